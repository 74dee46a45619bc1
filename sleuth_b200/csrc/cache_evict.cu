// Eviction from a cache of bounded size: of the rows that a sequence holds, `budget` stay.
//
// For every (sequence, kv head): n = lengths[s] rows; row j has gathered weights[j] and stands for the token at positions[j], or, for the rows
// of the last step (j >= past[s]), at seen[s] - (n - j). With n <= budget all stay. Otherwise those stay that come first by
//   (position < first or position >= seen - recent, before the others; then the larger weight, NaN last; then the lower row),
// and the rows that stay but lie at budget or behind move, in ascending order, into the places below budget of those that go, in ascending
// order: the least that has to be moved, and no place is read and written both. Rows of a cache are in no order of positions after that,
// which attention over all rows does not ask for.
//
// A block takes one (sequence, kv head). The order is one 32-bit key a row: the weight's bits made ascending, all ones for protected rows.
//   * Few rows go (a token or a short turn a step): the keys stay in registers, and the rows that go are taken out one after the other, each
//     a minimum over the block (the highest row among equals). The block moves the few rows itself.
//   * Many go (after a prompt): the keys lie in shared memory; a radix descent of 11, 11 and 10 bits finds the key of the last row that stays, and how
//     many of the rows with that very key stay (the lowest). Counts are whole numbers, so no order of threads matters. Rows are dealt to the threads in
//     runs, so that ranks are sums of a block-wide scan; the lists of places and rows go to scratch. The block, or where the rows are many a second
//     kernel, moves them, 16 threads a row.
// Bound by latency: loads, a descent, moves; the bytes are the weights and positions once and the moved rows twice. Measured: a row of 2,049 goes in each
// of 512 (sequence, kv head) pairs 7.6 us (17 MB, 2.3 TB/s; by the descent 37), of 16,000 in each of 32 pairs 11.5, of 16,386 18.8 and of 30,001 27.6 (32 keys a thread
// do not fit 64 registers: 504 bytes are spilled); 64 pairs of 2,500 to 8,192 rows come down to 1,024: the
// descent 15 us (18 with one row a thread in flight while the keys are made), the moves, 59 MB, 14 (4.2 TB/s; the same with four rows in flight a thread). 16 pairs of
// 40,000 rows to 3,000: 44 us, of 60,000: 114 (the keys do not fit shared memory and are made anew in every pass).
#include "common.cuh"

namespace slb {

constexpr int kEvictThreads = 1024;
constexpr int kFewGone = 16;       // rows that go one by one

struct EvictArgs {
  const float* weights;      // [slots, K, capacity]
  float* weights_out;
  const int* positions;
  int* positions_out;
  long long capacity;
  char* k_pool;
  char* v_pool;
  const int* block_table;
  const int* past;
  const int* lengths;
  const int* seen;
  const int* slots;
  int* scratch;              // with many moves: per (sequence, kv head) their number, the places, the rows
  int table_stride, n_seqs, kv_heads, row_bytes, budget, first, recent, max_length, keys_fit, most_moves, vector, moves_here;
};

__device__ __forceinline__ uint32_t order_key(float w, bool safe) {
  if (safe) return 0xffffffffu;
  if (w != w) return 0u;
  const uint32_t b = __float_as_uint(w + 0.0f);      // -0 counts as 0
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;   // between 0x007fffff (-inf) and 0xff800000 (inf)
}

// Exclusive sum over the block's threads of two counts packed in one word (each below 2^32), and the totals.
__device__ __forceinline__ unsigned long long block_scan(unsigned long long v, unsigned long long* warp_sums, unsigned long long& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned long long x = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const unsigned long long y = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    unsigned long long w = lane < (int)(blockDim.x >> 5) ? warp_sums[lane] : 0ull;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const unsigned long long y = __shfl_up_sync(0xffffffffu, w, d);
      if (lane >= d) w += y;
    }
    warp_sums[lane] = w;
  }
  __syncthreads();
  total = warp_sums[31];
  return x - v + (warp ? warp_sums[warp - 1] : 0ull);
}

__device__ __forceinline__ size_t pool_row(const EvictArgs& a, const int* table, int kh, int j) {
  return ((size_t)table[j / kPageTokens] * a.kv_heads + kh) * kPageTokens + j % kPageTokens;
}

// `lanes` threads copy one row of each pool.
__device__ __forceinline__ void move_row(const EvictArgs& a, const int* table, int kh, int to, int from, int lane, int lanes) {
  const size_t src = pool_row(a, table, kh, from) * a.row_bytes, dst = pool_row(a, table, kh, to) * a.row_bytes;
  if (a.vector) {
    for (int c = lane * 16; c < a.row_bytes; c += lanes * 16) {
      const uint4 k = *reinterpret_cast<const uint4*>(a.k_pool + src + c), v = *reinterpret_cast<const uint4*>(a.v_pool + src + c);
      *reinterpret_cast<uint4*>(a.k_pool + dst + c) = k;
      *reinterpret_cast<uint4*>(a.v_pool + dst + c) = v;
    }
  } else {
    for (int c = lane * 4; c < a.row_bytes; c += lanes * 4) {
      const uint32_t k = *reinterpret_cast<const uint32_t*>(a.k_pool + src + c), v = *reinterpret_cast<const uint32_t*>(a.v_pool + src + c);
      *reinterpret_cast<uint32_t*>(a.k_pool + dst + c) = k;
      *reinterpret_cast<uint32_t*>(a.v_pool + dst + c) = v;
    }
  }
}

// ---- few rows go ----
// THREADS threads with E keys each: row tid + e * THREADS.
template <int THREADS, int E>
__global__ void __launch_bounds__(THREADS) cache_evict_few_kernel(EvictArgs a) {
  pdl_enter();
  __shared__ unsigned long long mins[2][THREADS / 32];
  __shared__ int gone[kFewGone], to_s[kFewGone], from_s[kFewGone];
  __shared__ int s_moves;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, kh = blockIdx.x, seq = blockIdx.y;
  const size_t row0 = ((size_t)(a.slots ? a.slots[seq] : seq) * a.kv_heads + kh) * a.capacity;
  const float* weights = a.weights + row0;
  const int* positions = a.positions + row0;
  float* weights_out = a.weights_out + row0;
  int* positions_out = a.positions_out + row0;
  const int* table = a.block_table + (size_t)seq * a.table_stride;
  const int n = min(a.lengths[seq], a.max_length), past = min(a.past[seq], n), seen = a.seen[seq], left = min(n, a.budget);
  auto position = [&](int j) { return j < past ? positions[j] : seen - (n - j); };
  uint32_t key[E];
  {
    float w[E];
#pragma unroll
    for (int e = 0; e < E; ++e) w[e] = tid + e * THREADS < n ? weights[tid + e * THREADS] : 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int j = tid + e * THREADS, p = j < n ? position(j) : 0;
      key[e] = j < n ? order_key(w[e], p < a.first || p >= seen - a.recent) : 0xffffffffu;
    }
  }
  const int goes = n - left;           // 0 .. kFewGone
  uint32_t live = 0;                   // rows of this thread that stay so far
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (tid + e * THREADS < n) live |= 1u << e;
  // the least key of a thread, and its highest row: packed so that the smaller number goes first
  auto least = [&]() {
    unsigned long long best = ~0ull;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (live >> e & 1) {
        const unsigned long long v = (unsigned long long)key[e] << 32 | (uint32_t)~(tid + e * THREADS);
        best = v < best ? v : best;
      }
    return best;
  };
  unsigned long long mine = goes > 0 ? least() : 0ull;
  for (int g = 0; g < goes; ++g) {
    const uint32_t k = __reduce_min_sync(0xffffffffu, (uint32_t)(mine >> 32));
    const uint32_t r = __reduce_min_sync(0xffffffffu, (uint32_t)(mine >> 32) == k ? (uint32_t)mine : 0xffffffffu);
    if (lane == 0) mins[g & 1][warp] = (unsigned long long)k << 32 | r;
    __syncthreads();
    unsigned long long best = lane < THREADS / 32 ? mins[g & 1][lane] : ~0ull;
    const uint32_t bk = __reduce_min_sync(0xffffffffu, (uint32_t)(best >> 32));
    const uint32_t br = __reduce_min_sync(0xffffffffu, (uint32_t)(best >> 32) == bk ? (uint32_t)best : 0xffffffffu);
    const int row = (int)~br;
    if (tid == 0) gone[g] = row;
    if (row % THREADS == tid) {
      live &= ~(1u << (row / THREADS));
      mine = least();
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int j = tid + e * THREADS;
    if (j < left && (live >> e & 1)) {
      if (positions_out != positions || j >= past) positions_out[j] = position(j);
      if (weights_out != weights) weights_out[j] = weights[j];
    }
  }
  if (goes == 0) return;
  __syncthreads();
  if (warp == 0) {       // lane i: the i-th row that went, and the i-th row behind the budget
    const int out = lane < goes ? gone[lane] : 0x7fffffff, behind = left + lane;
    int rank = 0;
    bool stays = lane < goes;
#pragma unroll
    for (int i = 0; i < kFewGone; ++i) {
      const int o = __shfl_sync(0xffffffffu, out, i);
      rank += o < out;
      if (o == behind) stays = false;
    }
    const unsigned holes = __ballot_sync(0xffffffffu, out < left), movers = __ballot_sync(0xffffffffu, stays);
    if (out < left) to_s[rank] = out;          // (all rows below the budget come before those behind it)
    if (stays) from_s[__popc(movers & ((1u << lane) - 1))] = behind;
    if (lane == 0) s_moves = __popc(holes);
  }
  __syncthreads();
  const int moves = s_moves;
  if (tid < moves) {
    weights_out[to_s[tid]] = weights[from_s[tid]];
    positions_out[to_s[tid]] = position(from_s[tid]);
  }
  for (int i = tid >> 4; i < moves; i += THREADS / 16) move_row(a, table, kh, to_s[i], from_s[i], tid & 15, 16);
}

// ---- many rows go ----
template <int THREADS>
__global__ void __launch_bounds__(THREADS) cache_evict_kernel(EvictArgs a) {
  pdl_enter();
  extern __shared__ uint32_t keys[];
  __shared__ int hist[2048];
  __shared__ unsigned long long warp_sums[32];
  __shared__ uint32_t s_digit;
  __shared__ int s_need;
  const int tid = threadIdx.x, kh = blockIdx.x, seq = blockIdx.y;
  const size_t row0 = ((size_t)(a.slots ? a.slots[seq] : seq) * a.kv_heads + kh) * a.capacity;
  const float* weights = a.weights + row0;
  const int* positions = a.positions + row0;
  float* weights_out = a.weights_out + row0;
  int* positions_out = a.positions_out + row0;
  const int n = min(a.lengths[seq], a.max_length);
  const int past = min(a.past[seq], n), seen = a.seen[seq];
  const int left = min(n, a.budget);
  auto position = [&](int j) { return j < past ? positions[j] : seen - (n - j); };
  auto make_key = [&](int j) {
    const int p = position(j);
    return order_key(weights[j], p < a.first || p >= seen - a.recent);
  };
  const int* table = a.block_table + (size_t)seq * a.table_stride;
  int* lists = a.scratch ? a.scratch + ((size_t)seq * a.kv_heads + kh) * (2 * (size_t)a.most_moves + 1) : nullptr;
  if (n <= a.budget) {       // all stay (the whole block leaves)
    for (int j = tid; j < n; j += THREADS) {
      if (positions_out != positions || j >= past) positions_out[j] = position(j);
      if (weights_out != weights) weights_out[j] = weights[j];
    }
    if (lists && tid == 0) lists[0] = 0;
    return;
  }
#pragma unroll
  for (int i = 0; i < 2048 / THREADS; ++i) hist[tid + i * THREADS] = 0;
  __syncthreads();
  if (a.keys_fit) {
    // the keys and the counts of their first digit; kBatch rows a thread in flight (one after the other each would wait for the memory's answer)
    constexpr int kBatch = 8;
    for (int base = 0; base < n; base += kBatch * THREADS) {
      float w[kBatch];
      int p[kBatch];
#pragma unroll
      for (int e = 0; e < kBatch; ++e) {
        const int j = base + e * THREADS + tid;
        w[e] = j < n ? weights[j] : 0.0f;
        p[e] = j < past ? positions[j] : seen - (n - j);
      }
#pragma unroll
      for (int e = 0; e < kBatch; ++e) {
        const int j = base + e * THREADS + tid;
        const bool safe = p[e] < a.first || p[e] >= seen - a.recent;
        const uint32_t k = order_key(w[e], safe);
        const unsigned protect = __ballot_sync(0xffffffffu, safe && j < n);
        if (j < n) {
          keys[j] = k;
          if (!safe) atomicAdd(&hist[k >> 21], 1);
        }
        if (protect && (tid & 31) == 0) atomicAdd(&hist[2047], __popc(protect));      // (protected rows stand together: one addition a warp)
      }
    }
  }
  auto key_of = [&](int j) { return a.keys_fit ? keys[j] : make_key(j); };

  // the key of the last row that stays: digit by digit, the largest ones first
  uint32_t prefix = 0, mask = 0;
  int need = left;             // rows still to be chosen among those that agree with the prefix
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
    if (pass) {
#pragma unroll
      for (int i = 0; i < 2048 / THREADS; ++i) hist[tid + i * THREADS] = 0;
      __syncthreads();
    }
    if (pass || !a.keys_fit)
      for (int j = tid; j < n; j += THREADS) {
        const uint32_t k = key_of(j);
        if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & (bins - 1)], 1);
      }
    __syncthreads();
    // a thread a run of digits, the largest first: how many keys lie above them
    constexpr int RUN = 2048 / THREADS;
    int own = 0;
#pragma unroll
    for (int i = 0; i < RUN; ++i) own += hist[2047 - RUN * tid - i];
    unsigned long long all;
    int above = (int)block_scan((unsigned long long)own, warp_sums, all);
    if (above < need && above + own >= need) {
      int i = 0;
      for (; i < RUN - 1; ++i) {
        const int c = hist[2047 - RUN * tid - i];
        if (above + c >= need) break;
        above += c;
      }
      s_digit = (uint32_t)(2047 - RUN * tid - i);
      s_need = need - above;
    }
    __syncthreads();
    prefix |= s_digit << shift;
    mask |= (uint32_t)(bins - 1) << shift;
    need = s_need;
    __syncthreads();
  }
  const uint32_t last = prefix;

  // runs of rows a thread: an odd number, so that the threads of a warp meet different banks
  const int per = ((n + THREADS - 1) / THREADS) | 1, j0 = min(n, tid * per), j1 = min(n, j0 + per);
  unsigned long long ties = 0, total;
  for (int j = j0; j < j1; ++j) ties += key_of(j) == last;
  const int tie0 = (int)block_scan(ties, warp_sums, total);
  int tie = tie0;
  unsigned long long counts = 0;           // low word: places that become free below the budget; high word: rows that move
  for (int j = j0; j < j1; ++j) {
    const uint32_t k = key_of(j);
    const bool stays = k > last || (k == last && tie < need);
    tie += k == last;
    if (j < left) counts += !stays;
    else if (stays) counts += 1ull << 32;
  }
  const unsigned long long before = block_scan(counts, warp_sums, total);
  const int moves = (int)(total >> 32);
  int hole = (int)(before & 0xffffffffu), mover = (int)(before >> 32);
  tie = tie0;
  for (int j = j0; j < j1; ++j) {
    const uint32_t k = key_of(j);
    const bool stays = k > last || (k == last && tie < need);
    tie += k == last;
    if (j < left && !stays) lists[1 + hole++] = j;
    if (j >= left && stays) lists[1 + a.most_moves + mover++] = j;
    if (a.keys_fit) keys[j] = stays;      // (a row of this thread's own run)
    else if (j < left && stays) {
      if (positions_out != positions || j >= past) positions_out[j] = position(j);
      if (weights_out != weights) weights_out[j] = weights[j];
    }
  }
  if (tid == 0) lists[0] = moves;
  __syncthreads();
  // what stays in its place, a warp whole lines (in the loop above each copy would wait for the one before)
  if (a.keys_fit && (positions_out != positions || weights_out != weights || past < left))
#pragma unroll 4
    for (int j = tid; j < left; j += THREADS) {
      if (!keys[j]) continue;
      const float w = weights[j];
      const int p = position(j);
      if (positions_out != positions || j >= past) positions_out[j] = p;
      if (weights_out != weights) weights_out[j] = w;
    }
  for (int i = tid; i < moves; i += THREADS) {      // (the block's own stores are visible to it after the barrier)
    const int to = lists[1 + i], from = lists[1 + a.most_moves + i];
    weights_out[to] = weights[from];
    positions_out[to] = position(from);
  }
  if (a.moves_here)
    for (int i = tid >> 4; i < moves; i += THREADS / 16) move_row(a, table, kh, lists[1 + i], lists[1 + a.most_moves + i], tid & 15, 16);
}

// The moves of the lists: 16 threads a row of each pool.
__global__ void __launch_bounds__(256) cache_move_kernel(EvictArgs a) {
  pdl_enter();
  const int kh = blockIdx.y, seq = blockIdx.z;
  const int* lists = a.scratch + ((size_t)seq * a.kv_heads + kh) * (2 * (size_t)a.most_moves + 1);
  const int* table = a.block_table + (size_t)seq * a.table_stride;
  const int moves = lists[0];
  for (int i = blockIdx.x * 16 + (threadIdx.x >> 4); i < moves; i += gridDim.x * 16)
    move_row(a, table, kh, lists[1 + i], lists[1 + a.most_moves + i], threadIdx.x & 15, 16);
}

static int most_moves(int budget, int max_length) {
  const int behind = max_length - budget;
  return behind <= 0 ? 0 : behind < budget ? behind : budget;
}

constexpr int kMostKeysShared = 48 * 1024;      // 192 KB of keys

// Whether no sequence loses more rows than the kernel for that takes, nor holds more than its registers do.
static bool few_go(int budget, int max_length) { return max_length - budget <= kFewGone && max_length <= 32 * 1024; }

static int launch_evict_few(const EvictArgs& a, cudaStream_t s) {
  const dim3 grid(a.kv_heads, a.n_seqs);
  // a block of 256 threads up to 16 keys each, so that several share an SM; 1,024 beyond
  if (a.max_length <= 256 * 4) launch(cache_evict_few_kernel<256, 4>, grid, dim3(256), 0, s, a);
  else if (a.max_length <= 256 * 10) launch(cache_evict_few_kernel<256, 10>, grid, dim3(256), 0, s, a);
  else if (a.max_length <= 512 * 10) launch(cache_evict_few_kernel<512, 10>, grid, dim3(512), 0, s, a);
  else if (a.max_length <= 1024 * 10) launch(cache_evict_few_kernel<1024, 10>, grid, dim3(1024), 0, s, a);
  else if (a.max_length <= 1024 * 16) launch(cache_evict_few_kernel<1024, 16>, grid, dim3(1024), 0, s, a);
  else launch(cache_evict_few_kernel<1024, 32>, grid, dim3(1024), 0, s, a);
  return check_launch("cache_evict (few rows)");
}

}  // namespace slb

using namespace slb;

// 32-bit words of scratch that slb_cache_evict takes: the lists of moves, where a sequence may move more rows than a block does by itself.
extern "C" long long slb_cache_evict_scratch(int n_seqs, int kv_heads, int budget, int max_length) {
  const int moves = most_moves(budget, max_length);
  if (n_seqs <= 0 || kv_heads <= 0 || few_go(budget, max_length)) return 0;
  return (long long)n_seqs * kv_heads * (2ll * moves + 1);
}

// What a caller says, in one piece of memory (as KeptCall, kept.cuh).
struct EvictCall {
  const float* weights;                 // [slots, kv_heads, capacity]; a target may be its source
  float* weights_out;
  const int* positions;
  int* positions_out;
  void *k_pool, *v_pool;                // [pages, kv_heads, 64, row_bytes]
  const int *block_table, *past, *lengths, *seen, *slots;
  int* scratch;
  void* stream;
  long long capacity, scratch_words;
  int table_stride, n_seqs, kv_heads, row_bytes, budget, first, recent, max_length;
};
static_assert(sizeof(EvictCall) == 13 * 8 + 2 * 8 + 8 * 4, "as packed in kernels/ops.py");

// See the head of the file. max_length: no sequence holds more rows (0: as many as its table takes).
extern "C" int slb_cache_evict(const EvictCall* call) {
  SLB_REQUIRE(call != nullptr, "cache_evict: no call");
  const EvictCall c = *call;
  const int table_stride = c.table_stride, n_seqs = c.n_seqs, kv_heads = c.kv_heads, row_bytes = c.row_bytes, budget = c.budget, first = c.first, recent = c.recent;
  const long long capacity = c.capacity;
  int max_length = c.max_length;
  SLB_REQUIRE(n_seqs >= 0 && kv_heads > 0 && row_bytes > 0 && row_bytes % 4 == 0 && table_stride > 0 && capacity > 0 && n_seqs < 65536 && kv_heads < 65536,
              "cache_evict: n_seqs=%d kv_heads=%d row_bytes=%d table_stride=%d", n_seqs, kv_heads, row_bytes, table_stride);
  SLB_REQUIRE(budget > 0 && first >= 0 && recent >= 0 && (long long)first + recent <= budget,
              "cache_evict: %d first and %d recent rows do not fit a budget of %d", first, recent, budget);
  if (n_seqs == 0) return 0;
  const long long table_rows = (long long)table_stride * kPageTokens;
  if (max_length <= 0 || max_length > table_rows) max_length = (int)(table_rows < 0x7fffffffll ? table_rows : 0x7fffffffll);
  SLB_REQUIRE(capacity >= max_length, "cache_evict: weights and positions of %lld rows are shorter than the cache (%d)", capacity, max_length);
  const long long need = slb_cache_evict_scratch(n_seqs, kv_heads, budget, max_length);
  SLB_REQUIRE(need == 0 || (c.scratch != nullptr && c.scratch_words >= need), "cache_evict: the step needs %lld words of scratch, %lld were given", need,
              c.scratch ? c.scratch_words : 0ll);
  EvictArgs a{};
  a.weights = c.weights; a.weights_out = c.weights_out; a.positions = c.positions; a.positions_out = c.positions_out; a.capacity = capacity;
  a.k_pool = (char*)c.k_pool; a.v_pool = (char*)c.v_pool; a.block_table = c.block_table; a.past = c.past; a.lengths = c.lengths; a.seen = c.seen;
  a.slots = c.slots; a.scratch = need ? c.scratch : nullptr; a.table_stride = table_stride; a.n_seqs = n_seqs; a.kv_heads = kv_heads;
  a.row_bytes = row_bytes; a.budget = budget; a.first = first; a.recent = recent; a.max_length = max_length;
  a.most_moves = most_moves(budget, max_length);
  a.keys_fit = max_length <= kMostKeysShared;
  a.vector = row_bytes % 16 == 0 && (uintptr_t)c.k_pool % 16 == 0 && (uintptr_t)c.v_pool % 16 == 0;
  if (few_go(budget, max_length)) return launch_evict_few(a, (cudaStream_t)c.stream);
  const int smem = a.keys_fit ? max_length * 4 : 0;
  static std::atomic<unsigned long long> allowed;
  // few moves are made by the block that found them: a second kernel costs 3 us, 64 rows of 512 bytes a block less than one
  a.moves_here = a.most_moves * (long long)row_bytes <= 32 * 1024;
  if (max_length <= 2048) {      // small blocks, so that many share an SM
    launch(cache_evict_kernel<256>, dim3(kv_heads, n_seqs), dim3(256), smem, (cudaStream_t)c.stream, a);
  } else {
    const cudaError_t e = allow_shared((const void*)cache_evict_kernel<kEvictThreads>, kMostKeysShared * 4, allowed);
    if (e != cudaSuccess) return fail(2, "cache_evict: cannot reserve shared memory: %s", cudaGetErrorString(e));
    launch(cache_evict_kernel<kEvictThreads>, dim3(kv_heads, n_seqs), dim3(kEvictThreads), smem, (cudaStream_t)c.stream, a);
  }
  const int rc = check_launch("cache_evict");
  if (rc || a.moves_here) return rc;
  const long long pairs = (long long)n_seqs * kv_heads;
  long long blocks = 8ll * sm_count() / pairs;
  const long long most = (a.most_moves + 15) / 16;
  blocks = blocks < 1 ? 1 : blocks < most ? blocks : most;
  launch_prefetching(cache_move_kernel, dim3((unsigned)blocks, kv_heads, n_seqs), dim3(256), 0, (cudaStream_t)c.stream, a);
  return check_launch("cache_evict (moves)");
}
