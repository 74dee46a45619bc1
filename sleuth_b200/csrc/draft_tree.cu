// The tables of a step of drafted tokens, and the cache after it.
//
// slb_draft_tree: parents -> what each node sees of its step and its position. slb_cache_compact: the rows of the nodes that stay move
// together behind the rows from before the step.
#include "tree.cuh"

namespace slb {

// ---- what a node sees ----
// A node's way is itself and the nodes that it continues. Ways of up to 2^k nodes, A_k(i), and the node 2^k steps up, J_k(i), come by doubling:
//   A_{k+1}(i) = A_k(i) u A_k(J_k(i)),   J_{k+1}(i) = J_k(J_k(i)),
// eight rounds for 256 nodes, where walking up a chain would take 256 dependent reads. Under a window of w positions a node sees the first w nodes of its
// way: the union of A_k over the binary digits of w, each from where the digit before ended. Depth: nodes on the whole way, less one.
// All latency: a block a sequence, a thread a node, ways of 256 bits in registers and shared memory. One B200, device: one tree of 8 nodes 1.7 us, 64 of 17 to 250
// nodes 3.9; a call takes the host 7.
struct DraftTreeArgs {
  const int *parents, *seq_start, *past, *counts;
  uint32_t* seen;
  int* positions;
  long long tokens;
  int n_seqs, max_count, words, window;
};

template <int W>      // words of a way: 1, 2, 4 or 8
__global__ void __launch_bounds__(kMostNodes) draft_tree_kernel(DraftTreeArgs a) {
  pdl_enter();
  __shared__ uint32_t way_s[W * 32][W + (W > 1)];
  __shared__ int up_s[W * 32];
  const int i = threadIdx.x, seq = blockIdx.x;
  const int count = min(max(a.counts[seq], 0), a.max_count), tok0 = a.seq_start[seq];
  const bool real = i < count && tok0 >= 0 && (long long)tok0 + i < a.tokens;
  uint32_t way[W], seen[W];
  int up = -1, cur = i;       // cur: the node where the window's next digit begins, -1 behind the way's end
  if (real) {
    const int p = a.parents[tok0 + i];
    up = p >= 0 && p < i ? p : -1;
  }
#pragma unroll
  for (int w = 0; w < W; ++w) {
    way[w] = i >> 5 == w ? 1u << (i & 31) : 0u;
    seen[w] = 0u;
  }
  const int limit = a.window > 0 && a.window < W * 32 ? a.window : W * 32;
#pragma unroll 1
  for (int k = 0; 1 << k <= W * 32; ++k) {
#pragma unroll
    for (int w = 0; w < W; ++w) way_s[i][w] = way[w];
    up_s[i] = up;
    __syncthreads();
    if (limit >> k & 1 && cur >= 0) {
#pragma unroll
      for (int w = 0; w < W; ++w) seen[w] |= way_s[cur][w];
      cur = up_s[cur];
    }
    if (up >= 0) {
#pragma unroll
      for (int w = 0; w < W; ++w) way[w] |= way_s[up][w];
      up = up_s[up];
    }
    __syncthreads();
  }
  if (!real) return;
  int depth = -1;
#pragma unroll
  for (int w = 0; w < W; ++w) depth += __popc(way[w]);
  const size_t token = (size_t)tok0 + i;
#pragma unroll
  for (int w = 0; w < W; ++w)
    if (w < a.words) a.seen[token * a.words + w] = seen[w];
  for (int w = W; w < a.words; ++w) a.seen[token * a.words + w] = 0u;
  a.positions[token] = a.past[seq] + depth;
}

// What a caller says, in one piece of memory (as KeptCall, kept.cuh).
struct DraftTreeCall {
  const int *parents, *seq_start, *past, *counts;
  void* seen;
  int* positions;
  void* stream;
  long long tokens;
  int n_seqs, max_count, words, window;
};
static_assert(sizeof(DraftTreeCall) == 7 * 8 + 8 + 4 * 4, "as packed in kernels/ops.py");

extern "C" int slb_draft_tree(const DraftTreeCall* call) {
  SLB_REQUIRE(call != nullptr, "draft_tree: no call");
  const DraftTreeCall c = *call;
  const int n_seqs = c.n_seqs, max_count = c.max_count, words = c.words, window = c.window;
  const long long tokens = c.tokens;
  SLB_REQUIRE(n_seqs >= 0 && tokens >= 0 && window >= 0, "draft_tree: n_seqs=%d tokens=%lld window=%d", n_seqs, tokens, window);
  SLB_REQUIRE(max_count > 0 && max_count <= kMostNodes, "draft_tree: %d nodes of a sequence; 1 to %d are taken", max_count, kMostNodes);
  SLB_REQUIRE(words >= 1 && (long long)words * 32 >= max_count, "draft_tree: %d words of bits do not hold %d nodes", words, max_count);
  if (n_seqs == 0 || tokens == 0) return 0;
  const DraftTreeArgs a{c.parents, c.seq_start, c.past, c.counts, (uint32_t*)c.seen, c.positions, tokens, n_seqs, max_count, words, window};
  const cudaStream_t s = (cudaStream_t)c.stream;
  if (max_count <= 32) launch(draft_tree_kernel<1>, dim3(n_seqs), dim3(32), 0, s, a);
  else if (max_count <= 64) launch(draft_tree_kernel<2>, dim3(n_seqs), dim3(64), 0, s, a);
  else if (max_count <= 128) launch(draft_tree_kernel<4>, dim3(n_seqs), dim3(128), 0, s, a);
  else launch(draft_tree_kernel<8>, dim3(n_seqs), dim3(256), 0, s, a);
  return check_launch("draft_tree");
}

// ---- the cache after the step ----
// For every sequence, layer and kv head, for i = 0 .. lengths - 1 in this order: row past + i <- row past + path[i]. path rises, so path[i] >= i: a row
// that is written is never read afterwards, and a thread that takes the same 16 bytes of all rows, eight reads before eight writes, needs no barrier.
// All layers in one launch: a step's compaction is a few rows of each, 2 KB of a layer and row at 8 heads of 128. One B200, device: 28 layers of 8 heads of 128, one
// sequence with up to four rows 2.6 us, 24 sequences with up to seven 4.9 (12 MB read and written, in L2 mostly): three dependent reads (table, path, row) and the
// launch, and the host has 7.4 us a call.
struct CompactArgs {
  char *k_pool, *v_pool;                  // [layers, pages, kv_heads, 64, bytes]
  const int *block_table, *past, *path, *lengths;
  long long k_layer, v_layer;             // bytes of a layer
  long long k_pieces, pieces;             // (layer, kv head, piece) of the keys, and of keys and values
  int table_stride, kv_heads, k_row, v_row, path_width;      // bytes of a row
  long long pages;
};

constexpr int kCompactThreads = 256;

template <typename V>      // a piece: 16 or 4 bytes
__global__ void __launch_bounds__(kCompactThreads) cache_compact_kernel(CompactArgs a) {
  pdl_enter();
  __shared__ int from_s[kMostNodes];
  __shared__ int s_len;
  const int tid = threadIdx.x, seq = blockIdx.y, past = a.past[seq];
  const int* path = a.path + (size_t)seq * a.path_width;
  const int most = min(min(a.lengths[seq], a.path_width), kMostNodes);
  const long long rows = (long long)a.table_stride * kPageTokens;
  if (tid == 0) s_len = max(most, 0);
  __syncthreads();
  if (tid < most) {
    const int p = path[tid], before = tid ? path[tid - 1] : -1;
    from_s[tid] = p;
    bool good = p > before && p >= 0 && past >= 0 && (long long)past + p < rows;
    if (good) {
      const int* table = a.block_table + (size_t)seq * a.table_stride;
      const int from = table[(past + p) / kPageTokens], to = table[(past + tid) / kPageTokens];
      good = from >= 0 && from < a.pages && to >= 0 && to < a.pages;
    }
    if (!good) atomicMin(&s_len, tid);      // the path ends in front of it
  }
  __syncthreads();
  const int len = s_len;
  int first = 0;
  while (first < len && from_s[first] == first) ++first;      // rows that lie in place
  if (first >= len) return;
  const long long piece = (long long)blockIdx.x * kCompactThreads + tid;
  if (piece >= a.pieces) return;
  const bool value = piece >= a.k_pieces;
  const long long p = value ? piece - a.k_pieces : piece;
  const int row_bytes = value ? a.v_row : a.k_row, per = row_bytes / (int)sizeof(V);
  const int off = (int)(p % per), kh = (int)(p / per % a.kv_heads);
  char* pool = (value ? a.v_pool : a.k_pool) + p / per / a.kv_heads * (value ? a.v_layer : a.k_layer);
  const int* table = a.block_table + (size_t)seq * a.table_stride;
  auto at = [&](int i) {
    const int row = past + i;
    return reinterpret_cast<V*>(pool + (((long long)table[row / kPageTokens] * a.kv_heads + kh) * kPageTokens + row % kPageTokens) * row_bytes) + off;
  };
  for (int i0 = first; i0 < len; i0 += 8) {
    V v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i0 + i < len) v[i] = *at(from_s[i0 + i]);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i0 + i < len) *at(i0 + i) = v[i];
  }
}

struct CompactCall {
  void *k_pool, *v_pool;                 // [layers, pages, kv_heads, 64, k_row]; [v_layers, pages, kv_heads, 64, v_row] or null
  const int *block_table, *past, *path, *lengths;
  void* stream;
  long long layers, v_layers, pages;
  int table_stride, n_seqs, kv_heads, k_row, v_row, path_width;      // bytes of a row
};
static_assert(sizeof(CompactCall) == 7 * 8 + 3 * 8 + 6 * 4, "as packed in kernels/ops.py");

extern "C" int slb_cache_compact(const CompactCall* call) {
  SLB_REQUIRE(call != nullptr, "cache_compact: no call");
  const CompactCall c = *call;
  void *k_pool = c.k_pool, *v_pool = c.v_pool;
  const long long layers = c.layers, v_layers = c.v_layers, pages = c.pages;
  const int table_stride = c.table_stride, n_seqs = c.n_seqs, kv_heads = c.kv_heads, k_row = c.k_row, v_row = c.v_row, path_width = c.path_width;
  SLB_REQUIRE(n_seqs >= 0 && n_seqs < 65536 && layers >= 0 && v_layers >= 0 && pages > 0 && table_stride > 0 && kv_heads > 0 && path_width > 0,
              "cache_compact: n_seqs=%d layers=%lld pages=%lld table_stride=%d kv_heads=%d path_width=%d", n_seqs, layers, pages, table_stride, kv_heads, path_width);
  SLB_REQUIRE(path_width <= kMostNodes, "cache_compact: paths of %d nodes; at most %d are taken", path_width, kMostNodes);
  SLB_REQUIRE(k_row > 0 && k_row % 4 == 0 && v_row >= 0 && v_row % 4 == 0, "cache_compact: a row's bytes (%d, %d) are a multiple of four", k_row, v_row);
  SLB_REQUIRE((uintptr_t)k_pool % 4 == 0 && (uintptr_t)v_pool % 4 == 0, "cache_compact: pools must be 4-byte aligned");
  SLB_REQUIRE((long long)table_stride * kPageTokens < (1ll << 31) - kMostNodes, "cache_compact: a block table of %d pages is too long", table_stride);
  if (n_seqs == 0 || layers + v_layers == 0) return 0;
  CompactArgs a{};
  a.k_pool = (char*)k_pool; a.v_pool = (char*)v_pool; a.block_table = c.block_table; a.past = c.past; a.path = c.path; a.lengths = c.lengths;
  a.pages = pages;
  a.table_stride = table_stride; a.kv_heads = kv_heads; a.k_row = k_row; a.v_row = v_row; a.path_width = path_width;
  a.k_layer = pages * kv_heads * kPageTokens * k_row;
  a.v_layer = pages * kv_heads * kPageTokens * v_row;
  const bool wide = k_row % 16 == 0 && v_row % 16 == 0 && (uintptr_t)k_pool % 16 == 0 && (uintptr_t)v_pool % 16 == 0;
  const int piece = wide ? 16 : 4;
  a.k_pieces = layers * kv_heads * (k_row / piece);
  a.pieces = a.k_pieces + v_layers * kv_heads * (v_row / piece);
  const long long blocks = (a.pieces + kCompactThreads - 1) / kCompactThreads;
  SLB_REQUIRE(blocks < (1ll << 31), "cache_compact: too many layers for one launch");
  if (wide) launch(cache_compact_kernel<uint4>, dim3((unsigned)blocks, n_seqs), dim3(kCompactThreads), 0, (cudaStream_t)c.stream, a);
  else launch(cache_compact_kernel<uint32_t>, dim3((unsigned)blocks, n_seqs), dim3(kCompactThreads), 0, (cudaStream_t)c.stream, a);
  return check_launch("cache_compact");
}

}  // namespace slb
