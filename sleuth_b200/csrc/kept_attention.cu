// Attention over a cache of bounded size (kept.cuh), and the weights that its rows gather: the general kernels, for both dtypes, every
// even head size up to 256 and any number of new tokens.
//
//   out = sum_j softmax_j(scale q . k_j) v_j over the rows j that the query sees,   lse = log sum_j exp(scale q . k_j)
//   weights_out[j] = (weights[j] where row j was there before the step, else 0) + sum over the step's queries, and over the query heads
//                    of the key/value head, of exp(scale q . k_j - lse)
//
// A block of the first kernel takes 16 rows (row r is token r / G, query head r % G of the group) of one (sequence, kv head) and a share
// of the keys that some of them sees, 64 at a time: keys as float32 in shared memory, a thread a key and four rows; one pass with a running
// maximum and sum per row; values the same way, a thread four channels. Rows that are seen come in two runs, the first ones and the
// window; keys between them are not read. Shares are joined by a second kernel, in order. A key that a row does not see is left out of its sum,
// not multiplied by zero, so what lies in such a row of the pool (infinities, NaN) never reaches it.
// The weights need the finished denominators, so their kernel forms the scores again: a block takes 64 keys of one (sequence, kv head)
// and walks over the rows that see some of them, a thread a key; every sum has one order, and no two blocks add to the same place.
// Bound by the FMA pipe and shared memory.
#include <math.h>

#include "kept.cuh"

namespace slb {

constexpr int kGenThreads = 256, kGenRows = 16, kGenKeys = 64, kGenWeightRows = 64;

__host__ __device__ constexpr int padded_dim(int hd) { return (hd + 3) & ~3; }

// The virtual order of the keys that a tile sees: the first ones that lie before the window, then the window's rows up to `hi`.
struct KeyRun {
  int nf, lo, total;
  __device__ __forceinline__ KeyRun(int pos_first, int pos_last, int window, int first) {
    lo = window_lo(pos_first, window);
    nf = min(first, lo);
    total = nf + pos_last - lo + 1;
  }
  __device__ __forceinline__ int key(int v) const { return v < nf ? v : lo + v - nf; }
};

// 64 rows of a pool as float32 in shared memory, rows of hdp + 4 floats (16-byte reads of 8 lanes then meet 32 banks). Rows beyond the
// run are zeros.
template <typename T>
__device__ __forceinline__ void load_rows(float* dst, const T* pool, const KeptArgs& a, const int* table, int kh, const KeyRun& run, int v0, int v1) {
  const int hd = a.head_dim, hdp = padded_dim(hd);
  for (int e = threadIdx.x; e < kGenKeys * (hdp / 2); e += kGenThreads) {
    const int r = e / (hdp / 2), c = (e - r * (hdp / 2)) * 2;
    float x = 0.0f, y = 0.0f;
    if (v0 + r < v1 && c < hd) {
      const int key = run.key(v0 + r);
      const size_t row = ((size_t)table[key / kPageTokens] * a.kv_heads + kh) * kPageTokens + key % kPageTokens;
      const T* src = pool + row * hd + c;
      if constexpr (sizeof(T) == 4) {
        const float2 p = *reinterpret_cast<const float2*>(src);
        x = p.x;
        y = p.y;
      } else {
        const float2 p = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(src));
        x = p.x;
        y = p.y;
      }
    }
    *reinterpret_cast<float2*>(dst + r * (hdp + 4) + c) = make_float2(x, y);
  }
}

// ROWS rows of queries, times the scale, zeros behind the last row.
template <typename T, int ROWS>
__device__ __forceinline__ void load_queries(float* dst, const KeptArgs& a, size_t token0, int kh, int G, int r0, int rows_total) {
  const int hd = a.head_dim, hdp = padded_dim(hd);
  for (int e = threadIdx.x; e < ROWS * hdp; e += kGenThreads) {
    const int r = e / hdp, c = e - r * hdp, R = r0 + r;
    float v = 0.0f;
    if (R < rows_total && c < hd) v = to_f32(((const T*)a.q)[((token0 + R / G) * a.heads + kh * G + R % G) * hd + c]) * a.scale;
    dst[e] = v;
  }
}

__device__ __forceinline__ void dots(const float* krow, const float* q4, int hdp, float (&s)[4]) {
  s[0] = s[1] = s[2] = s[3] = 0.0f;
  for (int c = 0; c < hdp; c += 4) {
    const float4 k = *reinterpret_cast<const float4*>(krow + c);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 q = *reinterpret_cast<const float4*>(q4 + i * hdp + c);
      s[i] = fmaf(q.x, k.x, s[i]);
      s[i] = fmaf(q.y, k.y, s[i]);
      s[i] = fmaf(q.z, k.z, s[i]);
      s[i] = fmaf(q.w, k.w, s[i]);
    }
  }
}

__host__ __device__ constexpr int general_smem(int hd) { return (kGenKeys * (padded_dim(hd) + 4) + kGenRows * padded_dim(hd) + kGenRows * kGenKeys + 2 * kGenRows) * 4; }

// Scratch of a share: per (share, token, head) hd weighted values, maximum, sum.
__device__ __forceinline__ float* share_slot(const KeptArgs& a, int split, size_t token, int head, size_t tokens) {
  return a.scratch + (((size_t)split * tokens + token) * a.heads + head) * (a.head_dim + 2);
}

// RPT: rows a thread of the weighted sum, by how many groups of threads four channels each leave.
template <typename T, int RPT>
__global__ void __launch_bounds__(kGenThreads) kept_general_kernel(KeptArgs a, long long tokens) {
  pdl_enter();
  extern __shared__ __align__(16) float smem[];
  const int hd = a.head_dim, hdp = padded_dim(hd);
  float* rows_s = smem;                                  // [64][hdp + 4]
  float* q_s = rows_s + kGenKeys * (hdp + 4);            // [16][hdp]
  float* p_s = q_s + kGenRows * hdp;                     // [16][64]
  float* alpha_s = p_s + kGenRows * kGenKeys;            // [16]
  float* l_s = alpha_s + kGenRows;                       // [16]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int seq = blockIdx.z, kh = blockIdx.y, G = a.heads / a.kv_heads;
  const int tile = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
  const int count = a.counts[seq], past = a.past[seq], rows_total = count * G, r0 = tile * kGenRows;
  if (r0 >= rows_total) return;
  const size_t token0 = a.seq_start[seq];
  const int* table = a.block_table + (size_t)seq * a.table_stride;
  const int pos_first = past + r0 / G, pos_last = past + min(rows_total - 1, r0 + kGenRows - 1) / G;
  const KeyRun run(pos_first, pos_last, a.window, a.first);
  const int steps = (run.total + kGenKeys - 1) / kGenKeys, per = (steps + a.splits - 1) / a.splits;
  const int v_begin = split * per * kGenKeys, v_end = min(run.total, v_begin + per * kGenKeys);

  load_queries<T, kGenRows>(q_s, a, token0, kh, G, r0, rows_total);
  const int key_i = tid & 63, rg = tid >> 6;             // scores: a key, rows 4 rg .. 4 rg + 3
  int row_pos[4], row_lo[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int R = r0 + 4 * rg + i;
    row_pos[i] = R < rows_total ? past + R / G : -1;
    row_lo[i] = window_lo(row_pos[i], a.window);
  }
  const int quads = hdp / 4, groups = kGenThreads / quads;
  const int quad = tid % quads, group = tid / quads;     // weighted sum: channels 4 quad .., rows group, group + groups, ...
  const bool sums = group < groups;
  float acc[RPT][4];
#pragma unroll
  for (int i = 0; i < RPT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.0f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};      // rows 2 warp, 2 warp + 1
  for (int v0 = v_begin; v0 < v_end; v0 += kGenKeys) {
    __syncthreads();
    load_rows<T>(rows_s, (const T*)a.k_pool, a, table, kh, run, v0, v_end);
    __syncthreads();
    {
      float s[4];
      dots(rows_s + key_i * (hdp + 4), q_s + 4 * rg * hdp, hdp, s);
      const int key = run.key(v0 + key_i);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        p_s[(4 * rg + i) * kGenKeys + key_i] = v0 + key_i < v_end && sees(key, row_pos[i], row_lo[i], a.first) ? s[i] : -INFINITY;
    }
    __syncthreads();
    load_rows<T>(rows_s, (const T*)a.v_pool, a, table, kh, run, v0, v_end);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float* row = p_s + (2 * warp + i) * kGenKeys;
      const float x0 = row[lane], x1 = row[lane + 32];
      const float m_new = fmaxf(m[i], warp_max(fmaxf(x0, x1))), top = m_new == -INFINITY ? 0.0f : m_new;
      const float p0 = expf(x0 - top), p1 = expf(x1 - top), alpha = expf(m[i] - top);
      row[lane] = p0;
      row[lane + 32] = p1;
      l[i] = l[i] * alpha + warp_sum(p0 + p1);
      m[i] = m_new;
      if (lane == 0) alpha_s[2 * warp + i] = alpha;
    }
    __syncthreads();
    if (sums) {
#pragma unroll
      for (int i = 0; i < RPT; ++i) {
        const float f = alpha_s[min(group + i * groups, kGenRows - 1)];
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[i][c] *= f;
      }
      const int n = min(kGenKeys, v_end - v0);
      for (int j = 0; j < n; ++j) {
        const float4 v = *reinterpret_cast<const float4*>(rows_s + j * (hdp + 4) + 4 * quad);
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
          const float p = p_s[min(group + i * groups, kGenRows - 1) * kGenKeys + j];
          if (p != 0.0f) {
            acc[i][0] = fmaf(p, v.x, acc[i][0]);
            acc[i][1] = fmaf(p, v.y, acc[i][1]);
            acc[i][2] = fmaf(p, v.z, acc[i][2]);
            acc[i][3] = fmaf(p, v.w, acc[i][3]);
          }
        }
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int R = r0 + 2 * warp + i;
    if (lane == 0) {
      l_s[2 * warp + i] = l[i];
      if (R < rows_total) {
        const size_t token = token0 + R / G;
        const int head = kh * G + R % G;
        if (a.splits > 1) {
          float* slot = share_slot(a, split, token, head, tokens);
          slot[hd] = m[i];
          slot[hd + 1] = l[i];
        } else if (a.lse) {
          a.lse[token * a.heads + head] = l[i] == 0.0f ? -INFINITY : m[i] + logf(l[i]);
        }
      }
    }
  }
  __syncthreads();
  if (!sums) return;
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int r = group + i * groups, R = r0 + r;
    if (r >= kGenRows || R >= rows_total) continue;
    const size_t token = token0 + R / G;
    const int head = kh * G + R % G;
    const float inv = a.splits > 1 ? 1.0f : l_s[r] == 0.0f ? 0.0f : 1.0f / l_s[r];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if (4 * quad + c >= hd) continue;
      if (a.splits > 1) share_slot(a, split, token, head, tokens)[4 * quad + c] = acc[i][c];
      else ((T*)a.out)[(token * a.heads + head) * hd + 4 * quad + c] = from_f32<T>(acc[i][c] * inv);
    }
  }
}

// The shares of one (token, head), in order; a thread a channel.
template <typename T>
__global__ void kept_join_kernel(KeptArgs a, long long tokens) {
  pdl_enter();
  const int head = blockIdx.x, c = threadIdx.x, hd = a.head_dim;
  const size_t token = blockIdx.y + (size_t)blockIdx.z * 65535;
  if (token >= (size_t)tokens) return;
  float M = -INFINITY, L = 0.0f, o = 0.0f;
  for (int s = 0; s < a.splits; ++s) {
    const float* slot = share_slot(a, s, token, head, tokens);
    const float m = slot[hd], l = slot[hd + 1], v = c < hd ? slot[c] : 0.0f;
    const float m_new = fmaxf(M, m), top = m_new == -INFINITY ? 0.0f : m_new;
    const float fa = expf(M - top), fb = expf(m - top);
    L = L * fa + l * fb;
    o = o * fa + v * fb;
    M = m_new;
  }
  if (c < hd) ((T*)a.out)[(token * a.heads + head) * hd + c] = from_f32<T>(L == 0.0f ? 0.0f : o / L);
  if (c == 0 && a.lse) a.lse[token * a.heads + head] = L == 0.0f ? -INFINITY : M + logf(L);
}

__host__ __device__ constexpr int weights_smem(int hd) { return (kGenKeys * (padded_dim(hd) + 4) + kGenWeightRows * (padded_dim(hd) + 1) + kGenThreads) * 4; }

template <typename T>
__global__ void __launch_bounds__(kGenThreads) kept_weights_general_kernel(KeptArgs a) {
  pdl_enter();
  extern __shared__ __align__(16) float smem[];
  const int hd = a.head_dim, hdp = padded_dim(hd);
  float* rows_s = smem;                                  // [64][hdp + 4]
  float* q_s = rows_s + kGenKeys * (hdp + 4);            // [64][hdp]
  float* lse_s = q_s + kGenWeightRows * hdp;             // [64]
  float* part_s = lse_s + kGenWeightRows;                // [4][64]
  const int tid = threadIdx.x, key_i = tid & 63, rg = tid >> 6;
  const int seq = blockIdx.z, kh = blockIdx.y, G = a.heads / a.kv_heads;
  const int count = a.counts[seq], past = a.past[seq], end = past + count;
  const int key0 = blockIdx.x * kGenKeys, key = key0 + key_i;
  if (count <= 0 || key0 >= end) return;
  const size_t token0 = a.seq_start[seq];
  const int* table = a.block_table + (size_t)seq * a.table_stride;
  // the queries that see some key of the tile: from the tile's own rows on, and while the window reaches back to it (or all of them)
  const int last = min(end, key0 + kGenKeys) - 1;
  const int t_lo = max(0, key0 - past);
  const int t_hi = a.window > 0 && key0 >= a.first ? min(count - 1, last + a.window - 1 - past) : count - 1;
  float sum = 0.0f;
  if (t_lo <= t_hi) {
    KeyRun run(0, 0, 0, 0);
    run.lo = key0;       // 64 keys as they lie
    load_rows<T>(rows_s, (const T*)a.k_pool, a, table, kh, run, 0, last - key0 + 1);
    const int r_hi = (t_hi + 1) * G;
    for (int r0 = t_lo * G; r0 < r_hi; r0 += kGenWeightRows) {
      __syncthreads();
      load_queries<T, kGenWeightRows>(q_s, a, token0, kh, G, r0, r_hi);
      if (tid < kGenWeightRows) {
        const int R = r0 + tid;
        lse_s[tid] = R < r_hi ? a.lse[(token0 + R / G) * a.heads + kh * G + R % G] : -INFINITY;
      }
      __syncthreads();
      const int n = min(kGenWeightRows, r_hi - r0);
      for (int q0 = 4 * rg; q0 < n; q0 += 16) {      // a thread's group of four rows, then the next but three
        float s[4];
        dots(rows_s + key_i * (hdp + 4), q_s + q0 * hdp, hdp, s);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int R = r0 + q0 + i, pos = R < r_hi ? past + R / G : -1;
          const float d = lse_s[q0 + i];
          if (sees(key, pos, window_lo(pos, a.window), a.first) && d != -INFINITY) sum += expf(s[i] - d);
        }
      }
    }
  }
  part_s[tid] = sum;
  __syncthreads();
  if (tid < kGenKeys && key < end && key < a.capacity) {
    const size_t at = ((size_t)(a.slots ? a.slots[seq] : seq) * a.kv_heads + kh) * a.capacity + key;
    const float before = key < past ? a.weights[at] : 0.0f;
    a.weights_out[at] = before + ((part_s[tid] + part_s[64 + tid]) + (part_s[128 + tid] + part_s[192 + tid]));
  }
}

template <typename T, int RPT>
static int launch_general(const KeptArgs& a, int max_count, long long tokens, cudaStream_t s) {
  const int smem = general_smem(a.head_dim), G = a.heads / a.kv_heads;
  static std::atomic<unsigned long long> allowed;
  const cudaError_t e = allow_shared((const void*)kept_general_kernel<T, RPT>, general_smem(256), allowed);
  if (e != cudaSuccess) return fail(2, "attention_kept: cannot reserve shared memory: %s", cudaGetErrorString(e));
  const long long tiles = ((long long)max_count * G + kGenRows - 1) / kGenRows;
  SLB_REQUIRE(tiles * a.splits < (1ll << 31), "attention_kept: too many tiles (%lld)", tiles);
  launch(kept_general_kernel<T, RPT>, dim3((unsigned)(tiles * a.splits), a.kv_heads, a.n_seqs), dim3(kGenThreads), smem, s, a, tokens);
  int rc = check_launch("attention_kept (general kernel)");
  if (rc || a.splits == 1) return rc;
  launch_prefetching(kept_join_kernel<T>, dim3(a.heads, (unsigned)(tokens < 65535 ? tokens : 65535), (unsigned)((tokens + 65534) / 65535)),
         dim3((a.head_dim + 31) / 32 * 32), 0, s, a, tokens);
  return check_launch("attention_kept (join)");
}

template <typename T>
static int general(const KeptArgs& a, int max_count, long long tokens, cudaStream_t s) {
  const int groups = kGenThreads / (padded_dim(a.head_dim) / 4);
  if (groups >= 16) return launch_general<T, 1>(a, max_count, tokens, s);
  if (groups >= 8) return launch_general<T, 2>(a, max_count, tokens, s);
  return launch_general<T, 4>(a, max_count, tokens, s);
}

template <typename T>
static int general_weights(const KeptArgs& a, int max_keys, cudaStream_t s) {
  static std::atomic<unsigned long long> allowed;
  const cudaError_t e = allow_shared((const void*)kept_weights_general_kernel<T>, weights_smem(256), allowed);
  if (e != cudaSuccess) return fail(2, "attention_kept: cannot reserve shared memory: %s", cudaGetErrorString(e));
  launch_prefetching(kept_weights_general_kernel<T>, dim3((max_keys + kGenKeys - 1) / kGenKeys, a.kv_heads, a.n_seqs), dim3(kGenThreads),
         weights_smem(a.head_dim), s, a);
  return check_launch("attention_kept (weights, general kernel)");
}

// Shares of the keys: as many as give every SM about four blocks, of at least one step of 64 keys (a step takes a block 3 us, a share more takes
// the joining kernel 0.1: five sequences of 33 to 700 rows in shares of 256 keys 20 us).
static int general_splits(int n_seqs, int max_count, int heads, int kv_heads, int max_keys) {
  const long long tiles = ((long long)max_count * (heads / kv_heads) + kGenRows - 1) / kGenRows * kv_heads * n_seqs;
  long long splits = 4ll * sm_count() / (tiles > 0 ? tiles : 1);
  const long long most = (max_keys + kGenKeys - 1) / kGenKeys;
  splits = splits < most ? splits : most;
  return splits < 1 ? 1 : splits > 64 ? 64 : (int)splits;
}

}  // namespace slb

using namespace slb;

// Which kernels a step takes: few rows are cut along the keys (kept_few.cu), many go to the tcgen05 tensor cores, what neither takes to the
// general kernels above.
enum KeptForm : int { kKeptGeneral = 0, kKeptFew = 1, kKeptTc = 2 };
static int kept_form(long long tokens, int max_count, int heads, int kv_heads, int head_dim, int max_keys, int dtype, bool weights) {
  if (kept_few_takes(tokens, max_count, heads, kv_heads, head_dim, max_keys, dtype, weights)) return kKeptFew;
  const int G = heads / kv_heads;
  if (dtype == kBF16 && (head_dim == 64 || head_dim == 128) && G <= 128 && 128 % G == 0) return kKeptTc;
  return kKeptGeneral;
}

// Floats of scratch that slb_attention_kept takes for a step of these sizes: shares of results, with weights denominators and scores.
extern "C" long long slb_attention_kept_scratch(long long tokens, int n_seqs, int max_count, int heads, int kv_heads, int head_dim, int max_keys,
                                                int dtype, int weights) {
  if (tokens <= 0 || n_seqs <= 0 || max_count <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || max_keys <= 0) return 0;
  const int form = kept_form(tokens, max_count, heads, kv_heads, head_dim, max_keys, dtype, weights != 0);
  if (form == kKeptFew) return kept_few_floats(tokens, n_seqs, max_count, heads, kv_heads, head_dim, max_keys, weights != 0);
  if (form == kKeptTc) return weights ? tokens * heads : 0;
  const int splits = general_splits(n_seqs, max_count, heads, kv_heads, max_keys);
  return (weights ? tokens * heads : 0) + (splits > 1 ? (long long)splits * tokens * heads * (head_dim + 2) : 0);
}

// Attention of a step over a cache of bounded size (kept.cuh). Pools of pool_pages pages; lse [tokens, heads] float32 or null; weights and
// weights_out [slots, kv_heads, capacity] float32 (the same memory or apart) or both null; slots [n_seqs] or null. max_keys: no sequence has
// more rows after the step (0: as many as its table takes). Scratch as slb_attention_kept_scratch says. `status`: a zeroed device word that
// receives a code if a bounded wait inside a kernel gave up.
extern "C" int slb_attention_kept(const void* q, const void* k_pool, const void* v_pool, void* out, const int* seq_start, const int* past,
                                  const int* counts, const int* block_table, int table_stride, int n_seqs, long long tokens, int max_count,
                                  int max_keys, int heads, int kv_heads, int head_dim, int window, int first, float scale, float* lse,
                                  const int* slots, const float* weights, float* weights_out, long long capacity, float* scratch,
                                  long long scratch_floats, long long pool_pages, int* status, int dtype, void* stream) {
  SLB_REQUIRE(n_seqs >= 0 && tokens >= 0 && max_count >= 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0,
              "attention_kept: n_seqs=%d heads=%d kv_heads=%d", n_seqs, heads, kv_heads);
  SLB_REQUIRE(head_dim > 0 && head_dim <= 256 && head_dim % 2 == 0, "attention_kept: head_dim %d is not supported (even, at most 256)", head_dim);
  SLB_REQUIRE(window >= 0 && first >= 0 && table_stride > 0, "attention_kept: window=%d first=%d table_stride=%d", window, first, table_stride);
  SLB_REQUIRE(dtype == kF32 || dtype == kBF16, "attention_kept: unknown dtype %d", dtype);
  SLB_REQUIRE((weights == nullptr) == (weights_out == nullptr) && (weights == nullptr || capacity > 0), "attention_kept: weights and their target go together");
  SLB_REQUIRE(n_seqs < 65536 && kv_heads < 65536 && tokens < (1ll << 31), "attention_kept: n_seqs=%d tokens=%lld", n_seqs, tokens);
  if (n_seqs == 0 || tokens == 0 || max_count == 0) return 0;
  if (max_keys <= 0 || max_keys > table_stride * (long long)kPageTokens) {
    SLB_REQUIRE(table_stride < (1 << 25), "attention_kept: table_stride=%d", table_stride);
    max_keys = table_stride * kPageTokens;
  }
  const bool gather = weights != nullptr;
  const long long need = slb_attention_kept_scratch(tokens, n_seqs, max_count, heads, kv_heads, head_dim, max_keys, dtype, gather);
  SLB_REQUIRE(need == 0 || (scratch != nullptr && scratch_floats >= need), "attention_kept: the step needs %lld floats of scratch, %lld were given",
              need, scratch ? scratch_floats : 0ll);
  KeptArgs a{};
  a.q = q; a.k_pool = k_pool; a.v_pool = v_pool; a.out = out; a.seq_start = seq_start; a.past = past; a.counts = counts;
  a.block_table = block_table; a.table_stride = table_stride; a.n_seqs = n_seqs; a.heads = heads; a.kv_heads = kv_heads;
  a.head_dim = head_dim; a.window = window; a.first = window > 0 ? first : 0; a.scale = scale; a.slots = slots; a.weights = weights;
  a.weights_out = weights_out; a.capacity = capacity; a.lse = lse; a.scratch = scratch;
  const cudaStream_t s = (cudaStream_t)stream;
  SLB_REQUIRE(scale > 0.0f, "attention_kept: the scale is positive, got %g", (double)scale);
  const int form = kept_form(tokens, max_count, heads, kv_heads, head_dim, max_keys, dtype, gather);
  if (form == kKeptFew) return kept_few(a, tokens, max_count, max_keys, pool_pages, status, s);
  if (form == kKeptTc) {
    float* lse2 = gather ? scratch : nullptr;
    const int rc = attention_tc_kept(a, lse2, tokens, max_count, max_keys, pool_pages, status, s);
    return rc || !gather ? rc : kept_weights_tc(a, lse2, tokens, max_count, max_keys, pool_pages, status, s);
  }
  if (gather && lse == nullptr) {
    a.lse = scratch;
    a.scratch = scratch + tokens * heads;
  }
  a.splits = general_splits(n_seqs, max_count, heads, kv_heads, max_keys);
  int rc = dtype == kF32 ? general<float>(a, max_count, tokens, s) : general<__nv_bfloat16>(a, max_count, tokens, s);
  if (rc || !gather) return rc;
  return dtype == kF32 ? general_weights<float>(a, max_keys, s) : general_weights<__nv_bfloat16>(a, max_keys, s);
}
