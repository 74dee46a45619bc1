// Attention over a cache of bounded size (kept.cuh), and the weights that its rows gather: the general kernels, for both dtypes, every
// even head size up to 256 and any number of new tokens.
//
//   out = sum_j softmax_j(scale q . k_j) v_j over the rows j that the query sees,   lse = log sum_j exp(scale q . k_j)
//   weights_out[j] = (weights[j] where row j was there before the step, else 0) + sum over the step's queries, and over the query heads
//                    of the key/value head, of exp(scale q . k_j - lse)
//
// Few rows (up to 16 of a sequence and kv head): a block takes 16 rows (row r is token r / G, query head r % G of the group) and a share of the keys
// that some of them sees, 64 at a time, keys as float32 in shared memory, a thread a key and four rows. Many rows: tiles of 64 rows, a thread 4 x 4
// scores, so that eight 16-byte reads of shared memory feed 64 FMAs. Both make one pass with a running maximum and sum per row; values come the
// same way. Rows that are seen come in two runs, the first ones and the window; keys between them are not read. Shares are joined by a second
// kernel, in order. A key that a row does not see is left out of its sum, not multiplied by zero, so what lies in such a row of the pool
// (infinities, NaN) never reaches it.
// The weights need the finished denominators, so their kernel forms the scores again: a block takes 64 keys of one (sequence, kv head)
// and walks over the rows that see some of them, 64 at a time, a thread 4 x 4 scores; where such blocks are few a cluster shares the rows and its first
// block adds the sums in the order of the ranks. For one cut every sum has one order, and no two blocks add to the same place; the cut goes by the step (how many
// sequences, the longest share, the rows that the table holds, the window), so a token's bits may differ between batches.
// Bound by the FMA pipe (39 per cent busy) and shared memory. Measured (device time): float32, a prompt of 700 tokens, 16 / 8 heads of 128, 144 us, with weights 215
// (one pass of 16-row tiles 425); five tokens on 33 to 700 rows, 8 / 4 heads of 64, 12 us, with weights 20, three launches of which each waits for the one before.
// bfloat16 prompts come here where the tensor-core kernels do not take them: other head sizes (2,000 tokens, 8 / 8 heads of 96, 445 us, with weights 647), and groups
// that do not divide their tiles of 128 rows (6,000 tokens, 28 / 4 heads of 128, 8.8 ms, with weights 15.5; 40 / 8 heads 12.8 and 21.3; 32 / 8 heads there 0.32 and 0.48).
#include <math.h>

#include <algorithm>

#include "kept.cuh"
#include "tcgen05.cuh"      // clusters

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

// Four channels of a row as float32; `whole`: rows start where 16 bytes (bfloat16: 8) may be read at once, and end with a whole group of four.
template <typename T>
__device__ __forceinline__ float4 load_quad(const T* src, int left, bool whole) {
  if constexpr (sizeof(T) == 4) {
    if (whole) return *reinterpret_cast<const float4*>(src);
  } else if (whole) {
    const uint2 p = *reinterpret_cast<const uint2*>(src);
    const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&p.x)), b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&p.y));
    return make_float4(a.x, a.y, b.x, b.y);
  }
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  v.x = to_f32(src[0]);
  if (left > 1) v.y = to_f32(src[1]);
  if (left > 2) v.z = to_f32(src[2]);
  if (left > 3) v.w = to_f32(src[3]);
  return v;
}
template <typename T>
__device__ __forceinline__ bool whole_quads(const T* base, int hd) { return hd % 4 == 0 && (reinterpret_cast<uintptr_t>(base) & (4 * sizeof(T) - 1)) == 0; }

// 64 rows of a pool as float32 in shared memory, rows of hdp + 4 floats (16-byte reads of 8 lanes then meet 32 banks); zeros beyond the run. Sixteen
// threads a row and four rows a thread: no division, and a thread's loads are under way together.
template <typename T>
__device__ __forceinline__ void load_rows(float* dst, const T* pool, const KeptArgs& a, const int* table, int kh, const KeyRun& run, int v0, int v1) {
  const int hd = a.head_dim, hdp = padded_dim(hd), r0 = threadIdx.x >> 4;
  const bool whole = whole_quads(pool, hd);
  const T* src[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int v = v0 + r0 + 16 * i;
    src[i] = nullptr;
    if (v < v1) {
      const int key = run.key(v);
      src[i] = pool + (((size_t)table[key / kPageTokens] * a.kv_heads + kh) * kPageTokens + key % kPageTokens) * hd;
    }
  }
#pragma unroll 2
  for (int c = 4 * (threadIdx.x & 15); c < hdp; c += 64) {
    float4 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = src[i] ? load_quad(src[i] + c, hd - c, whole) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<float4*>(dst + (r0 + 16 * i) * (hdp + 4) + c) = x[i];
  }
}

// ROWS rows of queries, times the scale, zeros behind the last row.
template <typename T, int ROWS>
__device__ __forceinline__ void load_queries(float* dst, const KeptArgs& a, size_t token0, int kh, int G, int r0, int rows_total, int pitch) {
  const int hd = a.head_dim, hdp = padded_dim(hd), first = threadIdx.x >> 4;
  const bool whole = whole_quads((const T*)a.q, hd);
  const T* src[ROWS / 16];
#pragma unroll
  for (int i = 0; i < ROWS / 16; ++i) {
    const int R = r0 + first + 16 * i;
    src[i] = R < rows_total ? (const T*)a.q + ((token0 + R / G) * a.heads + kh * G + R % G) * hd : nullptr;
  }
#pragma unroll 2
  for (int c = 4 * (threadIdx.x & 15); c < hdp; c += 64) {
    float4 x[ROWS / 16];
#pragma unroll
    for (int i = 0; i < ROWS / 16; ++i) x[i] = src[i] ? load_quad(src[i] + c, hd - c, whole) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < ROWS / 16; ++i)
      *reinterpret_cast<float4*>(dst + (first + 16 * i) * pitch + c) = make_float4(x[i].x * a.scale, x[i].y * a.scale, x[i].z * a.scale, x[i].w * a.scale);
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

  load_queries<T, kGenRows>(q_s, a, token0, kh, G, r0, rows_total, hdp);
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

// Scores of 64 rows and 64 keys: rows 4 ry .. + 3, keys kx + 16 j; q_s and rows_s in rows of hdp + 4 floats.
__device__ __forceinline__ void dots_tile(const float* rows_s, const float* q_s, int hdp, int kx, int ry, float (&s)[4][4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) s[i][j] = 0.0f;
  const float* k0 = rows_s + kx * (hdp + 4);
  const float* q0 = q_s + 4 * ry * (hdp + 4);
#pragma unroll 2
  for (int c = 0; c < hdp; c += 4) {
    float4 k[4], q[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) k[j] = *reinterpret_cast<const float4*>(k0 + 16 * j * (hdp + 4) + c);
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = *reinterpret_cast<const float4*>(q0 + i * (hdp + 4) + c);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = fmaf(q[i].x, k[j].x, s[i][j]);
        s[i][j] = fmaf(q[i].y, k[j].y, s[i][j]);
        s[i][j] = fmaf(q[i].z, k[j].z, s[i][j]);
        s[i][j] = fmaf(q[i].w, k[j].w, s[i][j]);
      }
  }
}

constexpr int kTileRows = 64, kTilePitch = kGenKeys + 4;
__host__ __device__ constexpr int tile_smem(int hd) { return (2 * 64 * (padded_dim(hd) + 4) + kTileRows * kTilePitch + 2 * kTileRows) * 4; }

// Tiles of 64 rows. CH: groups of 64 channels.
template <typename T, int CH>
__global__ void __launch_bounds__(kGenThreads, CH <= 2 ? 2 : 1) kept_tile_kernel(KeptArgs a, long long tokens) {
  pdl_enter();
  extern __shared__ __align__(16) float smem[];
  const int hd = a.head_dim, hdp = padded_dim(hd);
  float* rows_s = smem;                                  // [64][hdp + 4]
  float* q_s = rows_s + kGenKeys * (hdp + 4);            // [64][hdp + 4]
  float* p_s = q_s + kTileRows * (hdp + 4);              // [64][68]
  float* alpha_s = p_s + kTileRows * kTilePitch;         // [64]
  float* l_s = alpha_s + kTileRows;                      // [64]
  const int tid = threadIdx.x, kx = tid & 15, ry = tid >> 4;
  // the longest walks first: tiles of the highest rows of all sequences and heads
  const int seq = blockIdx.x % a.n_seqs, kh = blockIdx.y, G = a.heads / a.kv_heads;
  const int tiles = gridDim.x / a.n_seqs / a.splits, part = blockIdx.x / a.n_seqs;
  const int tile = tiles - 1 - part / a.splits, split = part % a.splits;
  const int count = a.counts[seq], past = a.past[seq], rows_total = count * G, r0 = tile * kTileRows;
  if (r0 >= rows_total) return;
  const size_t token0 = a.seq_start[seq];
  const int* table = a.block_table + (size_t)seq * a.table_stride;
  const int pos_first = past + r0 / G, pos_last = past + min(rows_total - 1, r0 + kTileRows - 1) / G;
  const KeyRun run(pos_first, pos_last, a.window, a.first);
  const int steps = (run.total + kGenKeys - 1) / kGenKeys, per = (steps + a.splits - 1) / a.splits;
  const int v_begin = split * per * kGenKeys, v_end = min(run.total, v_begin + per * kGenKeys);
  const int all_lo = window_lo(pos_last, a.window);      // keys from here to pos_first, and the first ones, are seen by every row

  load_queries<T, kTileRows>(q_s, a, token0, kh, G, r0, rows_total, hdp + 4);
  int row_pos[4], row_lo[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int R = r0 + 4 * ry + i;
    row_pos[i] = R < rows_total ? past + R / G : -1;
    row_lo[i] = window_lo(row_pos[i], a.window);
  }
  float acc[4][CH][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int h = 0; h < CH; ++h) acc[i][h][0] = acc[i][h][1] = acc[i][h][2] = acc[i][h][3] = 0.0f;
  float m = -INFINITY, l = 0.0f;                         // row tid / 4, its keys 16 (tid % 4) .. + 15
  const int sr = tid >> 2, sq = tid & 3;
  for (int v0 = v_begin; v0 < v_end; v0 += kGenKeys) {
    __syncthreads();
    load_rows<T>(rows_s, (const T*)a.k_pool, a, table, kh, run, v0, v_end);
    __syncthreads();
    const int k_first = run.key(v0), k_last = run.key(min(v0 + kGenKeys, v_end) - 1), n = min(kGenKeys, v_end - v0);
    const bool whole = n == kGenKeys && k_last <= pos_first && (k_first >= all_lo || k_last < a.first) && r0 + kTileRows <= rows_total;
    {
      float s[4][4];
      dots_tile(rows_s, q_s, hdp, kx, ry, s);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = kx + 16 * j, key = run.key(v0 + c);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          p_s[(4 * ry + i) * kTilePitch + c] = whole || (v0 + c < v_end && sees(key, row_pos[i], row_lo[i], a.first)) ? s[i][j] : -INFINITY;
      }
    }
    __syncthreads();
    load_rows<T>(rows_s, (const T*)a.v_pool, a, table, kh, run, v0, v_end);
    {
      float4 x[4];
      float* row = p_s + sr * kTilePitch + 16 * sq;
#pragma unroll
      for (int g = 0; g < 4; ++g) x[g] = *reinterpret_cast<const float4*>(row + 4 * g);
      float top = -INFINITY;
#pragma unroll
      for (int g = 0; g < 4; ++g) top = fmaxf(top, fmaxf(fmaxf(x[g].x, x[g].y), fmaxf(x[g].z, x[g].w)));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float m_new = fmaxf(m, top), use = m_new == -INFINITY ? 0.0f : m_new, alpha = expf(m - use);
      float sum = 0.0f;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        x[g].x = expf(x[g].x - use); x[g].y = expf(x[g].y - use);
        x[g].z = expf(x[g].z - use); x[g].w = expf(x[g].w - use);
        sum += (x[g].x + x[g].y) + (x[g].z + x[g].w);
        *reinterpret_cast<float4*>(row + 4 * g) = x[g];
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      l = l * alpha + sum;
      m = m_new;
      if (sq == 0) alpha_s[sr] = alpha;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float f = alpha_s[4 * ry + i];
#pragma unroll
      for (int h = 0; h < CH; ++h)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[i][h][c] *= f;
    }
    const float* v_at = rows_s + 4 * kx;
    if (whole) {
#pragma unroll 2
      for (int j = 0; j < kGenKeys; j += 4) {
        float4 p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = *reinterpret_cast<const float4*>(p_s + (4 * ry + i) * kTilePitch + j);
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int h = 0; h < CH; ++h) {
            if (64 * h + 4 * kx >= hdp) continue;
            const float4 v = *reinterpret_cast<const float4*>(v_at + (j + u) * (hdp + 4) + 64 * h);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float w = u == 0 ? p[i].x : u == 1 ? p[i].y : u == 2 ? p[i].z : p[i].w;
              acc[i][h][0] = fmaf(w, v.x, acc[i][h][0]);
              acc[i][h][1] = fmaf(w, v.y, acc[i][h][1]);
              acc[i][h][2] = fmaf(w, v.z, acc[i][h][2]);
              acc[i][h][3] = fmaf(w, v.w, acc[i][h][3]);
            }
          }
      }
    } else {
#pragma unroll 4
      for (int j = 0; j < n; ++j) {
        float w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = p_s[(4 * ry + i) * kTilePitch + j];
#pragma unroll
        for (int h = 0; h < CH; ++h) {
          if (64 * h + 4 * kx >= hdp) continue;
          const float4 v = *reinterpret_cast<const float4*>(v_at + j * (hdp + 4) + 64 * h);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (w[i] != 0.0f) {
              acc[i][h][0] = fmaf(w[i], v.x, acc[i][h][0]);
              acc[i][h][1] = fmaf(w[i], v.y, acc[i][h][1]);
              acc[i][h][2] = fmaf(w[i], v.z, acc[i][h][2]);
              acc[i][h][3] = fmaf(w[i], v.w, acc[i][h][3]);
            }
        }
      }
    }
  }
  __syncthreads();
  if (sq == 0) {
    l_s[sr] = l;
    const int R = r0 + sr;
    if (R < rows_total) {
      const size_t token = token0 + R / G;
      const int head = kh * G + R % G;
      if (a.splits > 1) {
        float* slot = share_slot(a, split, token, head, tokens);
        slot[hd] = m;
        slot[hd + 1] = l;
      } else if (a.lse) {
        a.lse[token * a.heads + head] = l == 0.0f ? -INFINITY : m + logf(l);
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 4 * ry + i, R = r0 + r;
    if (R >= rows_total) continue;
    const size_t token = token0 + R / G;
    const int head = kh * G + R % G;
    const float inv = a.splits > 1 ? 1.0f : l_s[r] == 0.0f ? 0.0f : 1.0f / l_s[r];
#pragma unroll
    for (int h = 0; h < CH; ++h)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int ch = 64 * h + 4 * kx + c;
        if (ch >= hd) continue;
        if (a.splits > 1) share_slot(a, split, token, head, tokens)[ch] = acc[i][h][c];
        else ((T*)a.out)[(token * a.heads + head) * hd + ch] = from_f32<T>(acc[i][h][c] * inv);
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

__host__ __device__ constexpr int weights_smem(int hd) { return ((kGenKeys + kGenWeightRows) * (padded_dim(hd) + 4) + kGenWeightRows + (16 + 8) * kGenKeys) * 4; }

template <typename T>
__global__ void __launch_bounds__(kGenThreads) kept_weights_general_kernel(KeptArgs a) {
  pdl_enter();
  extern __shared__ __align__(16) float smem[];
  const int hd = a.head_dim, hdp = padded_dim(hd);
  float* rows_s = smem;                                  // [64][hdp + 4]
  float* q_s = rows_s + kGenKeys * (hdp + 4);            // [64][hdp + 4]
  float* lse_s = q_s + kGenWeightRows * (hdp + 4);       // [64]
  float* part_s = lse_s + kGenWeightRows;                // [16 groups of rows][64]
  float* rank_s = part_s + 16 * kGenKeys;                // [8 ranks][64] (the first block's)
  const int tid = threadIdx.x, kx = tid & 15, ry = tid >> 4;
  const int ranks = a.splits, rank = (int)cluster_ctarank();
  const int seq = blockIdx.z, kh = blockIdx.y, G = a.heads / a.kv_heads;
  const int count = a.counts[seq], past = a.past[seq], end = past + count;
  const int key0 = (int)(blockIdx.x / ranks) * kGenKeys;
  if (count <= 0 || key0 >= end) {                       // (the whole cluster)
    if (count <= 0 && rank == 0) carry_weights(a, seq, kh, key0, key0 + kGenKeys, tid, kGenThreads);
    return;
  }
  const size_t token0 = a.seq_start[seq];
  const int* table = a.block_table + (size_t)seq * a.table_stride;
  // the queries that see some key of the tile: from the tile's own rows on, and while the window reaches back to it (or all of them)
  const int last = min(end, key0 + kGenKeys) - 1;
  const int t_lo = max(0, key0 - past);
  const int t_hi = a.window > 0 && key0 >= a.first ? min(count - 1, last + a.window - 1 - past) : count - 1;
  float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (t_lo <= t_hi) {
    KeyRun run(0, 0, 0, 0);
    run.lo = key0;       // 64 keys as they lie
    load_rows<T>(rows_s, (const T*)a.k_pool, a, table, kh, run, 0, last - key0 + 1);
    const int r_hi = (t_hi + 1) * G;
    for (int r0 = t_lo * G + rank * kGenWeightRows; r0 < r_hi; r0 += ranks * kGenWeightRows) {
      __syncthreads();
      load_queries<T, kGenWeightRows>(q_s, a, token0, kh, G, r0, r_hi, hdp + 4);
      if (tid < kGenWeightRows) {
        const int R = r0 + tid;
        lse_s[tid] = R < r_hi ? a.lse[(token0 + R / G) * a.heads + kh * G + R % G] : -INFINITY;
      }
      __syncthreads();
      float s[4][4];
      dots_tile(rows_s, q_s, hdp, kx, ry, s);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int R = r0 + 4 * ry + i, pos = R < r_hi ? past + R / G : -1, lo = window_lo(pos, a.window);
        const float d = lse_s[4 * ry + i];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (sees(key0 + kx + 16 * j, pos, lo, a.first) && d != -INFINITY) sum[j] += expf(s[i][j] - d);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) part_s[ry * kGenKeys + kx + 16 * j] = sum[j];
  __syncthreads();
  float total = 0.0f;
  if (tid < kGenKeys)
#pragma unroll
    for (int g = 0; g < 16; ++g) total += part_s[g * kGenKeys + tid];
  if (ranks > 1) {
    cluster_sync_all();      // (the first block has begun; whole warps come here)
    if (tid < kGenKeys)
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cluster_map(smem_addr(rank_s + rank * kGenKeys + tid), 0)), "f"(total) : "memory");
    __syncthreads();
    cluster_sync_all();
    if (rank != 0) return;
    total = 0.0f;
    if (tid < kGenKeys)
      for (int i = 0; i < ranks; ++i) total += rank_s[i * kGenKeys + tid];
  }
  const int key = key0 + tid;
  if (tid < kGenKeys && key < end && key < a.capacity) {
    const size_t at = ((size_t)(a.slots ? a.slots[seq] : seq) * a.kv_heads + kh) * a.capacity + key;
    a.weights_out[at] = (key < past ? a.weights[at] : 0.0f) + total;
  }
}

// A step without any token, whose weights go elsewhere.
__global__ void __launch_bounds__(256) kept_carry_kernel(KeptArgs a) {
  pdl_enter();
  carry_weights(a, blockIdx.z, blockIdx.y, 0, a.capacity, blockIdx.x * 256 + threadIdx.x, gridDim.x * 256);
}

template <typename T>
static int launch_join(const KeptArgs& a, long long tokens, cudaStream_t s) {
  if (a.splits == 1) return 0;
  launch_prefetching(kept_join_kernel<T>, dim3(a.heads, (unsigned)(tokens < 65535 ? tokens : 65535), (unsigned)((tokens + 65534) / 65535)),
                     dim3((a.head_dim + 31) / 32 * 32), 0, s, a, tokens);
  return check_launch("attention_kept (join)");
}

template <typename T, int RPT>
static int launch_general(const KeptArgs& a, int max_count, long long tokens, cudaStream_t s) {
  const int smem = general_smem(a.head_dim), G = a.heads / a.kv_heads;
  static std::atomic<unsigned long long> allowed;
  const cudaError_t e = allow_shared((const void*)kept_general_kernel<T, RPT>, general_smem(256), allowed);
  if (e != cudaSuccess) return fail(2, "attention_kept: cannot reserve shared memory: %s", cudaGetErrorString(e));
  const long long tiles = ((long long)max_count * G + kGenRows - 1) / kGenRows;
  launch(kept_general_kernel<T, RPT>, dim3((unsigned)(tiles * a.splits), a.kv_heads, a.n_seqs), dim3(kGenThreads), smem, s, a, tokens);
  const int rc = check_launch("attention_kept (general kernel)");
  return rc ? rc : launch_join<T>(a, tokens, s);
}

template <typename T, int CH>
static int launch_tiles(const KeptArgs& a, int max_count, long long tokens, cudaStream_t s) {
  const int smem = tile_smem(a.head_dim), G = a.heads / a.kv_heads;
  static std::atomic<unsigned long long> allowed;
  const cudaError_t e = allow_shared((const void*)kept_tile_kernel<T, CH>, tile_smem(64 * CH), allowed);
  if (e != cudaSuccess) return fail(2, "attention_kept: cannot reserve shared memory: %s", cudaGetErrorString(e));
  const long long blocks = ((long long)max_count * G + kTileRows - 1) / kTileRows * a.splits * a.n_seqs;
  SLB_REQUIRE(blocks < (1ll << 31), "attention_kept: too many tiles (%lld)", blocks);
  launch(kept_tile_kernel<T, CH>, dim3((unsigned)blocks, a.kv_heads), dim3(kGenThreads), smem, s, a, tokens);
  const int rc = check_launch("attention_kept (tiles)");
  return rc ? rc : launch_join<T>(a, tokens, s);
}

// Tiles of 64 rows from 17 rows on.
static int general_rows(int max_count, int G) { return (long long)max_count * G <= kGenRows ? kGenRows : kTileRows; }

template <typename T>
static int general(const KeptArgs& a, int max_count, long long tokens, cudaStream_t s) {
  if (general_rows(max_count, a.heads / a.kv_heads) == kTileRows)
    return a.head_dim <= 64 ? launch_tiles<T, 1>(a, max_count, tokens, s) : a.head_dim <= 128 ? launch_tiles<T, 2>(a, max_count, tokens, s)
                                                                                             : launch_tiles<T, 4>(a, max_count, tokens, s);
  const int groups = kGenThreads / (padded_dim(a.head_dim) / 4);
  if (groups >= 16) return launch_general<T, 1>(a, max_count, tokens, s);
  if (groups >= 8) return launch_general<T, 2>(a, max_count, tokens, s);
  return launch_general<T, 4>(a, max_count, tokens, s);
}

template <typename T>
static int general_weights(KeptArgs a, int max_count, int max_keys, cudaStream_t s) {
  static std::atomic<unsigned long long> allowed;
  const cudaError_t e = allow_shared((const void*)kept_weights_general_kernel<T>, weights_smem(256), allowed);
  if (e != cudaSuccess) return fail(2, "attention_kept: cannot reserve shared memory: %s", cudaGetErrorString(e));
  // blocks that share 64 keys: up to two an SM in all, and no more than there are steps of rows
  const int tiles = (max_keys + kGenKeys - 1) / kGenKeys;
  const long long blocks = (long long)tiles * a.kv_heads * a.n_seqs, steps = ((long long)max_count * (a.heads / a.kv_heads) + kGenWeightRows - 1) / kGenWeightRows;
  a.splits = 1;
  while (a.splits < 8 && a.splits < steps && blocks * a.splits < 2 * sm_count()) a.splits *= 2;
  launch_clusters(pdl_mode() != 0, (unsigned)a.splits, kept_weights_general_kernel<T>, dim3(tiles * a.splits, a.kv_heads, a.n_seqs), dim3(kGenThreads),
                  weights_smem(a.head_dim), s, a);
  return check_launch("attention_kept (weights, general kernel)");
}

// Shares of the keys: as many as give every SM about four blocks (a prompt's tiles grow with their rows: 176 tiles of 1 to 11 steps, whole, 239 us,
// in three shares 152), of at least one step of 64 keys (a step takes a block 3 us, a
// share more takes the joining kernel 0.1: five sequences of 33 to 700 rows in shares of 256 keys 20 us). A tile walks the first rows and its
// tokens' windows at most, however long the cache is.
static int general_splits(int n_seqs, int max_count, int heads, int kv_heads, int max_keys, int window, int first) {
  const int G = heads / kv_heads, rows = general_rows(max_count, G);
  const long long tiles = ((long long)max_count * G + rows - 1) / rows * kv_heads * n_seqs;
  long long splits = 4ll * sm_count() / (tiles > 0 ? tiles : 1);
  long long keys = max_keys;
  if (window > 0) keys = std::min(keys, (long long)first + window + std::min(max_count, (rows + G - 2) / G + 1) - 1);
  const long long most = (keys + kGenKeys - 1) / kGenKeys;
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

// No sequence brings more tokens than the step has, or than it has rows afterwards.
static int least_count(int max_count, long long tokens, int max_keys) { return (int)std::min({(long long)max_count, tokens, (long long)max_keys}); }

// Floats of scratch that slb_attention_kept takes for a step of these sizes: shares of results, with weights denominators and scores.
extern "C" long long slb_attention_kept_scratch(long long tokens, int n_seqs, int max_count, int heads, int kv_heads, int head_dim, int max_keys,
                                                int dtype, int weights) {
  if (tokens <= 0 || n_seqs <= 0 || max_count <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || max_keys <= 0) return 0;
  max_count = least_count(max_count, tokens, max_keys);
  const int form = kept_form(tokens, max_count, heads, kv_heads, head_dim, max_keys, dtype, weights != 0);
  if (form == kKeptFew) return kept_few_floats(tokens, n_seqs, max_count, heads, kv_heads, head_dim, max_keys, weights != 0);
  if (form == kKeptTc) return weights ? tokens * heads : 0;
  const int splits = general_splits(n_seqs, max_count, heads, kv_heads, max_keys, 0, 0);      // (under a window no more)
  return (weights ? tokens * heads : 0) + (splits > 1 ? (long long)splits * tokens * heads * (head_dim + 2) : 0);
}

// Attention of a step over a cache of bounded size (kept.cuh). max_keys: no sequence has more rows after the step (0: as many as its table
// takes). Scratch as slb_attention_kept_scratch says.
extern "C" int slb_attention_kept(const KeptCall* call) {
  SLB_REQUIRE(call != nullptr, "attention_kept: no call");
  const KeptCall c = *call;
  const int n_seqs = c.n_seqs, heads = c.heads, kv_heads = c.kv_heads, head_dim = c.head_dim, table_stride = c.table_stride, dtype = c.dtype;
  int max_count = c.max_count, window = c.window, first = c.first;
  const long long tokens = c.tokens;
  const float scale = c.scale;
  int max_keys = c.max_keys;
  SLB_REQUIRE(n_seqs >= 0 && tokens >= 0 && max_count >= 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0,
              "attention_kept: n_seqs=%d heads=%d kv_heads=%d", n_seqs, heads, kv_heads);
  SLB_REQUIRE(head_dim > 0 && head_dim <= 256 && head_dim % 2 == 0, "attention_kept: head_dim %d is not supported (even, at most 256)", head_dim);
  SLB_REQUIRE(window >= 0 && first >= 0 && table_stride > 0, "attention_kept: window=%d first=%d table_stride=%d", window, first, table_stride);
  SLB_REQUIRE(dtype == kF32 || dtype == kBF16, "attention_kept: unknown dtype %d", dtype);
  SLB_REQUIRE((c.weights == nullptr) == (c.weights_out == nullptr) && (c.weights == nullptr || c.capacity > 0), "attention_kept: weights and their target go together");
  SLB_REQUIRE(n_seqs < 65536 && kv_heads < 65536 && tokens < (1ll << 31), "attention_kept: n_seqs=%d tokens=%lld", n_seqs, tokens);
  if (n_seqs == 0) return 0;
  KeptArgs a{};
  a.q = c.q; a.k_pool = c.k_pool; a.v_pool = c.v_pool; a.out = c.out; a.seq_start = c.seq_start; a.past = c.past; a.counts = c.counts;
  a.block_table = c.block_table; a.table_stride = table_stride; a.n_seqs = n_seqs; a.heads = heads; a.kv_heads = kv_heads;
  a.head_dim = head_dim; a.scale = scale; a.slots = c.slots; a.weights = c.weights; a.weights_out = c.weights_out; a.capacity = c.capacity; a.lse = c.lse;
  a.scratch = c.scratch;
  const cudaStream_t s = (cudaStream_t)c.stream;
  if (tokens == 0 || max_count == 0) {
    if (c.weights == nullptr || c.weights_out == c.weights) return 0;
    launch(kept_carry_kernel, dim3((unsigned)std::min((c.capacity + 255) / 256, 8ll), kv_heads, n_seqs), dim3(256), 0, s, a);
    return check_launch("attention_kept (no tokens)");
  }
  if (max_keys <= 0 || max_keys > table_stride * (long long)kPageTokens) {
    SLB_REQUIRE(table_stride < (1 << 25), "attention_kept: table_stride=%d", table_stride);
    max_keys = table_stride * kPageTokens;
  }
  // What hides nothing is taken out and what is beyond the last row is cut, so that sums of these numbers stay within 32 bits whatever a caller
  // says for "no limit": a window as long as the longest sequence is none, first rows behind it are all.
  SLB_REQUIRE(max_keys <= (1 << 30), "attention_kept: a sequence of %d rows", max_keys);
  if (window >= max_keys) window = 0;
  first = window > 0 ? std::min(first, max_keys) : 0;
  max_count = least_count(max_count, tokens, max_keys);
  const bool gather = c.weights != nullptr;
  const long long need = slb_attention_kept_scratch(tokens, n_seqs, max_count, heads, kv_heads, head_dim, max_keys, dtype, gather);
  SLB_REQUIRE(need == 0 || (c.scratch != nullptr && c.scratch_floats >= need), "attention_kept: the step needs %lld floats of scratch, %lld were given",
              need, c.scratch ? c.scratch_floats : 0ll);
  a.window = window;
  a.first = first;
  SLB_REQUIRE(scale > 0.0f, "attention_kept: the scale is positive, got %g", (double)scale);
  const int form = kept_form(tokens, max_count, heads, kv_heads, head_dim, max_keys, dtype, gather);
  if (form == kKeptFew) return kept_few(a, tokens, max_count, max_keys, c.pool_pages, c.status, s);
  if (form == kKeptTc) {
    float* lse2 = gather ? c.scratch : nullptr;
    const int rc = attention_tc_kept(a, lse2, tokens, max_count, max_keys, c.pool_pages, c.status, s);
    return rc || !gather ? rc : kept_weights_tc(a, lse2, tokens, max_count, max_keys, c.pool_pages, c.status, s);
  }
  if (gather && c.lse == nullptr) {
    a.lse = c.scratch;
    a.scratch = c.scratch + tokens * heads;
  }
  a.splits = general_splits(n_seqs, max_count, heads, kv_heads, max_keys, window, first);
  int rc = dtype == kF32 ? general<float>(a, max_count, tokens, s) : general<__nv_bfloat16>(a, max_count, tokens, s);
  if (rc || !gather) return rc;
  return dtype == kF32 ? general_weights<float>(a, max_count, max_keys, s) : general_weights<__nv_bfloat16>(a, max_count, max_keys, s);
}
