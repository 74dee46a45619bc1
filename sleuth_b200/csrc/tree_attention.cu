// Attention of a step's drafted nodes over the paged cache (tree.cuh): the general kernels, for both dtypes and every even head size up to 256.
//
//   out = sum_j softmax_j(scale q . k_j) v_j over the rows j that the node sees; zeros where it sees none
//
// A block takes 16 rows of queries of a (sequence, kv head) (row r is node r / G, query head r % G of the group) and a share of the keys, 64 at a
// time: keys as float32 in shared memory, a thread a key and four rows; then the values the same way, with a running maximum and sum a row. A key
// that a row does not see is left out of its sum, not multiplied by zero, so what lies in such a row of the pool (infinities, NaN) never
// reaches it. Shares are joined by a second kernel, in their order: no two blocks add to the same place.
#include <math.h>

#include <algorithm>

#include "tree.cuh"

namespace slb {

constexpr int kTreeThreads = 256, kTreeRows = 16, kTreeKeys = 64;

__host__ __device__ constexpr int tree_pad(int hd) { return (hd + 3) & ~3; }
__host__ __device__ constexpr int tree_smem(int hd) {
  return (2 * kTreeKeys * (tree_pad(hd) + 4) + kTreeRows * tree_pad(hd) + kTreeRows * kTreeKeys + 2 * kTreeRows) * 4;
}

// Scratch of a share: per (share, token, head) hd weighted values, maximum, sum.
__device__ __forceinline__ float* tree_slot(const TreeArgs& a, int split, size_t token, int head) {
  return a.scratch + (((size_t)split * a.tokens + token) * a.heads + head) * (a.head_dim + 2);
}

// 64 rows of a pool from row `key0` on as float32 in shared memory, rows of hdp + 4 floats; zeros from row `end` on, and for pages that the pool has not (as TMA reads them).
template <typename T>
__device__ __forceinline__ void tree_rows(float* dst, const T* pool, const TreeArgs& a, const int* table, int kh, int key0, int end) {
  const int hd = a.head_dim, hdp = tree_pad(hd), r0 = threadIdx.x >> 4;
  const bool whole = hd % 4 == 0 && (reinterpret_cast<uintptr_t>(pool) & (4 * sizeof(T) - 1)) == 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int key = key0 + r0 + 16 * i;
    const int page = key < end ? table[key / kPageTokens] : -1;
    const T* src = page >= 0 && page < a.pool_pages ? pool + (((size_t)page * a.kv_heads + kh) * kPageTokens + key % kPageTokens) * hd : nullptr;
    for (int c = 4 * (threadIdx.x & 15); c < hdp; c += 64) {
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (src) {
        if (whole) {
          if constexpr (sizeof(T) == 4) {
            v = *reinterpret_cast<const float4*>(src + c);
          } else {
            const uint2 p = *reinterpret_cast<const uint2*>(src + c);
            const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&p.x)), y = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&p.y));
            v = make_float4(x.x, x.y, y.x, y.y);
          }
        } else {
          v.x = to_f32(src[c]);
          if (c + 1 < hd) v.y = to_f32(src[c + 1]);
          if (c + 2 < hd) v.z = to_f32(src[c + 2]);
          if (c + 3 < hd) v.w = to_f32(src[c + 3]);
        }
      }
      *reinterpret_cast<float4*>(dst + (r0 + 16 * i) * (hdp + 4) + c) = v;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kTreeThreads) tree_general_kernel(TreeArgs a) {
  pdl_enter();
  extern __shared__ __align__(16) float smem[];
  const int hd = a.head_dim, hdp = tree_pad(hd);
  float* rows_s = smem;                                  // [64][hdp + 4]
  float* values_s = rows_s + kTreeKeys * (hdp + 4);      // [64][hdp + 4]
  float* q_s = values_s + kTreeKeys * (hdp + 4);         // [16][hdp]
  float* p_s = q_s + kTreeRows * hdp;                    // [16][64]
  float* alpha_s = p_s + kTreeRows * kTreeKeys;          // [16]
  float* l_s = alpha_s + kTreeRows;                      // [16]
  __shared__ unsigned long long bits_s[kTreeRows];
  __shared__ int lo_s[kTreeRows];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, G = a.heads / a.kv_heads;
  const int split = blockIdx.x, kh = blockIdx.y % a.kv_heads, tile = blockIdx.y / a.kv_heads, seq = blockIdx.z;
  const TreeSeq s(a, seq);
  const int rows_total = s.count * G, r0 = tile * kTreeRows, end = s.past + s.count;
  if (r0 >= rows_total) return;
  const int* table = a.block_table + (size_t)seq * a.table_stride;
  if (tid < kTreeRows) lo_s[tid] = r0 + tid < rows_total ? tree_lo(a, s.tok0 + (r0 + tid) / G, s.past) : s.past;
  for (int e = tid; e < kTreeRows * hdp; e += kTreeThreads) {
    const int r = e / hdp, c = e % hdp, R = r0 + r;
    q_s[e] = R < rows_total && c < hd ? to_f32(((const T*)a.q)[((size_t)(s.tok0 + R / G) * a.heads + kh * G + R % G) * hd + c]) * a.scale : 0.0f;
  }
  __syncthreads();
  int first = s.past;
  for (int r = 0; r < kTreeRows; ++r) first = min(first, lo_s[r]);
  first &= ~(kTreeKeys - 1);
  const int steps = (end - first + kTreeKeys - 1) / kTreeKeys, per = (steps + a.splits - 1) / a.splits;
  const int step0 = min(steps, split * per), step1 = min(steps, step0 + per);

  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};        // rows 2 warp, 2 warp + 1
  constexpr int kQuads = kTreeRows * 256 / 4 / kTreeThreads;       // row and four channels: kTreeRows * hdp / 4 of them
  float acc[kQuads][4];
#pragma unroll
  for (int i = 0; i < kQuads; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.0f;
  const int quads = hdp / 4;
  for (int step = step0; step < step1; ++step) {
    const int key0 = first + step * kTreeKeys;
    __syncthreads();
    tree_rows<T>(rows_s, (const T*)a.k_pool, a, table, kh, key0, end);
    tree_rows<T>(values_s, (const T*)a.v_pool, a, table, kh, key0, end);
    if (tid < kTreeRows) {      // what a row sees of these 64 keys
      const int R = r0 + tid;
      unsigned long long b = 0ull;
      if (R < rows_total) {
        const int from = lo_s[tid] - key0, to = s.past - key0;      // old keys: from .. to - 1
        if (from < 64 && to > 0) b = (to >= 64 ? ~0ull : (1ull << to) - 1ull) & (from <= 0 ? ~0ull : ~0ull << from);
        if (from >= to) b = 0ull;
        b |= tree_bits(a.seen + (size_t)(s.tok0 + R / G) * a.words, a.words, key0 - s.past, s.count);
      }
      bits_s[tid] = b;
    }
    __syncthreads();
    {
      const int key = tid & 63, group = tid >> 6;
      float sc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      const float* k = rows_s + key * (hdp + 4);
      for (int c = 0; c < hdp; c += 4) {
        const float4 kv = *reinterpret_cast<const float4*>(k + c);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 q = *reinterpret_cast<const float4*>(q_s + (group * 4 + i) * hdp + c);
          sc[i] = fmaf(q.x, kv.x, sc[i]);
          sc[i] = fmaf(q.y, kv.y, sc[i]);
          sc[i] = fmaf(q.z, kv.z, sc[i]);
          sc[i] = fmaf(q.w, kv.w, sc[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) p_s[(group * 4 + i) * kTreeKeys + key] = bits_s[group * 4 + i] >> key & 1ull ? sc[i] : -INFINITY;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float* p = p_s + (2 * warp + i) * kTreeKeys;
      const float s0 = p[lane], s1 = p[lane + 32], top = fmaxf(m[i], warp_max(fmaxf(s0, s1)));
      const float use = top == -INFINITY ? 0.0f : top, keep = expf(m[i] - use);
      const unsigned long long b = bits_s[2 * warp + i];
      const float p0 = b >> lane & 1ull ? expf(s0 - use) : 0.0f, p1 = b >> (lane + 32) & 1ull ? expf(s1 - use) : 0.0f;
      p[lane] = p0;
      p[lane + 32] = p1;
      l[i] = l[i] * keep + warp_sum(p0 + p1);
      m[i] = top;
      if (lane == 0) alpha_s[2 * warp + i] = keep;
    }
    __syncthreads();
    const int n = min(kTreeKeys, end - key0);
#pragma unroll
    for (int i = 0; i < kQuads; ++i) {
      const int e = tid + i * kTreeThreads, r = e / quads, c = e % quads * 4;
      if (r >= kTreeRows) continue;
      const float keep = alpha_s[r];
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[i][k] *= keep;
      const unsigned long long b = bits_s[r];
#pragma unroll 4
      for (int j = 0; j < n; ++j) {
        if (!(b >> j & 1ull)) continue;
        const float p = p_s[r * kTreeKeys + j];
        const float4 v = *reinterpret_cast<const float4*>(values_s + j * (hdp + 4) + c);
        acc[i][0] = fmaf(p, v.x, acc[i][0]);
        acc[i][1] = fmaf(p, v.y, acc[i][1]);
        acc[i][2] = fmaf(p, v.z, acc[i][2]);
        acc[i][3] = fmaf(p, v.w, acc[i][3]);
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int R = r0 + 2 * warp + i;
    if (lane != 0) continue;
    l_s[2 * warp + i] = l[i];
    if (R < rows_total && a.splits > 1) {
      float* slot = tree_slot(a, split, s.tok0 + R / G, kh * G + R % G);
      slot[hd] = m[i];
      slot[hd + 1] = l[i];
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kQuads; ++i) {
    const int e = tid + i * kTreeThreads, r = e / quads, c = e % quads * 4, R = r0 + r;
    if (r >= kTreeRows || R >= rows_total) continue;
    const size_t token = s.tok0 + R / G;
    const int head = kh * G + R % G;
    const float inv = l_s[r] == 0.0f ? 0.0f : 1.0f / l_s[r];
    for (int k = 0; k < 4 && c + k < hd; ++k) {
      if (a.splits > 1) tree_slot(a, split, token, head)[c + k] = acc[i][k];
      else ((T*)a.out)[(token * a.heads + head) * hd + c + k] = from_f32<T>(acc[i][k] * inv);
    }
  }
}

// A warp joins the shares of a (token, head), in their order: a lane a share's factor, then the lanes along the channels, eight shares on the way at once.
constexpr int kMostSplits = 64;
template <typename T>
__global__ void __launch_bounds__(128) tree_join_kernel(TreeArgs a) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, seq = blockIdx.y;
  const TreeSeq s(a, seq);      // (in front of the wait: what the kernel before this one has waited for is there)
  const long long row = (long long)blockIdx.x * 4 + warp;
  pdl_wait();
  if (row >= (long long)s.count * a.heads) return;
  __shared__ float factor_s[4][kMostSplits];
  const size_t token = s.tok0 + row / a.heads;
  const int head = (int)(row % a.heads), hd = a.head_dim;
  float m[kMostSplits / 32], l[kMostSplits / 32], top = -INFINITY;
#pragma unroll
  for (int k = 0; k < kMostSplits / 32; ++k) {
    const int i = lane + 32 * k;
    m[k] = -INFINITY;
    l[k] = 0.0f;
    if (i < a.splits) {
      const float* slot = tree_slot(a, i, token, head);
      m[k] = slot[hd];
      l[k] = slot[hd + 1];
    }
    top = fmaxf(top, m[k]);
  }
  top = warp_max(top);
  const float use = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f;
#pragma unroll
  for (int k = 0; k < kMostSplits / 32; ++k) {
    const float f = l[k] == 0.0f ? 0.0f : expf(m[k] - use);      // (0: a share that saw nothing)
    factor_s[warp][lane + 32 * k] = f;
    sum += l[k] * f;
  }
  sum = warp_sum(sum);
  __syncwarp();
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  for (int c = lane; c < hd; c += 32) {
    float acc = 0.0f;
    for (int i0 = 0; i0 < a.splits; i0 += 8) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = i0 + i < a.splits ? tree_slot(a, i0 + i, token, head)[c] : 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i0 + i < a.splits && factor_s[warp][i0 + i] != 0.0f) acc = fmaf(v[i], factor_s[warp][i0 + i], acc);
    }
    ((T*)a.out)[(token * a.heads + head) * hd + c] = from_f32<T>(acc * inv);
  }
}

// Shares of the keys: as many as give every SM four blocks, of at least 64 keys.
static int general_tree_splits(int n_seqs, int max_count, int heads, int kv_heads, int max_keys) {
  const long long tiles = (long long)n_seqs * kv_heads * (((long long)max_count * (heads / kv_heads) + kTreeRows - 1) / kTreeRows);
  const long long steps = ((long long)max_keys + kTreeKeys - 1) / kTreeKeys + 1, wanted = (4ll * sm_count() + tiles - 1) / tiles;
  return (int)std::max(1ll, std::min(std::min(steps, wanted), (long long)kMostSplits));
}

static long long general_tree_floats(long long tokens, int n_seqs, int max_count, int heads, int kv_heads, int head_dim, int max_keys) {
  const int splits = general_tree_splits(n_seqs, max_count, heads, kv_heads, max_keys);
  return splits == 1 ? 0 : (long long)splits * tokens * heads * (head_dim + 2);
}

template <typename T>
static int launch_tree_general(TreeArgs a, cudaStream_t s) {
  static std::atomic<unsigned long long> allowed;
  a.splits = general_tree_splits(a.n_seqs, a.max_count, a.heads, a.kv_heads, a.max_keys);
  const cudaError_t e = allow_shared((const void*)tree_general_kernel<T>, tree_smem(256), allowed);
  if (e != cudaSuccess) return fail(2, "attention_tree: cannot reserve shared memory: %s", cudaGetErrorString(e));
  const long long tiles = ((long long)a.max_count * (a.heads / a.kv_heads) + kTreeRows - 1) / kTreeRows * a.kv_heads;
  SLB_REQUIRE(tiles < 65536, "attention_tree: %d nodes of %d heads are too many for one launch", a.max_count, a.heads);
  launch(tree_general_kernel<T>, dim3(a.splits, (unsigned)tiles, a.n_seqs), dim3(kTreeThreads), (size_t)tree_smem(a.head_dim), s, a);
  const int rc = check_launch("attention_tree");
  if (rc || a.splits == 1) return rc;
  launch_prefetching(tree_join_kernel<T>, dim3((unsigned)(((long long)a.max_count * a.heads + 3) / 4), a.n_seqs), dim3(128), 0, s, a);
  return check_launch("attention_tree (joined)");
}

// Floats of scratch that slb_attention_tree takes; negative: sizes that it refuses.
extern "C" long long slb_attention_tree_scratch(long long tokens, int n_seqs, int max_count, int heads, int kv_heads, int head_dim, int max_keys, int dtype) {
  if (tokens < 0 || n_seqs < 0 || max_count <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || head_dim <= 0 || max_keys <= 0) return -1;
  if (tokens == 0 || n_seqs == 0) return 0;
  if (tree_tc_takes(n_seqs, max_count, heads, kv_heads, head_dim, max_keys, dtype)) return tree_tc_floats(n_seqs, max_count, heads, kv_heads, head_dim, max_keys);
  return general_tree_floats(tokens, n_seqs, max_count, heads, kv_heads, head_dim, max_keys);
}

extern "C" int slb_attention_tree(const TreeCall* call) {
  SLB_REQUIRE(call != nullptr, "attention_tree: no call");
  const TreeCall c = *call;
  SLB_REQUIRE(c.dtype == kF32 || c.dtype == kBF16, "attention_tree: dtype %d", c.dtype);
  SLB_REQUIRE(c.head_dim > 0 && c.head_dim <= 256 && c.head_dim % 2 == 0, "attention_tree: head_dim %d must be even and at most 256", c.head_dim);
  SLB_REQUIRE(c.heads > 0 && c.kv_heads > 0 && c.heads % c.kv_heads == 0, "attention_tree: %d heads of %d key/value heads", c.heads, c.kv_heads);
  SLB_REQUIRE(c.n_seqs >= 0 && c.n_seqs < 65536 && c.tokens >= 0 && c.table_stride > 0 && c.pool_pages > 0 && c.window >= 0 && c.scale > 0.0f && c.scale < INFINITY,
              "attention_tree: n_seqs=%d tokens=%lld table_stride=%d window=%d", c.n_seqs, c.tokens, c.table_stride, c.window);
  SLB_REQUIRE(c.max_count > 0 && c.max_count <= kMostNodes, "attention_tree: %d nodes of a sequence; 1 to %d are taken", c.max_count, kMostNodes);
  SLB_REQUIRE(c.words >= 1 && (long long)c.words * 32 >= c.max_count, "attention_tree: %d words of bits do not hold %d nodes", c.words, c.max_count);
  SLB_REQUIRE(c.window == 0 || c.positions != nullptr, "attention_tree: a window needs the nodes' positions");
  if (c.n_seqs == 0 || c.tokens == 0) return 0;
  const long long table_rows = (long long)c.table_stride * kPageTokens;
  SLB_REQUIRE(table_rows < (1ll << 31) - 64, "attention_tree: a block table of %d pages is too long", c.table_stride);
  TreeArgs a{};
  a.q = c.q; a.k_pool = c.k_pool; a.v_pool = c.v_pool; a.out = c.out; a.seq_start = c.seq_start; a.past = c.past; a.counts = c.counts;
  a.seen = (const uint32_t*)c.seen; a.positions = c.positions; a.block_table = c.block_table; a.table_stride = c.table_stride; a.n_seqs = c.n_seqs;
  a.heads = c.heads; a.kv_heads = c.kv_heads; a.head_dim = c.head_dim; a.window = c.window; a.words = c.words; a.max_count = c.max_count;
  a.tokens = c.tokens; a.pool_pages = c.pool_pages; a.scale = c.scale; a.scratch = c.scratch;
  a.max_keys = c.max_keys > 0 && c.max_keys < table_rows ? c.max_keys : (int)table_rows;
  const long long need = slb_attention_tree_scratch(c.tokens, c.n_seqs, c.max_count, c.heads, c.kv_heads, c.head_dim, a.max_keys, c.dtype);
  SLB_REQUIRE(need == 0 || (c.scratch != nullptr && c.scratch_floats >= need), "attention_tree: the step needs %lld floats of scratch, %lld were given", need,
              c.scratch ? c.scratch_floats : 0ll);
  if (tree_tc_takes(c.n_seqs, c.max_count, c.heads, c.kv_heads, c.head_dim, a.max_keys, c.dtype)) return tree_tc(a, c.pool_pages, c.status, (cudaStream_t)c.stream);
  return c.dtype == kF32 ? launch_tree_general<float>(a, (cudaStream_t)c.stream) : launch_tree_general<__nv_bfloat16>(a, (cudaStream_t)c.stream);
}

}  // namespace slb
