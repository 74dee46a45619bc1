// Attention of a step's drafted nodes over the paged cache (tree.cuh): the general kernels, for both dtypes and every even head size up to 256.
//
//   out = sum_j softmax_j(scale q . k_j) v_j over the rows j that the node sees; zeros where it sees none
//
// A block takes 16 rows of queries of a (sequence, kv head) (row r is node r / G, query head r % G of the group) and a share of the keys, a page of 64 at a time,
// keys and values as float32 in shared memory. Scores: a thread has four keys by four rows of every fourth piece of four channels, and four neighbours meet by
// shuffles (eight 16-byte reads of shared memory for 64 FMAs; with a key and four rows a thread it was five for 16). Then the running maximum and sum, two rows a
// warp; then the values, four rows by four channels a thread, the keys dealt to as many groups of threads as there are, whose sums meet at the end. A key that a row
// does not see is left out of its sum, not multiplied by zero, so what lies in such a row of the pool (infinities, NaN) never reaches it. Shares are joined by a
// second kernel, in their order: no two blocks add to the same place.
// Measured (one B200, device): five sequences of 33 to 700 rows in float32, 8 / 4 heads of 64 under a window of 256, 17 us, two dependent launches of a page a
// block. 64 sequences of 150 to 4,096 rows in float32, 32 / 8 heads of 128: 772 us, FMA pipe 43 %, issue 67 %, shared memory 53 % (the one key a thread 2,018);
// eight trees of 40 to 64 nodes 1,354 (3,550). bfloat16 with heads of 80, eight sequences: 68 (155).
#include <math.h>

#include <algorithm>

#include "tree.cuh"

namespace slb {

constexpr int kTreeThreads = 256, kTreeRows = 16, kTreeKeys = 64;
constexpr int kTreePitch = kTreeRows + 4;      // of a key's weights: 16-byte reads of four rows

__host__ __device__ constexpr int tree_pad(int hd) { return (hd + 3) & ~3; }
// A row's floats in shared memory: half the banks and a whole number of times all of them, so that two neighbouring keys' pieces of 64 bytes lie in different banks.
__host__ __device__ constexpr int tree_row(int hd) { return ((hd + 31) & ~31) + 16; }
__host__ __device__ constexpr int tree_smem(int hd) {
  return ((2 * kTreeKeys + kTreeRows) * tree_row(hd) + kTreeKeys * kTreePitch + 2 * kTreeRows) * 4;
}

// Scratch of a share: per (share, token, head) hd weighted values, maximum, sum.
__device__ __forceinline__ float* tree_slot(const TreeArgs& a, int split, size_t token, int head) {
  return a.scratch + (((size_t)split * a.tokens + token) * a.heads + head) * (a.head_dim + 2);
}

// Four channels of a row from channel c on, zeros behind the last one.
template <typename T>
__device__ __forceinline__ float4 tree_load(const T* src, int c, int hd, bool whole) {
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
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
  return v;
}

// The page of rows key0 .. key0 + 63, keys and values, as float32 in shared memory: 64 channels of eight rows of each on their way at once. Zeros from row `end` on,
// and for a page that the pool has not (as TMA reads them).
template <typename T>
__device__ __forceinline__ void tree_rows(float* ks, float* vs, const TreeArgs& a, const int* table, int kh, int key0, int end) {
  const int hd = a.head_dim, hdp = tree_pad(hd), pitch = tree_row(hd), r0 = threadIdx.x >> 4;
  const int page = table[key0 / kPageTokens];
  const bool there = page >= 0 && page < a.pool_pages;
  const size_t at = there ? ((size_t)page * a.kv_heads + kh) * kPageTokens * hd : 0;
  const T *kp = (const T*)a.k_pool + at, *vp = (const T*)a.v_pool + at;
  const bool whole = hd % 4 == 0 && ((reinterpret_cast<uintptr_t>(a.k_pool) | reinterpret_cast<uintptr_t>(a.v_pool)) & (4 * sizeof(T) - 1)) == 0;
#pragma unroll 1
  for (int c = 4 * (threadIdx.x & 15); c < hdp; c += 64) {
    float4 k[4], v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = r0 + 16 * i;
      k[i] = v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (there && key0 + r < end) {
        k[i] = tree_load(kp + (size_t)r * hd, c, hd, whole);
        v[i] = tree_load(vp + (size_t)r * hd, c, hd, whole);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      *reinterpret_cast<float4*>(ks + (r0 + 16 * i) * pitch + c) = k[i];
      *reinterpret_cast<float4*>(vs + (r0 + 16 * i) * pitch + c) = v[i];
    }
  }
}

// The same for one pool of float32 in whole 16-byte pieces, asynchronously: a group of copies a thread, empty where there is no such page.
__device__ __forceinline__ void tree_rows_async(float* dst, const float* pool, const TreeArgs& a, const int* table, int kh, int key0, int end, bool more) {
  if (more) {
    const int hd = a.head_dim, pitch = tree_row(hd), r0 = threadIdx.x >> 4, page = table[key0 / kPageTokens];
    const bool there = page >= 0 && page < a.pool_pages;
    const float* src = pool + (there ? ((size_t)page * a.kv_heads + kh) * kPageTokens * hd : 0);
    for (int c = 4 * (threadIdx.x & 15); c < hd; c += 64)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = r0 + 16 * i;
        const bool real = there && key0 + r < end;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst + r * pitch + c)), "l"(real ? src + (size_t)r * hd + c : pool), "r"(real ? 16 : 0) : "memory");
      }
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
}

template <typename T>
__global__ void __launch_bounds__(kTreeThreads) tree_general_kernel(TreeArgs a) {
  pdl_enter();
  extern __shared__ __align__(16) float smem[];
  const int hd = a.head_dim, hdp = tree_pad(hd), pitch = tree_row(hd);
  float* rows_s = smem;                                  // [64][pitch]
  float* values_s = rows_s + kTreeKeys * pitch;          // [64][pitch]
  float* q_s = values_s + kTreeKeys * pitch;             // [16][pitch]
  float* p_s = q_s + kTreeRows * pitch;                  // [64][20]: a score, then a weight; below zero where the row does not see the key
  float* alpha_s = p_s + kTreeKeys * kTreePitch;         // [16]
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
    q_s[r * pitch + c] = R < rows_total && c < hd ? to_f32(((const T*)a.q)[((size_t)(s.tok0 + R / G) * a.heads + kh * G + R % G) * hd + c]) * a.scale : 0.0f;
  }
  __syncthreads();
  int first = s.past;
  for (int r = 0; r < kTreeRows; ++r) first = min(first, lo_s[r]);
  first &= ~(kTreeKeys - 1);
  const int steps = (end - first + kTreeKeys - 1) / kTreeKeys, per = (steps + a.splits - 1) / a.splits;
  const int step0 = min(steps, split * per), step1 = min(steps, step0 + per);

  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};        // rows 2 warp, 2 warp + 1
  // values: a thread has four rows, four channels and every `parts`-th key
  const int quads = hdp / 4, parts = min(8, kTreeThreads / (4 * quads)), part = tid / (4 * quads), vrow = tid % (4 * quads) / quads * 4, vc = tid % quads * 4;
  float acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.0f;
  // Where the copies can be asynchronous the next page's keys come while this one's scores become weights and results, its values while the next scores form (64
  // sequences of 150 to 4,096 rows 843 us without, 772 so); a share of one page has nothing to gain and the longer way in (five sequences under a window of 256:
  // 16.7 us without, 17.8 so).
  const bool ahead = sizeof(T) == 4 && step1 - step0 > 1 && hd % 4 == 0 && ((reinterpret_cast<uintptr_t>(a.k_pool) | reinterpret_cast<uintptr_t>(a.v_pool)) & 15) == 0;
  if (ahead) {
    tree_rows_async(rows_s, (const float*)a.k_pool, a, table, kh, first + step0 * kTreeKeys, end, true);
    tree_rows_async(values_s, (const float*)a.v_pool, a, table, kh, first + step0 * kTreeKeys, end, true);
  }
#pragma unroll 1
  for (int step = step0; step < step1; ++step) {
    const int key0 = first + step * kTreeKeys;
    if (!ahead) __syncthreads();
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
    if (ahead) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else tree_rows<T>(rows_s, values_s, a, table, kh, key0, end);
    __syncthreads();
    {
      // scores: a thread has four keys, sixteen apart, four rows and every fourth piece of four channels; its neighbours the other pieces
      const int piece = tid & 3, key = tid >> 2 & 15, row = (tid >> 6) * 4;
      float sc[4][4];      // [key][row]
#pragma unroll
      for (int k = 0; k < 4; ++k) sc[k][0] = sc[k][1] = sc[k][2] = sc[k][3] = 0.0f;
#pragma unroll 2
      for (int c = 4 * piece; c < hdp; c += 16) {
        float4 kv[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) kv[k] = *reinterpret_cast<const float4*>(rows_s + (key + 16 * k) * pitch + c);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 q = *reinterpret_cast<const float4*>(q_s + (row + i) * pitch + c);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            sc[k][i] = fmaf(q.x, kv[k].x, sc[k][i]);
            sc[k][i] = fmaf(q.y, kv[k].y, sc[k][i]);
            sc[k][i] = fmaf(q.z, kv[k].z, sc[k][i]);
            sc[k][i] = fmaf(q.w, kv[k].w, sc[k][i]);
          }
        }
      }
      // the neighbours' sums come together: lane `piece` ends with key + 16 piece
      float two[2][4], one[4];
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float other = __shfl_xor_sync(0xffffffffu, piece & 2 ? sc[k][i] : sc[k + 2][i], 2);
          two[k][i] = (piece & 2 ? sc[k + 2][i] : sc[k][i]) + other;
        }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float other = __shfl_xor_sync(0xffffffffu, piece & 1 ? two[0][i] : two[1][i], 1);
        const float mine = (piece & 1 ? two[1][i] : two[0][i]) + other;
        one[i] = bits_s[row + i] >> (key + 16 * piece) & 1ull ? mine : -INFINITY;
      }
      *reinterpret_cast<float4*>(p_s + (key + 16 * piece) * kTreePitch + row) = make_float4(one[0], one[1], one[2], one[3]);
    }
    __syncthreads();
    if (ahead) tree_rows_async(rows_s, (const float*)a.k_pool, a, table, kh, key0 + kTreeKeys, end, step + 1 < step1);
    {
      float2* at0 = reinterpret_cast<float2*>(p_s + lane * kTreePitch + 2 * warp);
      float2* at1 = reinterpret_cast<float2*>(p_s + (lane + 32) * kTreePitch + 2 * warp);
      const float2 s0 = *at0, s1 = *at1;
      float2 w0, w1;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float x0 = i ? s0.y : s0.x, x1 = i ? s1.y : s1.x, top = fmaxf(m[i], warp_max(fmaxf(x0, x1)));
        const float use = top == -INFINITY ? 0.0f : top, keep = expf(m[i] - use);
        const unsigned long long b = bits_s[2 * warp + i];
        const bool sees0 = b >> lane & 1ull, sees1 = b >> (lane + 32) & 1ull;
        const float p0 = expf(x0 - use), p1 = expf(x1 - use);
        l[i] = l[i] * keep + warp_sum((sees0 ? p0 : 0.0f) + (sees1 ? p1 : 0.0f));
        m[i] = top;
        (i ? w0.y : w0.x) = sees0 ? p0 : -1.0f;
        (i ? w1.y : w1.x) = sees1 ? p1 : -1.0f;
        if (lane == 0) alpha_s[2 * warp + i] = keep;
      }
      *at0 = w0;
      *at1 = w1;
    }
    if (ahead) asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncthreads();
    if (part < parts) {
      const int n = min(kTreeKeys, end - key0);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float keep = alpha_s[vrow + i];
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[i][k] *= keep;
      }
#pragma unroll 4
      for (int j = part; j < n; j += parts) {
        const float4 v = *reinterpret_cast<const float4*>(values_s + j * pitch + vc), w = *reinterpret_cast<const float4*>(p_s + j * kTreePitch + vrow);
        const float p[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!(p[i] < 0.0f)) {      // (a weight that is no number is one that was seen)
            acc[i][0] = fmaf(p[i], v.x, acc[i][0]);
            acc[i][1] = fmaf(p[i], v.y, acc[i][1]);
            acc[i][2] = fmaf(p[i], v.z, acc[i][2]);
            acc[i][3] = fmaf(p[i], v.w, acc[i][3]);
          }
      }
    }
    if (ahead) {
      __syncthreads();
      tree_rows_async(values_s, (const float*)a.v_pool, a, table, kh, key0 + kTreeKeys, end, step + 1 < step1);
    }
  }
  if (ahead) asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  float* sums_s = rows_s;      // [parts][16][hdp], where keys and values lay
  if (part < parts)
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<float4*>(sums_s + (part * kTreeRows + vrow + i) * hdp + vc) = make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
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
  for (int e = tid; e < kTreeRows * hdp; e += kTreeThreads) {
    const int r = e / hdp, c = e % hdp, R = r0 + r;
    if (R >= rows_total || c >= hd) continue;
    float v = 0.0f;
    for (int k = 0; k < parts; ++k) v += sums_s[(k * kTreeRows + r) * hdp + c];
    const size_t token = s.tok0 + R / G;
    const int head = kh * G + R % G;
    if (a.splits > 1) tree_slot(a, split, token, head)[c] = v;
    else ((T*)a.out)[(token * a.heads + head) * hd + c] = from_f32<T>(l_s[r] == 0.0f ? 0.0f : v / l_s[r]);
  }
}

// A warp joins the shares of a (token, head), in their order: a lane a share's factor, then the lanes along the channels, eight shares on the way at once.
constexpr int kMostSplits = 64;
template <typename T>
__global__ void __launch_bounds__(128) tree_join_kernel(TreeArgs a) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, seq = blockIdx.y;
  const long long row = (long long)blockIdx.x * 4 + warp;
  pdl_wait();      // (the kernel before this one lets it begin before it has waited itself: the tables may still be on their way)
  const TreeSeq s(a, seq);
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

// Shares of the keys: as many as give every SM four blocks (at heads of 128 two run at a time; a share's sums cross memory once more), of at least 64 keys.
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
  // (begins early, call after call: five sequences under a window 17.1 us, 18.5 otherwise)
  launch_prefetching(tree_general_kernel<T>, dim3(a.splits, (unsigned)tiles, a.n_seqs), dim3(kTreeThreads), (size_t)tree_smem(a.head_dim), s, a);
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
