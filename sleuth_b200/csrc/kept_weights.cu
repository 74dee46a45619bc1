// The weights that the rows of a cache of bounded size gather in a step of many tokens (kept.cuh), on the tcgen05 tensor cores:
//   weights_out[j] = (weights[j] if row j was there before, else 0) + sum over queries i, heads h of the group, of 2^(s_ihj - d_ih),
// s = scale log2(e) q . k and d the rows' finished denominators in log2 units, which the attention has left.
//
// The scores are formed again with the keys as the instruction's rows, so that a thread of the epilogue owns one key and adds its
// weights over the queries in registers: no sum crosses threads until the end. A block takes 128 keys (two pages) of one (sequence, kv
// head) and walks over the (token, head) rows that see some of them, 128 at a time:
//   * warp 0, one lane: TMA loads of the key tile (once) and of the queries, a ring of five stages (eight at heads of 64): what a step reads from L2, 32
//     KB, takes about as long as its products, and arrives late with two;
//   * warp 1, one lane: S^T = K Q^T (M = 128, N = 128) into one of four accumulators of 128 columns, all of tensor memory;
//   * warp 2: the 128 denominators of a step into shared memory, asked for a step early;
//   * warps 3 to 18: two sets of eight take the steps in turn, a warp 32 keys and 64 columns, a thread 64 scores, 32 at a time. Per score one FMA,
//     one power of two, one addition (in pairs). Only steps with a key that some row does not see run a mask, a range of columns for each key.
// Clusters start in the order of their number: the first keys of all sequences and heads, whose walk is the longest, before the next ones. Where
// blocks are too few for the SMs, a cluster shares a key tile: the steps are dealt to its blocks in turn, the first block adds the sums in the
// order of the ranks.
// Measured: a prompt of 6,000 tokens, 32 / 8 heads of 128, 192 us by itself (0.77 PFLOP/s at 1.84 GHz), 160 to 170 added to the attention in front of it back to
// back. What bounds it: the powers of two (576 M scores at 16 a cycle and SM: 132 us at that clock, their unit 81 per cent busy), then
// the epilogue's waits between its stages. Tried, at 205 us then: 256 queries a step with two stages of them 333 us; three powers of eight by a
// polynomial on the FMA pipe 215, two of eight 201 (issue slots take what the unit gives back); 64 scores at once 211; 24 warps 201.
#include <math.h>

#include <algorithm>

#include "kept.cuh"
#include "packed_f32.cuh"
#include "tcgen05.cuh"

namespace slb {

constexpr int kKwThreads = 608, kKwRows = 128, kKwKeys = 128, kKwBuffers = 4;

struct KeptWeightsArgs {
  KeptArgs k;
  const float* lse2;
  float scale_log2;
  int* status;
  int tile0;            // the first key tile of the launch
};

template <int HD>
struct KwLayout {
  static constexpr int K_BYTES = kKwKeys * HD * 2, Q_BYTES = kKwRows * HD * 2, STAGES = HD == 128 ? 5 : 8;
  static constexpr int K_OFF = 0, Q_OFF = K_BYTES;
  static constexpr int D_OFF = Q_OFF + STAGES * Q_BYTES;                // denominators, [4 buffers][128]
  static constexpr int SUM_OFF = D_OFF + kKwBuffers * kKwRows * 4;      // [4 parts][128 keys]
  static constexpr int RANK_OFF = SUM_OFF + 4 * kKwKeys * 4;            // [8 ranks][128 keys] (the first block's)
  static constexpr int BAR_OFF = RANK_OFF + 8 * kKwKeys * 4;
  static constexpr int N_BARS = 1 + 2 * STAGES + 4 * kKwBuffers;
  static constexpr int TOTAL = BAR_OFF + N_BARS * 8 + 8;
  static_assert(TOTAL <= 226 * 1024, "the block must fit on an SM");
};

__device__ __forceinline__ float kw_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int HD>
__global__ void __launch_bounds__(kKwThreads, 1)
kept_weights_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, KeptWeightsArgs w) {
  using L = KwLayout<HD>;
  extern __shared__ __align__(1024) unsigned char smem[];
  const KeptArgs& a = w.k;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = smem_addr(smem);
  const int rank = (int)cluster_ctarank(), ranks = a.splits;
  const int G = a.heads / a.kv_heads, pairs = (int)(gridDim.y * gridDim.z);
  const int lin = (int)(blockIdx.x / ranks + gridDim.x / ranks * (blockIdx.y + gridDim.y * blockIdx.z));
  const int seq = (lin % pairs) / (int)gridDim.y, kh = (lin % pairs) % (int)gridDim.y, key0 = (w.tile0 + lin / pairs) * kKwKeys;
  const uint32_t bars = base + L::BAR_OFF;
  const uint32_t k_full = bars, q_full = bars + 8, q_free = q_full + 8 * L::STAGES, s_full = q_free + 8 * L::STAGES, s_free = s_full + 8 * kKwBuffers,
                 d_full = s_free + 8 * kKwBuffers, d_free = d_full + 8 * kKwBuffers;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::BAR_OFF + L::N_BARS * 8);
  pdl_wait();
  const int count = a.counts[seq], past = a.past[seq], end = past + count;
  if (count <= 0 || key0 >= end) {             // (the whole cluster)
    if (count <= 0 && rank == 0) carry_weights(a, seq, kh, key0, key0 + kKwKeys, tid, kKwThreads);
    return;
  }
  // that all blocks of the cluster have begun is waited for before the first store into another's shared memory
  if (ranks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const size_t tok0 = a.seq_start[seq];
  const int last = min(end, key0 + kKwKeys) - 1;
  const int t_lo = max(0, key0 - past);
  const int t_hi = a.window > 0 && key0 >= a.first ? min(count - 1, last + a.window - 1 - past) : count - 1;
  const int row_lo = t_lo * G, row_hi = (t_hi + 1) * G;
  const int all_steps = t_lo <= t_hi ? (row_hi - row_lo + kKwRows - 1) / kKwRows : 0;
  const int steps = all_steps > rank ? (all_steps - rank + ranks - 1) / ranks : 0;      // rank, rank + ranks, ...
  const bool aligned = (base & 1023u) == 0;
  float sum = 0.0f;
  const int quad = warp & 3, part = (warp - 3) >> 2;      // lanes of tensor memory; part = 2 * set + half of the columns
  if (all_steps > 0 && aligned) {
    if (tid == 0) {
      mbar_init(k_full, 1);
      for (int i = 0; i < L::STAGES; ++i) {
        mbar_init(q_full + 8 * i, 1);
        mbar_init(q_free + 8 * i, 1);
      }
      for (int i = 0; i < kKwBuffers; ++i) {
        mbar_init(s_full + 8 * i, 1);
        mbar_init(s_free + 8 * i, 8);
        mbar_init(d_full + 8 * i, 32);
        mbar_init(d_free + 8 * i, 8);
      }
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) {
      __syncwarp();
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(tmem_slot)) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    if (warp == 0) {
      if (elect_one() && steps > 0) {
        const int* table = a.block_table + (size_t)seq * a.table_stride;
        int pages[2] = {-1, -1};
        for (int i = 0; i < 2; ++i)
          if (key0 + 64 * i < end) pages[i] = table[key0 / 64 + i];
        const int held = (pages[0] >= 0) + (pages[1] >= 0);      // a page that no query sees may be gone: its rows are masked
        mbar_expect_tx(k_full, held * (L::K_BYTES / 2));
        for (int i = 0; i < 2; ++i)
          if (pages[i] >= 0)
#pragma unroll
            for (int h = 0; h < HD / 64; ++h)
              tma_load_2d(base + L::K_OFF + h * (kKwKeys * 128) + i * 8192, &map_k, h * 64, (pages[i] * a.kv_heads + kh) * 64, k_full);
        for (int i = 0, st = 0, lap = 0; i < steps; ++i) {
          if (lap > 0 && !mbar_wait(q_free + 8 * st, (lap - 1) & 1)) { atomicExch(w.status, 85); break; }
          const int token = t_lo + (rank + i * ranks) * (kKwRows / G);
          mbar_expect_tx(q_full + 8 * st, L::Q_BYTES);
#pragma unroll
          for (int h = 0; h < HD / 64; ++h)
            tma_load_3d(base + L::Q_OFF + st * L::Q_BYTES + h * (kKwRows * 128), &map_q, h * 64, kh * G, (int)tok0 + token, q_full + 8 * st);
          if (++st == L::STAGES) { st = 0; ++lap; }
        }
      }
    } else if (warp == 1) {
      if (elect_one() && steps > 0) {
        constexpr uint32_t idesc = instr_desc(kKwKeys, kKwRows);
        bool ok = mbar_wait(k_full, 0);
        if (!ok) atomicExch(w.status, 86);
        for (int i = 0, st = 0, lap = 0; i < steps && ok; ++i) {
          const int b = i % kKwBuffers;
          if (!mbar_wait(q_full + 8 * st, lap & 1)) { atomicExch(w.status, 87); break; }
          if (i >= kKwBuffers && !mbar_wait(s_free + 8 * b, (i / kKwBuffers - 1) & 1)) { atomicExch(w.status, 88); break; }
          tc_fence_after();
#pragma unroll
          for (int h = 0; h < HD / 64; ++h) {
            const uint64_t dk = smem_desc(base + L::K_OFF + h * (kKwKeys * 128)), dq = smem_desc(base + L::Q_OFF + st * L::Q_BYTES + h * (kKwRows * 128));
#pragma unroll
            for (int k4 = 0; k4 < 4; ++k4)
              mma_bf16_ss(tmem + (uint32_t)(b * kKwRows), dk + (uint64_t)(k4 * 2), dq + (uint64_t)(k4 * 2), idesc, (h > 0 || k4 > 0) ? 1u : 0u);
          }
          mma_commit(q_free + 8 * st);
          mma_commit(s_full + 8 * b);
          if (++st == L::STAGES) { st = 0; ++lap; }
        }
      }
    } else if (warp == 2) {
      float* d = reinterpret_cast<float*>(smem + L::D_OFF);
      const int shift = 31 - __clz(G);      // (a divisor of 128)
      float v[4], next[4];
      auto ask = [&](int i, float (&x)[4]) {
        const int R0 = row_lo + (rank + i * ranks) * kKwRows;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int R = R0 + c * 32 + lane;
          x[c] = -INFINITY;
          if (i < steps && R < row_hi) x[c] = w.lse2[(tok0 + (R >> shift)) * a.heads + kh * G + (R & (G - 1))];
        }
      };
      ask(0, v);
      for (int i = 0; i < steps; ++i) {
        const int b = i % kKwBuffers;
        ask(i + 1, next);
        if (i >= kKwBuffers && !mbar_wait(d_free + 8 * b, (i / kKwBuffers - 1) & 1)) {
          if (lane == 0) atomicExch(w.status, 89);
          break;
        }
        // the negative, to be added; a row without weight or behind the last gives none
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          d[b * kKwRows + c * 32 + lane] = v[c] == -INFINITY ? -INFINITY : -v[c];
          v[c] = next[c];
        }
        mbar_arrive(d_full + 8 * b);
      }
    } else {
      const int set = part >> 1, col0 = (part & 1) * 64;
      const int key = key0 + quad * 32 + lane;
      const float* d = reinterpret_cast<const float*>(smem + L::D_OFF);
      // rows that see this key: [see_lo, see_hi)
      const int see_lo = max(0, key - past) * G;
      const int see_hi = key >= end ? 0 : a.window > 0 && key >= a.first ? (int)min((long long)row_hi, max(0ll, (long long)key + a.window - past) * G) : row_hi;
      bool ok = true;
      f32x2 s0 = 0, s1 = 0;
      const f32x2 scale2 = both(w.scale_log2);
      for (int i = set; i < steps; i += 2) {
        const int b = i % kKwBuffers, R0 = row_lo + (rank + i * ranks) * kKwRows + col0;
        if (ok && !(mbar_wait(s_full + 8 * b, (i / kKwBuffers) & 1) && mbar_wait(d_full + 8 * b, (i / kKwBuffers) & 1))) {
          ok = false;
          if (lane == 0) atomicExch(w.status, 90);
        }
        tc_fence_after();
        const bool masked = __any_sync(0xffffffffu, R0 < see_lo || R0 + 64 > see_hi);
#pragma unroll
        for (int c0 = 0; c0 < 64; c0 += 32) {
          uint32_t sr[32];
          tmem_ld32(tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(b * kKwRows + col0 + c0), sr);
          if (c0 == 32) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(s_free + 8 * b);      // the next product may overwrite the scores
          }
          const ulonglong2* dd = reinterpret_cast<const ulonglong2*>(d + b * kKwRows + col0 + c0);
          if (masked) {
            // what a row does not give is left out of the sum, not added as 2^(-inf - d): d is NaN where a query is
            const int first_c = see_lo - R0 - c0, end_c = see_hi - R0 - c0;
#pragma unroll
            for (int c = 0; c < 32; c += 4) {
              const ulonglong2 n = dd[c >> 2];
              const f32x2 x0 = fma2(pair_of(__uint_as_float(sr[c]), __uint_as_float(sr[c + 1])), scale2, n.x);
              const f32x2 x1 = fma2(pair_of(__uint_as_float(sr[c + 2]), __uint_as_float(sr[c + 3])), scale2, n.y);
              auto given = [&](int i, float p) { return i >= first_c && i < end_c ? p : 0.0f; };
              s0 = add2(s0, pair_of(given(c, kw_ex2(low_half(x0))), given(c + 1, kw_ex2(high_half(x0)))));
              s1 = add2(s1, pair_of(given(c + 2, kw_ex2(low_half(x1))), given(c + 3, kw_ex2(high_half(x1)))));
            }
            continue;
          }
#pragma unroll
          for (int c = 0; c < 32; c += 4) {
            const ulonglong2 n = dd[c >> 2];
            const f32x2 x0 = fma2(pair_of(__uint_as_float(sr[c]), __uint_as_float(sr[c + 1])), scale2, n.x);
            const f32x2 x1 = fma2(pair_of(__uint_as_float(sr[c + 2]), __uint_as_float(sr[c + 3])), scale2, n.y);
            s0 = add2(s0, pair_of(kw_ex2(low_half(x0)), kw_ex2(high_half(x0))));
            s1 = add2(s1, pair_of(kw_ex2(low_half(x1)), kw_ex2(high_half(x1))));
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(d_free + 8 * b);
      }
      sum = halves_sum(s0) + halves_sum(s1);
    }
    if (warp >= 3) reinterpret_cast<float*>(smem + L::SUM_OFF)[part * kKwKeys + quad * 32 + lane] = sum;
    tc_fence_before();
    __syncthreads();
    if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  } else if (!aligned && tid == 0) {
    atomicExch(w.status, 84);
  }
  pdl_launch_dependents();
  float total = 0.0f;
  if (all_steps > 0 && aligned && tid < kKwKeys) {
    const float* p = reinterpret_cast<const float*>(smem + L::SUM_OFF) + tid;
    total = (p[0] + p[kKwKeys]) + (p[2 * kKwKeys] + p[3 * kKwKeys]);
  }
  if (ranks > 1) {
    __syncwarp();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (tid < kKwKeys) {
      const uint32_t to = cluster_map(base + L::RANK_OFF + (rank * kKwKeys + tid) * 4, 0);
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(total) : "memory");
    }
    __syncthreads();
    cluster_sync_all();
    if (rank != 0) return;
    if (tid < kKwKeys) {
      const float* p = reinterpret_cast<const float*>(smem + L::RANK_OFF) + tid;
      total = 0.0f;
      for (int i = 0; i < ranks; ++i) total += p[i * kKwKeys];
    }
  }
  const int key = key0 + tid;
  if (tid < kKwKeys && key < end && key < a.capacity) {
    const size_t at = ((size_t)(a.slots ? a.slots[seq] : seq) * a.kv_heads + kh) * a.capacity + key;
    a.weights_out[at] = (key < past ? a.weights[at] : 0.0f) + total;
  }
}

// Blocks that share each of `tiles` key tiles whose walks are at most `longest` steps and `total` in all: while the longest walk is longer than an SM's
// share of all, or blocks are fewer than two an SM; a block keeps four steps of the longest.
static int kw_ranks(long long tiles, long long longest, long long total) {
  const long long sms = sm_count();
  int ranks = 1;
  while (ranks < 8 && longest / (2 * ranks) >= 4 && (longest * sms > total * ranks || tiles * ranks < 2 * sms)) ranks *= 2;
  return ranks;
}

static int kw_encode(CUtensorMap* map, int rank, const void* base, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box, const char* what) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(2, "attention_kept: the driver does not offer cuTensorMapEncodeTiled");
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (cuuint32_t)rank, const_cast<void*>(base), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : fail(2, "attention_kept: cuTensorMapEncodeTiled failed for %s with code %d", what, (int)r);
}

template <int HD>
static int launch_kw(const CUtensorMap& mq, const CUtensorMap& mk, KeptWeightsArgs w, int tile0, int tiles, int ranks, cudaStream_t s) {
  static std::atomic<unsigned long long> allowed;
  const cudaError_t e = allow_shared((const void*)kept_weights_kernel<HD>, KwLayout<HD>::TOTAL, allowed);
  if (e != cudaSuccess) return fail(2, "attention_kept: cannot reserve %d bytes of shared memory: %s", KwLayout<HD>::TOTAL, cudaGetErrorString(e));
  w.tile0 = tile0;
  w.k.splits = ranks;
  const dim3 grid((unsigned)(tiles * ranks), w.k.kv_heads, w.k.n_seqs);
  launch_clusters(pdl_mode() != 0, (unsigned)ranks, kept_weights_kernel<HD>, grid, dim3(kKwThreads), (size_t)KwLayout<HD>::TOTAL, s, mq, mk, w);
  return check_launch("attention_kept (weights)");
}

template <int HD>
static int launch_all(const CUtensorMap& mq, const CUtensorMap& mk, const KeptWeightsArgs& w, int max_count, int max_keys, cudaStream_t s) {
  const KeptArgs& k = w.k;
  const int G = k.heads / k.kv_heads, tiles = (max_keys + kKwKeys - 1) / kKwKeys;
  const long long pairs = (long long)k.n_seqs * k.kv_heads, longest = ((long long)max_count * G + kKwRows - 1) / kKwRows;
  if (k.window == 0) return launch_kw<HD>(mq, mk, w, 0, tiles, kw_ranks(pairs * tiles, longest, pairs * tiles * ((longest + 1) / 2)), s);
  // Under a window most keys are seen by a few steps' queries, the first ones by all: launches of their own where that is far apart (two prompts of 875
  // and 2,626 tokens, 32 / 8 heads, a window of 8, 4 first: one launch 102 us, with eight blocks a tile or one)
  const long long usual = std::min(longest, ((long long)(k.window + kKwKeys) * G + kKwRows - 1) / kKwRows + 1);
  const int all = std::min(tiles, (k.first + kKwKeys - 1) / kKwKeys);
  const int apart = all < tiles && longest > 2 * usual ? all : 0;
  if (apart) {
    const int rc = launch_kw<HD>(mq, mk, w, 0, apart, kw_ranks(pairs * apart, longest, pairs * apart * longest), s);
    if (rc) return rc;
  }
  const long long rest = pairs * (tiles - apart), walk = apart ? usual : longest;
  return launch_kw<HD>(mq, mk, w, apart, tiles - apart, kw_ranks(rest, walk, rest * usual), s);
}

int kept_weights_tc(const KeptArgs& k, const float* lse2, long long tokens, int max_count, int max_keys, long long pool_pages, int* status, cudaStream_t s) {
  const int G = k.heads / k.kv_heads;
  CUtensorMap mq, mk;
  {
    cuuint64_t dims[3] = {(cuuint64_t)k.head_dim, (cuuint64_t)k.heads, (cuuint64_t)tokens};
    cuuint64_t strides[2] = {(cuuint64_t)k.head_dim * 2, (cuuint64_t)k.heads * k.head_dim * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)G, (cuuint32_t)(kKwRows / G)};
    int rc = kw_encode(&mq, 3, k.q, dims, strides, box, "q");
    if (rc) return rc;
  }
  {
    cuuint64_t dims[2] = {(cuuint64_t)k.head_dim, (cuuint64_t)(pool_pages * k.kv_heads * 64)};
    cuuint64_t strides[1] = {(cuuint64_t)k.head_dim * 2};
    cuuint32_t box[2] = {64, 64};
    int rc = kw_encode(&mk, 2, k.k_pool, dims, strides, box, "the key pool");
    if (rc) return rc;
  }
  KeptWeightsArgs w{};
  w.k = k;
  w.lse2 = lse2;
  w.scale_log2 = k.scale * kKeptLog2e;
  w.status = status;
  return k.head_dim == 64 ? launch_all<64>(mq, mk, w, max_count, max_keys, s) : launch_all<128>(mq, mk, w, max_count, max_keys, s);
}

}  // namespace slb
