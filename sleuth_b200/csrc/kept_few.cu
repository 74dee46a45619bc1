// Attention over a cache of bounded size (kept.cuh) for steps of few tokens, bfloat16, heads of 64 and 128: single tokens, short turns.
//
// What such a step costs is the read of the keys and values that its queries see, so the work is the pages: every sequence has so many
// (kv head, page) units, and each block takes an equal run of the list of all units, whatever the sequences' lengths. A
// (sequence, kv head) that lies in one run is finished by its block; the others' shares wait in scratch for a second kernel.
//   * the last warp: asks TMA for the pages of the block's run, keys and values, into a ring (32 KB a stage at heads of 128; about 190 KB an SM,
//     where 43 KB hide a memory latency of a microsecond at full bandwidth);
//   * the other warps: mma.sync on the pages as they land. A (sequence, kv head) has up to R times 16 rows, row r being token r / G, query head r % G of
//     the group; R is 1, 2 or 4, by the longest share of a sequence, and all rows meet a page at once.
//     R = 1: four warps, a warp 16 of a page's keys, and two blocks an SM, so that one reads while the other joins its warps' results;
//     R = 2 and 4: eight warps, four or two for each 16 rows, a block an SM. Each warp keeps a running maximum, sum and weighted values of its own
//     keys; they are joined at the end of a (sequence, kv head), in the order of the warps. The weights of the softmax are rounded to bfloat16
//     for their product, as in the prompt kernels (the instruction takes no wider ones beside bfloat16 values); sums and maxima stay in 32 bits.
// (tcgen05 has nothing to win here: its tiles are 128 rows high, and rows are 2 to 64.)
// With weights wanted the scores go to scratch as they are formed (log2 units, 4 bytes for each row and key against 4 x head_dim for the
// key and value: 1 to 4 per cent more bytes), because the denominators are known at the end only; the second kernel turns them into weights.
// Where the units are few (few_cluster) a cluster of blocks shares one (sequence, kv head) instead: the shares meet in distributed shared memory, the
// scores stay in shared memory, and there is neither a second kernel nor scratch.
// Measured (device time): 64 sequences of 150 to 4,096 rows, a window of 2,048, 32 / 8 heads of 128, 76 us = 5.4 TB/s of 6.46; six of 9,000 to 30,000
// 76 us = 5.9 TB/s, with weights 90; eight of 2,049 with weights, 16 / 8 heads, by clusters 15.8 us = 4.3 TB/s (rows that L2 holds); four turns of 3 to 13
// tokens on 1,024 to 2,048 rows, 32 / 8 heads, 23 us, with weights 29; a token on 1,028 rows 7.8 us: launch, tables, one page, two meetings.
// Keys that no row of the 16 sees (stale rows of the last page, what lies between the first rows and the window) have their values
// replaced by zeros in registers, so that infinities or NaN in them do not meet a zero weight.
#include <math.h>

#include <algorithm>

#include "kept.cuh"
#include "mma_sync.cuh"
#include "tcgen05.cuh"

namespace slb {

constexpr int few_warps(int R) { return R == 1 ? 4 : 8; }
constexpr int few_blocks_an_sm(int R) { return R == 1 ? 2 : 1; }
constexpr int kFewMostRows = 64;      // rows of a (sequence, kv head)

// Shared memory: the ring (keys then values of a stage), queries [16 R][HD] as the ring's tiles lie, the warps' results [warps][rows][HD] float
// and [warps][rows][2], barriers, in clusters what the blocks exchange. As many stages as fit.
struct FewLayout {
  int stages, q_off, merge_off, ml_off, bar_off, total, merge_rows;
  int part_off, score_off, score_pitch;      // clusters: the block's joined results with maximum, sum, all blocks' maximum and denominator a row; its scores [rows][pitch]
};
// (228 KB an SM; a block has 1 KB of static shared memory and 1 KB that the driver takes)
constexpr int few_room(int R) { return (R == 1 ? 112 : 226) * 1024; }
static FewLayout few_layout(int HD, int R, int rows, int cluster_pages = 0, bool weights = false) {
  FewLayout l;
  const int stage = 2 * 64 * HD * 2;
  l.merge_rows = rows < 16 ? rows : 16;
  l.score_pitch = cluster_pages * 64 + 8;
  const int shared = cluster_pages ? rows * (HD * 4 + 16) + (weights ? rows * l.score_pitch * 4 : 0) + 32 : 0;
  const int rest = 16 * R * HD * 2 + few_warps(R) * l.merge_rows * (HD * 4 + 8) + 2 * 8 * 8 + shared;
  const int room = few_room(R);
  l.stages = (room - rest) / stage;
  if (l.stages > 8) l.stages = 8;
  if (cluster_pages && l.stages > cluster_pages) l.stages = cluster_pages;
  l.q_off = l.stages * stage;
  l.merge_off = l.q_off + 16 * R * HD * 2;
  l.ml_off = l.merge_off + few_warps(R) * l.merge_rows * HD * 4;
  l.bar_off = (l.ml_off + few_warps(R) * l.merge_rows * 8 + 7) & ~7;
  l.part_off = (l.bar_off + 2 * l.stages * 8 + 15) & ~15;
  l.score_off = l.part_off + rows * (HD * 4 + 16);      // (the last 8 bytes a row: its denominator)
  l.total = l.part_off + shared;
  return l;
}

struct FewArgs {
  KeptArgs k;
  float scale_log2;
  int max_count;        // no sequence brings more tokens (the room below is made for that)
  float* part;          // [blocks][2][16 R][HD] weighted values, then [blocks][2][16 R][2] maximum and sum
  float* part_ml;
  int2* info;           // [n, kv_heads] first block and number of blocks
  float* lse2;          // [tokens, H] denominators in log2 units
  float* scores;        // [tokens, H, score_stride] or null
  long long score_stride;
  int* status;
  FewLayout lay;
  int cluster, cluster_pages;        // blocks that share a (sequence, kv head), and the pages that each takes at most; 0: runs of all units
  int out_blocks, keys_a_block;      // the second kernel's blocks of a (sequence, kv head): some for outputs, one for so many keys
};

// The pages of a step of one sequence: the first ones and the window's, as one list.
struct PageRun {
  int nf, lo, count;      // pages 0 .. nf - 1, then lo ..
  __device__ __forceinline__ PageRun(int past, int tokens, int window, int first) {
    if (tokens <= 0) { nf = lo = count = 0; return; }
    const int key_lo = window_lo(past, window);
    nf = (min(first, key_lo) + 63) / 64;
    lo = max(key_lo / 64, nf);
    count = nf + (past + tokens - 1) / 64 - lo + 1;
  }
  __device__ __forceinline__ int page(int i) const { return i < nf ? i : lo + i - nf; }
};

__device__ __forceinline__ float few_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float2 peer_ld2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 peer_ld4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

// 16-byte piece of channel `col` of row `row` in a tile of 64 rows as TMA leaves it: 64 channels a half, pieces exchanged by the row.
template <int ROWS>
__device__ __forceinline__ uint32_t tile_at(int row, int col) {
  return (uint32_t)((col >> 6) * (ROWS * 128) + row * 128 + (((col >> 3) & 7) ^ (row & 7)) * 16);
}

template <int HD, int R, bool CLUSTER>
__global__ void __launch_bounds__((few_warps(R) + 1) * 32, few_blocks_an_sm(R))
kept_few_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, FewArgs fa) {
  constexpr int ROWS = 16 * R, KW = R == 4 ? 32 : 16, KB = KW / 16, WARPS = few_warps(R), GROUPS = WARPS / R, THREADS = (WARPS + 1) * 32, PAGE = 64 * HD * 2;
  const FewLayout& L = fa.lay;
  extern __shared__ __align__(1024) unsigned char smem[];
  __shared__ long long warp_units[WARPS + 1];
  __shared__ long long s_first;
  __shared__ int s_seq;
  const KeptArgs& a = fa.k;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = smem_addr(smem);
  if ((base & 1023u) != 0) {
    if (tid == 0) atomicExch(fa.status, 81);
    return;
  }
  const uint32_t bars = base + L.bar_off;
  if (tid == 0) {
    for (int i = 0; i < L.stages; ++i) {
      mbar_init(bars + 8 * i, 1);
      mbar_init(bars + 8 * (L.stages + i), WARPS);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_wait();

  // units of the sequences, and where this block's run begins
  const int G = a.heads / a.kv_heads;
  auto units_of = [&](int s) -> long long { return (long long)PageRun(a.past[s], min(a.counts[s], fa.max_count), a.window, a.first).count * a.kv_heads; };
  // CLUSTER: the blocks of a cluster share the pages of one (sequence, kv head); `u` counts the pages of that pair alone
  int seq, rank = 0;
  long long seq_first, u, u_hi, blocks = 1, total = 0;
  const int pair_kh = CLUSTER ? (int)(blockIdx.x / fa.cluster) % a.kv_heads : 0;
  if constexpr (CLUSTER) {
    rank = (int)cluster_ctarank();
    seq = (int)(blockIdx.x / fa.cluster) / a.kv_heads;
    const int pages = PageRun(a.past[seq], min(a.counts[seq], fa.max_count), a.window, a.first).count;
    if (pages == 0) {      // (the whole cluster)
      carry_weights(a, seq, pair_kh, 0, a.capacity, rank * THREADS + tid, fa.cluster * THREADS);
      return;
    }
    const int share = min((pages + fa.cluster - 1) / fa.cluster, fa.cluster_pages);
    seq_first = -(long long)pair_kh * pages;      // as if the kv head's units were the first
    u = min(pages, rank * share);
    u_hi = min(pages, (int)u + share);
    __syncthreads();
  } else {
    const int per = (a.n_seqs + THREADS - 1) / THREADS, q0 = min(a.n_seqs, tid * per), q1 = min(a.n_seqs, q0 + per);
    long long own = 0;
    for (int s = q0; s < q1; ++s) own += units_of(s);
    long long incl = own;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += y;
    }
    if (lane == 31) warp_units[warp] = incl;
    __syncthreads();
    long long before = 0;
#pragma unroll
    for (int w = 0; w <= WARPS; ++w) {
      if (w < warp) before += warp_units[w];
      total += warp_units[w];
    }
    blocks = min((long long)gridDim.x, total);
    if ((long long)blockIdx.x >= blocks) return;
    u = blockIdx.x * total / blocks;
    u_hi = (blockIdx.x + 1) * total / blocks;
    before += incl - own;
    if (own > 0 && u >= before && u < before + own) {
      for (int s = q0; s < q1; ++s) {
        const long long units = units_of(s);
        if (u < before + units) {
          s_seq = s;
          s_first = before;
          break;
        }
        before += units;
      }
    }
    __syncthreads();
    seq = s_seq;
    seq_first = s_first;      // units before this sequence
  }

  if (warp == WARPS) {
    // ---- the ring's pages ----
    int st = 0, lap = 0;
    bool ok = true;
    while (u < u_hi && ok) {
      const int count = min(a.counts[seq], fa.max_count), past = a.past[seq];
      const PageRun run(past, count, a.window, a.first);
      const long long units = (long long)run.count * a.kv_heads;
      const int* table = a.block_table + (size_t)seq * a.table_stride;
      const long long stop = min(u_hi, seq_first + units);
      while (u < stop && ok) {
        const int off = (int)((u - seq_first) % run.count), kh = (int)((u - seq_first) / run.count);
        const int n = (int)min((long long)(run.count - off), stop - u);
        for (int i0 = 0; i0 < n && ok; i0 += 32) {
          const int mine = i0 + lane < n ? table[run.page(off + i0 + lane)] : 0;
          for (int i = 0; i < min(32, n - i0); ++i) {
            const int page = __shfl_sync(0xffffffffu, mine, i);
            if (lap > 0 && !mbar_wait(bars + 8 * (L.stages + st), (lap - 1) & 1)) {
              if (lane == 0) atomicExch(fa.status, 82);
              ok = false;
              break;
            }
            if (elect_one()) {
              const int row = (page * a.kv_heads + kh) * 64;
              const uint32_t dst = base + st * 2 * PAGE;
              mbar_expect_tx(bars + 8 * st, 2 * PAGE);
#pragma unroll
              for (int h = 0; h < HD / 64; ++h) tma_load_2d(dst + h * 8192, &map_k, h * 64, row, bars + 8 * st);
#pragma unroll
              for (int h = 0; h < HD / 64; ++h) tma_load_2d(dst + PAGE + h * 8192, &map_v, h * 64, row, bars + 8 * st);
            }
            __syncwarp();
            if (++st == L.stages) { st = 0; ++lap; }
          }
        }
        u += n;
      }
      if (CLUSTER) break;
      seq_first += units;
      ++seq;
    }
    pdl_launch_dependents();
    if (!CLUSTER) return;
  } else {

  // ---- the products ----
  const int g = lane >> 2, t4 = lane & 3;
  const int rt = warp % R, key_in = warp / R * KW;      // which 16 of the rows; which keys of a page
  auto sync = [&]() { asm volatile("bar.sync 1, %0;" ::"n"(WARPS * 32) : "memory"); };
  int st = 0, lap = 0;
  bool ok = true;
  if constexpr (CLUSTER) {
    // a block without pages leaves an empty share
    if (u >= u_hi)
      for (int r = tid; r < min(16 * R, min(a.counts[seq], fa.max_count) * G); r += WARPS * 32)
        *reinterpret_cast<float2*>(smem + L.part_off + r * (HD * 4 + 16) + HD * 4) = make_float2(-INFINITY, 0.0f);
  }
  while (u < u_hi) {
    const int count = min(a.counts[seq], fa.max_count), past = a.past[seq];
    const PageRun run(past, count, a.window, a.first);
    const long long units = (long long)run.count * a.kv_heads;
    const int tok0 = a.seq_start[seq];
    const long long stop = min(u_hi, seq_first + units);
    while (u < stop) {
      const int off = (int)((u - seq_first) % run.count), kh = (int)((u - seq_first) / run.count);
      const int n = (int)min((long long)(run.count - off), stop - u);
      const int rows = min(ROWS, count * G);
      // queries (the previous kv head's results have been read: every warp has passed its last barrier)
      for (int e = tid; e < ROWS * (HD / 8); e += WARPS * 32) {
        const int r = e / (HD / 8), col = (e % (HD / 8)) * 8;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (r < rows) v = *reinterpret_cast<const uint4*>((const __nv_bfloat16*)a.q + ((size_t)(tok0 + r / G) * a.heads + kh * G + r % G) * HD + col);
        *reinterpret_cast<uint4*>(smem + L.q_off + tile_at<ROWS>(r, col)) = v;
      }
      sync();
      // (with 64 rows the fragments are read anew for every page: held they push others out of 168 registers, four turns of 3 to 13 tokens 31.0 us against 29.8)
      constexpr bool HOLD = R != 4;
      uint32_t qf[HOLD ? HD / 16 : 1][4];
      if constexpr (HOLD)
#pragma unroll
      for (int kb = 0; kb < HD / 16; ++kb) ldmatrix_x4(qf[kb], base + L.q_off + tile_at<ROWS>(rt * 16 + (lane & 15), kb * 16 + ((lane >> 4) << 3)));
      int pos[2], lo[2];
      float* score_row[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = rt * 16 + g + 8 * h;
        pos[h] = r < rows ? past + r / G : -1;
        lo[h] = window_lo(pos[h], a.window);
        if (CLUSTER) score_row[h] = a.weights && r < rows ? reinterpret_cast<float*>(smem + L.score_off) + r * L.score_pitch : nullptr;
        else score_row[h] = fa.scores && r < rows ? fa.scores + ((size_t)(tok0 + r / G) * a.heads + kh * G + r % G) * fa.score_stride : nullptr;
      }
      // what the 16 rows of this warp see: all of them from see_lo (or below `first`) to see_hi, none beyond any_hi or below any_lo
      const int r_first = rt * 16, r_last = min(rows, r_first + 16) - 1;
      const bool idle = r_first > r_last;
      const int any_lo = window_lo(past + r_first / G, a.window), any_hi = past + r_last / G;
      const int all_lo = window_lo(any_hi, a.window), all_hi = past + r_first / G;

      float o[HD / 8][4];
#pragma unroll
      for (int i = 0; i < HD / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
      float m_r[2] = {-INFINITY, -INFINITY}, l_r[2] = {0.0f, 0.0f};
      for (int i = 0; i < n; ++i) {
        if (ok && !mbar_wait(bars + 8 * st, lap & 1)) {
          ok = false;
          if (lane == 0) atomicExch(fa.status, 83);
        }
        const int key0 = run.page(off + i) * 64 + key_in;
        const bool none = idle || key0 > any_hi || (key0 + KW - 1 < any_lo && key0 >= a.first);
        if (!none) {
          const uint32_t kS = base + st * 2 * PAGE, vS = kS + PAGE;
          float s[2 * KB][4];
#pragma unroll
          for (int j = 0; j < 2 * KB; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.0f;
#pragma unroll
          for (int kb = 0; kb < HD / 16; ++kb) {
            if constexpr (!HOLD) ldmatrix_x4(qf[0], base + L.q_off + tile_at<ROWS>(rt * 16 + (lane & 15), kb * 16 + ((lane >> 4) << 3)));
            const uint32_t (&q)[4] = qf[HOLD ? kb : 0];
#pragma unroll
            for (int b = 0; b < KB; ++b) {
              uint32_t kf[4];
              ldmatrix_x4(kf, kS + tile_at<64>(key_in + b * 16 + (lane & 7) + ((lane >> 4) << 3), kb * 16 + (((lane >> 3) & 1) << 3)));
              mma_bf16(s[2 * b], q, kf[0], kf[1]);
              mma_bf16(s[2 * b + 1], q, kf[2], kf[3]);
            }
          }
          const bool whole = key0 + KW - 1 <= all_hi && (key0 >= all_lo || key0 + KW <= a.first);
#pragma unroll
          for (int j = 0; j < 2 * KB; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int key = key0 + j * 8 + 2 * t4 + (e & 1);
              s[j][e] *= fa.scale_log2;
              if (!whole && !sees(key, pos[e >> 1], lo[e >> 1], a.first)) s[j][e] = -INFINITY;
            }
          if (CLUSTER ? a.weights != nullptr : fa.scores != nullptr) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (score_row[h] != nullptr) {
#pragma unroll
                for (int j = 0; j < 2 * KB; ++j) {
                  const int key = (CLUSTER ? i * 64 + key_in : key0) + j * 8 + 2 * t4;      // (clusters: by the page's place in the block)
                  if (CLUSTER || key < fa.score_stride) *reinterpret_cast<float2*>(score_row[h] + key) = make_float2(s[j][2 * h], s[j][2 * h + 1]);
                }
              }
          }
          float alpha[2], m_use[2];
          bool moved = false;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < 2 * KB; ++j) mx = fmaxf(mx, fmaxf(s[j][2 * h], s[j][2 * h + 1]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float m_new = fmaxf(m_r[h], mx);
            m_use[h] = m_new == -INFINITY ? 0.0f : m_new;
            alpha[h] = few_ex2(m_r[h] - m_use[h]);
            moved = moved || m_new > m_r[h];
            m_r[h] = m_new;
          }
          uint32_t pf[KB][4];
          float sum[2] = {0.0f, 0.0f};
#pragma unroll
          for (int j = 0; j < 2 * KB; ++j) {
            const float p0 = few_ex2(s[j][0] - m_use[0]), p1 = few_ex2(s[j][1] - m_use[0]);
            const float p2 = few_ex2(s[j][2] - m_use[1]), p3 = few_ex2(s[j][3] - m_use[1]);
            sum[0] += p0 + p1;
            sum[1] += p2 + p3;
            pf[j >> 1][(j & 1) * 2 + 0] = pack_bf16(p0, p1);
            pf[j >> 1][(j & 1) * 2 + 1] = pack_bf16(p2, p3);
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) l_r[h] = l_r[h] * alpha[h] + sum[h];
          if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int c = 0; c < HD / 8; ++c) {
              o[c][0] *= alpha[0]; o[c][1] *= alpha[0];
              o[c][2] *= alpha[1]; o[c][3] *= alpha[1];
            }
          }
          if (whole) {
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
              for (int dp = 0; dp < HD / 16; ++dp) {
                uint32_t vf[4];
                ldmatrix_x4_trans(vf, vS + tile_at<64>(key_in + b * 16 + (lane & 15), dp * 16 + ((lane >> 4) << 3)));
                mma_bf16(o[2 * dp], pf[b], vf[0], vf[1]);
                mma_bf16(o[2 * dp + 1], pf[b], vf[2], vf[3]);
              }
          } else {
#pragma unroll
            for (int b = 0; b < KB; ++b) {
              // a lane holds the values of keys 2 t4, 2 t4 + 1 (and + 8) in the halves of a register
              uint32_t live[2];
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int key = key0 + b * 16 + h * 8 + 2 * t4;
                live[h] = (sees(key, any_hi, any_lo, a.first) ? 0x0000ffffu : 0u) | (sees(key + 1, any_hi, any_lo, a.first) ? 0xffff0000u : 0u);
              }
#pragma unroll
              for (int dp = 0; dp < HD / 16; ++dp) {
                uint32_t vf[4];
                ldmatrix_x4_trans(vf, vS + tile_at<64>(key_in + b * 16 + (lane & 15), dp * 16 + ((lane >> 4) << 3)));
                mma_bf16(o[2 * dp], pf[b], vf[0] & live[0], vf[1] & live[1]);
                mma_bf16(o[2 * dp + 1], pf[b], vf[2] & live[0], vf[3] & live[1]);
              }
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bars + 8 * (L.stages + st));
        if (++st == L.stages) { st = 0; ++lap; }
      }

      // join the warps that share these rows
      float* mo = reinterpret_cast<float*>(smem + L.merge_off);      // [warps][rows][HD]
      float* ml = reinterpret_cast<float*>(smem + L.ml_off);         // [warps][rows][2]
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        l_r[h] += __shfl_xor_sync(0xffffffffu, l_r[h], 1);
        l_r[h] += __shfl_xor_sync(0xffffffffu, l_r[h], 2);
        const int r = g + 8 * h;
        if (rt * 16 + r >= rows) continue;
        if (t4 == 0) *reinterpret_cast<float2*>(ml + (warp * L.merge_rows + r) * 2) = make_float2(m_r[h], l_r[h]);
        // (rows of a warp start 8 x 4-byte banks apart by the row, so that the eight rows of a store meet different banks)
#pragma unroll
        for (int c = 0; c < HD / 8; ++c)
          *reinterpret_cast<float2*>(mo + (warp * L.merge_rows + r) * HD + ((c * 8 + 2 * t4) ^ ((r & 3) << 3))) = make_float2(o[c][2 * h], o[c][2 * h + 1]);
      }
      sync();
      const bool begins = off == 0, complete = begins && n == run.count;
      const long long pair_lo = seq_first + (long long)kh * run.count;
      const int first_block = blockIdx.x;
      if (!CLUSTER && begins && tid == 0) {
        const long long last = pair_lo + run.count - 1;
        const int last_block = (int)(((last + 1) * blocks - 1) / total);
        fa.info[(size_t)seq * a.kv_heads + kh] = make_int2(first_block, last_block - first_block + 1);
      }
      const size_t slot = ((size_t)blockIdx.x * 2 + (begins ? 1 : 0)) * ROWS;
      for (int e = tid; e < rows * (HD / 4); e += WARPS * 32) {
        const int r = e / (HD / 4), d = (e % (HD / 4)) * 4, in = r & 15;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < GROUPS; ++w) M = fmaxf(M, ml[((w * R + (r >> 4)) * L.merge_rows + in) * 2]);
        const float top = M == -INFINITY ? 0.0f : M;
        float sum = 0.0f;
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < GROUPS; ++w) {
          const int at = (w * R + (r >> 4)) * L.merge_rows + in;
          const float f = few_ex2(ml[at * 2] - top);
          const float4 v = *reinterpret_cast<const float4*>(mo + at * HD + (d ^ ((in & 3) << 3)));
          sum += ml[at * 2 + 1] * f;
          acc.x += v.x * f; acc.y += v.y * f; acc.z += v.z * f; acc.w += v.w * f;
        }
        const size_t row = (size_t)(tok0 + r / G) * a.heads + kh * G + r % G;
        if (CLUSTER) {
          float* slot = reinterpret_cast<float*>(smem + L.part_off + r * (HD * 4 + 16));
          *reinterpret_cast<float4*>(slot + d) = acc;
          if (d == 0) *reinterpret_cast<float2*>(slot + HD) = make_float2(M, sum);
        } else if (complete) {
          const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
          uint2 pk;
          pk.x = pack_bf16(acc.x * inv, acc.y * inv);
          pk.y = pack_bf16(acc.z * inv, acc.w * inv);
          *reinterpret_cast<uint2*>((__nv_bfloat16*)a.out + row * HD + d) = pk;
          if (d == 0) {
            const float lse2 = sum == 0.0f ? -INFINITY : top + log2f(sum);
            if (fa.lse2) fa.lse2[row] = lse2;
            if (a.lse) a.lse[row] = lse2 * 0.6931471805599453f;
          }
        } else {
          *reinterpret_cast<float4*>(fa.part + (slot + r) * HD + d) = acc;
          if (d == 0) *reinterpret_cast<float2*>(fa.part_ml + (slot + r) * 2) = make_float2(M, sum);
        }
      }
      sync();
      u += n;
    }
    if (CLUSTER) break;
    seq_first += units;
    ++seq;
  }
  }
  if constexpr (CLUSTER) {
    const int count = min(a.counts[seq], fa.max_count), past = a.past[seq], tok0 = a.seq_start[seq], rows = min(ROWS, count * G);
    const PageRun run(past, count, a.window, a.first);
    const int share = min((run.count + fa.cluster - 1) / fa.cluster, fa.cluster_pages), first_page = min(run.count, rank * share);
    const int my_pages = min(run.count, first_page + share) - first_page;
    __syncthreads();         // (the cluster's barrier counts warps: they have to come to it whole)
    cluster_sync_all();
    auto peer = [&](int c, int r, int word) { return cluster_map(base + L.part_off + r * (HD * 4 + 16) + word * 4, c); };
    // denominators: a thread a row
    for (int r = tid; r < rows; r += THREADS) {
      float M = -INFINITY, D = 0.0f;
      for (int c = 0; c < fa.cluster; ++c) {
        const float2 p = peer_ld2(peer(c, r, HD));
        const float top = fmaxf(M, p.x), use = top == -INFINITY ? 0.0f : top;
        D = D * few_ex2(M - use) + p.y * few_ex2(p.x - use);
        M = top;
      }
      const float lse2 = D == 0.0f ? -INFINITY : M + log2f(D);
      float* slot = reinterpret_cast<float*>(smem + L.part_off + r * (HD * 4 + 16));
      *reinterpret_cast<float2*>(slot + HD + 2) = make_float2(M, lse2 == -INFINITY ? INFINITY : lse2);
      if (rank == 0 && a.lse) a.lse[(size_t)(tok0 + r / G) * a.heads + pair_kh * G + r % G] = lse2 * 0.6931471805599453f;
    }
    __syncthreads();
    for (int e = rank * THREADS + tid; e < rows * (HD / 4); e += fa.cluster * THREADS) {
      const int r = e / (HD / 4), d = (e % (HD / 4)) * 4;
      const float M = reinterpret_cast<const float*>(smem + L.part_off + r * (HD * 4 + 16))[HD + 2], use = M == -INFINITY ? 0.0f : M;
      float D = 0.0f;
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int c = 0; c < fa.cluster; ++c) {
        const float2 p = peer_ld2(peer(c, r, HD));
        const float f = few_ex2(p.x - use);
        if (p.x == -INFINITY && p.y == 0.0f) continue;      // a share without keys (its values were never written)
        const float4 v = peer_ld4(peer(c, r, d));
        D += p.y * f;
        acc.x += v.x * f; acc.y += v.y * f; acc.z += v.z * f; acc.w += v.w * f;
      }
      const float inv = D == 0.0f ? 0.0f : 1.0f / D;
      uint2 pk;
      pk.x = pack_bf16(acc.x * inv, acc.y * inv);
      pk.y = pack_bf16(acc.z * inv, acc.w * inv);
      *reinterpret_cast<uint2*>((__nv_bfloat16*)a.out + ((size_t)(tok0 + r / G) * a.heads + pair_kh * G + r % G) * HD + d) = pk;
    }
    if (a.weights) {
      const int end = past + count;
      const size_t at0 = ((size_t)(a.slots ? a.slots[seq] : seq) * a.kv_heads + pair_kh) * a.capacity;
      const float* scores = reinterpret_cast<const float*>(smem + L.score_off);
      for (int k = tid; k < my_pages * 64; k += THREADS) {
        const int key = run.page(first_page + (k >> 6)) * 64 + (k & 63);
        if (key >= end || key >= a.capacity) continue;
        float w = key < past ? a.weights[at0 + key] : 0.0f, gained = 0.0f;
        for (int r = 0; r < rows; ++r) {
          const int pos = past + r / G;
          const float d = reinterpret_cast<const float*>(smem + L.part_off + r * (HD * 4 + 16))[HD + 3];
          if (sees(key, pos, window_lo(pos, a.window), a.first)) gained += few_ex2(scores[r * L.score_pitch + k] - d);
        }
        a.weights_out[at0 + key] = w + gained;
      }
      // rows that no query of the step sees: nothing is gathered
      if (a.weights_out != a.weights)
        for (int key = run.nf * 64 + rank * THREADS + tid; key < min(run.lo * 64, end); key += fa.cluster * THREADS)
          if (key < a.capacity) a.weights_out[at0 + key] = a.weights[at0 + key];
    }
    __syncthreads();
    cluster_sync_all();      // the others may still be reading this block's results
  }
}

// Joins the shares of what no block finished alone, and turns scores into weights: of the blocks of a (sequence, kv head) the first few take
// outputs, the others `keys_a_block` keys each.
template <int HD, int R>
__global__ void __launch_bounds__(256, 4) kept_few_finish_kernel(FewArgs fa) {
  pdl_wait();
  const KeptArgs& a = fa.k;
  constexpr int ROWS = 16 * R;
  __shared__ float lse_s[kFewMostRows];
  __shared__ int pos_s[kFewMostRows];
  __shared__ long long row_s[kFewMostRows];
  __shared__ float sum_s[4][256];
  const int tid = threadIdx.x;
  const int kh = blockIdx.y, seq = blockIdx.z, G = a.heads / a.kv_heads;
  const int count = min(a.counts[seq], fa.max_count), past = a.past[seq], tok0 = a.seq_start[seq], rows_total = count * G;
  if (count <= 0) {
    if ((int)blockIdx.x >= fa.out_blocks) {
      const long long lo = (long long)((int)blockIdx.x - fa.out_blocks) * fa.keys_a_block;
      carry_weights(a, seq, kh, lo, lo + fa.keys_a_block, tid, 256);
    }
    return;
  }
  const int2 in = fa.info[(size_t)seq * a.kv_heads + kh];
  auto row_of = [&](int r) { return (size_t)(tok0 + r / G) * a.heads + kh * G + r % G; };
  auto slot_of = [&](int i) { return ((size_t)(in.x + i) * 2 + (i == 0 ? 1 : 0)) * ROWS; };
  const bool outputs = (int)blockIdx.x < fa.out_blocks;
  const int key_begin = ((int)blockIdx.x - fa.out_blocks) * fa.keys_a_block, end = past + count;
  if (!outputs && key_begin >= end) return;
  if (outputs) {
    if (in.y == 1) return;      // its block has finished it
    for (int e = blockIdx.x * 256 + tid; e < rows_total * (HD / 4); e += fa.out_blocks * 256) {
      const int r = e / (HD / 4), d = (e % (HD / 4)) * 4;
      float M = -INFINITY, L = 0.0f;
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int i0 = 0; i0 < in.y; i0 += 8) {
        float2 p[8];
        float4 v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const size_t at = slot_of(i0 + i < in.y ? i0 + i : 0) + r;
          p[i] = *reinterpret_cast<const float2*>(fa.part_ml + at * 2);
          v[i] = *reinterpret_cast<const float4*>(fa.part + at * HD + d);
          if (i0 + i >= in.y) p[i].x = -INFINITY;
        }
        float top = M;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, p[i].x);
        const float use = top == -INFINITY ? 0.0f : top, keep = few_ex2(M - use);
        L *= keep;
        acc.x *= keep; acc.y *= keep; acc.z *= keep; acc.w *= keep;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float f = few_ex2(p[i].x - use);
          if (i0 + i < in.y) {      // (a share whose scores were all NaN has maximum -inf and a sum of NaN)
            L += p[i].y * f;
            acc.x += v[i].x * f; acc.y += v[i].y * f; acc.z += v[i].z * f; acc.w += v[i].w * f;
          }
        }
        M = top;
      }
      const float inv = L == 0.0f ? 0.0f : 1.0f / L;
      uint2 pk;
      pk.x = pack_bf16(acc.x * inv, acc.y * inv);
      pk.y = pack_bf16(acc.z * inv, acc.w * inv);
      *reinterpret_cast<uint2*>((__nv_bfloat16*)a.out + row_of(r) * HD + d) = pk;
      if (d == 0 && a.lse) a.lse[row_of(r)] = L == 0.0f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
    }
    return;
  }
  // denominators, a thread a row
  if (tid < rows_total) {
    const size_t row = row_of(tid);
    float v;
    if (in.y == 1) {
      v = fa.lse2[row];
    } else {
      float M = -INFINITY, L = 0.0f;
      for (int i0 = 0; i0 < in.y; i0 += 8) {
        float2 p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          p[i] = *reinterpret_cast<const float2*>(fa.part_ml + (slot_of(i0 + i < in.y ? i0 + i : 0) + tid) * 2);
          if (i0 + i >= in.y) p[i] = make_float2(-INFINITY, 0.0f);
        }
        float top = M;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, p[i].x);
        const float use = top == -INFINITY ? 0.0f : top;
        L *= few_ex2(M - use);
#pragma unroll
        for (int i = 0; i < 8; ++i) L += p[i].y * few_ex2(p[i].x - use);
        M = top;
      }
      v = L == 0.0f ? -INFINITY : M + log2f(L);
    }
    lse_s[tid] = v == -INFINITY ? INFINITY : v;      // a row without weight gives none
    pos_s[tid] = past + tid / G;
    row_s[tid] = (long long)row * fa.score_stride;
  }
  __syncthreads();
  const size_t at0 = ((size_t)(a.slots ? a.slots[seq] : seq) * a.kv_heads + kh) * a.capacity;
  const int key_end = (int)min((long long)min(end, key_begin + fa.keys_a_block), a.capacity);
  // Four keys a thread. Up to eight rows a thread takes them all, their loads under way together; with more, four groups of threads take the rows
  // r = group, group + 4, ..., and the groups' sums are added in their order.
  const bool alone = rows_total <= 8;
  const int quads = alone ? 256 : 64, quad = tid & (quads - 1), group = alone ? 0 : tid >> 6, step = alone ? 1 : 4;
  for (int key0 = key_begin; key0 < key_end; key0 += 4 * quads) {
    const int key = key0 + 4 * quad;
    float4 gained = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float before[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) before[i] = alone && key + i < min(past, key_end) ? a.weights[at0 + key + i] : 0.0f;
    if (key < key_end) {
      for (int r0 = group; r0 < rows_total; r0 += 8 * step) {
        float4 v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = r0 + i * step;
          v[i] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
          if (r >= rows_total) continue;
          const int pos = pos_s[r], lo = window_lo(pos, a.window);
          if (key > pos || (key + 3 < lo && key >= a.first)) continue;
          v[i] = *reinterpret_cast<const float4*>(fa.scores + row_s[r] + key);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = r0 + i * step;
          if (r >= rows_total) continue;
          const int pos = pos_s[r], lo = window_lo(pos, a.window);
          const float d = lse_s[r];
          gained.x += sees(key, pos, lo, a.first) ? few_ex2(v[i].x - d) : 0.0f;
          gained.y += sees(key + 1, pos, lo, a.first) ? few_ex2(v[i].y - d) : 0.0f;
          gained.z += sees(key + 2, pos, lo, a.first) ? few_ex2(v[i].z - d) : 0.0f;
          gained.w += sees(key + 3, pos, lo, a.first) ? few_ex2(v[i].w - d) : 0.0f;
        }
      }
    }
    if (alone) {
      const float sum[4] = {before[0] + gained.x, before[1] + gained.y, before[2] + gained.z, before[3] + gained.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (key + i < key_end) a.weights_out[at0 + key + i] = sum[i];
      continue;
    }
    __syncthreads();
    *reinterpret_cast<float4*>(&sum_s[group][4 * quad]) = gained;
    __syncthreads();
    if (key0 + tid < key_end) {
      const float w = key0 + tid < past ? a.weights[at0 + key0 + tid] : 0.0f;
      a.weights_out[at0 + key0 + tid] = w + ((sum_s[0][tid] + sum_s[1][tid]) + (sum_s[2][tid] + sum_s[3][tid]));
    }
  }
}

// R: kept_few_takes admits 64 rows.
static int few_row_tiles(int max_count, int G) { return max_count * G <= 16 ? 1 : max_count * G <= 32 ? 2 : 4; }

// Where the pieces of scratch lie, in floats.
struct FewScratch {
  long long part, part_ml, info, lse2, scores, total, score_stride;
  int blocks, cluster, cluster_pages;
};

// Whether blocks of a cluster share each (sequence, kv head), and how many: then no second kernel and no scratch is needed (a chat's token on 17 pages:
// 10.1 us by runs of units, 7.9 by clusters; eight tokens on 2,049 rows 19.4 / 15.6), but a cluster waits for its longest sequence alone, so only where all clusters run at once and
// no block takes more than ten pages (8 KB of scores a row at most).
static void few_cluster(int n_seqs, int max_count, int heads, int kv_heads, int head_dim, int max_keys, bool weights, int window, int first, FewScratch& f) {
  const int G = heads / kv_heads, R = few_row_tiles(max_count, G);
  f.cluster = f.cluster_pages = 0;
  if (R > 2) return;
  long long pages = (max_keys + 63) / 64;
  if (window > 0) pages = std::min(pages, (long long)(window + max_count - 2) / 64 + 2 + (first + 63) / 64);
  const long long pairs = (long long)n_seqs * kv_heads, resident = (long long)sm_count() * few_blocks_an_sm(R);
  if (pairs > resident) return;
  int c = 8;
  while (c > 1 && (pairs * c > resident || c >= 2 * pages)) c /= 2;
  const int each = (int)((pages + c - 1) / c);
  if (each > 10 || few_layout(head_dim, R, max_count * G, each, weights).stages < std::min(2, each)) return;
  f.cluster = c;
  f.cluster_pages = each;
}

static FewScratch few_scratch(long long tokens, int n_seqs, int max_count, int heads, int kv_heads, int head_dim, int max_keys, bool weights, int window, int first) {
  FewScratch f{};
  const int G = heads / kv_heads, R = few_row_tiles(max_count, G);
  few_cluster(n_seqs, max_count, heads, kv_heads, head_dim, max_keys, weights, window, first, f);
  if (f.cluster) return f;
  const long long units = (long long)n_seqs * kv_heads * ((max_keys + 63) / 64);
  const long long most = (long long)sm_count() * few_blocks_an_sm(R);
  f.blocks = (int)(units < most ? units : most);      // as many as run at once; none without a page
  const long long slots = 2ll * f.blocks * 16 * R;
  long long at = 0;
  auto take = [&](long long n) { const long long o = at; at += (n + 3) & ~3ll; return o; };
  f.part = take(slots * head_dim);
  f.part_ml = take(slots * 2);
  f.info = take(2ll * n_seqs * kv_heads);
  f.lse2 = weights ? take(tokens * heads) : 0;
  f.score_stride = (max_keys + 3) & ~3;
  f.scores = weights ? take(tokens * heads * f.score_stride) : 0;
  f.total = at;
  return f;
}

template <int HD, int R>
static int launch_few_cluster(const CUtensorMap& mk, const CUtensorMap& mv, const FewArgs& fa, cudaStream_t s) {
  static std::atomic<unsigned long long> allowed;
  const cudaError_t e = allow_shared((const void*)kept_few_kernel<HD, R, true>, few_room(R), allowed);
  if (e != cudaSuccess) return fail(2, "attention_kept: cannot reserve shared memory: %s", cudaGetErrorString(e));
  launch_clusters(false, (unsigned)fa.cluster, kept_few_kernel<HD, R, true>, dim3(fa.cluster * fa.k.kv_heads * fa.k.n_seqs), dim3((few_warps(R) + 1) * 32),
                  (size_t)fa.lay.total, s, mk, mv, fa);
  return check_launch("attention_kept (few tokens, clusters)");
}

template <int HD, int R>
static int launch_few(const CUtensorMap& mk, const CUtensorMap& mv, FewArgs fa, int blocks, int max_keys, int max_count, cudaStream_t s) {
  const int rows = max_count * (fa.k.heads / fa.k.kv_heads);
  fa.lay = few_layout(HD, R, rows, fa.cluster_pages, fa.k.weights != nullptr);
  if constexpr (R <= 2)
    if (fa.cluster) return launch_few_cluster<HD, R>(mk, mv, fa, s);
  static std::atomic<unsigned long long> allowed;
  const cudaError_t e = allow_shared((const void*)kept_few_kernel<HD, R, false>, few_room(R), allowed);
  if (e != cudaSuccess) return fail(2, "attention_kept: cannot reserve shared memory: %s", cudaGetErrorString(e));
  launch(kept_few_kernel<HD, R, false>, dim3(blocks), dim3((few_warps(R) + 1) * 32), (size_t)fa.lay.total, s, mk, mv, fa);
  const int rc = check_launch("attention_kept (few tokens)");
  if (rc) return rc;
  const long long pairs = (long long)fa.k.n_seqs * fa.k.kv_heads;
  fa.out_blocks = (rows * (HD / 4) + 255) / 256;
  long long key_blocks = 0;
  if (fa.scores) {      // about eight blocks an SM in all; each works out the denominators for itself
    const long long wanted = 8ll * sm_count() / pairs;
    fa.keys_a_block = (int)((max_keys / (wanted < 1 ? 1 : wanted) + 256) / 256 * 256);
    key_blocks = (max_keys + fa.keys_a_block - 1) / fa.keys_a_block;
  }
  launch_prefetching(kept_few_finish_kernel<HD, R>, dim3((unsigned)(fa.out_blocks + key_blocks), fa.k.kv_heads, fa.k.n_seqs), dim3(256), 0, s, fa);
  return check_launch("attention_kept (few tokens, joined)");
}

static int encode_pool(CUtensorMap* map, const void* base, long long rows, int head_dim, const char* what) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(2, "attention_kept: the driver does not offer cuTensorMapEncodeTiled");
  cuuint64_t dims[2] = {(cuuint64_t)head_dim, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)head_dim * 2};
  cuuint32_t box[2] = {64, 64}, estr[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : fail(2, "attention_kept: cuTensorMapEncodeTiled failed for %s with code %d", what, (int)r);
}

// Floats of scratch for scores: a gigabyte (64 sequences of 32 heads in a table of 131,072 rows). Single tokens and turns with weights beyond it take the
// prompt kernels, whose tiles of 128 rows they leave mostly empty.
constexpr long long kMostScores = 1ll << 28;

bool kept_few_takes(long long tokens, int max_count, int heads, int kv_heads, int head_dim, int max_keys, int dtype, bool weights) {
  return dtype == kBF16 && (head_dim == 64 || head_dim == 128) && (long long)max_count * (heads / kv_heads) <= kFewMostRows &&
         (!weights || tokens * heads * max_keys <= kMostScores);
}

long long kept_few_floats(long long tokens, int n_seqs, int max_count, int heads, int kv_heads, int head_dim, int max_keys, bool weights) {
  // (asked without the window: what a step without one takes is enough for every other, by runs of units or by clusters)
  FewScratch runs = few_scratch(tokens, n_seqs, max_count, heads, kv_heads, head_dim, max_keys, weights, 0, 0);
  return runs.total;
}

int kept_few(const KeptArgs& a, long long tokens, int max_count, int max_keys, long long pool_pages, int* status, cudaStream_t s) {
  SLB_REQUIRE(pool_pages * a.kv_heads * 64 < (1ll << 31), "attention_kept: the pool has too many rows for one tensor map");
  SLB_REQUIRE((uintptr_t)a.q % 16 == 0 && (uintptr_t)a.k_pool % 16 == 0 && (uintptr_t)a.v_pool % 16 == 0 && (uintptr_t)a.out % 16 == 0 &&
              (uintptr_t)a.scratch % 16 == 0, "attention_kept: q, out, scratch and the pools must be 16-byte aligned");
  SLB_REQUIRE(status != nullptr, "attention_kept: no status word");
  CUtensorMap mk, mv;
  int rc = encode_pool(&mk, a.k_pool, pool_pages * a.kv_heads * 64, a.head_dim, "the key pool");
  if (rc == 0) rc = encode_pool(&mv, a.v_pool, pool_pages * a.kv_heads * 64, a.head_dim, "the value pool");
  if (rc) return rc;
  const bool weights = a.weights != nullptr;
  const FewScratch f = few_scratch(tokens, a.n_seqs, max_count, a.heads, a.kv_heads, a.head_dim, max_keys, weights, a.window, a.first);
  FewArgs fa{};
  fa.k = a;
  fa.scale_log2 = a.scale * kKeptLog2e;
  fa.max_count = max_count;
  fa.cluster = f.cluster;
  fa.cluster_pages = f.cluster_pages;
  fa.part = a.scratch + f.part;
  fa.part_ml = a.scratch + f.part_ml;
  fa.info = reinterpret_cast<int2*>(a.scratch + f.info);
  fa.lse2 = weights && !f.cluster ? a.scratch + f.lse2 : nullptr;
  fa.scores = weights && !f.cluster ? a.scratch + f.scores : nullptr;
  fa.score_stride = f.score_stride;
  fa.status = status;
  const int R = few_row_tiles(max_count, a.heads / a.kv_heads);
  if (a.head_dim == 128)
    return R == 1 ? launch_few<128, 1>(mk, mv, fa, f.blocks, max_keys, max_count, s) : R == 2 ? launch_few<128, 2>(mk, mv, fa, f.blocks, max_keys, max_count, s)
                                                                           : launch_few<128, 4>(mk, mv, fa, f.blocks, max_keys, max_count, s);
  return R == 1 ? launch_few<64, 1>(mk, mv, fa, f.blocks, max_keys, max_count, s) : R == 2 ? launch_few<64, 2>(mk, mv, fa, f.blocks, max_keys, max_count, s)
                                                                        : launch_few<64, 4>(mk, mv, fa, f.blocks, max_keys, max_count, s);
}

}  // namespace slb
