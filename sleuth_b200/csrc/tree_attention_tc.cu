// Attention of drafted nodes (tree.cuh) on the tcgen05 tensor cores: bfloat16, heads of 64 and 128, any number of query heads a key/value head.
//
// What such a step costs is the read of the keys and values (up to 256 rows of queries meet each: 512 FLOP a byte at most), so the work is the pages: every sequence
// has (kv head, tile of 256 rows, page) units, and each block, one an SM, takes an equal run of the list of all units, whatever the sequences' lengths. What a run
// holds of one (sequence, kv head, tile) is a segment. A (sequence, kv head, tile) that is one segment is finished by its block; the others' shares wait in scratch
// for a second kernel that joins them in their order.
//   warp 0       asks TMA for the pages of the run, keys and values, each into a ring of its own (128 KB on the way at most: 43 KB an SM hide a microsecond of latency, and it is more under load);
//   warp 1       S = Q K^T, 128 x 64, ahead of the softmax; two score buffers a group in tensor memory;
//   warp 2       O += P V as soon as P is written, P read from tensor memory where S was;
//   warp 3       walks the segments ahead of the others, leaves their descriptions and brings their queries, into the other of two buffers where they fit;
//   warps 4..19  the softmax: two groups of 256 threads, two threads a row (32 keys of a page each), that take the pages in turn where the tile has up to 128 rows (each with a maximum, a sum
//                and an accumulator of its own, joined at the segment's end), or every page for 128 rows each where it has more. The instruction takes no weights
//                wider than bfloat16 beside bfloat16 values, so P goes in two parts of 16 bits each, which are multiplied one after the other: a weight is off by 2^-14 at most. The sum is
//                of the whole weights, in 32 bits.
// What bounds it, measured on one B200 (calls back to back in a graph): 64 sequences of 150 to 4,096 rows, 8 nodes each, 32 / 8 heads of 128: 112 us, 4.7 TB/s,
// where a copy reads 6.57; four of 9,000 to 30,000 rows 94 us, 4.6 TB/s; eight trees of 40 to 64 nodes on 1,000 to 8,192 rows 70 us where the bytes take 22; one
// chat, 5 tokens in a row on 2,000 rows, 16 / 8 heads, in clusters, 11.2 us, a chain of latencies around four pages a block. Tensor pipe 46 to 48 % busy, issue 32
// to 50 %: neither, but a page's chain of scores, softmax and products, which the ring of pages covers while the pages come, and 4 to 5 us of a segment's last
// product, results and next queries, which nothing covers.
// The second part of the weights costs 8, 12 and 9 % in the first three (103, 83 and 64 us with one part, nothing in the chat) and takes the error against 64 bits
// from 2.3e-3 to 1.7e-3, that of the result's own rounding. With one part a block walked a page in 0.64 to 0.68 us (32 KB: 7 TB/s over all), one of 256 rows, 16,384
// powers of two or 1,024 cycles of their unit, in 0.93; the way in, 37 MB of shares and the joining were the rest of the trees' time.
// The layouts before this one, with one part (batch, trees): two blocks an SM 155 and 81 us, one with a thread a row 140 and 78, two threads a row 111 and 70,
// and with segments weighed (kTtEntry) and shares joined from a list 100 and 64. The next page's scores asked for before this one's weights leave spill registers
// (batch 112, trees 71); references before the scale throughout 106 and 67. With two parts: scores of two pages by one instruction of N = 128 gain nothing (batch 131
// cold, 131 otherwise; long texts 107, 109), for the pages then wait for one another.
// Where the sequences are few (tt_cluster) the blocks of a cluster share one (sequence, kv head, tile) instead: the shares meet in distributed shared memory, and
// there is neither a second kernel nor scratch.
// Rows are row r = node r / G, query head r % G of the group. Fewer than 128 rows leave the instruction's other rows to whatever lies behind the queries in shared
// memory: a row of A reaches that row of the result alone, and nobody reads it.
// Rows that a node does not see are masked by a bit each. Their values meet a zero weight in the product, which an infinity or a NaN among them would survive: so in
// pages that not all rows see alike (the step's own and those at a window's edge) values that are not finite are taken out in shared memory, and nodes that do see
// them get them back at the end, a bit pair for each (row, channel).
#include <math.h>

#include <algorithm>

#include "packed_f32.cuh"
#include "tcgen05.cuh"
#include "tree.cuh"

namespace slb {

constexpr int kTtRows = 128, kTtTile = 256, kTtThreads = 20 * 32, kTtSoftmax = 4 * 32;      // (the first thread of the softmax)
constexpr float kTtRescale = 8.0f;      // log2 units by which a maximum may be stale
// A row's maximum m serves its weights as 2^(score scale - m), one FMA each, and is off by up to half a step of 32 bits, a factor that all of them share; from 2^31 on
// that factor alone would be below the least number. So a maximum of 2^29 and more is kept as the score times the power of two at or above the scale, which is exact,
// and its weights are 2^((score - maximum) scale). Two such scores lie 32 units apart or are equal, so it does not matter that their distance looks up to twice as long.
constexpr float kTtFar = 536870912.0f;
__device__ __forceinline__ bool tt_far(float m) { return fabsf(m) >= kTtFar && fabsf(m) < INFINITY; }

__device__ __forceinline__ float tt_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float tt_max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ void tt_copy16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src)); }

struct TtLayout {
  int rows, queries, stages, q_bytes, k_off, v_off, poison_off, ml_off, xch_off, bar_off, total;      // queries: buffers for them
};
static TtLayout tt_layout(int HD, int rows) {
  TtLayout l;
  l.rows = std::min(kTtTile, (rows + 31) & ~31);
  l.queries = l.rows <= kTtRows ? 2 : 1;
  l.q_bytes = l.rows * HD * 2;
  const int page = 64 * HD * 2, rest = 2 * kTtRows * HD / 4 + 2 * 2 * kTtRows * 16 + 2 * 2 * 2 * kTtRows * 4 + 64 * 8;
  l.stages = std::min(8, (223 * 1024 - l.queries * l.q_bytes - rest) / (2 * page));      // (227 KB a block, up to 3 KB of it static)
  l.k_off = l.queries * l.q_bytes;
  l.v_off = l.k_off + l.stages * page;
  l.poison_off = l.v_off + l.stages * page;
  l.ml_off = l.poison_off + 2 * kTtRows * HD / 4;
  l.xch_off = l.ml_off + 2 * 2 * kTtRows * 16;
  l.bar_off = l.xch_off + 2 * 2 * 2 * kTtRows * 4;
  l.total = l.bar_off + 64 * 8;
  return l;
}

struct TtArgs {
  TreeArgs t;
  float scale_log2, far_scale, far_back;      // far_scale: the power of two at or above scale_log2, far_back: one over it
  float* part;          // [blocks][2][HD][rows] weighted values
  float2* part_ml;      // [blocks][2][rows] maximum (log2 units) and sum
  int2* info;           // [blocks] the (sequence, kv head, tile) whose first pages this block has and whose last ones it has not, and the blocks that share it (0: none)
  int* status;
  int cluster;          // blocks that share a (sequence, kv head, tile), or 0: runs of all units
  int tiles;            // most tiles of a sequence
  int q_by_tma;         // queries come by TMA: a group divides 32
  TtLayout lay;
};

// The pages of a sequence that some node may see: those from the window of a node at `past` on. A (sequence, kv head, tile) counts kTtEntry units more than it has
// pages: what a segment's beginning and end cost (runs of equal pages left blocks with many short segments behind: 64 sequences of 150 to 4,096 rows, of 148 blocks
// the median 99 us, the last 136; with it the call takes 104).
constexpr int kTtEntry = 5;
struct TtSeq {
  int past, count, tok0, page_lo, pages, tiles, units;
  __device__ __forceinline__ void read(const TreeArgs& a, int seq) {
    const TreeSeq s(a, seq);
    past = s.past; count = s.count; tok0 = s.tok0;
    const long long lo = a.window > 0 ? (long long)past - a.window + 1 : 0;
    page_lo = lo > 0 ? (int)(lo / 64) : 0;
    pages = count > 0 ? (past + count - 1) / 64 - page_lo + 1 : 0;
    tiles = (count * (a.heads / a.kv_heads) + kTtTile - 1) / kTtTile;
    units = (pages + kTtEntry) * tiles * a.kv_heads;      // (the launcher has seen that all units of a call stay below 2^31)
  }
};

// How units go to blocks: the first `more` blocks take each + 1 of them, the others each.
struct TtShare {
  int each, more;
  __device__ __forceinline__ TtShare(int total, int blocks) { each = total / blocks; more = total - each * blocks; }
  __device__ __forceinline__ int begin(int block) const { return block * each + min(block, more); }
  __device__ __forceinline__ int block_of(int unit) const {
    const int at = more * (each + 1);
    return unit < at ? unit / (each + 1) : more + (unit - at) / each;
  }
};

// A block's run of units, segment by segment.
struct TtWalk {
  int u, u_hi, seq, seq_first;      // the next unit, the run's end; the sequence and its first unit
  TtSeq s;
  int kh, tile, off, n, rows;       // the segment: its first page within the sequence, its pages, its rows
  int first;                        // the unit of its (sequence, kv head, tile)'s first page
  __device__ __forceinline__ bool next(const TreeArgs& a) {
    n = 0;
    while (u < u_hi) {
      const int rel = u - seq_first;
      if (rel >= s.units) {
        seq_first += s.units;
        s.read(a, ++seq);
        continue;
      }
      const int long_pages = s.pages + kTtEntry, at = rel / long_pages, place = rel - at * long_pages;
      kh = at / s.tiles;
      tile = at - kh * s.tiles;
      first = u - place + kTtEntry;
      const int end = min(first + s.pages, u_hi), begin = max(u, first);
      u = end;
      if (end <= begin) continue;      // the run ends before the first page
      off = begin - first;
      n = end - begin;
      rows = min(kTtTile, s.count * (a.heads / a.kv_heads) - tile * kTtTile);
      return true;
    }
    return false;
  }
};

__device__ __forceinline__ float2 tt_peer2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float tt_peer(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

template <int HD, bool CLUSTER>
__global__ void __launch_bounds__(kTtThreads, 1)
tree_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ TtArgs ta) {
  constexpr int PAGE = 64 * HD * 2, WORDS = HD / 16;      // words of a row's poison
  const TreeArgs& a = ta.t;
  const TtLayout& L = ta.lay;
  extern __shared__ __align__(1024) unsigned char smem[];
  __shared__ int warp_units[kTtThreads / 32];
  __shared__ int s_lo[2];
  __shared__ uint32_t s_odd[3][2][2], tmem_slot;      // rows of a page with values that are not finite: of either group's page, of a page of both; two places used in turn
  __shared__ TtWalk desc[2], s_run;
  __shared__ float2 s_ml[CLUSTER ? kTtTile : 1];      // a cluster's blocks: maximum and sum of each row
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = smem_addr(smem);
  if ((base & 1023u) != 0) {
    if (tid == 0) atomicExch(ta.status, 111);
    return;
  }
  const uint32_t sK = base + L.k_off, sV = base + L.v_off, bars = base + L.bar_off;
  const uint32_t k_full = bars, k_free = bars + 64, v_full = bars + 128, v_free = bars + 192, s_full = bars + 256, p_full = bars + 288, pv_done = bars + 320,
                 q_full = bars + 352, q_free = bars + 368, o_free = bars + 384;      // (s_full, p_full, pv_done: [group][buffer])
  if (warp == 0) {
    // one arrival each, but for p_full (eight softmax warps), q_free (all sixteen, the scores' and the values' thread) and o_free (sixteen)
    for (int i = lane; i < 49; i += 32) mbar_init(bars + 8 * i, i >= 36 && i < 40 ? 8 : i == 46 || i == 47 ? 18 : i == 48 ? 16 : 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (lane < 12) (&s_odd[0][0][0])[lane] = 0u;
    if (lane < 2) s_lo[lane] = 0;
    if (CLUSTER)      // (of a block without pages nothing else becomes)
      for (int r = lane; r < kTtTile; r += 32) s_ml[r] = make_float2(-INFINITY, 0.0f);
  }
  if (warp == 2) {
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_slot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_wait();
  if (!CLUSTER && tid == kTtSoftmax) ta.info[blockIdx.x] = make_int2(0, 0);      // (by the thread that may write it again; the scratch may have been another kernel's until now)

  // where this block's run of units begins
  const int G = a.heads / a.kv_heads;
  int total = 0;
  if constexpr (CLUSTER) {
    if (tid == 0) {      // the block's share of its cluster's pages, as units that begin with this (sequence, kv head, tile)
      const int pair = (int)blockIdx.x / ta.cluster, rank = (int)blockIdx.x % ta.cluster, at = pair % (a.kv_heads * ta.tiles);
      s_run.seq = pair / (a.kv_heads * ta.tiles);
      s_run.s.read(a, s_run.seq);
      const int kh = at / ta.tiles, tile = at % ta.tiles, share = (s_run.s.pages + ta.cluster - 1) / ta.cluster;
      s_run.kh = kh;
      s_run.tile = tile;
      s_run.seq_first = -(kh * s_run.s.tiles + tile) * (s_run.s.pages + kTtEntry);
      s_run.u = kTtEntry + min(s_run.s.pages, rank * share);
      s_run.u_hi = tile < s_run.s.tiles ? kTtEntry + min(s_run.s.pages, (rank + 1) * share) : 0;
    }
  } else {
    const int per = (a.n_seqs + kTtThreads - 1) / kTtThreads, q0 = min(a.n_seqs, tid * per), q1 = min(a.n_seqs, q0 + per);
    TtSeq one;
    int own = 0;
    for (int s = q0; s < q1; ++s) {
      one.read(a, s);
      own += one.units;
    }
    int incl = own;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += y;
    }
    if (lane == 31) warp_units[warp] = incl;
    __syncthreads();
    int before = 0;
#pragma unroll
    for (int w = 0; w < kTtThreads / 32; ++w) {
      if (w < warp) before += warp_units[w];
      total += warp_units[w];
    }
    const int blocks = min((int)gridDim.x, total);
    if ((int)blockIdx.x < blocks) {
      const TtShare share(total, blocks);
      const int u = share.begin(blockIdx.x);
      before += incl - own;
      if (own > 0 && u >= before && u < before + own) {
        int s = q0;
        if (per > 1) one.read(a, s);
        while (u >= before + one.units) {
          before += one.units;
          one.read(a, ++s);
        }
        s_run.u = u;
        s_run.u_hi = share.begin(blockIdx.x + 1);
        s_run.seq = s;
        s_run.seq_first = before;
        s_run.s = one;
      }
    } else if (tid == 0) {
      s_run.u = s_run.u_hi = 0;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch_dependents();      // (only now: a successor that also wants tensor memory must not take it before this block has its own)
  const uint32_t tmem = tmem_slot;

  if (warp == 0) {
    // ---- pages ----
    TtWalk run = s_run;
    int st = 0, lap = 0;
    bool ok = true;
    while (ok && run.next(a)) {
      const int* table = a.block_table + (size_t)run.seq * a.table_stride + run.s.page_lo + run.off;
      for (int i0 = 0; i0 < run.n && ok; i0 += 32) {
        int mine = i0 + lane < run.n ? table[i0 + lane] : 0;
        if (mine < 0 || mine >= a.pool_pages) mine = -1;      // (rows in front of the pool: zeros; another page's number times its rows might come back into it)
        for (int i = 0; i < min(32, run.n - i0) && ok; ++i) {
          const int row = (__shfl_sync(0xffffffffu, mine, i) * a.kv_heads + run.kh) * 64;
          if (lap > 0 && !mbar_wait(k_free + 8 * st, (lap - 1) & 1)) { ok = false; break; }
          if (elect_one()) {
            mbar_expect_tx(k_full + 8 * st, PAGE);
#pragma unroll
            for (int h = 0; h < HD / 64; ++h) tma_load_2d(sK + st * PAGE + h * 8192, &map_k, h * 64, row, k_full + 8 * st);
          }
          __syncwarp();
          if (lap > 0 && !mbar_wait(v_free + 8 * st, (lap - 1) & 1)) {
            mbar_wait(k_full + 8 * st, lap & 1);      // (the copy under way lands before the block goes)
            ok = false;
            break;
          }
          if (elect_one()) {
            mbar_expect_tx(v_full + 8 * st, PAGE);
#pragma unroll
            for (int h = 0; h < HD / 64; ++h) tma_load_2d(sV + st * PAGE + h * 8192, &map_v, h * 64, row, v_full + 8 * st);
          }
          __syncwarp();
          if (++st == L.stages) { st = 0; ++lap; }
        }
      }
    }
    if (!ok && lane == 0) atomicExch(ta.status, 112);
    // copies under way land before the block goes
    for (int i = 0; i < L.stages; ++i) {
      if (st == 0) { st = L.stages; --lap; }
      if (lap < 0) break;
      --st;
      mbar_wait(k_full + 8 * st, lap & 1);
      mbar_wait(v_full + 8 * st, lap & 1);
    }
  } else if (warp == 1) {
    if (elect_one()) {
      // ---- scores: item x is a page of one group, x & 1, whose item x >> 1 it is ----
      constexpr uint32_t idesc = instr_desc(kTtRows, 64);
      int st = 0, lap = 0, x = 0;
      for (int seg = 0;; ++seg) {
        const int qb = L.queries == 2 ? seg & 1 : 0, q_lap = L.queries == 2 ? seg >> 1 : seg;
        if (!mbar_wait(q_full + 8 * qb, q_lap & 1)) { atomicExch(ta.status, 113); break; }
        const int n = desc[qb].n;
        const bool dual = desc[qb].rows > kTtRows;
        if (n == 0) break;
        bool ok = true;
        for (int i = 0; i < n && ok; ++i) {
          if (!mbar_wait(k_full + 8 * st, lap & 1)) { atomicExch(ta.status, 114); ok = false; break; }
          for (int d = 0; d < (dual ? 2 : 1); ++d, ++x) {
            const int g = x & 1, c = x >> 1, b = c & 1;
            // S lands where S and then P of two items ago lay: the product that read that P must be through
            if (c >= 2 && !mbar_wait(pv_done + 8 * (2 * g + b), ((c >> 1) - 1) & 1)) { atomicExch(ta.status, 115); ok = false; break; }
            tc_fence_after();
            const uint32_t q = base + qb * L.q_bytes + (dual ? g * (kTtRows * 128) : 0);
#pragma unroll
            for (int h = 0; h < HD / 64; ++h) {
              const uint64_t dq = smem_desc(q + h * L.rows * 128), dk = smem_desc(sK + st * PAGE + h * 8192);
#pragma unroll
              for (int k4 = 0; k4 < 4; ++k4)
                mma_bf16_ss(tmem + (uint32_t)(g * 256 + b * 64), dq + (uint64_t)(k4 * 2), dk + (uint64_t)(k4 * 2), idesc, (h > 0 || k4 > 0) ? 1u : 0u);
            }
            mma_commit(s_full + 8 * (2 * g + b));
          }
          if (!ok) break;
          mma_commit(k_free + 8 * st);
          if (++st == L.stages) { st = 0; ++lap; }
        }
        if (!ok) break;
        mma_commit(q_free + 8 * qb);
      }
    }
  } else if (warp == 2) {
    if (elect_one()) {
      // ---- values ----
      constexpr uint32_t idesc = instr_desc(kTtRows, HD, true);
      int st = 0, lap = 0, x = 0;
      for (int seg = 0;; ++seg) {
        const int qb = L.queries == 2 ? seg & 1 : 0, q_lap = L.queries == 2 ? seg >> 1 : seg;
        if (!mbar_wait(q_full + 8 * qb, q_lap & 1)) { atomicExch(ta.status, 116); break; }
        const int n = desc[qb].n;
        const bool dual = desc[qb].rows > kTtRows;
        if (n == 0) break;
        mbar_arrive(q_free + 8 * qb);
        if (seg > 0 && !mbar_wait(o_free, (seg - 1) & 1)) { atomicExch(ta.status, 116); break; }
        uint32_t fresh = 3u;      // groups without a product in this segment
        bool ok = true;
        for (int i = 0; i < n && ok; ++i) {
          if (!mbar_wait(v_full + 8 * st, lap & 1)) { atomicExch(ta.status, 117); ok = false; break; }
          for (int d = 0; d < (dual ? 2 : 1); ++d, ++x) {
            const int g = x & 1, c = x >> 1, b = c & 1;
            if (!mbar_wait(p_full + 8 * (2 * g + b), (c >> 1) & 1)) { atomicExch(ta.status, 118); ok = false; break; }
            tc_fence_after();
#pragma unroll
            for (int k4 = 0; k4 < 4; ++k4) {
              const uint64_t dv = smem_desc_mn(sV + st * PAGE + k4 * 2048, 8192, 1024);
              mma_bf16_ts(tmem + (uint32_t)(g * 256 + 128), tmem + (uint32_t)(g * 256 + b * 64 + k4 * 8), dv, idesc, k4 > 0 || !(fresh >> g & 1u) ? 1u : 0u);
              mma_bf16_ts(tmem + (uint32_t)(g * 256 + 128), tmem + (uint32_t)(g * 256 + b * 64 + 32 + k4 * 8), dv, idesc, 1u);
            }
            fresh &= ~(1u << g);
            mma_commit(pv_done + 8 * (2 * g + b));
          }
          if (!ok) break;
          mma_commit(v_free + 8 * st);
          if (++st == L.stages) { st = 0; ++lap; }
        }
        if (!ok) break;
      }
    }
  } else if (warp == 3) {
    // ---- segments and their queries, as a tile that TMA would have left: 64 channels a half, 16-byte pieces exchanged by the row ----
    TtWalk run = s_run;
    for (int seg = 0;; ++seg) {
      const int qb = L.queries == 2 ? seg & 1 : 0, q_lap = L.queries == 2 ? seg >> 1 : seg;
      const bool more = run.next(a);
      if (q_lap > 0 && !mbar_wait(q_free + 8 * qb, (q_lap - 1) & 1)) {
        if (lane == 0) atomicExch(ta.status, 123);
        break;
      }
      const uint32_t q = base + qb * L.q_bytes;
      if (more && !ta.q_by_tma) {
        constexpr int PIECES = HD / 8, AT_ONCE = 32 / PIECES;
        const int piece = lane % PIECES;
        int r = lane / PIECES, node = (run.tile * kTtTile + r) / G, head = run.tile * kTtTile + r - node * G;
        for (; r < run.rows; r += AT_ONCE) {
          tt_copy16(q + (piece >> 3) * (L.rows * 128) + r * 128 + (((piece & 7) ^ (r & 7)) << 4),
                    (const __nv_bfloat16*)a.q + ((size_t)(run.s.tok0 + node) * a.heads + run.kh * G + head) * HD + piece * 8);
          for (head += AT_ONCE; head >= G; head -= G) ++node;
        }
      }
      if (lane == 0) desc[qb] = run;
      asm volatile("cp.async.wait_all;" ::: "memory");
      fence_smem_to_async();
      __syncwarp();
      if (elect_one()) {
        if (more && ta.q_by_tma) {      // a tile that begins with a whole group, zeros or another sequence's queries behind its rows
          mbar_expect_tx(q_full + 8 * qb, L.q_bytes);
#pragma unroll
          for (int h = 0; h < HD / 64; ++h) tma_load_3d(q + h * (L.rows * 128), &map_q, h * 64, run.kh * G, run.s.tok0 + run.tile * kTtTile / G, q_full + 8 * qb);
        } else {
          mbar_arrive(q_full + 8 * qb);
        }
      }
      if (!more) break;
    }
  } else {
    // ---- softmax: tensor-memory lanes 32 (warp % 4) .. + 31 hold the rows; two warps share them, keys 0..31 and 32..63 of a page ----
    const int quad = warp & 3, g = (warp - 4) >> 3, half = (warp - 4) >> 2 & 1, r = quad * 32 + lane, stid = tid - kTtSoftmax, gtid = stid & 255;
    const uint32_t lane_addr = tmem + ((uint32_t)(quad * 32) << 16), own = lane_addr + g * 256;
    uint32_t* poison = reinterpret_cast<uint32_t*>(smem + L.poison_off) + (g * kTtRows + r) * WORDS;      // [2 groups][128 rows][WORDS]; of the other group: other_poison words on
    const int other_poison = g ? -kTtRows * WORDS : kTtRows * WORDS;
    float4* ml = reinterpret_cast<float4*>(smem + L.ml_off);                  // [2 groups][2 halves][128 rows] maximum, sum, whether there is poison
    float* xch = reinterpret_cast<float*>(smem + L.xch_off) + g * 512 + r;      // [2 groups][2 buffers][2 halves][128 rows]
    // A wait that gives up ends nothing here: the warp notes it and walks on to the segment's end, because others meet it at barriers; the status word says so.
    bool ok = true;
    auto wait_warp = [&](uint32_t bar, uint32_t parity, int code) {
      if (ok && !mbar_wait(bar, parity)) {
        ok = false;
        if (lane == 0) atomicExch(ta.status, code);
      }
    };
    auto arrive_warp = [&](uint32_t bar) {
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    auto pair_sync = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(1 + 4 * g + quad) : "memory"); };
    auto look_sync = [&](bool both) {      // of a group, or of both
      asm volatile("bar.sync %0, %1;" ::"r"(both ? 11 : 9 + g), "r"(both ? 512 : 256) : "memory");
    };
    int page_no = 0, x = 0;      // pages and items so far, over all segments
    int looked[2] = {0, 0};      // pages whose values were looked through: of this group's, of both groups'
    for (int seg = 0;; ++seg) {
      const int qb = L.queries == 2 ? seg & 1 : 0, q_lap = L.queries == 2 ? seg >> 1 : seg;
      {
        const uint32_t lost = mbar_wait(q_full + 8 * qb, q_lap & 1) ? 0u : 1u;      // all or none go on
        uint32_t any;
        __syncwarp();
        asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, 11, 512, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(any) : "r"(lost) : "memory");
        if (any) {
          if (stid == 0) atomicExch(ta.status, 124);
          break;
        }
      }
      const TtWalk& w = desc[qb];
      const int n = w.n;
      if (n == 0) break;
      const int past = w.s.past, key_first = (w.s.page_lo + w.off) * 64;
      const bool dual = w.rows > kTtRows;
      const int in_tile = dual ? g * kTtRows + r : r;
      const bool live = in_tile < w.rows, warp_live = in_tile - lane < w.rows;
      const int node = w.s.tok0 + (live ? (w.tile * kTtTile + in_tile) / G : 0);
      const uint32_t* words = a.seen + (size_t)node * a.words;
      int lo = 0, lo_most = 0;
      if (a.window > 0) {      // the latest beginning of a window in the tile
        lo = live ? tree_lo(a, node, past) : 0;
        if (live && half == 0) atomicMax(&s_lo[seg & 1], lo);
        look_sync(true);
        lo_most = s_lo[seg & 1];
        if (stid == 0) s_lo[(seg + 1) & 1] = 0;      // (read for the last time before the barrier above)
      }
      float m_used = -INFINITY, l = 0.0f;
      bool poisoned = false;
      int done = 0;      // this group's items in the segment
      for (int i = 0; i < n; ++i, ++page_no) {
        if (dual) {
          x += 2;
        } else if ((x++ & 1) != g) {
          continue;
        }
        const int c = (dual ? x - 2 + ((x & 1) != g) : x - 1) >> 1, b = c & 1;      // the item's number among the group's
        const int key_page = key_first + i * 64, key0 = key_page + half * 32;
        wait_warp(s_full + 8 * (2 * g + b), (c >> 1) & 1, 119);
        const bool mixed = key_page + 63 >= past || key_page < lo_most;      // not all rows see all of the page
        uint32_t seen = 0xffffffffu;
        if (warp_live) {
          tc_fence_after();
          uint32_t sr[32];
          tmem_ld32(own + (uint32_t)(b * 64 + half * 32), sr);
          if (mixed) {
            const int to = past - key0, from = lo - key0;
            seen = (to >= 32 ? 0xffffffffu : to <= 0 ? 0u : (1u << to) - 1u) & (from <= 0 ? 0xffffffffu : from >= 32 ? 0u : 0xffffffffu << from);
            if (key0 + 31 >= past) seen |= (uint32_t)tree_bits(words, a.words, key0 - past, w.s.count);
            if (!live) seen = 0u;
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (!(seen >> k & 1u)) sr[k] = 0xff800000u;     // -inf
          }
          float mx = -INFINITY, mx1 = -INFINITY;
#pragma unroll
          for (int k = 0; k < 32; k += 4) {
            mx = tt_max3(mx, __uint_as_float(sr[k]), __uint_as_float(sr[k + 1]));
            mx1 = tt_max3(mx1, __uint_as_float(sr[k + 2]), __uint_as_float(sr[k + 3]));
          }
          // The row's maximum is the larger of the two halves', so that both threads of a row take the same decisions, and it is exchanged as it is: rounded up to 16
          // bits it lies up to 2^-7 of itself too high, 126 units of log2 where scores pass 10^4, and no weight is left beside it.
          {
            const float own_max = fmaxf(mx, mx1);
            xch[b * 256 + half * 128] = own_max;      // (a place per buffer: the partner passes the barrier of the next item only after reading this one)
            pair_sync();
            mx = fmaxf(own_max, xch[b * 256 + (half ^ 1) * 128]);
          }
          mx = fabsf(mx * ta.scale_log2) >= kTtFar ? mx * ta.far_scale : mx * ta.scale_log2;      // the scale is positive
          const float m_new = fmaxf(m_used, mx);
          const bool grow = m_new > m_used + kTtRescale;      // also true for the first finite maximum
          if (done > 0 && __any_sync(0xffffffffu, grow)) {
            wait_warp(pv_done + 8 * (2 * g + (b ^ 1)), ((c - 1) >> 1) & 1, 120);      // O must hold all of the last product
            tc_fence_after();
            const float alpha = grow ? tt_ex2(m_used - m_new) : 1.0f;
#pragma unroll 1
            for (int c0 = 0; c0 < HD / 2; c0 += 16) {      // this thread's half of the accumulator row
              uint32_t o[16];
              tmem_ld16(own + 128 + half * (HD / 2) + c0, o);
#pragma unroll
              for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
              tmem_st16(own + 128 + half * (HD / 2) + c0, o);
            }
            l *= alpha;
          }
          if (grow) m_used = m_new;
          const bool far = tt_far(m_used);
          if (__any_sync(0xffffffffu, far)) {
            const float ref = far ? m_used * ta.far_back : 0.0f;
#pragma unroll
            for (int k = 0; k < 32; ++k) sr[k] = __float_as_uint(__uint_as_float(sr[k]) - ref);
          }
          const f32x2 refs = both(m_used == -INFINITY || far ? 0.0f : -m_used), scales = both(ta.scale_log2);
          f32x2 sums = 0ull;
          // The weights' upper 16 bits, less one in the last place, and the upper 16 bits of what is left: only a weight of nothing has a part that is nothing, so an
          // infinity that all rows see is not multiplied by zero. What is lost is below 2^-14 of a weight.
          uint32_t pk[16], rest[16];
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            const f32x2 e = fma2(pair_of(__uint_as_float(sr[k]), __uint_as_float(sr[k + 1])), scales, refs);
            const float p0 = tt_ex2(__uint_as_float((uint32_t)e)), p1 = tt_ex2(__uint_as_float((uint32_t)(e >> 32)));
            const f32x2 p = pair_of(p0, p1);
            pk[k >> 1] = __viaddmax_s16x2(__byte_perm(__float_as_uint(p0), __float_as_uint(p1), 0x7632), 0xffffffffu, 0u);
            const f32x2 low = fma2(pair_of(__uint_as_float(pk[k >> 1] << 16), __uint_as_float(pk[k >> 1] & 0xffff0000u)), both(-1.0f), p);
            rest[k >> 1] = __byte_perm((uint32_t)low, (uint32_t)(low >> 32), 0x7632);
            sums = add2(sums, p);
          }
          tmem_st16(own + (uint32_t)(b * 64 + half * 16), pk);
          tmem_st16(own + (uint32_t)(b * 64 + 32 + half * 16), rest);      // (the partner has its scores from here: both met at the barrier above)
          l += __uint_as_float((uint32_t)sums) + __uint_as_float((uint32_t)(sums >> 32));
        }
        ++done;
        if (mixed) {
          // values that are not finite go; rows that see one remember it. Two groups on one page look together, since what one has taken out the other would miss
          const int st = page_no % L.stages, lap = page_no / L.stages;
          wait_warp(v_full + 8 * st, lap & 1, 121);
          const int held = past + w.s.count - key_page;      // rows of the page that belong to the sequence
          uint32_t* odd = dual ? s_odd[2][looked[1]++ & 1] : s_odd[g][looked[0]++ & 1];
          bool wrote = false;
#pragma unroll 1
          for (int e = dual ? stid : gtid; e < 64 * HD / 8; e += dual ? 512 : 256) {
            const int row = e >> 3 & 63;                 // a 16-byte piece of a row, as the pieces lie
            const uint32_t at = sV + st * PAGE + e * 16;
            uint4 v;
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
            auto carry = [](uint32_t y) { return (y & 0x7fff7fffu) + 0x00800080u; };      // bit 15 and 31: an exponent of all ones
            if ((carry(v.x) | carry(v.y) | carry(v.z) | carry(v.w)) & 0x80008000u) {
              auto bad = [](uint32_t y) { return ((y & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((y & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u); };
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x & ~bad(v.x)), "r"(v.y & ~bad(v.y)), "r"(v.z & ~bad(v.z)), "r"(v.w & ~bad(v.w)) : "memory");
              if (row < held) atomicOr(&odd[row >> 5], 1u << (row & 31));
              wrote = true;
            }
          }
          if (wrote) fence_smem_to_async();
          look_sync(dual);
          if (odd[0] | odd[1]) {
            uint32_t left = live ? odd[half] & seen : 0u;
            look_sync(dual);
            if (gtid < 2 && (g == 0 || !dual)) odd[gtid] = 0u;
            // the row's two threads one after the other: they share its words
            if (half == 0 && live && !poisoned)
              for (int k = 0; k < WORDS; ++k) poison[k] = 0u;
            poisoned = true;
            look_sync(dual);
            const int page = a.block_table[(size_t)w.seq * a.table_stride + key_page / 64];
            for (; left; left &= left - 1) {
              const uint32_t* v = reinterpret_cast<const uint32_t*>((const __nv_bfloat16*)a.v_pool + (((size_t)page * a.kv_heads + w.kh) * 64 + half * 32 + __ffs(left) - 1) * HD);
#pragma unroll 1
              for (int k = 0; k < HD; ++k) {
                const uint32_t y = v[k >> 1] >> (k & 1) * 16 & 0xffffu;
                if ((y & 0x7f80u) == 0x7f80u) atomicOr(&poison[k / 16], ((y & 0x7fu) ? 3u : y >> 15 ? 2u : 1u) << (k % 16 * 2));
              }
            }
          }
        }
        tc_fence_before();
        arrive_warp(p_full + 8 * (2 * g + b));
      }
      // ---- the segment's results: of a tile of up to 128 rows the groups join theirs, a quarter of the channels a thread; else half ----
      const int first_item = x - (dual ? 2 * n : n);
      auto items = [&](int group) { return dual ? n : (n + (((first_item & 1) == group) ? 1 : 0)) / 2; };      // of a group in the segment
      auto wait_done = [&](int group) {      // its last one
        const int last = (x - 1 - (((x - 1) & 1) != group)) >> 1;
        wait_warp(pv_done + 8 * (2 * group + (last & 1)), (last >> 1) & 1, 122);
      };
      if (live) ml[(g * 2 + half) * kTtRows + r] = make_float4(m_used, l, poisoned ? 1.0f : 0.0f, 0.0f);
      look_sync(true);
      const bool begins = w.off == 0, complete = begins && n == w.s.pages;
      if (!CLUSTER && begins && !complete && stid == 0)
        ta.info[blockIdx.x] = make_int2((w.seq * a.kv_heads + w.kh) * ta.tiles + w.tile,
                                        TtShare(total, min((int)gridDim.x, total)).block_of(w.first + w.s.pages - 1) - (int)blockIdx.x + 1);
      const bool mine_here = items(g) > 0, other_here = !dual && items(g ^ 1) > 0;
      if (warp_live) {
        if (mine_here) wait_done(g);
        if (other_here || (CLUSTER && dual)) wait_done(g ^ 1);      // (a cluster's share goes where the other group's values lay)
        tc_fence_after();
        float4 me = ml[(g * 2 + half) * kTtRows + r], them = make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
        me.y += ml[(g * 2 + (half ^ 1)) * kTtRows + r].y;
        if (other_here) {
          them = ml[((g ^ 1) * 2 + half) * kTtRows + r];
          them.y += ml[((g ^ 1) * 2 + (half ^ 1)) * kTtRows + r].y;
        }
        const float M = fmaxf(me.x, them.x), use = M == -INFINITY ? 0.0f : M;
        float f = mine_here ? tt_ex2(me.x - use) : 0.0f, fo = other_here ? tt_ex2(them.x - use) : 0.0f;
        const float sum = me.y * f + them.y * fo;
        if (!CLUSTER && complete) {
          const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
          f *= inv;
          fo *= inv;
        }
        // (a share that saw nothing, whose products are of nothing but zeros, stays out; one whose scores were all NaN has a sum of NaN)
        const bool take = mine_here && me.y != 0.0f, take_other = other_here && them.y != 0.0f;
        const size_t slot = (size_t)blockIdx.x * 2 + (begins ? 1 : 0);
        const int width = dual ? HD / 2 : HD / 4, ch0 = dual ? half * width : (2 * g + half) * width;
#pragma unroll 1
        for (int ch = ch0; ch < ch0 + width; ch += 16) {
          float v[16];
          uint32_t o[16];
          __syncwarp();
          if (mine_here) tmem_ld16(own + 128 + ch, o);
#pragma unroll
          for (int k = 0; k < 16; ++k) v[k] = take ? __uint_as_float(o[k]) * f : 0.0f;
          if (other_here) {
            __syncwarp();
            tmem_ld16(lane_addr + (g ^ 1) * 256 + 128 + ch, o);
#pragma unroll
            for (int k = 0; k < 16; ++k) v[k] = take_other ? fmaf(__uint_as_float(o[k]), fo, v[k]) : v[k];
          }
          if (live) {
            if (me.z != 0.0f || them.z != 0.0f) {
              const uint32_t bad = (me.z != 0.0f ? poison[ch / 16] : 0u) | (them.z != 0.0f ? poison[other_poison + ch / 16] : 0u);
#pragma unroll
              for (int k = 0; k < 16; ++k) {
                const uint32_t y = bad >> (2 * k) & 3u;
                if (y) v[k] += y == 1u ? INFINITY : y == 2u ? -INFINITY : NAN;
              }
            }
            if (!CLUSTER && complete) {
              uint32_t y[8];
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                __nv_bfloat162 h2 = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]);
                y[k] = *reinterpret_cast<uint32_t*>(&h2);
              }
              uint4* out = reinterpret_cast<uint4*>((__nv_bfloat16*)a.out + ((size_t)node * a.heads + w.kh * G + (w.tile * kTtTile + in_tile) % G) * HD + ch);
              if (ok) {
                out[0] = make_uint4(y[0], y[1], y[2], y[3]);
                out[1] = make_uint4(y[4], y[5], y[6], y[7]);
              }
            } else {      // (in a cluster where the ring was: its pages have been multiplied)
              float* part = (CLUSTER ? reinterpret_cast<float*>(smem + L.k_off) + (size_t)ch * L.rows : ta.part + (slot * HD + ch) * L.rows) + in_tile;
#pragma unroll
              for (int k = 0; k < 16; ++k) part[(size_t)k * L.rows] = v[k];
            }
          }
        }
        if (live && half == 0 && (dual || g == 0)) {
          if (CLUSTER) s_ml[in_tile] = make_float2(M, sum);
          else if (!complete) ta.part_ml[slot * L.rows + in_tile] = make_float2(M, sum);
        }
      }
      tc_fence_before();
      arrive_warp(o_free);
      arrive_warp(q_free + 8 * qb);
    }
  }
  tc_fence_before();
  if constexpr (!CLUSTER) __syncthreads();
  if constexpr (CLUSTER) {
    // the shares meet: every block adds up its part of the (row, four channels)
    const int kh = s_run.kh, tile = s_run.tile, rank = (int)cluster_ctarank();
    const TtSeq& s = s_run.s;
    const int rows = min(kTtTile, s.count * G - tile * kTtTile);
    __syncwarp();
    cluster_sync_all();
    const uint32_t ml_at = smem_addr(s_ml), part_at = base + L.k_off;
    // (dealt to the blocks by the warp: what a block's reads of the others can bring is what this waits for)
    for (int e = (warp * ta.cluster + rank) * 32 + lane; e < L.rows * (HD / 4); e += ta.cluster * kTtThreads) {
      const int r = e % L.rows, c0 = e / L.rows * 4;
      if (r >= rows) continue;
      float2 p[8];
      float v[8][4], M = -INFINITY;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[i] = make_float2(-INFINITY, 0.0f);
        if (i >= ta.cluster) continue;
        p[i] = tt_peer2(cluster_map(ml_at + r * 8, i));
        const uint32_t at = cluster_map(part_at + (c0 * L.rows + r) * 4, i);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[i][k] = tt_peer(at + k * L.rows * 4);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) M = fmaxf(M, p[i].x);
      const float use = M == -INFINITY ? 0.0f : M;
      float l = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i >= ta.cluster || p[i].y == 0.0f) continue;      // (a share that saw nothing, or has no pages)
        const float f = tt_ex2(p[i].x - use);
        l += p[i].y * f;
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[k] += v[i][k] * f;
      }
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      uint32_t w[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        __nv_bfloat162 h2 = __floats2bfloat162_rn(acc[2 * k] * inv, acc[2 * k + 1] * inv);
        w[k] = *reinterpret_cast<uint32_t*>(&h2);
      }
      const int R = tile * kTtTile + r;
      *reinterpret_cast<uint2*>((__nv_bfloat16*)a.out + ((size_t)(s.tok0 + R / G) * a.heads + kh * G + R % G) * HD + c0) = make_uint2(w[0], w[1]);
    }
    __syncwarp();
    cluster_sync_all();      // the others may still be reading this block's share
  }
  if (warp == 2) {
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// Joins the shares of what no block finished alone, of each block of the kernel before at most one (sequence, kv head, tile): the blocks make a list of them and go
// over its pieces of 256 (row, four channels), a thread each, eight shares on the way at once.
constexpr int kTtMostBlocks = 256;
template <int HD>
__global__ void __launch_bounds__(256) tree_tc_join_kernel(TtArgs ta, int blocks) {
  const TreeArgs& a = ta.t;
  __shared__ int2 info_s[kTtMostBlocks];
  __shared__ int block_s[kTtMostBlocks], warp_s[8];
  const int rows_pad = ta.lay.rows, G = a.heads / a.kv_heads, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, chunks = rows_pad * (HD / 4) / 256;
  pdl_wait();
  const int2 mine = tid < blocks ? ta.info[tid] : make_int2(0, 0);
  const uint32_t has = __ballot_sync(0xffffffffu, mine.y > 1);
  if (lane == 0) warp_s[warp] = __popc(has);
  __syncthreads();
  int before = 0, found = 0;
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    before += w < warp ? warp_s[w] : 0;
    found += warp_s[w];
  }
  if (mine.y > 1) {
    const int at = before + __popc(has & ((1u << lane) - 1u));
    info_s[at] = mine;
    block_s[at] = tid;
  }
  __syncthreads();
  for (int task = blockIdx.x; task < found * chunks; task += gridDim.x) {
    const int2 in = info_s[task / chunks];
    const int first = block_s[task / chunks], tile = in.x % ta.tiles, kh = in.x / ta.tiles % a.kv_heads, seq = in.x / ta.tiles / a.kv_heads;
    const TreeSeq s(a, seq);
    const int rows = min(kTtTile, s.count * G - tile * kTtTile), e = task % chunks * 256 + tid, r = e % rows_pad, c0 = e / rows_pad * 4;
    if (r >= rows) continue;
    auto slot_of = [&](int i) { return (size_t)(first + i) * 2 + (i == 0 ? 1 : 0); };
    float M = -INFINITY, l = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int i0 = 0; i0 < in.y; i0 += 8) {
      float2 ml[8];
      float v[8][4];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        ml[i] = make_float2(-INFINITY, 0.0f);
        if (i0 + i >= in.y) continue;
        const size_t slot = slot_of(i0 + i);
        ml[i] = ta.part_ml[slot * rows_pad + r];
#pragma unroll
        for (int c = 0; c < 4; ++c) v[i][c] = ta.part[(slot * HD + c0 + c) * rows_pad + r];
      }
      float top = M;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, ml[i].x);
      const float use = top == -INFINITY ? 0.0f : top, keep = tt_ex2(M - use);
      l *= keep;
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[c] *= keep;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i0 + i >= in.y || ml[i].y == 0.0f) continue;      // (a share that saw nothing; one whose scores were all NaN has a sum of NaN)
        const float f = tt_ex2(ml[i].x - use);
        l += ml[i].y * f;
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[c] += v[i][c] * f;
      }
      M = top;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    __nv_bfloat162 lo = __floats2bfloat162_rn(acc[0] * inv, acc[1] * inv), hi = __floats2bfloat162_rn(acc[2] * inv, acc[3] * inv);
    const int R = tile * kTtTile + r;
    *reinterpret_cast<uint2*>((__nv_bfloat16*)a.out + ((size_t)(s.tok0 + R / G) * a.heads + kh * G + R % G) * HD + c0) =
        make_uint2(*reinterpret_cast<uint32_t*>(&lo), *reinterpret_cast<uint32_t*>(&hi));
  }
}

bool tree_tc_takes(int n_seqs, int max_count, int heads, int kv_heads, int head_dim, int max_keys, int dtype) {
  const long long tiles = ((long long)max_count * (heads / kv_heads) + kTtTile - 1) / kTtTile;
  return dtype == kBF16 && (head_dim == 64 || head_dim == 128) && n_seqs * tiles * kv_heads * (max_keys / 64 + 2ll + kTtEntry) < (1ll << 31);
}

// Whether blocks of a cluster share each (sequence, kv head, tile), and how many: one chat (5 tokens on 2,000 rows, 16 / 8 heads) takes 11.2 us so and 20.6 by runs
// of units and a second kernel. A cluster waits for its longest sequence alone, so only where all clusters run at once (128 of the 148 blocks:
// clusters of eight lie within one of the GPU's partitions each) and no block takes more than ten pages.
static int tt_cluster(int n_seqs, int kv_heads, int tiles, int max_count, int max_keys, int window) {
  long long pages = ((long long)max_keys + 63) / 64;
  if (window > 0) pages = std::min(pages, ((long long)window + max_count + 62) / 64 + 1);
  const long long pairs = (long long)n_seqs * kv_heads * tiles;
  int c = 8;
  while (c > 1 && (pairs * c > 128 || c > pages)) c /= 2;
  return pairs * c <= 128 && pages <= 10ll * c ? c : 0;
}

struct TtScratch {
  long long part, part_ml, info, total;
  int blocks, tiles, cluster;
};
static TtScratch tt_scratch(int n_seqs, int max_count, int heads, int kv_heads, int head_dim, int max_keys, int window) {
  TtScratch f{};
  const long long rows = (long long)max_count * (heads / kv_heads);
  f.tiles = (int)((rows + kTtTile - 1) / kTtTile);
  f.cluster = tt_cluster(n_seqs, kv_heads, f.tiles, max_count, max_keys, window);
  if (f.cluster) return f;
  const long long units = (long long)n_seqs * kv_heads * f.tiles * (((long long)max_keys + 63) / 64 + 1), most = std::min(sm_count(), kTtMostBlocks);
  f.blocks = (int)std::min(units, most);      // one an SM
  const int rows_pad = tt_layout(head_dim, (int)std::min(rows, (long long)kTtTile)).rows;
  long long at = 0;
  auto take = [&](long long n) { const long long o = at; at += (n + 3) & ~3ll; return o; };
  f.part = take(2ll * f.blocks * rows_pad * head_dim);
  f.part_ml = take(4ll * f.blocks * rows_pad);
  f.info = take(2ll * f.blocks);
  f.total = at;
  return f;
}

long long tree_tc_floats(int n_seqs, int max_count, int heads, int kv_heads, int head_dim, int max_keys) {
  return tt_scratch(n_seqs, max_count, heads, kv_heads, head_dim, max_keys, 0).total;      // (a window makes no share longer: what a step without one takes is enough)
}

static int encode_tree_pool(CUtensorMap* map, const void* base, long long rows, int head_dim, const char* what) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(2, "attention_tree: the driver does not offer cuTensorMapEncodeTiled");
  cuuint64_t dims[2] = {(cuuint64_t)head_dim, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)head_dim * 2};
  cuuint32_t box[2] = {64, 64}, estr[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : fail(2, "attention_tree: cuTensorMapEncodeTiled failed for %s with code %d", what, (int)r);
}

template <int HD>
static int launch_tree_tc(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const TtArgs& ta, int blocks, cudaStream_t s) {
  static std::atomic<unsigned long long> allowed, allowed_clusters;
  cudaError_t e = ta.cluster ? allow_shared((const void*)tree_tc_kernel<HD, true>, 224 * 1024, allowed_clusters) : allow_shared((const void*)tree_tc_kernel<HD, false>, 224 * 1024, allowed);
  if (e != cudaSuccess) return fail(2, "attention_tree: cannot reserve shared memory: %s", cudaGetErrorString(e));
  // (both may begin early: barriers and tensor memory are made while the kernel before ends. One chat, call after call: 11.2 us so, two more one after the other)
  if (ta.cluster) {
    launch_clusters(pdl_mode() != 0, (unsigned)ta.cluster, tree_tc_kernel<HD, true>, dim3(ta.cluster * ta.t.kv_heads * ta.tiles * ta.t.n_seqs), dim3(kTtThreads), (size_t)ta.lay.total, s, mq, mk, mv, ta);
    return check_launch("attention_tree (tensor cores, clusters)");
  }
  launch_prefetching(tree_tc_kernel<HD, false>, dim3(blocks), dim3(kTtThreads), (size_t)ta.lay.total, s, mq, mk, mv, ta);
  const int rc = check_launch("attention_tree (tensor cores)");
  if (rc) return rc;
  if (blocks == 1) return 0;
  launch_prefetching(tree_tc_join_kernel<HD>, dim3(std::min(4 * blocks, blocks * (ta.lay.rows * (HD / 4) / 256))), dim3(256), 0, s, ta, blocks);
  return check_launch("attention_tree (tensor cores, joined)");
}

int tree_tc(const TreeArgs& a, long long pool_pages, int* status, cudaStream_t s) {
  SLB_REQUIRE(pool_pages * a.kv_heads * 64 < (1ll << 31), "attention_tree: the pool has too many rows for one tensor map");
  SLB_REQUIRE((uintptr_t)a.q % 16 == 0 && (uintptr_t)a.k_pool % 16 == 0 && (uintptr_t)a.v_pool % 16 == 0 && (uintptr_t)a.out % 16 == 0 &&
              (uintptr_t)a.scratch % 16 == 0, "attention_tree: q, out, scratch and the pools must be 16-byte aligned");
  SLB_REQUIRE(status != nullptr, "attention_tree: no status word");
  CUtensorMap mq{}, mk, mv;
  int rc = encode_tree_pool(&mk, a.k_pool, pool_pages * a.kv_heads * 64, a.head_dim, "the key pool");
  if (rc == 0) rc = encode_tree_pool(&mv, a.v_pool, pool_pages * a.kv_heads * 64, a.head_dim, "the value pool");
  if (rc) return rc;
  const TtScratch f = tt_scratch(a.n_seqs, a.max_count, a.heads, a.kv_heads, a.head_dim, a.max_keys, a.window);
  SLB_REQUIRE((long long)a.kv_heads * f.tiles < 65536, "attention_tree: too many heads for one launch");
  TtArgs ta{};
  ta.t = a;
  ta.scale_log2 = a.scale * 1.4426950408889634f;
  int exponent = 0;
  const float fraction = frexpf(ta.scale_log2, &exponent);
  ta.far_scale = ldexpf(1.0f, fraction == 0.5f ? exponent - 1 : exponent);
  ta.far_back = 1.0f / ta.far_scale;
  if (!f.cluster) {
    ta.part = a.scratch + f.part;
    ta.part_ml = reinterpret_cast<float2*>(a.scratch + f.part_ml);
    ta.info = reinterpret_cast<int2*>(a.scratch + f.info);
  }
  ta.cluster = f.cluster;
  ta.status = status;
  ta.tiles = f.tiles;
  ta.lay = tt_layout(a.head_dim, (int)std::min((long long)a.max_count * (a.heads / a.kv_heads), (long long)kTtTile));
  const int G = a.heads / a.kv_heads;
  ta.q_by_tma = 32 % G == 0 && a.tokens < (1ll << 31);
  if (ta.q_by_tma) {
    EncodeTiledFn fn = encode_fn();
    const int nodes = ta.lay.rows / G;
    cuuint64_t dims[3] = {(cuuint64_t)a.head_dim, (cuuint64_t)a.heads, (cuuint64_t)a.tokens};
    cuuint64_t strides[2] = {(cuuint64_t)a.head_dim * 2, (cuuint64_t)a.heads * a.head_dim * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)G, (cuuint32_t)nodes}, estr[3] = {1, 1, 1};
    const CUresult r = fn(&mq, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(a.q), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(2, "attention_tree: cuTensorMapEncodeTiled failed for the queries with code %d", (int)r);
  }
  return a.head_dim == 128 ? launch_tree_tc<128>(mq, mk, mv, ta, f.blocks, s) : launch_tree_tc<64>(mq, mk, mv, ta, f.blocks, s);
}

}  // namespace slb
