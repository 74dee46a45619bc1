// Attention of drafted nodes (tree.cuh) on the tcgen05 tensor cores: bfloat16, heads of 64 and 128, any number of query heads a key/value head.
//
// What such a step costs is the read of the keys and values (up to 256 rows of queries meet each: 512 FLOP a byte at most), so the work is the pages: every sequence has
// (kv head, tile of 128 rows, page) units, and each block takes an equal run of the list of all units, whatever the sequences' lengths. A (sequence, kv head, tile) that
// lies in one run is finished by its block; the others' shares wait in scratch for a second kernel that joins them in their order.
//   warp 0      asks TMA for the run's pages of keys, into a ring, and issues S = Q K^T, 128 x 64, one page ahead of the softmax (two score buffers in tensor memory);
//   warp 1      the same for the values, and O += P V as soon as P is written, P read from tensor memory where S was;
//   warps 2..9  the softmax, two threads a row (32 keys of a page each) that agree on the row's running maximum; P is rounded to bfloat16 (the instruction takes no wider
//                one beside bfloat16 values), the sum is of the unrounded weights, in 32 bits.
// Rows are row r = node r / G, query head r % G of the group. Fewer than 128 rows leave the tile's other rows to whatever lies behind the queries in shared memory: a row of
// A reaches that row of the result alone, and nobody reads it. Two blocks an SM, so that one loads and multiplies while the other stands in its chain of load, maximum, powers and store.
// Rows that a node does not see are masked by a bit each. Their values meet a zero weight in the product, which an infinity or a NaN among them would survive: so in pages that
// not all rows see alike (the step's own and those at a window's edge) values that are not finite are taken out in shared memory, and nodes that do see them get them back at the end, a bit pair for each (row, channel).
#include <math.h>

#include <algorithm>

#include "tcgen05.cuh"
#include "tree.cuh"

namespace slb {

constexpr int kTtRows = 128, kTtThreads = 10 * 32, kTtSoft = 256;
constexpr float kTtRescale = 8.0f;      // log2 units by which a maximum may be stale

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

struct TtLayout {
  int rows, stages, k_off, v_off, poison_off, xch_off, sum_off, bar_off, total;
};
static TtLayout tt_layout(int HD, int rows) {
  TtLayout l;
  l.rows = std::min(kTtRows, (rows + 31) & ~31);
  const int page = 64 * HD * 2, q = l.rows * HD * 2, rest = l.rows * HD / 4 + 2 * 2 * kTtRows * 2 + 2 * kTtRows * 4 + 32 * 8;
  l.stages = std::min(4, (112 * 1024 - q - rest) / (2 * page));      // (113 KB a block, 1 KB of it static)
  l.k_off = q;
  l.v_off = l.k_off + l.stages * page;
  l.poison_off = l.v_off + l.stages * page;
  l.xch_off = l.poison_off + l.rows * HD / 4;
  l.sum_off = l.xch_off + 2 * 2 * kTtRows * 2;
  l.bar_off = l.sum_off + 2 * kTtRows * 4;
  l.total = l.bar_off + 32 * 8;
  return l;
}

struct TtArgs {
  TreeArgs t;
  float scale_log2;
  float* part;          // [blocks][2][HD][rows] weighted values
  float2* part_ml;      // [blocks][2][rows] maximum (log2 units) and sum
  int2* info;           // [n, kv_heads, tiles] first block and number of blocks
  int* status;
  int tiles;            // most tiles of a sequence
  TtLayout lay;
};

// The pages of a sequence that some node may see: those from the window of a node at `past` on.
struct TtSeq {
  int page_lo, pages, tiles, rows, units;
  __device__ __forceinline__ TtSeq(const TreeArgs& a, const TreeSeq& s) {
    const int G = a.heads / a.kv_heads;
    const long long lo = a.window > 0 ? (long long)s.past - a.window + 1 : 0;
    page_lo = lo > 0 ? (int)(lo / 64) : 0;
    pages = s.count > 0 ? (s.past + s.count - 1) / 64 - page_lo + 1 : 0;
    rows = s.count * G;
    tiles = (rows + kTtRows - 1) / kTtRows;
    units = pages * tiles * a.kv_heads;      // (the launcher has seen that all units of a call stay below 2^31)
  }
};

// A block's run of units, segment by segment: a segment is what the run holds of one (sequence, kv head, tile).
struct TtWalk {
  int u, u_hi, seq, seq_first;      // the next unit, the run's end; the sequence and its first unit
  int kh, tile, off, n;             // the segment: its first page within the sequence, its pages
  int past, count, tok0, page_lo, pages, rows;
  __device__ __forceinline__ bool next(const TreeArgs& a) {
    if (u >= u_hi) return false;
    while (true) {
      const TreeSeq s(a, seq);
      const TtSeq t(a, s);
      if (u < seq_first + t.units) {
        const int rel = u - seq_first, at = rel / t.pages;
        off = rel - at * t.pages;
        kh = at / t.tiles;
        tile = at - kh * t.tiles;
        n = min(t.pages - off, u_hi - u);
        past = s.past; count = s.count; tok0 = s.tok0;
        page_lo = t.page_lo; pages = t.pages; rows = t.rows;
        u += n;
        return true;
      }
      seq_first += t.units;
      ++seq;
    }
  }
};

// The same run page by page, for loads that go ahead of the products: rows of a tensor map's pool.
struct TtPages {
  TtWalk w;
  int i, ahead;      // pages taken of the segment; the number of the next page, read one page early
  const int* table;
  __device__ __forceinline__ void segment(const TreeArgs& a) {
    i = 0;
    if (w.next(a)) {
      table = a.block_table + (size_t)w.seq * a.table_stride + w.page_lo + w.off;
      ahead = table[0];
    } else {
      w.n = 0;
    }
  }
  __device__ __forceinline__ TtPages(const TtWalk& from, const TreeArgs& a) : w(from) { segment(a); }
  __device__ __forceinline__ bool next(const TreeArgs& a, int& row) {
    if (w.n == 0) return false;
    row = (ahead * a.kv_heads + w.kh) * 64;
    if (++i == w.n) segment(a);
    else ahead = table[i];
    return true;
  }
};

template <int HD>
__global__ void __launch_bounds__(kTtThreads, 2)
tree_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ TtArgs ta) {
  constexpr int PAGE = 64 * HD * 2;
  const TreeArgs& a = ta.t;
  const TtLayout& L = ta.lay;
  extern __shared__ __align__(1024) unsigned char smem[];
  __shared__ int warp_units[kTtThreads / 32];
  __shared__ int s_first, s_seq, s_lo, s_poison;
  __shared__ uint32_t s_odd[2], tmem_slot;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = smem_addr(smem);
  if ((base & 1023u) != 0) {
    if (tid == 0) atomicExch(ta.status, 91);
    return;
  }
  const uint32_t sK = base + L.k_off, sV = base + L.v_off, bars = base + L.bar_off;
  const uint32_t k_full = bars, k_free = bars + 32, v_full = bars + 64, v_free = bars + 96, s_full = bars + 128, p_full = bars + 144, pv_done = bars + 160,
                 q_full = bars + 176, o_free = bars + 184;
  if (tid == 0) {
    for (int i = 0; i < L.stages; ++i) {
      mbar_init(k_full + 8 * i, 1);
      mbar_init(k_free + 8 * i, 1);
      mbar_init(v_full + 8 * i, 1);
      mbar_init(v_free + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + 8 * i, 1);
      mbar_init(p_full + 8 * i, 8);
      mbar_init(pv_done + 8 * i, 1);
    }
    mbar_init(q_full, 8);
    mbar_init(o_free, 8);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    s_lo = s_poison = 0;
    s_odd[0] = s_odd[1] = 0u;
  }
  pdl_wait();

  // where this block's run of units begins
  const int G = a.heads / a.kv_heads;
  TtWalk run;
  int total = 0, blocks;
  {
    const int per = (a.n_seqs + kTtThreads - 1) / kTtThreads, q0 = min(a.n_seqs, tid * per), q1 = min(a.n_seqs, q0 + per);
    auto units_of = [&](int s) { return TtSeq(a, TreeSeq(a, s)).units; };
    int own = 0;
    for (int s = q0; s < q1; ++s) own += units_of(s);
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
    blocks = min((int)gridDim.x, total);
    if ((int)blockIdx.x >= blocks) return;
    run.u = (int)((long long)blockIdx.x * total / blocks);
    run.u_hi = (int)((long long)(blockIdx.x + 1) * total / blocks);
    before += incl - own;
    if (own > 0 && run.u >= before && run.u < before + own) {
      for (int s = q0; s < q1; ++s) {
        const int units = units_of(s);
        if (run.u < before + units) {
          s_seq = s;
          s_first = before;
          break;
        }
        before += units;
      }
    }
  }
  if (warp == 1) {
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_slot)), "r"(256) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch_dependents();      // (only now: a successor that also wants tensor memory must not take it before this block has its own)
  const uint32_t tmem = tmem_slot, tO = tmem + 128;
  run.seq = s_seq;
  run.seq_first = s_first;

  if (warp == 0) {
    if (elect_one()) {
      // ---- scores ----
      constexpr uint32_t idesc = instr_desc(kTtRows, 64);
      TtPages pages(run, a);
      int st = 0, lap = 0, jj = 0, seg = 0, lst = 0, loaded = 0;      // lst: the stage of the next load
      auto load = [&]() {      // (a stage is free once S of the page that lay there is complete; the caller has seen to it)
        int row;
        if (!pages.next(a, row)) return;
        mbar_expect_tx(k_full + 8 * lst, PAGE);
#pragma unroll
        for (int h = 0; h < HD / 64; ++h) tma_load_2d(sK + lst * PAGE + h * 8192, &map_k, h * 64, row, k_full + 8 * lst);
        if (++lst == L.stages) lst = 0;
        ++loaded;
      };
      for (int i = 0; i + 1 < L.stages; ++i) load();
      bool ok = true;
      while (ok && run.next(a)) {
        if (!mbar_wait(q_full, seg & 1)) { atomicExch(ta.status, 93); break; }
        ++seg;
        for (int i = 0; i < run.n; ++i, ++jj) {
          const int b = jj & 1, before = st ? st - 1 : L.stages - 1;
          if (jj >= 1 && !mbar_wait(k_free + 8 * before, (st ? lap : lap - 1) & 1)) { atomicExch(ta.status, 92); ok = false; break; }
          load();      // into the stage of page jj - 1
          if (!mbar_wait(k_full + 8 * st, lap & 1)) { atomicExch(ta.status, 94); ok = false; break; }
          // S lands where S and then P of two pages ago lay: the product that read that P must be through
          if (jj >= 2 && !mbar_wait(pv_done + 8 * b, ((jj >> 1) - 1) & 1)) { atomicExch(ta.status, 95); ok = false; break; }
          tc_fence_after();
#pragma unroll
          for (int h = 0; h < HD / 64; ++h) {
            const uint64_t dq = smem_desc(base + h * L.rows * 128), dk = smem_desc(sK + st * PAGE + h * 8192);
#pragma unroll
            for (int k4 = 0; k4 < 4; ++k4)
              mma_bf16_ss(tmem + (uint32_t)(b * 64), dq + (uint64_t)(k4 * 2), dk + (uint64_t)(k4 * 2), idesc, (h > 0 || k4 > 0) ? 1u : 0u);
          }
          mma_commit(s_full + 8 * b);
          mma_commit(k_free + 8 * st);
          if (++st == L.stages) { st = 0; ++lap; }
        }
      }
      // copies under way land before the block goes
      for (; jj < loaded; ++jj) {
        mbar_wait(k_full + 8 * st, lap & 1);
        if (++st == L.stages) { st = 0; ++lap; }
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      // ---- values ----
      constexpr uint32_t idesc = instr_desc(kTtRows, HD, true);
      TtPages pages(run, a);
      int st = 0, lap = 0, jj = 0, seg = 0, lst = 0, loaded = 0;
      auto load = [&]() {
        int row;
        if (!pages.next(a, row)) return;
        mbar_expect_tx(v_full + 8 * lst, PAGE);
#pragma unroll
        for (int h = 0; h < HD / 64; ++h) tma_load_2d(sV + lst * PAGE + h * 8192, &map_v, h * 64, row, v_full + 8 * lst);
        if (++lst == L.stages) lst = 0;
        ++loaded;
      };
      for (int i = 0; i + 1 < L.stages; ++i) load();
      bool ok = true;
      while (ok && run.next(a)) {
        if (seg > 0 && !mbar_wait(o_free, (seg - 1) & 1)) { atomicExch(ta.status, 96); break; }
        ++seg;
        for (int i = 0; i < run.n; ++i, ++jj) {
          const int b = jj & 1, before = st ? st - 1 : L.stages - 1;
          if (jj >= 1 && !mbar_wait(v_free + 8 * before, (st ? lap : lap - 1) & 1)) { atomicExch(ta.status, 92); ok = false; break; }
          load();
          if (!mbar_wait(v_full + 8 * st, lap & 1)) { atomicExch(ta.status, 97); ok = false; break; }
          if (!mbar_wait(p_full + 8 * b, (jj >> 1) & 1)) { atomicExch(ta.status, 98); ok = false; break; }
          tc_fence_after();
#pragma unroll
          for (int k4 = 0; k4 < 4; ++k4) {
            const uint64_t dv = smem_desc_mn(sV + st * PAGE + k4 * 2048, 8192, 1024);
            mma_bf16_ts(tO, tmem + (uint32_t)(b * 64 + k4 * 8), dv, idesc, (i > 0 || k4 > 0) ? 1u : 0u);
          }
          mma_commit(pv_done + 8 * b);
          mma_commit(v_free + 8 * st);
          if (++st == L.stages) { st = 0; ++lap; }
        }
      }
      for (; jj < loaded; ++jj) {
        mbar_wait(v_full + 8 * st, lap & 1);
        if (++st == L.stages) { st = 0; ++lap; }
      }
    }
  } else {
    // ---- softmax: tensor-memory lanes 32 (warp % 4) .. + 31 hold the rows; two warps share them, keys 0..31 and 32..63 of a page ----
    const int quad = warp & 3, half = (warp - 2) >> 2, r = quad * 32 + lane, stid = tid - 64;
    const uint32_t lane_addr = tmem + ((uint32_t)(quad * 32) << 16);
    unsigned short* xch = reinterpret_cast<unsigned short*>(smem + L.xch_off);      // [2 pages][2 halves][128 rows]
    float* xl = reinterpret_cast<float*>(smem + L.sum_off);                          // [2 halves][128 rows]
    uint32_t* poison = reinterpret_cast<uint32_t*>(smem + L.poison_off);             // [rows][HD / 16]
    // A wait that gives up ends nothing here: the warp notes it and walks on to the end, because others meet it at barriers; the status word says so.
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
    auto pair_sync = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(1 + quad) : "memory"); };
    auto all_sync = [&]() { asm volatile("bar.sync 5, 256;" ::: "memory"); };
    int st = 0, lap = 0, jj = 0;
    while (run.next(a)) {
      const int kh = run.kh, R0 = run.tile * kTtRows, rows = min(kTtRows, run.rows - R0), R = R0 + r, n = run.n;
      // queries, as a tile that TMA would have left: 64 channels a half, 16-byte pieces exchanged by the row
      for (int e = stid; e < L.rows * (HD / 8); e += kTtSoft) {
        const int qr = e / (HD / 8), col = e % (HD / 8) * 8;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (qr < rows) v = *reinterpret_cast<const uint4*>((const __nv_bfloat16*)a.q + ((size_t)(run.tok0 + (R0 + qr) / G) * a.heads + kh * G + (R0 + qr) % G) * HD + col);
        *reinterpret_cast<uint4*>(smem + (col >> 6) * (L.rows * 128) + qr * 128 + ((((col >> 3) & 7) ^ (qr & 7)) << 4)) = v;
      }
      for (int e = stid; e < L.rows * (HD / 16); e += kTtSoft) poison[e] = 0u;
      fence_smem_to_async();
      arrive_warp(q_full);
      const bool live = r < rows, warp_live = quad * 32 < rows;
      const uint32_t* words = a.seen + (size_t)(run.tok0 + (live ? R / G : 0)) * a.words;
      int lo = 0, lo_most = 0;
      if (a.window > 0) {      // the latest beginning of a window in the tile
        lo = live ? tree_lo(a, run.tok0 + R / G, run.past) : 0;
        if (live) atomicMax(&s_lo, lo);
        all_sync();
        lo_most = s_lo;
      }
      float m_used = -INFINITY, l = 0.0f;
      for (int i = 0; i < n; ++i, ++jj) {
        const int b = jj & 1, key_page = (run.page_lo + run.off + i) * 64, key0 = key_page + half * 32;
        wait_warp(s_full + 8 * b, (jj >> 1) & 1, 99);
        const bool mixed = key_page + 63 >= run.past || key_page < lo_most;      // not all rows see all of the page
        uint32_t seen = 0xffffffffu;
        if (warp_live) {
          tc_fence_after();
          uint32_t sr[32];
          tmem_ld32(lane_addr + (uint32_t)(b * 64 + half * 32), sr);
          if (mixed) {
            const int to = run.past - key0, from = lo - key0;
            seen = (to >= 32 ? 0xffffffffu : to <= 0 ? 0u : (1u << to) - 1u) & (from <= 0 ? 0xffffffffu : from >= 32 ? 0u : 0xffffffffu << from);
            if (key0 + 31 >= run.past) seen |= (uint32_t)tree_bits(words, a.words, key0 - run.past, run.count);
            if (!live) seen = 0u;
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if (!(seen >> c & 1u)) sr[c] = 0xff800000u;     // -inf
          }
          float mx = -INFINITY;
#pragma unroll
          for (int c = 0; c < 32; c += 2) mx = tt_max3(mx, __uint_as_float(sr[c]), __uint_as_float(sr[c + 1]));
          // The row's maximum is the larger of the two halves'. They are exchanged rounded up to 16 bits (any common reference at or above the maximum serves a
          // softmax), so both threads of a row take the same decisions.
          {
            const uint32_t bits = __float_as_uint(mx);
            const unsigned short up = (unsigned short)(((bits & 0x80000000u) ? bits : bits + 0xffffu) >> 16);
            xch[b * 256 + half * 128 + r] = up;      // (a place per parity: the partner passes the barrier of the next page only after reading this one)
            pair_sync();
            const unsigned short other = xch[b * 256 + (half ^ 1) * 128 + r];
            mx = fmaxf(__uint_as_float((uint32_t)up << 16), __uint_as_float((uint32_t)other << 16));
          }
          const float m_new = fmaxf(m_used, mx * ta.scale_log2);      // the scale is positive
          const bool grow = m_new > m_used + kTtRescale;              // also true for the first finite maximum
          if (i > 0 && __any_sync(0xffffffffu, grow)) {
            wait_warp(pv_done + 8 * ((jj - 1) & 1), ((jj - 1) >> 1) & 1, 100);      // O must hold all of the last product
            tc_fence_after();
            const float alpha = grow ? tt_ex2(m_used - m_new) : 1.0f;
#pragma unroll
            for (int c0 = 0; c0 < HD / 2; c0 += 16) {      // this thread's half of the accumulator row
              uint32_t o[16];
              tmem_ld16(lane_addr + 128 + half * (HD / 2) + c0, o);
#pragma unroll
              for (int c = 0; c < 16; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * alpha);
              tmem_st16(lane_addr + 128 + half * (HD / 2) + c0, o);
            }
            l *= alpha;
          }
          if (grow) m_used = m_new;
          const float neg_m = m_used == -INFINITY ? 0.0f : -m_used;
          uint32_t pk[16];
          float l0 = 0.0f, l1 = 0.0f;
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            const float p0 = tt_ex2(fmaf(__uint_as_float(sr[c]), ta.scale_log2, neg_m)), p1 = tt_ex2(fmaf(__uint_as_float(sr[c + 1]), ta.scale_log2, neg_m));
            __nv_bfloat162 h2 = __floats2bfloat162_rn(p0, p1);
            pk[c >> 1] = *reinterpret_cast<uint32_t*>(&h2);
            l0 += p0;
            l1 += p1;
          }
          l += l0 + l1;
          tmem_st16(lane_addr + (uint32_t)(b * 64 + half * 16), pk);
        }
        if (mixed) {
          // values that are not finite go; rows that see one remember it
          wait_warp(v_full + 8 * st, lap & 1, 101);
          const int held = run.past + run.count - key_page;      // rows of the page that belong to the sequence
#pragma unroll
          for (int e = stid; e < 64 * HD / 8; e += kTtSoft) {
            const int row = e & 63, slab = e >> 6;           // a 16-byte piece of a row, in any order
            const uint32_t at = sV + st * PAGE + (slab >> 3) * 8192 + row * 128 + (slab & 7) * 16;
            uint4 v;
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
            auto bad = [](uint32_t x) { return ((x & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((x & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u); };
            const uint32_t b0 = bad(v.x), b1 = bad(v.y), b2 = bad(v.z), b3 = bad(v.w);
            if (b0 | b1 | b2 | b3) {
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x & ~b0), "r"(v.y & ~b1), "r"(v.z & ~b2), "r"(v.w & ~b3) : "memory");
              if (row < held) atomicOr(&s_odd[row >> 5], 1u << (row & 31));
            }
          }
          fence_smem_to_async();
          all_sync();
          const uint32_t odd0 = s_odd[0], odd1 = s_odd[1];
          if (odd0 | odd1) {
            const int page = a.block_table[(size_t)run.seq * a.table_stride + key_page / 64];
            for (uint32_t left = live ? (half ? odd1 : odd0) & seen : 0u; left; left &= left - 1) {
              const uint32_t* v = reinterpret_cast<const uint32_t*>((const __nv_bfloat16*)a.v_pool + (((size_t)page * a.kv_heads + kh) * 64 + half * 32 + __ffs(left) - 1) * HD);
              for (int c = 0; c < HD; ++c) {
                const uint32_t x = v[c >> 1] >> (c & 1) * 16 & 0xffffu;
                if ((x & 0x7f80u) == 0x7f80u) {
                  atomicOr(&poison[r * (HD / 16) + c / 16], ((x & 0x7fu) ? 3u : x >> 15 ? 2u : 1u) << (c % 16 * 2));
                  s_poison = 1;
                }
              }
            }
            all_sync();
            if (stid < 2) s_odd[stid] = 0u;
            all_sync();
          }
        }
        tc_fence_before();
        arrive_warp(p_full + 8 * b);
        if (++st == L.stages) { st = 0; ++lap; }
      }
      // ---- the segment's results ----
      wait_warp(pv_done + 8 * ((jj - 1) & 1), ((jj - 1) >> 1) & 1, 102);
      const bool begins = run.off == 0, complete = begins && n == run.pages;
      if (begins && stid == 0) {      // (the segment's first unit is u - n)
        const long long last = run.u - n + run.pages - 1;
        ta.info[((long long)run.seq * a.kv_heads + kh) * ta.tiles + run.tile] = make_int2((int)blockIdx.x, (int)(((last + 1) * blocks - 1) / total) - (int)blockIdx.x + 1);
      }
      if (warp_live) {
        xl[half * 128 + r] = l;
        pair_sync();
        l += xl[(half ^ 1) * 128 + r];
        tc_fence_after();
      }
      all_sync();      // (poison is complete)
      const float inv = !complete ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
      const size_t slot = (size_t)blockIdx.x * 2 + (begins ? 1 : 0);
#pragma unroll
      for (int c0 = 0; c0 < HD / 2; c0 += 16) {      // this thread's half of the accumulator row
        if (!warp_live) break;
        uint32_t o[16];
        __syncwarp();
        tmem_ld16(lane_addr + 128 + half * (HD / 2) + c0, o);
        if (!live) continue;
        const int ch = half * (HD / 2) + c0;
        const uint32_t x = s_poison ? poison[r * (HD / 16) + ch / 16] : 0u;
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          float v = l == 0.0f ? 0.0f : __uint_as_float(o[c]) * inv;      // (0: nothing seen)
          if (x >> (2 * c) & 3u) v += (x >> (2 * c) & 3u) == 1u ? INFINITY : (x >> (2 * c) & 3u) == 2u ? -INFINITY : NAN;
          o[c] = __float_as_uint(v);
        }
        if (complete) {
#pragma unroll
          for (int c = 0; c < 16; c += 8) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              __nv_bfloat162 h2 = __floats2bfloat162_rn(__uint_as_float(o[c + 2 * k]), __uint_as_float(o[c + 2 * k + 1]));
              w[k] = *reinterpret_cast<uint32_t*>(&h2);
            }
            const int piece = (ch + c) >> 3;      // (rows in the queries' place, pieces exchanged so that a warp's rows meet different banks)
            *reinterpret_cast<uint4*>(smem + r * (HD * 2) + (((piece & ~7) | ((piece ^ r) & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        } else {
          float* part = ta.part + (slot * HD + ch) * L.rows + r;
#pragma unroll
          for (int c = 0; c < 16; ++c) part[(size_t)c * L.rows] = __uint_as_float(o[c]);
        }
      }
      tc_fence_before();
      arrive_warp(o_free);
      if (complete) {
        all_sync();
        for (int e = stid; e < rows * (HD / 8); e += kTtSoft) {
          const int rr = e / (HD / 8), piece = e % (HD / 8);
          const uint4 v = *reinterpret_cast<const uint4*>(smem + rr * (HD * 2) + (((piece & ~7) | ((piece ^ rr) & 7)) << 4));
          if (ok) *reinterpret_cast<uint4*>((__nv_bfloat16*)a.out + ((size_t)(run.tok0 + (R0 + rr) / G) * a.heads + kh * G + (R0 + rr) % G) * HD + piece * 8) = v;
        }
      } else if (live && half == 0) {
        ta.part_ml[slot * L.rows + r] = make_float2(m_used, l);
      }
      all_sync();
      if (stid == 0) s_lo = s_poison = 0;
      all_sync();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256) : "memory");
}

// Joins the shares of what no block finished alone: a block takes 8 or more channels of a (sequence, kv head, tile), a thread a row and eight channels.
template <int HD>
__global__ void __launch_bounds__(256) tree_tc_join_kernel(TtArgs ta) {
  pdl_wait();
  const TreeArgs& a = ta.t;
  const int rows_pad = ta.lay.rows, seq = blockIdx.z, kh = blockIdx.y / ta.tiles, tile = blockIdx.y % ta.tiles, G = a.heads / a.kv_heads;
  const TreeSeq s(a, seq);
  const int rows = min(kTtRows, s.count * G - tile * kTtRows);
  if (rows <= 0) return;
  const int2 in = ta.info[((size_t)seq * a.kv_heads + kh) * ta.tiles + tile];
  if (in.y == 1) return;      // its block has finished it
  const int e = blockIdx.x * 256 + threadIdx.x, r = e % rows_pad, c0 = e / rows_pad * 8;
  if (r >= rows || c0 >= HD) return;
  auto slot_of = [&](int i) { return (size_t)(in.x + i) * 2 + (i == 0 ? 1 : 0); };
  float M = -INFINITY, l = 0.0f, acc[8];
#pragma unroll
  for (int c = 0; c < 8; ++c) acc[c] = 0.0f;
  for (int i0 = 0; i0 < in.y; i0 += 4) {
    float2 ml[4];
    float v[4][8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const size_t slot = slot_of(min(i0 + i, in.y - 1));
      ml[i] = ta.part_ml[slot * rows_pad + r];
      if (i0 + i >= in.y) ml[i] = make_float2(-INFINITY, 0.0f);
#pragma unroll
      for (int c = 0; c < 8; ++c) v[i][c] = ta.part[(slot * HD + c0 + c) * rows_pad + r];
    }
    float top = M;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = fmaxf(top, ml[i].x);
    const float use = top == -INFINITY ? 0.0f : top, keep = tt_ex2(M - use);
    l *= keep;
#pragma unroll
    for (int c = 0; c < 8; ++c) acc[c] *= keep;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i0 + i >= in.y || ml[i].y == 0.0f) continue;      // (a share that saw nothing; one whose scores were all NaN has a sum of NaN)
      const float f = tt_ex2(ml[i].x - use);
      l += ml[i].y * f;
#pragma unroll
      for (int c = 0; c < 8; ++c) acc[c] += v[i][c] * f;
    }
    M = top;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint32_t w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    __nv_bfloat162 h2 = __floats2bfloat162_rn(acc[2 * k] * inv, acc[2 * k + 1] * inv);
    w[k] = *reinterpret_cast<uint32_t*>(&h2);
  }
  const int R = tile * kTtRows + r;
  *reinterpret_cast<uint4*>((__nv_bfloat16*)a.out + ((size_t)(s.tok0 + R / G) * a.heads + kh * G + R % G) * HD + c0) = make_uint4(w[0], w[1], w[2], w[3]);
}

bool tree_tc_takes(int n_seqs, int max_count, int heads, int kv_heads, int head_dim, int max_keys, int dtype) {
  const long long tiles = ((long long)max_count * (heads / kv_heads) + kTtRows - 1) / kTtRows;
  return dtype == kBF16 && (head_dim == 64 || head_dim == 128) && n_seqs * tiles * kv_heads * (max_keys / 64 + 2ll) < (1ll << 31);
}

struct TtScratch {
  long long part, part_ml, info, total;
  int blocks, tiles;
};
static TtScratch tt_scratch(int n_seqs, int max_count, int heads, int kv_heads, int head_dim, int max_keys) {
  TtScratch f{};
  const long long rows = (long long)max_count * (heads / kv_heads);
  f.tiles = (int)((rows + kTtRows - 1) / kTtRows);
  const long long units = (long long)n_seqs * kv_heads * f.tiles * ((max_keys + 63) / 64 + 1), most = 2ll * sm_count();
  f.blocks = (int)std::min(units, most);      // as many as run at once
  const int rows_pad = tt_layout(head_dim, (int)std::min(rows, (long long)kTtRows)).rows;
  long long at = 0;
  auto take = [&](long long n) { const long long o = at; at += (n + 3) & ~3ll; return o; };
  f.part = take(2ll * f.blocks * rows_pad * head_dim);
  f.part_ml = take(4ll * f.blocks * rows_pad);
  f.info = take(2ll * n_seqs * kv_heads * f.tiles);
  f.total = at;
  return f;
}

long long tree_tc_floats(int n_seqs, int max_count, int heads, int kv_heads, int head_dim, int max_keys) {
  return tt_scratch(n_seqs, max_count, heads, kv_heads, head_dim, max_keys).total;
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
static int launch_tree_tc(const CUtensorMap& mk, const CUtensorMap& mv, const TtArgs& ta, int blocks, cudaStream_t s) {
  static std::atomic<unsigned long long> allowed;
  const cudaError_t e = allow_shared((const void*)tree_tc_kernel<HD>, 113 * 1024, allowed);
  if (e != cudaSuccess) return fail(2, "attention_tree: cannot reserve shared memory: %s", cudaGetErrorString(e));
  launch(tree_tc_kernel<HD>, dim3(blocks), dim3(kTtThreads), (size_t)ta.lay.total, s, mk, mv, ta);
  const int rc = check_launch("attention_tree (tensor cores)");
  if (rc) return rc;
  launch_prefetching(tree_tc_join_kernel<HD>, dim3((ta.lay.rows * (HD / 8) + 255) / 256, ta.t.kv_heads * ta.tiles, ta.t.n_seqs), dim3(256), 0, s, ta);
  return check_launch("attention_tree (tensor cores, joined)");
}

int tree_tc(const TreeArgs& a, long long pool_pages, int* status, cudaStream_t s) {
  SLB_REQUIRE(pool_pages * a.kv_heads * 64 < (1ll << 31), "attention_tree: the pool has too many rows for one tensor map");
  SLB_REQUIRE((uintptr_t)a.q % 16 == 0 && (uintptr_t)a.k_pool % 16 == 0 && (uintptr_t)a.v_pool % 16 == 0 && (uintptr_t)a.out % 16 == 0 &&
              (uintptr_t)a.scratch % 16 == 0, "attention_tree: q, out, scratch and the pools must be 16-byte aligned");
  SLB_REQUIRE(status != nullptr, "attention_tree: no status word");
  CUtensorMap mk, mv;
  int rc = encode_tree_pool(&mk, a.k_pool, pool_pages * a.kv_heads * 64, a.head_dim, "the key pool");
  if (rc == 0) rc = encode_tree_pool(&mv, a.v_pool, pool_pages * a.kv_heads * 64, a.head_dim, "the value pool");
  if (rc) return rc;
  const TtScratch f = tt_scratch(a.n_seqs, a.max_count, a.heads, a.kv_heads, a.head_dim, a.max_keys);
  SLB_REQUIRE((long long)a.kv_heads * f.tiles < 65536, "attention_tree: too many heads for one launch");
  TtArgs ta{};
  ta.t = a;
  ta.scale_log2 = a.scale * 1.4426950408889634f;
  ta.part = a.scratch + f.part;
  ta.part_ml = reinterpret_cast<float2*>(a.scratch + f.part_ml);
  ta.info = reinterpret_cast<int2*>(a.scratch + f.info);
  ta.status = status;
  ta.tiles = f.tiles;
  ta.lay = tt_layout(a.head_dim, (int)std::min((long long)a.max_count * (a.heads / a.kv_heads), (long long)kTtRows));
  return a.head_dim == 128 ? launch_tree_tc<128>(mk, mv, ta, f.blocks, s) : launch_tree_tc<64>(mk, mv, ta, f.blocks, s);
}

}  // namespace slb
