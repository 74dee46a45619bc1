// Which drafted tokens the target's probabilities accept, and the token behind the last of them.
//
// Every sequence brings a tree: node 0 is its newest certain token, row t of `logits` what the target says behind node t. With l the logits of the node reached,
// p(i) = exp(l_i / T) / Z over i < limit with l_i >= floor, q the distribution that its children were drawn from, independently, the children x are tried in their
// order: x is accepted with probability min(1, p(x) / q(x)); after a refusal p becomes max(p - q, 0) over its sum. Refusals in a row stay in one family:
//   p after k refusals = max(p - c_k q, 0) / F_k,   F_k = sum max(p - c_k q, 0),   c_0 = 0, F_0 = 1, c_{k+1} = c_k + F_k,
// because max(max(p - c q, 0) / F - q, 0) = max(p - (c + F) q, 0) / F. So child x with the number u goes through iff p(x) > (c + u F) q(x), and a refusal costs one
// sum over the row. Certain drafts are point masses: p(x) > u (1 - R), R the probability of the distinct tokens refused before. Where no child is left the next token is
// drawn from what p has become: the first token, in the order of their numbers, where the running sum passes u of the whole. Temperature 0: the child that is
// the row's first largest logit, and in the end that token.
//
// Two kernels: the first leaves the largest logit and the sum Z of every node that has children, the whole GPU over all of them; the second walks the sequences'
// ways, a cluster of up to sixteen blocks each, a run of the row a warp, and reads whole rows only where a draft is refused or the next token is drawn. (Where the
// rows of all nodes would be too much to read, kMostStatsBytes, the second finds Z by itself, row by row.) Results are whole numbers and have to be the
// definition's. Z comes from 32-bit powers summed in 64 bits, off by some 1e-7 (the power unit's 2^-22, rounded exponents and partial sums, 1e-5 at the very most), and
// where a child lies nearer to its number than kVerifyDoubt the row's exact sum decides, one pass that one child in 30,000 takes; a draw compares one number with
// 150,000 running sums. Those sums, and refusals', are of powers in pairs of 32-bit numbers, off by some 1e-12 (1e-11 where logits over temperature pass 1,000; a
// table of 64 and four terms of the series; in 64 bits, of which an SM does 16 operations a clock, a pass over a row took 7.5 us in eight blocks, four fifths of
// them waiting for that unit). A refusal takes one pass: the sums of exp, and of exp and of q over the tokens where exp / Z > c q as far as 32 bits tell, make both
// the exact Z and F (a token on the wrong side is off by 1e-7 of itself, and one in a million is).
// Measured (one B200, device, 151,936 tokens): one sequence of five drafts with distributions 21 us, 64 sequences of two to five 77 (the first kernel 32 for 137 MB,
// 4.2 TB/s; the second 50 in clusters of two, one pass of some 60 instructions a token and one of 300 tokens by the block that draws), eight trees of 15 to 23
// certain drafts 36 (19 and 23). Steps before: every row by the blocks of its sequence, in 64 bits 45, 128 and 27; sums of all nodes first, 64-bit powers 27, 91 and
// 45; pairs of 32-bit numbers, clusters of sixteen blocks of 512 threads 18, 86 and 38; of 1,024 threads 21, 75 and 37, which is kept: a batch has fewer blocks a
// sequence and gains most.
// Sums first or row by row, both in the present form, drafts certain (which need no pass for a refusal): eight trees whose first draft is refused 36 and 37 us, whose
// first drafts are right 43 and 108; 64 chains 62 and 85, 80 and 193; at temperature 0 the trees 28 and 18, 33 and 62, the chains 36 and 45, 56 and 106. Row by row
// gains 10 us where a greedy tree is refused at once and loses 30 to 110 where drafts are right; what will be accepted is not known before, so sums come first, with
// distributions and without.
#include <float.h>
#include <math.h>

#include "tcgen05.cuh"      // clusters
#include "tree.cuh"

namespace slb {

constexpr int kVerifyTeam = 16, kVerifyThreads = 1024, kVerifyWarps = kVerifyThreads / 32, kVerifyRuns = kVerifyTeam * kVerifyWarps;
constexpr double kVerifyDoubt = 0x1p-16;      // of a probability: what the rough sums may be off by, with room
constexpr long long kMostStatsBytes = 512ll << 20;      // 80 us of reading at most in front of the way; beyond it few rows of many lie on a way

// Of a piece of a row of logits: the largest kept one, its first place, and the sum of exp((l - top) / T).
struct VerifyStat {
  float top;
  int best;
  double z;
};

// What a caller says, in one piece of memory (as KeptCall, kept.cuh).
struct VerifyCall {
  const float *logits, *probs, *floors, *uniforms;
  const int *tokens, *parents, *seq_start, *counts;
  int *path, *lengths, *chosen, *scratch;
  void* stream;
  long long rows, ld, ldp, scratch_words;
  double temperature;
  int n_seqs, limit, max_count, path_width;
};
static_assert(sizeof(VerifyCall) == 13 * 8 + 4 * 8 + 8 + 4 * 4, "as packed in kernels/ops.py");

struct VerifyArgs {
  const float *logits, *probs, *floors, *uniforms;
  const int *tokens, *parents, *seq_start, *counts;
  int *path, *lengths, *chosen;
  long long rows, ld, ldp;
  double scale, unscale;      // log2 e / T, and one over it; 0: the largest logit alone counts
  float scale_hi, scale_lo, least;      // least: a difference of logits whose power is nothing
  VerifyStat* stats;          // [rows, pieces], or null
  int limit, max_count, path_width, run, vec;      // run: tokens of a warp, a multiple of 4
  int team, pieces, steps;    // blocks of a sequence; pieces of a row in the first kernel, and their steps
};

struct VerifyExchange {
  double sum[2][3][kVerifyWarps];      // two copies, used in turn: a block may write its next share while a slower one still reads the last
  double z[2];
  float max[2];
  int best[2];
};

struct VerifyShared {
  VerifyExchange x;
  float2 table[64];                 // 2^(j / 64), in two parts
  double runs[kVerifyRuns];         // sums up to and with each run
  double red_z[kVerifyWarps];
  double scan[kVerifyWarps];
  float red_m[kVerifyWarps];
  int red_i[kVerifyWarps];
  VerifyStat stat[kMostNodes];
  int inner[kMostNodes];            // whether a node has children
  int parent[kMostNodes], token[kMostNodes], refused[kMostNodes];
  double p[kMostNodes];
  float logit[kMostNodes], prob[kMostNodes], u[kMostNodes];
  double total_z;
  float top;
  int best, found, last;
};

__device__ __forceinline__ double peer_f64(uint32_t addr) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float peer_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A sum of numbers from 0 to 1 in two parts: each addition's error is kept. It begins at 4 so that no number is larger than the sum.
struct PairSum {
  float hi = 4.0f, lo = 0.0f;
  __device__ __forceinline__ void add(float x, float rest) {
    const float t = hi + x;
    lo += (x - (t - hi)) + rest;
    hi = t;
  }
  __device__ __forceinline__ double value() const { return ((double)hi - 4.0) + (double)lo; }
};

// 2^y scaled so that the row's largest logit has between 1/2 and 1, y = l * log2 e / T in two parts (the product's error is an FMA away): y = m + j / 64 + r with
// |r| <= 1 / 128, 2^r = 1 + a + b with a = r ln 2 rounded and b its error and the series' other terms up to the fourth, 2^(j / 64) from the table in two parts. Off
// by 1e-12 or less. Logits are counted from `base`: 0, or the largest where its y is beyond 1,000 (all that counts then lies so near that the difference is exact).
struct PairPower {
  float scale_hi, scale_lo, base, cap, least;      // below `least` nothing counts; from `base` no logit lies further up than `cap`
  int bias;                                   // what makes a power of two of the whole part
  bool none;                                  // nothing counts
  __device__ __forceinline__ PairPower() {}
  __device__ __forceinline__ PairPower(const VerifyArgs& a, float top, float floor) {
    const double y = (double)top * a.scale;
    scale_hi = a.scale_hi;
    scale_lo = a.scale_lo;
    const bool near = fabs(y) <= 1000.0;
    base = near ? 0.0f : top;
    cap = near ? FLT_MAX : 0.0f;
    bias = (127 - (near ? (int)ceil(y) : 0)) << 23;
    none = floor != floor || !(top > -INFINITY);
    least = top < INFINITY ? fmaxf(floor, (float)(top - 120.0 * a.unscale)) : INFINITY;
  }
  __device__ __forceinline__ float2 of(float l, const float2* table) const {
    constexpr double kLn2 = 0.6931471805599453;
    constexpr float kHi = (float)kLn2, kLo = (float)(kLn2 - (double)kHi);
    const bool counts = l >= least && !none;
    const float x = fminf(fmaxf(l, least) - base, cap);      // (inf - inf, beside an infinite logit, is no number and becomes `cap`: 0)
    const float p = __fmul_rn(x, scale_hi), e = fmaf(x, scale_lo, fmaf(x, scale_hi, -p));
    const float t = fmaf(p, 64.0f, 12582912.0f);      // 1.5 * 2^23: the nearest whole number in the low bits
    const uint32_t bits = __float_as_uint(t);
    const float r = fmaf(t - 12582912.0f, -0.015625f, p), r1 = r + e;
    const float a = __fmul_rn(r, kHi);
    float g = fmaf(r1, (float)(kLn2 * kLn2 * kLn2 * kLn2 / 24.0), (float)(kLn2 * kLn2 * kLn2 / 6.0));
    g = fmaf(r1, g, (float)(kLn2 * kLn2 / 2.0));
    const float b = fmaf(r1 * r1, g, fmaf(e, kHi, fmaf(r, kLo, fmaf(r, kHi, -a))));
    const float2 f = table[bits & 63u];
    const float h = __fmul_rn(f.x, a);                // (products that are also parts: never joined with a sum)
    float lo = fmaf(f.x, b, fmaf(f.x, a, -h)) + fmaf(f.y, a, f.y);
    const float s = f.x + h;
    lo += h - (s - f.x);
    const float two = counts ? __uint_as_float(((bits & ~63u) << 17) + (uint32_t)bias) : 0.0f;      // (from 2^-122 on; the magic number's own bits leave at the top)
    return make_float2(s * two, lo * two);
  }
};

// f(token, logit, q) for tokens lo .. hi - 1 of a row of logits and, if there is one, a row of q (else 0), by the lanes of a warp; `vec`: 16-byte reads, lo a
// multiple of 4. The next eight tokens of a lane are on their way while f works on four: loops that fetch their instructions once (unrolled twice as far every pass
// waited for instructions more than for anything else).
template <bool PAIR, typename F>
__device__ __forceinline__ void each_logit(const float* row, const float* other, int lo, int hi, int lane, bool vec, F f) {
  if (vec) {
    const int last = hi - 4;      // the last place of a whole 16-byte read
    int i = lo + 4 * lane;
    constexpr int AHEAD = 2;
    float4 v[AHEAD], q[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (i + 128 * k <= last) {
        v[k] = *reinterpret_cast<const float4*>(row + i + 128 * k);
        if (PAIR) q[k] = *reinterpret_cast<const float4*>(other + i + 128 * k);
      }
#pragma unroll 1
    for (; i <= last; i += 128) {
      const float4 x = v[0], y = PAIR ? q[0] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int k = 0; k + 1 < AHEAD; ++k) {
        v[k] = v[k + 1];
        if (PAIR) q[k] = q[k + 1];
      }
      if (i + 128 * AHEAD <= last) {
        v[AHEAD - 1] = *reinterpret_cast<const float4*>(row + i + 128 * AHEAD);
        if (PAIR) q[AHEAD - 1] = *reinterpret_cast<const float4*>(other + i + 128 * AHEAD);
      }
      f(i, x.x, y.x);
      f(i + 1, x.y, y.y);
      f(i + 2, x.z, y.z);
      f(i + 3, x.w, y.w);
    }
    // what is left of four
    const int tail = lo + ((hi - lo) & ~3) + lane;
    if (hi > lo && tail < hi) f(tail, row[tail], PAIR ? other[tail] : 0.0f);
  } else {
    int i = lo + lane;
#pragma unroll 1
    for (; i + 3 * 32 < hi; i += 4 * 32) {
      float v[4], q[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[k] = row[i + 32 * k];
        q[k] = PAIR ? other[i + 32 * k] : 0.0f;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) f(i + 32 * k, v[k], q[k]);
    }
#pragma unroll 1
    for (; i < hi; i += 32) f(i, row[i], PAIR ? other[i] : 0.0f);
  }
}

// exp((l - m) / T) from the 32-bit unit, l <= m
__device__ __forceinline__ float rough_exp(const VerifyArgs& a, float l, float m) {
  const float x = l - m, t = x * a.scale_hi;
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(fmaf(x, a.scale_hi, x * a.scale_lo)));
  return l == m ? 1.0f : t > -1e4f ? y : 0.0f;      // (infinities end here)
}

__device__ __forceinline__ float ex2_f32(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// What counts as a logit of row t: at or above its floor; -inf has no probability, nor has NaN.
__device__ __forceinline__ float floor_of(const VerifyArgs& a, size_t t) {
  if (a.floors == nullptr) return -FLT_MAX;
  const float f = a.floors[t];
  return f != f ? f : fmaxf(f, -FLT_MAX);
}

constexpr int kStatsThreads = 256, kStatsStep = 4096;      // tokens that a block holds at once, the next ones on their way
// A piece of the row of a node that has children: `steps` steps. A thread's sum is relative to its own largest logit, in units of log2 after the temperature.
__global__ void __launch_bounds__(kStatsThreads, 5) verify_stats_kernel(VerifyArgs a) {
  pdl_enter();
  __shared__ float top_s[kStatsThreads / 32];
  __shared__ int best_s[kStatsThreads / 32];
  __shared__ double z_s[kStatsThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, seq = blockIdx.y, node = blockIdx.z;
  const int tok0 = a.seq_start[seq], count = min(max(a.counts[seq], 0), a.max_count);
  if (node >= count || tok0 < 0 || (long long)tok0 + count > a.rows) return;
  bool child = false;
  for (int j = node + 1 + tid; j < count; j += kStatsThreads) child = child || a.parents[tok0 + j] == node;
  if (!__syncthreads_or(child)) return;
  const size_t t = (size_t)tok0 + node;
  const float* row = a.logits + t * a.ld;
  const float floor = floor_of(a, t);
  const long long piece = (long long)a.steps * kStatsStep;
  const int begin = (int)min((long long)a.limit, blockIdx.x * piece), end = (int)min((long long)a.limit, begin + piece);
  constexpr int PER = kStatsStep / kStatsThreads;
  // (vec: thread tid has tokens at + 4 tid + 1024 k .. + 3, else at + tid + 256 k)
  auto token = [&](int at, int k) { return a.vec ? at + 4 * tid + 4 * kStatsThreads * (k >> 2) + (k & 3) : at + tid + kStatsThreads * k; };
  auto load = [&](int at, float (&v)[PER]) {
    if (a.vec) {
#pragma unroll
      for (int k = 0; k < PER; k += 4) {
        const int i = at + 4 * tid + kStatsThreads * k;
        if (i + 3 < end) {
          const float4 x = *reinterpret_cast<const float4*>(row + i);
          v[k] = x.x; v[k + 1] = x.y; v[k + 2] = x.z; v[k + 3] = x.w;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[k + e] = i + e < end ? row[i + e] : -INFINITY;
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < PER; ++k) v[k] = token(at, k) < end ? row[token(at, k)] : -INFINITY;
    }
  };
  const bool greedy = a.scale == 0.0;
  float top = -INFINITY, v[PER];
  int best = 0x7fffffff;
  double z = 0.0;
  load(begin, v);
#pragma unroll 1
  for (int at = begin; at < end; at += kStatsStep) {
    float next[PER];
    if (at + kStatsStep < end) load(at + kStatsStep, next);
    if (greedy) {
#pragma unroll
      for (int k = 0; k < PER; ++k)
        if (token(at, k) < end && (v[k] > top || (v[k] == top && token(at, k) < best))) { top = v[k]; best = token(at, k); }
    } else {
      float high = top;
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        v[k] = v[k] >= floor ? v[k] : -INFINITY;
        high = fmaxf(high, v[k]);
      }
      if (high > top) {
        z = top > -INFINITY ? z * rough_exp(a, top, high) : 0.0;
        top = high;
      }
      float part = 0.0f;
      if (fabsf(top) < INFINITY) {
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          const float y = ex2_f32(fmaxf(v[k] - top, a.least) * a.scale_hi);      // (a difference: nothing is lost where logits over temperature are large)
          part += v[k] > -INFINITY ? y : 0.0f;
        }
      } else if (top > -INFINITY) {      // infinite: as many of them as there are
#pragma unroll
        for (int k = 0; k < PER; ++k) part += v[k] == top ? 1.0f : 0.0f;
      }
      z += part;
    }
#pragma unroll
    for (int k = 0; k < PER; ++k) v[k] = next[k];
  }
  if (greedy) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float x = __shfl_xor_sync(0xffffffffu, top, o);
      const int i = __shfl_xor_sync(0xffffffffu, best, o);
      if (x > top || (x == top && i < best)) { top = x; best = i; }
    }
  } else {
    const float all = warp_max(top);
    z = top > -INFINITY ? z * rough_exp(a, top, all) : 0.0;
    top = all;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
  }
  if (lane == 0) { top_s[warp] = top; best_s[warp] = best; z_s[warp] = z; }
  __syncthreads();
  if (tid != 0) return;
  VerifyStat out{-INFINITY, 0x7fffffff, 0.0};
  for (int w = 0; w < kStatsThreads / 32; ++w)
    if (top_s[w] > out.top || (top_s[w] == out.top && best_s[w] < out.best)) { out.top = top_s[w]; out.best = best_s[w]; }
  for (int w = 0; w < kStatsThreads / 32; ++w)
    if (top_s[w] > -INFINITY) out.z += z_s[w] * rough_exp(a, top_s[w], out.top);
  a.stats[t * a.pieces + blockIdx.x] = out;
}

struct Verifier {
  const VerifyArgs& a;
  VerifyShared& s;
  const int tid, lane, warp, rank;
  int flip = 0;
  const float* row = nullptr;       // logits of the node reached
  const float* probs = nullptr;     // what its children were drawn from
  float floor = -FLT_MAX, top = 0.0f;
  PairPower power;
  double inv_e = 0.0;               // one over the row's sum of powers, where sums() has formed it
  int node_at = 0;

  __device__ Verifier(const VerifyArgs& a_, VerifyShared& s_) : a(a_), s(s_), tid(threadIdx.x), lane(threadIdx.x & 31), warp(threadIdx.x >> 5), rank((int)cluster_ctarank()) {}

  __device__ __forceinline__ uint32_t peer(const void* p, int r) const { return cluster_map(smem_addr(p), r); }
  __device__ __forceinline__ int begin(int r, int w) const { return min((long long)a.limit, (long long)(r * kVerifyWarps + w) * a.run); }

  __device__ void at_node(int seq_row, int node) {
    const size_t t = (size_t)seq_row + node;
    node_at = node;
    row = a.logits + t * a.ld;
    probs = a.probs ? a.probs + t * a.ldp : nullptr;
    floor = floor_of(a, t);
  }
  __device__ __forceinline__ bool kept(float l) const { return l >= floor; }

  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    each_logit<false>(row, nullptr, begin(rank, warp), begin(rank, warp + 1), lane, a.vec, [&](int i, float l, float) { f(i, l); });
  }

  // which nodes have children, and the first kernel's findings of those, a warp a node
  __device__ void find(int tok0, int count) {
    for (int node = warp; node < count; node += kVerifyWarps) {
      bool child = false;
      for (int j = node + 1 + lane; j < count; j += 32) child = child || s.parent[j] == node;
      const bool inner = __any_sync(0xffffffffu, child);
      if (lane == 0) s.inner[node] = inner ? 1 : 0;
      if (!inner || a.stats == nullptr) continue;
      VerifyStat mine{-INFINITY, 0x7fffffff, 0.0};
      for (int i = lane; i < a.pieces; i += 32) {
        const VerifyStat x = a.stats[(size_t)(tok0 + node) * a.pieces + i];
        const float top = fmaxf(mine.top, x.top);
        if (x.top > mine.top || (x.top == mine.top && x.best < mine.best)) mine.best = x.best;
        if (top > -INFINITY)
          mine.z = (mine.top > -INFINITY ? mine.z * rough_exp(a, mine.top, top) : 0.0) + (x.top > -INFINITY ? x.z * rough_exp(a, x.top, top) : 0.0);
        mine.top = top;
      }
      const float top = warp_max(mine.top);
      const double z = warp_sum_f64(mine.top > -INFINITY ? mine.z * rough_exp(a, mine.top, top) : 0.0);
      const int best = __reduce_min_sync(0xffffffffu, mine.top == top ? mine.best : 0x7fffffff);
      if (lane == 0) s.stat[node] = VerifyStat{top, top > -INFINITY ? best : 0, z};
    }
  }

  // first largest logit of the row (0 where there is none), the same in all blocks
  __device__ int argmax(bool have) {
    if (have) return s.stat[node_at].best;
    float bv = -INFINITY;
    int bi = 0x7fffffff;
    each([&](int i, float l) {
      if (l > bv || (l == bv && i < bi)) { bv = l; bi = i; }
    });
    auto better = [&](float v, int i) {
      if (v > bv || (v == bv && i < bi)) { bv = v; bi = i; }
    };
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) better(__shfl_xor_sync(0xffffffffu, bv, o), __shfl_xor_sync(0xffffffffu, bi, o));
    if (lane == 0) { s.red_m[warp] = bv; s.red_i[warp] = bi; }
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < kVerifyWarps; ++w) better(s.red_m[w], s.red_i[w]);
      s.x.max[flip] = bv;
      s.x.best[flip] = bi;
    }
    __syncthreads();
    cluster_sync_all();
    if (tid == 0) {
      bv = -INFINITY;
      bi = 0x7fffffff;
      for (int r = 0; r < a.team; ++r) better(peer_f32(peer(&s.x.max[flip], r)), __float_as_int(peer_f32(peer(&s.x.best[flip], r))));
      s.best = bv > -INFINITY ? bi : 0;
    }
    __syncthreads();
    flip ^= 1;
    return s.best;
  }

  __device__ __forceinline__ float rough(float l, float m) const { return rough_exp(a, l, m); }
  __device__ __forceinline__ void set_top(float m) {
    top = m;
    power = PairPower(a, m, floor);
  }

  // largest kept logit (into `top`) and, unless that is all, the sum Z of exp((l - top) / T)
  __device__ double denominator(bool top_alone) {
    float m = -INFINITY;
    each([&](int, float l) {
      if (kept(l)) m = fmaxf(m, l);
    });
    m = warp_max(m);
    double z = 0.0;
    float part = 0.0f;
    int n = 0;
    if (!top_alone)
      each([&](int, float l) {
        if (kept(l)) part += rough(l, m);
        if ((++n & 15) == 0) { z += part; part = 0.0f; }
      });
    z = warp_sum_f64(z + part);
    if (lane == 0) { s.red_m[warp] = m; s.red_z[warp] = z; }
    __syncthreads();
    if (warp == 0) {
      const float mw = lane < kVerifyWarps ? s.red_m[lane] : -INFINITY, mb = warp_max(mw);
      const double zw = lane < kVerifyWarps && mw > -INFINITY ? s.red_z[lane] * rough(mw, mb) : 0.0, zb = warp_sum_f64(zw);
      if (lane == 0) { s.x.max[flip] = mb; s.x.z[flip] = zb; }
    }
    __syncthreads();
    cluster_sync_all();
    if (warp == 0) {
      const float mr = lane < a.team ? peer_f32(peer(&s.x.max[flip], lane)) : -INFINITY, mc = warp_max(mr);
      const double zr = lane < a.team && mr > -INFINITY ? peer_f64(peer(&s.x.z[flip], lane)) * rough(mr, mc) : 0.0, zc = warp_sum_f64(zr);
      if (lane == 0) { s.top = mc; s.total_z = zc; }
    }
    __syncthreads();
    flip ^= 1;
    set_top(s.top);
    const double all = s.total_z;
    __syncthreads();
    return all;
  }

  __device__ __forceinline__ double fine(float l) const {      // the power in 64 bits
    const float2 x = power.of(l, s.table);
    return (double)x.x + (double)x.y;
  }

  // Sums over the runs, into s.runs up to and with each run; returns the last. Without `pair` of the powers, less those of the refused tokens of certain drafts; with it of
  // max(p - c q, 0), `cz` being c times the rough Z in the unit of the powers.
  __device__ double sums(bool pair, double c, float cz, int n_refused) {
    const int lo = begin(rank, warp), hi = begin(rank, warp + 1);
    PairSum all, over, drawn;
    if (!pair) {
      each_logit<false>(row, nullptr, lo, hi, lane, a.vec, [&](int, float l, float) {
        const float2 x = power.of(l, s.table);
        all.add(x.x, x.y);
      });
    } else {
      each_logit<true>(row, probs, lo, hi, lane, a.vec, [&](int, float l, float q) {
        const float2 x = power.of(l, s.table);
        all.add(x.x, x.y);
        const bool more = x.x > cz * q;
        over.add(more ? x.x : 0.0f, more ? x.y : 0.0f);
        drawn.add(more ? q : 0.0f, 0.0f);
      });
    }
    double w = warp_sum_f64(all.value());
    const double wo = pair ? warp_sum_f64(over.value()) : 0.0, wq = pair ? warp_sum_f64(drawn.value()) : 0.0;
    for (int r = 0; r < n_refused; ++r) {
      const int x = s.refused[r];
      if (x >= lo && x < hi) w -= fine(row[x]);
    }
    if (lane == 0) {
      s.x.sum[flip][0][warp] = fmax(w, 0.0);
      s.x.sum[flip][1][warp] = wo;
      s.x.sum[flip][2][warp] = wq;
    }
    __syncthreads();
    cluster_sync_all();
    // a thread a run
    static_assert(kVerifyRuns <= kVerifyThreads && kVerifyWarps == 32, "a thread a run, a warp a block's runs");
    const int runs = a.team * kVerifyWarps;
    double own = 0.0, own_over = 0.0, own_drawn = 0.0, inv = 0.0;
    if (warp < a.team) {
      own = peer_f64(peer(&s.x.sum[flip][0][lane], warp));
      if (pair) {
        own_over = peer_f64(peer(&s.x.sum[flip][1][lane], warp));
        own_drawn = peer_f64(peer(&s.x.sum[flip][2][lane], warp));
        const double e = warp_sum_f64(own);
        if (lane == 0) s.red_z[warp] = e;
      }
    }
    if (pair) {
      __syncthreads();
      if (warp == 0) {
        const double e = warp_sum_f64(lane < a.team ? s.red_z[lane] : 0.0);
        if (lane == 0) s.total_z = e > 0.0 ? 1.0 / e : 0.0;
      }
      __syncthreads();
      inv = s.total_z;
      own = fmax(own_over * inv - c * own_drawn, 0.0);
    }
    if (warp < a.team) {
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, own, d);
        if (lane >= d) own += y;
      }
      if (lane == 31) s.scan[warp] = own;
    }
    __syncthreads();
    if (warp < a.team) {
      double off = 0.0;
      for (int w = 0; w < warp; ++w) off += s.scan[w];
      s.runs[tid] = off + own;
    }
    __syncthreads();
    flip ^= 1;
    if (pair) inv_e = inv;
    return s.runs[runs - 1];
  }

  // s.p of a node's children from the exact sum of its row, which a refusal of drafts with distributions (`formed`) has left
  __device__ void exact_children(int node, int count, bool formed) {
    if (!formed) {
      const double all = sums(false, 0.0, 0.0f, 0);
      inv_e = all > 0.0 ? 1.0 / all : 0.0;
    }
    __syncthreads();      // (others may still be reading)
    if (tid > node && tid < count && s.parent[tid] == node) s.p[tid] = s.token[tid] < 0 ? 0.0 : fine(s.logit[tid]) * inv_e;
    __syncthreads();
  }

  // the token where the running sum passes `target`; in the block that has its run, else -1
  __device__ int draw(double target, bool pair, double c, int n_refused) {
    const int runs = a.team * kVerifyWarps;
    int first = kVerifyRuns, last = -1;      // the first run whose sum passes it, else the last that adds something
    for (int i0 = runs - 32; i0 >= 0; i0 -= 32) {
      const int i = i0 + lane;
      const bool adds = s.runs[i] > (i ? s.runs[i - 1] : 0.0);
      const uint32_t hits = __ballot_sync(0xffffffffu, adds && s.runs[i] > target), any = __ballot_sync(0xffffffffu, adds);
      if (hits) first = i0 + __ffs(hits) - 1;
      if (any && last < 0) last = i0 + 31 - __clz(any);
    }
    const int g = first < kVerifyRuns ? first : max(last, 0);
    double at = g ? s.runs[g - 1] : 0.0;
    if (g / kVerifyWarps != rank) return -1;
    if (tid == 0) { s.found = 0x7fffffff; s.last = -1; }
    __syncthreads();
    const int lo = begin(rank, g % kVerifyWarps), hi = begin(rank, g % kVerifyWarps + 1);
    auto weight = [&](int i) {
      const double e = fine(row[i]);
      if (pair) return fmax(e * inv_e - c * (double)probs[i], 0.0);
      for (int r = 0; r < n_refused; ++r)
        if (s.refused[r] == i) return 0.0;
      return e;
    };
    const int per = (hi - lo + kVerifyThreads - 1) / kVerifyThreads, i0 = lo + tid * per, i1 = min(hi, i0 + per);
    double mine = 0.0;
    for (int i = i0; i < i1; ++i) mine += weight(i);
    double incl = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += y;
    }
    if (lane == 31) s.scan[warp] = incl;
    __syncthreads();
    for (int w = 0; w < warp; ++w) at += s.scan[w];
    at += incl - mine;
    if (mine > 0.0) {
      for (int i = i0; i < i1; ++i) {
        const double w = weight(i);
        at += w;
        if (w > 0.0) {
          atomicMax(&s.last, i);
          if (at > target) { atomicMin(&s.found, i); break; }
        }
      }
    }
    __syncthreads();
    return s.found != 0x7fffffff ? s.found : s.last < 0 ? 0 : s.last;
  }
};

__global__ void __launch_bounds__(kVerifyThreads) verify_kernel(VerifyArgs a) {
  pdl_enter();
  __shared__ VerifyShared s;
  Verifier v(a, s);
  const int tid = threadIdx.x, seq = blockIdx.x / a.team;
  const int tok0 = a.seq_start[seq];
  int count = min(max(a.counts[seq], 0), a.max_count);
  if (tok0 < 0 || (long long)tok0 + count > a.rows) count = 0;      // (never read behind the given rows)
  const bool writer = v.rank == 0 && tid == 0;
  if (count == 0) {      // the whole cluster
    if (v.rank == 0)
      for (int i = tid; i < a.path_width; i += kVerifyThreads) a.path[(size_t)seq * a.path_width + i] = -1;
    if (writer) { a.lengths[seq] = 0; a.chosen[seq] = -1; }
    return;
  }
  const bool greedy = a.scale == 0.0;
  if (tid < 64) {
    const double x = exp2(tid * 0.015625);
    s.table[tid] = make_float2((float)x, (float)(x - (double)(float)x));
  }
  if (tid < count) {
    const int p = a.parents[tok0 + tid], x = a.tokens[tok0 + tid];
    const bool child = p >= 0 && p < tid, inside = x >= 0 && x < a.limit;
    s.parent[tid] = child ? p : -1;
    s.token[tid] = inside ? x : -1;
    s.u[tid] = a.uniforms ? a.uniforms[tok0 + tid] : 0.0f;
    s.logit[tid] = child && inside ? a.logits[(size_t)(tok0 + p) * a.ld + x] : -INFINITY;
    s.prob[tid] = a.probs == nullptr ? 1.0f : child && inside ? a.probs[(size_t)(tok0 + p) * a.ldp + x] : 0.0f;
  }
  if (v.rank == 0)
    for (int i = tid; i < a.path_width; i += kVerifyThreads)
      if (i > 0) a.path[(size_t)seq * a.path_width + i] = -1;
  __syncthreads();
  v.find(tok0, count);
  __syncthreads();
  // the children's probabilities at their parents, where the first kernel has been over those
  auto child_p = [&](int j, const PairPower& power, float top, double z) {
    if (s.token[j] < 0 || !(z > 0.0)) return 0.0;
    const float2 x = power.of(s.logit[j], s.table), one = power.of(top, s.table);
    return ((double)x.x + (double)x.y) / (((double)one.x + (double)one.y) * z);
  };
  if (a.stats && !greedy && tid < count && s.parent[tid] >= 0) {
    const VerifyStat& x = s.stat[s.parent[tid]];
    s.p[tid] = child_p(tid, PairPower(a, x.top, floor_of(a, (size_t)tok0 + s.parent[tid])), x.top, x.z);
  }
  __syncthreads();
  int node = 0, length = 1, n_refused = 0, best = 0;
  double c = 0.0, total = -1.0;      // c: of what s.runs holds the sums; total < 0: not formed yet
  bool pair = false;
  while (true) {
    v.at_node(tok0, node);
    int taken = -1;
    n_refused = 0;
    c = 0.0;
    total = -1.0;
    pair = false;
    const bool inner = s.inner[node] != 0, have = inner && a.stats != nullptr;
    if (greedy) {
      best = v.argmax(have);
      for (int j = node + 1; j < count && taken < 0; ++j)
        if (s.parent[j] == node && s.token[j] == best) taken = j;
    } else {
      double z = have ? s.stat[node].z : 0.0;
      bool set = false;      // v's powers are the node's
      if (!have) {
        z = v.denominator(!inner);
        set = true;
        if (inner) {
          if (tid > node && tid < count && s.parent[tid] == node) s.p[tid] = child_p(tid, v.power, v.top, z);
          __syncthreads();
        }
      }
      double f = 1.0, gone = 0.0;
      bool exact = false;      // s.p of this node's children are
      for (int j = inner ? node + 1 : count; j < count; ++j) {
        if (s.parent[j] != node) continue;
        const double u = s.u[j];
        bool again = false;      // a certain draft that was refused before has no probability left
        for (int r = 0; r < n_refused; ++r) again = again || s.refused[r] == s.token[j];
        if (!again) {
          double p = s.p[j], border = a.probs ? (c + u * f) * (double)s.prob[j] : u * (1.0 - gone);
          if (!exact && p > 0.0 && fabs(p - border) <= kVerifyDoubt * (p + u * gone)) {      // the rough Z does not tell
            exact = true;
            if (!set) v.set_top(s.stat[node].top);
            set = true;
            v.exact_children(node, count, pair);
            gone = 0.0;
            for (int i = node + 1; i < j; ++i) {      // what was refused, every token once
              if (a.probs || s.parent[i] != node || s.token[i] < 0) continue;
              bool twice = false;
              for (int k = node + 1; k < i; ++k) twice = twice || (s.parent[k] == node && s.token[k] == s.token[i]);
              if (!twice) gone += s.p[i];
            }
            p = s.p[j];
            border = a.probs ? (c + u * f) * (double)s.prob[j] : u * (1.0 - gone);
          }
          if (p > border) {
            taken = j;
            break;
          }
        }
        if (a.probs) {
          if (!(z > 0.0)) continue;      // a row without probabilities: nothing to refuse
          c += f;
          if (!set) v.set_top(s.stat[node].top);
          set = pair = true;
          f = total = v.sums(true, c, (float)(c * z * v.fine(v.top)), 0);
        } else if (s.token[j] >= 0 && !again) {
          __syncthreads();
          if (tid == 0) s.refused[n_refused] = s.token[j];
          ++n_refused;
          gone += s.p[j];
          __syncthreads();
        }
      }
    }
    if (taken < 0) {
      if (!greedy && have && !pair) v.set_top(s.stat[node].top);
      break;
    }
    node = taken;
    if (writer && length < a.path_width) a.path[(size_t)seq * a.path_width + length] = node;
    ++length;
    __syncthreads();      // (s.p is written anew)
  }
  if (!greedy) {
    if (total < 0.0) total = v.sums(false, 0.0, 0.0f, n_refused);
    if (!(total > 0.0)) {      // refusals that had no probability have left nothing: all of p again
      pair = false;
      n_refused = 0;
      total = v.sums(false, 0.0, 0.0f, 0);
    }
    const int x = v.draw((double)s.u[0] * total, pair, c, n_refused);
    if (x >= 0 && tid == 0) a.chosen[seq] = x;
  }
  if (writer) {
    a.path[(size_t)seq * a.path_width] = 0;
    a.lengths[seq] = length;
    if (greedy) a.chosen[seq] = best;
  }
  __syncthreads();
  cluster_sync_all();      // the others may still be reading this block's sums
}

// Pieces of a row in the first kernel: small ones where the rows are few, else as many blocks as run at once three times over, of which those of nodes without
// children leave at once (a batch of 64: 73 to 77 us with 740 to 4,736 blocks, 83 with 500, 79 with 7,000; eight trees 36 to 37, 41, 42).
static int stats_steps(long long rows, int limit) {
  const long long steps = ((long long)limit + kStatsStep - 1) / kStatsStep, pieces = 2368 / rows + 1;
  return (int)(pieces >= steps ? 1 : (steps + pieces - 1) / pieces);
}
static int stats_pieces(long long rows, int limit) {
  const long long piece = (long long)stats_steps(rows, limit) * kStatsStep;
  return (int)((limit + piece - 1) / piece);
}
static bool stats_first(long long rows, int limit) { return rows * limit * 4 <= kMostStatsBytes; }
// 32-bit words of scratch that slb_verify_drafts takes.
extern "C" long long slb_verify_drafts_scratch(int n_seqs, long long rows, int limit, int drawn) {
  return n_seqs > 0 && n_seqs < 65536 && rows > 0 && limit > 0 && stats_first(rows, limit) ? rows * stats_pieces(rows, limit) * (long long)(sizeof(VerifyStat) / 4) : 0;
}

// How many clusters of sixteen blocks, an SM each, run at once on the current device: such clusters are to be allowed, and lie within one of the GPU's partitions.
static int wide_clusters() {
  static std::atomic<int> known[64];      // one more than the number; 0: not asked yet
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  int n = known[dev].load(std::memory_order_acquire);
  if (n > 0) return n - 1;
  int clusters = 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kVerifyTeam);
  cfg.blockDim = dim3(kVerifyThreads);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kVerifyTeam;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (allow_wide_clusters((const void*)verify_kernel) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&clusters, verify_kernel, &cfg) != cudaSuccess) {
    cudaGetLastError();
    clusters = 0;
  }
  known[dev].store(clusters + 1, std::memory_order_release);
  return clusters;
}

extern "C" int slb_verify_drafts(const VerifyCall* call) {
  SLB_REQUIRE(call != nullptr, "verify_drafts: no call");
  const VerifyCall c = *call;
  SLB_REQUIRE(c.n_seqs >= 0 && c.n_seqs < (1 << 24) && c.rows >= 0, "verify_drafts: n_seqs=%d rows=%lld", c.n_seqs, c.rows);
  SLB_REQUIRE(c.limit > 0 && c.ld >= c.limit && (c.probs == nullptr || c.ldp >= c.limit), "verify_drafts: %d tokens in rows of %lld and %lld", c.limit, c.ld, c.ldp);
  SLB_REQUIRE(c.max_count > 0 && c.max_count <= kMostNodes, "verify_drafts: %d nodes of a sequence; 1 to %d are taken", c.max_count, kMostNodes);
  SLB_REQUIRE(c.path_width >= c.max_count, "verify_drafts: paths of %d places do not hold %d nodes", c.path_width, c.max_count);
  SLB_REQUIRE(c.temperature < INFINITY, "verify_drafts: the temperature must be finite");
  SLB_REQUIRE(!(c.temperature > 0.0) || c.uniforms != nullptr || c.rows == 0, "verify_drafts: a temperature needs the random numbers");
  if (c.n_seqs == 0) return 0;
  VerifyArgs a{};
  a.logits = c.logits; a.probs = c.probs; a.floors = c.floors; a.uniforms = c.uniforms; a.tokens = c.tokens; a.parents = c.parents; a.seq_start = c.seq_start;
  a.counts = c.counts; a.path = c.path; a.lengths = c.lengths; a.chosen = c.chosen; a.rows = c.rows; a.ld = c.ld; a.ldp = c.ldp;
  a.limit = c.limit; a.max_count = c.max_count; a.path_width = c.path_width;
  if (c.temperature > 0.0) {
    a.scale = fmin(1.4426950408889634 / c.temperature, 1e30);      // (colder than that only the largest logit is left either way)
    a.unscale = 1.0 / a.scale;
    a.scale_hi = (float)a.scale;
    a.scale_lo = (float)(a.scale - (double)a.scale_hi);
    a.least = (float)fmax(-200.0 * a.unscale, -(double)FLT_MAX);
  }
  const long long need = slb_verify_drafts_scratch(c.n_seqs, c.rows, c.limit, c.probs != nullptr);
  SLB_REQUIRE(need == 0 || (c.scratch != nullptr && c.scratch_words >= need), "verify_drafts: the call needs %lld words of scratch, %lld were given", need,
              c.scratch ? c.scratch_words : 0ll);
  SLB_REQUIRE((uintptr_t)c.scratch % 16 == 0, "verify_drafts: scratch must be 16-byte aligned");
  a.team = kVerifyTeam;      // as many as give every block an SM of its own (one sequence: sixteen blocks 21 us, eight 26)
  while (a.team > 1 && (long long)c.n_seqs * a.team > sm_count()) a.team /= 2;
  if (a.team > 8 && c.n_seqs > wide_clusters()) a.team = 8;
  if (a.team == 8 && c.n_seqs > 16) a.team = 4;      // (a cluster lies within one of the GPU's partitions: eighteen of eight may not run at once)
  const int runs = a.team * kVerifyWarps;
  a.run = (int)((((long long)c.limit + runs - 1) / runs + 3) / 4 * 4);
  a.vec = (uintptr_t)c.logits % 16 == 0 && c.ld % 4 == 0 && (c.probs == nullptr || ((uintptr_t)c.probs % 16 == 0 && c.ldp % 4 == 0));
  if (need > 0) {
    a.steps = stats_steps(c.rows, c.limit);
    a.pieces = stats_pieces(c.rows, c.limit);
  }
  if (need > 0) {
    a.stats = reinterpret_cast<VerifyStat*>(c.scratch);
    // (begins early, call after call: one chat 21.9 us, 23.2 otherwise: a launch is on its way while the kernel before ends)
    launch_prefetching(verify_stats_kernel, dim3(a.pieces, c.n_seqs, c.max_count), dim3(kStatsThreads), 0, (cudaStream_t)c.stream, a);
    const int rc = check_launch("verify_drafts (sums)");
    if (rc) return rc;
  }
  launch_clusters(need > 0 ? pdl_mode() != 0 : pdl_mode() == 1, a.team, verify_kernel, dim3(c.n_seqs * a.team), dim3(kVerifyThreads), 0, (cudaStream_t)c.stream, a);
  return check_launch("verify_drafts");
}

}  // namespace slb
