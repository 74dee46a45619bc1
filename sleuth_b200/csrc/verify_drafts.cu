// Which drafted tokens the target's probabilities accept, and the token behind the last of them.
//
// Every sequence brings a tree: node 0 is its newest certain token, row t of `logits` what the target says behind node t. With l the logits of the node
// reached, p(i) = exp(l_i / T) / Z over i < limit with l_i >= floor, q the distribution that its children were drawn from, independently, the children x are tried in their order: x is
// accepted with probability min(1, p(x) / q(x)); after a refusal p becomes max(p - q, 0) over its sum. Refusals in a row stay in one family:
//   p after k refusals = max(p - c_k q, 0) / F_k,   F_k = sum max(p - c_k q, 0),   c_0 = 0, F_0 = 1, c_{k+1} = c_k + F_k,
// because max(max(p - c q, 0) / F - q, 0) = max(p - (c + F) q, 0) / F. So child x with the number u goes through iff p(x) > (c + u F) q(x), and a refusal costs one
// sum over the row. Certain drafts are point masses: p(x) > u (1 - R), R the probability of the distinct tokens refused before. Where no child is left the next token is
// drawn from what p has become: the first token, in the order of their numbers, where the running sum passes u of the whole. Temperature 0: the child that is
// the row's first largest logit, and in the end that token.
//
// A cluster of eight blocks walks a sequence's way, an eighth of a row each, a run of it a warp, so that only rows on the way are read. Results are whole numbers and have to be
// the definition's: what decides about a child (Z, p) comes from 32-bit powers summed in 64 bits, off by some 1e-8, which is the chance that a random number falls
// between; but a draw compares one number with 150,000 running sums, so sums for draws and refusals are of 64-bit powers of two (a table of 32 and five
// terms of the series, off by 3e-15).
#include <float.h>
#include <math.h>

#include "tcgen05.cuh"      // clusters
#include "tree.cuh"

namespace slb {

constexpr int kVerifyTeam = 8, kVerifyThreads = 512, kVerifyWarps = kVerifyThreads / 32, kVerifyRuns = kVerifyTeam * kVerifyWarps;

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
  double scale;               // log2 e / T; 0: the largest logit alone counts
  float scale_hi, scale_lo;
  int limit, max_count, path_width, run, vec;      // run: tokens of a warp, a multiple of 4
};

struct VerifyExchange {
  double sum[2][kVerifyWarps];      // two copies, used in turn: a block may write its next share while a slower one still reads the last
  double z[2];
  float max[2];
  int best[2];
};

struct VerifyShared {
  VerifyExchange x;
  double table[32];                 // 2^(j / 32)
  double runs[kVerifyRuns];         // sums before and with each run
  double red_z[kVerifyWarps];
  double scan[kVerifyWarps];
  float red_m[kVerifyWarps];
  int red_i[kVerifyWarps];
  int parent[kMostNodes], token[kMostNodes], refused[kMostNodes];
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

// 2^y for y <= 0: y = n + j / 32 + r with |r| <= 1 / 64, and 2^r from the series of exp(r ln 2), whose sixth power is below 3e-15.
__device__ __forceinline__ double pow2_f64(double y, const double* table) {
  if (!(y > -1000.0)) return y == y ? 0.0 : y;
  const double t = y * 32.0 + 6755399441055744.0;      // 1.5 * 2^52: the nearest whole number in the low bits
  const int k = __double2loint(t);
  const double x = (y - (t - 6755399441055744.0) * 0.03125) * 0.6931471805599453;
  double p = fma(x, 1.0 / 120.0, 1.0 / 24.0);
  p = fma(x, p, 1.0 / 6.0);
  p = fma(x, p, 0.5);
  p = fma(x, p, 1.0);
  p = fma(x, p, 1.0);
  p *= table[k & 31];
  return __hiloint2double(__double2hiint(p) + ((k >> 5) << 20), __double2loint(p));      // (p is in [0.98, 2), k >> 5 >= -1000: no underflow)
}

struct Verifier {
  const VerifyArgs& a;
  VerifyShared& s;
  const int tid, lane, warp, rank;
  int flip = 0;
  const float* row = nullptr;       // logits of the node reached
  const float* probs = nullptr;     // what its children were drawn from
  float floor = -FLT_MAX, top = 0.0f;

  __device__ Verifier(const VerifyArgs& a_, VerifyShared& s_) : a(a_), s(s_), tid(threadIdx.x), lane(threadIdx.x & 31), warp(threadIdx.x >> 5), rank((int)cluster_ctarank()) {}

  __device__ __forceinline__ uint32_t peer(const void* p, int r) const { return cluster_map(smem_addr(p), r); }
  __device__ __forceinline__ int begin(int r, int w) const { return min((long long)a.limit, (long long)(r * kVerifyWarps + w) * a.run); }

  __device__ void at_node(int seq_row, int node) {
    const size_t t = (size_t)seq_row + node;
    row = a.logits + t * a.ld;
    probs = a.probs ? a.probs + t * a.ldp : nullptr;
    floor = -FLT_MAX;             // -inf has no probability, nor has NaN
    if (a.floors) {
      const float f = a.floors[t];
      floor = f != f ? f : fmaxf(f, -FLT_MAX);
    }
  }
  __device__ __forceinline__ bool kept(float l) const { return l >= floor; }

  // f(token, logit) for this warp's run, four tokens of a lane at a time where rows are aligned
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    const int lo = begin(rank, warp), hi = begin(rank, warp + 1);
    if (a.vec) {
      int i = lo + 4 * lane;
      for (; i + 3 * 128 + 3 < hi; i += 4 * 128) {
        float4 v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = *reinterpret_cast<const float4*>(row + i + 128 * k);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          f(i + 128 * k, v[k].x);
          f(i + 128 * k + 1, v[k].y);
          f(i + 128 * k + 2, v[k].z);
          f(i + 128 * k + 3, v[k].w);
        }
      }
      for (; i < hi; i += 128)
        for (int k = 0; k < 4; ++k)
          if (i + k < hi) f(i + k, row[i + k]);
    } else {
      int i = lo + lane;
      for (; i + 3 * 32 < hi; i += 4 * 32) {
        float v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = row[i + 32 * k];
#pragma unroll
        for (int k = 0; k < 4; ++k) f(i + 32 * k, v[k]);
      }
      for (; i < hi; i += 32) f(i, row[i]);
    }
  }

  // first largest logit of the row (0 where there is none), the same in all blocks
  __device__ int argmax() {
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
      for (int r = 0; r < kVerifyTeam; ++r) better(peer_f32(peer(&s.x.max[flip], r)), __float_as_int(peer_f32(peer(&s.x.best[flip], r))));
      s.best = bi == 0x7fffffff ? 0 : bi;
    }
    __syncthreads();
    flip ^= 1;
    return s.best;
  }

  __device__ __forceinline__ float rough(float l, float m) const {      // exp((l - m) / T), l <= m
    const float x = l - m, t = x * a.scale_hi;
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(fmaf(x, a.scale_hi, x * a.scale_lo)));
    return l == m ? 1.0f : t > -1e4f ? y : 0.0f;      // (infinities end here)
  }

  // largest kept logit (into `top`) and the sum Z of exp((l - top) / T)
  __device__ double denominator() {
    float m = -INFINITY;
    each([&](int, float l) {
      if (kept(l)) m = fmaxf(m, l);
    });
    m = warp_max(m);
    double z = 0.0;
    float part = 0.0f;
    int n = 0;
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
      const float mr = lane < kVerifyTeam ? peer_f32(peer(&s.x.max[flip], lane)) : -INFINITY, mc = warp_max(mr);
      const double zr = lane < kVerifyTeam && mr > -INFINITY ? peer_f64(peer(&s.x.z[flip], lane)) * rough(mr, mc) : 0.0, zc = warp_sum_f64(zr);
      if (lane == 0) { s.top = mc; s.total_z = zc; }
    }
    __syncthreads();
    flip ^= 1;
    top = s.top;
    return s.total_z;
  }

  __device__ __forceinline__ double fine(float l) const {      // exp((l - top) / T) in 64 bits
    return !kept(l) ? 0.0 : l == top ? 1.0 : pow2_f64(((double)l - (double)top) * a.scale, s.table);
  }
  __device__ __forceinline__ double rest(double e, double inv_z, double c, int i) const { return fmax(fma(e, inv_z, -c * (double)probs[i]), 0.0); }

  // sums over the runs: of exp (inv_z 0) or of max(exp * inv_z - c q, 0), without the refused tokens of certain drafts; s.runs: sums up to and with each run
  __device__ double sums(double inv_z, double c, int n_refused) {
    double w = 0.0;
    if (inv_z == 0.0) each([&](int, float l) { w += fine(l); });
    else each([&](int i, float l) { w += rest(fine(l), inv_z, c, i); });
    w = warp_sum_f64(w);
    const int lo = begin(rank, warp), hi = begin(rank, warp + 1);
    for (int r = 0; r < n_refused; ++r) {
      const int x = s.refused[r];
      if (x >= lo && x < hi) w -= fine(row[x]);
    }
    if (lane == 0) s.x.sum[flip][warp] = fmax(w, 0.0);
    __syncthreads();
    cluster_sync_all();
    if (warp == 0) {
      double v[4], before = 0.0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int g = lane * 4 + k;
        v[k] = peer_f64(peer(&s.x.sum[flip][g % kVerifyWarps], g / kVerifyWarps));
        before += v[k];
        v[k] = before;
      }
      double incl = before;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += y;
      }
      const double off = __shfl_up_sync(0xffffffffu, incl, 1);
#pragma unroll
      for (int k = 0; k < 4; ++k) s.runs[lane * 4 + k] = (lane ? off : 0.0) + v[k];
    }
    __syncthreads();
    flip ^= 1;
    return s.runs[kVerifyRuns - 1];
  }

  // the token where the running sum passes `target`; in the block that has its run, else -1
  __device__ int draw(double target, double inv_z, double c, int n_refused) {
    int first = kVerifyRuns, last = -1;      // the first run whose sum passes it, else the last that adds something
#pragma unroll
    for (int k = kVerifyRuns / 32 - 1; k >= 0; --k) {
      const int i = 32 * k + lane;
      const bool adds = s.runs[i] > (i ? s.runs[i - 1] : 0.0);
      const uint32_t hits = __ballot_sync(0xffffffffu, adds && s.runs[i] > target), any = __ballot_sync(0xffffffffu, adds);
      if (hits) first = 32 * k + __ffs(hits) - 1;
      if (any && last < 0) last = 32 * k + 31 - __clz(any);
    }
    const int g = first < kVerifyRuns ? first : max(last, 0);
    double at = g ? s.runs[g - 1] : 0.0;
    if (g / kVerifyWarps != rank) return -1;
    if (tid == 0) { s.found = 0x7fffffff; s.last = -1; }
    __syncthreads();
    const int lo = begin(rank, g % kVerifyWarps), hi = begin(rank, g % kVerifyWarps + 1);
    auto weight = [&](int i) {
      const double e = fine(row[i]);
      if (inv_z != 0.0) return rest(e, inv_z, c, i);
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
  const int tid = threadIdx.x, seq = blockIdx.x / kVerifyTeam;
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
  if (tid < 32) s.table[tid] = exp2(tid * 0.03125);
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
  int node = 0, length = 1, n_refused = 0, best = 0;
  double inv_z = 0.0, c = 0.0, total = -1.0;      // inv_z, c: of what s.runs holds the sums; total < 0: not formed yet
  while (true) {
    v.at_node(tok0, node);
    int taken = -1;
    n_refused = 0;
    inv_z = c = 0.0;
    total = -1.0;
    if (greedy) {
      best = v.argmax();
      for (int j = node + 1; j < count && taken < 0; ++j)
        if (s.parent[j] == node && s.token[j] == best) taken = j;
    } else {
      const double z = v.denominator();
      double f = 1.0, gone = 0.0;
      for (int j = node + 1; j < count; ++j) {
        if (s.parent[j] != node) continue;
        const double p = s.token[j] >= 0 && z > 0.0 ? v.fine(s.logit[j]) / z : 0.0, u = s.u[j];
        if (a.probs ? p > (c + u * f) * (double)s.prob[j] : p > u * (1.0 - gone)) {
          bool again = false;      // a certain draft that was refused before has no probability left
          for (int r = 0; r < n_refused; ++r) again = again || s.refused[r] == s.token[j];
          if (!again) {
            taken = j;
            break;
          }
        }
        if (a.probs) {
          if (inv_z == 0.0) {
            const double fine_z = v.sums(0.0, 0.0, 0);
            if (!(fine_z > 0.0)) break;      // a row without probabilities: nothing to refuse
            inv_z = 1.0 / fine_z;
          }
          c += f;
          f = total = v.sums(inv_z, c, 0);
        } else if (s.token[j] >= 0) {
          bool again = false;
          for (int r = 0; r < n_refused; ++r) again = again || s.refused[r] == s.token[j];
          if (!again) {
            __syncthreads();
            if (tid == 0) s.refused[n_refused] = s.token[j];
            ++n_refused;
            gone += p;
            __syncthreads();
          }
        }
      }
    }
    if (taken < 0) break;
    node = taken;
    if (writer && length < a.path_width) a.path[(size_t)seq * a.path_width + length] = node;
    ++length;
  }
  if (!greedy) {
    if (total < 0.0) {
      inv_z = 0.0;
      total = v.sums(0.0, 0.0, n_refused);
    }
    if (!(total > 0.0)) {      // refusals that had no probability have left nothing: all of p again
      inv_z = 0.0;
      n_refused = 0;
      total = v.sums(0.0, 0.0, 0);
    }
    const int x = v.draw((double)s.u[0] * total, inv_z, c, n_refused);
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

// 32-bit words of scratch that slb_verify_drafts takes.
extern "C" long long slb_verify_drafts_scratch(int n_seqs, long long rows, int limit, int drawn) { return 0; }

extern "C" int slb_verify_drafts(const VerifyCall* call) {
  SLB_REQUIRE(call != nullptr, "verify_drafts: no call");
  const VerifyCall c = *call;
  SLB_REQUIRE(c.n_seqs >= 0 && c.n_seqs < (1 << 24) && c.rows >= 0, "verify_drafts: n_seqs=%d rows=%lld", c.n_seqs, c.rows);
  SLB_REQUIRE(c.limit > 0 && c.ld >= c.limit && (c.probs == nullptr || c.ldp >= c.limit), "verify_drafts: %d tokens in rows of %lld and %lld", c.limit, c.ld, c.ldp);
  SLB_REQUIRE(c.max_count > 0 && c.max_count <= kMostNodes, "verify_drafts: %d nodes of a sequence; 1 to %d are taken", c.max_count, kMostNodes);
  SLB_REQUIRE(c.path_width >= c.max_count, "verify_drafts: paths of %d places do not hold %d nodes", c.path_width, c.max_count);
  SLB_REQUIRE(c.temperature < INFINITY, "verify_drafts: the temperature must be finite");
  SLB_REQUIRE(!(c.temperature > 0.0) || c.uniforms != nullptr, "verify_drafts: a temperature needs the random numbers");
  if (c.n_seqs == 0) return 0;
  VerifyArgs a{};
  a.logits = c.logits; a.probs = c.probs; a.floors = c.floors; a.uniforms = c.uniforms; a.tokens = c.tokens; a.parents = c.parents; a.seq_start = c.seq_start;
  a.counts = c.counts; a.path = c.path; a.lengths = c.lengths; a.chosen = c.chosen; a.rows = c.rows; a.ld = c.ld; a.ldp = c.ldp;
  a.limit = c.limit; a.max_count = c.max_count; a.path_width = c.path_width;
  if (c.temperature > 0.0) {
    a.scale = 1.4426950408889634 / c.temperature;
    a.scale_hi = a.scale < 1e30 ? (float)a.scale : 1e30f;      // (colder than that only the largest logit is left either way)
    a.scale_lo = a.scale < 1e30 ? (float)(a.scale - (double)a.scale_hi) : 0.0f;
  }
  a.run = (int)((((long long)c.limit + kVerifyRuns - 1) / kVerifyRuns + 3) / 4 * 4);
  a.vec = (uintptr_t)c.logits % 16 == 0 && c.ld % 4 == 0;
  launch_clusters(pdl_mode() == 1, kVerifyTeam, verify_kernel, dim3(c.n_seqs * kVerifyTeam), dim3(kVerifyThreads), 0, (cudaStream_t)c.stream, a);
  return check_launch("verify_drafts");
}

}  // namespace slb
