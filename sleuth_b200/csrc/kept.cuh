// What the kernels of a cache of bounded size share: which rows of the cache a query sees, and the arguments of a step.
//
// Rows of a sequence are counted from 0 in the order of its block table (64 rows a page). A step appends counts[s] rows behind the
// past[s] rows that are there; the query of row p sees row j if j <= p and (window == 0, or j > p - window, or j < first): the latest
// `window` rows, its own included, and the first `first` ones.
#pragma once

#include "common.cuh"

namespace slb {

constexpr float kKeptLog2e = 1.4426950408889634f;

struct KeptArgs {
  const void* q;            // [tokens, H, hd]
  const void* k_pool;       // [pages, K, 64, hd]
  const void* v_pool;
  void* out;                // [tokens, H * hd]
  const int* seq_start;     // [n] first token row of each sequence
  const int* past;          // [n] rows before the step
  const int* counts;        // [n] new rows
  const int* block_table;   // [n, table_stride]
  int table_stride, n_seqs, heads, kv_heads, head_dim, window, first;
  float scale;
  float* lse;               // [tokens, H] log of the softmax denominator, or null
  float* scratch;
  int splits;
  const int* slots;         // [n] the row of `weights` of each sequence, or null: its own number
  const float* weights;     // [slots, K, capacity] what the rows have gathered before
  float* weights_out;
  long long capacity;
};

// What a caller of slb_attention_kept says, in one piece of memory (thirty arguments cost a call through ctypes 4 us, one 1).
struct KeptCall {
  const void *q, *k_pool, *v_pool;      // [tokens, heads, head_dim]; [pool_pages, kv_heads, 64, head_dim]
  void* out;                            // [tokens, heads * head_dim]
  const int *seq_start, *past, *counts, *block_table;
  float* lse;                           // [tokens, heads] or null
  const int* slots;                     // [n_seqs] or null
  const float* weights;                 // [slots, kv_heads, capacity]; with its target (the same memory or apart), or both null
  float *weights_out, *scratch;
  int* status;                          // a zeroed device word that receives a code if a bounded wait inside a kernel gave up
  void* stream;
  long long tokens, capacity, scratch_floats, pool_pages;
  int table_stride, n_seqs, max_count, max_keys, heads, kv_heads, head_dim, window, first, dtype;
  float scale;
};
static_assert(sizeof(KeptCall) == 15 * 8 + 4 * 8 + 11 * 4 + 4, "as packed in kernels/ops.py");

// First row of the window of the query at row p.
__host__ __device__ __forceinline__ int window_lo(int p, int window) { return window > 0 && p - window + 1 > 0 ? p - window + 1 : 0; }

__device__ __forceinline__ bool sees(int key, int pos, int lo, int first) { return key <= pos && (key >= lo || key < first); }

// A sequence that brings no token keeps what its rows have gathered: where the target lies apart, rows lo .. hi - 1 of it go over. `t` of `threads` threads.
__device__ __forceinline__ void carry_weights(const KeptArgs& a, int seq, int kh, long long lo, long long hi, int t, int threads) {
  if (a.weights == nullptr || a.weights_out == a.weights) return;
  const size_t at0 = ((size_t)(a.slots ? a.slots[seq] : seq) * a.kv_heads + kh) * a.capacity;
  hi = min(hi, min((long long)a.past[seq], a.capacity));
  for (long long key = lo + t; key < hi; key += threads) a.weights_out[at0 + key] = a.weights[at0 + key];
}

// Steps of few tokens (kept_few.cu): which they take, the floats of scratch (the first ones 16-byte aligned), the launch.
bool kept_few_takes(long long tokens, int max_count, int heads, int kv_heads, int head_dim, int max_keys, int dtype, bool weights);
long long kept_few_floats(long long tokens, int n_seqs, int max_count, int heads, int kv_heads, int head_dim, int max_keys, bool weights);
int kept_few(const KeptArgs& a, long long tokens, int max_count, int max_keys, long long pool_pages, int* status, cudaStream_t s);

// Steps of many tokens on the tcgen05 tensor cores: the attention (attention_tc.cu), which leaves the denominators in `lse2` (log2 units,
// [tokens, H], may be null), and the weights from them (kept_weights.cu).
int attention_tc_kept(const KeptArgs& a, float* lse2, long long tokens, int max_count, int max_keys, long long pool_pages, int* status, cudaStream_t s);
int kept_weights_tc(const KeptArgs& a, const float* lse2, long long tokens, int max_count, int max_keys, long long pool_pages, int* status, cudaStream_t s);

}  // namespace slb
