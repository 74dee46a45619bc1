// What the kernels of drafted tokens share: the arguments of a step whose new rows form trees, and what its queries see.
//
// Rows of a sequence are counted from 0 in the order of its block table (64 rows a page). A step appends counts[s] rows, the nodes of
// a tree, behind the past[s] rows that are there. The query of a node sees the row j < past[s] if window == 0 or j > max(positions[node], past[s]) - window,
// and the row past[s] + b of the step if bit b of its words of `seen` is set; a bit at counts[s] or behind says nothing.
#pragma once

#include "common.cuh"

namespace slb {

constexpr int kMostNodes = 256;      // of a sequence in a step

struct TreeArgs {
  const void* q;            // [tokens, H, hd]
  const void* k_pool;       // [pages, K, 64, hd]
  const void* v_pool;
  void* out;                // [tokens, H * hd]
  const int* seq_start;     // [n] first token row of each sequence
  const int* past;          // [n] rows before the step
  const int* counts;        // [n] new rows
  const uint32_t* seen;     // [tokens, words]
  const int* positions;     // [tokens], or null without a window
  const int* block_table;   // [n, table_stride]
  int table_stride, n_seqs, heads, kv_heads, head_dim, window, words, max_count;
  long long tokens, pool_pages;
  float scale;
  float* scratch;
  int splits, max_keys;
};

// What a caller of slb_attention_tree says, in one piece of memory (as KeptCall, kept.cuh).
struct TreeCall {
  const void *q, *k_pool, *v_pool;
  void* out;
  const int *seq_start, *past, *counts;
  const void* seen;
  const int *positions, *block_table;
  float* scratch;
  int* status;              // a zeroed device word that receives a code if a bounded wait inside a kernel gave up
  void* stream;
  long long tokens, scratch_floats, pool_pages;
  int table_stride, n_seqs, max_count, max_keys, heads, kv_heads, head_dim, window, words, dtype;
  float scale;
};
static_assert(sizeof(TreeCall) == 13 * 8 + 3 * 8 + 10 * 4 + 4 + 4, "as packed in kernels/ops.py");

// A sequence's share of a step: its rows before it and its nodes, both inside what the call promised and the given tokens.
struct TreeSeq {
  int past, count, tok0;
  __device__ __forceinline__ TreeSeq(const TreeArgs& a, int seq) {
    tok0 = a.seq_start[seq];
    past = min(max(a.past[seq], 0), a.max_keys);
    count = min(min(max(a.counts[seq], 0), a.max_count), a.max_keys - past);
    if (tok0 < 0 || tok0 >= a.tokens) count = 0;
    else if (count > a.tokens - tok0) count = (int)(a.tokens - tok0);
  }
};

// First row of those before the step that a node sees.
__device__ __forceinline__ int tree_lo(const TreeArgs& a, int token, int past) {
  if (a.window <= 0) return 0;
  const long long lo = (long long)max(a.positions[token], past) - a.window + 1;
  return lo <= 0 ? 0 : lo >= past ? past : (int)lo;
}

// Bits b .. b + 63 of a node's words (zeros outside 0 .. count - 1), for any b.
__device__ __forceinline__ unsigned long long tree_bits(const uint32_t* words, int n_words, int b, int count) {
  auto word = [&](int w) { return w >= 0 && w < n_words ? words[w] : 0u; };
  const int w = b >> 5, sh = b & 31;      // (floor, for negative b too)
  const uint32_t x0 = word(w), x1 = word(w + 1), x2 = sh ? word(w + 2) : 0u;
  unsigned long long v = (unsigned long long)__funnelshift_r(x0, x1, sh) | (unsigned long long)__funnelshift_r(x1, x2, sh) << 32;
  const int left = count - b;             // bits at count and behind go
  if (left <= 0) return 0ull;
  if (left < 64) v &= (1ull << left) - 1ull;
  return v;
}

// On the tensor cores (tree_attention_tc.cu): which calls it takes, the floats of scratch (the first ones 16-byte aligned), the launch.
bool tree_tc_takes(int n_seqs, int max_count, int heads, int kv_heads, int head_dim, int max_keys, int dtype);
long long tree_tc_floats(int n_seqs, int max_count, int heads, int kv_heads, int head_dim, int max_keys);
int tree_tc(const TreeArgs& a, long long pool_pages, int* status, cudaStream_t s);

}  // namespace slb
