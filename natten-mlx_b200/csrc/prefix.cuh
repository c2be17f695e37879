// Attention of a batch's queries to one prefix of keys and values that all samples share: what the launchers of the
// two kernel families have in common.
#pragma once

#include "launch.cuh"

namespace nb {

struct PrefixArgs {
  const void *q, *k, *v;
  const void* window_out;    // result of the same queries over other keys, to be merged in; null (both) without
  const float* window_lse;
  void* out;                 // [tokens, Hq, D]
  float* lse;                // [tokens, Hq]; may be null
  const int* lens;           // [batch] tokens of the prefix a sample sees; null: all
  long long q_token, q_head, k_token, k_head, v_token, v_head;   // strides in elements
  long long tokens;          // query tokens of the batch
  uint32_t per_sample;       // query tokens of one sample
  int Hq, Hkv, G, D;         // G = Hq / Hkv: the queries of one key/value head are tokens x G rows
  int prefix;                // keys
  float scale;
  // With splits > 1 the prefix is cut into so many parts, for all rows (CUDA cores) or for the last `cut` pairs of row
  // tiles (tensor cores; a pair is 256 rows).  Every part leaves its normalised result and log-sum-exp in
  // part_out [splits, part_rows, D] and part_lse [splits, part_rows], and a second kernel joins them.
  int splits;
  long long cut;
  long long part_rows;
  float *part_out, *part_lse;
};

// How two results over disjoint keys are joined: out = a * o0 + b * o1, lse as returned.  -inf stands for no keys.
__device__ __forceinline__ float join_weights(float l0, float l1, float& a, float& b) {
  const float m = fmaxf(l0, l1);
  if (m == -INFINITY) { a = b = 0.f; return m; }
  a = expf(l0 - m);
  b = expf(l1 - m);
  const float t = a + b;
  a /= t;
  b /= t;
  return m + logf(t);
}

// Tokens of the prefix that the queries of `token` see.
__device__ __forceinline__ int prefix_limit(const PrefixArgs& a, long long token) {
  if (a.lens == nullptr) return a.prefix;
  const int n = __ldg(a.lens + (uint32_t)token / a.per_sample);
  return n < 0 ? 0 : n > a.prefix ? a.prefix : n;
}

// The row of out and lse that row `i` of the parts belongs to; -1 for rows of a tile that are not there.
__host__ __device__ inline long long prefix_part_row(const PrefixArgs& a, long long i) {
  if (a.cut == 0) return i;
  const int tile_tokens = 128 / a.G;
  const long long tiles = (a.tokens + tile_tokens - 1) / tile_tokens, pairs = (tiles + 1) / 2;
  const long long item = pairs * a.Hkv - a.cut + i / 256, hk = item / pairs;
  const long long tile = (item - hk * pairs) * 2 + (i >> 7 & 1);
  const int r = (int)(i & 127), tl = r / a.G;
  const long long token = tile * tile_tokens + tl;
  return tl < tile_tokens && token < a.tokens ? token * a.Hq + hk * a.G + (r - tl * a.G) : -1;
}

int prefix_simt_splits(const PrefixArgs& a);
int run_prefix_simt(const PrefixArgs& a, int dtype, cudaStream_t s);
// nullptr when the tensor-core kernel takes the problem, else why not
const char* prefix_sm100_unsupported(const PrefixArgs& a, int dtype);
void prefix_sm100_plan(PrefixArgs* a);   // sets splits and cut
int run_prefix_sm100(const PrefixArgs& a, int dtype, cudaStream_t s);

}  // namespace nb
