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
  // the prefix in `splits` parts: with more than one, every part leaves its normalised result and log-sum-exp in
  // part_out [splits, tokens, Hq, D] and part_lse [splits, tokens, Hq], and a second kernel joins them
  int splits;
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

int prefix_simt_splits(const PrefixArgs& a);
int run_prefix_simt(const PrefixArgs& a, int dtype, cudaStream_t s);
// nullptr when the tensor-core kernel takes the problem, else why not
const char* prefix_sm100_unsupported(const PrefixArgs& a, int dtype);
int prefix_sm100_splits(const PrefixArgs& a);
int run_prefix_sm100(const PrefixArgs& a, int dtype, cudaStream_t s);

}  // namespace nb
