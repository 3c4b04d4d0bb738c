// What the attention kernels share: a sequence's lengths, which keys a query sees, and the
// launchers of the two families (attention_rows.cu on the CUDA cores, attention_tiles.cu on the
// tensor cores), which attention.cu chooses between.
#pragma once
#include "relative.cuh"

namespace b200 {
namespace attention {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// keys, queries and shift of sequence b; a length outside its range is clamped and flagged
struct Sequence {
  int keys, queries, shift;
  __device__ __forceinline__ Sequence(const b200_attention& a, int64_t b) {
    keys = one(a, a.lengths, b, (int)a.keys);
    queries = one(a, a.query_lengths, b, (int)a.queries);
    shift = keys - queries;
  }
  static __device__ __forceinline__ int one(const b200_attention& a, const void* lengths, int64_t b, int all) {
    if (!lengths) return all;
    const int64_t n = a.length_dtype == B200_I64 ? reinterpret_cast<const long long*>(lengths)[b] : (int64_t)reinterpret_cast<const int*>(lengths)[b];
    if (n < 0 || n > all) raise_device_error(B200_ERR_ARG);
    return (int)max((int64_t)0, min((int64_t)all, n));
  }
  // keys that query i (< queries) sees: [first, end)
  __device__ __forceinline__ int first_key(const b200_attention& a, int i) const {
    return a.window ? (int)max((int64_t)0, (int64_t)i + shift - a.window + 1) : 0;
  }
  __device__ __forceinline__ int end_key(const b200_attention& a, int i) const {
    if (a.causal) return min(keys, i + shift + 1);
    return a.window ? (int)min((int64_t)keys, (int64_t)i + shift + a.window) : keys;
  }
  // queries that see key j (< keys): [first, end)
  __device__ __forceinline__ int first_query(const b200_attention& a, int j) const {
    if (a.causal) return max(0, j - shift);
    return a.window ? (int)max((int64_t)0, (int64_t)j - shift - a.window + 1) : 0;
  }
  __device__ __forceinline__ int end_query(const b200_attention& a, int j) const {
    return a.window ? (int)min((int64_t)queries, max((int64_t)0, (int64_t)j - shift + a.window)) : queries;
  }
};

// The gradient makes p = exp(z - lse) again. lse holds the scores' size and log sum exp(z - max) in 24 bits, so the exponent is off by
// the roundings of numbers of that size: five of at most 2^-24 each (z, max + log2 sum, to lse, back, the constants), 0.02 at |lse| =
// 2^16 (p off by 1.2 %), 0.27 at 2^20 (a fifth), hundreds at 1e9. From 2^20 on a row has no probabilities to make again: p = 0, and the
// error flag is set unless its dout is zero.
constexpr float LSE_LIMIT = 1048576.f * LOG2E;  // in the log2 domain
// lse in the log2 domain as the gradient takes it away; infinite where there are no probabilities
__device__ __forceinline__ float exponent_of(float lse) {
  const float x = lse * LOG2E;
  return fabsf(x) >= LSE_LIMIT ? INFINITY : x;
}

// a table entry in the log2 domain; what is finite stays finite
__device__ __forceinline__ float table_log2(const void* table, int64_t at, int dtype) {
  const float v = dtype == B200_BF16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(table)[at]) : reinterpret_cast<const float*>(table)[at];
  const float w = v * LOG2E;
  return isinf(w) && !isinf(v) ? copysignf(3.402823466e38f, w) : w;
}

// attention_rows.cu
size_t rows_forward_workspace(const b200_attention& a);
int rows_forward(const b200_attention& a, void* out, float* lse, void* workspace, cudaStream_t st);
size_t rows_grad_workspace(const b200_attention& a);
int rows_grad(const b200_attention& a, const b200_attention_grads& g, const float* delta, int64_t padded, void* workspace, cudaStream_t st);
// dtable from [batch][heads][blocks][buckets] partial sums, in order
int table_sum(const b200_attention& a, const float* part, int64_t blocks, void* dtable, cudaStream_t st);

// attention_tiles.cu
bool tiles_take(const b200_attention& a);       // whether they make the forward,
bool tiles_take_grad(const b200_attention& a);  // and the gradient
size_t tiles_forward_workspace(const b200_attention& a);
int tiles_forward(const b200_attention& a, void* out, float* lse, void* workspace, cudaStream_t st);
size_t tiles_grad_workspace(const b200_attention& a, const b200_attention_grads* g);  // g NULL: for any dout
// lse2 (log2) and delta: [batch x heads][padded], both negated (so that a query that sees nothing, or is none, has p = 2^-inf),
// padded a multiple of 128
int tiles_grad(const b200_attention& a, const b200_attention_grads& g, const float* lse2, const float* delta, int64_t padded, void* workspace,
               cudaStream_t st);

}  // namespace attention
}  // namespace b200
