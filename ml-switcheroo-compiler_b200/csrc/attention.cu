// The attention entry points: checks, and the choice of the kernels.
#include <algorithm>

#include "attention.cuh"

namespace b200 {
namespace attention {

static int check_attention(const char* what, const b200_attention* a) {
  B200_REQUIRE(a, "%s: no description", what);
  B200_REQUIRE(a->batch >= 0 && a->queries >= 0 && a->keys >= 0 && a->heads >= 1 && a->kv_heads >= 1 && a->heads % a->kv_heads == 0,
               "%s: batch %lld, %lld queries, %lld keys, %lld heads, %lld key heads", what, (long long)a->batch, (long long)a->queries,
               (long long)a->keys, (long long)a->heads, (long long)a->kv_heads);
  B200_REQUIRE(a->batch <= 65535 && a->heads <= 65535 && a->queries < (1 << 30) && a->keys < (1 << 30),
               "%s: batch and heads up to 65535, queries and keys below 2^30", what);
  B200_REQUIRE(a->queries * (a->heads / a->kv_heads) < (1ll << 30), "%s: %lld queries times %lld heads a key head reach 2^30", what,
               (long long)a->queries, (long long)(a->heads / a->kv_heads));
  B200_REQUIRE(a->dim >= 1 && a->dim <= 256, "%s: dim %lld (1 to 256)", what, (long long)a->dim);
  // the kernels multiply by scale log2 e, which has to be a number too
  B200_REQUIRE(a->scale > 0 && a->scale < 3.402823466e38f / LOG2E, "%s: scale %g is not a positive number below 2.3e38", what, (double)a->scale);
  B200_REQUIRE(a->window >= 0, "%s: window %lld", what, (long long)a->window);
  if (a->dtype != B200_F32 && a->dtype != B200_BF16) {
    set_error("%s: dtype %d (F32 and BF16)", what, a->dtype);
    return B200_ERR_DTYPE;
  }
  if (a->lengths || a->query_lengths)
    if (a->length_dtype != B200_I32 && a->length_dtype != B200_I64) {
      set_error("%s: lengths of dtype %d (I32 and I64)", what, a->length_dtype);
      return B200_ERR_DTYPE;
    }
  if (a->table) {
    if (int rc = relative::check(what, &a->relative)) return rc;
    if (a->table_dtype != B200_F32 && a->table_dtype != B200_BF16) {
      set_error("%s: table of dtype %d (F32 and BF16)", what, a->table_dtype);
      return B200_ERR_DTYPE;
    }
  }
  B200_REQUIRE(a->batch == 0 || a->queries == 0 || a->q, "%s: null queries", what);
  B200_REQUIRE(a->batch == 0 || a->keys == 0 || (a->k && a->v), "%s: null keys or values", what);
  return B200_OK;
}

// The description with a window that positions can be added to: 2^31 is more than queries and keys together and hides nothing.
static b200_attention within(const b200_attention& a) {
  b200_attention own = a;
  own.window = std::min<int64_t>(a.window, 1ll << 31);
  return own;
}

// What the gradient needs of each query beside its own row, negated: delta = dout . out, and lse in the log2 domain, infinite where
// the query sees nothing, is none or has lost its probabilities (so that p = 0). out is the caller's, rounded to the heads' type: bf16
// moves all dz of a row by p times one error, and with it an fp32 table's gradient (2.9e-3 of its norm); keeping out in fp32 would
// double its bytes.
// [batch x heads][padded]; 8 lanes a query, FOUR queries of theirs under way.
constexpr int FOUR = 4;
template <typename T>
__global__ void __launch_bounds__(256) delta_kernel(const __grid_constant__ b200_attention a, const T* dout, const T* out, const float* lse, int64_t sb,
                                                    int64_t ss, int64_t sh, float* lse2, float* delta, int padded, int vec) {
  const int64_t b = blockIdx.y;
  const int lane = threadIdx.x & 7, heads = (int)a.heads, dim = (int)a.dim;
  const uint32_t rows = (uint32_t)padded * (uint32_t)heads;  // [padded, heads]
  const uint32_t row0 = blockIdx.x * (32u * FOUR) + (threadIdx.x >> 3);
  const int queries = Sequence(a, b).queries;
  constexpr int V = 16 / sizeof(T);
  float s[FOUR], e[FOUR];
  uint32_t h[FOUR], i[FOUR];
  const T *x[FOUR], *y[FOUR];
#pragma unroll
  for (int n = 0; n < FOUR; ++n) {
    const uint32_t row = row0 + 32u * n;
    i[n] = row / (uint32_t)heads, h[n] = row - i[n] * (uint32_t)heads;
    s[n] = 0.f, e[n] = -INFINITY;
    // a row that is none reads the last one's: no load waits behind a branch
    const int64_t at = min(i[n], (uint32_t)max(queries - 1, 0));
    x[n] = dout + b * sb + at * ss + h[n] * sh, y[n] = out + ((b * a.queries + at) * heads + h[n]) * dim;
    if (queries > 0) e[n] = lse[(b * heads + h[n]) * a.queries + at] * -LOG2E;
  }
  if (queries > 0) {
    for (int c = lane * V; c < dim; c += 8 * V) {
      if (vec) {
        uint4 u[FOUR], w[FOUR];
#pragma unroll
        for (int n = 0; n < FOUR; ++n) u[n] = *reinterpret_cast<const uint4*>(x[n] + c), w[n] = *reinterpret_cast<const uint4*>(y[n] + c);
#pragma unroll
        for (int n = 0; n < FOUR; ++n) {
          const T *p = reinterpret_cast<const T*>(&u[n]), *q = reinterpret_cast<const T*>(&w[n]);
#pragma unroll
          for (int k = 0; k < V; ++k) s[n] = fmaf((float)p[k], (float)q[k], s[n]);
        }
      } else {  // the same elements in the same order
        for (int n = 0; n < FOUR; ++n)
          for (int k = 0; k < V && c + k < dim; ++k) s[n] = fmaf((float)x[n][c + k], (float)y[n][c + k], s[n]);
      }
    }
  }
#pragma unroll
  for (int n = 0; n < FOUR; ++n)
    if ((int)i[n] >= queries) {
      e[n] = -INFINITY, s[n] = 0.f;
    } else if (fabsf(e[n]) >= LSE_LIMIT) {  // as exponent_of
      if (!isinf(e[n])) {
        bool any = false;
        for (int c = lane; c < dim; c += 8) any |= (float)x[n][c] != 0.f;
        if (any) raise_device_error(B200_ERR_ARG);
      }
      e[n] = -INFINITY;
    }
#pragma unroll
  for (int n = 0; n < FOUR; ++n) {
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) s[n] += __shfl_xor_sync(0xffffffffu, s[n], o);
    if (row0 + 32u * n < rows && lane == 0) {
      const int64_t to = (b * heads + h[n]) * padded + i[n];
      delta[to] = -s[n];
      lse2[to] = e[n];
    }
  }
}

static int64_t padded_of(const b200_attention& a) { return ceil_div(a.queries, 128) * 128; }
static size_t delta_bytes(const b200_attention& a) { return (size_t)(2 * a.batch * a.heads * padded_of(a)) * sizeof(float); }

}  // namespace attention
}  // namespace b200

using namespace b200;
using namespace b200::attention;

extern "C" size_t b200_attention_workspace_bytes(const b200_attention* a) {
  if (check_attention("attention", a) || a->batch == 0 || a->queries == 0) return 0;
  return tiles_take(*a) ? tiles_forward_workspace(*a) : rows_forward_workspace(*a);
}

extern "C" int b200_attention_forward(const b200_attention* a, void* out, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_attention("attention", a)) return rc;
  if (a->batch == 0 || a->queries == 0) return B200_OK;
  B200_REQUIRE(out && lse, "attention: null result");
  const size_t need = b200_attention_workspace_bytes(a);
  B200_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0),
               "attention: workspace of %zu bytes, %zu needed on a 256-byte boundary", workspace_bytes, need);
  const b200_attention own = within(*a);
  return tiles_take(own) ? tiles_forward(own, out, lse, workspace, as_stream(stream)) : rows_forward(own, out, lse, workspace, as_stream(stream));
}

extern "C" size_t b200_attention_grad_workspace_bytes_of(const b200_attention* a, const b200_attention_grads* g) {
  if (check_attention("attention_grad", a) || a->batch == 0) return 0;
  return delta_bytes(*a) + (tiles_take_grad(*a) ? tiles_grad_workspace(*a, g) : rows_grad_workspace(*a));
}
extern "C" size_t b200_attention_grad_workspace_bytes(const b200_attention* a) { return b200_attention_grad_workspace_bytes_of(a, nullptr); }

extern "C" int b200_attention_grad(const b200_attention* a, const b200_attention_grads* g, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  if (int rc = check_attention("attention_grad", a)) return rc;
  B200_REQUIRE(g, "attention_grad: no gradients");
  B200_REQUIRE(!a->table || g->dtable, "attention_grad: no place for the table's gradient");
  cudaStream_t st = as_stream(stream);
  const size_t size = a->dtype == B200_F32 ? 4 : 2;
  if (a->batch == 0 || a->queries == 0 || a->keys == 0) {
    if (a->batch * a->queries) cudaMemsetAsync(g->dq, 0, (size_t)(a->batch * a->queries * a->heads * a->dim) * size, st);
    if (a->batch * a->keys) {
      cudaMemsetAsync(g->dk, 0, (size_t)(a->batch * a->keys * a->kv_heads * a->dim) * size, st);
      cudaMemsetAsync(g->dv, 0, (size_t)(a->batch * a->keys * a->kv_heads * a->dim) * size, st);
    }
    if (a->table)
      cudaMemsetAsync(g->dtable, 0, (size_t)(relative::buckets_of(a->relative) * a->heads) * (a->table_dtype == B200_F32 ? 4 : 2), st);
    return check_launch("attention_grad");
  }
  B200_REQUIRE(g->dout && g->out && g->lse && g->dq && g->dk && g->dv, "attention_grad: null operand");
  const size_t need = b200_attention_grad_workspace_bytes_of(a, g);
  B200_REQUIRE(workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0,
               "attention_grad: workspace of %zu bytes, %zu needed on a 256-byte boundary", workspace_bytes, need);
  const b200_attention own = within(*a);
  const int64_t padded = padded_of(*a);
  float *lse2 = reinterpret_cast<float*>(workspace), *delta = lse2 + a->batch * a->heads * padded;
  B200_REQUIRE(padded * a->heads < (1ll << 31), "attention_grad: %lld queries of %lld heads are too many", (long long)a->queries, (long long)a->heads);
  const dim3 grid((unsigned)ceil_div(padded * a->heads, 32 * FOUR), (unsigned)a->batch);
  const int64_t* s = g->dout_stride;
  const int vec = ((reinterpret_cast<uintptr_t>(g->dout) | reinterpret_cast<uintptr_t>(g->out) | (uint64_t)((s[0] | s[1] | s[2] | a->dim) * size)) & 15) == 0;
  if (a->dtype == B200_F32)
    delta_kernel<float><<<grid, 256, 0, st>>>(own, (const float*)g->dout, (const float*)g->out, g->lse, s[0], s[1], s[2], lse2, delta, (int)padded, vec);
  else
    delta_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(own, (const __nv_bfloat16*)g->dout, (const __nv_bfloat16*)g->out, g->lse, s[0], s[1], s[2], lse2,
                                                      delta, (int)padded, vec);
  if (int rc = check_launch("attention_grad")) return rc;
  void* rest = reinterpret_cast<uint8_t*>(workspace) + delta_bytes(*a);
  return tiles_take_grad(own) ? tiles_grad(own, *g, lse2, delta, padded, rest, st) : rows_grad(own, *g, delta, padded, rest, st);
}
