// The output head and its softmax cross entropy over a large vocabulary, without the logits
// in memory, and the gradients.
//
//   z = x w  [N, V],  lse_t = log sum_v exp z_tv,  loss_t = lse_t - z_t,label(t)
//   d_tv = dloss_t (exp(z_tv - lse_t) - [v = label(t)]),  dx = d w^T,  dw = x^T d
//
// Forward: one tcgen05 product whose epilogue keeps, per row and half tile, the
// running maximum and the sum of exponentials of the accumulator (fp32, base 2), and the
// label's logit; a second kernel joins a row's halves. z is never written: 8 bytes leave the
// SM for a half tile's 128 logits.
// Backward: the vocabulary is walked in pieces. A piece's logits are made again (a fourth
// product: the price of not keeping 4 bytes per token and word), its epilogue turns them
// into d, written in the operands' precision to a workspace that one piece fills; the
// piece's columns of dw and its share of dx are two more products over it. dx is added up
// over the pieces in fp32 and rounded once.
// bf16 operands multiply directly; d is rounded to bf16 (half a step of 2^-8 per value, the
// precision of the gradients themselves). fp32 operands are split into two bf16 planes
// (x = hi + lo, 16 bits), three products each (tc_tile.cuh); d likewise.
// Bound by the tensor cores: 2 N D V flop forward, 6 N D V backward.
//
// Up to 8 tokens of fp32, or one of bf16, take kernels of their own (below): reading w bounds them.
// Rows whose label is ignore_index, or outside the vocabulary: loss 0, no gradient, and the row
// of x they hold is replaced by zeros where dw is made, so whatever it contains stays out.
#include "tc_tile.cuh"

namespace b200 {
namespace lx {

using namespace tile;

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ int64_t label_at(const void* labels, int i32, int64_t row) {
  return i32 ? (int64_t) reinterpret_cast<const int*>(labels)[row] : reinterpret_cast<const long long*>(labels)[row];
}

// whether a row of this label takes part in the gradients
__device__ __forceinline__ bool counts(int64_t label, int64_t ignore, int64_t V) { return label != ignore && label >= 0 && label < V; }

// ---- forward epilogue: maxima, sums and the label's logit ----
struct LseEpi {
  struct Args {
    float2* part;  // [parts][N]: (maximum, sum of exp2((z - maximum) log2 e)) of a half tile's columns
    int width;     // columns of a half tile
    float* picked;
    const void* labels;
    int labels_i32;
    int64_t N, V;
  };
  static constexpr bool SINGLE_WIDE = true, SINGLE_NARROW = false, TEAMS = false, INIT = false;
  const Args& a;
  float m, s, at_label;
  int64_t label;
  __device__ explicit LseEpi(const Args& args) : a(args) {}

  __device__ __forceinline__ void begin(const Spot& sp) {
    m = -INFINITY;
    s = 0.f;
    label = sp.row < a.N ? label_at(a.labels, a.labels_i32, sp.row) : -1;
    at_label = 0.f;
  }
  __device__ __forceinline__ void chunk(const Spot& sp, int64_t col, float (&v)[32]) {
    if (col + 32 > a.V) {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (col + i >= a.V) v[i] = -INFINITY;
    }
    const int64_t at = label - col;
    if (at >= 0 && at < 32) {
      const int k = (int)at;
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (k == i) at_label = v[i];
    }
    float top[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
    for (int i = 4; i < 32; ++i) top[i & 3] = fmaxf(top[i & 3], v[i]);
    const float t = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
    if (t > m) {
      s *= ex2((m - t) * LOG2E);  // 0 from -inf
      m = t;
    }
    const float shift = m == -INFINITY ? 0.f : m * LOG2E;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 32; ++i) sum[i & 3] += ex2(fmaf(v[i], LOG2E, -shift));
    s += (sum[0] + sum[1]) + (sum[2] + sum[3]);
  }
  __device__ __forceinline__ void finish(int) {}
  __device__ __forceinline__ void end(const Spot& sp) {
    if (sp.row >= a.N) return;
    a.part[(int64_t)(sp.nt * 2 + sp.half) * a.N + sp.row] = make_float2(m, s);
    const int64_t k = label - sp.col0;
    if (k >= 0 && k < a.width && label < a.V) a.picked[sp.row] = at_label;
  }
};

// lse and loss of each row from its half tiles: 32 threads a row (a row's 250 parts, read one
// after the other, took 9 us at 777 rows), joined in a fixed order
constexpr int JOIN = 32;
__global__ void __launch_bounds__(32 * JOIN) lse_join_kernel(const float2* __restrict__ part, int parts, const float* __restrict__ picked,
                                                             const void* labels, int labels_i32, int64_t ignore,
                                                             float* __restrict__ loss, float* __restrict__ lse, int64_t N, int64_t V) {
  __shared__ float2 red[JOIN][33];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int64_t row = (int64_t)blockIdx.x * 32 + lane;
  float m = -INFINITY, s = 0.f;
  bool nan = false;
  auto join = [&](float2 p) {
    if (isnan(p.x) || isnan(p.y)) nan = true;
    const float M = fmaxf(m, p.x);
    if (M == -INFINITY) return;
    s = s * ex2((m - M) * LOG2E) + p.y * ex2((p.x - M) * LOG2E);
    m = M;
  };
  if (row < N) {
    int i = slice;
    for (; i + 3 * JOIN < parts; i += 4 * JOIN) {
      float2 p[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) p[j] = part[(int64_t)(i + j * JOIN) * N + row];
#pragma unroll
      for (int j = 0; j < 4; ++j) join(p[j]);
    }
    for (; i < parts; i += JOIN) join(part[(int64_t)i * N + row]);
  }
  red[slice][lane] = make_float2(nan ? NAN : m, s);
  __syncthreads();
  if (slice || row >= N) return;
  for (int i = 1; i < JOIN; ++i) join(red[i][lane]);
  const float out = nan ? NAN : m + LN2 * log2f(s);
  lse[row] = out;
  const int64_t label = label_at(labels, labels_i32, row);
  if (label == ignore) {
    loss[row] = 0.f;
  } else if (label < 0 || label >= V) {
    raise_device_error(B200_ERR_ARG);
    loss[row] = 0.f;
  } else {
    loss[row] = out - picked[row];
  }
}

// ---- backward: the gradient of the logits of one piece of the vocabulary ----
struct GradEpi {
  struct Args {
    CUtensorMap map;  // d [planes][N][ld], stored 32 x 32 at a time
    int planes;
    const float *dloss, *lse;
    const void* labels;
    int labels_i32;
    int64_t ignore, N, V, first;  // first: the piece's first column of w
  };
  static constexpr bool SINGLE_WIDE = true, SINGLE_NARROW = false, TEAMS = false, INIT = false;
  const Args& a;
  float g, shift;
  int64_t label;  // relative to the piece
  uint32_t kept;  // all ones, or zero for an ignored row
  uint32_t turn;
  __device__ explicit GradEpi(const Args& args) : a(args), turn(0) {}

  __device__ __forceinline__ void begin(const Spot& sp) {
    g = shift = 0.f;
    label = -1;
    kept = 0u;
    if (sp.row >= a.N) return;
    const int64_t l = label_at(a.labels, a.labels_i32, sp.row);
    if (!counts(l, a.ignore, a.V)) return;
    label = l - a.first;
    kept = ~0u;
    g = a.dloss[sp.row];
    shift = a.lse[sp.row] * LOG2E;
  }
  __device__ __forceinline__ void chunk(const Spot& sp, int64_t col, float (&v)[32]) {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = g * ex2(fmaf(v[i], LOG2E, -shift));
    const int64_t at = label - col;
    if (at >= 0 && at < 32) {
      const int k = (int)at;
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (k == i) v[i] -= g;
    }
    for (int plane = 0; plane < a.planes; ++plane) {
      uint32_t w[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) w[i] = pack_bf16(v[2 * i], v[2 * i + 1]) & kept;
      // two 2 KB buffers: the bulk store before the last one has been read
      const uint32_t buf = sp.buf + (turn++ & 1) * 2048;
      if (sp.lane == 0) bulk_wait_read1();
      __syncwarp();
      stage_chunk<2>(buf, sp.lane, w);
      fence_proxy_async_smem();
      __syncwarp();
      if (sp.lane == 0) {
        tma_store_4d(&a.map, buf, (int)col, (int)sp.row0, plane, 0);
        bulk_commit();
      }
      if (plane + 1 < a.planes) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const __nv_bfloat162 h = *reinterpret_cast<const __nv_bfloat162*>(&w[i]);
          v[2 * i] -= __low2float(h);
          v[2 * i + 1] -= __high2float(h);
        }
      }
    }
  }
  __device__ __forceinline__ void end(const Spot&) {}
  __device__ __forceinline__ void finish(int lane) {
    if (lane == 0) bulk_wait0();
  }
};

// ---- plain result: C = acc (+ an fp32 addend), fp32 or bf16; K splits write partials ----
struct StoreEpi {
  struct Args {
    void* C;
    const float* add;  // same element offsets as an fp32 C of leading dimension ld_add, or NULL
    int64_t ld, ld_add, split_stride, M, N;
    int bf16;
  };
  static constexpr bool SINGLE_WIDE = true, SINGLE_NARROW = true, TEAMS = false, INIT = true;
  static constexpr float scale = 1.f;
  const Args& a;
  __device__ explicit StoreEpi(const Args& args) : a(args) {}
  __device__ __forceinline__ void begin(const Spot&) {}
  __device__ __forceinline__ void end(const Spot&) {}
  __device__ __forceinline__ void finish(int) {}
  __device__ __forceinline__ bool dense(int64_t col) const {  // 16-byte rows of whole chunks
    return col + 32 <= a.N && (a.ld_add & 3) == 0 && (reinterpret_cast<uintptr_t>(a.add) & 15) == 0;
  }
  __device__ __forceinline__ bool adds() const { return a.add != nullptr; }
  __device__ __forceinline__ void fetch(const Spot& sp, int64_t col, float (&v)[32]) {
    if (!a.add) return;
    const int rows = (int)min((int64_t)32, a.M - sp.row0);
    const float* p = a.add + sp.row0 * a.ld_add + col;
    if (dense(col)) {
      rows_load<4>(reinterpret_cast<const uint8_t*>(p), a.ld_add * 4, rows, 8, sp.lane, v, 0);
    } else if (sp.lane < rows) {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (col + i < a.N) v[i] = p[sp.lane * a.ld_add + i];
    }
  }
  __device__ __forceinline__ void ready(const Spot& sp, int64_t col, float (&v)[32]) {
    if (a.add && dense(col)) rows_in<4>(sp.buf, sp.lane, v, 0);
  }
  __device__ __forceinline__ void chunk(const Spot& sp, int64_t col, float (&v)[32]) {
    const int rows = (int)min((int64_t)32, a.M - sp.row0);
    const int64_t cols = min((int64_t)32, a.N - col);
    const int64_t at = sp.split * a.split_stride + sp.row0 * a.ld + col;
    __syncwarp();
    if (a.bf16) {
      uint32_t w[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) w[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
      stage_chunk<2>(sp.buf, sp.lane, w);
      __syncwarp();
      put_chunk<2>(sp.buf, sp.lane, reinterpret_cast<uint8_t*>(reinterpret_cast<__nv_bfloat16*>(a.C) + at), a.ld, rows, (int)cols);
    } else {
      uint32_t w[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) w[i] = __float_as_uint(v[i]);
      stage_chunk<4>(sp.buf, sp.lane, w);
      __syncwarp();
      put_chunk<4>(sp.buf, sp.lane, reinterpret_cast<uint8_t*>(reinterpret_cast<float*>(a.C) + at), a.ld, rows, (int)cols);
    }
  }
};

// partial results [splits][n] (fp32), added in order (+ add), rounded once
__global__ void __launch_bounds__(256) join_splits_kernel(const float* __restrict__ part, int splits, int64_t n, int64_t cols,
                                                          const float* __restrict__ add, void* out, int bf16, int64_t ld) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    float v = add ? add[i] : 0.f;
    for (int k = 0; k < splits; ++k) v += part[k * n + i];
    const int64_t at = i / cols * ld + i % cols;
    if (bf16) reinterpret_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(v);
    else reinterpret_cast<float*>(out)[at] = v;
  }
}

// A dense 16-bit operand with 16-byte rows from src [rows, cols] (row stride ld): bf16 copied,
// fp32 split into two bf16 planes. With labels, the rows of tokens that do not count become zeros.
template <bool F32>
__global__ void __launch_bounds__(256) pack_kernel(const void* __restrict__ src, int64_t ld, __nv_bfloat16* __restrict__ out, int64_t ldo,
                                                   int64_t plane, int64_t rows, int64_t cols, const void* labels, int labels_i32,
                                                   int64_t ignore, int64_t V) {
  const int64_t per = ldo / 8, total = rows * per;  // 8 elements a thread
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per, c = i % per * 8;
    const bool zero = labels && !counts(label_at(labels, labels_i32, r), ignore, V);
    float v[8];
    const int64_t at = r * ld + c;
    if constexpr (F32) {
      const float* p = reinterpret_cast<const float*>(src) + at;
      if (c + 8 <= cols && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
        const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
      } else {
        for (int j = 0; j < 8; ++j) v[j] = c + j < cols ? p[j] : 0.f;
      }
    } else {
      const __nv_bfloat16* p = reinterpret_cast<const __nv_bfloat16*>(src) + at;
      if (c + 8 <= cols && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
        uint4 u = *reinterpret_cast<const uint4*>(p);
        if (zero) u = make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(out + r * ldo + c) = u;
        continue;
      }
      for (int j = 0; j < 8; ++j) v[j] = c + j < cols ? __bfloat162float(p[j]) : 0.f;
    }
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float a = zero ? 0.f : v[2 * j], b = zero ? 0.f : v[2 * j + 1];
      const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
      hi[j] = *reinterpret_cast<const uint32_t*>(&h);
      // a value that is not finite has no low part (inf - inf)
      const float la = a - __low2float(h), lb = b - __high2float(h);
      lo[j] = pack_bf16(isfinite(la) ? la : 0.f, isfinite(lb) ? lb : 0.f);
    }
    *reinterpret_cast<uint4*>(out + r * ldo + c) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    if constexpr (F32) *reinterpret_cast<uint4*>(out + plane + r * ldo + c) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
  }
}

// ---- few tokens: up to 8 rows of fp32 x, or one of bf16, on the CUDA cores ----
// With N rows a weight is worth 2 N flop forward and 6 N backward: below about a dozen rows
// reading w (and writing dw) bounds the call, a 128-row tile is mostly padding, and splitting
// fp32 weights into planes triples the bytes. x (fp32) stays in shared memory, w is read
// once forward, twice backward (the second time for dx, from the L2 where it fits). Products
// and sums are fp32 throughout.
namespace few {

constexpr int MOST = 8, WARPS = 8, T = 32 * WARPS, X_FLOATS = 12288;

struct Args {
  const void *x, *w, *labels;
  const float *dloss, *lse;
  int64_t ldx, ldw, ignore;
  int labels_i32, N, D, V;
  float2* part;    // forward: [blocks][N]
  float* picked;
  float* d;        // backward: [N][V]
  void* dw;
  int dw_bf16;
};

template <typename E>
__device__ __forceinline__ float value(E v);
template <>
__device__ __forceinline__ float value<float>(float v) { return v; }
template <>
__device__ __forceinline__ float value<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// W adjacent elements (one 8- or 16-byte access where W > 1)
template <typename E, int W>
__device__ __forceinline__ void get(const E* p, float (&v)[W]) {
  if constexpr (W == 1) {
    v[0] = value(*p);
  } else if constexpr (sizeof(E) == 4) {
    const float4 u = *reinterpret_cast<const float4*>(p);
    v[0] = u.x, v[1] = u.y, v[2] = u.z, v[3] = u.w;
  } else {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    v[0] = __uint_as_float(u.x << 16), v[1] = __uint_as_float(u.x & 0xffff0000u);
    v[2] = __uint_as_float(u.y << 16), v[3] = __uint_as_float(u.y & 0xffff0000u);
  }
}
template <typename E, int W>
__device__ __forceinline__ void set(E* p, const float (&v)[W]) {
  if constexpr (sizeof(E) == 4) {
    if constexpr (W == 1) *p = v[0];
    else *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    if constexpr (W == 1) *p = __float2bfloat16_rn(v[0]);
    else *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
  }
}

// W elements of dw from the at-th on
template <int W>
__device__ __forceinline__ void set_dw(const Args& a, int64_t at, const float (&v)[W]) {
  if (a.dw_bf16) set<__nv_bfloat16, W>(reinterpret_cast<__nv_bfloat16*>(a.dw) + at, v);
  else set<float, W>(reinterpret_cast<float*>(a.dw) + at, v);
}

// x as fp32 [NT][D] (rows that do not exist, and with `masked` those of tokens that do not count, zeros)
template <typename E, int NT>
__device__ __forceinline__ void load_x(const Args& a, float* xs, bool masked) {
  for (int t = 0; t < NT; ++t) {
    const bool in = t < a.N && !(masked && !counts(label_at(a.labels, a.labels_i32, t), a.ignore, a.V));
    for (int k = threadIdx.x; k < a.D; k += T) xs[t * a.D + k] = in ? value(reinterpret_cast<const E*>(a.x)[t * a.ldx + k]) : 0.f;
  }
}

// gradient of a logit z of token t at word v
struct Row {
  float g, shift;
  int64_t label;
  bool kept;
  __device__ __forceinline__ void load(const Args& a, int t) {
    kept = false, g = shift = 0.f, label = -1;
    if (t >= a.N) return;
    const int64_t l = label_at(a.labels, a.labels_i32, t);
    if (!counts(l, a.ignore, a.V)) return;
    kept = true, label = l, g = a.dloss[t], shift = a.lse[t] * LOG2E;
  }
  __device__ __forceinline__ float grad(float z, int64_t v) const {
    return kept ? g * ex2(fmaf(z, LOG2E, -shift)) - (v == label ? g : 0.f) : 0.f;
  }
};

__device__ __forceinline__ void online(float& m, float& s, float z) {
  const float M = fmaxf(m, z);
  if (M != -INFINITY || isnan(z)) {
    s = s * ex2((m - M) * LOG2E) + ex2((z - M) * LOG2E);
    m = M;
  }
}

// w stored [V, D]: a warp takes P words at a time (each element of x read from shared memory
// serves P products), lanes along D
template <typename E, int NT, int W, bool GRAD>
__global__ void __launch_bounds__(T) words_kernel(const __grid_constant__ Args a) {
  constexpr int P = NT >= 4 ? 4 : 2;
  extern __shared__ float xs[];
  __shared__ float2 red[WARPS][NT];
  load_x<E, NT>(a, xs, GRAD);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Row row[NT];
  int64_t label[NT];
  float m[NT], s[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    if (GRAD) row[t].load(a, t);
    label[t] = t < a.N ? label_at(a.labels, a.labels_i32, t) : -1;
    m[t] = -INFINITY, s[t] = 0.f;
  }
  __syncthreads();
  const E* w = reinterpret_cast<const E*>(a.w);
  for (int64_t v0 = ((int64_t)blockIdx.x * WARPS + warp) * P; v0 < a.V; v0 += (int64_t)gridDim.x * WARPS * P) {
    float z[P][NT] = {};
    const E* p[P];
#pragma unroll
    for (int j = 0; j < P; ++j) p[j] = w + min(v0 + j, (int64_t)a.V - 1) * a.ldw;
#pragma unroll(P == 2 ? 4 : 2)
    for (int k = lane * W; k < a.D; k += 32 * W) {
      float u[P][W];
#pragma unroll
      for (int j = 0; j < P; ++j) get<E, W>(p[j] + k, u[j]);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float xv[W];
        get<float, W>(xs + t * a.D + k, xv);
#pragma unroll
        for (int i = 0; i < W; ++i)
#pragma unroll
          for (int j = 0; j < P; ++j) z[j][t] = fmaf(u[j][i], xv[i], z[j][t]);
      }
    }
#pragma unroll
    for (int j = 0; j < P; ++j)
#pragma unroll
      for (int t = 0; t < NT; ++t) z[j][t] = warp_sum(z[j][t]);
#pragma unroll
    for (int j = 0; j < P; ++j) {
      if (v0 + j >= a.V) break;
      if constexpr (!GRAD) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          online(m[t], s[t], z[j][t]);
          if (lane == 0 && label[t] == v0 + j) a.picked[t] = z[j][t];
        }
      } else {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          z[j][t] = row[t].grad(z[j][t], v0 + j);
          if (lane == 0 && t < a.N) a.d[(int64_t)t * a.V + v0 + j] = z[j][t];
        }
      }
    }
    if constexpr (GRAD) {
      if (!a.dw) continue;
      for (int k = lane * W; k < a.D; k += 32 * W) {
        float o[P][W] = {};
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          float xv[W];
          get<float, W>(xs + t * a.D + k, xv);
#pragma unroll
          for (int i = 0; i < W; ++i)
#pragma unroll
            for (int j = 0; j < P; ++j) o[j][i] = fmaf(z[j][t], xv[i], o[j][i]);
        }
#pragma unroll
        for (int j = 0; j < P; ++j)
          if (v0 + j < a.V) set_dw<W>(a, (v0 + j) * a.D + k, o[j]);
      }
    }
  }
  if constexpr (!GRAD) {
    if (lane == 0)
#pragma unroll
      for (int t = 0; t < NT; ++t) red[warp][t] = make_float2(m[t], s[t]);
    __syncthreads();
    if (threadIdx.x < NT && (int)threadIdx.x < a.N) {
      const int t = threadIdx.x;
      float M = -INFINITY, S = 0.f;
      for (int i = 0; i < WARPS; ++i) M = fmaxf(M, red[i][t].x);
      for (int i = 0; i < WARPS; ++i)
        if (red[i][t].x != -INFINITY || isnan(red[i][t].y)) S += red[i][t].y * ex2((red[i][t].x - M) * LOG2E);
      a.part[(int64_t)blockIdx.x * a.N + t] = make_float2(M, S);
    }
  }
}

// w stored [D, V]: a block takes 32 W columns, its warps share out D
template <typename E, int NT, int W, bool GRAD>
__global__ void __launch_bounds__(T) columns_kernel(const __grid_constant__ Args a) {
  extern __shared__ float xs[];
  float* red = xs + NT * a.D;  // [WARPS][NT][32 W]; then d in [0][..]
  load_x<E, NT>(a, xs, GRAD);
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c0 = (int64_t)blockIdx.x * 32 * W, c = c0 + lane * W;
  const E* w = reinterpret_cast<const E*>(a.w) + c;
  float z[NT][W] = {};
  if (c < a.V) {  // W divides V where W > 1
#pragma unroll 4
    for (int k = warp; k < a.D; k += WARPS) {
      float u[W];
      get<E, W>(w + (int64_t)k * a.ldw, u);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < W; ++i) z[t][i] = fmaf(u[i], xs[t * a.D + k], z[t][i]);
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < W; ++i) red[(warp * NT + t) * 32 * W + lane * W + i] = z[t][i];
  __syncthreads();
  // warp t finishes token t (NT <= WARPS): 32 W columns
  if (warp < NT && warp < a.N) {
    const int t = warp;
    Row row;
    if (GRAD) row.load(a, t);
    const int64_t label = label_at(a.labels, a.labels_i32, t);
    float m = -INFINITY, s = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const int at = i * 32 + lane;
      if (c0 + at >= a.V) continue;
      float v = 0.f;
#pragma unroll
      for (int j = 0; j < WARPS; ++j) v += red[(j * NT + t) * 32 * W + at];
      if constexpr (GRAD) {
        v = row.grad(v, c0 + at);
        a.d[(int64_t)t * a.V + c0 + at] = v;
        red[t * 32 * W + at] = v;  // this token's first slot: read above by this lane alone
      } else {
        online(m, s, v);
        if (label == c0 + at) a.picked[t] = v;
      }
    }
    if constexpr (!GRAD) {
      const bool nan = isnan(s);
      const float M = warp_max(m);
      s = warp_sum(nan ? NAN : (m == -INFINITY ? 0.f : s * ex2((m - M) * LOG2E)));
      if (lane == 0) a.part[(int64_t)blockIdx.x * a.N + t] = make_float2(M, s);
    }
  }
  if constexpr (GRAD) {
    __syncthreads();
    if (!a.dw || c >= a.V) return;
    float d[NT][W];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < W; ++i) d[t][i] = t < a.N ? red[t * 32 * W + lane * W + i] : 0.f;
#pragma unroll 2
    for (int k = warp; k < a.D; k += WARPS) {
      float o[W] = {};
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < W; ++i) o[i] = fmaf(d[t][i], xs[t * a.D + k], o[i]);
      set_dw<W>(a, c + (int64_t)k * a.V, o);
    }
  }
}

// dx = d w^T over one slice of the words (blockIdx.y): part [slices][N][D]
template <typename E, int NT, int W>
__global__ void __launch_bounds__(T) dx_words_kernel(const __grid_constant__ Args a, float* part, int64_t per) {
  __shared__ float ds[NT][64];
  const int k = (blockIdx.x * T + threadIdx.x) * W;
  const int64_t lo = blockIdx.y * per, hi = min((int64_t)a.V, lo + per);
  const E* w = reinterpret_cast<const E*>(a.w) + k;
  float o[NT][W] = {};
  for (int64_t v0 = lo; v0 < hi; v0 += 64) {
    __syncthreads();
    for (int i = threadIdx.x; i < NT * 64; i += T)
      ds[i / 64][i % 64] = i / 64 < a.N && v0 + i % 64 < hi ? a.d[(int64_t)(i / 64) * a.V + v0 + i % 64] : 0.f;
    __syncthreads();
    if (k >= a.D) continue;
    const int n = (int)min((int64_t)64, hi - v0);
#pragma unroll 8
    for (int j = 0; j < n; ++j) {
      float u[W];
      get<E, W>(w + (v0 + j) * a.ldw, u);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < W; ++i) o[t][i] = fmaf(ds[t][j], u[i], o[t][i]);
    }
  }
  if (k < a.D)
#pragma unroll
    for (int t = 0; t < NT; ++t)
      if (t < a.N)
#pragma unroll
        for (int i = 0; i < W; ++i) part[((int64_t)blockIdx.y * a.N + t) * a.D + k + i] = o[t][i];
}

// the same for w stored [D, V]: a warp takes 4 features, lanes along the slice's words, 256 of
// d at a time in shared memory
template <typename E, int NT, int W>
__global__ void __launch_bounds__(T) dx_columns_kernel(const __grid_constant__ Args a, float* part, int64_t per) {
  __shared__ __align__(16) float ds[NT][256];
  const int lane = threadIdx.x & 31, k0 = (blockIdx.x * WARPS + (threadIdx.x >> 5)) * 4;
  const int64_t lo = blockIdx.y * per, hi = min((int64_t)a.V, lo + per);
  const E* w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = reinterpret_cast<const E*>(a.w) + (int64_t)min(k0 + j, a.D - 1) * a.ldw;
  float o[4][NT] = {};
  for (int64_t v0 = lo; v0 < hi; v0 += 256) {
    __syncthreads();
    for (int i = threadIdx.x; i < NT * 256; i += T)
      ds[i / 256][i % 256] = i / 256 < a.N && v0 + i % 256 < hi ? a.d[(int64_t)(i / 256) * a.V + v0 + i % 256] : 0.f;
    __syncthreads();
    const int n = (int)min((int64_t)256, hi - v0);
#pragma unroll(256 / (32 * W) < 4 ? 256 / (32 * W) : 4)
    for (int c = lane * W; c < n; c += 32 * W) {
      float u[4][W];
#pragma unroll
      for (int j = 0; j < 4; ++j) get<E, W>(w[j] + v0 + c, u[j]);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float d[W];
        get<float, W>(&ds[t][c], d);
#pragma unroll
        for (int i = 0; i < W; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[j][t] = fmaf(d[i], u[j][i], o[j][t]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const float v = warp_sum(o[j][t]);
      if (lane == 0 && t < a.N && k0 + j < a.D) part[((int64_t)blockIdx.y * a.N + t) * a.D + k0 + j] = v;
    }
}

// the slices' parts [slices][n], 32 threads a value, added in a fixed order, rounded once
__global__ void __launch_bounds__(1024) join_slices_kernel(const float* __restrict__ part, int slices, int64_t n, void* out, int bf16) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, at = threadIdx.x >> 5;
  const int64_t i = (int64_t)blockIdx.x * 32 + lane;
  float v = 0.f;
  if (i < n)
#pragma unroll 4
    for (int k = at; k < slices; k += 32) v += part[(int64_t)k * n + i];
  red[at][lane] = v;
  __syncthreads();
  if (at || i >= n) return;
  for (int k = 1; k < 32; ++k) v += red[k][lane];
  if (bf16) reinterpret_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(v);
  else reinterpret_cast<float*>(out)[i] = v;
}

// tokens rounded up to a kernel's 1, 2, 4 or 8
static int rounded(int64_t N) { return N <= 1 ? 1 : (N <= 2 ? 2 : (N <= 4 ? 4 : 8)); }
// Where these kernels are the faster ones for both layouts of w (1024 x 32000, us forward / gradient,
// w stored [V, D] and [D, V]): fp32 up to 8 tokens (1: 28 / 73 and 42 / 91, 8: 52 / 143 and
// 53 / 147, the tiles 94 / 147 at 9), bf16 for one (15 / 47 and 19 / 56). Two bf16 tokens take 18 / 58
// and 31 / 77 here, 19 / 63 and 20 / 63 by the tiles, which have them: [V, D] alone gains too little
// for a rule of its own. x has to fit shared memory.
static bool fits(int dtype, int64_t N, int64_t D) { return N <= (dtype == B200_F32 ? MOST : 1) && rounded(N) * D <= X_FLOATS; }
// blocks of the first kernel: word rows by the SMs, or one per 32 W columns
static int64_t blocks(int w_dn, int wide, int64_t V) {
  return w_dn ? ceil_div(V, wide ? 128 : 32) : std::min<int64_t>(ceil_div(V, 4 * WARPS), 4 * num_sms());
}
// whole vectors of 4 words (or features) at every row
static int vectors(int dtype, const void* w, int64_t ldw, int64_t row) {
  const uint64_t unit = dtype == B200_F32 ? 16 : 8;
  return row % 4 == 0 && ldw % 4 == 0 && reinterpret_cast<uintptr_t>(w) % unit == 0;
}
// slices of the words for dx: 4 blocks an SM, as far as a slice keeps 64 words
static int64_t slices(int w_dn, int wide, int64_t D, int64_t V) {
  const int64_t across = w_dn ? ceil_div(D, 4 * WARPS) : ceil_div(D, (int64_t)T * (wide ? 4 : 1));
  return std::max<int64_t>(1, std::min(ceil_div(4 * (int64_t)num_sms(), across), ceil_div(V, w_dn ? 256 : 64)));
}

template <typename E, int NT, int W>
static int launch(const Args& a, int w_dn, bool grad, float* dx_part, int64_t n_slices, cudaStream_t s, const char* what) {
  // The limit on shared memory is the function's, for all its callers: raised to the most that
  // any call needs, never to this call's size, below which another thread's launch may need more.
  constexpr size_t MOST_X = (size_t)X_FLOATS * 4, RED = (size_t)WARPS * NT * 32 * W * 4;
  const size_t x_bytes = (size_t)NT * a.D * 4;
  const unsigned grid = (unsigned)blocks(w_dn, W > 1, a.V);
  if (w_dn) {
    auto* fn = grad ? columns_kernel<E, NT, W, true> : columns_kernel<E, NT, W, false>;
    if (x_bytes + RED > 48 * 1024) cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(MOST_X + RED));
    fn<<<grid, T, x_bytes + RED, s>>>(a);
  } else {
    auto* fn = grad ? words_kernel<E, NT, W, true> : words_kernel<E, NT, W, false>;
    if (x_bytes + 1024 > 48 * 1024) cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)MOST_X);
    fn<<<grid, T, x_bytes, s>>>(a);
  }
  int rc = check_launch(what);
  if (rc || !dx_part) return rc;
  const int64_t per = ceil_div(ceil_div(a.V, n_slices), 4) * 4;
  if (w_dn) dx_columns_kernel<E, NT, W><<<dim3((unsigned)ceil_div(a.D, 4 * WARPS), (unsigned)n_slices), T, 0, s>>>(a, dx_part, per);
  else dx_words_kernel<E, NT, W><<<dim3((unsigned)ceil_div(a.D, (int64_t)T * W), (unsigned)n_slices), T, 0, s>>>(a, dx_part, per);
  return check_launch(what);
}

static int run(int dtype, const Args& a, int w_dn, int wide, bool grad, float* dx_part, int64_t n_slices, cudaStream_t s, const char* what) {
  if (dtype == B200_BF16)
    return wide ? launch<__nv_bfloat16, 1, 4>(a, w_dn, grad, dx_part, n_slices, s, what)
                : launch<__nv_bfloat16, 1, 1>(a, w_dn, grad, dx_part, n_slices, s, what);
  switch (rounded(a.N) * 2 + wide) {
    case 2: return launch<float, 1, 1>(a, w_dn, grad, dx_part, n_slices, s, what);
    case 3: return launch<float, 1, 4>(a, w_dn, grad, dx_part, n_slices, s, what);
    case 4: return launch<float, 2, 1>(a, w_dn, grad, dx_part, n_slices, s, what);
    case 5: return launch<float, 2, 4>(a, w_dn, grad, dx_part, n_slices, s, what);
    case 8: return launch<float, 4, 1>(a, w_dn, grad, dx_part, n_slices, s, what);
    case 9: return launch<float, 4, 4>(a, w_dn, grad, dx_part, n_slices, s, what);
    case 16: return launch<float, 8, 1>(a, w_dn, grad, dx_part, n_slices, s, what);
    default: return launch<float, 8, 4>(a, w_dn, grad, dx_part, n_slices, s, what);
  }
}

}  // namespace few

// ---------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------

static int64_t up8(int64_t v) { return (v + 7) / 8 * 8; }
static int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }

// A 16-bit operand that TMA can read needs 16-byte rows and base; anything else, and fp32,
// is packed into the workspace.
static bool needs_pack(int dtype, const void* p, int64_t ld) {
  return dtype == B200_F32 || (reinterpret_cast<uintptr_t>(p) & 15) || ld % 8;
}

static int pack(int dtype, const void* src, int64_t ld, __nv_bfloat16* out, int64_t rows, int64_t cols, const void* labels, int labels_i32,
                int64_t ignore, int64_t V, cudaStream_t s) {
  const int64_t ldo = up8(cols), total = rows * (ldo / 8);
  const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(total, 256), (int64_t)num_sms() * 16);
  if (dtype == B200_F32)
    pack_kernel<true><<<grid, 256, 0, s>>>(src, ld, out, ldo, rows * ldo, rows, cols, labels, labels_i32, ignore, V);
  else
    pack_kernel<false><<<grid, 256, 0, s>>>(src, ld, out, ldo, rows * ldo, rows, cols, labels, labels_i32, ignore, V);
  return check_launch("linear_cross_entropy pack");
}

// Sizes of one call and where its scratch lies in the workspace (offsets in bytes)
struct Plan {
  int64_t N, D, V;
  int planes, w_dn;       // w_dn: w is stored [D, V] (V adjacent), else [V, D]
  int64_t w_rows, w_cols; // of the stored matrix
  size_t x, w, part, picked, d, xg, acc, split, dw_acc, bytes;
  int64_t width;          // columns of one piece
  int64_t tokens, words;  // of one product for dw, and for dx
  bool few;               // the kernels for up to 8 tokens
  int wide;               // their vectors of 4
  int64_t parts, slices;
};

static size_t align256(size_t v) { return (v + 255) & ~size_t(255); }

constexpr size_t PIECE_BYTES = size_t(512) << 20;
// Tokens of a dw product, or words of a dx product, that one accumulator takes where operands are one
// plane: its additions are cut towards zero (tc_tile.cuh), and sums of one sign fall short by
// 1.7e-4 over 32768 terms, 3.7e-4 over 65536, 7.8e-4 over 131072. More terms than this are several
// products, added up in fp32 with rounding; the shortfall stays at a twentieth of bf16's half step.
constexpr int64_t MOST_TERMS = 32768;

// The piece: as few as keep d (2 bytes per token, column and plane) within 512 MiB, and of
// those counts the one whose dw tiles fill the CTA pairs best, since each piece ends with
// a partial wave.
static int64_t piece_width(int64_t N, int64_t D, int64_t V, int planes) {
  const int64_t most = std::max<int64_t>(256, (int64_t)(PIECE_BYTES / (size_t)(2 * planes) / (size_t)std::max<int64_t>(N, 1)) / 256 * 256);
  const int64_t cols = ceil_div(V, 256), units = std::max(1, num_sms() / 2), per_col = ceil_div(D, 256);
  const int64_t least = ceil_div(cols, most / 256);
  int64_t best = 0, best_waves = INT64_MAX;
  for (int64_t n = least; n <= least + 3; ++n) {
    const int64_t w = ceil_div(cols, n);
    int64_t waves = 0;
    for (int64_t c = 0; c < cols; c += w) waves += ceil_div(std::min(w, cols - c) * per_col, units);
    if (waves < best_waves) best_waves = waves, best = w;
  }
  return std::min(best * 256, up256(V));
}

// splits of the K axis so that few output tiles still occupy the SMs; each split keeps at
// least 8 K blocks
static int splits_for(int64_t M, int64_t N, int64_t K) {
  const int64_t tiles = ceil_div(M, 256) * ceil_div(N, 256), units = num_sms() / 2;
  return (int)std::max<int64_t>(1, std::min(units / std::max<int64_t>(tiles, 1), ceil_div(K, BK) / 8));
}

static Plan plan(bool grad, int dtype, const void* x, int64_t ldx, const void* w, int64_t ldw, int w_dn, int64_t N, int64_t D, int64_t V) {
  Plan p = {};
  p.N = N, p.D = D, p.V = V, p.w_dn = w_dn;
  p.planes = dtype == B200_F32 ? 2 : 1;
  p.w_rows = w_dn ? D : V;
  p.w_cols = w_dn ? V : D;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at = align256(at + bytes);
    return here;
  };
  p.few = few::fits(dtype, N, D);
  if (p.few) {
    p.wide = few::vectors(dtype, w, ldw, w_dn ? V : D);
    p.parts = few::blocks(w_dn, p.wide, V);
    p.slices = few::slices(w_dn, p.wide, D, V);
    if (!grad) {
      p.part = take((size_t)p.parts * N * sizeof(float2));
      p.picked = take((size_t)N * 4);
    } else {
      p.d = take((size_t)N * V * 4);
      p.split = take((size_t)p.slices * N * D * 4);
    }
    p.bytes = at;
    return p;
  }
  const size_t xb = (size_t)p.planes * N * up8(D) * 2;
  // forward x is read as it is where it can be; the gradient's copy has zeros for rows that do not count
  if (!grad && needs_pack(dtype, x, ldx)) p.x = take(xb);
  if (needs_pack(dtype, w, ldw)) p.w = take((size_t)p.planes * p.w_rows * up8(p.w_cols) * 2);
  if (!grad) {
    p.part = take((size_t)ceil_div(V, p.planes > 1 && N <= 128 ? 128 : 256) * 2 * N * sizeof(float2));
    p.picked = take((size_t)N * 4);
  } else {
    p.width = piece_width(N, D, V, p.planes);
    p.d = take((size_t)p.planes * N * p.width * 2);
    p.xg = take(xb);
    const int64_t width = std::min(p.width, V);
    p.words = p.planes > 1 ? width : std::min(width, MOST_TERMS * splits_for(N, D, width));
    p.tokens = p.planes > 1 ? N : std::min(N, MOST_TERMS * splits_for(D, width, N));
    if (p.words < V) p.acc = take((size_t)N * D * 4);
    if (p.tokens < N) p.dw_acc = take((size_t)D * p.width * 4);
    // splits x tiles of 256 x 256 never exceed the pairs of SMs
    p.split = take((size_t)(num_sms() / 2) * 256 * 256 * 4);
  }
  p.bytes = at;
  return p;
}

// C [M, N] (+ add) over K, in `splits` parts where the tiles are few
static int product(const Operand& A, const Operand& B, int64_t M, int64_t N, int64_t K, int planes, void* C, int64_t ldc, int bf16,
                   const float* add, float* split_ws, cudaStream_t s, const char* what) {
  Loop lp = {};
  lp.bf16 = 1;
  lp.group_m = 16;
  lp.splits = splits_for(M, N, K);
  const int64_t nk = ceil_div(K, BK);
  lp.splits = (int)ceil_div(nk, ceil_div(nk, lp.splits));
  StoreEpi::Args a = {C, add, ldc, N, 0, M, N, bf16};
  const int splits = lp.splits;
  if (splits > 1) a = {split_ws, nullptr, N, N, M * N, M, N, 0};
  int rc;
  rc = launch<StoreEpi>(A, B, M, N, K, 1, planes, M > 128 && N > 128, lp, a, s, what);
  if (rc || splits == 1) return rc;
  const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(M * N, 256), (int64_t)num_sms() * 16);
  join_splits_kernel<<<grid, 256, 0, s>>>(split_ws, splits, M * N, N, add, C, bf16, ldc);
  return check_launch(what);
}

static int check(const char* what, int dtype, const void* x, int64_t ldx, const void* w, int64_t ldw, int w_dn, const void* labels,
                 int label_dtype, int64_t N, int64_t D, int64_t V, void* ws, size_t ws_bytes, size_t need) {
  if (label_dtype != B200_I64 && label_dtype != B200_I32) {
    set_error("%s: labels of dtype %d (int32 and int64)", what, label_dtype);
    return B200_ERR_DTYPE;
  }
  B200_REQUIRE(N == 0 || (x && labels), "%s: null tensor", what);
  B200_REQUIRE(w, "%s: null weight", what);
  B200_REQUIRE(ldx >= D && ldw >= (w_dn ? V : D), "%s: row stride below the row", what);
  B200_REQUIRE(need == 0 || (ws && ws_bytes >= need && (reinterpret_cast<uintptr_t>(ws) & 255) == 0),
               "%s: workspace of %zu bytes, %zu needed (256-byte aligned)", what, ws_bytes, need);
  return B200_OK;
}

static int check_sizes(const char* what, int dtype, int64_t N, int64_t D, int64_t V) {
  if (dtype != B200_F32 && dtype != B200_BF16) {
    set_error("%s: operands of dtype %d (fp32 and bf16)", what, dtype);
    return B200_ERR_DTYPE;
  }
  B200_REQUIRE(N >= 0 && D >= 1 && V >= 1, "%s: %lld tokens, %lld features, %lld words", what, (long long)N, (long long)D, (long long)V);
  B200_REQUIRE(N < (1ll << 30) && D < (1ll << 30) && V < (1ll << 30), "%s: a size of 2^30 or more", what);
  return B200_OK;
}

// operands of the logits' product for columns [first, first + width) of w
static Operand w_columns(const Plan& p, const void* w, int64_t ldw, int64_t first) {
  Operand o;
  o.base = reinterpret_cast<const __nv_bfloat16*>(w) + (p.w_dn ? first : first * ldw);
  o.ld = ldw;
  o.plane_stride = p.w_rows * ldw;
  o.mn = p.w_dn;
  return o;
}

}  // namespace lx
}  // namespace b200

using namespace b200;

extern "C" size_t b200_linear_xent_workspace_bytes(int dtype, const void* x, int64_t ldx, const void* w, int64_t ldw, int w_dn, int64_t N,
                                                   int64_t D, int64_t V) {
  if (lx::check_sizes("linear_cross_entropy", dtype, N, D, V) || N == 0) return 0;
  return lx::plan(false, dtype, x, ldx, w, ldw, w_dn != 0, N, D, V).bytes;
}

extern "C" size_t b200_linear_xent_grad_workspace_bytes(int dtype, const void* x, int64_t ldx, const void* w, int64_t ldw, int w_dn,
                                                        int64_t N, int64_t D, int64_t V) {
  if (lx::check_sizes("linear_cross_entropy_grad", dtype, N, D, V) || N == 0) return 0;
  return lx::plan(true, dtype, x, ldx, w, ldw, w_dn != 0, N, D, V).bytes;
}

extern "C" int b200_linear_xent(int dtype, const void* x, int64_t ldx, const void* w, int64_t ldw, int w_dn, const void* labels,
                                int label_dtype, int64_t ignore_index, float* loss, float* lse, int64_t N, int64_t D, int64_t V,
                                void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "linear_cross_entropy";
  int rc = lx::check_sizes(what, dtype, N, D, V);
  if (rc) return rc;
  const lx::Plan p = lx::plan(false, dtype, x, ldx, w, ldw, w_dn != 0, N, D, V);
  rc = lx::check(what, dtype, x, ldx, w, ldw, w_dn, labels, label_dtype, N, D, V, workspace, workspace_bytes, N ? p.bytes : 0);
  if (rc || N == 0) return rc;
  B200_REQUIRE(loss && lse, "%s: null result", what);
  cudaStream_t s = as_stream(stream);
  uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
  const int i32 = label_dtype == B200_I32;
  if (p.few) {
    lx::few::Args f = {x, w, labels, nullptr, nullptr, ldx, ldw, ignore_index, i32, (int)N, (int)D, (int)V,
                       reinterpret_cast<float2*>(ws + p.part), reinterpret_cast<float*>(ws + p.picked), nullptr, nullptr, 0};
    if ((rc = lx::few::run(dtype, f, p.w_dn, p.wide, false, nullptr, 0, s, what))) return rc;
    lx::lse_join_kernel<<<1, 32 * lx::JOIN, 0, s>>>(f.part, (int)p.parts, f.picked, labels, i32, ignore_index, loss, lse, N, V);
    return check_launch(what);
  }
  if (lx::needs_pack(dtype, x, ldx)) {
    auto* out = reinterpret_cast<__nv_bfloat16*>(ws + p.x);
    if ((rc = lx::pack(dtype, x, ldx, out, N, D, nullptr, 0, 0, 0, s))) return rc;
    x = out, ldx = lx::up8(D);
  }
  if (lx::needs_pack(dtype, w, ldw)) {
    auto* out = reinterpret_cast<__nv_bfloat16*>(ws + p.w);
    if ((rc = lx::pack(dtype, w, ldw, out, p.w_rows, p.w_cols, nullptr, 0, 0, 0, s))) return rc;
    w = out, ldw = lx::up8(p.w_cols);
  }
  auto* part = reinterpret_cast<float2*>(ws + p.part);
  float* picked = reinterpret_cast<float*>(ws + p.picked);
  tile::Operand A, B = lx::w_columns(p, w, ldw, 0);
  A.base = x, A.ld = ldx, A.plane_stride = N * ldx;
  tile::Loop lp = {};
  lp.bf16 = 1;
  lp.group_m = 16;
  const int width = p.planes > 1 && N <= 128 ? 64 : 128;  // fp32 operands on single CTAs: 128-wide tiles
  const lx::LseEpi::Args a = {part, width, picked, labels, i32, N, V};
  // a pair's 256 rows; one CTA's 128 when there are no more tokens than that
  rc = tile::launch<lx::LseEpi>(A, B, N, V, D, 1, p.planes, N > 128, lp, a, s, what);
  if (rc) return rc;
  lx::lse_join_kernel<<<(unsigned)ceil_div(N, 32), 32 * lx::JOIN, 0, s>>>(part, (int)(ceil_div(V, 2 * width) * 2), picked, labels, i32, ignore_index, loss,
                                                                lse, N, V);
  return check_launch(what);
}

extern "C" int b200_linear_xent_grad(int dtype, const float* dloss, const void* x, int64_t ldx, const void* w, int64_t ldw, int w_dn,
                                     const void* labels, int label_dtype, int64_t ignore_index, const float* lse, void* dx, void* dw,
                                     int64_t N, int64_t D, int64_t V, void* workspace, size_t workspace_bytes, void* stream) {
  return b200_linear_xent_grad_mixed(dtype, dloss, x, ldx, w, ldw, w_dn, labels, label_dtype, ignore_index, lse, dx, dtype, dw, dtype, N, D,
                                     V, workspace, workspace_bytes, stream);
}

extern "C" int b200_linear_xent_grad_mixed(int dtype, const float* dloss, const void* x, int64_t ldx, const void* w, int64_t ldw, int w_dn,
                                           const void* labels, int label_dtype, int64_t ignore_index, const float* lse, void* dx,
                                           int dx_dtype, void* dw, int dw_dtype, int64_t N, int64_t D, int64_t V, void* workspace,
                                           size_t workspace_bytes, void* stream) {
  const char* what = "linear_cross_entropy_grad";
  int rc = lx::check_sizes(what, dtype, N, D, V);
  if (!rc) rc = lx::check_sizes(what, dx_dtype, N, D, V);
  if (!rc) rc = lx::check_sizes(what, dw_dtype, N, D, V);
  if (rc) return rc;
  w_dn = w_dn != 0;
  const lx::Plan p = lx::plan(true, dtype, x, ldx, w, ldw, w_dn, N, D, V);
  rc = lx::check(what, dtype, x, ldx, w, ldw, w_dn, labels, label_dtype, N, D, V, workspace, workspace_bytes, N ? p.bytes : 0);
  if (rc) return rc;
  cudaStream_t s = as_stream(stream);
  const int64_t size = dw_dtype == B200_F32 ? 4 : 2;
  if (N == 0) {
    if (dw && cudaMemsetAsync(dw, 0, (size_t)(D * V * size), s) != cudaSuccess) return check_launch(what);
    return B200_OK;
  }
  B200_REQUIRE(dloss && lse, "%s: null tensor", what);
  B200_REQUIRE(dx || dw, "%s: no result asked for", what);
  uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
  const int i32 = label_dtype == B200_I32, dx_bf16 = dx_dtype == B200_BF16, dw_bf16 = dw_dtype == B200_BF16;
  if (p.few) {
    lx::few::Args f = {x, w, labels, dloss, lse, ldx, ldw, ignore_index, i32, (int)N, (int)D, (int)V,
                       nullptr, nullptr, reinterpret_cast<float*>(ws + p.d), dw, dw_bf16};
    // dw is written dense: its rows too have to take vectors
    const int wide = p.wide && reinterpret_cast<uintptr_t>(dw) % (dw_bf16 ? 8 : 16) == 0;
    float* part = dx ? reinterpret_cast<float*>(ws + p.split) : nullptr;
    if ((rc = lx::few::run(dtype, f, w_dn, wide, true, part, p.slices, s, what)) || !dx) return rc;
    lx::few::join_slices_kernel<<<(unsigned)ceil_div(N * D, 32), 1024, 0, s>>>(part, (int)p.slices, N * D, dx, dx_bf16);
    return check_launch(what);
  }
  auto* xg = reinterpret_cast<__nv_bfloat16*>(ws + p.xg);
  const int64_t ldg = lx::up8(D);
  // (their logits come out as zeros, which gives no gradient either)
  if ((rc = lx::pack(dtype, x, ldx, xg, N, D, labels, i32, ignore_index, V, s))) return rc;
  if (lx::needs_pack(dtype, w, ldw)) {
    auto* out = reinterpret_cast<__nv_bfloat16*>(ws + p.w);
    if ((rc = lx::pack(dtype, w, ldw, out, p.w_rows, p.w_cols, nullptr, 0, 0, 0, s))) return rc;
    w = out, ldw = lx::up8(p.w_cols);
  }
  auto* d = reinterpret_cast<__nv_bfloat16*>(ws + p.d);
  float* acc = reinterpret_cast<float*>(ws + p.acc);
  float* split = reinterpret_cast<float*>(ws + p.split);
  tile::Operand X;
  X.base = xg, X.ld = ldg, X.plane_stride = N * ldg;
  for (int64_t first = 0; first < V; first += p.width) {
    const int64_t width = std::min(p.width, V - first);
    const tile::Operand W = lx::w_columns(p, w, ldw, first);
    tile::Loop lp = {};
    lp.bf16 = 1;
    lp.group_m = 16;
    lx::GradEpi::Args a = {{}, p.planes, dloss, lse, labels, i32, ignore_index, N, V, first};
    if (!tc::make_store_map(&a.map, d, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, width, N, p.planes, 1, p.width, N * p.width, 0)) {
      set_error("%s: no tensor map for the logits' gradient (%lld x %lld)", what, (long long)N, (long long)width);
      return B200_ERR_CUDA;
    }
    rc = tile::launch<lx::GradEpi>(X, W, N, width, D, 1, p.planes, N > 128, lp, a, s, what);
    if (rc) return rc;
    tile::Operand Dk, Dm;  // d as [N, width] with the tokens, or the columns, as its major axis
    Dk.base = Dm.base = d, Dk.ld = Dm.ld = p.width, Dk.plane_stride = Dm.plane_stride = N * p.width;
    Dm.mn = 1;
    if (dx) {
      // dx (+)= d w^T over the piece: w's features are the result's columns
      for (int64_t c = 0; c < width; c += p.words) {
        const int64_t n = std::min(p.words, width - c);
        tile::Operand Wt = lx::w_columns(p, w, ldw, first + c);
        Wt.mn = !w_dn;
        Dk.base = d + c;
        const bool last = first + c + n >= V;
        rc = lx::product(Dk, Wt, N, D, n, p.planes, last ? dx : acc, D, last ? dx_bf16 : 0, first + c ? acc : nullptr, split, s, what);
        if (rc) return rc;
      }
    }
    if (dw) {
      tile::Operand Xm = X;
      Xm.mn = 1;
      uint8_t* out = reinterpret_cast<uint8_t*>(dw) + (w_dn ? first : first * D) * size;
      float* sums = reinterpret_cast<float*>(ws + p.dw_acc);
      for (int64_t t = 0; t < N; t += p.tokens) {
        const int64_t n = std::min(p.tokens, N - t);
        const bool last = t + n >= N;
        void* to = last ? static_cast<void*>(out) : sums;
        const float* add = t ? sums : nullptr;
        Xm.base = xg + t * ldg, Dm.base = d + t * p.width;
        rc = w_dn ? lx::product(Xm, Dm, D, width, n, p.planes, to, last ? V : width, last ? dw_bf16 : 0, add, split, s, what)
                  : lx::product(Dm, Xm, width, D, n, p.planes, to, D, last ? dw_bf16 : 0, add, split, s, what);
        if (rc) return rc;
      }
    }
  }
  return B200_OK;
}
