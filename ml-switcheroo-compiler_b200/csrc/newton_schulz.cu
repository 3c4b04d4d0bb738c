// Orthogonalising a matrix by Newton-Schulz products, and the optimizer step that uses it.
//
//   X0 = G / (|G|_F + eps);  each step: S = X X^T, P = b S + c S S, X <- a X + P X
// (X X^T for rows <= cols, X^T X and X <- a X + X P otherwise: the Gram matrix of the
// shorter side, without a transpose). Step update: m' = mu m + g, G = g + mu m' (Nesterov)
// or m', p' = p (1 - lr wd) - lr sqrt(max(1, rows / cols)) X.
//
// Per step 3 products on the tensor cores (tc_tile.cuh). S and P are symmetric: only the
// tiles on and above the diagonal are computed, each written twice, so a step costs
// 3 m^2 n + m^3 flop (m the shorter side) instead of 4 m^2 n + 2 m^3.
// Precision. The iterates live in fp16, scaled by 2^8: |X|_F = 1 at the start and the
// singular values stay below about 1.3, so no entry can pass 2^9 while entries of 2^-20
// of the largest keep their bits. bf16 matrices take one fp16 plane (11 bits: 2e-3 of the
// result after 5 steps, below bf16's own rounding; with bf16 iterates it is 2e-2). fp32
// matrices take two planes, hi + lo (22 bits), three products: 2e-6, as with fp32 products.
// Where eps outweighs |G| the iterates start far below 1: each matrix carries a power of two
// t = 2^e >= 1, Y = 2^8 t X is what is stored, b and c are divided by t^2 and t^4, and t
// shrinks as a makes X grow. t is 1 for any |G| above eps.
// The sum of squares is in 64 bits. Every sum has a fixed order.
// Bound by the tensor cores for large matrices, by the chain of 15 launches for one small.
#include <cuda_fp16.h>

#include <cmath>

#include "tc_tile.cuh"

namespace b200 {
namespace ns {

using namespace tile;

constexpr float SCALE = 256.f;
constexpr int NORM_BLOCKS = 296, NT = 256;

__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const __half2 t = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&t);
}
__device__ __forceinline__ void unpack_f16(uint32_t u, float& a, float& b) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
  a = f.x, b = f.y;
}

constexpr int GRAM = 0, POLY = 1, NEXT = 2;

// result = cc acc + ca source, as fp16 planes (and mirrored), or out = fa add + fb result
struct NsEpi {
  struct Args {
    const __half* src;  // planes at the result's offsets, or NULL
    __half* dst;        // planes, or NULL: the last product
    int64_t ld, plane, batch;
    float ca, cc;
    int planes, mirror;
    void* out;
    const float* add;  // fp32, dense as out
    int64_t M, N;
    float fa, fb;
    int bf16;
    const int* e0;               // [batch]: the exponent of t at the start
    int e_down, e_down_next;     // how far it has shrunk, and will have after this product
    int which;                   // GRAM, POLY, NEXT
  };
  const Args& a;
  float ca, cc, fb;
  __device__ explicit NsEpi(const Args& args) : a(args) {}
  __device__ __forceinline__ void begin(const Spot& sp) {
    ca = a.ca, cc = a.cc, fb = a.fb;
    const int e0 = a.e0[sp.z];
    if (e0 == 0) return;
    const int e = max(0, e0 - a.e_down), next = a.dst ? max(0, e0 - a.e_down_next) : 0;
    if (a.which == POLY) {
      ca = ldexpf(ca, -2 * e);
      cc = ldexpf(cc, -4 * e);
    } else if (a.which == NEXT && a.dst) {
      ca = ldexpf(ca, next - e);
      cc = ldexpf(cc, next - e);
    } else if (a.which == NEXT) {
      fb = ldexpf(fb, -e);
    }
  }
  __device__ __forceinline__ void end(const Spot&) {}

  __device__ __forceinline__ void chunk(const Spot& sp, int64_t col, float (&v)[32]) {
    const int rows = (int)min((int64_t)32, a.M - sp.row0);
    const int64_t cols = min((int64_t)32, a.N - col);
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] *= cc;
    if (a.src && sp.row < a.M) {
      const __half* p = a.src + sp.z * a.batch + sp.row * a.ld + col;
      for (int k = 0; k < a.planes; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (8 * j < cols) {  // rows are padded to 8 elements
            const uint4 u = *reinterpret_cast<const uint4*>(p + k * a.plane + 8 * j);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float x, y;
              unpack_f16(w[i], x, y);
              v[8 * j + 2 * i] = fmaf(ca, x, v[8 * j + 2 * i]);
              v[8 * j + 2 * i + 1] = fmaf(ca, y, v[8 * j + 2 * i + 1]);
            }
          }
    }
    if (!a.dst) {
      const int64_t at = (sp.z * a.M + sp.row0) * a.N + col;
      if (a.add) {
        const float* p = a.add + at + sp.lane * a.N;
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = (sp.lane < rows && i < cols ? p[i] * a.fa : 0.f) + fb * v[i];
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] *= fb;
      }
      __syncwarp();
      if (a.bf16) {
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
        stage_chunk<2>(sp.buf, sp.lane, w);
        __syncwarp();
        write_chunk<2>(sp.buf, sp.lane, reinterpret_cast<uint8_t*>(reinterpret_cast<__nv_bfloat16*>(a.out) + at), a.N, rows, cols);
      } else {
        uint32_t w[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) w[i] = __float_as_uint(v[i]);
        stage_chunk<4>(sp.buf, sp.lane, w);
        __syncwarp();
        write_chunk<4>(sp.buf, sp.lane, reinterpret_cast<uint8_t*>(reinterpret_cast<float*>(a.out) + at), a.N, rows, cols);
      }
      return;
    }
    for (int k = 0; k < a.planes; ++k) {
      __half* d = a.dst + sp.z * a.batch + k * a.plane;
      uint32_t w[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) w[i] = pack_f16(v[2 * i], v[2 * i + 1]);
      __syncwarp();
      stage_chunk<2>(sp.buf, sp.lane, w);
      __syncwarp();
      write_chunk<2>(sp.buf, sp.lane, reinterpret_cast<uint8_t*>(d + sp.row0 * a.ld + col), a.ld, rows, cols);
      if (a.mirror && sp.mt != sp.nt && sp.lane < rows) {
        // the transposed tile: 32 lanes store 32 adjacent elements of each of its rows
        __half* m = d + col * a.ld + sp.row;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const __half2 h = *reinterpret_cast<const __half2*>(&w[i]);
          if (2 * i < cols) m[(2 * i) * a.ld] = __low2half(h);
          if (2 * i + 1 < cols) m[(2 * i + 1) * a.ld] = __high2half(h);
        }
      }
      if (k + 1 < a.planes) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float x, y;
          unpack_f16(w[i], x, y);
          v[2 * i] -= x;
          v[2 * i + 1] -= y;
        }
      }
    }
  }
};

__device__ __forceinline__ float value_at(const void* g, int bf16, int64_t i) {
  return bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(g)[i]) : reinterpret_cast<const float*>(g)[i];
}

// Sums of squares of each matrix, a part per block. With a momentum: m' = mu m + g is
// written and G = g + mu m' (nesterov) or m' is what is summed.
__global__ void __launch_bounds__(NT) square_kernel(const void* g, int bf16, const float* mom, float* mom_out, float mu, int nesterov,
                                                    double* part, int64_t n) {
  __shared__ double red[NT / 32];
  const int64_t base = (int64_t)blockIdx.y * n;
  double s = 0.0;
  for (int64_t i = (int64_t)blockIdx.x * NT + threadIdx.x; i < n; i += (int64_t)gridDim.x * NT) {
    float v = value_at(g, bf16, base + i);
    if (mom) {
      const float m = mu * mom[base + i] + v;
      mom_out[base + i] = m;
      v = nesterov ? v + mu * m : m;
    }
    s += (double)v * (double)v;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < NT / 32; ++i) s += red[i];
    part[(int64_t)blockIdx.y * gridDim.x + blockIdx.x] = s;
  }
}

// X0 = 2^8 G / (|G| + eps) as fp16 planes with rows padded to 8 elements
__global__ void __launch_bounds__(NT) start_kernel(const void* g, int bf16, const float* mom, float mu, int nesterov, const double* part,
                                                   int parts, float eps, int* e0, __half* x, int64_t ld, int64_t plane, int64_t batch, int planes,
                                                   int64_t rows, int64_t cols) {
  __shared__ double red[NT / 32];
  double s = 0.0;
  for (int i = threadIdx.x; i < parts; i += NT) s += part[(int64_t)blockIdx.y * parts + i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  s = red[0];
  for (int i = 1; i < NT / 32; ++i) s += red[i];
  const double norm = sqrt(s), share = norm / (norm + (double)eps);
  const int e = share > 0.0 && share < 0.5 ? min(96, -1 - ilogb(share)) : 0;  // t share in [1/2, 1)
  if (blockIdx.x == 0 && threadIdx.x == 0) e0[blockIdx.y] = e;
  const float scale = (float)(ldexp((double)SCALE, e) / (norm + (double)eps));
  const int64_t base = (int64_t)blockIdx.y * rows * cols, per = ld / 8;
  for (int64_t i = (int64_t)blockIdx.x * NT + threadIdx.x; i < rows * per; i += (int64_t)gridDim.x * NT) {
    const int64_t r = i / per, c = i % per * 8;
    float v[8];
    for (int j = 0; j < 8; ++j) {
      v[j] = 0.f;
      if (c + j < cols) {
        const int64_t at = base + r * cols + c + j;
        float t = value_at(g, bf16, at);
        if (mom) t = nesterov ? t + mu * mom[at] : mom[at];  // mom: the new momentum
        v[j] = t * scale;
      }
    }
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = pack_f16(v[2 * j], v[2 * j + 1]);
    __half* d = x + (int64_t)blockIdx.y * batch + r * ld + c;
    *reinterpret_cast<uint4*>(d) = make_uint4(w[0], w[1], w[2], w[3]);
    if (planes > 1) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float a, b;
        unpack_f16(w[j], a, b);
        w[j] = pack_f16(v[2 * j] - a, v[2 * j + 1] - b);
      }
      *reinterpret_cast<uint4*>(d + plane) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

static int64_t up8(int64_t v) { return (v + 7) / 8 * 8; }
static size_t align256(size_t v) { return (v + 255) & ~size_t(255); }

struct Plan {
  int planes;
  int64_t side, ldx, ldg, xn, gn;  // shorter side; row strides and sizes of one X and one Gram plane
  size_t x0, x1, s, p, part, e0, bytes;
};

static Plan plan(int dtype, int64_t batch, int64_t rows, int64_t cols) {
  Plan q = {};
  q.planes = dtype == B200_F32 ? 2 : 1;
  q.side = std::min(rows, cols);
  q.ldx = up8(cols);
  q.ldg = up8(q.side);
  q.xn = rows * q.ldx;
  q.gn = q.side * q.ldg;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at = align256(at + bytes);
    return here;
  };
  const size_t xb = (size_t)batch * q.planes * q.xn * 2, gb = (size_t)batch * q.planes * q.gn * 2;
  q.x0 = take(xb), q.x1 = take(xb), q.s = take(gb), q.p = take(gb);
  q.part = take((size_t)batch * NORM_BLOCKS * 8);
  q.e0 = take((size_t)batch * 4);
  q.bytes = at;
  return q;
}

// One product, on CTA pairs (256 x 256 tiles) when those alone fill two thirds of them, else
// on 128 x 128 tiles of single CTAs: a 1024 x 1024 product has 16 of the former (10 above
// the diagonal) for 74 pairs, 64 (36) of the latter.
static int product(const Operand& A, const Operand& B, int64_t M, int64_t N, int64_t K, int64_t batch, int planes, bool triangle,
                   const NsEpi::Args& a, cudaStream_t s, const char* what) {
  Loop lp = {};
  lp.group_m = 16;
  lp.walk = triangle ? WALK_TRIANGLE : WALK_GROUPED;
  const int64_t tm = ceil_div(M, 256), tn = ceil_div(N, 256);
  const int64_t tiles = (triangle ? tn * (tn + 1) / 2 : tm * tn) * batch;
  if (M > 128 && N > 128 && tiles * 3 >= num_sms()) return launch<256, true, NsEpi>(A, B, M, N, K, batch, planes, lp, a, s, what);
  return launch<128, false, NsEpi>(A, B, M, N, K, batch, planes, lp, a, s, what);
}

struct Finish {  // out = fa add + fb X
  void* out;
  const float* add;
  float fa, fb;
  int bf16;
};

static int run(const Plan& q, const void* g, int dtype, const float* mom, float* mom_out, float mu, int nesterov, const Finish& f,
               int64_t batch, int64_t rows, int64_t cols, const float* coef, int steps, float eps, void* workspace, cudaStream_t s,
               const char* what) {
  uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
  __half* x[2] = {reinterpret_cast<__half*>(ws + q.x0), reinterpret_cast<__half*>(ws + q.x1)};
  __half *S = reinterpret_cast<__half*>(ws + q.s), *P = reinterpret_cast<__half*>(ws + q.p);
  double* part = reinterpret_cast<double*>(ws + q.part);
  int* e0 = reinterpret_cast<int*>(ws + q.e0);
  const int64_t n = rows * cols;
  const int parts = (int)std::min<int64_t>(NORM_BLOCKS, ceil_div(n, NT * 8));
  const int bf16 = dtype == B200_BF16;
  square_kernel<<<dim3((unsigned)parts, (unsigned)batch), NT, 0, s>>>(g, bf16, mom, mom_out, mu, nesterov, part, n);
  int rc = check_launch(what);
  if (rc) return rc;
  const int64_t xb = q.planes * q.xn, gb = q.planes * q.gn;
  const unsigned gx = (unsigned)std::min<int64_t>(ceil_div(rows * (q.ldx / 8), NT), 4 * num_sms());
  start_kernel<<<dim3(gx, (unsigned)batch), NT, 0, s>>>(g, bf16, mom ? mom_out : nullptr, mu, nesterov, part, parts, eps, e0, x[0], q.ldx, q.xn,
                                                        xb, q.planes, rows, cols);
  if ((rc = check_launch(what))) return rc;
  const bool tall = rows > cols;
  double grown = 0.0;  // log2 of how far a has made the smallest X grow
  for (int i = 0; i < steps; ++i) {
    const float a = coef[3 * i], b = coef[3 * i + 1], c = coef[3 * i + 2];
    Operand X, Gm;
    X.base = x[i & 1], X.ld = q.ldx, X.plane_stride = q.xn, X.batch_stride = xb, X.mn = tall;
    Gm.ld = q.ldg, Gm.plane_stride = q.gn, Gm.batch_stride = gb;
    NsEpi::Args e = {};
    e.e0 = e0;
    e.e_down = (int)std::floor(grown);
    grown += std::max(0.0, std::log2((double)std::fabs(a)));
    e.e_down_next = (int)std::floor(grown);
    e.which = GRAM;
    e.planes = q.planes;
    e.M = e.N = q.side;
    e.ld = q.ldg, e.plane = q.gn, e.batch = gb;
    e.cc = 1.f / SCALE;
    e.mirror = 1;
    e.dst = S;
    rc = product(X, X, q.side, q.side, tall ? rows : cols, batch, q.planes, true, e, s, what);
    if (rc) return rc;
    e.which = POLY;
    e.src = S, e.dst = P, e.ca = b, e.cc = c / SCALE;
    Gm.base = S;
    rc = product(Gm, Gm, q.side, q.side, q.side, batch, q.planes, true, e, s, what);
    if (rc) return rc;
    Gm.base = P;
    const bool last = i + 1 == steps;
    NsEpi::Args r = {};
    r.e0 = e0, r.e_down = e.e_down, r.e_down_next = e.e_down_next, r.which = NEXT;
    r.planes = q.planes;
    r.M = rows, r.N = cols;
    r.ld = q.ldx, r.plane = q.xn, r.batch = xb;
    r.src = x[i & 1], r.ca = a, r.cc = 1.f / SCALE;
    r.dst = last ? nullptr : x[(i + 1) & 1];
    r.out = f.out, r.add = f.add, r.fa = f.fa, r.fb = f.fb / SCALE, r.bf16 = f.bf16;
    // P X (wide: X's columns are the result's) or X P (tall); P's rows serve as its columns
    Operand Xo = X;
    Xo.mn = tall ? 0 : 1;
    rc = tall ? product(Xo, Gm, rows, cols, q.side, batch, q.planes, false, r, s, what)
              : product(Gm, Xo, rows, cols, q.side, batch, q.planes, false, r, s, what);
    if (rc) return rc;
  }
  return B200_OK;
}

static int check(const char* what, int64_t batch, int64_t rows, int64_t cols, const float* coef, int steps, float eps, void* ws,
                 size_t bytes, size_t need) {
  B200_REQUIRE(batch >= 0 && rows >= 0 && cols >= 0, "%s: negative size", what);
  B200_REQUIRE(batch <= 65535 && rows < (1 << 24) && cols < (1 << 24), "%s: %lld matrices of %lld x %lld are too many or too large", what,
               (long long)batch, (long long)rows, (long long)cols);
  B200_REQUIRE(coef && steps >= 1 && steps <= 100, "%s: %d steps not in [1, 100], or no coefficients", what, steps);
  B200_REQUIRE(eps >= 0.f, "%s: eps %g is negative", what, (double)eps);
  B200_REQUIRE(need == 0 || (ws && bytes >= need), "%s: workspace of %zu bytes, %zu needed", what, bytes, need);
  return B200_OK;
}

}  // namespace ns
}  // namespace b200

using namespace b200;

extern "C" size_t b200_newton_schulz_workspace_bytes(int dtype, int64_t batch, int64_t rows, int64_t cols) {
  if (batch <= 0 || rows <= 0 || cols <= 0 || batch > 65535 || rows >= (1 << 24) || cols >= (1 << 24)) return 0;
  return ns::plan(dtype, batch, rows, cols).bytes;
}

extern "C" int b200_newton_schulz(int dtype, const void* g, void* out, int64_t batch, int64_t rows, int64_t cols, const float* coefficients,
                                  int steps, float eps, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "newton_schulz";
  if (dtype != B200_F32 && dtype != B200_BF16) {
    set_error("%s: dtype %d (fp32 and bf16)", what, dtype);
    return B200_ERR_DTYPE;
  }
  int rc = ns::check(what, batch, rows, cols, coefficients, steps, eps, workspace, workspace_bytes,
                     b200_newton_schulz_workspace_bytes(dtype, batch, rows, cols));
  if (rc || batch == 0 || rows == 0 || cols == 0) return rc;
  B200_REQUIRE(g && out, "%s: null tensor", what);
  const ns::Plan q = ns::plan(dtype, batch, rows, cols);
  const ns::Finish f = {out, nullptr, 0.f, 1.f, dtype == B200_BF16};
  return ns::run(q, g, dtype, nullptr, nullptr, 0.f, 0, f, batch, rows, cols, coefficients, steps, eps, workspace, as_stream(stream), what);
}

extern "C" int b200_apply_muon_f32(const float* param, const float* momentum, const float* grad, float* param_out, float* momentum_out,
                                   int64_t batch, int64_t rows, int64_t cols, float lr, float mu, int nesterov, float weight_decay,
                                   const float* coefficients, int steps, float eps, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "apply_muon";
  int rc = ns::check(what, batch, rows, cols, coefficients, steps, eps, workspace, workspace_bytes,
                     b200_newton_schulz_workspace_bytes(B200_F32, batch, rows, cols));
  if (rc || batch == 0 || rows == 0 || cols == 0) return rc;
  B200_REQUIRE(param && momentum && grad && param_out && momentum_out, "%s: null tensor", what);
  const ns::Plan q = ns::plan(B200_F32, batch, rows, cols);
  const float tall = rows > cols ? sqrtf((float)((double)rows / (double)cols)) : 1.f;
  const ns::Finish f = {param_out, param, 1.f - lr * weight_decay, -lr * tall, 0};
  return ns::run(q, grad, B200_F32, momentum, momentum_out, mu, nesterov != 0, f, batch, rows, cols, coefficients, steps, eps, workspace,
                 as_stream(stream), what);
}
