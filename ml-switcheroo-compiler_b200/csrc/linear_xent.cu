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
// Rows whose label is ignore_index: loss 0, no gradient, and the row of x they hold is
// replaced by zeros where dw is made, so whatever it contains stays out.
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
    if (l == a.ignore || l < 0 || l >= a.V) return;
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
  __device__ __forceinline__ void init(const Spot& sp, int64_t col, float (&v)[32]) {
    if (a.add && sp.row < a.M) {
      const float* p = a.add + sp.row * a.ld_add + col;
      if (col + 32 <= a.N && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          const float4 t = *reinterpret_cast<const float4*>(p + i);
          v[i] = t.x, v[i + 1] = t.y, v[i + 2] = t.z, v[i + 3] = t.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (col + i < a.N) v[i] = p[i];
      }
    }
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
// fp32 split into two bf16 planes. With labels, the rows of ignored tokens become zeros.
template <bool F32>
__global__ void __launch_bounds__(256) pack_kernel(const void* __restrict__ src, int64_t ld, __nv_bfloat16* __restrict__ out, int64_t ldo,
                                                   int64_t plane, int64_t rows, int64_t cols, const void* labels, int labels_i32,
                                                   int64_t ignore) {
  const int64_t per = ldo / 8, total = rows * per;  // 8 elements a thread
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per, c = i % per * 8;
    const bool zero = labels && label_at(labels, labels_i32, r) == ignore;
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
                int64_t ignore, cudaStream_t s) {
  const int64_t ldo = up8(cols), total = rows * (ldo / 8);
  const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(total, 256), (int64_t)num_sms() * 16);
  if (dtype == B200_F32)
    pack_kernel<true><<<grid, 256, 0, s>>>(src, ld, out, ldo, rows * ldo, rows, cols, labels, labels_i32, ignore);
  else
    pack_kernel<false><<<grid, 256, 0, s>>>(src, ld, out, ldo, rows * ldo, rows, cols, labels, labels_i32, ignore);
  return check_launch("linear_cross_entropy pack");
}

// Sizes of one call and where its scratch lies in the workspace (offsets in bytes)
struct Plan {
  int64_t N, D, V;
  int planes, w_dn;       // w_dn: w is stored [D, V] (V adjacent), else [V, D]
  int64_t w_rows, w_cols; // of the stored matrix
  size_t x, w, part, picked, d, xg, acc, split, bytes;
  int64_t width;          // columns of one piece
};

static size_t align256(size_t v) { return (v + 255) & ~size_t(255); }

constexpr size_t PIECE_BYTES = size_t(512) << 20;

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
  const size_t xb = (size_t)p.planes * N * up8(D) * 2;
  // the forward product reads x as it is where it can; dw's operand has the ignored rows zeroed
  if (needs_pack(dtype, x, ldx)) p.x = take(xb);
  if (needs_pack(dtype, w, ldw)) p.w = take((size_t)p.planes * p.w_rows * up8(p.w_cols) * 2);
  if (!grad) {
    p.part = take((size_t)ceil_div(V, p.planes > 1 && N <= 128 ? 128 : 256) * 2 * N * sizeof(float2));
    p.picked = take((size_t)N * 4);
  } else {
    p.width = piece_width(N, D, V, p.planes);
    p.d = take((size_t)p.planes * N * p.width * 2);
    p.xg = take(xb);
    if (p.width < V) p.acc = take((size_t)N * D * 4);
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
  B200_REQUIRE(ws_bytes >= need && (need == 0 || ws), "%s: workspace of %zu bytes, %zu needed", what, ws_bytes, need);
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
  if (lx::needs_pack(dtype, x, ldx)) {
    auto* out = reinterpret_cast<__nv_bfloat16*>(ws + p.x);
    if ((rc = lx::pack(dtype, x, ldx, out, N, D, nullptr, 0, 0, s))) return rc;
    x = out, ldx = lx::up8(D);
  }
  if (lx::needs_pack(dtype, w, ldw)) {
    auto* out = reinterpret_cast<__nv_bfloat16*>(ws + p.w);
    if ((rc = lx::pack(dtype, w, ldw, out, p.w_rows, p.w_cols, nullptr, 0, 0, s))) return rc;
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
  const char* what = "linear_cross_entropy_grad";
  int rc = lx::check_sizes(what, dtype, N, D, V);
  if (rc) return rc;
  w_dn = w_dn != 0;
  const lx::Plan p = lx::plan(true, dtype, x, ldx, w, ldw, w_dn, N, D, V);
  rc = lx::check(what, dtype, x, ldx, w, ldw, w_dn, labels, label_dtype, N, D, V, workspace, workspace_bytes, N ? p.bytes : 0);
  if (rc) return rc;
  cudaStream_t s = as_stream(stream);
  const int64_t size = dtype == B200_F32 ? 4 : 2;
  if (N == 0) {
    if (dw && cudaMemsetAsync(dw, 0, (size_t)(D * V * size), s) != cudaSuccess) return check_launch(what);
    return B200_OK;
  }
  B200_REQUIRE(dloss && lse, "%s: null tensor", what);
  B200_REQUIRE(dx || dw, "%s: no result asked for", what);
  uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
  const int i32 = label_dtype == B200_I32, bf16 = dtype == B200_BF16;
  auto* xg = reinterpret_cast<__nv_bfloat16*>(ws + p.xg);
  const int64_t ldg = lx::up8(D);
  if (dw && (rc = lx::pack(dtype, x, ldx, xg, N, D, labels, i32, ignore_index, s))) return rc;
  if (lx::needs_pack(dtype, x, ldx)) {
    auto* out = reinterpret_cast<__nv_bfloat16*>(ws + p.x);
    if ((rc = lx::pack(dtype, x, ldx, out, N, D, nullptr, 0, 0, s))) return rc;
    x = out, ldx = ldg;
  }
  if (lx::needs_pack(dtype, w, ldw)) {
    auto* out = reinterpret_cast<__nv_bfloat16*>(ws + p.w);
    if ((rc = lx::pack(dtype, w, ldw, out, p.w_rows, p.w_cols, nullptr, 0, 0, s))) return rc;
    w = out, ldw = lx::up8(p.w_cols);
  }
  auto* d = reinterpret_cast<__nv_bfloat16*>(ws + p.d);
  float* acc = reinterpret_cast<float*>(ws + p.acc);
  float* split = reinterpret_cast<float*>(ws + p.split);
  tile::Operand X;
  X.base = x, X.ld = ldx, X.plane_stride = N * ldx;
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
      tile::Operand Wt = W;
      Wt.mn = !w_dn;
      const bool last = first + width >= V;
      rc = lx::product(Dk, Wt, N, D, width, p.planes, last ? dx : acc, D, last ? bf16 : 0, first ? acc : nullptr, split, s, what);
      if (rc) return rc;
    }
    if (dw) {
      tile::Operand Xm;
      Xm.base = xg, Xm.ld = ldg, Xm.plane_stride = N * ldg, Xm.mn = 1;
      uint8_t* out = reinterpret_cast<uint8_t*>(dw) + (w_dn ? first : first * D) * size;
      rc = w_dn ? lx::product(Xm, Dm, D, width, N, p.planes, out, V, bf16, nullptr, split, s, what)
                : lx::product(Dm, Xm, width, D, N, p.planes, out, D, bf16, nullptr, split, s, what);
      if (rc) return rc;
    }
  }
  return B200_OK;
}
