// A block's output added to the residual stream, with the norms on either side of the sum:
//
//   p = post_norm ? N(f; post_gamma, post_beta) : f        the block's output f, normed
//   s = scale x + gate p                                   the new residual stream
//   h = N(s; gamma, beta)                                  what the next block reads
//
// N is the RMS norm  t rstd gamma, rstd = 1 / sqrt(mean(t^2) + eps),  or the layer norm, which
// takes the mean from t first and adds beta. The gate is one value per channel, per channel and
// group of rows (a sequence), or per element. With u = the normed row before gamma, the gradient
// of a norm is  dt = rstd (d - [mean d] - u mean(d u)),  d = dy gamma, so
//
//   ds = ds' + rstd_s (t - [mean t] - u_s mean(t u_s)), t = dh gamma;  dx = scale ds
//   dp = gate ds;  dgate = sum ds p;  df = dp, or the norm's gradient of dp post_gamma
//   dgamma = sum dh u_s, dbeta = sum dh, dpost_gamma = sum dp u_f, dpost_beta = sum dp
//
// One block holds one row in registers (8 elements a thread and register set) and walks its rows;
// the next row's loads are issued before the current one's reductions. Everything is fp32 between
// one load and one rounding per output; h is made of the sum before its rounding, and the
// gradient makes the sums again from x and f. Bound by HBM: each array is read or written once.
// The weights' gradients are kept per thread over the block's rows (a thread owns columns), go to
// the workspace once a block, and are added up in a fixed order by a second launch; a gate's
// gradient whose group one block covers alone is written by that block.
#include <algorithm>

#include "common.cuh"

namespace b200 {
namespace rnorm {

constexpr int MAX_THREADS = 512, MAX_COLS = MAX_THREADS * 8 * 4;

struct Args {
  // weights that were not given point at another one, or at x, and are not asked for: no address is null
  const void *x, *f, *gate, *gamma, *beta, *post_gamma, *post_beta;
  int has_gate, has_gamma, has_beta, has_post_gamma, has_post_beta;
  const void *ds, *dh;                  // gradient only
  void *out0, *out1;                    // s and h, or dx and df
  float* part;                          // [blocks][weights][cols]
  float* gate_part;                     // [groups][chunks][cols] (chunks > 1)
  void* dgate;                          // written here where chunks == 1
  int64_t rows, groups, per_group;      // per_group = rows / groups
  int64_t chunks, per_chunk;            // a group's rows are cut into chunks
  int cols;
  int x_bf16, f_bf16, w_bf16, gate_bf16;
  float scale, eps;
};

// Where a thread's element i (of 8 NV) of a row is: vectors of 8 neighbours, or one column in
// blockDim where rows are no multiple of 8 elements or not aligned.
template <int V>
__device__ __forceinline__ int column(int i) {
  if constexpr (V == 8) return ((i >> 3) * (int)blockDim.x + (int)threadIdx.x) * 8 + (i & 7);
  else return i * (int)blockDim.x + (int)threadIdx.x;
}

// 8 NV elements of one row as they are in memory (two register sets of four words per 8 fp32)
template <int V, int NV>
struct Raw {
  uint4 w[V == 8 ? NV * 2 : 1];
  float s[V == 8 ? 1 : NV * 8];

  __device__ __forceinline__ void load(const void* base, int64_t row, int cols, int bf16) {
    if constexpr (V == 8) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int c = column<V>(8 * v);
        if (c < cols) {
          if (bf16) {
            w[2 * v] = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(base) + row * cols + c));
          } else {
            const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(base) + row * cols + c);
            w[2 * v] = __ldg(p);
            w[2 * v + 1] = __ldg(p + 1);
          }
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8 * NV; ++i) {
        const int c = column<V>(i);
        if (c < cols)
          s[i] = bf16 ? __bfloat162float(__ldg(reinterpret_cast<const __nv_bfloat16*>(base) + row * cols + c))
                      : __ldg(reinterpret_cast<const float*>(base) + row * cols + c);
      }
    }
  }
  // as fp32; zeros behind the row's end
  __device__ __forceinline__ void get(float (&o)[8 * NV], int cols, int bf16) const {
    if constexpr (V == 8) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const bool in = column<V>(8 * v) < cols;
        const uint32_t a[8] = {w[2 * v].x, w[2 * v].y, w[2 * v].z, w[2 * v].w, w[2 * v + 1].x, w[2 * v + 1].y, w[2 * v + 1].z, w[2 * v + 1].w};
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t b = bf16 ? ((k & 1) ? a[k >> 1] & 0xFFFF0000u : a[k >> 1] << 16) : a[k];
          o[8 * v + k] = in ? __uint_as_float(b) : 0.f;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8 * NV; ++i) o[i] = column<V>(i) < cols ? s[i] : 0.f;
    }
  }
};

template <int V, int NV>
__device__ __forceinline__ void fetch(float (&o)[8 * NV], const void* base, int64_t row, int cols, int bf16) {
  Raw<V, NV> r;
  r.load(base, row, cols, bf16);
  r.get(o, cols, bf16);
}

template <int V, int NV>
__device__ __forceinline__ void put(void* base, int64_t row, int cols, int bf16, const float (&o)[8 * NV]) {
  if constexpr (V == 8) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = column<V>(8 * v);
      if (c >= cols) continue;
      if (bf16) {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const __nv_bfloat162 t = __floats2bfloat162_rn(o[8 * v + 2 * k], o[8 * v + 2 * k + 1]);
          w[k] = *reinterpret_cast<const uint32_t*>(&t);
        }
        *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(base) + row * cols + c) = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
        float4* p = reinterpret_cast<float4*>(reinterpret_cast<float*>(base) + row * cols + c);
        p[0] = make_float4(o[8 * v], o[8 * v + 1], o[8 * v + 2], o[8 * v + 3]);
        p[1] = make_float4(o[8 * v + 4], o[8 * v + 5], o[8 * v + 6], o[8 * v + 7]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8 * NV; ++i) {
      const int c = column<V>(i);
      if (c >= cols) continue;
      if (bf16) reinterpret_cast<__nv_bfloat16*>(base)[row * cols + c] = __float2bfloat16_rn(o[i]);
      else reinterpret_cast<float*>(base)[row * cols + c] = o[i];
    }
  }
}

// Sums over the block, the same on every thread: one barrier, the area alternates between two
// halves so that the next sum may write while slow warps still read this one.
struct Sums {
  float (*area)[2][16];  // [half][value][warp]
  int half;
  __device__ __forceinline__ void operator()(float& a, float& b) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      a += __shfl_xor_sync(0xffffffffu, a, o);
      b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if (warps == 1) return;
    if (lane == 0) area[half][0][warp] = a, area[half][1][warp] = b;
    __syncthreads();
    a = b = 0.f;
    for (int w = 0; w < warps; ++w) a += area[half][0][w], b += area[half][1][w];
    half ^= 1;
  }
  __device__ __forceinline__ void operator()(float& a) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    a = warp_sum(a);
    if (warps == 1) return;
    if (lane == 0) area[half][0][warp] = a;
    __syncthreads();
    a = 0.f;
    for (int w = 0; w < warps; ++w) a += area[half][0][w];
    half ^= 1;
  }
};

// t (zeros behind the row's end) -> the normed row u before gamma; returns rstd
template <int V, int NV, bool LAYER>
__device__ __forceinline__ float unit(float (&t)[8 * NV], int cols, float eps, Sums& sums) {
  if constexpr (LAYER) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8 * NV; ++i) m += t[i];
    sums(m);
    m /= (float)cols;
#pragma unroll
    for (int i = 0; i < 8 * NV; ++i) t[i] = column<V>(i) < cols ? t[i] - m : 0.f;
  }
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < 8 * NV; ++i) q = fmaf(t[i], t[i], q);
  sums(q);
  const float rstd = 1.f / sqrtf(q / (float)cols + eps);
#pragma unroll
  for (int i = 0; i < 8 * NV; ++i) t[i] *= rstd;
  return rstd;
}

// d = dy gamma -> the gradient rstd (d - [mean d] - u mean(d u))
template <int V, int NV, bool LAYER>
__device__ __forceinline__ void unit_grad(float (&d)[8 * NV], const float (&u)[8 * NV], float rstd, int cols, Sums& sums) {
  float a = 0.f, b = 0.f;
#pragma unroll
  for (int i = 0; i < 8 * NV; ++i) {
    a = fmaf(d[i], u[i], a);
    if constexpr (LAYER) b += d[i];
  }
  if constexpr (LAYER) sums(a, b);
  else sums(a);
  a /= (float)cols;
  b /= (float)cols;
#pragma unroll
  for (int i = 0; i < 8 * NV; ++i) {
    d[i] = rstd * (d[i] - b - u[i] * a);
    if (LAYER && column<V>(i) >= cols) d[i] = 0.f;  // what a later mean adds up
  }
}

// the rows of block `b`: a group's chunk, or (chunks == 1) whole groups in turn
struct Walk {
  int64_t group, row, end, step_groups;
  __device__ __forceinline__ Walk(const Args& a) {
    if (a.chunks > 1) {
      group = blockIdx.x / a.chunks;
      const int64_t c = blockIdx.x % a.chunks;
      row = group * a.per_group + c * a.per_chunk;
      end = min(row + a.per_chunk, (group + 1) * a.per_group);
      step_groups = a.groups;
    } else {
      group = blockIdx.x;
      row = group * a.per_group;
      end = row + a.per_group;
      step_groups = gridDim.x;
    }
  }
  __device__ __forceinline__ bool more(const Args& a) const { return group < a.groups && row < end; }
  __device__ __forceinline__ void next(const Args& a) {
    if (++row < end) return;
    group += step_groups;
    row = group * a.per_group;
    end = row + a.per_group;
  }
};

template <int V, int NV, bool LAYER, bool POST>
__global__ void __launch_bounds__(MAX_THREADS) forward_kernel(const __grid_constant__ Args a) {
  __shared__ float area[2][2][16];
  Sums sums{area, 0};
  constexpr int E = 8 * NV;
  Walk w(a);
  Raw<V, NV> rx, rf;
  if (w.more(a)) {
    rx.load(a.x, w.row, a.cols, a.x_bf16);
    rf.load(a.f, w.row, a.cols, a.f_bf16);
  }
  while (w.more(a)) {
    const int64_t row = w.row, group = w.group;
    float s[E], p[E], t[E];
    rx.get(s, a.cols, a.x_bf16);
    rf.get(p, a.cols, a.f_bf16);
    w.next(a);
    if (w.more(a)) {
      rx.load(a.x, w.row, a.cols, a.x_bf16);
      rf.load(a.f, w.row, a.cols, a.f_bf16);
    }
    if constexpr (POST) {
      unit<V, NV, LAYER>(p, a.cols, a.eps, sums);
      if (a.has_post_gamma) {
        fetch<V, NV>(t, a.post_gamma, 0, a.cols, a.w_bf16);
#pragma unroll
        for (int i = 0; i < E; ++i) p[i] *= t[i];
      }
      if (LAYER && a.has_post_beta) {
        fetch<V, NV>(t, a.post_beta, 0, a.cols, a.w_bf16);
#pragma unroll
        for (int i = 0; i < E; ++i) p[i] += t[i];
      }
    }
    if (a.has_gate) {
      fetch<V, NV>(t, a.gate, group, a.cols, a.gate_bf16);
#pragma unroll
      for (int i = 0; i < E; ++i) p[i] *= t[i];
    }
#pragma unroll
    for (int i = 0; i < E; ++i) s[i] = fmaf(a.scale, s[i], p[i]);
    put<V, NV>(a.out0, row, a.cols, a.x_bf16, s);
    unit<V, NV, LAYER>(s, a.cols, a.eps, sums);
    if (a.has_gamma) {
      fetch<V, NV>(t, a.gamma, 0, a.cols, a.w_bf16);
#pragma unroll
      for (int i = 0; i < E; ++i) s[i] *= t[i];
    }
    if (LAYER && a.has_beta) {
      fetch<V, NV>(t, a.beta, 0, a.cols, a.w_bf16);
#pragma unroll
      for (int i = 0; i < E; ++i) s[i] += t[i];
    }
    put<V, NV>(a.out1, row, a.cols, a.f_bf16, s);
  }
}

// weights' gradients that a block keeps, in the order of the workspace
template <bool LAYER, bool POST>
struct Kept {
  static constexpr int N = (1 + (POST ? 1 : 0)) * (LAYER ? 2 : 1);
  static constexpr int GAMMA = 0, BETA = 1, POST_GAMMA = LAYER ? 2 : 1, POST_BETA = 3;
};

template <int V, int NV, bool LAYER, bool POST, bool GATE>
__global__ void __launch_bounds__(MAX_THREADS) gradient_kernel(const __grid_constant__ Args a) {
  using K = Kept<LAYER, POST>;
  __shared__ float area[2][2][16];
  Sums sums{area, 0};
  constexpr int E = 8 * NV;
  float kept[K::N][E], dgate[GATE ? E : 1];
#pragma unroll
  for (int n = 0; n < K::N; ++n)
#pragma unroll
    for (int i = 0; i < E; ++i) kept[n][i] = 0.f;
  constexpr bool AHEAD = NV == 1;  // wider rows have no registers for the next one
  Walk w(a);
  Raw<V, NV> rx, rf, rs, rh;
  auto load = [&]() {
    rx.load(a.x, w.row, a.cols, a.x_bf16);
    rf.load(a.f, w.row, a.cols, a.f_bf16);
    rs.load(a.ds, w.row, a.cols, a.x_bf16);
    rh.load(a.dh, w.row, a.cols, a.f_bf16);
  };
  if (AHEAD && w.more(a)) load();
  int64_t current = -1;
  while (w.more(a)) {
    const int64_t row = w.row, group = w.group;
    if constexpr (GATE) {
      if (group != current) {
        current = group;
#pragma unroll
        for (int i = 0; i < E; ++i) dgate[i] = 0.f;
      }
    }
    float s[E], p[E], ds[E], d[E], t[E];
    if constexpr (!AHEAD) load();
    rx.get(s, a.cols, a.x_bf16);
    rf.get(p, a.cols, a.f_bf16);
    rs.get(ds, a.cols, a.x_bf16);
    rh.get(d, a.cols, a.f_bf16);
    w.next(a);
    const bool last = !w.more(a) || w.group != group;  // of this group
    if (AHEAD && w.more(a)) load();
    float rstd_f = 0.f;
    float u[POST ? E : 1];
    if constexpr (POST) {
      rstd_f = unit<V, NV, LAYER>(p, a.cols, a.eps, sums);
#pragma unroll
      for (int i = 0; i < E; ++i) u[i] = p[i];
      if (a.has_post_gamma) {
        fetch<V, NV>(t, a.post_gamma, 0, a.cols, a.w_bf16);
#pragma unroll
        for (int i = 0; i < E; ++i) p[i] *= t[i];
      }
      if (LAYER && a.has_post_beta) {
        fetch<V, NV>(t, a.post_beta, 0, a.cols, a.w_bf16);
#pragma unroll
        for (int i = 0; i < E; ++i) p[i] += t[i];
      }
    }
    if constexpr (GATE) {
      fetch<V, NV>(t, a.gate, group, a.cols, a.gate_bf16);
#pragma unroll
      for (int i = 0; i < E; ++i) s[i] = fmaf(a.scale, s[i], p[i] * t[i]);
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) s[i] = fmaf(a.scale, s[i], p[i]);
    }
    const float rstd = unit<V, NV, LAYER>(s, a.cols, a.eps, sums);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      kept[K::GAMMA][i] = fmaf(d[i], s[i], kept[K::GAMMA][i]);
      if constexpr (LAYER) kept[K::BETA][i] += d[i];
    }
    if (a.has_gamma) {
      fetch<V, NV>(t, a.gamma, 0, a.cols, a.w_bf16);
#pragma unroll
      for (int i = 0; i < E; ++i) d[i] *= t[i];
    }
    unit_grad<V, NV, LAYER>(d, s, rstd, a.cols, sums);
#pragma unroll
    for (int i = 0; i < E; ++i) d[i] += ds[i];  // the sum's whole gradient
#pragma unroll
    for (int i = 0; i < E; ++i) s[i] = a.scale * d[i];
    put<V, NV>(a.out0, row, a.cols, a.x_bf16, s);
    if constexpr (GATE) {
#pragma unroll
      for (int i = 0; i < E; ++i) dgate[i] = fmaf(d[i], p[i], dgate[i]);
      fetch<V, NV>(t, a.gate, group, a.cols, a.gate_bf16);
#pragma unroll
      for (int i = 0; i < E; ++i) d[i] *= t[i];
      if (last) {
        if (a.chunks == 1) put<V, NV>(a.dgate, group, a.cols, a.gate_bf16, dgate);
        else put<V, NV>(a.gate_part, (int64_t)blockIdx.x, a.cols, 0, dgate);
      }
    }
    if constexpr (POST) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        kept[K::POST_GAMMA][i] = fmaf(d[i], u[i], kept[K::POST_GAMMA][i]);
        if constexpr (LAYER) kept[K::POST_BETA][i] += d[i];
      }
      if (a.has_post_gamma) {
        fetch<V, NV>(t, a.post_gamma, 0, a.cols, a.w_bf16);
#pragma unroll
        for (int i = 0; i < E; ++i) d[i] *= t[i];
      }
      unit_grad<V, NV, LAYER>(d, u, rstd_f, a.cols, sums);
    }
    put<V, NV>(a.out1, row, a.cols, a.f_bf16, d);
  }
#pragma unroll
  for (int n = 0; n < K::N; ++n) put<V, NV>(a.part, (int64_t)blockIdx.x * K::N + n, a.cols, 0, kept[n]);
}

// out[z][c] = sum over i of part[(z count + i) pitch + first + c]: 32 columns a block, eight threads
// each, four loads in flight, a fixed order
struct Fold {
  const float* part;
  int64_t count, pitch;
  int cols;
  struct Out {
    void* p;
    int64_t first;
    int bf16;
  } out[4];
};
__global__ void __launch_bounds__(256) fold_kernel(const __grid_constant__ Fold a) {
  __shared__ float area[8][33];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  const Fold::Out o = a.out[blockIdx.y];
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  if (c < a.cols) {
    const float* p = a.part + (int64_t)blockIdx.z * a.count * a.pitch + o.first + c;
    int64_t i = slice;
    for (; i + 24 < a.count; i += 32)
#pragma unroll
      for (int k = 0; k < 4; ++k) s[k] += __ldg(p + (i + 8 * k) * a.pitch);
    for (; i < a.count; i += 8) s[0] += __ldg(p + i * a.pitch);
  }
  area[slice][lane] = (s[0] + s[1]) + (s[2] + s[3]);
  __syncthreads();
  if (slice == 0 && c < a.cols) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) t += area[k][lane];
    const int64_t at = (int64_t)blockIdx.z * a.cols + c;
    if (o.bf16) reinterpret_cast<__nv_bfloat16*>(o.p)[at] = __float2bfloat16_rn(t);
    else reinterpret_cast<float*>(o.p)[at] = t;
  }
}

// threads of a block, register sets of 8 elements a thread
static void shape(int64_t cols, int* threads, int* nv) {
  *nv = cols <= MAX_THREADS * 8 ? 1 : (cols <= MAX_THREADS * 16 ? 2 : 4);
  *threads = (int)(ceil_div(cols, 8 * *nv * 32) * 32);
}

// Blocks, and the chunks that each group's rows are cut into: `fill` blocks at most, but one a group.
struct Split {
  int64_t chunks, per_chunk, blocks;
};
static Split split(int64_t rows, int64_t groups, int64_t fill) {
  const int64_t per_group = rows / groups;
  Split s{1, per_group, std::min(groups, fill)};
  if (groups < fill) {
    s.per_chunk = ceil_div(per_group, std::min(per_group, std::max<int64_t>(1, fill / groups)));
    s.chunks = ceil_div(per_group, s.per_chunk);
    s.blocks = groups * s.chunks;
  }
  return s;
}
static int64_t fill_of(int threads, bool grad) {
  // 20 warps an SM forward, 16 in the gradient (its registers); 24 blocks
  return (int64_t)num_sms() * std::max(1, std::min(24, (grad ? 512 : 640) / threads));
}

static int check(const char* what, const b200_residual_norm* n, const void* const* ptr, int count) {
  B200_REQUIRE(n, "%s: no description", what);
  B200_REQUIRE(n->rows >= 0 && n->cols >= 1 && n->cols <= MAX_COLS, "%s: %lld x %lld (1 to %d columns)", what, (long long)n->rows,
               (long long)n->cols, MAX_COLS);
  B200_REQUIRE(n->kind == B200_NORM_RMS || n->kind == B200_NORM_LAYER, "%s: kind %d", what, n->kind);
  B200_REQUIRE(n->groups >= 0 && (n->gate == nullptr) == (n->groups == 0), "%s: %lld groups %s a gate", what, (long long)n->groups,
               n->gate ? "with" : "without");
  B200_REQUIRE(n->groups == 0 || n->rows % n->groups == 0, "%s: %lld rows in %lld groups", what, (long long)n->rows, (long long)n->groups);
  B200_REQUIRE(n->post || (!n->post_gamma && !n->post_beta), "%s: post weights without a post norm", what);
  B200_REQUIRE(n->kind == B200_NORM_LAYER || (!n->beta && !n->post_beta), "%s: beta is for layer norms", what);
  for (int d : {n->x_dtype, n->f_dtype, n->weight_dtype, n->gate_dtype})
    if (d != B200_F32 && d != B200_BF16) {
      set_error("%s: dtype %d (F32 and BF16)", what, d);
      return B200_ERR_DTYPE;
    }
  for (int i = 0; i < count; ++i) B200_REQUIRE(n->rows == 0 || ptr[i], "%s: null operand %d", what, i);
  return B200_OK;
}

static Args fill_args(const b200_residual_norm* n, const void* x, const void* f) {
  Args a = {};
  a.x = x, a.f = f;
  a.has_gate = n->gate != nullptr, a.has_gamma = n->gamma != nullptr, a.has_beta = n->beta != nullptr;
  a.has_post_gamma = n->post_gamma != nullptr, a.has_post_beta = n->post_beta != nullptr;
  const bool weights = a.has_gamma || a.has_beta || a.has_post_gamma || a.has_post_beta;
  const void* spare = n->gamma ? n->gamma : (n->beta ? n->beta : (n->post_gamma ? n->post_gamma : (n->post_beta ? n->post_beta : x)));
  a.gate = n->gate ? n->gate : x;
  a.gamma = n->gamma ? n->gamma : spare, a.beta = n->beta ? n->beta : spare;
  a.post_gamma = n->post_gamma ? n->post_gamma : spare, a.post_beta = n->post_beta ? n->post_beta : spare;
  a.rows = n->rows, a.groups = n->groups ? n->groups : 1, a.cols = (int)n->cols;
  a.per_group = a.rows / a.groups;
  a.x_bf16 = n->x_dtype == B200_BF16, a.f_bf16 = n->f_dtype == B200_BF16;
  a.w_bf16 = (weights ? n->weight_dtype : n->x_dtype) == B200_BF16, a.gate_bf16 = (n->gate ? n->gate_dtype : n->x_dtype) == B200_BF16;
  a.scale = n->scale, a.eps = n->eps;
  return a;
}

// whether every row of every array starts on 16 bytes and holds whole vectors
static bool vectors(const b200_residual_norm* n, std::initializer_list<const void*> ptr) {
  if (n->cols % 8) return false;
  uintptr_t u = 0;
  for (const void* p : ptr) u |= reinterpret_cast<uintptr_t>(p);
  for (const void* p : {n->gate, n->gamma, n->beta, n->post_gamma, n->post_beta}) u |= reinterpret_cast<uintptr_t>(p);
  return (u & 15) == 0;
}

template <int V, int NV>
static void launch_forward(const Args& a, int64_t blocks, int threads, bool layer, bool post, cudaStream_t st) {
  const dim3 g((unsigned)blocks), b((unsigned)threads);
  if (layer) post ? forward_kernel<V, NV, true, true><<<g, b, 0, st>>>(a) : forward_kernel<V, NV, true, false><<<g, b, 0, st>>>(a);
  else post ? forward_kernel<V, NV, false, true><<<g, b, 0, st>>>(a) : forward_kernel<V, NV, false, false><<<g, b, 0, st>>>(a);
}
template <int V, int NV, bool GATE>
static void launch_gradient(const Args& a, int64_t blocks, int threads, bool layer, bool post, cudaStream_t st) {
  const dim3 g((unsigned)blocks), b((unsigned)threads);
  if (layer) post ? gradient_kernel<V, NV, true, true, GATE><<<g, b, 0, st>>>(a) : gradient_kernel<V, NV, true, false, GATE><<<g, b, 0, st>>>(a);
  else post ? gradient_kernel<V, NV, false, true, GATE><<<g, b, 0, st>>>(a) : gradient_kernel<V, NV, false, false, GATE><<<g, b, 0, st>>>(a);
}

}  // namespace rnorm
}  // namespace b200

using namespace b200;
using namespace b200::rnorm;

extern "C" int b200_residual_norm_forward(const b200_residual_norm* n, const void* x, const void* f, void* sum, void* normed,
                                          void* stream) {
  const void* ptr[] = {x, f, sum, normed};
  if (int rc = check("residual_norm", n, ptr, 4)) return rc;
  if (n->rows == 0) return B200_OK;
  Args a = fill_args(n, x, f);
  a.out0 = sum, a.out1 = normed;
  int threads, nv;
  shape(n->cols, &threads, &nv);
  const Split s = split(a.rows, a.groups, fill_of(threads, false));
  a.chunks = s.chunks, a.per_chunk = s.per_chunk;
  const bool layer = n->kind == B200_NORM_LAYER, post = n->post != 0, vec = vectors(n, {x, f, sum, normed});
  cudaStream_t st = as_stream(stream);
#define B200_GO(V, NV) launch_forward<V, NV>(a, s.blocks, threads, layer, post, st)
  if (vec) nv == 1 ? B200_GO(8, 1) : (nv == 2 ? B200_GO(8, 2) : B200_GO(8, 4));
  else nv == 1 ? B200_GO(1, 1) : (nv == 2 ? B200_GO(1, 2) : B200_GO(1, 4));
#undef B200_GO
  return check_launch("residual_norm");
}

static int kept_of(int kind, int post) { return (post ? 2 : 1) * (kind == B200_NORM_LAYER ? 2 : 1); }

extern "C" size_t b200_residual_norm_grad_workspace_bytes(const b200_residual_norm* n) {
  if (!n || n->rows <= 0 || n->cols < 1 || n->cols > MAX_COLS || n->groups < 0 || (n->groups && n->rows % n->groups)) return 0;
  int threads, nv;
  shape(n->cols, &threads, &nv);
  const Split s = split(n->rows, n->groups ? n->groups : 1, fill_of(threads, true));
  const int64_t gate = n->groups && s.chunks > 1 ? s.blocks : 0;
  return (size_t)((s.blocks * kept_of(n->kind, n->post) + gate) * n->cols) * sizeof(float);
}

extern "C" int b200_residual_norm_grad(const b200_residual_norm* n, const void* dsum, const void* dnormed, const void* x, const void* f,
                                       void* dx, void* df, const b200_residual_norm_grads* g, void* workspace, size_t workspace_bytes,
                                       void* stream) {
  const void* ptr[] = {dsum, dnormed, x, f, dx, df};
  if (int rc = check("residual_norm_grad", n, ptr, 6)) return rc;
  B200_REQUIRE(g, "residual_norm_grad: no place for the weights' gradients");
  const bool layer = n->kind == B200_NORM_LAYER, post = n->post != 0, gate = n->groups > 0;
  cudaStream_t st = as_stream(stream);
  const size_t wsize = n->weight_dtype == B200_BF16 ? 2 : 4, gsize = n->gate_dtype == B200_BF16 ? 2 : 4;
  if (n->rows == 0) {
    // sums over no rows
    for (void* p : {g->dgamma, g->dbeta, g->dpost_gamma, g->dpost_beta})
      if (p && cudaMemsetAsync(p, 0, (size_t)n->cols * wsize, st) != cudaSuccess) return check_launch("residual_norm_grad");
    if (g->dgate && cudaMemsetAsync(g->dgate, 0, (size_t)(n->groups * n->cols) * gsize, st) != cudaSuccess)
      return check_launch("residual_norm_grad");
    return B200_OK;
  }
  B200_REQUIRE(!gate || g->dgate, "residual_norm_grad: no place for the gate's gradient");
  const size_t need = b200_residual_norm_grad_workspace_bytes(n);
  B200_REQUIRE(workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
               "residual_norm_grad: workspace of %zu bytes, %zu needed on a 16-byte boundary", workspace_bytes, need);
  Args a = fill_args(n, x, f);
  a.ds = dsum, a.dh = dnormed, a.out0 = dx, a.out1 = df, a.dgate = g->dgate;
  int threads, nv;
  shape(n->cols, &threads, &nv);
  const Split s = split(a.rows, a.groups, fill_of(threads, true));
  a.chunks = s.chunks, a.per_chunk = s.per_chunk;
  const int kept = kept_of(n->kind, n->post);
  a.part = reinterpret_cast<float*>(workspace);
  a.gate_part = a.part + s.blocks * kept * n->cols;
  const bool vec = vectors(n, {dsum, dnormed, x, f, dx, df, g->dgate});
#define B200_GO(V, NV) \
  gate ? launch_gradient<V, NV, true>(a, s.blocks, threads, layer, post, st) : launch_gradient<V, NV, false>(a, s.blocks, threads, layer, post, st)
  if (vec) nv == 1 ? (B200_GO(8, 1)) : (nv == 2 ? (B200_GO(8, 2)) : (B200_GO(8, 4)));
  else nv == 1 ? (B200_GO(1, 1)) : (nv == 2 ? (B200_GO(1, 2)) : (B200_GO(1, 4)));
#undef B200_GO
  if (int rc = check_launch("residual_norm_grad")) return rc;
  // the sums over blocks of the weights that are asked for
  Fold fold = {};
  fold.part = a.part, fold.count = s.blocks, fold.pitch = kept * n->cols, fold.cols = a.cols;
  int outs = 0;
  auto ask = [&](void* p, int slot) {
    if (p) fold.out[outs++] = {p, (int64_t)slot * n->cols, n->weight_dtype == B200_BF16};
  };
  ask(g->dgamma, 0);
  if (layer) ask(g->dbeta, 1);
  if (post) ask(g->dpost_gamma, layer ? 2 : 1);
  if (post && layer) ask(g->dpost_beta, 3);
  const unsigned wide = (unsigned)ceil_div(n->cols, 32);
  if (outs) {
    fold_kernel<<<dim3(wide, (unsigned)outs, 1), 256, 0, st>>>(fold);
    if (int rc = check_launch("residual_norm_grad")) return rc;
  }
  if (gate && s.chunks > 1) {
    Fold fg = {};
    fg.part = a.gate_part, fg.count = s.chunks, fg.pitch = n->cols, fg.cols = a.cols;
    fg.out[0] = {g->dgate, 0, a.gate_bf16};
    fold_kernel<<<dim3(wide, 1, (unsigned)a.groups), 256, 0, st>>>(fg);
    return check_launch("residual_norm_grad");
  }
  return B200_OK;
}
