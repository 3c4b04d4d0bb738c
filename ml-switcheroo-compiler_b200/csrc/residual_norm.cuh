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
// One block holds one row in registers (8 elements a thread and register set) and walks its rows.
// Everything is fp32 between one load and one rounding per output; h is made of the sum before its
// rounding, and the gradient makes the sums again from x and f. Each array is read or written once.
// What bounds it is the chain of a row: its loads, and two (rms) to four (layer) reductions over the block
// forward, up to six in the gradient, a barrier each. So many blocks share an SM (registers are capped for it)
// rather than that a block loads ahead, a thread of the gradient has 16 elements (fewer threads to a barrier, more rows under way),
// and weights stay in shared memory. Measured: 64 x 512 x 1024 layer norm, fp32 stream, 71 us (141 with the next row loaded early
// and types looked up at run time), the gradients of 16 x 1000 x 2048 with post norm and gate 124 to 127 us (430; 206 with 8
// elements a thread). Most gradients spill: 4 to 416 bytes a thread for whole vectors up to 8192 columns (152 in the measured one), up
// to 2154 for wider or ragged rows.
// The weights' gradients are kept per thread over the block's rows (a thread owns columns), go to
// the workspace once a block, and are added up in a fixed order by a second launch; a gate's
// gradient whose group one block covers alone is written by that block.
#pragma once
#include <algorithm>

#include "common.cuh"

namespace b200 {
namespace rnorm {

constexpr int MAX_THREADS = 512, MAX_COLS = MAX_THREADS * 8 * 4;
// threads of a block at most, and blocks an SM that its registers are capped for
template <int NV>
struct Bounds {
  static constexpr int THREADS = NV == 1 ? 256 : 512, FORWARD = NV == 1 ? 4 : (NV == 2 ? 2 : 1), GRADIENT = NV == 1 ? 3 : 1;
};

struct Args {
  const void *x, *f, *ds, *dh;  // ds, dh: gradient only
  // weights that were not given point at another one, or at x, and are not asked for: no address is null
  const void *gate, *gamma, *beta, *post_gamma, *post_beta;
  int has_gate, has_gamma, has_beta, has_post_gamma, has_post_beta;
  int w_bf16, gate_bf16;
  int gate_kept;                        // groups are long enough for the gate to be kept like the weights
  int shared;                           // the weights fit shared memory
  void *out0, *out1;                    // s and h, or dx and df
  float* part;                          // [blocks][weights][cols]
  float* gate_part;                     // [groups][chunks][cols] (chunks > 1)
  void* dgate;                          // written here where chunks == 1
  int64_t rows, groups, per_group;      // per_group = rows / groups
  int64_t chunks, per_chunk;            // a group's rows are cut into chunks
  int cols;
  float scale, eps, inv_cols;
};

// Where a thread's element i (of 8 NV) of a row is: vectors of 8 neighbours, or one column in
// blockDim where rows are no multiple of 8 elements or not aligned.
template <int V>
__device__ __forceinline__ int column(int i) {
  if constexpr (V == 8) return ((i >> 3) * (int)blockDim.x + (int)threadIdx.x) * 8 + (i & 7);
  else return i * (int)blockDim.x + (int)threadIdx.x;
}

// 16 bytes that are read once: not kept in the L1. An ordinary load in its place among the stores: results may lie over the arrays
// that are read here (a row's elements are read by the thread that writes them, before it does).
__device__ __forceinline__ uint4 load_once(const void* p) {
  uint4 u;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "l"(p) : "memory");
  return u;
}
__device__ __forceinline__ void widen(const uint4& u, float* o) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) o[2 * k] = __uint_as_float(w[k] << 16), o[2 * k + 1] = __uint_as_float(w[k] & 0xFFFF0000u);
}

// A thread's 8 NV elements of one row as they are in memory; zeros behind the row's end
template <int V, int NV, typename T>
struct Raw {
  static constexpr int WORDS = sizeof(T) == 2 ? 1 : 2;  // 16-byte words of 8 elements
  uint4 w[V == 8 ? NV * WORDS : 1];
  T s[V == 8 ? 1 : NV * 8];

  __device__ __forceinline__ void load(const void* base, int64_t row, int cols) {
    const T* p = reinterpret_cast<const T*>(base) + row * cols;
    if constexpr (V == 8) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int c = column<V>(8 * v);
#pragma unroll
        for (int k = 0; k < WORDS; ++k) w[v * WORDS + k] = c < cols ? load_once(p + c + k * (8 / WORDS)) : make_uint4(0, 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8 * NV; ++i) s[i] = column<V>(i) < cols ? p[column<V>(i)] : (T)0.f;
    }
  }
  __device__ __forceinline__ void get(float (&o)[8 * NV]) const {
    if constexpr (V == 8) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        if constexpr (sizeof(T) == 2) {
          widen(w[v], o + 8 * v);
        } else {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint4 u = w[2 * v + k];
            o[8 * v + 4 * k] = __uint_as_float(u.x), o[8 * v + 4 * k + 1] = __uint_as_float(u.y);
            o[8 * v + 4 * k + 2] = __uint_as_float(u.z), o[8 * v + 4 * k + 3] = __uint_as_float(u.w);
          }
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8 * NV; ++i) o[i] = (float)s[i];
    }
  }
};

// a row of weights or of the gate, of either type; zeros behind the end
template <int V, int NV>
__device__ __forceinline__ void fetch(float (&o)[8 * NV], const void* base, int64_t row, int cols, int bf16) {
  if constexpr (V == 8) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = column<V>(8 * v);
#pragma unroll
      for (int k = 0; k < 8; ++k) o[8 * v + k] = 0.f;
      if (c < cols) {
        if (bf16) {
          widen(__ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(base) + row * cols + c)), o + 8 * v);
        } else {
          const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(base) + row * cols + c);
          const float4 a = __ldg(p), b = __ldg(p + 1);
          o[8 * v] = a.x, o[8 * v + 1] = a.y, o[8 * v + 2] = a.z, o[8 * v + 3] = a.w;
          o[8 * v + 4] = b.x, o[8 * v + 5] = b.y, o[8 * v + 6] = b.z, o[8 * v + 7] = b.w;
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8 * NV; ++i) {
      const int c = column<V>(i);
      o[i] = 0.f;
      if (c < cols)
        o[i] = bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(base)[row * cols + c]) : reinterpret_cast<const float*>(base)[row * cols + c];
    }
  }
}

template <int V, int NV, typename T>
__device__ __forceinline__ void put(T* base, int64_t row, int cols, const float (&o)[8 * NV]) {
  base += row * cols;
  if constexpr (V == 8) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = column<V>(8 * v);
      if (c >= cols) continue;
      if constexpr (sizeof(T) == 2) {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const __nv_bfloat162 t = __floats2bfloat162_rn(o[8 * v + 2 * k], o[8 * v + 2 * k + 1]);
          w[k] = *reinterpret_cast<const uint32_t*>(&t);
        }
        *reinterpret_cast<uint4*>(base + c) = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
        float4* p = reinterpret_cast<float4*>(base + c);
        p[0] = make_float4(o[8 * v], o[8 * v + 1], o[8 * v + 2], o[8 * v + 3]);
        p[1] = make_float4(o[8 * v + 4], o[8 * v + 5], o[8 * v + 6], o[8 * v + 7]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8 * NV; ++i)
      if (column<V>(i) < cols) base[column<V>(i)] = (T)o[i];
  }
}
template <int V, int NV>
__device__ __forceinline__ void put_any(void* base, int64_t row, int cols, int bf16, const float (&o)[8 * NV]) {
  if (bf16) put<V, NV>(reinterpret_cast<__nv_bfloat16*>(base), row, cols, o);
  else put<V, NV>(reinterpret_cast<float*>(base), row, cols, o);
}

// Weights that a block keeps in shared memory as fp32, each thread its own columns (so without a barrier), laid out so that a
// thread's four neighbours are 16 bytes; or, where they do not fit, reads again from global memory.
template <int NV>
struct Slot {
  uint32_t at, step;  // shared-memory address of this thread's first 16 bytes, bytes to the next
  __device__ __forceinline__ void put(const float (&o)[8 * NV]) {
#pragma unroll
    for (int i = 0; i < 2 * NV; ++i)
      asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at + i * step), "f"(o[4 * i]), "f"(o[4 * i + 1]), "f"(o[4 * i + 2]), "f"(o[4 * i + 3])
                   : "memory");
  }
  __device__ __forceinline__ void get(float (&o)[8 * NV]) const {
#pragma unroll
    for (int i = 0; i < 2 * NV; ++i)
      asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                   : "=f"(o[4 * i]), "=f"(o[4 * i + 1]), "=f"(o[4 * i + 2]), "=f"(o[4 * i + 3])
                   : "r"(at + i * step)
                   : "memory");
  }
};
constexpr int GAMMA = 0, BETA = 1, POST_GAMMA = 2, POST_BETA = 3, GATE_SLOT = 4, SLOTS = 5;

template <int V, int NV>
struct Weights {
  const Args& a;
  uint32_t slot[SLOTS], step;
  int64_t gate_group;  // whose gate its slot holds

  __device__ __forceinline__ Weights(const Args& a_, float4* s) : a(a_), step(blockDim.x * 16u), gate_group(-1) {
    const uint32_t base = (uint32_t)__cvta_generic_to_shared(s + threadIdx.x);
    const int has[SLOTS] = {a.has_gamma, a.has_beta, a.has_post_gamma, a.has_post_beta, a.has_gate && a.gate_kept};
    int n = 0;
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) slot[i] = base + (has[i] ? n++ : 0) * (2 * NV * step);
    if (!a.shared) return;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (has[i]) {
        float t[8 * NV];
        fetch<V, NV>(t, pointer(i), 0, a.cols, a.w_bf16);
        at(i).put(t);
      }
  }
  __device__ __forceinline__ const void* pointer(int i) const { return i == GAMMA ? a.gamma : (i == BETA ? a.beta : (i == POST_GAMMA ? a.post_gamma : a.post_beta)); }
  __device__ __forceinline__ Slot<NV> at(int i) const { return {slot[i], step}; }
  __device__ __forceinline__ void get(float (&o)[8 * NV], int i) const {
    if (a.shared) at(i).get(o);
    else fetch<V, NV>(o, pointer(i), 0, a.cols, a.w_bf16);
  }
  __device__ __forceinline__ void gate(float (&o)[8 * NV], int64_t group) {
    if (a.shared && a.gate_kept) {
      if (group != gate_group) {
        gate_group = group;
        fetch<V, NV>(o, a.gate, group, a.cols, a.gate_bf16);
        at(GATE_SLOT).put(o);
        return;
      }
      at(GATE_SLOT).get(o);
    } else {
      fetch<V, NV>(o, a.gate, group, a.cols, a.gate_bf16);
    }
  }
};

// Sums over the block, the same on every thread: one barrier, the area alternates between two
// halves so that the next sum may write while slow warps still read this one. Places of warps that the block does not have stay zero.
struct Sums {
  float (*area)[2][16];  // [half][value][warp]
  int half, quads;       // quads: fours of warps
  __device__ __forceinline__ Sums(float (*s)[2][16]) : area(s), half(0), quads(((int)blockDim.x + 127) >> 7) {
    for (int i = threadIdx.x; i < 64; i += blockDim.x) (&s[0][0][0])[i] = 0.f;
    __syncthreads();
  }
  __device__ __forceinline__ float read(const float* p) const {
    const float4* v = reinterpret_cast<const float4*>(p);
    float4 u = v[0];
    float s = (u.x + u.y) + (u.z + u.w);
    if (quads > 1) u = v[1], s += (u.x + u.y) + (u.z + u.w);
    if (quads > 2) {
      u = v[2], s += (u.x + u.y) + (u.z + u.w);
      u = v[3], s += (u.x + u.y) + (u.z + u.w);
    }
    return s;
  }
  __device__ __forceinline__ void operator()(float& a, float& b) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      a += __shfl_xor_sync(0xffffffffu, a, o);
      b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if (blockDim.x == 32) return;
    if ((threadIdx.x & 31) == 0) area[half][0][threadIdx.x >> 5] = a, area[half][1][threadIdx.x >> 5] = b;
    __syncthreads();
    a = read(area[half][0]), b = read(area[half][1]);
    half ^= 1;
  }
  __device__ __forceinline__ void operator()(float& a) {
    a = warp_sum(a);
    if (blockDim.x == 32) return;
    if ((threadIdx.x & 31) == 0) area[half][0][threadIdx.x >> 5] = a;
    __syncthreads();
    a = read(area[half][0]);
    half ^= 1;
  }
};

// t (zeros behind the row's end) -> the normed row u before gamma; returns rstd
template <int V, int NV, bool LAYER>
__device__ __forceinline__ float unit(float (&t)[8 * NV], const Args& a, Sums& sums) {
  const int cols = a.cols;
  if constexpr (LAYER) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8 * NV; ++i) m += t[i];
    sums(m);
    m *= a.inv_cols;
#pragma unroll
    for (int i = 0; i < 8 * NV; ++i) t[i] = column<V>(i) < cols ? t[i] - m : 0.f;
  }
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < 8 * NV; ++i) q = fmaf(t[i], t[i], q);
  sums(q);
  const float rstd = rsqrtf(fmaf(q, a.inv_cols, a.eps));
#pragma unroll
  for (int i = 0; i < 8 * NV; ++i) t[i] *= rstd;
  return rstd;
}

// d = dy gamma -> the gradient rstd (d - [mean d] - u mean(d u))
template <int V, int NV, bool LAYER>
__device__ __forceinline__ void unit_grad(float (&d)[8 * NV], const float (&u)[8 * NV], float rstd, const Args& args, Sums& sums) {
  const int cols = args.cols;
  float a = 0.f, b = 0.f;
#pragma unroll
  for (int i = 0; i < 8 * NV; ++i) {
    a = fmaf(d[i], u[i], a);
    if constexpr (LAYER) b += d[i];
  }
  if constexpr (LAYER) sums(a, b);
  else sums(a);
  a *= -rstd * args.inv_cols;
  b *= args.inv_cols;
#pragma unroll
  for (int i = 0; i < 8 * NV; ++i) {
    d[i] = LAYER ? fmaf(a, u[i], rstd * (d[i] - b)) : fmaf(a, u[i], rstd * d[i]);
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

template <int NV>
__device__ __forceinline__ void times(float (&x)[8 * NV], const float (&y)[8 * NV]) {
#pragma unroll
  for (int i = 0; i < 8 * NV; ++i) x[i] *= y[i];
}
template <int NV>
__device__ __forceinline__ void plus(float (&x)[8 * NV], const float (&y)[8 * NV]) {
#pragma unroll
  for (int i = 0; i < 8 * NV; ++i) x[i] += y[i];
}

template <int V, int NV, bool LAYER, bool POST, typename TX, typename TF>
__global__ void __launch_bounds__(Bounds<NV>::THREADS, Bounds<NV>::FORWARD) forward_kernel(const __grid_constant__ Args a) {
  __shared__ __align__(16) float area[2][2][16];
  extern __shared__ float4 slots[];
  Sums sums(area);
  Weights<V, NV> weights(a, slots);
  constexpr int E = 8 * NV;
  for (Walk w(a); w.more(a); w.next(a)) {
    float s[E], p[E], t[E];
    {
      Raw<V, NV, TX> rx;
      Raw<V, NV, TF> rf;
      rf.load(a.f, w.row, a.cols);
      rx.load(a.x, w.row, a.cols);
      rf.get(p);
      rx.get(s);
    }
    if constexpr (POST) {
      unit<V, NV, LAYER>(p, a, sums);
      if (a.has_post_gamma) {
        weights.get(t, POST_GAMMA);
        times<NV>(p, t);
      }
      if (LAYER && a.has_post_beta) {
        weights.get(t, POST_BETA);
        plus<NV>(p, t);
      }
    }
    if (a.has_gate) {
      weights.gate(t, w.group);
      times<NV>(p, t);
    }
#pragma unroll
    for (int i = 0; i < E; ++i) s[i] = fmaf(a.scale, s[i], p[i]);
    put<V, NV>(reinterpret_cast<TX*>(a.out0), w.row, a.cols, s);
    unit<V, NV, LAYER>(s, a, sums);
    if (a.has_gamma) {
      weights.get(t, GAMMA);
      times<NV>(s, t);
    }
    if (LAYER && a.has_beta) {
      weights.get(t, BETA);
      plus<NV>(s, t);
    }
    put<V, NV>(reinterpret_cast<TF*>(a.out1), w.row, a.cols, s);
  }
}

// weights' gradients that a block keeps, in the order of the workspace
template <bool LAYER, bool POST>
struct Kept {
  static constexpr int N = (1 + (POST ? 1 : 0)) * (LAYER ? 2 : 1);
  static constexpr int GAMMA = 0, BETA = 1, POST_GAMMA = LAYER ? 2 : 1, POST_BETA = 3;
};

template <int V, int NV, bool LAYER, bool POST, bool GATE, typename TX, typename TF>
__global__ void __launch_bounds__(Bounds<NV>::THREADS, Bounds<NV>::GRADIENT) gradient_kernel(const __grid_constant__ Args a) {
  using K = Kept<LAYER, POST>;
  __shared__ __align__(16) float area[2][2][16];
  extern __shared__ float4 slots[];
  Sums sums(area);
  Weights<V, NV> weights(a, slots);
  constexpr int E = 8 * NV;
  float kept[K::N][E], dgate[GATE ? E : 1];
#pragma unroll
  for (int n = 0; n < K::N; ++n)
#pragma unroll
    for (int i = 0; i < E; ++i) kept[n][i] = 0.f;
  Walk w(a);
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
    // all four rows are on their way at once; the gradients stay packed until they are needed
    Raw<V, NV, TX> rs;
    Raw<V, NV, TF> rh;
    float s[E], p[E], t[E];  // p: the block's output, normed without its weights
    {
      Raw<V, NV, TX> rx;
      Raw<V, NV, TF> rf;
      rf.load(a.f, row, a.cols);
      rx.load(a.x, row, a.cols);
      rh.load(a.dh, row, a.cols);
      rs.load(a.ds, row, a.cols);
      rf.get(p);
      rx.get(s);
    }
    w.next(a);
    const bool last = !w.more(a) || w.group != group;  // of this group
    // the block's output with its norm's weights
    auto block = [&](float (&o)[E]) {
#pragma unroll
      for (int i = 0; i < E; ++i) o[i] = p[i];
      if constexpr (POST) {
        float v[E];
        if (a.has_post_gamma) {
          weights.get(v, POST_GAMMA);
          times<NV>(o, v);
        }
        if (LAYER && a.has_post_beta) {
          weights.get(v, POST_BETA);
          plus<NV>(o, v);
        }
      }
    };
    float rstd_f = 0.f;
    if constexpr (POST) rstd_f = unit<V, NV, LAYER>(p, a, sums);
    {
      float o[E];
      block(o);
      if constexpr (GATE) {
        weights.gate(t, group);
        times<NV>(o, t);
      }
#pragma unroll
      for (int i = 0; i < E; ++i) s[i] = fmaf(a.scale, s[i], o[i]);
    }
    const float rstd = unit<V, NV, LAYER>(s, a, sums);
    float d[E];
    rh.get(d);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      kept[K::GAMMA][i] = fmaf(d[i], s[i], kept[K::GAMMA][i]);
      if constexpr (LAYER) kept[K::BETA][i] += d[i];
    }
    if (a.has_gamma) {
      weights.get(t, GAMMA);
      times<NV>(d, t);
    }
    unit_grad<V, NV, LAYER>(d, s, rstd, a, sums);
    rs.get(t);
    plus<NV>(d, t);  // the sum's whole gradient
#pragma unroll
    for (int i = 0; i < E; ++i) s[i] = a.scale * d[i];
    put<V, NV>(reinterpret_cast<TX*>(a.out0), row, a.cols, s);
    if constexpr (GATE) {
      block(s);
#pragma unroll
      for (int i = 0; i < E; ++i) dgate[i] = fmaf(d[i], s[i], dgate[i]);
      weights.gate(t, group);
      times<NV>(d, t);
      if (last) {
        if (a.chunks == 1) put_any<V, NV>(a.dgate, group, a.cols, a.gate_bf16, dgate);
        else put<V, NV>(a.gate_part, (int64_t)blockIdx.x, a.cols, dgate);
      }
    }
    if constexpr (POST) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        kept[K::POST_GAMMA][i] = fmaf(d[i], p[i], kept[K::POST_GAMMA][i]);
        if constexpr (LAYER) kept[K::POST_BETA][i] += d[i];
      }
      if (a.has_post_gamma) {
        weights.get(t, POST_GAMMA);
        times<NV>(d, t);
      }
      unit_grad<V, NV, LAYER>(d, p, rstd_f, a, sums);
    }
    put<V, NV>(reinterpret_cast<TF*>(a.out1), row, a.cols, d);
  }
#pragma unroll
  for (int n = 0; n < K::N; ++n) put<V, NV>(a.part, (int64_t)blockIdx.x * K::N + n, a.cols, kept[n]);
}

// What to launch: the shape of a block, which kernel.
struct Launch {
  int64_t blocks;
  int threads, nv, vec, layer, post, gate;
  size_t shared;
};
// for rows of TX (the stream) and TF (the block's output); the four are compiled in files of their own
template <typename TX, typename TF>
int run_forward(const Args& a, const Launch& l, cudaStream_t st);
template <typename TX, typename TF>
int run_gradient(const Args& a, const Launch& l, cudaStream_t st);

template <typename Kernel>
static int go(Kernel kernel, const Args& a, const Launch& l, cudaStream_t st) {
  kernel<<<(unsigned)l.blocks, l.threads, l.shared, st>>>(a);
  return check_launch("residual_norm");
}
template <int V, int NV, typename TX, typename TF>
static int forward_of(const Args& a, const Launch& l, cudaStream_t st) {
  if (l.layer) return l.post ? go(forward_kernel<V, NV, true, true, TX, TF>, a, l, st) : go(forward_kernel<V, NV, true, false, TX, TF>, a, l, st);
  return l.post ? go(forward_kernel<V, NV, false, true, TX, TF>, a, l, st) : go(forward_kernel<V, NV, false, false, TX, TF>, a, l, st);
}
template <int V, int NV, bool GATE, typename TX, typename TF>
static int gradient_of(const Args& a, const Launch& l, cudaStream_t st) {
  if (l.layer) return l.post ? go(gradient_kernel<V, NV, true, true, GATE, TX, TF>, a, l, st) : go(gradient_kernel<V, NV, true, false, GATE, TX, TF>, a, l, st);
  return l.post ? go(gradient_kernel<V, NV, false, true, GATE, TX, TF>, a, l, st) : go(gradient_kernel<V, NV, false, false, GATE, TX, TF>, a, l, st);
}
// rows that are no vectors take the register sets of wider ones: one kernel for all
#define B200_RESIDUAL_NORM(TX, TF)                                                                                                      \
  template <>                                                                                                                           \
  int run_forward<TX, TF>(const Args& a, const Launch& l, cudaStream_t st) {                                                            \
    if (!l.vec) return l.nv == 1 ? forward_of<1, 1, TX, TF>(a, l, st) : forward_of<1, 4, TX, TF>(a, l, st);                             \
    return l.nv == 1 ? forward_of<8, 1, TX, TF>(a, l, st) : (l.nv == 2 ? forward_of<8, 2, TX, TF>(a, l, st) : forward_of<8, 4, TX, TF>(a, l, st)); \
  }                                                                                                                                     \
  template <>                                                                                                                           \
  int run_gradient<TX, TF>(const Args& a, const Launch& l, cudaStream_t st) {                                                           \
    if (!l.vec) {                                                                                                                       \
      if (l.nv == 1) return l.gate ? gradient_of<1, 1, true, TX, TF>(a, l, st) : gradient_of<1, 1, false, TX, TF>(a, l, st);            \
      return l.gate ? gradient_of<1, 4, true, TX, TF>(a, l, st) : gradient_of<1, 4, false, TX, TF>(a, l, st);                           \
    }                                                                                                                                   \
    if (l.nv == 1) return l.gate ? gradient_of<8, 1, true, TX, TF>(a, l, st) : gradient_of<8, 1, false, TX, TF>(a, l, st);              \
    if (l.nv == 2) return l.gate ? gradient_of<8, 2, true, TX, TF>(a, l, st) : gradient_of<8, 2, false, TX, TF>(a, l, st);              \
    return l.gate ? gradient_of<8, 4, true, TX, TF>(a, l, st) : gradient_of<8, 4, false, TX, TF>(a, l, st);                             \
  }

}  // namespace rnorm
}  // namespace b200
