// Rotary positions of heads, and the RMS norm of queries and keys per head with the same
// rotation in one pass; both directions.
//
//   forward          y  = R(u gamma),  u = x rsqrt(mean(x^2) + eps)      (norm)
//                    y  = R(x)                                           (rotation alone)
//   backward (norm)  g  = R^-1(dy), h = g gamma, dx = rstd (h - u mean(h u)), dgamma = sum g u
//   R rotates pair j of a head by t_j = position * w_j and scales it by `factor`:
//                    (a, b) -> factor (a cos t - b sin t, b cos t + a sin t)
// The pairs are (j, j + rotary_dim / 2) or, interleaved, (2j, 2j + 1); elements from
// rotary_dim on pass through (normed, not rotated).
//
// Angles. w_j comes as a fraction of a turn per position in 64-bit fixed point, so
// position * w_j modulo one turn is one wrapping integer product: exact for any position
// (an fp32 product would be off by 0.06 rad at position 10^6). The nearest quarter turn is
// taken off in integers, what is left (within pi / 4) goes through the Taylor polynomials of
// sine (to x^9) and cosine (to x^10), off by less than 2^-28 there. The table travels in the
// kernel's parameters: nothing is uploaded or kept.
//
// Layout of the work. A lane owns one unit of a head: two vectors of V = 4 elements that
// hold whole pairs (the two halves of V pairs, or 2V neighbours), so a rotation needs no
// shuffle; the units of a head take L lanes (a power of two for the norms), a warp holds R = 32 / L
// heads. A warp takes a token and walks its heads, R at a time: the lane's angles are the
// same for every head, so cosines and sines are made once per token, while the first heads'
// loads are under way. Few tokens (a decoding batch) are split over head groups, so that the
// heads of one token run on many warps; each then makes the angles again.
// Bound by HBM: x (and dy) are read once, y (dx) written once. BATCH groups of heads are
// loaded before any is worked on: with 8 to 16 bytes a lane and vector the SM's warps have
// to have 50 KB or more under way. The issue slots come next: elements are worked on two at a
// time (f32x2 products), the weights are folded into the rotation's coefficients
// (y = rstd (x k1 + partner k2)), and row pointers advance by additions.
// The launch bounds (4, 3 and 2 blocks an SM) leave some kernels short of registers: the forward
// norm of heads up to 256 spills 8 to 88 bytes a thread, two units of vectors 40 to 360, and the
// five units of odd 512-element heads up to 770.
#include <algorithm>
#include <limits>

#include "common.cuh"

namespace b200 {
namespace rot {

constexpr int WARPS = 8, THREADS = 32 * WARPS;
constexpr int ROTATE = 0, NORM = 1, NORM_GRAD = 2;

struct Seg {  // one tensor of heads; element strides over batch, sequence, head (the head's elements are adjacent)
  const void* x;
  const void* dy;
  void* y;
  int64_t x_b, x_s, x_h, d_b, d_s, d_h, y_b, y_s, y_h;
  const void* gamma;
  int heads;
  int groups;  // ceil(heads / R)
};

struct Args {
  Seg seg[2];
  const void* pos;  // NULL: offset + index in the sequence
  int64_t pos_b, pos_s, offset;
  int pos_i32, gamma_bf16;
  int tokens, seq, dim, part;
  int L, chunks, per_chunk;  // lanes per head; head groups per token are cut into chunks of per_chunk
  int n_rot, n_units;        // units that rotate (by halves), units in all
  float eps, factor, sign;
  float* partial;  // [grid, 2, dim] sums of g u (NORM_GRAD)
  uint64_t freq[B200_ROTARY_MAX_DIM / 2];
};

// ---- two fp32 values in a 64-bit register pair ----
typedef uint64_t f2;
__device__ __forceinline__ f2 pair(float a, float b) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void halves(f2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f2 swapped(f2 v) {
  float a, b;
  halves(v, a, b);
  return pair(b, a);
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float sum2(f2 v) {
  float a, b;
  halves(v, a, b);
  return a + b;
}

// cosine and sine of phase / 2^64 of a turn
__device__ __forceinline__ void cos_sin(uint64_t phase, float& c, float& s) {
  const uint32_t top = (uint32_t)(phase >> 32);
  const uint32_t quarter = (top + 0x20000000u) >> 30;        // the nearest quarter turn
  const float x = (float)(int32_t)(top - (quarter << 30)) * 1.4629180792671596e-9f;  // 2 pi 2^-32: within pi / 4
  const float q = x * x;
  float sn = fmaf(q, 2.7557319223985893e-6f, -1.984126984126984e-4f);
  sn = fmaf(q, sn, 8.333333333333333e-3f);
  sn = fmaf(q, sn, -1.6666666666666666e-1f);
  sn = fmaf(q * sn, x, x);
  float cs = fmaf(q, -2.755731922398589e-7f, 2.48015873015873e-5f);
  cs = fmaf(q, cs, -1.388888888888889e-3f);
  cs = fmaf(q, cs, 4.1666666666666664e-2f);
  cs = fmaf(q, cs, -0.5f);
  cs = fmaf(q, cs, 1.f);
  const float u = quarter & 1 ? sn : cs, v = quarter & 1 ? cs : sn;
  c = __uint_as_float(__float_as_uint(u) ^ (((quarter + 1) & 2) << 30));
  s = __uint_as_float(__float_as_uint(v) ^ ((quarter & 2) << 30));
}

// V elements as loaded: the words of one vector access (FAST; all there or none), or floats
template <typename T, int V, bool FAST>
struct Vec {
  static constexpr int WORDS = FAST ? V * (int)sizeof(T) / 4 : V;
  uint32_t w[WORDS];

  __device__ __forceinline__ void load(const T* p, int n) {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) w[i] = 0u;
    if constexpr (!FAST) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i < n) w[i] = __float_as_uint((float)p[i]);
    } else if constexpr (WORDS == 4) {
      // predicated, where `if` would branch around every load (17 % of all instructions); volatile
      // keeps loads and stores in order for a result written over its input
      asm volatile("{\n .reg .pred p;\n setp.ne.s32 p, %5, 0;\n @p ld.global.v4.u32 {%0, %1, %2, %3}, [%4];\n}\n"
                   : "+r"(w[0]), "+r"(w[1]), "+r"(w[2]), "+r"(w[3])
                   : "l"(p), "r"(n)
                   : "memory");
    } else {
      asm volatile("{\n .reg .pred p;\n setp.ne.s32 p, %3, 0;\n @p ld.global.v2.u32 {%0, %1}, [%2];\n}\n"
                   : "+r"(w[0]), "+r"(w[1])
                   : "l"(p), "r"(n)
                   : "memory");
    }
  }
  __device__ __forceinline__ f2 get(int i) const {  // elements 2 i and 2 i + 1
    if constexpr (FAST && sizeof(T) == 2) return pair(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    else return pair(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
  }
};

__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

template <typename T, int V, bool FAST>
__device__ __forceinline__ void store_vec(T* p, const f2 (&x)[V / 2], int n) {
  float v[V];
#pragma unroll
  for (int i = 0; i < V / 2; ++i) halves(x[i], v[2 * i], v[2 * i + 1]);
  if constexpr (!FAST) {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n) put(p + i, v[i]);
  } else if constexpr (sizeof(T) == 4) {
    asm volatile("{\n .reg .pred p;\n setp.ne.s32 p, %5, 0;\n @p st.global.v4.f32 [%4], {%0, %1, %2, %3};\n}\n" ::"f"(v[0]), "f"(v[1]),
                 "f"(v[2]), "f"(v[3]), "l"(p), "r"(n)
                 : "memory");
  } else {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
    asm volatile("{\n .reg .pred p;\n setp.ne.s32 p, %3, 0;\n @p st.global.v2.u32 [%2], {%0, %1};\n}\n" ::"r"(
                     *reinterpret_cast<const uint32_t*>(&a)),
                 "r"(*reinterpret_cast<const uint32_t*>(&b)), "l"(p), "r"(n)
                 : "memory");
  }
}

template <typename T, int V, int NU, bool FAST>
struct Row {
  Vec<T, V, FAST> a[NU], b[NU];
};

template <typename T, int V, int NU, bool FAST, bool INTER, int MODE, int LANES>
__global__ void __launch_bounds__(THREADS, MODE == ROTATE ? 4 : (MODE == NORM ? 3 : 2)) heads_kernel(const __grid_constant__ Args A) {
  constexpr int BATCH = NU > 1 ? 1 : (MODE == NORM_GRAD || sizeof(T) == 4 ? 2 : 4);
  constexpr int P = V / 2;  // f32x2 values per vector
  __shared__ uint64_t freq[B200_ROTARY_MAX_DIM / 2];
  const int half = A.part / 2;
  __shared__ float gamma[MODE == ROTATE ? 1 : 2][MODE == ROTATE ? 1 : B200_ROTARY_MAX_DIM];
  for (int i = threadIdx.x; i < half; i += THREADS) freq[i] = A.freq[i];
  if constexpr (MODE != ROTATE) {
    const int dt = A.gamma_bf16 ? B200_BF16 : B200_F32;
    for (int i = threadIdx.x; i < 2 * B200_ROTARY_MAX_DIM; i += THREADS) {
      const int t = i / B200_ROTARY_MAX_DIM, d = i % B200_ROTARY_MAX_DIM;
      gamma[t][d] = A.seg[t].gamma && d < A.dim ? load_as_f32(A.seg[t].gamma, d, dt) : 1.f;
    }
  }
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int L = LANES ? LANES : A.L, sub = lane / L, u0 = lane % L, R = 32 / L;
  // this lane's units: element offsets, how many elements of each vector exist, first pair
  int o0[NU], o1[NU], n0[NU], n1[NU], f0[NU];
  bool rot[NU], rot_b[NU];  // whether the unit's first vector turns, and its second
#pragma unroll
  for (int k = 0; k < NU; ++k) {
    const int u = sub < R ? u0 + L * k : A.n_units;  // lanes beyond the last whole head have none
    rot[k] = u < A.n_rot;
    f0[k] = u * V;
    rot_b[k] = rot[k];
    if (INTER) {
      o0[k] = 2 * u * V;
      o1[k] = o0[k] + V;
      rot[k] = o0[k] < A.part;
      rot_b[k] = o1[k] < A.part;
      n0[k] = u < A.n_units ? max(0, min(V, A.dim - o0[k])) : 0;
      n1[k] = u < A.n_units ? max(0, min(V, A.dim - o1[k])) : 0;
    } else if (rot[k]) {
      o0[k] = u * V;
      o1[k] = half + u * V;
      n0[k] = n1[k] = min(V, half - u * V);
    } else {
      o0[k] = A.part + 2 * (u - A.n_rot) * V;
      o1[k] = o0[k] + V;
      n0[k] = u < A.n_units ? max(0, min(V, A.dim - o0[k])) : 0;
      n1[k] = u < A.n_units ? max(0, min(V, A.dim - o1[k])) : 0;
    }
  }
  f2 acc[2][2][NU][P];  // [tensor][vector][unit][elements]: sums of g u
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int k = 0; k < NU; ++k)
#pragma unroll
      for (int i = 0; i < P; ++i) acc[t][0][k][i] = acc[t][1][k][i] = 0;
  const float inv_dim = 1.f / (float)A.dim;
  const int total_groups = A.seg[0].groups + A.seg[1].groups;
  const int64_t items = (int64_t)A.tokens * A.chunks;
  for (int64_t item = (int64_t)blockIdx.x * WARPS + warp; item < items; item += (int64_t)gridDim.x * WARPS) {
    const int token = A.chunks == 1 ? (int)item : (int)(item / A.chunks), chunk = (int)(item - (int64_t)token * A.chunks);
    const int bt = token / A.seq, st = token - bt * A.seq;
    const int g_begin = chunk * A.per_chunk, g_end = min(total_groups, g_begin + A.per_chunk);
    Row<T, V, NU, FAST> xr[BATCH], dr[BATCH];
    const T *xp = nullptr, *dp = nullptr;  // this lane's head of the next group to load
    int head = 0;
    // the pointers of one tensor from group g on
    auto point = [&](const Seg& S, int g) {
      head = g * R + sub;
      xp = reinterpret_cast<const T*>(S.x) + bt * S.x_b + st * S.x_s + head * S.x_h;
      if constexpr (MODE == NORM_GRAD) dp = reinterpret_cast<const T*>(S.dy) + bt * S.d_b + st * S.d_s + head * S.d_h;
    };
    // BATCH groups of heads; `end`: the heads that this warp has to do end before it
    auto fetch = [&](const Seg& S, int end) {
#pragma unroll
      for (int j = 0; j < BATCH; ++j) {
        const bool in = head < end;
#pragma unroll
        for (int k = 0; k < NU; ++k) {
          xr[j].a[k].load(xp + o0[k], in ? n0[k] : 0);
          xr[j].b[k].load(xp + o1[k], in ? n1[k] : 0);
          if constexpr (MODE == NORM_GRAD) {
            dr[j].a[k].load(dp + o0[k], in ? n0[k] : 0);
            dr[j].b[k].load(dp + o1[k], in ? n1[k] : 0);
          }
        }
        head += R;
        xp += R * S.x_h;
        if constexpr (MODE == NORM_GRAD) dp += R * S.d_h;
      }
    };
    const int t_first = g_begin < A.seg[0].groups ? 0 : 1;
    {
      const Seg& S = A.seg[t_first];
      const int first = t_first ? A.seg[0].groups : 0;
      point(S, g_begin - first);
      fetch(S, min(S.heads, (g_end - first) * R));
    }
    int64_t p = A.offset + st;
    if (A.pos) {
      const int64_t i = bt * A.pos_b + st * A.pos_s;
      p = A.pos_i32 ? (int64_t) reinterpret_cast<const int*>(A.pos)[i] : reinterpret_cast<const long long*>(A.pos)[i];
    }
    // y = x k1 + partner k2, the partner being the other vector, or each pair's other element
    f2 k1[2][NU][P], k2[2][NU][P];
#pragma unroll
    for (int k = 0; k < NU; ++k) {
      float c[V], s[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        c[i] = 1.f;
        s[i] = 0.f;
        if (rot[k] && f0[k] + i < half) {
          cos_sin((uint64_t)p * freq[f0[k] + i], c[i], s[i]);
          c[i] *= A.factor;
          s[i] *= A.factor * A.sign;
        }
      }
#pragma unroll
      for (int i = 0; i < P; ++i) {
        if constexpr (INTER) {
          k1[0][k][i] = pair(c[i], c[i]);
          k2[0][k][i] = pair(-s[i], s[i]);
          k1[1][k][i] = pair(c[P + i], c[P + i]);
          k2[1][k][i] = pair(-s[P + i], s[P + i]);
        } else {
          k1[0][k][i] = k1[1][k][i] = pair(c[2 * i], c[2 * i + 1]);
          k2[0][k][i] = pair(-s[2 * i], -s[2 * i + 1]);
          k2[1][k][i] = pair(s[2 * i], s[2 * i + 1]);
        }
      }
    }
    auto turn = [&](f2 (&a)[NU][P], f2 (&b)[NU][P], const f2 (&m1)[2][NU][P], const f2 (&m2)[2][NU][P]) {
#pragma unroll
      for (int k = 0; k < NU; ++k)
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const f2 x = a[k][i], y = b[k][i];
          a[k][i] = mul2(x, m1[0][k][i]);
          b[k][i] = mul2(y, m1[1][k][i]);
          // elements that only pass see nothing of a partner
          if (rot[k]) a[k][i] = fma2(INTER ? swapped(x) : y, m2[0][k][i], a[k][i]);
          if (INTER ? rot_b[k] : rot[k]) b[k][i] = fma2(INTER ? swapped(y) : x, m2[1][k][i], b[k][i]);
        }
    };
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const Seg& S = A.seg[t];
      const int first = t == 0 ? 0 : A.seg[0].groups;
      const int lo = max(0, g_begin - first), hi = min(S.groups, g_end - first);
      if (lo >= hi) continue;
      const int end = min(S.heads, hi * R);
      f2 gam[2][NU][P], w1[2][NU][P], w2[2][NU][P];  // the weights; the coefficients with them
      if constexpr (MODE != ROTATE) {
#pragma unroll
        for (int k = 0; k < NU; ++k)
#pragma unroll
          for (int i = 0; i < P; ++i) {
            // beyond the head: any weight will do, the elements are zeros and are not stored
            const int ia = min(o0[k] + 2 * i, B200_ROTARY_MAX_DIM - 2), ib = min(o1[k] + 2 * i, B200_ROTARY_MAX_DIM - 2);
            const f2 ga = gam[0][k][i] = pair(gamma[t][ia], gamma[t][ia + 1]);
            const f2 gb = gam[1][k][i] = pair(gamma[t][ib], gamma[t][ib + 1]);
            if constexpr (MODE == NORM) {
              w1[0][k][i] = mul2(k1[0][k][i], ga);
              w1[1][k][i] = mul2(k1[1][k][i], gb);
              w2[0][k][i] = mul2(k2[0][k][i], INTER ? swapped(ga) : gb);
              w2[1][k][i] = mul2(k2[1][k][i], INTER ? swapped(gb) : ga);
            }
          }
      }
      if (t != t_first) point(S, lo);
      int out = lo * R + sub;
      T* yp = reinterpret_cast<T*>(S.y) + bt * S.y_b + st * S.y_s + out * S.y_h;
      // The gradient's few warps keep the next batch's loads in flight; the other modes load
      // a batch and work on it (more warps, and more rows a batch, do as well there).
      constexpr bool AHEAD = MODE == NORM_GRAD && NU == 1;
      if (AHEAD && t != t_first) fetch(S, end);
      for (int g = lo; g < hi; g += BATCH) {
        Row<T, V, NU, FAST> xc[BATCH], dc[BATCH];
        if (!AHEAD && (t != t_first || g != lo)) fetch(S, end);
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
          xc[j] = xr[j];
          if constexpr (MODE == NORM_GRAD) dc[j] = dr[j];
        }
        if (AHEAD && g + BATCH < hi) fetch(S, end);
        auto work = [&](int j) {
          f2 a[NU][P], b[NU][P];
          f2 ss = 0;
#pragma unroll
          for (int k = 0; k < NU; ++k)
#pragma unroll
            for (int i = 0; i < P; ++i) {
              a[k][i] = xc[j].a[k].get(i);
              b[k][i] = xc[j].b[k].get(i);
              if constexpr (MODE != ROTATE) ss = fma2(a[k][i], a[k][i], fma2(b[k][i], b[k][i], ss));
            }
          if constexpr (MODE == ROTATE) {
            turn(a, b, k1, k2);
          } else if constexpr (MODE == NORM) {
            float sq = sum2(ss);
            #pragma unroll
            for (int o = L >> 1; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
            const float rstd = rsqrtf(sq * inv_dim + A.eps);
            const f2 r2 = pair(rstd, rstd);
            turn(a, b, w1, w2);
#pragma unroll
            for (int k = 0; k < NU; ++k)
#pragma unroll
              for (int i = 0; i < P; ++i) {
                a[k][i] = mul2(a[k][i], r2);
                b[k][i] = mul2(b[k][i], r2);
              }
          } else {
            f2 ga[NU][P], gb[NU][P];
#pragma unroll
            for (int k = 0; k < NU; ++k)
#pragma unroll
              for (int i = 0; i < P; ++i) {
                ga[k][i] = dc[j].a[k].get(i);
                gb[k][i] = dc[j].b[k].get(i);
              }
            turn(ga, gb, k1, k2);
            f2 hh = 0;
#pragma unroll
            for (int k = 0; k < NU; ++k)
#pragma unroll
              for (int i = 0; i < P; ++i)
                hh = fma2(mul2(ga[k][i], gam[0][k][i]), a[k][i], fma2(mul2(gb[k][i], gam[1][k][i]), b[k][i], hh));
            float sq = sum2(ss), hx = sum2(hh);
#pragma unroll
            for (int o = L >> 1; o > 0; o >>= 1) {
              sq += __shfl_xor_sync(0xffffffffu, sq, o);
              hx += __shfl_xor_sync(0xffffffffu, hx, o);
            }
            const float rstd = rsqrtf(sq * inv_dim + A.eps);
            const float m = -hx * inv_dim * rstd * rstd * rstd;  // -rstd mean(h u) / (u / x)
            const f2 r2 = pair(rstd, rstd), m2 = pair(m, m);
#pragma unroll
            for (int k = 0; k < NU; ++k)
#pragma unroll
              for (int i = 0; i < P; ++i) {
                ga[k][i] = mul2(ga[k][i], r2);  // rstd g
                gb[k][i] = mul2(gb[k][i], r2);
                acc[t][0][k][i] = fma2(ga[k][i], a[k][i], acc[t][0][k][i]);
                acc[t][1][k][i] = fma2(gb[k][i], b[k][i], acc[t][1][k][i]);
                a[k][i] = fma2(ga[k][i], gam[0][k][i], mul2(a[k][i], m2));
                b[k][i] = fma2(gb[k][i], gam[1][k][i], mul2(b[k][i], m2));
              }
          }
#pragma unroll
          for (int k = 0; k < NU; ++k) {
            store_vec<T, V, FAST>(yp + o0[k], a[k], out < end ? n0[k] : 0);
            store_vec<T, V, FAST>(yp + o1[k], b[k], out < end ? n1[k] : 0);
          }
          out += R;
          yp += R * S.y_h;
        };
        // whole batches without a branch between their rows, so that one's shuffles hide another's
        if (g + BATCH <= hi) {
#pragma unroll
          for (int j = 0; j < BATCH; ++j) work(j);
        } else {
#pragma unroll
          for (int j = 0; j < BATCH; ++j) {
            if (g + j >= hi) break;  // warp-uniform
            work(j);
          }
        }
      }
    }
  }
  if constexpr (MODE == NORM_GRAD) {
    // the block's sums: over the warp's R heads by shuffles, over its warps in order
    __shared__ float sums[WARPS][B200_ROTARY_MAX_DIM];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < NU; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float a, b, x0, x1, y0, y1;
          halves(acc[t][0][k][i / 2], x0, x1);
          halves(acc[t][1][k][i / 2], y0, y1);
          a = i & 1 ? x1 : x0;
          b = i & 1 ? y1 : y0;
          for (int o = L; o < 32; o <<= 1) {
            a += __shfl_xor_sync(0xffffffffu, a, o);
            b += __shfl_xor_sync(0xffffffffu, b, o);
          }
          if (sub == 0) {
            if (i < n0[k]) sums[warp][o0[k] + i] = a;
            if (i < n1[k]) sums[warp][o1[k] + i] = b;
          }
        }
      __syncthreads();
      for (int d = threadIdx.x; d < A.dim; d += THREADS) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) v += sums[w][d];
        A.partial[((int64_t)blockIdx.x * 2 + t) * A.dim + d] = v;
      }
    }
  }
}

// dgamma of both tensors from the blocks' partials, added in block order by 8 threads per
// column and a fixed tree
__global__ void __launch_bounds__(256) gamma_sum_kernel(const float* __restrict__ partial, float* dgq, float* dgk, int dim, int blocks) {
  __shared__ float red[8][33];
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), part = threadIdx.x >> 5;
  float v = 0.f;
  if (col < 2 * dim)
    for (int b = part; b < blocks; b += 8) v += partial[(int64_t)b * 2 * dim + col];
  red[part][threadIdx.x & 31] = v;
  __syncthreads();
  if (part == 0 && col < 2 * dim) {
#pragma unroll
    for (int i = 1; i < 8; ++i) v += red[i][threadIdx.x];
    float* out = col < dim ? dgq : dgk;
    if (out) out[col < dim ? col : col - dim] = v;
  }
}

template <typename T, int V, int NU, bool FAST, int MODE, int LANES = 0>
static int launch(const Args& a, bool inter, int grid, cudaStream_t s) {
  if (inter) heads_kernel<T, V, NU, FAST, true, MODE, LANES><<<grid, THREADS, 0, s>>>(a);
  else heads_kernel<T, V, NU, FAST, false, MODE, LANES><<<grid, THREADS, 0, s>>>(a);
  return check_launch(MODE == ROTATE ? "rotary" : (MODE == NORM ? "qk_norm_rotary" : "qk_norm_rotary_grad"));
}

// heads of up to 256 elements in whole vectors; the norms' reductions over 8 or 16 lanes (heads
// of 64 or 128) are unrolled
template <typename T, int MODE>
static int launch_fast(const Args& a, bool inter, int grid, cudaStream_t s) {
  if constexpr (MODE != ROTATE) {
    if (a.L == 8) return launch<T, 4, 1, true, MODE, 8>(a, inter, grid, s);
    if (a.L == 16) return launch<T, 4, 1, true, MODE, 16>(a, inter, grid, s);
  }
  return launch<T, 4, 1, true, MODE>(a, inter, grid, s);
}

// Units a lane: a head of 512 elements is 64 units of whole vectors, or up to 129 of 2-element
// vectors; an idle unit costs as much as a full one.
template <typename T, int MODE>
static int launch_type(const Args& a, bool fast, int nu, bool inter, int grid, cudaStream_t s) {
  if (nu > (fast ? 2 : 5)) {
    set_error("rotary: %d units a head, more than any kernel takes", a.n_units);
    return B200_ERR_UNSUPPORTED;
  }
  if (fast) return nu == 1 ? launch_fast<T, MODE>(a, inter, grid, s) : launch<T, 4, 2, true, MODE>(a, inter, grid, s);
  if (nu == 1) return launch<T, 2, 1, false, MODE>(a, inter, grid, s);
  if (nu == 2) return launch<T, 2, 2, false, MODE>(a, inter, grid, s);
  return nu == 3 ? launch<T, 2, 3, false, MODE>(a, inter, grid, s) : launch<T, 2, 5, false, MODE>(a, inter, grid, s);
}

static int grad_blocks() { return 2 * num_sms(); }

template <int MODE>
static int run(const b200_rotary* r, int dtype, Args& a, cudaStream_t s, int* blocks_out = nullptr) {
  const int size = dtype == B200_F32 ? 4 : 2;
  const int wide = 4;
  const int half = r->rotary_dim / 2, rest = r->head_dim - r->rotary_dim;
  // vectors of 4 elements when they tile the head's parts and every row starts on one's
  // boundary; otherwise units of 2 elements, loaded one by one (16 x 1024 x 8 x 128 bf16: 15 us
  // with 64 rotated, 33 with 62 by halves, 23 with 62 interleaved; staging whole rows through shared
  // memory took 40)
  bool fast = rest % wide == 0 && (r->interleaved ? r->rotary_dim : half) % wide == 0;
  for (const Seg& g : a.seg) {
    if (!g.heads) continue;
    uint64_t bits = reinterpret_cast<uintptr_t>(g.x) | reinterpret_cast<uintptr_t>(g.y) | reinterpret_cast<uintptr_t>(g.dy);
    bits |= (uint64_t)(g.x_b | g.x_s | g.x_h | g.y_b | g.y_s | g.y_h | g.d_b | g.d_s | g.d_h) * (uint64_t)size;
    if (bits & (uint64_t)(wide * size - 1)) fast = false;
  }
  const int V = fast ? wide : 2;
  // (interleaved, a unit may hold the rotated part's last vector and the first that passes)
  a.n_rot = (int)ceil_div(half, V);
  a.n_units = r->interleaved ? (int)ceil_div(r->head_dim, 2 * V) : a.n_rot + (int)ceil_div(rest, 2 * V);
  a.L = 1;
  while (a.L < a.n_units && a.L < 32) a.L *= 2;
  // without a reduction the lanes of a head need be no power of two: three heads of 10 units
  // share a warp instead of two
  if (MODE == ROTATE && a.n_units <= 32) a.L = std::max(1, a.n_units);
  const int nu = (int)ceil_div(a.n_units, a.L);
  const int R = 32 / a.L;
  for (Seg& g : a.seg) g.groups = (int)ceil_div(g.heads, R);
  const int groups = a.seg[0].groups + a.seg[1].groups;
  // one warp per token while the tokens fill the SMs (32 warps each); below that a token's
  // head groups are spread over as many warps as it takes
  const int64_t want = ceil_div((int64_t)num_sms() * 32, a.tokens);
  a.chunks = (int)std::max<int64_t>(1, std::min<int64_t>(groups, want));
  a.per_chunk = (int)ceil_div(groups, a.chunks);
  a.chunks = (int)ceil_div(groups, a.per_chunk);
  const int64_t blocks = ceil_div((int64_t)a.tokens * a.chunks, WARPS);
  const int grid = (int)std::min<int64_t>(blocks, MODE == NORM_GRAD ? grad_blocks() : 16 * num_sms());
  if (blocks_out) *blocks_out = grid;
  return dtype == B200_F32 ? launch_type<float, MODE>(a, fast, nu, r->interleaved, grid, s)
                           : launch_type<__nv_bfloat16, MODE>(a, fast, nu, r->interleaved, grid, s);
}

static int check_rotary(const char* what, const b200_rotary* r, int dtype, int64_t batch, int64_t seq, const void* pos, int pos_dtype) {
  B200_REQUIRE(r, "%s: null rotary description", what);
  B200_REQUIRE(r->head_dim >= 1 && r->head_dim <= B200_ROTARY_MAX_DIM, "%s: head_dim %d not in [1, %d]", what, r->head_dim,
               B200_ROTARY_MAX_DIM);
  B200_REQUIRE(r->rotary_dim >= 0 && r->rotary_dim <= r->head_dim && r->rotary_dim % 2 == 0,
               "%s: rotary_dim %d must be even and in [0, head_dim = %d]", what, r->rotary_dim, r->head_dim);
  B200_REQUIRE(batch >= 0 && seq >= 0, "%s: negative size", what);
  B200_REQUIRE(batch == 0 || seq <= INT32_MAX / batch, "%s: more than 2^31 - 1 tokens", what);
  if (dtype != B200_F32 && dtype != B200_BF16) {
    set_error("%s: dtype %d (fp32 and bf16 heads)", what, dtype);
    return B200_ERR_DTYPE;
  }
  if (pos && pos_dtype != B200_I64 && pos_dtype != B200_I32) {
    set_error("%s: positions of dtype %d (int32 and int64)", what, pos_dtype);
    return B200_ERR_DTYPE;
  }
  return B200_OK;
}

static int check_norm(const char* what, int64_t heads_q, int64_t heads_k, bool gamma, int gamma_dtype, float eps) {
  B200_REQUIRE(heads_q >= 0 && heads_k >= 0 && heads_q <= 65535 && heads_k <= 65535, "%s: %lld and %lld heads not in [0, 65535]", what,
               (long long)heads_q, (long long)heads_k);
  B200_REQUIRE(eps >= 0.f, "%s: eps %g is negative", what, (double)eps);
  if (gamma && gamma_dtype != B200_F32 && gamma_dtype != B200_BF16) {
    set_error("%s: weights of dtype %d (fp32 and bf16)", what, gamma_dtype);
    return B200_ERR_DTYPE;
  }
  return B200_OK;
}

static void fill(Args& a, const b200_rotary* r, int64_t batch, int64_t seq, const void* pos, int pos_dtype, int64_t pos_b,
                 int64_t pos_s, int64_t offset) {
  a.pos = pos;
  a.pos_i32 = pos_dtype == B200_I32;
  a.pos_b = pos_b;
  a.pos_s = pos_s;
  a.offset = offset;
  a.tokens = (int)(batch * seq);
  a.seq = (int)seq;
  a.dim = r->head_dim;
  a.part = r->rotary_dim;
  a.factor = r->factor;
  a.sign = 1.f;
  for (int i = 0; i < r->rotary_dim / 2; ++i) a.freq[i] = r->turns[i];
}

}  // namespace rot
}  // namespace b200

using namespace b200;

extern "C" int b200_rotary_heads(const b200_rotary* r, int dtype, const void* x, void* y, int64_t batch, int64_t seq, int64_t heads,
                                 int64_t x_b, int64_t x_s, int64_t x_h, int64_t y_b, int64_t y_s, int64_t y_h, const void* positions,
                                 int pos_dtype, int64_t pos_b, int64_t pos_s, int64_t offset, int inverse, void* stream) {
  const int rc = rot::check_rotary("rotary", r, dtype, batch, seq, positions, pos_dtype);
  if (rc) return rc;
  B200_REQUIRE(heads >= 0 && heads <= 65535, "rotary: %lld heads not in [0, 65535]", (long long)heads);
  if (batch == 0 || seq == 0 || heads == 0) return B200_OK;
  B200_REQUIRE(x && y, "rotary: null tensor");
  rot::Args a = {};
  rot::fill(a, r, batch, seq, positions, pos_dtype, pos_b, pos_s, offset);
  if (inverse) a.sign = -1.f;
  a.seg[0] = {x, nullptr, y, x_b, x_s, x_h, 0, 0, 0, y_b, y_s, y_h, nullptr, (int)heads, 0};
  return rot::run<rot::ROTATE>(r, dtype, a, as_stream(stream));
}

extern "C" int b200_qk_norm_rotary(const b200_rotary* r, int dtype, const void* q, const void* k, void* yq, void* yk, int64_t batch,
                                   int64_t seq, int64_t heads_q, int64_t heads_k, int64_t q_b, int64_t q_s, int64_t q_h, int64_t k_b,
                                   int64_t k_s, int64_t k_h, int64_t yq_b, int64_t yq_s, int64_t yq_h, int64_t yk_b, int64_t yk_s,
                                   int64_t yk_h, const void* gamma_q, const void* gamma_k, int gamma_dtype, float eps,
                                   const void* positions, int pos_dtype, int64_t pos_b, int64_t pos_s, int64_t offset, void* stream) {
  int rc = rot::check_rotary("qk_norm_rotary", r, dtype, batch, seq, positions, pos_dtype);
  if (!rc) rc = rot::check_norm("qk_norm_rotary", heads_q, heads_k, gamma_q || gamma_k, gamma_dtype, eps);
  if (rc) return rc;
  if (batch == 0 || seq == 0 || heads_q + heads_k == 0) return B200_OK;
  B200_REQUIRE((!heads_q || (q && yq)) && (!heads_k || (k && yk)), "qk_norm_rotary: null tensor");
  rot::Args a = {};
  rot::fill(a, r, batch, seq, positions, pos_dtype, pos_b, pos_s, offset);
  a.eps = eps;
  a.gamma_bf16 = gamma_dtype == B200_BF16;
  a.seg[0] = {q, nullptr, yq, q_b, q_s, q_h, 0, 0, 0, yq_b, yq_s, yq_h, gamma_q, (int)heads_q, 0};
  a.seg[1] = {k, nullptr, yk, k_b, k_s, k_h, 0, 0, 0, yk_b, yk_s, yk_h, gamma_k, (int)heads_k, 0};
  return rot::run<rot::NORM>(r, dtype, a, as_stream(stream));
}

extern "C" size_t b200_qk_norm_rotary_grad_workspace_bytes(int64_t head_dim) {
  return head_dim > 0 ? (size_t)rot::grad_blocks() * 2 * (size_t)head_dim * sizeof(float) : 0;
}

extern "C" int b200_qk_norm_rotary_grad(const b200_rotary* r, int dtype, const void* dyq, const void* dyk, const void* q, const void* k,
                                        void* dq, void* dk, int64_t batch, int64_t seq, int64_t heads_q, int64_t heads_k,
                                        const int64_t* strides, const void* gamma_q, const void* gamma_k, int gamma_dtype, float eps,
                                        const void* positions, int pos_dtype, int64_t pos_b, int64_t pos_s, int64_t offset,
                                        float* dgamma_q, float* dgamma_k, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = rot::check_rotary("qk_norm_rotary_grad", r, dtype, batch, seq, positions, pos_dtype);
  if (!rc) rc = rot::check_norm("qk_norm_rotary_grad", heads_q, heads_k, gamma_q || gamma_k, gamma_dtype, eps);
  if (rc) return rc;
  B200_REQUIRE(strides, "qk_norm_rotary_grad: null strides");
  cudaStream_t s = as_stream(stream);
  if (batch == 0 || seq == 0 || heads_q + heads_k == 0) {
    for (float* g : {dgamma_q, dgamma_k})
      if (g && cudaMemsetAsync(g, 0, (size_t)r->head_dim * sizeof(float), s) != cudaSuccess) return check_launch("qk_norm_rotary_grad");
    return B200_OK;
  }
  B200_REQUIRE((!heads_q || (q && dyq && dq)) && (!heads_k || (k && dyk && dk)), "qk_norm_rotary_grad: null tensor");
  B200_REQUIRE(workspace && workspace_bytes >= b200_qk_norm_rotary_grad_workspace_bytes(r->head_dim) &&
                   reinterpret_cast<uintptr_t>(workspace) % alignof(float) == 0,
               "qk_norm_rotary_grad: workspace of %zu bytes, %zu needed (4-byte aligned)", workspace_bytes,
               b200_qk_norm_rotary_grad_workspace_bytes(r->head_dim));
  rot::Args a = {};
  rot::fill(a, r, batch, seq, positions, pos_dtype, pos_b, pos_s, offset);
  a.sign = -1.f;
  // Lanes beyond the last head carry zeros into the sums. Without eps their rstd would be infinite,
  // and 0 * inf NaN; the smallest number that is not zero makes it 2.7e22 and changes no mean square of
  // 2^-124 or more. (A select per row in the kernel cost 1 % of its time.)
  a.eps = std::max(eps, std::numeric_limits<float>::denorm_min());
  a.gamma_bf16 = gamma_dtype == B200_BF16;
  a.partial = reinterpret_cast<float*>(workspace);
  const int64_t* t = strides;
  a.seg[0] = {q, dyq, dq, t[0], t[1], t[2], t[3], t[4], t[5], t[6], t[7], t[8], gamma_q, (int)heads_q, 0};
  t += 9;
  a.seg[1] = {k, dyk, dk, t[0], t[1], t[2], t[3], t[4], t[5], t[6], t[7], t[8], gamma_k, (int)heads_k, 0};
  int blocks = 0;
  rc = rot::run<rot::NORM_GRAD>(r, dtype, a, s, &blocks);
  if (rc || (!dgamma_q && !dgamma_k)) return rc;
  rot::gamma_sum_kernel<<<(unsigned)ceil_div(2 * a.dim, 32), 256, 0, s>>>(a.partial, dgamma_q, dgamma_k, a.dim, blocks);
  return check_launch("qk_norm_rotary_grad sums");
}
