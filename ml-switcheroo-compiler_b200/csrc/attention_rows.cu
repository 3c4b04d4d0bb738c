// Attention on the CUDA cores: few queries against a long cache, fp32, heads of any size.
//
// A block holds R rows (queries of the heads that share a key head; for dk and dv, keys) and its
// four warps stream the other side past them, KEYS = 32 / R tokens a step, each warp steps of its own.
// The lanes of a warp lie over the head's elements (E each), so a token is one coalesced load and no
// shared memory. A step has R x KEYS = 32 scores, one a lane in the end: every lane sums its elements
// of all 32, then 16 + 8 + 4 + 2 + 1 exchanges leave score l in lane l, where mask, bias and exponential
// are done once each; the probabilities go back to all lanes through 128 bytes of shared memory a warp.
// Forward: running maximum and sum per row (exp2 in the log2 domain), the warps' results joined at the end;
// where rows leave SMs idle the keys are split over blocks and a second launch joins the parts.
// Backward: p = exp2(z - lse) made again; dq has rows of queries, dk and dv rows of keys, so every sum
// stays in registers, in a fixed order. Everything is fp32.
// bf16 queries (rows of whole 16 bytes) make their scores by mma.sync instead, 8 tokens a step, whose operands a lane loads as
// they are: without the sums over lanes and the conversions of K a step has half the instructions.
// What bounds it: for single tokens latency and issue on the way to HBM (32 caches of 4096 places, 32 + 8 heads of 128 bf16: 96 us, 4.2
// TB/s; 661 us with loads that waited behind branches, 132 without mma.sync), else issue: of 2 x 777 tokens, 8 heads of 80 fp32 the
// forward takes 190, dq 257, dk and dv 322 us, with 61, 59 and 54 % of the issue slots in use but the FMA pipe only for 34, 33 and
// 34 %. The rest are the sums over lanes (31 exchanges and 62 selects for 32 scores, twice in the gradients), the probabilities' way
// through shared memory, and 48 of 128 lanes' elements behind a head of 80. Heads above 128 spill: 168 to 1360 bytes a thread.
#include <algorithm>

#include "attention.cuh"

namespace b200 {
namespace attention {
namespace rows {

constexpr int WARPS = 4, THREADS = 32 * WARPS;
constexpr int FWD = 0, DQ = 1, DKV = 2;
constexpr int AREA = 80;  // floats that a warp hands scores round by

struct Io {
  int64_t out_rows;             // blocks of rows of one (batch, head or key head)
  int splits;                   // FWD: blocks that share a row block's keys
  int vec;                      // vector loads: 16-byte aligned tokens, dim a multiple of the lane's elements
  void* out;                    // FWD: out; DQ: dq; DKV: dk
  void* out2;                   // DKV: dv
  float* lse;                   // FWD: written; else read
  const void* dout;
  int64_t dout_stride[3];
  const float* delta;           // [batch x heads][padded], negated
  int64_t padded;
  float* part;                  // FWD with splits: [row blocks][splits][R][dim + 2]; DQ with a table: [row blocks][buckets]
};

// A lane's E elements of a token as they are in memory. Lanes behind the head's end read its first elements, whose factors are
// zero, and tokens behind the last are the last again: no load waits behind a branch.
template <typename T, int E>
struct Token {
  static constexpr int WORDS = E * (int)sizeof(T) / 4;
  uint32_t w[WORDS];

  __device__ __forceinline__ void load(const T* p, int c, int dim, int vec) {
    if (vec) {
      const uint32_t* q = reinterpret_cast<const uint32_t*>(p + (c < dim ? c : 0));
      if constexpr (WORDS == 1) {
        w[0] = *q;
      } else if constexpr (WORDS == 2) {
        const uint2 u = *reinterpret_cast<const uint2*>(q);
        w[0] = u.x, w[1] = u.y;
      } else {
#pragma unroll
        for (int i = 0; i < WORDS; i += 4) {
          const uint4 u = *reinterpret_cast<const uint4*>(q + i);
          w[i] = u.x, w[i + 1] = u.y, w[i + 2] = u.z, w[i + 3] = u.w;
        }
      }
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < E; ++i) w[i] = __float_as_uint(c + i < dim ? (float)p[c + i] : 0.f);
    } else {
#pragma unroll
      for (int i = 0; i < E / 2; ++i) {
        const __nv_bfloat162 u = __floats2bfloat162_rn(c + 2 * i < dim ? (float)p[c + 2 * i] : 0.f, c + 2 * i + 1 < dim ? (float)p[c + 2 * i + 1] : 0.f);
        w[i] = *reinterpret_cast<const uint32_t*>(&u);
      }
    }
  }
  __device__ __forceinline__ void get(float (&v)[E]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < E; ++i) v[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < E / 2; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
};
// a row that stays: zeros behind the head's end
template <typename T, int E>
__device__ __forceinline__ void load_row(float (&v)[E], const T* p, int c, int dim, int vec) {
  Token<T, E> x;
  x.load(p, c, dim, vec);
  x.get(v);
#pragma unroll
  for (int i = 0; i < E; ++i)
    if (c + i >= dim) v[i] = 0.f;
}
template <int E>
__device__ __forceinline__ void zero(float (&v)[E]) {
#pragma unroll
  for (int i = 0; i < E; ++i) v[i] = 0.f;
}

// D += A B for 16 rows, 8 columns and 16 elements in bf16; rows 8 to 15 of A are zeros
__device__ __forceinline__ void mma_16x8(float& d0, float& d1, float& d2, float& d3, uint32_t a0, uint32_t a2, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d0), "+f"(d1), "+f"(d2), "+f"(d3)
      : "r"(a0), "r"(0), "r"(a2), "r"(0), "r"(b0), "r"(b1));
}

// 32 values a lane -> the sum over lanes of value `lane`
__device__ __forceinline__ float sum_to_lane(float (&v)[32], int lane) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const bool up = lane & o;
      const float send = up ? v[i] : v[i + o], keep = up ? v[i + o] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
    }
  return v[0];
}

template <typename T, int E, int R, int MODE, bool MMA>
__global__ void __launch_bounds__(THREADS, MODE == DKV ? 2 : (MMA ? 4 : 3))
    rows_kernel(const __grid_constant__ b200_attention a, const __grid_constant__ Io io) {
  static_assert(!MMA || (MODE == FWD && sizeof(T) == 2), "queries of bf16");
  // tokens of a step, lanes that share a row's scores
  constexpr int KEYS = MMA ? 8 : 32 / R, LANES = MMA ? 4 : KEYS;
  extern __shared__ __align__(16) uint8_t smem[];
  float* s_p = reinterpret_cast<float*>(smem);             // [WARPS][AREA]: p; corrections or dz
  float* s_join = s_p + WARPS * AREA;                        // [WARPS][R][32 E] (DKV: twice), then FWD's m and l [WARPS][R] each
  constexpr int JOIN = WARPS * R * 32 * E * (MODE == DKV ? 2 : 1) + 2 * WARPS * R;
  float* s_near = s_join + JOIN;                           // DQ with a table: [WARPS][2 far + 1] sums by rel
  const int far = a.table ? relative::far_of(a.relative) : 0;
  const int bins = 2 * far + 1;
  uint8_t* s_bucket = reinterpret_cast<uint8_t*>(s_near + (MODE == DQ && a.table ? WARPS * bins : 0));  // [2 far + 1]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane * E;
  const int group = (int)(a.heads / a.kv_heads), dim = (int)a.dim;
  const int64_t b = blockIdx.z;
  const int hy = blockIdx.y;  // key head (FWD, DKV) or head (DQ)
  const int kvh = MODE == DQ ? hy / group : hy;
  const Sequence seq(a, b);
  const int rb = MODE == FWD ? (int)(blockIdx.x / io.splits) : (int)blockIdx.x, part = MODE == FWD ? (int)(blockIdx.x % io.splits) : 0;
  if (a.table) {
    for (int i = threadIdx.x; i < bins; i += THREADS) s_bucket[i] = (uint8_t)relative::bucket_of(a.relative, i - far);
    if constexpr (MODE == DQ)
      for (int i = threadIdx.x; i < WARPS * bins; i += THREADS) s_near[i] = 0.f;
    __syncthreads();
  }
  const T *q = reinterpret_cast<const T*>(a.q) + b * a.q_stride[0], *dout = reinterpret_cast<const T*>(io.dout) + (MODE == FWD ? 0 : b * io.dout_stride[0]);
  const T *k = reinterpret_cast<const T*>(a.k) + b * a.k_stride[0] + kvh * a.k_stride[2],
          *v = reinterpret_cast<const T*>(a.v) + b * a.v_stride[0] + kvh * a.v_stride[2];
  // row r of the block: its query and head, or its key
  auto row_query = [&](int r) { return MODE == FWD ? (rb * R + r) / group : rb * R + r; };
  auto row_head = [&](int r) { return MODE == FWD ? kvh * group + (rb * R + r) % group : hy; };
  const int row_end = MODE == DKV ? seq.keys : seq.queries;  // rows inside the sequence

  // this lane's score is row lr, token lk of a step (MMA: tokens 2 lk and 2 lk + 1)
  const int lr = lane / LANES, lk = lane % LANES;
  const int my_row = MODE == DKV ? rb * R + lr : row_query(lr);
  const int my_head = MODE == DKV ? 0 : row_head(lr);
  const bool my_in = my_row < row_end && lr < R;
  int lo, hi;  // tokens that this lane's row takes part with
  if (MODE == DKV) lo = my_in ? seq.first_query(a, my_row) : 0, hi = my_in ? seq.end_query(a, my_row) : 0;
  else lo = my_in ? seq.first_key(a, my_row) : 0, hi = my_in ? seq.end_key(a, my_row) : 0;
  // the block's tokens: from the smallest to the largest of its rows' (whose ranges move one way)
  int first = __reduce_min_sync(0xffffffffu, hi > lo ? lo : 0x7fffffff), end = __reduce_max_sync(0xffffffffu, hi > lo ? hi : 0);
  if (first > end) first = end;
  if (MODE == FWD && io.splits > 1) {
    const int unit = io.splits * KEYS * WARPS;
    const int each = (end - first + unit - 1) / unit * KEYS * WARPS;
    first = min(end, first + part * each);
    end = min(end, first + each);
  }

  float x1[R][E], x2[MODE == FWD ? 1 : R][E], acc[R][E], acc2[MODE == DKV ? R : 1][E];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    zero(acc[r]);
    zero(x1[r]);
    if constexpr (MODE == DKV) zero(acc2[r]);
    if constexpr (MODE != FWD) zero(x2[r]);
    if constexpr (MODE == DKV) {
      const int j = rb * R + r;
      if (j < row_end) {
        load_row<T, E>(x1[r], k + j * a.k_stride[1], c, dim, io.vec);
        load_row<T, E>(x2[r], v + j * a.v_stride[1], c, dim, io.vec);
      }
    } else {
      const int i = row_query(r), h = row_head(r);
      if (!MMA && i < row_end) {
        load_row<T, E>(x1[r], q + i * a.q_stride[1] + h * a.q_stride[2], c, dim, io.vec);
        if constexpr (MODE == DQ) load_row<T, E>(x2[r], dout + i * io.dout_stride[1] + h * io.dout_stride[2], c, dim, io.vec);
      }
    }
  }
  const float sl = a.scale * LOG2E;
  float m = -INFINITY, l = 0.f;            // FWD: this lane's row's maximum, this lane's share of its sum
  float my_lse = INFINITY, my_delta = 0.f;  // DQ
  float before = 0.f, after = 0.f;          // DQ with a table: sums of dz at rel <= -far, >= far
  if (MODE == DQ && my_in) {
    const int64_t at = (b * a.heads + my_head) * a.queries + my_row;
    my_lse = exponent_of(io.lse[at]);
    my_delta = -io.delta[(b * a.heads + my_head) * io.padded + my_row];
  }
  float* sp = s_p + warp * AREA;

  if constexpr (MMA) {
    // S = Q K^T of 8 rows and 8 tokens by mma.m16n8k16 (rows 8 to 15 are zeros). The order of the products' elements is free: lane
    // (g, t) = (lane / 4, lane % 4) brings 16 bytes of token g's elements 32 j + 8 t .. + 7 and has the same ones of row g, which
    // are two K steps of 16 elements. So a token goes from its load to the tensor core as it is.
    const int g8 = lane >> 2, t8 = lane & 3;
    uint4 qf[E], kf[E];
    Token<T, E> y2[KEYS];
    auto piece = [&](const T* p, int j) {  // zeros for rows, the first elements again for tokens, behind the head's end
      const int d = 32 * j + 8 * t8;
      return *reinterpret_cast<const uint4*>(p + (d < dim ? d : 0));
    };
    {
      const int i = row_query(min(g8, R - 1)), h = row_head(min(g8, R - 1));
      const bool in = g8 < R && i < row_end;
      const T* p = q + (in ? i * a.q_stride[1] + h * a.q_stride[2] : 0);
#pragma unroll
      for (int j = 0; j < E; ++j) {
        qf[j] = make_uint4(0, 0, 0, 0);
        if (in && 32 * j + 8 * t8 < dim) qf[j] = piece(p, j);
      }
    }
    auto load1 = [&](int t) {
      const T* p = k + min(t + g8, end - 1) * a.k_stride[1];
#pragma unroll
      for (int j = 0; j < E; ++j) kf[j] = piece(p, j);
    };
    auto load2 = [&](int t) {
#pragma unroll
      for (int n = 0; n < KEYS; ++n) y2[n].load(v + min(t + n, end - 1) * a.v_stride[1], c, dim, 1);
    };
    int t0 = first + warp * KEYS;
    if (t0 < end) load1(t0), load2(t0);
    for (; t0 < end; t0 += WARPS * KEYS) {
      const bool more = t0 + WARPS * KEYS < end;
      float d0 = 0.f, d1 = 0.f, d2 = 0.f, d3 = 0.f;
#pragma unroll
      for (int j = 0; j < E; ++j) {
        mma_16x8(d0, d1, d2, d3, qf[j].x, qf[j].y, kf[j].x, kf[j].y);
        mma_16x8(d0, d1, d2, d3, qf[j].z, qf[j].w, kf[j].z, kf[j].w);
      }
      if (more) load1(t0 + WARPS * KEYS);
      float s[2] = {d0 * sl, d1 * sl};
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int j = t0 + 2 * t8 + u;
        const bool seen = j < end && j >= lo && j < hi;
        if (a.table && seen)
          s[u] += table_log2(a.table, (int64_t)s_bucket[max(-far, min(far, j - my_row - seq.shift)) + far] * a.heads + my_head, a.table_dtype);
        if (!seen) s[u] = -INFINITY;
      }
      float top = fmaxf(s[0], s[1]);
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      top = fmaxf(m, top);
      const float base = top == -INFINITY ? 0.f : top;
      const float p0 = exp2f(s[0] - base), p1 = exp2f(s[1] - base), fix = exp2f(m - base);
      const bool grown = __any_sync(0xffffffffu, top != m);
      l = l * fix + (p0 + p1);
      m = top;
      __syncwarp();
      if (g8 < R) {
        *reinterpret_cast<float2*>(sp + g8 * KEYS + 2 * t8) = make_float2(p0, p1);
        if (t8 == 0) sp[64 + g8] = fix;
      }
      __syncwarp();
      if (grown) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float f = sp[64 + r];
#pragma unroll
          for (int e = 0; e < E; ++e) acc[r][e] *= f;
        }
      }
#pragma unroll
      for (int n0 = 0; n0 < KEYS; n0 += 4) {
        float4 f[R];
#pragma unroll
        for (int r = 0; r < R; ++r) f[r] = *reinterpret_cast<const float4*>(sp + r * KEYS + n0);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          float y[E];
          y2[n0 + n].get(y);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const float w = n == 0 ? f[r].x : (n == 1 ? f[r].y : (n == 2 ? f[r].z : f[r].w));
#pragma unroll
            for (int e = 0; e < E; ++e) acc[r][e] = fmaf(w, y[e], acc[r][e]);
          }
        }
      }
      if (more) load2(t0 + WARPS * KEYS);
    }
  } else {
  constexpr int WORDS = Token<T, E>::WORDS;
  // both sides' tokens are on their way before the first product where registers allow; forward, the next step's as soon as
  // this one's are used up
  constexpr bool BOTH = KEYS * WORDS <= 32, AHEAD = MODE == FWD && BOTH;
  Token<T, E> y1[KEYS], y2[BOTH ? KEYS : 1];
  // dk and dv: the tokens of one head of the group after the other
  for (int head = MODE == DKV ? kvh * group : 0, heads = MODE == DKV ? group : 1; heads > 0; ++head, --heads) {
    auto token1 = [&](int t) {  // K, or Q for dk and dv
      t = min(t, end - 1);
      return MODE == DKV ? q + t * a.q_stride[1] + head * a.q_stride[2] : k + t * a.k_stride[1];
    };
    auto token2 = [&](int t) {  // V, or dout for dk and dv
      t = min(t, end - 1);
      return MODE == DKV ? dout + t * io.dout_stride[1] + head * io.dout_stride[2] : v + t * a.v_stride[1];
    };
    auto load1 = [&](int t) {
#pragma unroll
      for (int n = 0; n < KEYS; ++n) y1[n].load(token1(t + n), c, dim, io.vec);
    };
    auto load2 = [&](int t) {
      if constexpr (BOTH)
#pragma unroll
        for (int n = 0; n < KEYS; ++n) y2[n].load(token2(t + n), c, dim, io.vec);
    };
    int t0 = first + warp * KEYS;
    if (AHEAD && t0 < end) load1(t0), load2(t0);
    for (; t0 < end; t0 += WARPS * KEYS) {
      const bool more = t0 + WARPS * KEYS < end;
      if constexpr (!AHEAD) load1(t0), load2(t0);
      float z[32];
#pragma unroll
      for (int n = 0; n < KEYS; ++n) {
        float y[E];
        y1[n].get(y);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          float s = 0.f;
#pragma unroll
          for (int e = 0; e < E; ++e) s = fmaf(x1[r][e], y[e], s);
          z[r * KEYS + n] = s;
        }
      }
      auto second = [&](float (&y)[E], int n) {
        if constexpr (BOTH) {
          y2[n].get(y);
        } else {
          Token<T, E> u;
          u.load(token2(t0 + n), c, dim, io.vec);
          u.get(y);
        }
      };
      if (AHEAD && more) load1(t0 + WARPS * KEYS);
      const float dot = sum_to_lane(z, lane);
      // the lane's score
      const int t = t0 + lk;
      const int i = MODE == DKV ? t : my_row, j = MODE == DKV ? my_row : t;
      const int other = MODE == DKV ? i : j;
      const bool seen = t < end && other >= lo && other < hi;
      const int rel = j - i - seq.shift;
      float s = dot * sl;
      if (a.table && seen) {
        const int h = MODE == DKV ? head : my_head;
        s += table_log2(a.table, (int64_t)s_bucket[max(-far, min(far, rel)) + far] * a.heads + h, a.table_dtype);
      }
      if (!seen) s = -INFINITY;
      if constexpr (MODE == FWD) {
        float top = s;
#pragma unroll
        for (int o = KEYS / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        top = fmaxf(m, top);
        const float base = top == -INFINITY ? 0.f : top;
        const float p = exp2f(s - base), fix = exp2f(m - base);
        const bool grown = __any_sync(0xffffffffu, top != m);
        l = l * fix + p;
        m = top;
        __syncwarp();
        sp[lane] = p;
        if (lk == 0) sp[32 + lr] = fix;
        __syncwarp();
        if (grown) {
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const float f = sp[32 + r];
#pragma unroll
            for (int e = 0; e < E; ++e) acc[r][e] *= f;
          }
        }
#pragma unroll
        for (int n = 0; n < KEYS; ++n) {
          float y[E];
          second(y, n);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const float f = sp[r * KEYS + n];
#pragma unroll
            for (int e = 0; e < E; ++e) acc[r][e] = fmaf(f, y[e], acc[r][e]);
          }
        }
        if (AHEAD && more) load2(t0 + WARPS * KEYS);
      } else {
#pragma unroll
        for (int n = 0; n < KEYS; ++n) {
          float y[E];
          second(y, n);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            float d = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) d = fmaf(x2[r][e], y[e], d);
            z[r * KEYS + n] = d;
          }
        }
        const float dp = sum_to_lane(z, lane);
        float lse = my_lse, delta = my_delta;
        if constexpr (MODE == DKV) {
          lse = INFINITY, delta = 0.f;
          if (seen) {
            lse = exponent_of(io.lse[(b * a.heads + head) * a.queries + i]);
            delta = -io.delta[(b * a.heads + head) * io.padded + i];
          }
        }
        const float p = seen ? exp2f(s - lse) : 0.f;
        const float dz = seen ? p * (dp - delta) : 0.f;
        __syncwarp();
        sp[lane] = p;
        sp[32 + lane] = dz;
        __syncwarp();
        if constexpr (MODE == DQ) {
          if (a.table) {
            if (rel >= far) after += dz;
            else if (rel <= -far) before += dz;
            // the step's near diagonals rel = t0 + d - (R - 1) - first query - shift, one a lane: no lane adds to another's
            const int d = lane - (R - 1);
            const int at = t0 + d - rb * R - seq.shift;
            if (lane < R + KEYS - 1 && at > -far && at < far) {
              float sum = 0.f;
#pragma unroll
              for (int r = 0; r < R; ++r)
                if (d + r >= 0 && d + r < KEYS) sum += sp[32 + r * KEYS + d + r];
              s_near[warp * bins + at + far] += sum;
            }
          }
        }
#pragma unroll
        for (int n = 0; n < KEYS; ++n) {
          float y[E];
          y1[n].get(y);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const float f = sp[32 + r * KEYS + n];
#pragma unroll
            for (int e = 0; e < E; ++e) acc[r][e] = fmaf(f, y[e], acc[r][e]);
          }
          if constexpr (MODE == DKV) {
            second(y, n);
#pragma unroll
            for (int r = 0; r < R; ++r) {
              const float f = sp[r * KEYS + n];
#pragma unroll
              for (int e = 0; e < E; ++e) acc2[r][e] = fmaf(f, y[e], acc2[r][e]);
            }
          }
        }
      }
    }
  }
  }

  // the warps' results joined, in order
  float *jm = s_join + JOIN - 2 * WARPS * R, *jl = jm + WARPS * R;
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int e = 0; e < E; ++e) {
      s_join[(warp * R + r) * 32 * E + c + e] = acc[r][e];
      if constexpr (MODE == DKV) s_join[((WARPS + warp) * R + r) * 32 * E + c + e] = acc2[r][e];
    }
  if constexpr (MODE == FWD) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if (lk == 0 && lr < R) jm[warp * R + lr] = m, jl[warp * R + lr] = l;
  }
  if constexpr (MODE == DQ) {
    if (a.table) {
      before = warp_sum(before), after = warp_sum(after);
      if (lane == 0) s_near[warp * bins] = before, s_near[warp * bins + 2 * far] = after;
    }
  }
  __syncthreads();
  const int64_t row_block = ((int64_t)b * gridDim.y + hy) * io.out_rows + rb;
  for (int at = threadIdx.x; at < R * dim; at += THREADS) {
    const int r = at / dim, col = at % dim;
    if constexpr (MODE == FWD) {
      const int i = row_query(r), h = row_head(r);
      if (i >= a.queries) continue;
      float top = -INFINITY, sum = 0.f, o = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) top = fmaxf(top, jm[w * R + r]);
      const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float f = exp2f(jm[w * R + r] - base);
        sum = fmaf(f, jl[w * R + r], sum);
        o = fmaf(f, s_join[(w * R + r) * 32 * E + col], o);
      }
      if (io.splits > 1) {
        float* p = io.part + ((row_block * io.splits + part) * R + r) * (dim + 2);
        p[col] = o;
        if (col == 0) p[dim] = top, p[dim + 1] = sum;
      } else {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        reinterpret_cast<T*>(io.out)[((b * a.queries + i) * a.heads + h) * dim + col] = (T)(o * inv);
        if (col == 0) io.lse[(b * a.heads + h) * a.queries + i] = sum == 0.f ? -INFINITY : (base + log2f(sum)) * LN2;
      }
    } else {
      float o = 0.f, o2 = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        o += s_join[(w * R + r) * 32 * E + col];
        if constexpr (MODE == DKV) o2 += s_join[((WARPS + w) * R + r) * 32 * E + col];
      }
      const int row = rb * R + r;
      if (MODE == DQ) {
        if (row < a.queries) reinterpret_cast<T*>(io.out)[((b * a.queries + row) * a.heads + hy) * dim + col] = (T)(o * a.scale);
      } else if (row < a.keys) {
        const int64_t to = ((b * a.keys + row) * a.kv_heads + hy) * dim + col;
        reinterpret_cast<T*>(io.out)[to] = (T)(o * a.scale);
        reinterpret_cast<T*>(io.out2)[to] = (T)o2;
      }
    }
  }
  if constexpr (MODE == DQ) {
    if (a.table) {
      for (int i = threadIdx.x; i < bins; i += THREADS) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) s += s_near[w * bins + i];
        s_near[i] = s;  // this thread's column alone
      }
      __syncthreads();
      const int nb = relative::buckets_of(a.relative);
      for (int n = threadIdx.x; n < nb; n += THREADS) io.part[row_block * nb + n] = relative::bucket_sum(a.relative, far, s_near, n);
    }
  }
}

// joins the splits of a row, a block each: their factors once, then a thread a column
constexpr int MOST_SPLITS = 256;
template <typename T>
__global__ void __launch_bounds__(128)
    join_kernel(const __grid_constant__ b200_attention a, const float* part, int splits, int64_t row_blocks, int R, T* out, float* lse) {
  __shared__ float factor[MOST_SPLITS], red[32];
  const int64_t at = blockIdx.x;  // [batch][key head][query][head of the group]
  const int dim = (int)a.dim;
  const int64_t group = a.heads / a.kv_heads, per = a.queries * group;
  const int64_t bk = at / per, rr = at % per, b = bk / a.kv_heads, i = rr / group, h = bk % a.kv_heads * group + rr % group;
  const float* p = part + ((bk * row_blocks + rr / R) * splits * R + rr % R) * (dim + 2);
  const int64_t step = (int64_t)R * (dim + 2);
  float m[MOST_SPLITS / 128], l[MOST_SPLITS / 128], top = -INFINITY, sum = 0.f;
#pragma unroll
  for (int k = 0; k < MOST_SPLITS / 128; ++k) {
    const int s = threadIdx.x + 128 * k;
    m[k] = s < splits ? p[s * step + dim] : -INFINITY;
    l[k] = s < splits ? p[s * step + dim + 1] : 0.f;
    top = fmaxf(top, m[k]);
  }
  top = block_max(top, red);
  const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
  for (int k = 0; k < MOST_SPLITS / 128; ++k) {
    const float f = exp2f(m[k] - base);
    factor[threadIdx.x + 128 * k] = f;
    sum = fmaf(f, l[k], sum);
  }
  sum = block_sum(sum, red);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  for (int c = threadIdx.x; c < dim; c += 128) {
    float o[4] = {0.f, 0.f, 0.f, 0.f};
    int s = 0;
    for (; s + 8 <= splits; s += 8)
#pragma unroll
      for (int k = 0; k < 8; ++k) o[k & 3] = fmaf(factor[s + k], p[(s + k) * step + c], o[k & 3]);
    for (; s < splits; ++s) o[0] = fmaf(factor[s], p[s * step + c], o[0]);
    out[((b * a.queries + i) * a.heads + h) * dim + c] = (T)(((o[0] + o[1]) + (o[2] + o[3])) * inv);
  }
  if (threadIdx.x == 0) lse[(b * a.heads + h) * a.queries + i] = sum == 0.f ? -INFINITY : (base + log2f(sum)) * LN2;
}

// dtable[bucket, h]: the blocks' sums, batch by batch; 32 lanes a value
template <typename T>
__global__ void __launch_bounds__(256) table_kernel(const float* part, T* dtable, int64_t batch, int heads, int64_t blocks, int nb) {
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (at >= (int64_t)heads * nb) return;
  const int n = (int)(at / heads), h = (int)(at % heads);
  float s = 0.f;
  for (int64_t i = lane; i < batch * blocks; i += 32) s += part[(((i / blocks) * heads + h) * blocks + i % blocks) * nb + n];
  s = warp_sum(s);
  if (lane == 0) dtable[at] = (T)s;
}

static bool vectors(const b200_attention& a, int elements, const void* dout, const int64_t* ds) {
  const int64_t size = a.dtype == B200_F32 ? 4 : 2;
  uint64_t u = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) | reinterpret_cast<uintptr_t>(dout);
  for (int i = 0; i < 3; ++i) u |= (uint64_t)((a.q_stride[i] | a.k_stride[i] | a.v_stride[i] | (ds ? ds[i] : 0)) * size);
  return (u & 15) == 0 && a.dim % elements == 0;
}

static int elements(const b200_attention& a) { return a.dim <= 64 ? 2 : (a.dim <= 128 ? 4 : 8); }

// rows of a block: as few as there are, so that a step has more tokens
static int rows_of(const b200_attention& a, int64_t rows) {
  const int most = a.dim <= 128 ? 8 : 4;
  for (int r = 1; r < most; r *= 2)
    if (rows <= r) return r;
  return most;
}

struct Shape {
  int R, splits;
  int64_t blocks;  // row blocks of a (batch, key head)
};
static Shape forward_shape(const b200_attention& a) {
  Shape s;
  const int64_t rows = a.queries * (a.heads / a.kv_heads);
  s.R = rows_of(a, rows);
  s.blocks = ceil_div(rows, s.R);
  // splits that bring 12 blocks to every SM (four waves, so that caches of several lengths even out), of 64 keys at least;
  // none where the rows alone fill the SMs twice
  const int64_t have = s.blocks * a.batch * a.kv_heads, sms = num_sms();
  s.splits = have >= 6 * sms ? 1 : (int)std::max<int64_t>(1, std::min({12 * sms / have, ceil_div(a.keys, 64), (int64_t)MOST_SPLITS}));
  return s;
}

template <int MODE>
static size_t shared_bytes(const b200_attention& a, int R, int E) {
  size_t n = WARPS * AREA + (size_t)WARPS * R * 32 * E * (MODE == DKV ? 2 : 1) + 2 * WARPS * R;
  const size_t bins = a.table ? 2 * relative::far_of(a.relative) + 1 : 0;
  if (MODE == DQ) n += WARPS * bins;
  return n * sizeof(float) + bins;
}

template <typename T, int E, int R, int MODE, bool MMA = false>
static int launch(const b200_attention& a, const Io& io, dim3 grid, cudaStream_t st) {
  const size_t shared = shared_bytes<MODE>(a, R, E);
  const auto kernel = rows_kernel<T, E, R, MODE, MMA>;
  if (shared > 48 * 1024) {
    // the largest that any call needs, so that calls of several threads do not lower it
    const size_t most = sizeof(float) * (WARPS * AREA + WARPS * R * 32 * E * 2 + 2 * WARPS * R + WARPS * (2 * B200_RELATIVE_MAX_FAR + 1)) + 2 * B200_RELATIVE_MAX_FAR + 1;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most) != cudaSuccess) return check_launch("attention");
  }
  kernel<<<grid, THREADS, shared, st>>>(a, io);
  return check_launch("attention");
}

template <typename T, int E, int MODE>
static int launch_r(const b200_attention& a, const Io& io, int R, dim3 grid, cudaStream_t st) {
  if constexpr (MODE == FWD && sizeof(T) == 2) {
    // whole 16-byte pieces of a head
    if (io.vec && a.dim % 8 == 0) {
      if (R == 1) return launch<T, E, 1, MODE, true>(a, io, grid, st);
      if (R == 2) return launch<T, E, 2, MODE, true>(a, io, grid, st);
      if (R == 4) return launch<T, E, 4, MODE, true>(a, io, grid, st);
      if constexpr (E < 8) return launch<T, E, 8, MODE, true>(a, io, grid, st);
    }
  }
  if constexpr (E < 8)
    if (R == 8) return launch<T, E, 8, MODE>(a, io, grid, st);
  if constexpr (MODE == FWD) {
    if (R == 1) return launch<T, E, 1, MODE>(a, io, grid, st);
    if (R == 2) return launch<T, E, 2, MODE>(a, io, grid, st);
    return launch<T, E, 4, MODE>(a, io, grid, st);
  } else if constexpr (E == 8) {
    return launch<T, E, 4, MODE>(a, io, grid, st);
  }
  return B200_ERR_UNSUPPORTED;
}
template <int MODE>
static int launch_any(const b200_attention& a, const Io& io, int R, dim3 grid, cudaStream_t st) {
  const int e = elements(a);
  if (a.dtype == B200_F32)
    return e == 2 ? launch_r<float, 2, MODE>(a, io, R, grid, st) : (e == 4 ? launch_r<float, 4, MODE>(a, io, R, grid, st) : launch_r<float, 8, MODE>(a, io, R, grid, st));
  using B = __nv_bfloat16;
  return e == 2 ? launch_r<B, 2, MODE>(a, io, R, grid, st) : (e == 4 ? launch_r<B, 4, MODE>(a, io, R, grid, st) : launch_r<B, 8, MODE>(a, io, R, grid, st));
}

}  // namespace rows

size_t rows_forward_workspace(const b200_attention& a) {
  const rows::Shape s = rows::forward_shape(a);
  return s.splits == 1 ? 0 : (size_t)(a.batch * a.kv_heads * s.blocks * s.splits * s.R * (a.dim + 2)) * sizeof(float);
}

int rows_forward(const b200_attention& a, void* out, float* lse, void* workspace, cudaStream_t st) {
  using namespace rows;
  const Shape s = forward_shape(a);
  Io io = {};
  io.out_rows = s.blocks, io.splits = s.splits, io.vec = vectors(a, elements(a), nullptr, nullptr), io.out = out, io.lse = lse;
  io.part = reinterpret_cast<float*>(workspace);
  B200_REQUIRE(s.blocks * s.splits < (1ll << 31), "attention: too many queries");
  if (int rc = launch_any<FWD>(a, io, s.R, dim3((unsigned)(s.blocks * s.splits), (unsigned)a.kv_heads, (unsigned)a.batch), st)) return rc;
  if (s.splits == 1) return B200_OK;
  const unsigned grid = (unsigned)(a.batch * a.heads * a.queries);
  if (a.dtype == B200_F32) join_kernel<float><<<grid, 128, 0, st>>>(a, io.part, s.splits, s.blocks, s.R, (float*)out, lse);
  else join_kernel<__nv_bfloat16><<<grid, 128, 0, st>>>(a, io.part, s.splits, s.blocks, s.R, (__nv_bfloat16*)out, lse);
  return check_launch("attention");
}

int table_sum(const b200_attention& a, const float* part, int64_t blocks, void* dtable, cudaStream_t st) {
  const int nb = relative::buckets_of(a.relative);
  const unsigned grid = (unsigned)ceil_div(a.heads * nb, 8);
  if (a.table_dtype == B200_F32) rows::table_kernel<float><<<grid, 256, 0, st>>>(part, (float*)dtable, a.batch, (int)a.heads, blocks, nb);
  else rows::table_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(part, (__nv_bfloat16*)dtable, a.batch, (int)a.heads, blocks, nb);
  return check_launch("attention_grad");
}

size_t rows_grad_workspace(const b200_attention& a) {
  if (!a.table) return 0;
  const int R = a.dim <= 128 ? 8 : 4;
  return (size_t)(a.batch * a.heads * ceil_div(a.queries, R) * relative::buckets_of(a.relative)) * sizeof(float);
}

int rows_grad(const b200_attention& a, const b200_attention_grads& g, const float* delta, int64_t padded, void* workspace, cudaStream_t st) {
  using namespace rows;
  const int R = a.dim <= 128 ? 8 : 4;
  Io io = {};
  io.splits = 1, io.vec = vectors(a, elements(a), g.dout, g.dout_stride), io.dout = g.dout, io.delta = delta, io.padded = padded;
  for (int i = 0; i < 3; ++i) io.dout_stride[i] = g.dout_stride[i];
  io.lse = const_cast<float*>(g.lse);
  io.out_rows = ceil_div(a.queries, R), io.out = g.dq, io.part = reinterpret_cast<float*>(workspace);
  if (int rc = launch_any<DQ>(a, io, R, dim3((unsigned)io.out_rows, (unsigned)a.heads, (unsigned)a.batch), st)) return rc;
  if (a.table)
    if (int rc = table_sum(a, io.part, io.out_rows, g.dtable, st)) return rc;
  io.out_rows = ceil_div(a.keys, R), io.out = g.dk, io.out2 = g.dv, io.part = nullptr;
  return launch_any<DKV>(a, io, R, dim3((unsigned)io.out_rows, (unsigned)a.kv_heads, (unsigned)a.batch), st);
}

}  // namespace attention
}  // namespace b200
