// Attention on the tensor cores: bf16 heads of up to 128 elements, many queries.
//
// Forward. A block takes two tiles of 128 queries of one head past the keys, 128 at a time:
//   warp 0       TMA: both query tiles once, then K and V tiles into a ring;
//   warp 1       owns TMEM, issues S_w = Q_w K^T (operands in shared memory) and O_w += P_w V (P from TMEM);
//   warps 4-7, 8-11   softmax of tile 0, tile 1: a thread owns a query's row of S.
// TMEM: S_0, S_1 (128 columns each; P, bf16, over its own S), O_0, O_1. While one tile's threads make their
// exponentials, the tensor cores work for the other. S_w of the next keys is issued right behind O_w's product: MMAs
// run in their order, so it overwrites P only when that is used up, and its completion says that O_w is at rest.
// The running maximum moves only when a row's has grown by 2^8 (probabilities stay below 2^8, sums are
// fp32), so O is hardly ever rescaled.
//
// Backward, one kernel in two forms. 128 rows stay, tiles of the other side go past:
//   dq:      rows are queries (Q, dO), tiles are keys (K, V):     S = Q K^T, dP = dO V^T, dQ += dS K
//   dk, dv:  rows are keys (K, V), tiles are queries (Q, dO):     S = K Q^T, dP = V dO^T, dV += P dO, dK += dS Q
// so p and dz of a tile are made by the threads that own its rows, go back to TMEM as bf16 and are the A operand of the
// sums from there: nothing is transposed, no sum leaves its block, every order is fixed. S and dP are made
// twice for that (7 products instead of 5). Threads read S and dP early, so the MMAs of the next tile run
// under their exponentials.
//
// Probabilities and dz are rounded to bf16 for the products that they are operands of; scores, maxima, sums and
// all accumulators are fp32. Every wait is bounded (tc_common.cuh); on expiry the error flag is set and the
// block winds down.
#include <algorithm>

#include "attention.cuh"
#include "tc_common.cuh"

namespace b200 {
namespace attention {
namespace tiles {

using namespace tc;

constexpr int THREADS = 384, ROWS = 128;
constexpr uint32_t SMEM_LIMIT = 232448;

// Bounded wait of whoever calls it. A look at the timer takes longer than a tile's MMAs, so it comes every 256 polls. After
// WAIT_LIMIT_NS the block gives up: every later wait ends at once, results are not valid, the error flag says so.
__device__ __forceinline__ void wait(uint64_t* bar, uint32_t parity, int* gave_up) {
  unsigned long long t0 = 0;
  while (true) {
#pragma unroll 1
    for (int k = 0; k < 256; ++k)
      if (mbar_try_wait(bar, parity)) return;
    if (*reinterpret_cast<volatile int*>(gave_up)) return;
    const unsigned long long now = globaltimer();
    if (t0 == 0) t0 = now;
    else if (now - t0 > WAIT_LIMIT_NS) {
      raise_device_error(B200_ERR_TIMEOUT);
      *reinterpret_cast<volatile int*>(gave_up) = 1;
    }
  }
}
// by all lanes, together again behind it
__device__ __forceinline__ void warp_wait(uint64_t* bar, uint32_t parity, int* gave_up) {
  wait(bar, parity, gave_up);
  __syncwarp();
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The warp that issues MMAs walks its code with all lanes, and only the instruction itself is the elected lane's: under a
// branch of one lane every operand is fetched into the uniform registers anew, 95 clocks an MMA of 64. A descriptor is
// two words, of which tiles and K steps change the low one.
struct Desc {
  uint32_t lo, hi;
};
__device__ __forceinline__ Desc desc_at(uint32_t addr, uint32_t lbo_bytes) {
  const uint64_t d = smem_desc(addr, lbo_bytes, 1024);
  return {(uint32_t)d, (uint32_t)(d >> 32)};
}
__device__ __forceinline__ int elect_one() {
  int e;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.s32 %0, 1, 0, p;\n}\n" : "=r"(e));
  return e;
}
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }
__device__ __forceinline__ void mma(int elected, uint32_t d, Desc a, uint32_t a_off, Desc b, uint32_t b_off, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p, e;\n .reg .b64 x, y;\n mov.b64 x, {%1, %2};\n mov.b64 y, {%3, %4};\n setp.ne.b32 p, %6, 0;\n setp.ne.b32 e, %7, 0;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %5, p;\n}\n" ::"r"(d),
      "r"(a.lo + a_off), "r"(a.hi), "r"(b.lo + b_off), "r"(b.hi), "r"(idesc), "r"(acc), "r"(elected));
}
// D += A B with A (16-bit, two K a column) in TMEM
__device__ __forceinline__ void mma_from_tmem(int elected, uint32_t d, uint32_t a, Desc b, uint32_t b_off, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p, e;\n .reg .b64 y;\n mov.b64 y, {%2, %3};\n setp.ne.b32 p, %5, 0;\n setp.ne.b32 e, %6, 0;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %4, p;\n}\n" ::"r"(d),
      "r"(a), "r"(b.lo + b_off), "r"(b.hi), "r"(idesc), "r"(acc), "r"(elected));
}
__device__ __forceinline__ void commit(int elected, uint64_t* bar) {
  asm volatile(
      "{\n .reg .pred e;\n setp.ne.b32 e, %1, 0;\n @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(smem_u32(bar)),
      "r"(elected)
      : "memory");
}
#define B200_R16(r, o)                                                                                                              \
  "r"(r[o]), "r"(r[o + 1]), "r"(r[o + 2]), "r"(r[o + 3]), "r"(r[o + 4]), "r"(r[o + 5]), "r"(r[o + 6]), "r"(r[o + 7]), "r"(r[o + 8]), \
      "r"(r[o + 9]), "r"(r[o + 10]), "r"(r[o + 11]), "r"(r[o + 12]), "r"(r[o + 13]), "r"(r[o + 14]), "r"(r[o + 15])
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr), B200_R16(r, 0));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,"
      "%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
      B200_R16(r, 0), B200_R16(r, 16));
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ uint32_t idesc_of(int m, int n, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// A tile of R rows is DP / 64 pieces of [R][64] elements, 128-byte rows, swizzled. K-major, elements 16 k .. 16 k + 15 of every row
// are at off_k<R>(k) of its descriptor (in 16 bytes); with the elements as N, rows 16 k .. 16 k + 15 at off_mn(k).
template <int R>
__device__ __forceinline__ constexpr uint32_t off_k(int k) {
  return (uint32_t)(k >> 2) * (R * 8u) + (uint32_t)(k & 3) * 2u;
}
__device__ __forceinline__ constexpr uint32_t off_mn(int k) { return (uint32_t)k * 128u; }
// rows [from, R) of a tile set to zero by one warp
template <int R, int DP>
__device__ __forceinline__ void zero_rows(uint32_t base, int from, int lane) {
  for (int p = 0; p < DP / 64; ++p)
    for (uint32_t o = (uint32_t)from * 128u + lane * 16u; o < R * 128u; o += 512u) st_shared_v4(base + p * (R * 128u) + o, 0, 0, 0, 0);
}

// the bias of a head by relative position, log2 domain: shared memory, [2 far + 1]
__device__ __forceinline__ void fill_bias(float* lut, const b200_attention& a, int far, int head) {
  for (int i = threadIdx.x; i <= 2 * far; i += blockDim.x)
    lut[i] = table_log2(a.table, (int64_t)relative::bucket_of(a.relative, i - far) * a.heads + head, a.table_dtype);
}

// 32 fp32 columns of a row, scaled, to a row of the result from column `col` on
__device__ __forceinline__ void store32(__nv_bfloat16* row, int col, int dim, bool vec, const uint32_t (&v)[32], float f) {
  if (vec) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (col + 8 * k < dim) {
        uint4 u;
        u.x = pack_bf16(__uint_as_float(v[8 * k]) * f, __uint_as_float(v[8 * k + 1]) * f);
        u.y = pack_bf16(__uint_as_float(v[8 * k + 2]) * f, __uint_as_float(v[8 * k + 3]) * f);
        u.z = pack_bf16(__uint_as_float(v[8 * k + 4]) * f, __uint_as_float(v[8 * k + 5]) * f);
        u.w = pack_bf16(__uint_as_float(v[8 * k + 6]) * f, __uint_as_float(v[8 * k + 7]) * f);
        *reinterpret_cast<uint4*>(row + col + 8 * k) = u;
      }
  } else {
#pragma unroll
    for (int k = 0; k < 32; ++k)
      if (col + k < dim) row[col + k] = __float2bfloat16_rn(__uint_as_float(v[k]) * f);
  }
}

// ------------------------------------------------------------------------------------
// forward
// ------------------------------------------------------------------------------------

constexpr int KEYS = 128;
constexpr float LAZY = 8.f;  // log2 by which a maximum may grow before O is rescaled

template <int DP>
struct Fwd {
  static constexpr int STAGES = DP == 64 ? 4 : 2;
  static constexpr uint32_t TILE = 128 * DP * 2;
  static constexpr uint32_t BARS = 2 * TILE + STAGES * 2 * TILE;
  static constexpr uint32_t LUT = BARS + 256;
  static constexpr uint32_t TMEM_O = 256;
};

template <int DP, bool BIAS>
__global__ void __launch_bounds__(THREADS, 1)
    forward_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                   const __grid_constant__ b200_attention a, __nv_bfloat16* out, float* lse, int vec) {
  using F = Fwd<DP>;
  constexpr int ST = F::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t s_q = smem_u32(smem), s_k = s_q + 2 * F::TILE, s_v = s_k + ST * F::TILE;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + F::BARS);
  uint64_t *q_full = bars, *k_full = bars + 1, *k_empty = k_full + ST, *v_full = k_empty + ST, *v_empty = v_full + ST, *s_full = v_empty + ST,
           *p_full = s_full + 2, *o_full = p_full + 2, *idle = o_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(idle + 1);
  int* gave_up = reinterpret_cast<int*>(tmem_slot + 1);
  float* lut = reinterpret_cast<float*>(smem + F::LUT);

  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int head = blockIdx.y, kvh = head / (int)(a.heads / a.kv_heads), dim = (int)a.dim;
  const int64_t b = blockIdx.z;
  const Sequence seq(a, b);
  // causal blocks with the most keys start first
  const int pair = a.causal ? (int)(gridDim.x - 1 - blockIdx.x) : (int)blockIdx.x;
  int t0[2], t1[2];  // key tiles of each query tile
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const int i0 = (2 * pair + w) * ROWS, i1 = min(i0 + ROWS, seq.queries) - 1;
    t0[w] = t1[w] = 0;
    if (i1 >= i0) {
      const int lo = seq.first_key(a, i0), hi = seq.end_key(a, i1);
      if (hi > lo) t0[w] = lo / KEYS, t1[w] = (hi + KEYS - 1) / KEYS;
    }
    t0[w] = uniform(t0[w]), t1[w] = uniform(t1[w]);
  }
  const bool any0 = t1[0] > t0[0], any1 = t1[1] > t0[1];
  const int T0 = any0 ? (any1 ? min(t0[0], t0[1]) : t0[0]) : t0[1], T1 = max(t1[0], t1[1]);
  const int far = BIAS ? relative::far_of(a.relative) : 0;

  if (threadIdx.x == 0) {
    *gave_up = 0;
    for (const CUtensorMap* m : {&map_q, &map_k, &map_v}) asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(m)) : "memory");
    mbar_init(q_full, 1);
    for (int s = 0; s < ST; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(&s_full[w], 1);
      mbar_init(&p_full[w], 4);
      mbar_init(&o_full[w], 1);
    }
    mbar_init(idle, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if constexpr (BIAS) fill_bias(lut, a, far, head);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = (uint32_t)uniform((int)*tmem_slot);

  if (warp == 0) {
    if (lane == 0 && T1 > T0) {
      mbar_expect_tx(q_full, ((any0 ? 1 : 0) + (any1 ? 1 : 0)) * F::TILE);
      for (int w = 0; w < 2; ++w)
        if (t1[w] > t0[w])
          for (int p = 0; p < DP / 64; ++p)
            tma_load_4d(smem + w * F::TILE + p * (ROWS * 128), &map_q, q_full, p * 64, (2 * pair + w) * ROWS, head, (int)b);
      int n = 0;
      for (int t = T0; t < T1; ++t, ++n) {
        const int s = n % ST;
        const uint32_t par = ((n / ST) & 1) ^ 1;
        wait(&k_empty[s], par, gave_up);
        mbar_expect_tx(&k_full[s], F::TILE);
        for (int p = 0; p < DP / 64; ++p)
          tma_load_4d(smem + 2 * F::TILE + s * F::TILE + p * (KEYS * 128), &map_k, &k_full[s], p * 64, t * KEYS, kvh, (int)b);
        wait(&v_empty[s], par, gave_up);
        mbar_expect_tx(&v_full[s], F::TILE);
        for (int p = 0; p < DP / 64; ++p)
          tma_load_4d(smem + (2 + ST) * F::TILE + s * F::TILE + p * (KEYS * 128), &map_v, &v_full[s], p * 64, t * KEYS, kvh, (int)b);
      }
      // every load has landed before the block may end
      wait(q_full, 0, gave_up);
      for (int m = max(0, n - ST); m < n; ++m) {
        wait(&k_full[m % ST], (m / ST) & 1, gave_up);
        wait(&v_full[m % ST], (m / ST) & 1, gave_up);
      }
    }
  } else if (warp == 1) {
    const int ks = (dim + 15) / 16, elected = elect_one();
    const uint32_t id_s = idesc_of(ROWS, KEYS, false), id_o = idesc_of(ROWS, ks * 16, true);
    if (T1 > T0) warp_wait(q_full, 0, gave_up);
    const Desc dq = desc_at(s_q, 16), dk = desc_at(s_k, 16), dv = desc_at(s_v, KEYS * 128);
    auto product_s = [&](int w, int s) {  // S_w of the tile in stage s, whose K has landed
      tc_fence_after();
      const Desc kd = {dk.lo + s * (F::TILE >> 4), dk.hi}, qd = {dq.lo + w * (F::TILE >> 4), dq.hi};
#pragma unroll
      for (int k = 0; k < DP / 16; ++k)
        if (k < ks) mma(elected, tmem + w * KEYS, qd, off_k<ROWS>(k), kd, off_k<KEYS>(k), id_s, k > 0);
      commit(elected, &s_full[w]);
    };
    int done[2] = {0, 0};
    if (T1 > T0) {
      warp_wait(&k_full[0], 0, gave_up);
      for (int w = 0; w < 2; ++w)
        if (t0[w] == T0 && t1[w] > t0[w]) product_s(w, 0);
      commit(elected, &k_empty[0]);
    }
    for (int t = T0, s = 0, par = 0, next = 0, next_par = 0; t < T1; ++t, s = next, par = next_par) {
      next = s + 1 == ST ? 0 : s + 1, next_par = s + 1 == ST ? par ^ 1 : par;
      warp_wait(&v_full[s], par, gave_up);
      const int have = seq.keys - t * KEYS;
      if (have < KEYS && seq.keys < a.keys) {
        // what lies behind the sequence's end may be anything, and is multiplied by zeros
        zero_rows<KEYS, DP>(s_v + s * F::TILE, max(have, 0), lane);
        fence_proxy_async_smem();
        __syncwarp();
      }
      const Desc vd = {dv.lo + s * (F::TILE >> 4), dv.hi};
      if (t + 1 < T1) warp_wait(&k_full[next], next_par, gave_up);
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        if (t >= t0[w] && t < t1[w]) {
          warp_wait(&p_full[w], done[w] & 1, gave_up);
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < KEYS / 16; ++k)
            mma_from_tmem(elected, tmem + F::TMEM_O + w * DP, tmem + w * KEYS + k * 8, vd, off_mn(k), id_o, done[w] > 0 || k > 0);
          if (t + 1 == t1[w]) commit(elected, &o_full[w]);
          ++done[w];
        }
        if (t + 1 >= t0[w] && t + 1 < t1[w]) product_s(w, next);
      }
      commit(elected, &v_empty[s]);
      if (t + 1 < T1) commit(elected, &k_empty[next]);
    }
    // no MMA and no commit is on its way when the block ends
    commit(elected, idle);
    warp_wait(idle, 0, gave_up);
  } else if (warp >= 4) {
    const int w = (warp - 4) >> 2, q = warp & 3;
    const int i0 = (2 * pair + w) * ROWS + q * 32, i = i0 + lane;
    const bool valid = i < seq.queries;
    const int lo = valid ? seq.first_key(a, i) : 0, hi = valid ? seq.end_key(a, i) : 0;
    // every key of [full0, full1) is seen by all rows of the warp
    const int last = min(i0 + 31, seq.queries - 1);
    const int full0 = seq.first_key(a, last), full1 = seq.end_key(a, i0);
    const uint32_t lanes = (uint32_t)(q * 32) << 16;
    const uint32_t t_s = tmem + lanes + w * KEYS, t_o = tmem + lanes + F::TMEM_O + w * DP;
    const float sl = a.scale * LOG2E;
    float m = -INFINITY, l = 0.f;
    for (int t = t0[w]; t < t1[w]; ++t) {
      const int n = t - t0[w], j0 = t * KEYS;
      warp_wait(&s_full[w], n & 1, gave_up);
      tc_fence_after();
      uint32_t v[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32_issue(t_s + c * 32, v[c]);
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_wait(v[c]);
      float mul = sl;
      if constexpr (BIAS) {
        mul = 1.f;
        const int r0 = j0 - i - seq.shift;  // of column 0
        const int w0 = j0 - i0 - seq.shift;  // of lane 0
        if (w0 - 31 >= far || w0 + KEYS - 1 <= -far) {
          const float c0 = lut[w0 >= far ? 2 * far : 0];
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int k = 0; k < 32; ++k) v[c][k] = __float_as_uint(fmaf(__uint_as_float(v[c][k]), sl, c0));
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int k = 0; k < 32; ++k)
              v[c][k] = __float_as_uint(fmaf(__uint_as_float(v[c][k]), sl, lut[max(-far, min(far, r0 + c * 32 + k)) + far]));
        }
      }
      if (j0 < full0 || j0 + KEYS > full1) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int k = 0; k < 32; ++k) {
            const int j = j0 + c * 32 + k;
            if (j < lo || j >= hi) v[c][k] = 0xff800000u;
          }
      }
      float tops[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) tops[k] = -INFINITY;
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int k = 0; k < 32; ++k) tops[k & 7] = fmaxf(tops[k & 7], __uint_as_float(v[c][k]));
      const float top = mul * fmaxf(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])), fmaxf(fmaxf(tops[4], tops[5]), fmaxf(tops[6], tops[7])));
      if (__any_sync(0xffffffffu, top > m + LAZY)) {
        const float grown = fmaxf(m, top);
        const float fix = ex2(m - (grown == -INFINITY ? 0.f : grown));
        l *= fix;
        m = grown;
        if (n > 0) {
#pragma unroll 1
          for (int c = 0; c < DP; c += 32) {
            uint32_t o[32];
            tmem_ld32_issue(t_o + c, o);
            tmem_wait(o);
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * fix);
            tmem_st32(t_o + c, o);
          }
        }
      }
      const float base = m == -INFINITY ? 0.f : m;
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t p[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const float x = ex2(fmaf(__uint_as_float(v[c][2 * k]), mul, -base)), y = ex2(fmaf(__uint_as_float(v[c][2 * k + 1]), mul, -base));
          sum[k & 3] += x + y;
          p[k] = pack_bf16(x, y);
        }
        tmem_st16(t_s + c * 16, p);
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[w]);
    }
    const bool some = t1[w] > t0[w];
    if (some) warp_wait(&o_full[w], 0, gave_up);
    tc_fence_after();
    const bool live = valid && l != 0.f;
    const float inv = live ? 1.f / l : 0.f;
    __nv_bfloat16* row = out + ((b * a.queries + i) * a.heads + head) * dim;
    for (int c = 0; c < DP && c < dim; c += 32) {
      uint32_t o[32];
      if (some) {
        tmem_ld32_issue(t_o + c, o);
        tmem_wait(o);
      }
      if (!some || !live) {
#pragma unroll
        for (int k = 0; k < 32; ++k) o[k] = 0;
      }
      if (i < a.queries) store32(row, c, dim, vec, o, inv);
    }
    if (i < a.queries) lse[(b * a.heads + head) * a.queries + i] = live ? (m + log2f(l)) * LN2 : -INFINITY;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
}

// ------------------------------------------------------------------------------------
// backward
// ------------------------------------------------------------------------------------

template <int DP>
struct Bwd {
  static constexpr int BN = DP == 64 ? 128 : 64;  // tokens of a tile
  static constexpr uint32_t X = ROWS * DP * 2, Y = BN * DP * 2;
  // TMEM columns: S, dP, then P and dS (bf16), then the sums
  static constexpr uint32_t T_DP = BN, T_P = 2 * BN, T_DS = 2 * BN + BN / 2, T_ACC = 3 * BN;
  static constexpr int MOST = 3;  // ring stages at most
};

struct BwdIo {
  const float *lse, *delta;
  __nv_bfloat16 *d0, *d1;  // dq; or dv and dk
  float* part;             // dq with a table: [batch][heads][row tiles][buckets]
  int stages, vec;
};

// the diagonal sums of a 32 x 32 piece (lane = row, x = its columns): lane l gets the sum over column - row = l - 31, and
// (l < 31) that over column - row = 31 - l. A sum moves down one lane a column; lane 31 ends one a step.
__device__ __forceinline__ void diagonals(const float (&x)[32], int lane, float& upper, float& lower) {
  float s = 0.f;
#pragma unroll
  for (int c = 0; c < 32; ++c) {
    const float from = __shfl_up_sync(0xffffffffu, s, 1);
    s = (lane ? from : 0.f) + x[c];
    const float end = __shfl_sync(0xffffffffu, s, 31);
    if (lane == c) upper = end;
  }
  lower = s;
}

template <int DP, bool DKV, bool BIAS>
__global__ void __launch_bounds__(THREADS, 1)
    backward_kernel(const __grid_constant__ CUtensorMap map_x0, const __grid_constant__ CUtensorMap map_x1, const __grid_constant__ CUtensorMap map_y0,
                    const __grid_constant__ CUtensorMap map_y1, const __grid_constant__ b200_attention a, const __grid_constant__ BwdIo io) {
  using G = Bwd<DP>;
  constexpr int BN = G::BN, HALF = BN / 2;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int ST = io.stages;
  const uint32_t s_x = smem_u32(smem), s_y = s_x + 2 * G::X;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + 2 * G::X + ST * 2 * G::Y);
  uint64_t *x_full = bars, *y_full = bars + 1, *y_empty = y_full + G::MOST, *st_full = y_empty + G::MOST, *sp_full = st_full + G::MOST, *sp_free = sp_full + 1,
           *pd_full = sp_full + 2, *pd_free = sp_full + 3, *acc_full = sp_full + 4, *idle = sp_full + 5;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(idle + 1);
  int* gave_up = reinterpret_cast<int*>(tmem_slot + 1);
  float* s_stat = reinterpret_cast<float*>(bars + 32);           // DKV: [stages][lse, delta][BN]
  float* lut = s_stat + (DKV ? G::MOST * 2 * BN : 0);            // BIAS: [2 far + 1]
  float* near = lut + (BIAS ? 2 * relative::far_of(a.relative) + 1 : 0);  // dq with BIAS: [8 warps][2 far + 1]

  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int group = (int)(a.heads / a.kv_heads), dim = (int)a.dim;
  const int hy = blockIdx.y, kvh = DKV ? hy : hy / group;
  const int64_t b = blockIdx.z;
  const Sequence seq(a, b);
  // causal blocks with the most tiles start first
  const int rt = !DKV && a.causal ? (int)(gridDim.x - 1 - blockIdx.x) : (int)blockIdx.x;
  const int r0 = rt * ROWS, row_end = DKV ? seq.keys : seq.queries, r1 = min(r0 + ROWS, row_end) - 1;
  int first = 0, per = 0;  // tiles of one head
  if (r1 >= r0) {
    const int lo = DKV ? seq.first_query(a, r0) : seq.first_key(a, r0), hi = DKV ? seq.end_query(a, r1) : seq.end_key(a, r1);
    if (hi > lo) first = lo / BN, per = (hi + BN - 1) / BN - first;
  }
  first = uniform(first), per = uniform(per);
  const int total = per * (DKV ? group : 1);
  const int far = BIAS ? relative::far_of(a.relative) : 0, bins = 2 * far + 1;
  // tile n: its head and first token
  auto head_of = [&](int n) { return DKV ? kvh * group + n / per : hy; };
  auto token_of = [&](int n) { return (first + (DKV ? n % per : n)) * BN; };

  if (threadIdx.x == 0) {
    *gave_up = 0;
    for (const CUtensorMap* m : {&map_x0, &map_x1, &map_y0, &map_y1})
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(m)) : "memory");
    mbar_init(x_full, 1);
    for (int s = 0; s < ST; ++s) {
      mbar_init(&y_full[s], 1);
      mbar_init(&y_empty[s], 1);
      mbar_init(&st_full[s], 1);
    }
    mbar_init(sp_full, 1);
    mbar_init(sp_free, 8);
    mbar_init(pd_full, 8);
    mbar_init(pd_free, 1);
    mbar_init(acc_full, 1);
    mbar_init(idle, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if constexpr (BIAS && !DKV) {
    fill_bias(lut, a, far, hy);
    for (int i = threadIdx.x; i < 8 * bins; i += THREADS) near[i] = 0.f;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = (uint32_t)uniform((int)*tmem_slot);

  if (warp == 0) {
    if (lane == 0 && total > 0) {
      const int xh = DKV ? kvh : hy;
      mbar_expect_tx(x_full, 2 * G::X);
      for (int p = 0; p < DP / 64; ++p) {
        tma_load_4d(smem + p * (ROWS * 128), &map_x0, x_full, p * 64, r0, xh, (int)b);
        tma_load_4d(smem + G::X + p * (ROWS * 128), &map_x1, x_full, p * 64, r0, xh, (int)b);
      }
      int n = 0;
      for (; n < total; ++n) {
        const int s = n % ST;
        wait(&y_empty[s], ((n / ST) & 1) ^ 1, gave_up);
        mbar_expect_tx(&y_full[s], 2 * G::Y);
        const int yh = DKV ? head_of(n) : kvh;
        for (int p = 0; p < DP / 64; ++p) {
          uint8_t* y = smem + 2 * G::X + s * 2 * G::Y + p * (BN * 128);
          tma_load_4d(y, &map_y0, &y_full[s], p * 64, token_of(n), yh, (int)b);
          tma_load_4d(y + G::Y, &map_y1, &y_full[s], p * 64, token_of(n), yh, (int)b);
        }
      }
      // every load has landed before the block may end
      wait(x_full, 0, gave_up);
      for (int m = max(0, n - ST); m < n; ++m) wait(&y_full[m % ST], (m / ST) & 1, gave_up);
    }
  } else if (warp == 1) {
    const int ks = (dim + 15) / 16, elected = elect_one();
    const uint32_t id_s = idesc_of(ROWS, BN, false), id_a = idesc_of(ROWS, ks * 16, true);
    if (total > 0) warp_wait(x_full, 0, gave_up);
    const Desc x0 = desc_at(s_x, 16), x1 = desc_at(s_x + G::X, 16), yk = desc_at(s_y, 16), ymn = desc_at(s_y, BN * 128);
    auto scores = [&](int n, int s, int par) {  // S and dP of tile n, in stage s
      warp_wait(&y_full[s], par, gave_up);
      const uint32_t y = s_y + s * 2 * G::Y;
      const int have = (DKV ? seq.queries : seq.keys) - token_of(n);
      if (have < BN && (DKV ? seq.queries < a.queries : seq.keys < a.keys)) {
        // what lies behind the sequence's end may be anything, and is multiplied by zeros in the sums
        zero_rows<BN, DP>(y, max(have, 0), lane);
        zero_rows<BN, DP>(y + G::Y, max(have, 0), lane);
        fence_proxy_async_smem();
        __syncwarp();
      }
      tc_fence_after();
      const Desc y0 = {yk.lo + s * (2 * G::Y >> 4), yk.hi}, y1 = {y0.lo + (G::Y >> 4), yk.hi};
#pragma unroll
      for (int k = 0; k < DP / 16; ++k)
        if (k < ks) mma(elected, tmem, x0, off_k<ROWS>(k), y0, off_k<BN>(k), id_s, k > 0);
#pragma unroll
      for (int k = 0; k < DP / 16; ++k)
        if (k < ks) mma(elected, tmem + G::T_DP, x1, off_k<ROWS>(k), y1, off_k<BN>(k), id_s, k > 0);
      commit(elected, sp_full);
    };
    if (total > 0) scores(0, 0, 0);
    for (int n = 0, s = 0, par = 0, next = 0; n < total; ++n, s = next) {
      next = s + 1 == ST ? 0 : s + 1;
      par ^= next == 0;
      if (n + 1 < total) {
        warp_wait(sp_free, n & 1, gave_up);
        scores(n + 1, next, par);
      }
      warp_wait(pd_full, n & 1, gave_up);
      tc_fence_after();
      const Desc y0 = {ymn.lo + s * (2 * G::Y >> 4), ymn.hi}, y1 = {y0.lo + (G::Y >> 4), ymn.hi};
      if constexpr (DKV) {
#pragma unroll
        for (int k = 0; k < BN / 16; ++k)  // dV += P dO
          mma_from_tmem(elected, tmem + G::T_ACC, tmem + G::T_P + k * 8, y1, off_mn(k), id_a, n > 0 || k > 0);
#pragma unroll
        for (int k = 0; k < BN / 16; ++k)  // dK += dS Q
          mma_from_tmem(elected, tmem + G::T_ACC + DP, tmem + G::T_DS + k * 8, y0, off_mn(k), id_a, n > 0 || k > 0);
      } else {
#pragma unroll
        for (int k = 0; k < BN / 16; ++k)  // dQ += dS K
          mma_from_tmem(elected, tmem + G::T_ACC, tmem + G::T_DS + k * 8, y0, off_mn(k), id_a, n > 0 || k > 0);
      }
      commit(elected, &y_empty[s]);
      commit(elected, pd_free);
      if (n + 1 == total) commit(elected, acc_full);
    }
    // no MMA and no commit is on its way when the block ends
    commit(elected, idle);
    warp_wait(idle, 0, gave_up);
  } else if (DKV && warp == 2) {
    // the queries' lse (log2; infinite where nothing is to be had) and delta
    for (int n = 0; n < total; ++n) {
      const int s = n % ST;
      warp_wait(&y_empty[s], ((n / ST) & 1) ^ 1, gave_up);
      const int64_t at = (b * a.heads + head_of(n)) * a.queries;
      for (int c = lane; c < BN; c += 32) {
        const int i = token_of(n) + c;
        float x = INFINITY, d = 0.f;
        if (i < seq.queries) {
          x = io.lse[at + i] * LOG2E;
          if (x == -INFINITY) x = INFINITY;
          d = io.delta[at + i];
        }
        s_stat[s * 2 * BN + c] = x;
        s_stat[s * 2 * BN + BN + c] = d;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&st_full[s]);
    }
  } else if (warp >= 4) {
    const int g = (warp - 4) >> 2, q = warp & 3;
    const int w0 = r0 + q * 32, r = w0 + lane;
    const bool valid = r < row_end;
    const int lo = !valid ? 0 : (DKV ? seq.first_query(a, r) : seq.first_key(a, r)), hi = !valid ? 0 : (DKV ? seq.end_query(a, r) : seq.end_key(a, r));
    // every token of [full0, full1) goes with all rows of the warp
    const int last = min(w0 + 31, row_end - 1);
    const int full0 = DKV ? seq.first_query(a, last) : seq.first_key(a, last), full1 = DKV ? seq.end_query(a, w0) : seq.end_key(a, w0);
    const uint32_t lanes = (uint32_t)(q * 32) << 16, tm = tmem + lanes;
    const float sl = a.scale * LOG2E;
    float row_lse = INFINITY, row_delta = 0.f, before = 0.f, after = 0.f;
    if (!DKV && valid) {
      const int64_t at = (b * a.heads + hy) * a.queries + r;
      row_lse = io.lse[at] * LOG2E;
      if (row_lse == -INFINITY) row_lse = INFINITY;
      row_delta = io.delta[at];
    }
    float* my_near = near + (warp - 4) * bins;
    int lut_head = -1;
    for (int n = 0; n < total; ++n) {
      if constexpr (BIAS && DKV) {
        // the lookup of the tile's head, by the threads that read it
        if (head_of(n) != lut_head) {
          lut_head = head_of(n);
          asm volatile("bar.sync 1, 256;" ::: "memory");
          for (int i = threadIdx.x - 128; i < bins; i += 256)
            lut[i] = table_log2(a.table, (int64_t)relative::bucket_of(a.relative, i - far) * a.heads + lut_head, a.table_dtype);
          asm volatile("bar.sync 1, 256;" ::: "memory");
        }
      }
      warp_wait(sp_full, n & 1, gave_up);
      if constexpr (DKV) warp_wait(&st_full[n % ST], (n / ST) & 1, gave_up);
      tc_fence_after();
      const float* stat = s_stat + (n % ST) * 2 * BN + g * HALF;
#pragma unroll
      for (int c0 = 0; c0 < HALF; c0 += 32) {
        const int t0 = token_of(n) + g * HALF + c0;  // first token of these columns
        uint32_t s[32], d[32];
        tmem_ld32_issue(tm + g * HALF + c0, s);
        tmem_ld32_issue(tm + G::T_DP + g * HALF + c0, d);
        tmem_wait(s);
        tmem_wait(d);
        if (c0 + 32 == HALF) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(sp_free);
        }
        float x[32];
        int w_rel = 0;  // key - query - shift of lane 0, column 0; + 1 a column for dq, - 1 for dk and dv
        bool is_near = false;
        if constexpr (BIAS) {
          w_rel = DKV ? w0 - t0 - seq.shift : t0 - w0 - seq.shift;
          const int low = w_rel - 31, high = w_rel + 31;  // over the 32 x 32 piece
          is_near = low < far && high > -far;
          if (!is_near) {
            const float c = lut[low >= far ? 2 * far : 0];
#pragma unroll
            for (int k = 0; k < 32; ++k) x[k] = fmaf(__uint_as_float(s[k]), sl, c);
          } else {
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              const int rel = DKV ? w_rel + lane - k : w_rel + k - lane;
              x[k] = fmaf(__uint_as_float(s[k]), sl, lut[max(-far, min(far, rel)) + far]);
            }
          }
        }
#pragma unroll
        for (int k = 0; k < 32; k += 4) {
          float4 ls, de;
          if constexpr (DKV) {
            ls = *reinterpret_cast<const float4*>(stat + c0 + k);
            de = *reinterpret_cast<const float4*>(stat + BN + c0 + k);
          } else {
            ls = make_float4(row_lse, row_lse, row_lse, row_lse);
            de = make_float4(row_delta, row_delta, row_delta, row_delta);
          }
          const float l4[4] = {ls.x, ls.y, ls.z, ls.w}, d4[4] = {de.x, de.y, de.z, de.w};
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const float p = ex2(BIAS ? x[k + u] - l4[u] : fmaf(__uint_as_float(s[k + u]), sl, -l4[u]));
            x[k + u] = p * (__uint_as_float(d[k + u]) - d4[u]);
            s[k + u] = __float_as_uint(p);
          }
        }
        if (t0 < full0 || t0 + 32 > full1) {
#pragma unroll
          for (int k = 0; k < 32; ++k)
            if (t0 + k < lo || t0 + k >= hi) {
              x[k] = 0.f;
              s[k] = 0;
            }
        }
        if constexpr (BIAS && !DKV) {
          if (!valid) {
#pragma unroll
            for (int k = 0; k < 32; ++k) x[k] = 0.f;
          }
          if (is_near) {
            float upper = 0.f, lower = 0.f;
            diagonals(x, lane, upper, lower);
            const int ru = w_rel + lane - 31, rl = w_rel + 31 - lane;
            if (ru >= far) after += upper;
            else if (ru <= -far) before += upper;
            else my_near[ru + far] += upper;
            __syncwarp();
            if (lane < 31) {
              if (rl >= far) after += lower;
              else if (rl <= -far) before += lower;
              else my_near[rl + far] += lower;
            }
            __syncwarp();
          } else {
            float sum = 0.f;
#pragma unroll
            for (int k = 0; k < 32; ++k) sum += x[k];
            if (w_rel - 31 >= far) after += sum;
            else before += sum;
          }
        }
        if (c0 == 0 && n > 0) {
          // the sums of the tile before have read P and dS
          warp_wait(pd_free, (n - 1) & 1, gave_up);
          tc_fence_after();
        }
        uint32_t p[16];
        if constexpr (DKV) {
#pragma unroll
          for (int k = 0; k < 16; ++k) p[k] = pack_bf16(__uint_as_float(s[2 * k]), __uint_as_float(s[2 * k + 1]));
          tmem_st16(tm + G::T_P + (g * HALF + c0) / 2, p);
        }
#pragma unroll
        for (int k = 0; k < 16; ++k) p[k] = pack_bf16(x[2 * k], x[2 * k + 1]);
        tmem_st16(tm + G::T_DS + (g * HALF + c0) / 2, p);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(pd_full);
    }
    const bool some = total > 0;
    if (some) warp_wait(acc_full, 0, gave_up);
    tc_fence_after();
    const int rows = DKV ? (int)a.keys : (int)a.queries, heads = DKV ? (int)a.kv_heads : (int)a.heads;
    // dk, dv: a warpgroup each; dq: half of the columns each
    const int from = DKV ? 0 : g * (DP / 2), to = DKV ? DP : from + DP / 2;
    const uint32_t acc = tm + G::T_ACC + (DKV ? g * DP : 0);
    __nv_bfloat16* row = (DKV && g ? io.d1 : io.d0) + ((b * rows + r) * heads + hy) * dim;
    for (int c = from; c < to && c < dim; c += 32) {
      uint32_t o[32];
      if (some) {
        tmem_ld32_issue(acc + c, o);
        tmem_wait(o);
      }
      if (!some || !valid) {
#pragma unroll
        for (int k = 0; k < 32; ++k) o[k] = 0;
      }
      if (r < rows) store32(row, c, dim, io.vec, o, DKV && !g ? 1.f : a.scale);
    }
    if constexpr (BIAS && !DKV) {
      before = warp_sum(before), after = warp_sum(after);
      if (lane == 0) my_near[0] = before, my_near[2 * far] = after;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
  if constexpr (BIAS && !DKV) {
    // the warps' sums by rel to buckets, in order
    const int nb = relative::buckets_of(a.relative);
    float* part = io.part + (((int64_t)b * gridDim.y + hy) * gridDim.x + rt) * nb;
    for (int n = threadIdx.x; n < nb; n += THREADS) {
      float s = 0.f;
      for (int i = 0; i < bins; ++i)
        if (relative::bucket_of(a.relative, i - far) == n)
#pragma unroll
          for (int w = 0; w < 8; ++w) s += near[w * bins + i];
      part[n] = s;
    }
  }
}

// ------------------------------------------------------------------------------------
// host
// ------------------------------------------------------------------------------------

// tokens whose rows TMA cannot address, copied dense with rows of whole 16 bytes
__global__ void __launch_bounds__(256)
    pack_kernel(const __nv_bfloat16* x, __nv_bfloat16* y, int64_t n, int tokens, int heads, int dim, int wide, int64_t sb, int64_t ss, int64_t sh) {
  const int64_t step = (int64_t)gridDim.x * 256;
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < n; e += step) {
    const int c = (int)(e % wide);
    const int64_t row = e / wide, h = row % heads, s = row / heads % tokens, b = row / heads / tokens;
    y[e] = c < dim ? x[b * sb + s * ss + h * sh + c] : __float2bfloat16_rn(0.f);
  }
}

struct Operand {
  const void* p;
  int64_t tokens, heads, stride[3];
};
static bool addressable(const b200_attention& a, const Operand& x) {
  if (reinterpret_cast<uintptr_t>(x.p) & 15) return false;
  const int64_t size[3] = {a.batch, x.tokens, x.heads};
  for (int i = 0; i < 3; ++i)
    if (size[i] > 1 && (x.stride[i] <= 0 || x.stride[i] % 8 || x.stride[i] >= (1ll << 38))) return false;
  return true;
}
static int64_t wide_of(const b200_attention& a) { return (a.dim + 7) / 8 * 8; }
static size_t up256(size_t n) { return (n + 255) & ~size_t(255); }
static size_t packed_bytes(const b200_attention& a, const Operand& x) {
  return addressable(a, x) ? 0 : up256((size_t)(a.batch * x.tokens * x.heads * wide_of(a)) * 2);
}
// x as TMA can address it: itself, or copied to the workspace
static int make_addressable(const b200_attention& a, Operand& x, uint8_t*& ws, cudaStream_t st) {
  if (addressable(a, x)) return B200_OK;
  const int64_t wide = wide_of(a), n = a.batch * x.tokens * x.heads * wide;
  const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(n, 256), (int64_t)num_sms() * 16);
  pack_kernel<<<grid, 256, 0, st>>>(reinterpret_cast<const __nv_bfloat16*>(x.p), reinterpret_cast<__nv_bfloat16*>(ws), n, (int)x.tokens, (int)x.heads,
                                    (int)a.dim, (int)wide, x.stride[0], x.stride[1], x.stride[2]);
  if (int rc = check_launch("attention")) return rc;
  x.p = ws;
  x.stride[0] = x.tokens * x.heads * wide, x.stride[1] = x.heads * wide, x.stride[2] = wide;
  ws += up256((size_t)n * 2);
  return B200_OK;
}
static int map_of(CUtensorMap* m, const b200_attention& a, const Operand& x, uint32_t rows) {
  const uint64_t row = (uint64_t)wide_of(a) * 2;  // a stride that is never walked
  auto bytes = [&](int64_t size, int64_t stride) { return size > 1 ? (uint64_t)stride * 2 : row; };
  return make_map(m, x.p, (uint64_t)a.dim, (uint64_t)x.tokens, (uint64_t)x.heads, (uint64_t)a.batch, bytes(x.tokens, x.stride[1]),
                  bytes(x.heads, x.stride[2]), bytes(a.batch, x.stride[0]), 64, rows);
}
static Operand operand(const void* p, int64_t tokens, int64_t heads, const int64_t* s) { return {p, tokens, heads, {s[0], s[1], s[2]}}; }
static Operand queries_of(const b200_attention& a) { return operand(a.q, a.queries, a.heads, a.q_stride); }
static Operand keys_of(const b200_attention& a) { return operand(a.k, a.keys, a.kv_heads, a.k_stride); }
static Operand values_of(const b200_attention& a) { return operand(a.v, a.keys, a.kv_heads, a.v_stride); }

static size_t bias_bytes(const b200_attention& a, int copies) {
  return a.table ? (size_t)(2 * relative::far_of(a.relative) + 1) * 4 * copies : 0;
}

template <typename Kernel>
static int allow(Kernel k) {
  // always the limit itself, so that calls of several threads do not lower it
  return cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_LIMIT) == cudaSuccess ? B200_OK : check_launch("attention");
}

template <int DP, bool BIAS>
static int launch_forward(const b200_attention& a, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, void* out, float* lse,
                          cudaStream_t st) {
  const size_t shared = 1024 + Fwd<DP>::LUT + bias_bytes(a, 1);
  const auto kernel = forward_kernel<DP, BIAS>;
  if (int rc = allow(kernel)) return rc;
  const int vec = a.dim % 8 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  kernel<<<dim3((unsigned)ceil_div(a.queries, 2 * ROWS), (unsigned)a.heads, (unsigned)a.batch), THREADS, shared, st>>>(
      q, k, v, a, reinterpret_cast<__nv_bfloat16*>(out), lse, vec);
  return check_launch("attention");
}

template <int DP, bool DKV, bool BIAS>
static int launch_backward(const b200_attention& a, const Operand (&x)[2], const Operand (&y)[2], BwdIo io, cudaStream_t st) {
  using G = Bwd<DP>;
  CUtensorMap m[4];
  for (int i = 0; i < 2; ++i) {
    if (int rc = map_of(&m[i], a, x[i], ROWS)) return rc;
    if (int rc = map_of(&m[2 + i], a, y[i], G::BN)) return rc;
  }
  auto shared = [&](int stages) {
    return 1024 + 2 * (size_t)G::X + stages * 2 * (size_t)G::Y + 256 + (DKV ? G::MOST * 2 * G::BN * 4 : 0) + bias_bytes(a, DKV ? 1 : 9);
  };
  io.stages = shared(G::MOST) <= SMEM_LIMIT ? G::MOST : 2;
  const auto kernel = backward_kernel<DP, DKV, BIAS>;
  if (int rc = allow(kernel)) return rc;
  const int64_t rows = DKV ? a.keys : a.queries;
  kernel<<<dim3((unsigned)ceil_div(rows, ROWS), (unsigned)(DKV ? a.kv_heads : a.heads), (unsigned)a.batch), THREADS, shared(io.stages), st>>>(
      m[0], m[1], m[2], m[3], a, io);
  return check_launch("attention_grad");
}

}  // namespace tiles

bool tiles_take(const b200_attention& a) { return a.dtype == B200_BF16 && a.dim <= 128 && a.queries >= 16 && a.keys >= 1; }

size_t tiles_forward_workspace(const b200_attention& a) {
  using namespace tiles;
  return packed_bytes(a, queries_of(a)) + packed_bytes(a, keys_of(a)) + packed_bytes(a, values_of(a));
}

int tiles_forward(const b200_attention& a, void* out, float* lse, void* workspace, cudaStream_t st) {
  using namespace tiles;
  uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
  Operand x[3] = {queries_of(a), keys_of(a), values_of(a)};
  CUtensorMap m[3];
  for (int i = 0; i < 3; ++i) {
    if (int rc = make_addressable(a, x[i], ws, st)) return rc;
    if (int rc = map_of(&m[i], a, x[i], 128)) return rc;
  }
  if (a.dim <= 64)
    return a.table ? launch_forward<64, true>(a, m[0], m[1], m[2], out, lse, st) : launch_forward<64, false>(a, m[0], m[1], m[2], out, lse, st);
  return a.table ? launch_forward<128, true>(a, m[0], m[1], m[2], out, lse, st) : launch_forward<128, false>(a, m[0], m[1], m[2], out, lse, st);
}

static size_t part_bytes(const b200_attention& a) {
  return a.table ? tiles::up256((size_t)(a.batch * a.heads * ceil_div(a.queries, tiles::ROWS) * relative::buckets_of(a.relative)) * 4) : 0;
}

size_t tiles_grad_workspace(const b200_attention& a, const b200_attention_grads* g) {
  using namespace tiles;
  // the gradient's own strides are not known to a caller who asks for the size: room for its copy
  const size_t d = g ? packed_bytes(a, operand(g->dout, a.queries, a.heads, g->dout_stride)) : up256((size_t)(a.batch * a.queries * a.heads * wide_of(a)) * 2);
  return part_bytes(a) + tiles_forward_workspace(a) + d;
}

int tiles_grad(const b200_attention& a, const b200_attention_grads& g, const float* delta, void* workspace, cudaStream_t st) {
  using namespace tiles;
  uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
  BwdIo io = {};
  io.lse = g.lse, io.delta = delta, io.part = reinterpret_cast<float*>(ws);
  ws += part_bytes(a);
  Operand q = queries_of(a), k = keys_of(a), v = values_of(a), d = operand(g.dout, a.queries, a.heads, g.dout_stride);
  for (Operand* x : {&q, &k, &v, &d})
    if (int rc = make_addressable(a, *x, ws, st)) return rc;
  const Operand qd[2] = {q, d}, kv[2] = {k, v};
  auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  io.d0 = reinterpret_cast<__nv_bfloat16*>(g.dq), io.vec = a.dim % 8 == 0 && aligned(g.dq);
  int rc;
  if (a.dim <= 64) rc = a.table ? launch_backward<64, false, true>(a, qd, kv, io, st) : launch_backward<64, false, false>(a, qd, kv, io, st);
  else rc = a.table ? launch_backward<128, false, true>(a, qd, kv, io, st) : launch_backward<128, false, false>(a, qd, kv, io, st);
  if (rc) return rc;
  if (a.table)
    if (int rc = table_sum(a, io.part, ceil_div(a.queries, ROWS), g.dtable, st)) return rc;
  io.d0 = reinterpret_cast<__nv_bfloat16*>(g.dv), io.d1 = reinterpret_cast<__nv_bfloat16*>(g.dk);
  io.vec = a.dim % 8 == 0 && aligned(g.dv) && aligned(g.dk);
  if (a.dim <= 64) return a.table ? launch_backward<64, true, true>(a, kv, qd, io, st) : launch_backward<64, true, false>(a, kv, qd, io, st);
  return a.table ? launch_backward<128, true, true>(a, kv, qd, io, st) : launch_backward<128, true, false>(a, kv, qd, io, st);
}

}  // namespace attention
}  // namespace b200
