// Attention on the tensor cores: bf16 heads of up to 128 elements, many queries.
//
// Forward. A block takes 128 queries of one head past the keys; two blocks share an SM, so that one's exponentials run under
// the other's MMAs, and its start and end under the other's middle:
//   warp 0      TMA: the queries once, then K and V tiles into a ring;
//   warp 1      owns 256 columns of TMEM, issues S = Q K^T (operands in shared memory) and O += P V (P from TMEM);
//   warps 2-5   softmax, a row of S a thread.
// Tiles of 64 keys: two S take turns, P lies over its S (bf16 in the lower half), O has the rest (64 + 64 + 128 columns), so that the
// next tile's S is made under this one's exponentials. MMAs run in their order: an S is overwritten only when the P over it is used up.
// (One S of 128 keys with P over it, whose successor waited for P, took 314 us for 2 x 4096 causal tokens of 32 heads of 128, this 276;
// S of 128 keys beside P, with two threads a row that exchange its maximum, 167 us for 64 x 512 tokens of 16 heads of 64, this 151.)
// The running maximum moves only when a row's has grown by 2^8 (probabilities stay below 2^8, sums are fp32), so O is hardly ever
// rescaled.
// Making up to 3 of 8 exponentials on the FMA pipe changed nothing (the special function unit is busy for 60 % of the time): not done.
//
// Backward, one kernel in two forms. 128 rows stay, tiles of 64 tokens of the other side go past:
//   dq:      rows are queries (Q, dO), tiles are keys (K, V):     S = Q K^T, dP = dO V^T, dQ += dS K
//   dk, dv:  rows are keys (K, V), tiles are queries (Q, dO):     S = K Q^T, dP = V dO^T, dV += P dO, dK += dS Q
// so p and dz of a tile are made by the threads that own its rows, go back to TMEM as bf16 over the S and dP that they come
// from, and are the A operand of the sums there: nothing is transposed, no sum leaves its block, every order is fixed. S and
// dP are made twice for that (7 products instead of 5). Two warpgroups share a tile, 32 columns each (one for all 64 took as long).
// Heads of up to 64: 256 columns of TMEM a block and two blocks an SM; wider heads: two pairs of warpgroups that take tiles in turn,
// each with an S and dP of its own (one pair: 739 us for 4 x 2048 tokens of 16 heads of 128, two: 537).
// Tiles of 64 because of TMEM; an MMA of 128 x 64 from shared memory takes 48 clocks, of 128 x 128 64 (measured).
// dk and dv are capped at 96 registers (two blocks of 10 warps or one of 18: five warps to a quarter of an SM) and spill 84 to 116 bytes
// a thread, dq of heads of 64 with a bias 56.
// What bounds both directions is the chain of a tile, with two tiles under way on an SM: the tensor pipe is active for 29 to 36 % of
// the time, the special function unit for 29 to 62 %, issue slots for 40 to 46 % (8 x 2048 tokens of 16 heads of 64: forward 216, dq 274,
// dk and dv 441 us).
//
// Probabilities and dz are rounded to bf16 for the products that they are operands of: both operands of an MMA have one type, the
// heads', and a second plane for what is lost would double those products, against an error of 2.0e-3 (outputs) to 2.9e-3 (gradients)
// where the results' own rounding is 1.7e-3. Scores, maxima, sums and all accumulators are fp32; exponentials are ex2.approx, whose
// error of 2^-22 is far below a bf16 operand's 2^-8 (the row kernels use exp2f, so their bits differ).
// Every wait is bounded (tc_common.cuh); on expiry the error flag is set and the block winds down.
#include <algorithm>

#include "attention.cuh"
#include "tc_common.cuh"

namespace b200 {
namespace attention {
namespace tiles {

using namespace tc;

constexpr int ROWS = 128;
constexpr uint32_t SMEM_LIMIT = 232448;

// Which rows and head a block has. Blocks of one group of heads come one after the other, and in it the row tiles in turn: causal
// calls with the most tiles first and as many heads a group as have their tokens in the L2, others head by head.
struct Order {
  int row_tiles, heads, pairs, group, last_first;  // pairs: batch x heads
};
struct Place {
  int tile, head;
  int64_t batch;
  __device__ __forceinline__ Place(const Order& o) {
    const int per = o.group * o.row_tiles;
    const int g = (int)blockIdx.x / per, r = (int)blockIdx.x % per;
    const int size = min(o.group, o.pairs - g * o.group);
    const int pair = g * o.group + r % size;
    tile = r / size;
    if (o.last_first) tile = o.row_tiles - 1 - tile;
    head = pair % o.heads, batch = pair / o.heads;
  }
};

// Bounded wait of whoever calls it. A look at the timer takes longer than a tile's MMAs, so it comes every 256 polls. After
// WAIT_LIMIT_NS the block gives up: every later wait ends at once, results are not valid, the error flag says so.
__device__ __forceinline__ bool given_up(const int* gave_up) { return *reinterpret_cast<const volatile int*>(gave_up) != 0; }
template <bool EVEN_THEN = false>
__device__ __forceinline__ void wait(uint64_t* bar, uint32_t parity, int* gave_up) {
  unsigned long long t0 = 0;
  while (true) {
#pragma unroll 1
    for (int k = 0; k < 256; ++k) {
      if (mbar_try_wait(bar, parity)) return;
      if (!EVEN_THEN && given_up(gave_up)) return;
    }
    const unsigned long long now = globaltimer();
    if (t0 == 0) t0 = now;
    else if (now - t0 > WAIT_LIMIT_NS) {
      raise_device_error(B200_ERR_TIMEOUT);
      *reinterpret_cast<volatile int*>(gave_up) = 1;
      return;
    }
  }
}
// for what is in flight when a block ends (copies into its shared memory, its MMAs): waited for even by a block that has given up,
// with a limit of its own
__device__ __forceinline__ void settle(uint64_t* bar, uint32_t parity, int* gave_up) { wait<true>(bar, parity, gave_up); }
// by all lanes, together again behind it (61 clocks where it is satisfied; one polling lane and the others' wait for it 136)
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
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr)
      : "memory");
}
// `bytes` (a multiple of 16, both addresses too) of global memory, counted on the barrier
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes),
               "r"(smem_u32(bar))
               : "memory");
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

// two fp32 in one instruction
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(__float_as_uint(a)), "r"(__float_as_uint(b)));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t r, float& a, float& b) {
  uint32_t x, y;
  asm("mov.b64 {%0, %1}, %2;" : "=r"(x), "=r"(y) : "l"(r));
  a = __uint_as_float(x), b = __uint_as_float(y);
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// first in a block of code that few tiles run: keeps it behind a branch (as selects of every element it is a third of all
// instructions)
__device__ __forceinline__ void seldom() { asm volatile("" ::: "memory"); }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
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

constexpr int KEYS = 64, FWD_THREADS = 192;
constexpr float LAZY = 8.f;  // log2 by which a maximum may grow before O is rescaled

template <int DP>
struct Fwd {
  static constexpr int STAGES = DP == 64 ? 4 : 2;
  static constexpr uint32_t Q = ROWS * DP * 2, TILE = KEYS * DP * 2;
  static constexpr uint32_t BARS = Q + STAGES * 2 * TILE, LUT = BARS + 256;
  static constexpr uint32_t TMEM = 256, T_O = TMEM - DP;
};

template <int DP, bool BIAS>
__global__ void __launch_bounds__(FWD_THREADS, 2)
    forward_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                   const __grid_constant__ b200_attention a, const __grid_constant__ Order order, __nv_bfloat16* out, float* lse, int vec) {
  using F = Fwd<DP>;
  constexpr int ST = F::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t s_q = smem_u32(smem), s_k = s_q + F::Q, s_v = s_k + ST * F::TILE;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + F::BARS);
  uint64_t *q_full = bars, *k_full = bars + 1, *k_empty = k_full + ST, *v_full = k_empty + ST, *v_empty = v_full + ST, *s_full = v_empty + ST,
           *p_full = s_full + 2, *o_done = s_full + 4, *idle = s_full + 6;  // s_full, p_full, o_done: one each for even and odd tiles
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(idle + 1);
  int* gave_up = reinterpret_cast<int*>(tmem_slot + 1);
  float* lut = reinterpret_cast<float*>(smem + F::LUT);

  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const Place at(order);
  const int head = at.head, kvh = head / (int)(a.heads / a.kv_heads), dim = (int)a.dim;
  const int64_t b = at.batch;
  const Sequence seq(a, b);
  const int r0 = at.tile * ROWS;
  int T0 = 0, n_tiles = 0;  // key tiles
  {
    const int r1 = min(r0 + ROWS, seq.queries) - 1;
    if (r1 >= r0) {
      const int lo = seq.first_key(a, r0), hi = seq.end_key(a, r1);
      if (hi > lo) T0 = lo / KEYS, n_tiles = (hi + KEYS - 1) / KEYS - T0;
    }
    T0 = uniform(T0), n_tiles = uniform(n_tiles);
  }
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
    for (int e = 0; e < 2; ++e) {
      // two sets: a tile's scores are full before every warp has seen the ones before, and a warp may hand over a tile's P before
      // another has the last one's; the next but one needs both
      mbar_init(&s_full[e], 1);
      mbar_init(&p_full[e], 4);
      mbar_init(&o_done[e], 1);
    }
    mbar_init(idle, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(F::TMEM));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if constexpr (BIAS) fill_bias(lut, a, far, head);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = (uint32_t)uniform((int)*tmem_slot);

  if (warp == 0) {
    if (lane == 0 && n_tiles > 0) {
      mbar_expect_tx(q_full, F::Q);
      for (int p = 0; p < DP / 64; ++p) tma_load_4d(smem + p * (ROWS * 128), &map_q, q_full, p * 64, r0, head, (int)b);
      int keys = 0, values = 0;  // tiles under way: none into a stage that a block which gave up may still read or fill
      for (int n = 0; n < n_tiles; ++n) {
        const int s = n % ST;
        const uint32_t par = ((n / ST) & 1) ^ 1;
        wait(&k_empty[s], par, gave_up);
        if (given_up(gave_up)) break;
        ++keys;
        mbar_expect_tx(&k_full[s], F::TILE);
        for (int p = 0; p < DP / 64; ++p)
          tma_load_4d(smem + F::Q + s * F::TILE + p * (KEYS * 128), &map_k, &k_full[s], p * 64, (T0 + n) * KEYS, kvh, (int)b);
        wait(&v_empty[s], par, gave_up);
        if (given_up(gave_up)) break;
        ++values;
        mbar_expect_tx(&v_full[s], F::TILE);
        for (int p = 0; p < DP / 64; ++p)
          tma_load_4d(smem + F::Q + (ST + s) * F::TILE + p * (KEYS * 128), &map_v, &v_full[s], p * 64, (T0 + n) * KEYS, kvh, (int)b);
      }
      // every load has landed before the block may end
      settle(q_full, 0, gave_up);
      for (int m = max(0, keys - ST); m < keys; ++m) settle(&k_full[m % ST], (m / ST) & 1, gave_up);
      for (int m = max(0, values - ST); m < values; ++m) settle(&v_full[m % ST], (m / ST) & 1, gave_up);
    }
  } else if (warp == 1) {
    const int ks = (dim + 15) / 16, elected = elect_one();
    const uint32_t id_s = idesc_of(ROWS, KEYS, false), id_o = idesc_of(ROWS, ks * 16, true);
    const Desc dq = desc_at(s_q, 16), dk = desc_at(s_k, 16), dv = desc_at(s_v, KEYS * 128);
    auto scores = [&](int s, int par, int n) {  // S of tile n, in stage s
      warp_wait(&k_full[s], par, gave_up);
      tc_fence_after();
      const Desc kd = {dk.lo + s * (F::TILE >> 4), dk.hi};
#pragma unroll
      for (int k = 0; k < DP / 16; ++k)
        if (k < ks) mma(elected, tmem + (n & 1) * KEYS, dq, off_k<ROWS>(k), kd, off_k<KEYS>(k), id_s, k > 0);
      commit(elected, &s_full[n & 1]);
      commit(elected, &k_empty[s]);
    };
    if (n_tiles > 0) {
      warp_wait(q_full, 0, gave_up);
      scores(0, 0, 0);
    }
    for (int n = 0, s = 0, par = 0, next = 0, next_par = 0; n < n_tiles; ++n, s = next, par = next_par) {
      next = s + 1 == ST ? 0 : s + 1, next_par = s + 1 == ST ? par ^ 1 : par;
      if (n + 1 < n_tiles) scores(next, next_par, n + 1);  // over the P before this one, which is used up
      warp_wait(&v_full[s], par, gave_up);
      const int have = seq.keys - (T0 + n) * KEYS;
      if (have < KEYS && seq.keys < a.keys) {
        // what lies behind the sequence's end may be anything, and is multiplied by zeros
        zero_rows<KEYS, DP>(s_v + s * F::TILE, max(have, 0), lane);
        fence_proxy_async_smem();
        __syncwarp();
      }
      const Desc vd = {dv.lo + s * (F::TILE >> 4), dv.hi};
      warp_wait(&p_full[n & 1], (n >> 1) & 1, gave_up);
      tc_fence_after();
#pragma unroll
      for (int k = 0; k < KEYS / 16; ++k)
        mma_from_tmem(elected, tmem + F::T_O, tmem + (n & 1) * KEYS + k * 8, vd, off_mn(k), id_o, n > 0 || k > 0);
      commit(elected, &v_empty[s]);
      commit(elected, &o_done[n & 1]);
    }
    // no MMA and no commit is on its way when the block ends
    commit(elected, idle);
    settle(idle, 0, gave_up);
    __syncwarp();
  } else {
    const int q = warp & 3;
    const int i0 = r0 + q * 32, i = i0 + lane;
    const bool valid = i < seq.queries;
    const int lo = valid ? seq.first_key(a, i) : 0, hi = valid ? seq.end_key(a, i) : 0;
    // every key of [full0, full1) is seen by all rows of the warp
    const int full0 = seq.first_key(a, min(i0 + 31, seq.queries - 1)), full1 = seq.end_key(a, i0);
    const uint32_t t_row = tmem + ((uint32_t)(q * 32) << 16), t_o = t_row + F::T_O;
    const float sl = a.scale * LOG2E;
    float m = -INFINITY, l = 0.f;
    for (int n = 0; n < n_tiles; ++n) {
      const int j0 = (T0 + n) * KEYS;
      const uint32_t t_s = t_row + (n & 1) * KEYS;
      warp_wait(&s_full[n & 1], (n >> 1) & 1, gave_up);
      tc_fence_after();
      uint32_t v[2][32];
      tmem_ld32_issue(t_s, v[0]);
      tmem_ld32_issue(t_s + 32, v[1]);
      tmem_wait(v[0]);
      tmem_wait(v[1]);
      float mul = sl;
      if constexpr (BIAS) {
        mul = 1.f;
        const int rel0 = j0 - i - seq.shift;   // of column 0
        const int w_rel = j0 - i0 - seq.shift;  // of lane 0
        if (w_rel - 31 >= far || w_rel + 63 <= -far) {
          const float c0 = lut[w_rel >= far ? 2 * far : 0];
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int k = 0; k < 32; ++k) v[c][k] = __float_as_uint(fmaf(__uint_as_float(v[c][k]), sl, c0));
        } else {
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int k = 0; k < 32; ++k)
              v[c][k] = __float_as_uint(fmaf(__uint_as_float(v[c][k]), sl, lut[max(-far, min(far, rel0 + c * 32 + k)) + far]));
        }
      }
      const bool cut = j0 < full0 || j0 + 64 > full1;
      if (cut) {
        seldom();
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int k = 0; k < 32; ++k) {
            const int j = j0 + c * 32 + k;
            if (j < lo || j >= hi) v[c][k] = 0xff800000u;
          }
      }
      float tops[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        tops[c] = __uint_as_float(v[c >> 1][16 * (c & 1)]);
#pragma unroll
        for (int k = 1; k < 15; k += 2)
          tops[c] = fmaxf(fmaxf(tops[c], __uint_as_float(v[c >> 1][16 * (c & 1) + k])), __uint_as_float(v[c >> 1][16 * (c & 1) + k + 1]));
        tops[c] = fmaxf(tops[c], __uint_as_float(v[c >> 1][16 * (c & 1) + 15]));
      }
      const float top = mul * fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
      float fix = 1.f;
      const bool moved = __any_sync(0xffffffffu, top > m + LAZY);
      if (moved) {
        const float grown = fmaxf(m, top);
        fix = ex2(m - (grown == -INFINITY ? 0.f : grown));
        l *= fix;
        m = grown;
      }
      const float base = m == -INFINITY ? 0.f : m;
      const uint64_t mul22 = pack2(mul, mul), base2 = pack2(-base, -base);
      uint64_t sum[2] = {0, 0};  // two zeros each
      uint32_t p[32];
#pragma unroll
      for (int k = 0; k < 32; ++k) {
        const int c = k >> 4, e = 2 * (k & 15);
        float x, y;
        unpack2(fma2(pack2(__uint_as_float(v[c][e]), __uint_as_float(v[c][e + 1])), mul22, base2), x, y);
        x = ex2(x), y = ex2(y);
        sum[k & 1] = add2(sum[k & 1], pack2(x, y));
        p[k] = pack_bf16(x, y);
      }
      if (n > 0 && moved) {
        warp_wait(&o_done[(n - 1) & 1], ((n - 1) >> 1) & 1, gave_up);  // O at rest
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < DP; c += 16) {
          uint32_t o[16];
          tmem_ld16(t_o + c, o);
#pragma unroll
          for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * fix);
          tmem_st16(t_o + c, o);
        }
      }
      tmem_st32(t_s, p);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[n & 1]);
      float s0, s1, s2, s3;
      unpack2(sum[0], s0, s1);
      unpack2(sum[1], s2, s3);
      l += (s0 + s1) + (s2 + s3);
    }
    if (n_tiles > 0) warp_wait(&o_done[(n_tiles - 1) & 1], ((n_tiles - 1) >> 1) & 1, gave_up);
    tc_fence_after();
    const bool live = valid && l != 0.f;
    const float inv = live ? 1.f / l : 0.f;
    __nv_bfloat16* row = out + ((b * a.queries + i) * a.heads + head) * dim;
    for (int c = 0; c < DP && c < dim; c += 32) {
      uint32_t o[32];
      if (n_tiles > 0) {
        tmem_ld32_issue(t_o + c, o);
        tmem_wait(o);
      }
      if (n_tiles == 0 || !live) {
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
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(F::TMEM));
  }
}

// ------------------------------------------------------------------------------------
// backward
// ------------------------------------------------------------------------------------

constexpr int BN = 64;  // tokens of a tile

template <int DP, bool DKV, bool BIAS>
struct Bwd {
  // pairs of warpgroups, which take tiles in turn (32 columns of a tile a warpgroup); dq's sums by diagonal, a set a warp, leave
  // room for one
  static constexpr int GROUPS = DP == 64 || (BIAS && !DKV) ? 1 : 2;
  static constexpr int THREADS = 64 + 256 * GROUPS, STAGES = 3;
  static constexpr uint32_t X = ROWS * DP * 2, Y = BN * DP * 2;
  // TMEM: each warpgroup's S and dP (P and dS over them), then the sums
  static constexpr uint32_t TMEM = DP == 64 ? 256 : 512, T_ACC = GROUPS * 2 * BN;
};

struct BwdIo {
  const float *lse, *delta;  // [batch x heads][padded], both negated: lse in the log2 domain (-inf where nothing is seen), dout . out
  int padded, stages, vec;
  __nv_bfloat16 *d0, *d1;  // dq; or dv and dk
  float* part;             // dq with a table: [batch][heads][row tiles][buckets]
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
__global__ void __launch_bounds__(Bwd<DP, DKV, BIAS>::THREADS, DP == 64 ? 2 : 1)
    backward_kernel(const __grid_constant__ CUtensorMap map_x0, const __grid_constant__ CUtensorMap map_x1, const __grid_constant__ CUtensorMap map_y0,
                    const __grid_constant__ CUtensorMap map_y1, const __grid_constant__ b200_attention a, const __grid_constant__ Order order,
                    const __grid_constant__ BwdIo io) {
  using G = Bwd<DP, DKV, BIAS>;
  constexpr int WG = G::GROUPS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int ST = io.stages;
  const uint32_t s_x = smem_u32(smem), s_y = s_x + 2 * G::X;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + 2 * G::X + ST * 2 * G::Y);
  uint64_t *x_full = bars, *y_full = bars + 1, *y_empty = y_full + G::STAGES, *sp_full = y_empty + G::STAGES, *pd_full = sp_full + 2, *acc_full = pd_full + 2,
           *idle = acc_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(idle + 1);
  int* gave_up = reinterpret_cast<int*>(tmem_slot + 1);
  float* s_stat = reinterpret_cast<float*>(bars + 32);           // DKV: [stages][lse, delta][BN]
  float* lut0 = s_stat + (DKV ? G::STAGES * 2 * BN : 0);         // BIAS: [2 far + 1], for dk and dv one a pair of warpgroups
  const int far = BIAS ? relative::far_of(a.relative) : 0, bins = 2 * far + 1;
  float* near = lut0 + bins;                                     // dq with BIAS: [warps][2 far + 1]

  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const Place at(order);
  const int group = (int)(a.heads / a.kv_heads), dim = (int)a.dim;
  const int hy = at.head, kvh = DKV ? hy : hy / group;
  const int64_t b = at.batch;
  const Sequence seq(a, b);
  const int rt = at.tile, r0 = rt * ROWS, row_end = DKV ? seq.keys : seq.queries;
  int first = 0, per = 0;  // tiles of one head
  {
    const int r1 = min(r0 + ROWS, row_end) - 1;
    if (r1 >= r0) {
      const int lo = DKV ? seq.first_query(a, r0) : seq.first_key(a, r0), hi = DKV ? seq.end_query(a, r1) : seq.end_key(a, r1);
      if (hi > lo) first = lo / BN, per = (hi + BN - 1) / BN - first;
    }
    first = uniform(first), per = uniform(per);
  }
  const int total = per * (DKV ? group : 1);
  // a warp's way through the tiles: head and first token, ring stage and its parity, without divisions
  struct Step {
    int head, tile, stage, parity;
  };
  auto start = [&]() { return Step{DKV ? kvh * group : hy, 0, 0, 0}; };
  auto advance = [&](Step& x) {
    if (++x.stage == ST) x.stage = 0, x.parity ^= 1;
    if (++x.tile == per && DKV) x.tile = 0, ++x.head;
  };
  auto token_of = [&](const Step& x) { return (first + x.tile) * BN; };

  if (threadIdx.x == 0) {
    *gave_up = 0;
    for (const CUtensorMap* m : {&map_x0, &map_x1, &map_y0, &map_y1})
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(m)) : "memory");
    mbar_init(x_full, 1);
    for (int s = 0; s < ST; ++s) {
      mbar_init(&y_full[s], 1);
      mbar_init(&y_empty[s], 1);
    }
    for (int g = 0; g < 2; ++g) {
      mbar_init(&sp_full[g], 1);
      mbar_init(&pd_full[g], 8);
    }
    mbar_init(acc_full, 1);
    mbar_init(idle, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(G::TMEM));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if constexpr (BIAS && !DKV) {
    fill_bias(lut0, a, far, hy);
    for (int i = threadIdx.x; i < 8 * WG * bins; i += G::THREADS) near[i] = 0.f;
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
      Step x = start();
      int n = 0;  // tiles under way, as in the forward
      for (; n < total; ++n, advance(x)) {
        const int s = x.stage, token = token_of(x), yh = DKV ? x.head : kvh;
        wait(&y_empty[s], x.parity ^ 1, gave_up);
        if (given_up(gave_up)) break;
        mbar_expect_tx(&y_full[s], 2 * G::Y + (DKV ? 2 * BN * 4 : 0));
        for (int p = 0; p < DP / 64; ++p) {
          uint8_t* y = smem + 2 * G::X + s * 2 * G::Y + p * (BN * 128);
          tma_load_4d(y, &map_y0, &y_full[s], p * 64, token, yh, (int)b);
          tma_load_4d(y + G::Y, &map_y1, &y_full[s], p * 64, token, yh, (int)b);
        }
        if constexpr (DKV) {  // 256 bytes each, on 256-byte boundaries; rows are padded to whole tiles
          const int64_t from = (b * a.heads + yh) * io.padded + token;
          bulk_load(s_stat + s * 2 * BN, io.lse + from, BN * 4, &y_full[s]);
          bulk_load(s_stat + s * 2 * BN + BN, io.delta + from, BN * 4, &y_full[s]);
        }
      }
      // every load has landed before the block may end
      settle(x_full, 0, gave_up);
      for (int m = max(0, n - ST); m < n; ++m) settle(&y_full[m % ST], (m / ST) & 1, gave_up);
    }
  } else if (warp == 1) {
    const int ks = (dim + 15) / 16, elected = elect_one();
    const uint32_t id_s = idesc_of(ROWS, BN, false), id_a = idesc_of(ROWS, ks * 16, true);
    const Desc x0 = desc_at(s_x, 16), x1 = desc_at(s_x + G::X, 16), yk = desc_at(s_y, 16), ymn = desc_at(s_y, BN * 128);
    Step next = start();
    auto scores = [&](int g) {  // S and dP of the next tile, for warpgroups g
      const int ls = next.stage;
      warp_wait(&y_full[ls], next.parity, gave_up);
      const int have = (DKV ? seq.queries : seq.keys) - token_of(next);
      if (have < BN && (DKV ? seq.queries < a.queries : seq.keys < a.keys)) {
        // what lies behind the sequence's end may be anything, and is multiplied by zeros in the sums
        const uint32_t y = s_y + ls * 2 * G::Y;
        zero_rows<BN, DP>(y, max(have, 0), lane);
        zero_rows<BN, DP>(y + G::Y, max(have, 0), lane);
        fence_proxy_async_smem();
        __syncwarp();
      }
      tc_fence_after();
      const uint32_t t_s = tmem + g * 2 * BN;
      const Desc y0 = {yk.lo + ls * (2 * G::Y >> 4), yk.hi}, y1 = {y0.lo + (G::Y >> 4), yk.hi};
#pragma unroll
      for (int k = 0; k < DP / 16; ++k)
        if (k < ks) mma(elected, t_s, x0, off_k<ROWS>(k), y0, off_k<BN>(k), id_s, k > 0);
#pragma unroll
      for (int k = 0; k < DP / 16; ++k)
        if (k < ks) mma(elected, t_s + BN, x1, off_k<ROWS>(k), y1, off_k<BN>(k), id_s, k > 0);
      commit(elected, &sp_full[g]);
      advance(next);
    };
    if (total > 0) {
      warp_wait(x_full, 0, gave_up);
      for (int n = 0; n < WG && n < total; ++n) scores(n);
    }
    for (int n = 0, s = 0, g = 0, par = 0; n < total; ++n, s = s + 1 == ST ? 0 : s + 1) {
      warp_wait(&pd_full[g], par, gave_up);
      tc_fence_after();
      const uint32_t t_s = tmem + g * 2 * BN;
      const Desc y0 = {ymn.lo + s * (2 * G::Y >> 4), ymn.hi}, y1 = {y0.lo + (G::Y >> 4), ymn.hi};
      if constexpr (DKV) {
#pragma unroll
        for (int k = 0; k < BN / 16; ++k)  // dV += P dO
          mma_from_tmem(elected, tmem + G::T_ACC, t_s + k * 8, y1, off_mn(k), id_a, n > 0 || k > 0);
#pragma unroll
        for (int k = 0; k < BN / 16; ++k)  // dK += dS Q
          mma_from_tmem(elected, tmem + G::T_ACC + DP, t_s + BN + k * 8, y0, off_mn(k), id_a, n > 0 || k > 0);
      } else {
#pragma unroll
        for (int k = 0; k < BN / 16; ++k)  // dQ += dS K
          mma_from_tmem(elected, tmem + G::T_ACC, t_s + BN + k * 8, y0, off_mn(k), id_a, n > 0 || k > 0);
      }
      commit(elected, &y_empty[s]);
      if (n + 1 == total) commit(elected, acc_full);
      // behind the sums in the MMAs' order: their P and dS are used up when it overwrites them
      if (n + WG < total) scores(g);
      if (++g == WG) g = 0, par ^= 1;
    }
    // no MMA and no commit is on its way when the block ends
    commit(elected, idle);
    settle(idle, 0, gave_up);
    __syncwarp();
  } else {
    const int g = (warp - 2) >> 3, half = ((warp - 2) >> 2) & 1, q = warp & 3;
    const int w0 = r0 + q * 32, r = w0 + lane;
    const bool valid = r < row_end;
    const int lo = !valid ? 0 : (DKV ? seq.first_query(a, r) : seq.first_key(a, r)), hi = !valid ? 0 : (DKV ? seq.end_query(a, r) : seq.end_key(a, r));
    // every token of [full0, full1) goes with all rows of the warp
    const int last = min(w0 + 31, row_end - 1);
    const int full0 = DKV ? seq.first_query(a, last) : seq.first_key(a, last), full1 = DKV ? seq.end_query(a, w0) : seq.end_key(a, w0);
    const uint32_t tm = tmem + ((uint32_t)(q * 32) << 16), t_s = tm + g * 2 * BN;
    const float sl = a.scale * LOG2E;
    const uint64_t sl2 = pack2(sl, sl);
    float row_lse = -INFINITY, row_delta = 0.f, before = 0.f, after = 0.f;
    if (!DKV && valid) {
      const int64_t from = (b * a.heads + hy) * io.padded + r;
      row_lse = io.lse[from];
      row_delta = io.delta[from];
    }
    float* lut = lut0 + (DKV ? g * bins : 0);
    float* my_near = near + (warp - 2) * bins;
    int lut_head = -1, par = 0;
    Step at_tile = start();
    if (g && total > 0) advance(at_tile);
    for (int n = g; n < total; n += WG, par ^= 1) {
      const Step x_at = at_tile;
      const int token = token_of(x_at);
#pragma unroll
      for (int k = 0; k < WG; ++k) advance(at_tile);
      if constexpr (BIAS && DKV) {
        // the lookup of the tile's head, by the threads that read it
        if (x_at.head != lut_head) {
          lut_head = x_at.head;
          asm volatile("bar.sync %0, 256;" ::"r"(1 + g) : "memory");
          for (int i = ((half * 4 + q) << 5) + lane; i < bins; i += 256)
            lut[i] = table_log2(a.table, (int64_t)relative::bucket_of(a.relative, i - far) * a.heads + lut_head, a.table_dtype);
          asm volatile("bar.sync %0, 256;" ::"r"(1 + g) : "memory");
        }
      }
      if constexpr (DKV) warp_wait(&y_full[x_at.stage], x_at.parity, gave_up);  // lse and delta
      warp_wait(&sp_full[g], par, gave_up);
      tc_fence_after();
      const float* stat = s_stat + x_at.stage * 2 * BN;
      {
        const int c0 = half * 32, t0 = token + c0;  // this warp's columns, and the first's token
        uint32_t s[32], d[32];
        tmem_ld32_issue(t_s + c0, s);
        tmem_ld32_issue(t_s + BN + c0, d);
        tmem_wait(s);
        tmem_wait(d);
        // P and dS go over what the other half's warp of these rows may not have read yet
        tc_fence_before();
        asm volatile("bar.sync %0, 64;" ::"r"(3 + g * 4 + q) : "memory");
        tc_fence_after();
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
        // p = 2^(x - lse), dz = p (dP - delta), two columns at a time
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
          const uint64_t l2[2] = {pack2(ls.x, ls.y), pack2(ls.z, ls.w)}, d2[2] = {pack2(de.x, de.y), pack2(de.z, de.w)};
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int e = k + 2 * u;
            const uint64_t z = BIAS ? add2(pack2(x[e], x[e + 1]), l2[u]) : fma2(pack2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), sl2, l2[u]);
            float p0, p1;
            unpack2(z, p0, p1);
            p0 = ex2(p0), p1 = ex2(p1);
            unpack2(mul2(pack2(p0, p1), add2(pack2(__uint_as_float(d[e]), __uint_as_float(d[e + 1])), d2[u])), x[e], x[e + 1]);
            s[e] = __float_as_uint(p0), s[e + 1] = __float_as_uint(p1);
          }
        }
        if (t0 < full0 || t0 + 32 > full1) {
          seldom();
#pragma unroll
          for (int k = 0; k < 32; ++k)
            if (t0 + k < lo || t0 + k >= hi) {
              x[k] = 0.f;
              s[k] = 0;
            }
        }
        uint32_t p[16];
        if constexpr (DKV) {
#pragma unroll
          for (int k = 0; k < 16; ++k) p[k] = pack_bf16(__uint_as_float(s[2 * k]), __uint_as_float(s[2 * k + 1]));
          tmem_st16(t_s + c0 / 2, p);
        }
#pragma unroll
        for (int k = 0; k < 16; ++k) p[k] = pack_bf16(x[2 * k], x[2 * k + 1]);
        tmem_st16(t_s + BN + c0 / 2, p);
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
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&pd_full[g]);
    }
    if (total > 0) warp_wait(acc_full, 0, gave_up);
    tc_fence_after();
    const int part = g * 2 + half, parts = 2 * WG;  // dv and dk: half of the warpgroups each; each a share of the columns
    const int rows = DKV ? (int)a.keys : (int)a.queries, heads = DKV ? (int)a.kv_heads : (int)a.heads;
    const int which = DKV ? part & 1 : 0, share = DKV ? part >> 1 : part, shares = DKV ? WG : parts;
    const uint32_t acc = tm + G::T_ACC + which * DP;
    __nv_bfloat16* row = (which ? io.d1 : io.d0) + ((b * rows + r) * heads + hy) * dim;
    for (int c = share * 32; c < DP && c < dim; c += shares * 32) {
      uint32_t o[32];
      if (total > 0) {
        tmem_ld32_issue(acc + c, o);
        tmem_wait(o);
      }
      if (total == 0 || !valid) {
#pragma unroll
        for (int k = 0; k < 32; ++k) o[k] = 0;
      }
      if (r < rows) store32(row, c, dim, io.vec, o, DKV && !which ? 1.f : a.scale);
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
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(G::TMEM));
  }
  if constexpr (BIAS && !DKV) {
    // the warps' sums by rel, then to buckets, in order
    for (int i = threadIdx.x; i < bins; i += G::THREADS) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < 8 * WG; ++w) s += near[w * bins + i];
      lut0[i] = s;
    }
    __syncthreads();
    const int nb = relative::buckets_of(a.relative);
    float* part = io.part + ((b * a.heads + hy) * order.row_tiles + rt) * nb;
    for (int n = threadIdx.x; n < nb; n += G::THREADS) part[n] = relative::bucket_sum(a.relative, far, lut0, n);
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

// `heads` of rows, row tiles of them; `bytes`: the tokens that go past a head's rows
static int order_of(Order* o, const b200_attention& a, int64_t heads, int64_t rows, int64_t bytes, bool last_first) {
  const int64_t tiles = ceil_div(rows, ROWS), pairs = a.batch * heads;
  B200_REQUIRE(tiles * pairs < (1ll << 31), "attention: %lld rows of %lld heads are too many", (long long)rows, (long long)pairs);
  // causal: 32 MB of them at a time, a quarter of the L2
  const int64_t group = a.causal ? std::max<int64_t>(1, (32ll << 20) / std::max<int64_t>(1, bytes)) : 1;
  *o = {(int)tiles, (int)heads, (int)pairs, (int)std::min(group, pairs), a.causal && last_first};
  return B200_OK;
}

template <int DP, bool BIAS>
static int launch_forward(const b200_attention& a, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, void* out, float* lse,
                          cudaStream_t st) {
  Order order;
  if (int rc = order_of(&order, a, a.heads, a.queries, a.keys * a.dim * 4 * a.kv_heads / a.heads, true)) return rc;
  const size_t shared = 1024 + Fwd<DP>::LUT + bias_bytes(a, 1);
  const auto kernel = forward_kernel<DP, BIAS>;
  if (int rc = allow(kernel)) return rc;
  const int vec = a.dim % 8 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  kernel<<<(unsigned)(order.row_tiles * order.pairs), FWD_THREADS, shared, st>>>(q, k, v, a, order, reinterpret_cast<__nv_bfloat16*>(out), lse, vec);
  return check_launch("attention");
}

template <int DP, bool DKV, bool BIAS>
static int launch_backward(const b200_attention& a, const Operand (&x)[2], const Operand (&y)[2], BwdIo io, cudaStream_t st) {
  using G = Bwd<DP, DKV, BIAS>;
  CUtensorMap m[4];
  for (int i = 0; i < 2; ++i) {
    if (int rc = map_of(&m[i], a, x[i], ROWS)) return rc;
    if (int rc = map_of(&m[2 + i], a, y[i], BN)) return rc;
  }
  Order order;
  const int64_t token = a.dim * 4;
  if (int rc = DKV ? order_of(&order, a, a.kv_heads, a.keys, a.queries * token * a.heads / a.kv_heads, false)
                   : order_of(&order, a, a.heads, a.queries, a.keys * token * a.kv_heads / a.heads, true))
    return rc;
  auto shared = [&](int stages) {
    return 1024 + 2 * (size_t)G::X + stages * 2 * (size_t)G::Y + 256 + (DKV ? G::STAGES * 2 * BN * 4 : 0) +
           bias_bytes(a, DKV ? G::GROUPS : 1 + 8 * G::GROUPS);
  };
  io.stages = shared(G::STAGES) <= SMEM_LIMIT ? G::STAGES : 2;
  const auto kernel = backward_kernel<DP, DKV, BIAS>;
  if (int rc = allow(kernel)) return rc;
  kernel<<<(unsigned)(order.row_tiles * order.pairs), G::THREADS, shared(io.stages), st>>>(m[0], m[1], m[2], m[3], a, order, io);
  return check_launch("attention_grad");
}

}  // namespace tiles

bool tiles_take_grad(const b200_attention& a) { return a.dtype == B200_BF16 && a.dim <= 128 && a.queries >= 16 && a.keys >= 1; }

// Forward, the row kernels split long keys over the SMs, which a tile's block walks alone (0.6 us for 64 keys). They take few queries
// over 2048 keys or more, while queries x heads x elements stay below 75000. Measured, kernels of rows (with the join) against tiles:
// 16 queries of 8 heads of 64 over 2048 keys 12.5 and 24.9 us, 64 queries 28.7 and 25.2, 128 queries 39 and 26; calls over 16384 keys,
// 16 queries 45 and 168 us, 64 queries 90 and 168, 128 queries 167 and 168, 256 queries 312 and 168; 32 + 8 heads of 128 over 16384
// keys, 16 queries 143 and 218, 32 queries 264 and 210; 16 queries of 4 x 32 heads of 128 over 4096 keys 158 and 55.
bool tiles_take(const b200_attention& a) {
  return tiles_take_grad(a) && (a.keys < 2048 || a.batch * a.heads * a.queries * a.dim >= 75000);
}

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
    if (int rc = map_of(&m[i], a, x[i], i == 0 ? ROWS : KEYS)) return rc;
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
  // a caller who does not say where dout is gets room for its copy
  const size_t d = g ? packed_bytes(a, operand(g->dout, a.queries, a.heads, g->dout_stride)) : up256((size_t)(a.batch * a.queries * a.heads * wide_of(a)) * 2);
  return part_bytes(a) + tiles_forward_workspace(a) + d;
}

int tiles_grad(const b200_attention& a, const b200_attention_grads& g, const float* lse2, const float* delta, int64_t padded, void* workspace,
               cudaStream_t st) {
  using namespace tiles;
  uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
  BwdIo io = {};
  io.lse = lse2, io.delta = delta, io.padded = (int)padded, io.part = reinterpret_cast<float*>(ws);
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
