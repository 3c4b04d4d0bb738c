// Persistent tcgen05 tile loop shared by the vocabulary loss and the Newton-Schulz
// products: C tile = A . B over K blocks of 64, 16-bit operands, fp32 accumulators in TMEM,
// and an epilogue object that gets each accumulator 32 columns at a time.
//
// Two things are wider than in the graph GEMM (gemm_tc.cu):
//  * an operand may come as two 16-bit planes, hi + lo of fp32 values (SPLIT; 16 or 22
//    bits). Each K block then brings all four planes and runs hi.lo + lo.hi + hi.hi, which is
//    the fp32 product up to lo.lo: a third of the tensor rate instead of the CUDA cores'. The
//    tensor cores cut (not round) each sum to fp32, all towards zero: sums of one sign lose
//    0.76 2^-23 of their value per 16 products, which over K = 50000 was 1e-4. So the
//    accumulator is drained every CHUNK K blocks and added up in registers with rounding (48
//    cuts; 16 in the 128-wide tiles, where hi.lo + lo.hi, 2^-8 to 2^-11 of the whole, have an
//    accumulator of their own);
//  * the tiles are walked in groups of M tiles (their A rows stay in L2 while B streams
//    past once per group), over the upper triangle of a symmetric result, or over splits of
//    the K axis, each with its own partial result.
//
// Roles as in gemm_tc.cu: warp 0 issues TMA loads, warp 1 owns TMEM and issues the MMAs,
// warps 4 to 11 (two per TMEM lane quarter) drain the double-buffered accumulator while the
// next MMAs run. PAIR: two CTAs of a cluster share a 256 x BN tile (cta_group::2), each
// loading its 128 rows of A and half of B: a single CTA's 128 x 128 tile reads and writes
// 64 KB of shared memory per K block, twice the time of its MMAs; a pair's 256 x 256 tile
// half its MMAs' time.
// What bounds split operands is the L2 (9 to 11 TB/s): a 256 x 128 tile reads 98 KB a K block
// for 786 clocks of MMAs and took 1480, a 256 x 256 tile 131 KB for 1572. Its drained
// accumulator is 128 registers a thread of the epilogue, so the two warpgroups there take over
// most of the first one's (setmaxnreg; ptxas honours it only in files compiled without -rdc).
// TEAM: where single tiles would leave most SMs idle, a cluster of 2 or 4 CTAs shares one
// tile's K axis; each then sends its partial sums of the columns that another one owns
// through shared memory (in place of the operands, all read by then) and finishes its own.
// The loop walks one product, or a chain of them whose tiles wait for each other (run_tiles).
// Every wait is bounded (tc_common.cuh); on expiry the device error flag is set and the
// block winds down.
#pragma once
#include <algorithm>

#include "tc_common.cuh"

namespace b200 {
namespace tile {

using namespace tc;

constexpr int BM = 128, BK = 64, EPI_WARPS = 8, EPI_FIRST = 4, THREADS = 32 * (EPI_FIRST + EPI_WARPS);
// registers a thread: at launch, then in the first warpgroup and in the epilogue's two; a sum
// beyond what the launch gave would wait forever (checked here and before the launch)
constexpr int REGS = 168, REGS_ISSUE = 56, REGS_EPI = 224, REGS_SUM = 128 * REGS_ISSUE + 256 * REGS_EPI;
static_assert(REGS_SUM <= THREADS * REGS, "setmaxnreg beyond the launch's registers");
constexpr uint32_t EPI_BUF = 4096;  // staging bytes per epilogue warp
constexpr uint32_t LEADER = 0xFEFFFFFFu;  // shared-memory address mask of a pair's CTA 0

template <int BN, bool PAIR, bool SPLIT>
struct Geo {
  static constexpr int PLANES = SPLIT ? 2 : 1;
  static constexpr bool LEND = SPLIT && BN == 256;   // the epilogue needs the first warpgroup's registers
  static constexpr bool APART = SPLIT && BN == 128;  // the small products' accumulators fit beside the others
  static_assert(!LEND || PAIR, "256-wide split tiles are for pairs");
  static constexpr int STAGES = SPLIT ? 3 : (BN == 256 && !PAIR ? 4 : 6);
  static constexpr int TM = PAIR ? 2 * BM : BM;
  static constexpr uint32_t A_BYTES = BM * BK * 2, B_BYTES = (PAIR ? BN / 2 : BN) * BK * 2;
  static constexpr uint32_t TMEM = (APART ? 4 : 2) * BN;  // columns
  static constexpr uint32_t STAGE = PLANES * (A_BYTES + B_BYTES);
  static constexpr size_t SMEM = (size_t)STAGES * STAGE + EPI_WARPS * EPI_BUF + 1024 + 256;
  static_assert(SMEM <= 232448, "operand ring and staging must fit 227 KB");
};

constexpr int CHUNK = 4;  // K blocks per accumulator of split operands
constexpr int WALK_GROUPED = 0, WALK_TRIANGLE = 1;

struct Loop {
  int nk;        // K blocks in all
  int nk_split;  // K blocks per split (= nk without splits)
  int chunk;     // K blocks that one accumulator takes before it is drained
  int a_mn, b_mn, bf16;
  int tiles_m, tiles_n, group_m, walk;
  int per_batch, total;  // tiles of one batch entry (splits included), of all
  int splits;
  int team;      // CTAs of a cluster that share a tile's K axis (TEAM)
};

struct Tile {
  int z, split, mt, nt;
  int product, step;  // which product of a chain, in which round
};

// the i-th tile of one product
__device__ __forceinline__ void place(Tile& r, int i, int walk, int tiles_m, int tiles_n, int group_m) {
  if (walk == WALK_TRIANGLE) {
    // square tiles on and above the diagonal: i = nt (nt + 1) / 2 + mt, mt <= nt
    int nt = (int)((sqrtf(8.f * (float)i + 1.f) - 1.f) * 0.5f);
    while ((nt + 1) * (nt + 2) / 2 <= i) ++nt;
    while (nt * (nt + 1) / 2 > i) --nt;
    r.nt = nt;
    r.mt = i - nt * (nt + 1) / 2;
    return;
  }
  const int per_group = group_m * tiles_n;
  const int first = i / per_group * group_m;
  const int size = min(group_m, tiles_m - first);
  const int j = i % per_group;
  r.mt = first + j % size;
  r.nt = j / size;
}

// What the tile loop walks: tile t of `total`, its K blocks, its operands, the result's size. This one: one product over all of its batch.
struct Product {
  static constexpr bool CHAIN = false;
  const CUtensorMap &a, &b;
  const Loop& lp;
  int64_t M, N;
  __device__ __forceinline__ int total() const { return lp.total; }
  __device__ __forceinline__ Tile at(int t) const {
    Tile r;
    r.product = r.step = 0;
    r.z = t / lp.per_batch;
    int i = t % lp.per_batch;
    const int per_split = lp.per_batch / lp.splits;
    r.split = i / per_split;
    i %= per_split;
    place(r, i, lp.walk, lp.tiles_m, lp.tiles_n, lp.group_m);
    return r;
  }
  __device__ __forceinline__ Tile kind(int t) const {  // what the MMAs need of it
    Tile r = {};
    r.split = t % lp.per_batch / (lp.per_batch / lp.splits);
    return r;
  }
  __device__ __forceinline__ int blocks(const Tile&) const { return lp.nk; }
  __device__ __forceinline__ int blocks_each(const Tile&) const { return lp.nk_split; }
  __device__ __forceinline__ int chunk(const Tile&) const { return lp.chunk; }
  struct Side {  // an operand: its map at a K block, whether it has M (N) adjacent there
    const CUtensorMap* m;
    int adjacent;
    __device__ __forceinline__ const CUtensorMap* map(int) const { return m; }
    __device__ __forceinline__ int mn(int) const { return adjacent; }
  };
  __device__ __forceinline__ Side side_a(const Tile&) const { return {&a, lp.a_mn}; }
  __device__ __forceinline__ Side side_b(const Tile&) const { return {&b, lp.b_mn}; }
  __device__ __forceinline__ int64_t rows(const Tile&) const { return M; }
  __device__ __forceinline__ int64_t cols(const Tile&) const { return N; }
  __device__ __forceinline__ void prefetch() const {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&a)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&b)) : "memory");
  }
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release;\n barrier.cluster.wait.acquire;" ::: "memory");
}
template <bool PAIR>
__device__ __forceinline__ void load4(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2, int c3) {
  if constexpr (PAIR) {
    // the completed bytes count on the leader's barrier
    asm volatile(
        "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, "
        "%5}], [%6];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar) & LEADER)
        : "memory");
  } else {
    tma_load_4d(dst, map, bar, c0, c1, c2, c3);
  }
}
template <bool PAIR>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  if constexpr (PAIR) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a),
        "l"(b), "r"(idesc), "r"(acc));
  } else {
    mma_bf16(d, a, b, idesc, acc);  // kind::f16: fp16 or bf16 operands by idesc
  }
}
template <bool PAIR>
__device__ __forceinline__ void commit(uint64_t* bar) {
  if constexpr (PAIR) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                     smem_u32(bar)),
                 "h"((uint16_t)3)
                 : "memory");
  } else {
    mma_commit(bar);
  }
}

// A chunk staged by stage_chunk<ESZ> to rows of an output whose rows start anywhere: 16 bytes a
// lane where every row allows it, else an element a lane. The loops stay small: an epilogue's
// chunks are unrolled, and code beyond the instruction caches cost the first tile of a launch
// three times the others.
template <int ESZ>
__device__ __forceinline__ void put_chunk(uint32_t buf, int lane, uint8_t* base, int64_t ld, int rows, int cols) {
  constexpr int PIECES = 2 * ESZ;
  auto word_at = [&](int r, int byte) {
    const uint32_t sw = ESZ == 4 ? (uint32_t)(r & 7) : (uint32_t)((r >> 1) & 3);
    return buf + (uint32_t)r * (32u * ESZ) + ((((uint32_t)byte >> 4) ^ sw) << 4) + ((uint32_t)byte & 15u);
  };
  if (cols == 32 && ((reinterpret_cast<uintptr_t>(base) | (uint64_t)ld * ESZ) & 15) == 0) {
    const int j = lane % PIECES;
#pragma unroll 2
    for (int r = lane / PIECES; r < rows; r += 32 / PIECES)
      *reinterpret_cast<uint4*>(base + (int64_t)r * ld * ESZ + 16 * j) = ld_shared_v4(word_at(r, 16 * j));
    return;
  }
#pragma unroll 1
  for (int r = 0; r < rows; ++r)
    if (lane < cols) {
      uint8_t* d = base + ((int64_t)r * ld + lane) * ESZ;
      if constexpr (ESZ == 4) {
        uint32_t v;
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(word_at(r, 4 * lane)) : "memory");
        *reinterpret_cast<uint32_t*>(d) = v;
      } else {
        uint16_t v;
        asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"(word_at(r, 2 * lane)) : "memory");
        *reinterpret_cast<uint16_t*>(d) = v;
      }
    }
}

// 32 rows of 32 ESZ bytes (16-byte aligned, `ld` bytes apart) as the lanes can load them together:
// whole rows per instruction, so that a warp's load touches 8 (ESZ 2) or 4 lines, not 32, whose
// lookups alone took as long as the tile's MMAs. A row per lane comes out of rows_in.
template <int ESZ>
__device__ __forceinline__ void rows_load(const uint8_t* base, int64_t ld, int rows, int pieces, int lane, float (&w)[32], int first) {
  constexpr int PIECES = 2 * ESZ, PER = 32 / PIECES;
  const int j = lane % PIECES;
  base += (int64_t)(lane / PIECES) * ld + 16 * j;
#pragma unroll
  for (int i = 0; i < PIECES; ++i)
    if (i * PER + lane / PIECES < rows && j < pieces) {
      const float4 u = *reinterpret_cast<const float4*>(base + (int64_t)(i * PER) * ld);
      w[first + 4 * i] = u.x, w[first + 4 * i + 1] = u.y, w[first + 4 * i + 2] = u.z, w[first + 4 * i + 3] = u.w;
    }
}
template <int ESZ>
__device__ __forceinline__ void rows_in(uint32_t buf, int lane, float (&w)[32], int first) {
  constexpr int PIECES = 2 * ESZ, PER = 32 / PIECES;
  auto at = [&](int r, int j) {
    const int sw = ESZ == 4 ? r & 7 : ((r >> 1) ^ (r >> 3)) & 3;
    return buf + (uint32_t)r * (32u * ESZ) + ((uint32_t)(j ^ sw) << 4);
  };
  __syncwarp();
#pragma unroll
  for (int i = 0; i < PIECES; ++i)
    st_shared_v4(at(i * PER + lane / PIECES, lane % PIECES), __float_as_uint(w[first + 4 * i]), __float_as_uint(w[first + 4 * i + 1]),
                 __float_as_uint(w[first + 4 * i + 2]), __float_as_uint(w[first + 4 * i + 3]));
  __syncwarp();
#pragma unroll
  for (int j = 0; j < PIECES; ++j) {
    const uint4 u = ld_shared_v4(at(lane, j));
    w[first + 4 * j] = __uint_as_float(u.x), w[first + 4 * j + 1] = __uint_as_float(u.y);
    w[first + 4 * j + 2] = __uint_as_float(u.z), w[first + 4 * j + 3] = __uint_as_float(u.w);
  }
}

// What an epilogue warp knows about its chunk: `row` is this lane's output row, `row0` the
// warp's first one, `buf` its staging buffer
struct Spot {
  int64_t row, row0, col0;  // col0: first of this warp's columns
  int z, split, mt, nt, half, lane;
  uint32_t buf;
};

// Epi: begin(spot) once per tile; where INIT, fetch(spot, column, values[32]) loads (into zeros)
// what ready(spot, column, values[32]) turns into what the product is added to (result =
// values + scale * product); chunk(spot, column, values[32]) for each 32 columns
// inside the result, end(spot); adds(): whether there is something to add; finish(lane) at the
// end of the kernel. A chain's epilogue has enter(tile, spot) in begin's place.
// Work: Product, whose tiles are dealt out in turn, or a chain of them (CHAIN) whose tiles wait
// for earlier ones and are taken by tickets, in order, by whichever pair comes next. Two warps
// see to that, since a look at a counter in global memory takes 1200 clocks under load and the
// fence behind a tile's stores 4000 (a tile 23000). Warp 2 (scout) takes a ticket once the loader
// has begun the tile before (the leader's, for both CTAs), waits for ready(tile) and shows it to
// the other warps through a ring in shared memory; warp 3 (herald) waits for the epilogue's
// warps and publishes the tile by done(tile).
template <int BN, bool PAIR, bool SPLIT, bool TEAM, typename Work, typename Epi>
__device__ __forceinline__ void run_tiles(const Work& work, int team, bool bf16, Epi& epi) {
  using G = Geo<BN, PAIR, SPLIT>;
  constexpr int STG = G::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* s_epi = smem + STG * G::STAGE;  // a stage: A's planes, then B's
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(s_epi + EPI_WARPS * EPI_BUF);
  uint64_t* empty_bar = full_bar + STG;
  uint64_t* acc_full = empty_bar + STG;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* fin_bar = acc_empty + 2;  // CHAIN: the epilogue's warps have stored a tile
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(fin_bar + 1);
  // CHAIN, counted in tiles of this CTA: shown to its warps (-1: given up), handed over by the
  // leader's scout, begun by the loader, taken over by the herald and the peer's; tiles by number % 4
  int *seen = reinterpret_cast<int*>(tmem_slot + 1), *given = seen + 1, *begun = seen + 2, *passed = seen + 3, *peer_passed = seen + 4;
  int* ring = seen + 5;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_rank() : 0u;
  const int member = TEAM ? (int)cluster_rank() : 0;
  const int per_unit = PAIR ? 2 : (TEAM ? team : 1);
  const int total = work.total();
  const int unit = (int)blockIdx.x / per_unit, units = (int)gridDim.x / per_unit;

  if (threadIdx.x == 0) {
    work.prefetch();
    for (int s = 0; s < STG; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], (PAIR ? 2 : 1) * EPI_WARPS);
    }
    if constexpr (Work::CHAIN) {
      mbar_init(fin_bar, EPI_WARPS);
      *seen = *given = *begun = *passed = *peer_passed = 0;
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(G::TMEM));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(G::TMEM));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
  }
  tc_fence_before();
  if constexpr (PAIR) cluster_sync_all();
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // The next kernel of the stream may start its own set-up now; this one has waited for the
  // kernels before it from here on (it reads and writes no global memory earlier).
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");

  // a counter in shared memory at `least` or more; false if its writer gave up or takes too long
  auto counted = [&](const int* count, int least) {
    unsigned long long t0 = 0;
    while (true) {
      int v;
      asm volatile("ld.acquire.cluster.shared::cta.s32 %0, [%1];" : "=r"(v) : "r"(smem_u32(count)) : "memory");
      if (v >= least) return true;
      if (v < 0) return false;
      if (t0 == 0) t0 = globaltimer();
      if (globaltimer() - t0 > WAIT_LIMIT_NS) {
        raise_device_error(B200_ERR_TIMEOUT);
        return false;
      }
    }
  };
  auto count = [&](int* count, int value) {
    asm volatile("st.release.cta.shared::cta.s32 [%0], %1;" ::"r"(smem_u32(count)), "r"(value) : "memory");
  };
  auto at_peer = [&](const int* p) {
    uint32_t far;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(far) : "r"(smem_u32(p)), "r"(rank ^ 1u));
    return far;
  };
  // the n-th tile of this CTA; `total`: no more
  auto nth = [&](int n) {
    if constexpr (Work::CHAIN) return counted(seen, n + 1) ? *(volatile int*)&ring[n & 3] : total;
    else return unit + n * units;
  };

  if (warp < EPI_FIRST) {
    if constexpr (G::LEND) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_ISSUE));
    if (warp == 0 && lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      for (int n = 0, t; ok && (t = nth(n)) < total; ++n) {
        const Tile at = work.at(t);
        if constexpr (Work::CHAIN) count(begun, n + 1);
        const int each = work.blocks_each(at);
        const auto a = work.side_a(at);
        const auto b = work.side_b(at);
        const int m0 = at.mt * G::TM + (int)rank * BM;
        const int n0 = at.nt * BN + (PAIR ? (int)rank * (BN / 2) : 0);
        const int kb0 = (TEAM ? member : at.split) * each, kb1 = min(work.blocks(at), kb0 + each);
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const int s = it % STG;
          if (!mbar_wait(&empty_bar[s], ((it / STG) & 1) ^ 1)) {
            ok = false;
            break;
          }
          if (rank == 0) mbar_expect_tx(&full_bar[s], (PAIR ? 2u : 1u) * G::STAGE);
          const int k0 = kb * BK;
          const CUtensorMap *map_a = a.map(kb), *map_b = b.map(kb);
          const int a_mn = a.mn(kb), b_mn = b.mn(kb);
#pragma unroll
          for (int p = 0; p < G::PLANES; ++p) {
            uint8_t* a_dst = smem + s * G::STAGE + p * G::A_BYTES;
            uint8_t* b_dst = smem + s * G::STAGE + G::PLANES * G::A_BYTES + p * G::B_BYTES;
            if (!a_mn) {
              load4<PAIR>(a_dst, map_a, &full_bar[s], k0, m0, p, at.z);
            } else {
              load4<PAIR>(a_dst, map_a, &full_bar[s], m0, k0, p, at.z);
              load4<PAIR>(a_dst + 8192, map_a, &full_bar[s], m0 + 64, k0, p, at.z);
            }
            if (!b_mn) {
              load4<PAIR>(b_dst, map_b, &full_bar[s], k0, n0, p, at.z);
            } else {
#pragma unroll
              for (int j = 0; j < (PAIR ? BN / 2 : BN) / 64; ++j)
                load4<PAIR>(b_dst + j * 8192, map_b, &full_bar[s], n0 + 64 * j, k0, p, at.z);
            }
          }
        }
      }
      if constexpr (PAIR) {
        // wait until the MMAs released every stage this CTA filled, so that no commit of the
        // leader arrives on this CTA's barriers after it has exited
        for (int i = 0; i < STG && ok; ++i, ++it) ok = mbar_wait(&empty_bar[it % STG], ((it / STG) & 1) ^ 1, 64);
      }
    }
    if (warp == 1 && lane == 0 && rank == 0) {
      const uint32_t fmt = bf16 ? (1u << 7) | (1u << 10) : 0u;
      uint32_t it = 0, local = 0;
      bool ok = true;
      uint32_t tiles = 0;
      for (int t; ok && (t = nth((int)tiles)) < total; ++tiles) {
        const Tile at = work.kind(t);
        const int each = work.blocks_each(at), chunk = work.chunk(at);
        const auto a = work.side_a(at);
        const auto sb = work.side_b(at);
        const int kb0 = (TEAM ? member : at.split) * each, kb1 = min(work.blocks(at), kb0 + each);
        for (int c0 = kb0; c0 < kb1 && ok; c0 += chunk, ++local) {
          const int b = local & 1;
          if (!mbar_wait(&acc_empty[b], ((local >> 1) & 1) ^ 1)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t d = tmem + (uint32_t)(b * BN);
          const int c1 = min(kb1, c0 + chunk);
          for (int kb = c0; kb < c1; ++kb, ++it) {
            const int s = it % STG;
            if (!mbar_wait(&full_bar[s], (it / STG) & 1)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const int a_mn = a.mn(kb), b_mn = sb.mn(kb);
            const uint32_t idesc = (1u << 4) | fmt | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) | ((uint32_t)(BN >> 3) << 17) |
                                   ((uint32_t)(G::TM >> 4) << 24);
            const uint32_t a0 = smem_u32(smem + s * G::STAGE), b0 = a0 + G::PLANES * G::A_BYTES;
#pragma unroll
            for (int seg = SPLIT ? 0 : 2; seg < 3; ++seg) {
              // hi.lo and lo.hi into the tile's accumulator of small products (APART), hi.hi into the chunk's
              const uint32_t as = a0 + (SPLIT && seg == 1 ? G::A_BYTES : 0u), bs = b0 + (SPLIT && seg == 0 ? G::B_BYTES : 0u);
              const uint32_t to = G::APART && seg < 2 ? tmem + (uint32_t)((2 + (tiles & 1)) * BN) : d;
              const bool fresh = G::APART ? (seg == 0 ? kb == kb0 : (seg == 2 && kb == c0)) : (seg == (SPLIT ? 0 : 2) && kb == c0);
#pragma unroll
              for (int k = 0; k < BK / 16; ++k) {
                const uint64_t ad = a_mn ? smem_desc(as + k * 2048, 8192, 1024) : smem_desc(as + k * 32, 16, 1024);
                const uint64_t bd = b_mn ? smem_desc(bs + k * 2048, 8192, 1024) : smem_desc(bs + k * 32, 16, 1024);
                mma<PAIR>(to, ad, bd, idesc, (!fresh || k > 0) ? 1u : 0u);
              }
            }
            commit<PAIR>(&empty_bar[s]);
          }
          if (ok) commit<PAIR>(&acc_full[b]);
        }
      }
    }
    if constexpr (Work::CHAIN) {
      if (warp == 2 && lane == 0) {
        bool shown = true;
        for (int n = 0, t = 0; shown && t < total; ++n) {
          shown = false;
          if (rank == 0) {
            if (!counted(begun, n) || !counted(passed, n - 3) || !counted(peer_passed, n - 3)) break;
            t = work.ticket();
            ring[n & 3] = t;
            asm volatile("st.relaxed.cluster.shared::cluster.s32 [%0], %1;" ::"r"(at_peer(&ring[n & 3])), "r"(t) : "memory");
            asm volatile("st.release.cluster.shared::cluster.s32 [%0], %1;" ::"r"(at_peer(given)), "r"(n + 1) : "memory");
          } else {
            if (!counted(given, n + 1)) break;
            t = *(volatile int*)&ring[n & 3];
          }
          shown = t >= total || work.ready(work.at(t));
          if (shown) count(seen, n + 1);
        }
        if (!shown) count(seen, -1);
      }
      if (warp == 3 && lane == 0) {
        for (int n = 0, t; (t = nth(n)) < total; ++n) {
          if (!mbar_wait(fin_bar, n & 1, 64)) break;
          count(passed, n + 1);
          if (rank != 0) asm volatile("st.release.cluster.shared::cluster.s32 [%0], %1;" ::"r"(at_peer(peer_passed)), "r"(n + 1) : "memory");
          work.done(work.at(t));
        }
      }
    }
    if constexpr (TEAM) {  // the epilogue's two meetings
      cluster_sync_all();
      cluster_sync_all();
    }
  } else {
    if constexpr (G::LEND) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_EPI));
    Spot sp;
    const int q = warp & 3;
    sp.half = (warp - EPI_FIRST) >> 2;
    sp.lane = lane;
    sp.buf = smem_u32(s_epi) + (uint32_t)(warp - EPI_FIRST) * EPI_BUF;
    constexpr int CH = BN / 64;  // chunks of 32 columns per warp
    static_assert(!TEAM || CH == 2, "teams share 128-wide tiles");
    uint32_t local = 0, tiles = 0;
    bool ok = true;
    // the accumulator may be overwritten once every epilogue warp has read it
    auto release = [&](int b) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (PAIR)
          asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(smem_u32(&acc_empty[b]) & LEADER) : "memory");
        else mbar_arrive(&acc_empty[b]);
      }
    };
    for (int n = 0, t; ok && (t = nth(n)) < total; ++n) {
      const Tile at = work.at(t);
      const int64_t M = work.rows(at), N = work.cols(at);
      sp.z = at.z;
      sp.split = at.split;
      sp.mt = at.mt;
      sp.nt = at.nt;
      sp.row0 = (int64_t)at.mt * G::TM + (int64_t)rank * BM + q * 32;
      sp.row = sp.row0 + lane;
      const int64_t col0 = sp.col0 = (int64_t)at.nt * BN + sp.half * (BN / 2);
      const uint32_t base = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(sp.half * (BN / 2));
      if constexpr (Work::CHAIN) {
        epi.enter(at, sp);
      } else {
        epi.begin(sp);
      }
      // the member that finishes chunk c of this warp: of two, each takes a chunk of every warp
      auto owner = [&](int c) { return !TEAM ? 0 : (team == 2 ? c : sp.half * CH + c); };
      if constexpr (SPLIT || TEAM) {
        // What the product is added to comes first where registers last for it (EARLY); 256-wide
        // tiles, whose MMAs wait as long as the accumulator is not drained, take it a
        // chunk ahead while the chunks are stored.
        constexpr bool EARLY = CH == 2;
        float acc[CH][32], more[Epi::INIT && !EARLY ? 32 : 1];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
#pragma unroll
          for (int i = 0; i < 32; ++i) acc[c][i] = 0.f;
          // every chunk's loads are issued before the first is waited for
          if constexpr (Epi::INIT && EARLY)
            if (owner(c) == member && col0 + c * 32 < N && sp.row0 < M) epi.fetch(sp, col0 + c * 32, acc[c]);
        }
        if constexpr (Epi::INIT && EARLY) {
#pragma unroll
          for (int c = 0; c < CH; ++c)
            if (owner(c) == member && col0 + c * 32 < N && sp.row0 < M) epi.ready(sp, col0 + c * 32, acc[c]);
        }
        auto add = [&](uint32_t at_col, float (&to)[32]) {
          uint32_t cur[32];
          tmem_ld32_issue(base + at_col, cur);
          tmem_wait(cur);
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            if constexpr (Epi::INIT && EARLY) to[i] = fmaf(epi.scale, __uint_as_float(cur[i]), to[i]);
            else to[i] += __uint_as_float(cur[i]);
          }
        };
        auto ahead = [&](int c) {
          if constexpr (Epi::INIT && !EARLY) {
            if (!epi.adds()) return;
#pragma unroll
            for (int i = 0; i < 32; ++i) more[i] = 0.f;
            if (col0 + c * 32 < N && sp.row0 < M) epi.fetch(sp, col0 + c * 32, more);
          }
        };
        const int each = work.blocks_each(at), chunk = work.chunk(at);
        const int kb0 = (TEAM ? member : at.split) * each, kb1 = min(work.blocks(at), kb0 + each);
        for (int c0 = kb0; c0 < kb1; c0 += chunk, ++local) {
          const int b = local & 1;
          if constexpr (Epi::INIT && !EARLY)
            if (c0 + chunk >= kb1) ahead(0);
          if (!mbar_wait(&acc_full[b], (local >> 1) & 1)) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < CH; ++c) {
            add((uint32_t)(b * BN + c * 32), acc[c]);
            if (G::APART && c0 + chunk >= kb1) add((uint32_t)((2 + (tiles & 1)) * BN + c * 32), acc[c]);
          }
          release(b);
        }
        ++tiles;
        if constexpr (TEAM) {
          // every member's MMAs are done: the operand ring takes the partial sums, 16 KB (128 rows
          // of 32, 16-byte pieces swizzled by row) per chunk and sender
          cluster_sync_all();
          const int share = 2 * CH / team, mine = team == 2 ? sp.half : 0;
          const uint32_t line = smem_u32(smem) + (uint32_t)(q * 32 + lane) * 128u;
#pragma unroll
          for (int c = 0; c < CH; ++c) {
            const int to = owner(c);
            if (to == member) continue;
            const int slot = (member < to ? member : member - 1) * share + mine;
            uint32_t far;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(far) : "r"(line + (uint32_t)slot * 16384u), "r"(to));
#pragma unroll
            for (int p = 0; p < 8; ++p)
              asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(far + (uint32_t)((p ^ (lane & 7)) << 4)),
                           "f"(acc[c][4 * p]), "f"(acc[c][4 * p + 1]), "f"(acc[c][4 * p + 2]), "f"(acc[c][4 * p + 3])
                           : "memory");
          }
          cluster_sync_all();
#pragma unroll
          for (int c = 0; c < CH; ++c) {
            if (owner(c) != member) continue;
            for (int from = 0; from < team - 1; ++from) {
              const uint32_t at_line = line + (uint32_t)(from * share + mine) * 16384u;
#pragma unroll
              for (int p = 0; p < 8; ++p) {
                const uint4 u = ld_shared_v4(at_line + (uint32_t)((p ^ (lane & 7)) << 4));
                acc[c][4 * p] += __uint_as_float(u.x);
                acc[c][4 * p + 1] += __uint_as_float(u.y);
                acc[c][4 * p + 2] += __uint_as_float(u.z);
                acc[c][4 * p + 3] += __uint_as_float(u.w);
              }
            }
          }
        }
        if (!ok) break;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          if (owner(c) == member && col0 + c * 32 < N && sp.row0 < M) {  // warp-uniform
            if constexpr (Epi::INIT && !EARLY) {
              if (epi.adds()) {
                epi.ready(sp, col0 + c * 32, more);
#pragma unroll
                for (int i = 0; i < 32; ++i) acc[c][i] = fmaf(epi.scale, acc[c][i], more[i]);
                if (c + 1 < CH) ahead(c + 1);
              } else {
#pragma unroll
                for (int i = 0; i < 32; ++i) acc[c][i] *= epi.scale;
              }
            }
            epi.chunk(sp, col0 + c * 32, acc[c]);
          }
          asm volatile("" ::: "memory");  // one chunk at a time: the others wait in registers
        }
      } else {
        const int b = local & 1;
        float more[Epi::INIT ? 32 : 1];
        auto ahead = [&](int64_t col) {
          if constexpr (Epi::INIT) {
#pragma unroll
            for (int i = 0; i < 32; ++i) more[i] = 0.f;
            if (col < N && sp.row0 < M) epi.fetch(sp, col, more);
          }
        };
        ahead(col0);
        if (!mbar_wait(&acc_full[b], (local >> 1) & 1)) break;
        tc_fence_after();
        uint32_t cur[32];
        tmem_ld32_issue(base + (uint32_t)(b * BN), cur);
#pragma unroll 1
        for (int c = 0; c < CH; ++c) {
          const int64_t col = col0 + c * 32;
          tmem_wait(cur);
          if (!(col < N && sp.row0 < M)) break;  // warp-uniform
          float v[32];
          if constexpr (Epi::INIT) epi.ready(sp, col, more);
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            if constexpr (Epi::INIT) v[i] = fmaf(epi.scale, __uint_as_float(cur[i]), more[i]);
            else v[i] = __uint_as_float(cur[i]);
          }
          // the next chunk's loads are under way while this one is worked on
          if (c + 1 < CH) {
            tmem_ld32_issue(base + (uint32_t)(b * BN + (c + 1) * 32), cur);
            ahead(col + 32);
          }
          epi.chunk(sp, col, v);
        }
        tmem_wait(cur);
        release(b);
        ++local;
      }
      epi.end(sp);
      if constexpr (Work::CHAIN) {
        __syncwarp();
        // (an arrival two tiles ahead of warp 3 would turn the barrier's phase back)
        if (lane == 0 && counted(passed, n)) mbar_arrive(fin_bar);
      }
    }
    epi.finish(lane);
  }
  tc_fence_before();
  if constexpr (PAIR) cluster_sync_all();
  else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(G::TMEM));
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(G::TMEM));
  }
}

template <int BN, bool PAIR, bool SPLIT, bool TEAM, typename Epi>
__global__ void __launch_bounds__(THREADS, 1) tile_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                                                          const __grid_constant__ Loop lp, const int64_t M, const int64_t N,
                                                          const __grid_constant__ typename Epi::Args args) {
  Epi epi(args);
  run_tiles<BN, PAIR, SPLIT, TEAM>(Product{map_a, map_b, lp, M, N}, lp.team, lp.bf16 != 0, epi);
}

// ---------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------

// One 16-bit operand of `major` rows and K: element (i, k) of plane p, batch z at
//   base + 2 (z batch_stride + p plane_stride + (mn ? k ld + i : i ld + k)).
struct Operand {
  const void* base = nullptr;
  int64_t ld = 0, plane_stride = 0, batch_stride = 0;
  int mn = 0;
};

// The map of an operand of `major` rows and K, boxes of 64 elements of K by `box` rows (64 x 64
// where the rows are adjacent)
static int operand_map(CUtensorMap* m, const Operand& o, int64_t major, int64_t K, int planes, int64_t batch, int box) {
  const uint64_t span = (uint64_t)o.ld * 2 * (uint64_t)(o.mn ? K : major);
  const uint64_t ps = planes > 1 ? (uint64_t)o.plane_stride * 2 : span, bs = batch > 1 ? (uint64_t)o.batch_stride * 2 : ps * planes;
  return o.mn ? make_map(m, o.base, major, K, planes, batch, o.ld * 2, ps, bs, 64, 64)
              : make_map(m, o.base, K, major, planes, batch, o.ld * 2, ps, bs, 64, box);
}

// Clusters (of `size` CTAs; 1: none) of a kernel of geometry G that can be resident at once, per
// kernel, size and device; 0 where it was compiled to fewer registers than its warpgroups trade
template <typename G, auto KERNEL>
static int resident(int size) {
  static int units[64][5] = {{0}};
  int dev = 0;
  cudaGetDevice(&dev);
  const bool known = dev >= 0 && dev < 64;
  if (known && units[dev][size]) return units[dev][size];
  auto* fn = KERNEL;
  if constexpr (G::LEND) {
    cudaFuncAttributes at;
    if (cudaFuncGetAttributes(&at, fn) != cudaSuccess || at.numRegs * THREADS < REGS_SUM) return 0;
  }
  cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)G::SMEM);
  int n = num_sms() / size;
  if (size > 1) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(size * n), 1, 1);
    cfg.blockDim = dim3(THREADS, 1, 1);
    cfg.dynamicSmemBytes = G::SMEM;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)size;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int k = 0;
    if (cudaOccupancyMaxActiveClusters(&k, fn, &cfg) == cudaSuccess && k > 0) n = std::min(n, k);
    else cudaGetLastError();
  }
  if (known) units[dev][size] = n;
  return n;
}

// C [batch][M, N] = A . B with operands of one 16-bit plane, or of two (SPLIT). Fills in the
// loop's tile counts and launches as many CTAs (or pairs) as are resident, each walking its
// share of the tiles.
template <int BN, bool PAIR, bool SPLIT, bool TEAM, typename Epi>
static int launch_as(const Operand& A, const Operand& B, int64_t M, int64_t N, int64_t K, int64_t batch, Loop lp,
                     const typename Epi::Args& args, cudaStream_t s, const char* what) {
  using G = Geo<BN, PAIR, SPLIT>;
  constexpr auto kernel = tile_kernel<BN, PAIR, SPLIT, TEAM, Epi>;
  constexpr int planes = SPLIT ? 2 : 1;
  lp.a_mn = A.mn;
  lp.b_mn = B.mn;
  lp.nk = (int)ceil_div(K, BK);
  if (lp.splits < 1) lp.splits = 1;
  lp.nk_split = (int)ceil_div(lp.nk, lp.splits);
  lp.splits = (int)ceil_div(lp.nk, lp.nk_split);  // no split without K blocks
  lp.chunk = SPLIT ? CHUNK : lp.nk_split;
  lp.tiles_m = (int)ceil_div(M, G::TM);
  lp.tiles_n = (int)ceil_div(N, BN);
  const int64_t per = lp.walk == WALK_TRIANGLE ? (int64_t)lp.tiles_n * (lp.tiles_n + 1) / 2 : (int64_t)lp.tiles_m * lp.tiles_n;
  B200_REQUIRE(per * lp.splits * batch < (1ll << 30), "%s: too many tiles", what);
  lp.per_batch = (int)(per * lp.splits);
  lp.total = (int)(per * lp.splits * batch);
  int size = PAIR ? 2 : 1, units;
  if constexpr (TEAM) {
    // one tile per team; 4 or 2 members where that many teams fit and each has 2 K blocks or more
    size = 4;
    while (size > 1 && (lp.nk < 2 * size || resident<G, kernel>(size) < lp.total)) size /= 2;
    if (size == 1) return -1;
    lp.team = size;
    lp.nk_split = (int)ceil_div(lp.nk, size);
    if (!SPLIT) lp.chunk = lp.nk_split;
    units = lp.total;
  } else {
    units = std::min(resident<G, kernel>(size), lp.total);
  }
  if (units < 1) {
    set_error("%s: the kernel cannot be resident (registers)", what);
    return B200_ERR_CUDA;
  }
  CUtensorMap ma, mb;
  int rc = operand_map(&ma, A, M, K, planes, batch, BM);
  if (!rc) rc = operand_map(&mb, B, N, K, planes, batch, PAIR ? BN / 2 : BN);
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(size * units), 1, 1);
  cfg.blockDim = dim3(THREADS, 1, 1);
  cfg.dynamicSmemBytes = G::SMEM;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)size;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = size > 1 ? 2 : 1;
  cudaLaunchKernelEx(&cfg, kernel, ma, mb, lp, M, N, args);
  return check_launch(what);
}

// 256 x 256 tiles on pairs; else 128 x 128 of split operands, and of plain ones 128 x 256 for
// more than 128 columns or 128 x 128, as far as the epilogue has them; 128 x 128 tiles on teams
// where it has those and they fit.
template <typename Epi>
static int launch(const Operand& A, const Operand& B, int64_t M, int64_t N, int64_t K, int64_t batch, int planes, bool pair, const Loop& lp,
                  const typename Epi::Args& args, cudaStream_t s, const char* what) {
  if constexpr (Epi::TEAMS) {
    if (!pair) {
      const int rc = planes > 1 ? launch_as<128, false, true, true, Epi>(A, B, M, N, K, batch, lp, args, s, what)
                                : launch_as<128, false, false, true, Epi>(A, B, M, N, K, batch, lp, args, s, what);
      if (rc >= 0) return rc;
    }
  }
  if (planes > 1)
    return pair ? launch_as<256, true, true, false, Epi>(A, B, M, N, K, batch, lp, args, s, what)
                : launch_as<128, false, true, false, Epi>(A, B, M, N, K, batch, lp, args, s, what);
  if (pair) return launch_as<256, true, false, false, Epi>(A, B, M, N, K, batch, lp, args, s, what);
  if constexpr (Epi::SINGLE_WIDE) {
    if (!Epi::SINGLE_NARROW || N > 128) return launch_as<256, false, false, false, Epi>(A, B, M, N, K, batch, lp, args, s, what);
  }
  if constexpr (Epi::SINGLE_NARROW) return launch_as<128, false, false, false, Epi>(A, B, M, N, K, batch, lp, args, s, what);
  return B200_ERR_UNSUPPORTED;
}

}  // namespace tile
}  // namespace b200
