// Persistent tcgen05 tile loop shared by the vocabulary loss and the Newton-Schulz
// products: C tile = A . B over K blocks of 64, 16-bit operands, fp32 accumulators in TMEM,
// and an epilogue object that gets each accumulator 32 columns at a time.
//
// Two things are wider than in the graph GEMM (gemm_tc.cu):
//  * an operand may come as two 16-bit planes, hi + lo of fp32 values (16 or 22 bits). The
//    loop then runs three segments into the same accumulator, hi.lo + lo.hi + hi.hi, which
//    is the fp32 product up to lo.lo: a third of the tensor rate instead of the CUDA cores'.
//    The tensor cores cut (not round) each sum to fp32: 2^-24 of it per 16 products, all
//    towards zero, which over K = 50000 is 1e-4. So the accumulator is drained every 512 of
//    K and added up in registers with rounding (SPLIT), the small segments first: at most
//    32 cuts at full size;
//  * the tiles are walked in groups of M tiles (their A rows stay in L2 while B streams
//    past once per group), over the upper triangle of a symmetric result, or over splits of
//    the K axis, each with its own partial result.
//
// Roles as in gemm_tc.cu: warp 0 issues TMA loads, warp 1 owns TMEM and issues the MMAs,
// eight epilogue warps (two per TMEM lane quarter) drain the double-buffered accumulator
// while the next tile's MMAs run. PAIR: two CTAs of a cluster share a 256 x BN tile
// (cta_group::2), each loading its 128 rows of A and half of B.
// Every wait is bounded (tc_common.cuh); on expiry the device error flag is set and the
// block winds down.
#pragma once
#include <algorithm>

#include "tc_common.cuh"

namespace b200 {
namespace tile {

using namespace tc;

constexpr int BM = 128, BK = 64, EPI_WARPS = 8, THREADS = 64 + 32 * EPI_WARPS;
constexpr uint32_t EPI_BUF = 4096;  // staging bytes per epilogue warp
constexpr uint32_t LEADER = 0xFEFFFFFFu;  // shared-memory address mask of a pair's CTA 0

template <int BN, bool PAIR>
struct Geo {
  static constexpr int STAGES = BN == 256 ? (PAIR ? 6 : 4) : 6;
  static constexpr int TM = PAIR ? 2 * BM : BM;
  static constexpr uint32_t A_BYTES = BM * BK * 2, B_BYTES = (PAIR ? BN / 2 : BN) * BK * 2;
  static constexpr size_t SMEM = (size_t)STAGES * (A_BYTES + B_BYTES) + EPI_WARPS * EPI_BUF + 1024 + 256;
  static_assert(SMEM <= 232448, "operand ring and staging must fit 227 KB");
};

constexpr int CHUNK = 8;  // K blocks per accumulator of split operands
constexpr int WALK_GROUPED = 0, WALK_TRIANGLE = 1;

struct Loop {
  int nk;        // K blocks in all
  int nk_split;  // K blocks per split (= nk without splits)
  int nseg;      // 1, or 3 for hi.lo + lo.hi + hi.hi
  int chunk;     // K blocks that one accumulator takes before it is drained
  int a_mn, b_mn, bf16;
  int tiles_m, tiles_n, group_m, walk;
  int per_batch, total;  // tiles of one batch entry (splits included), of all
  int splits;
};

struct Tile {
  int z, split, mt, nt;
};

__device__ __forceinline__ Tile tile_at(const Loop& lp, int t) {
  Tile r;
  r.z = t / lp.per_batch;
  int i = t % lp.per_batch;
  const int per_split = lp.per_batch / lp.splits;
  r.split = i / per_split;
  i %= per_split;
  if (lp.walk == WALK_TRIANGLE) {
    // i = nt (nt + 1) / 2 + mt, mt <= nt
    int nt = (int)((sqrtf(8.f * (float)i + 1.f) - 1.f) * 0.5f);
    while ((nt + 1) * (nt + 2) / 2 <= i) ++nt;
    while (nt * (nt + 1) / 2 > i) --nt;
    r.nt = nt;
    r.mt = i - nt * (nt + 1) / 2;
    return r;
  }
  const int per_group = lp.group_m * lp.tiles_n;
  const int first = i / per_group * lp.group_m;
  const int size = min(lp.group_m, lp.tiles_m - first);
  const int j = i % per_group;
  r.mt = first + j % size;
  r.nt = j / size;
  return r;
}

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

// What an epilogue warp knows about its chunk: `row` is this lane's output row, `row0` the
// warp's first one, `buf` its staging buffer
struct Spot {
  int64_t row, row0;
  int z, split, mt, nt, half, lane;
  uint32_t buf;
};

// Epi: begin(spot) once per tile, chunk(spot, column, values[32]) for each 32 columns
// inside the result, end(spot).
template <int BN, bool PAIR, bool SPLIT, typename Epi>
__device__ __forceinline__ void run_tiles(const CUtensorMap& map_a, const CUtensorMap& map_b, const Loop& lp, int64_t M, int64_t N,
                                          Epi& epi) {
  using G = Geo<BN, PAIR>;
  constexpr int STG = G::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* s_a = smem;
  uint8_t* s_b = smem + STG * G::A_BYTES;
  uint8_t* s_epi = s_b + STG * G::B_BYTES;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(s_epi + EPI_WARPS * EPI_BUF);
  uint64_t* empty_bar = full_bar + STG;
  uint64_t* acc_full = empty_bar + STG;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_rank() : 0u;
  const int unit = PAIR ? (int)(blockIdx.x >> 1) : (int)blockIdx.x;
  const int units = PAIR ? (int)(gridDim.x >> 1) : (int)gridDim.x;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STG; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], (PAIR ? 2 : 1) * EPI_WARPS);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(2 * BN));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(2 * BN));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
  }
  tc_fence_before();
  if constexpr (PAIR) cluster_sync_all();
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      for (int t = unit; t < lp.total && ok; t += units) {
        const Tile at = tile_at(lp, t);
        const int m0 = at.mt * G::TM + (int)rank * BM;
        const int n0 = at.nt * BN + (PAIR ? (int)rank * (BN / 2) : 0);
        const int kb0 = at.split * lp.nk_split, kb1 = min(lp.nk, kb0 + lp.nk_split);
        for (int c0 = kb0; c0 < kb1 && ok; c0 += lp.chunk) {
          const int c1 = min(kb1, c0 + lp.chunk);
          for (int seg = 0; seg < lp.nseg && ok; ++seg) {
            const int pa = lp.nseg == 3 && seg == 1, pb = lp.nseg == 3 && seg == 0;  // planes: hi.lo, lo.hi, hi.hi
            for (int kb = c0; kb < c1; ++kb, ++it) {
              const int s = it % STG;
              if (!mbar_wait(&empty_bar[s], ((it / STG) & 1) ^ 1)) {
                ok = false;
                break;
              }
              if (rank == 0) mbar_expect_tx(&full_bar[s], (PAIR ? 2u : 1u) * (G::A_BYTES + G::B_BYTES));
              const int k0 = kb * BK;
              uint8_t* a_dst = s_a + s * G::A_BYTES;
              uint8_t* b_dst = s_b + s * G::B_BYTES;
              if (!lp.a_mn) {
                load4<PAIR>(a_dst, &map_a, &full_bar[s], k0, m0, pa, at.z);
              } else {
                load4<PAIR>(a_dst, &map_a, &full_bar[s], m0, k0, pa, at.z);
                load4<PAIR>(a_dst + 8192, &map_a, &full_bar[s], m0 + 64, k0, pa, at.z);
              }
              if (!lp.b_mn) {
                load4<PAIR>(b_dst, &map_b, &full_bar[s], k0, n0, pb, at.z);
              } else {
#pragma unroll
                for (int j = 0; j < (PAIR ? BN / 2 : BN) / 64; ++j)
                  load4<PAIR>(b_dst + j * 8192, &map_b, &full_bar[s], n0 + 64 * j, k0, pb, at.z);
              }
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
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      const uint32_t fmt = lp.bf16 ? (1u << 7) | (1u << 10) : 0u;
      const uint32_t idesc = (1u << 4) | fmt | ((uint32_t)lp.a_mn << 15) | ((uint32_t)lp.b_mn << 16) | ((uint32_t)(BN >> 3) << 17) |
                             ((uint32_t)(G::TM >> 4) << 24);
      uint32_t it = 0, local = 0;
      bool ok = true;
      for (int t = unit; t < lp.total && ok; t += units) {
        const int split = t % lp.per_batch / (lp.per_batch / lp.splits);
        const int kb0 = split * lp.nk_split, kb1 = min(lp.nk, kb0 + lp.nk_split);
        for (int c0 = kb0; c0 < kb1 && ok; c0 += lp.chunk, ++local) {
          const int b = local & 1;
          if (!mbar_wait(&acc_empty[b], ((local >> 1) & 1) ^ 1)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t d = tmem + (uint32_t)(b * BN);
          const int steps = lp.nseg * (min(kb1, c0 + lp.chunk) - c0);
          for (int i = 0; i < steps; ++i, ++it) {
            const int s = it % STG;
            if (!mbar_wait(&full_bar[s], (it / STG) & 1)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t a0 = smem_u32(s_a + s * G::A_BYTES), b0 = smem_u32(s_b + s * G::B_BYTES);
#pragma unroll
            for (int k = 0; k < BK / 16; ++k) {
              const uint64_t ad = lp.a_mn ? smem_desc(a0 + k * 2048, 8192, 1024) : smem_desc(a0 + k * 32, 16, 1024);
              const uint64_t bd = lp.b_mn ? smem_desc(b0 + k * 2048, 8192, 1024) : smem_desc(b0 + k * 32, 16, 1024);
              mma<PAIR>(d, ad, bd, idesc, (i > 0 || k > 0) ? 1u : 0u);
            }
            commit<PAIR>(&empty_bar[s]);
          }
          if (ok) commit<PAIR>(&acc_full[b]);
        }
      }
    }
  } else {
    Spot sp;
    const int q = warp & 3;
    sp.half = (warp - 2) >> 2;
    sp.lane = lane;
    sp.buf = smem_u32(s_epi) + (uint32_t)(warp - 2) * EPI_BUF;
    constexpr int CH = BN / 64;  // chunks of 32 columns per warp
    uint32_t local = 0;
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
    for (int t = unit; t < lp.total && ok; t += units) {
      const Tile at = tile_at(lp, t);
      sp.z = at.z;
      sp.split = at.split;
      sp.mt = at.mt;
      sp.nt = at.nt;
      sp.row0 = (int64_t)at.mt * G::TM + (int64_t)rank * BM + q * 32;
      sp.row = sp.row0 + lane;
      const int64_t col0 = (int64_t)at.nt * BN + sp.half * (BN / 2);
      const uint32_t base = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(sp.half * (BN / 2));
      epi.begin(sp);
      if constexpr (SPLIT) {
        float acc[CH][32];
        const int kb0 = at.split * lp.nk_split, kb1 = min(lp.nk, kb0 + lp.nk_split);
        for (int c0 = kb0; c0 < kb1; c0 += lp.chunk, ++local) {
          const int b = local & 1;
          if (!mbar_wait(&acc_full[b], (local >> 1) & 1)) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < CH; ++c) {
            uint32_t cur[32];
            tmem_ld32_issue(base + (uint32_t)(b * BN + c * 32), cur);
            tmem_wait(cur);
#pragma unroll
            for (int i = 0; i < 32; ++i) acc[c][i] = c0 == kb0 ? __uint_as_float(cur[i]) : acc[c][i] + __uint_as_float(cur[i]);
          }
          release(b);
        }
        if (!ok) break;
#pragma unroll
        for (int c = 0; c < CH; ++c)
          if (col0 + c * 32 < N && sp.row0 < M) epi.chunk(sp, col0 + c * 32, acc[c]);  // warp-uniform
      } else {
        const int b = local & 1;
        if (!mbar_wait(&acc_full[b], (local >> 1) & 1)) break;
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < CH; ++c) {
          const int64_t col = col0 + c * 32;
          if (col >= N || sp.row0 >= M) break;  // warp-uniform
          uint32_t cur[32];
          tmem_ld32_issue(base + (uint32_t)(b * BN + c * 32), cur);
          tmem_wait(cur);
          float v[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(cur[i]);
          epi.chunk(sp, col, v);
        }
        release(b);
        ++local;
      }
      epi.end(sp);
    }
  }
  tc_fence_before();
  if constexpr (PAIR) cluster_sync_all();
  else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * BN));
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * BN));
  }
}

template <int BN, bool PAIR, bool SPLIT, typename Epi>
__global__ void __launch_bounds__(THREADS, 1) tile_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                                                          const __grid_constant__ Loop lp, const int64_t M, const int64_t N,
                                                          const __grid_constant__ typename Epi::Args args) {
  Epi epi(args);
  run_tiles<BN, PAIR, SPLIT>(map_a, map_b, lp, M, N, epi);
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

// CTAs (pairs count twice) that can be resident at once, per kernel and device
template <int BN, bool PAIR, bool SPLIT, typename Epi>
static int resident_units() {
  static int units[64] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  const int slot = dev >= 0 && dev < 64 ? dev : 0;
  if (units[slot] && slot == dev) return units[slot];
  auto* fn = tile_kernel<BN, PAIR, SPLIT, Epi>;
  cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Geo<BN, PAIR>::SMEM);
  int n = num_sms();
  if constexpr (PAIR) {
    n = num_sms() / 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(2 * n), 1, 1);
    cfg.blockDim = dim3(THREADS, 1, 1);
    cfg.dynamicSmemBytes = Geo<BN, PAIR>::SMEM;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 2;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int k = 0;
    if (cudaOccupancyMaxActiveClusters(&k, fn, &cfg) == cudaSuccess && k > 0) n = std::min(n, k);
    else cudaGetLastError();
  }
  units[slot] = n;
  return n;
}

// C [batch][M, N] = A . B with operands of one 16-bit plane, or of two (SPLIT). Fills in the loop's tile counts and launches as many CTAs (or
// pairs) as are resident, each walking its share of the tiles.
template <int BN, bool PAIR, bool SPLIT, typename Epi>
static int launch_as(const Operand& A, const Operand& B, int64_t M, int64_t N, int64_t K, int64_t batch, Loop lp,
                     const typename Epi::Args& args, cudaStream_t s, const char* what) {
  using G = Geo<BN, PAIR>;
  constexpr int planes = SPLIT ? 2 : 1;
  CUtensorMap ma, mb;
  auto map = [&](CUtensorMap* m, const Operand& o, int64_t major, int box) {
    const uint64_t span = (uint64_t)o.ld * 2 * (uint64_t)(o.mn ? K : major);
    const uint64_t ps = planes > 1 ? (uint64_t)o.plane_stride * 2 : span, bs = batch > 1 ? (uint64_t)o.batch_stride * 2 : ps * planes;
    return o.mn ? make_map(m, o.base, major, K, planes, batch, o.ld * 2, ps, bs, 64, 64)
                : make_map(m, o.base, K, major, planes, batch, o.ld * 2, ps, bs, 64, box);
  };
  int rc = map(&ma, A, M, BM);
  if (!rc) rc = map(&mb, B, N, PAIR ? BN / 2 : BN);
  if (rc) return rc;
  lp.a_mn = A.mn;
  lp.b_mn = B.mn;
  lp.nseg = planes > 1 ? 3 : 1;
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
  const int units = std::min(resident_units<BN, PAIR, SPLIT, Epi>(), lp.total);
  if constexpr (PAIR) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(2 * units), 1, 1);
    cfg.blockDim = dim3(THREADS, 1, 1);
    cfg.dynamicSmemBytes = G::SMEM;
    cfg.stream = s;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 2;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, tile_kernel<BN, PAIR, SPLIT, Epi>, ma, mb, lp, M, N, args);
  } else {
    tile_kernel<BN, PAIR, SPLIT, Epi><<<(unsigned)units, THREADS, G::SMEM, s>>>(ma, mb, lp, M, N, args);
  }
  return check_launch(what);
}

template <int BN, bool PAIR, typename Epi>
static int launch(const Operand& A, const Operand& B, int64_t M, int64_t N, int64_t K, int64_t batch, int planes, const Loop& lp,
                  const typename Epi::Args& args, cudaStream_t s, const char* what) {
  return planes > 1 ? launch_as<BN, PAIR, true, Epi>(A, B, M, N, K, batch, lp, args, s, what)
                    : launch_as<BN, PAIR, false, Epi>(A, B, M, N, K, batch, lp, args, s, what);
}

}  // namespace tile
}  // namespace b200
