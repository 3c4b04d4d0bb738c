// Orthogonalising a matrix by Newton-Schulz products, and the optimizer step that uses it.
//
//   X0 = G / (|G|_F + eps);  each step: S = X X^T, P = a I + b S + c S S, X <- P X
// (X X^T for rows <= cols, X^T X and X <- X P otherwise: the Gram matrix of the shorter
// side, without a transpose; a on P's diagonal, so that only P's epilogue reads a matrix).
// Step update: m' = mu m + g, G = g + mu m' (Nesterov) or m', p' = p (1 - lr wd) - lr sqrt(max(1, rows / cols)) X.
//
// Per step 3 products on the tensor cores (tc_tile.cuh). S and P are symmetric: only the
// tiles on and above the diagonal are computed (each written twice where products are
// launches of their own), so a step costs
// 3 m^2 n + m^3 flop (m the shorter side) instead of 4 m^2 n + 2 m^3.
// Precision. The iterates live in fp16, scaled by 2^8: |X|_F = 1 at the start and the
// singular values stay below about 1.3, so no entry can pass 2^9 while entries of 2^-20
// of the largest keep their bits. bf16 matrices take one fp16 plane (11 bits: 2e-3 of the
// result after 5 steps, below bf16's own rounding; with bf16 iterates it is 2e-2). fp32
// matrices take two planes, hi + lo (22 bits), three products: 2e-6, as with fp32 products. So
// do bf16 ones of few rows or columns, where no error averages out and a small singular value
// makes it grow: of 1600 matrices each with one plane, 2 x 2 were off by up to 3.8e-2, 8 x 8 by
// 1.8e-2, 16 x 16 by 6.4e-3 (24 x 24: 4.3e-3), with two by 3.2e-3 at most, bf16's rounding; a
// call takes 12 % longer (57 -> 64 us).
// Where eps outweighs |G| the iterates start far below 1: each matrix carries a power of two
// t = 2^e >= 1, Y = 2^8 t X is what is stored, b and c are divided by t^2 and t^4, and t
// shrinks as a makes X grow. t is 1 for any |G| above eps.
// The sum of squares is in 64 bits. Every sum has a fixed order.
// Stacks that fill the GPU run all products of all steps in one launch (below): 16 x 1024 x 1024
// fp32 in 0.91 ms, a pair's 256 x 256 tile of 16 K blocks every 29000 clocks (37000 POLY) for
// 22900 of MMAs, which write and read shared memory at nearly its rate while the
// epilogue stages through it. One small matrix is bound by its chain of 15 launches (1024 x 1024
// fp32: 222 us).
#include <cuda_fp16.h>

#include <cmath>

#include "tc_tile.cuh"

namespace b200 {
namespace ns {

using namespace tile;

constexpr float SCALE = 256.f, MOST_A = 250.f;
constexpr int64_t NARROW = 16;  // bf16 matrices up to this side take two planes
constexpr int NORM_BLOCKS = 296, NT = 256;

__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const __half2 t = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&t);
}
__device__ __forceinline__ void unpack_f16(uint32_t u, float& a, float& b) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
  a = f.x, b = f.y;
}

constexpr int GRAM = 0, POLY = 1, NEXT = 2, LAST = 3;

// result = cc product + ca source + diag I (POLY), as fp16 planes; LAST: out = cc product + fa add
struct NsArgs {
  const __half* src;  // planes at the result's offsets, or NULL
  __half* dst;        // planes, or NULL: the last product
  int64_t ld, plane, batch;
  float ca, cc, diag;
  int planes, mirror;
  void* out;
  const float* add;  // fp32, dense as out
  int64_t M, N;
  float fa;
  int bf16;
  const int* e0;               // [batch]: the exponent of t at the start
  int e_down, e_down_next;     // how far it has shrunk, and will have after this step
  int which;                   // GRAM, POLY, NEXT, LAST
};

// MIRROR: symmetric results (`mirror`) are written on both sides of the diagonal
template <bool MIRROR>
struct NsEpi {
  using Args = NsArgs;
  static constexpr bool SINGLE_WIDE = false, SINGLE_NARROW = true, TEAMS = true, INIT = true;
  const Args* a;
  __half* dst;
  float scale, ca, diag;
  __device__ explicit NsEpi(const Args& args) : a(&args), dst(args.dst) {}
  __device__ __forceinline__ void begin(const Spot& sp) {
    scale = a->cc, ca = a->ca, diag = a->diag;
    shrunk(a->e0[sp.z], a->e_down, a->e_down_next);
  }
  // the coefficients where t is not 1
  __device__ __forceinline__ void shrunk(int e0, int e_down, int e_down_next) {
    if (e0 != 0) {
      const int e = max(0, e0 - e_down), shrink = max(0, e0 - e_down_next) - e;
      if (a->which == POLY) {
        ca = ldexpf(ca, shrink - 2 * e);
        scale = ldexpf(scale, shrink - 4 * e);
        diag = ldexpf(diag, shrink);
      } else if (a->which == LAST) {
        scale = ldexpf(scale, -e);
      }
    }
  }
  __device__ __forceinline__ void end(const Spot&) {}
  __device__ __forceinline__ void finish(int) {}

  // What the product is added to: ca source + diag I (POLY), fa add (LAST). The source arrives as
  // its planes' 16 words each, in the chunk's own registers.
  __device__ __forceinline__ bool dense(const Spot& sp, int64_t col) const {  // 16-byte rows of whole chunks
    return col + 32 <= a->N && (a->N & 3) == 0 && (reinterpret_cast<uintptr_t>(a->add) & 15) == 0;
  }
  __device__ __forceinline__ bool adds() const { return a->which == POLY || (a->which == LAST && a->add); }
  __device__ __forceinline__ void fetch(const Spot& sp, int64_t col, float (&v)[32]) {
    const int rows = (int)min((int64_t)32, a->M - sp.row0), cols = (int)min((int64_t)32, a->N - col);
    if (a->which == POLY) {
      const __half* p = a->src + sp.z * a->batch + sp.row0 * a->ld + col;  // rows are padded to 8 elements
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (k < a->planes) rows_load<2>(reinterpret_cast<const uint8_t*>(p + k * a->plane), a->ld * 2, rows, (cols + 7) / 8, sp.lane, v, 16 * k);
    } else if (a->which == LAST && a->add) {
      const float* p = a->add + (sp.z * a->M + sp.row0) * a->N + col;
      if (dense(sp, col)) {
        rows_load<4>(reinterpret_cast<const uint8_t*>(p), a->N * 4, rows, 8, sp.lane, v, 0);
      } else if (sp.lane < rows) {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (i < cols) v[i] = p[sp.lane * a->N + i];
      }
    }
  }
  __device__ __forceinline__ void ready(const Spot& sp, int64_t col, float (&v)[32]) {
    if (a->which == POLY) {
      rows_in<2>(sp.buf, sp.lane, v, 0);
      if (a->planes > 1) rows_in<2>(sp.buf + 2048u, sp.lane, v, 16);
      uint32_t w[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) w[i] = __float_as_uint(v[i]);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float x, y, lx, ly;  // (one plane: its partner's words are zeros)
        unpack_f16(w[i], x, y);
        unpack_f16(w[16 + i], lx, ly);
        v[2 * i] = ca * (x + lx);
        v[2 * i + 1] = ca * (y + ly);
      }
      const int k = (int)(sp.row - col);
      if (k >= 0 && k < 32) {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (k == i) v[i] += diag;
      }
    } else if (a->which == LAST && a->add) {
      if (dense(sp, col)) rows_in<4>(sp.buf, sp.lane, v, 0);
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] *= a->fa;
    }
  }

  __device__ __forceinline__ void chunk(const Spot& sp, int64_t col, float (&v)[32]) {
    const int rows = (int)min((int64_t)32, a->M - sp.row0);
    const int64_t cols = min((int64_t)32, a->N - col);
    if (a->which == LAST) {
      const int64_t at = (sp.z * a->M + sp.row0) * a->N + col;
      __syncwarp();
      if (a->bf16) {
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
        stage_chunk<2>(sp.buf, sp.lane, w);
        __syncwarp();
        put_chunk<2>(sp.buf, sp.lane, reinterpret_cast<uint8_t*>(reinterpret_cast<__nv_bfloat16*>(a->out) + at), a->N, rows, (int)cols);
      } else {
        uint32_t w[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) w[i] = __float_as_uint(v[i]);
        stage_chunk<4>(sp.buf, sp.lane, w);
        __syncwarp();
        put_chunk<4>(sp.buf, sp.lane, reinterpret_cast<uint8_t*>(reinterpret_cast<float*>(a->out) + at), a->N, rows, (int)cols);
      }
      return;
    }
    // The chunk goes through shared memory, 64-byte rows whose four 16-byte pieces are swizzled by
    // (row / 2) ^ (row / 8): rows written and read, and 8 x 8 blocks read transposed, are then free
    // of bank conflicts. Rows leave as 64 adjacent bytes each way.
    const int lane = sp.lane;
    const bool mirror = MIRROR && a->mirror && sp.mt != sp.nt;
    for (int k = 0; k < a->planes; ++k) {
      __half* d = dst + sp.z * a->batch + k * a->plane;
      const uint32_t buf = sp.buf + (uint32_t)(k & 1) * 2048u;
      uint32_t w[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) w[i] = pack_f16(v[2 * i], v[2 * i + 1]);
      __syncwarp();
      const uint32_t f = (uint32_t)((lane >> 1) ^ (lane >> 3)) & 3u;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        st_shared_v4(buf + (uint32_t)lane * 64u + (((uint32_t)j ^ f) << 4), w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
      __syncwarp();
      // 8 rows of 4 pieces at a time (rows are padded to 8 elements: whole pieces)
      const int piece = lane & 3;
      uint4 u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 8 * i + (lane >> 2);
        u[i] = ld_shared_v4(buf + (uint32_t)r * 64u + (((uint32_t)piece ^ (((r >> 1) ^ (r >> 3)) & 3u)) << 4));
      }
      __half* row = d + (sp.row0 + (lane >> 2)) * a->ld + col + 8 * piece;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (8 * i + (lane >> 2) < rows && 8 * piece < cols) *reinterpret_cast<uint4*>(row + 8 * i * a->ld) = u[i];
      if (mirror) {
        // four 8 x 8 blocks transposed: block m's rows are 8 c/2 + 2 m + c%2 (c = 0..7), so that
        // thread l ends up with rows 8 (l % 4) .. + 7 of source column 8 g + l / 4
        const int c = lane & 7, r = 8 * (c >> 1) + 2 * (lane >> 3) + (c & 1);
#pragma unroll
        for (int g = 0; g < 4; ++g)
          asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                       : "=r"(u[g].x), "=r"(u[g].y), "=r"(u[g].z), "=r"(u[g].w)
                       : "r"(buf + (uint32_t)r * 64u + (((uint32_t)g ^ (((r >> 1) ^ (r >> 3)) & 3u)) << 4))
                       : "memory");
        // the mirrored rows are as long as the result: whole pieces up to the padding
        row = d + (col + (lane >> 2)) * a->ld + sp.row0 + 8 * piece;
#pragma unroll
        for (int g = 0; g < 4; ++g)
          if (8 * g + (lane >> 2) < cols && 8 * piece < rows) *reinterpret_cast<uint4*>(row + 8 * g * a->ld) = u[g];
      }
      if (k + 1 < a->planes) {
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

// ---- all products of all steps in one launch ----
// Where the products fill the CTA pairs, each one's last wave of tiles is partial (16 matrices of
// 1024 x 1024: 160, 160 and 256 tiles for 74 pairs, 10 waves for 7.8) and each launch fills and
// drains its pipeline (the optimizer step: 1.39 ms as launches, 1.09 in one). So all tiles
// of all products form one list, taken by the pairs in order. A tile waits until its matrix's
// previous product is complete: counters in the workspace, one per matrix, of the CTAs that
// have finished a tile. Every tile depends on earlier ones of the list only, which running
// pairs have taken: the first unfinished one never waits, however many pairs are resident.
// A matrix's buffers are overwritten two products after their last reader at the
// earliest, which the same counter orders.
// S and P, symmetric, are stored on and above the diagonal's tiles only (the mirrored half
// took 6000 clocks a tile, of 15000 for the epilogue): a K block left of the diagonal is read as the
// transposed block above it, with the rows adjacent.
constexpr int MAX_STEPS = 100, ARRIVALS = 2;  // of a tile

struct Chain {
  static constexpr bool CHAIN = true;
  struct One {
    int64_t M, N;
    int nk, chunk, tiles_m, tiles_n, walk, per;  // per: tiles of one matrix
  };
  CUtensorMap x_gram[2], x_next[2], s[2], p[2];  // s, p: [1] with the rows adjacent
  One one[3];     // GRAM, POLY, NEXT
  int* finished;  // [batch], then the tickets
  int batch, steps, tall;
  __device__ __forceinline__ int per_step() const { return one[0].per + one[1].per + one[2].per; }
  __device__ __forceinline__ int total() const { return steps * batch * per_step(); }
  __device__ __forceinline__ Tile at(int t) const {
    Tile r = {};
    r.step = t / (batch * per_step());
    t -= r.step * batch * per_step();
    while (r.product < NEXT && t >= batch * one[r.product].per) t -= batch * one[r.product++].per;
    const One& o = one[r.product];
    r.z = t / o.per;
    place(r, t % o.per, o.walk, o.tiles_m, o.tiles_n, 16);
    return r;
  }
  __device__ __forceinline__ Tile kind(int t) const { return at(t); }
  __device__ __forceinline__ int blocks(const Tile& t) const { return one[t.product].nk; }
  __device__ __forceinline__ int blocks_each(const Tile& t) const { return one[t.product].nk; }
  __device__ __forceinline__ int chunk(const Tile& t) const { return one[t.product].chunk; }
  __device__ __forceinline__ int64_t rows(const Tile& t) const { return one[t.product].M; }
  __device__ __forceinline__ int64_t cols(const Tile& t) const { return one[t.product].N; }
  struct Side {  // an operand: K blocks below `until` are read with the rows adjacent
    const CUtensorMap *adjacent, *rest;
    int until;
    __device__ __forceinline__ const CUtensorMap* map(int kb) const { return kb < until ? adjacent : rest; }
    __device__ __forceinline__ int mn(int kb) const { return kb < until; }
  };
  // the symmetric operand's tile row i: what lies left of the diagonal, transposed
  __device__ __forceinline__ Side symmetric(const CUtensorMap (&m)[2], int i) const { return {&m[1], &m[0], i * (256 / BK)}; }
  __device__ __forceinline__ Side plain(const CUtensorMap& m, int adjacent) const { return {&m, &m, adjacent ? 1 << 30 : 0}; }
  __device__ __forceinline__ Side side_a(const Tile& t) const {
    if (t.product == GRAM) return plain(x_gram[t.step & 1], tall);
    return t.product == POLY ? symmetric(s, t.mt) : (tall ? plain(x_next[t.step & 1], 0) : symmetric(p, t.mt));
  }
  __device__ __forceinline__ Side side_b(const Tile& t) const {
    if (t.product == GRAM) return plain(x_gram[t.step & 1], tall);
    return t.product == POLY ? symmetric(s, t.nt) : (tall ? symmetric(p, t.nt) : plain(x_next[t.step & 1], 1));
  }
  __device__ __forceinline__ void prefetch() const {
    for (const CUtensorMap* m : {&x_gram[0], &s[0], &p[0], &x_next[0]})
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(m)) : "memory");
  }
  __device__ __forceinline__ int ticket() const { return atomicAdd(finished + batch, 1); }
  // true once the tile's matrix has seen every product before this one (by one thread); false
  // (and the device error flag set) if that takes too long
  __device__ __forceinline__ bool ready(const Tile& t) const {
    int need = t.step * per_step();
    if (t.product > 0) need += one[0].per;
    if (t.product > 1) need += one[1].per;
    need *= ARRIVALS;
    unsigned long long t0 = 0;
    while (true) {
      int v;
      asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(finished + t.z) : "memory");
      if (v >= need) break;
      if (t0 == 0) t0 = globaltimer();
      if (globaltimer() - t0 > WAIT_LIMIT_NS) {
        raise_device_error(B200_ERR_TIMEOUT);
        return false;
      }
      __nanosleep(64);
    }
    asm volatile("fence.proxy.async;" ::: "memory");  // TMA reads next
    return true;
  }
  // this CTA's part of the tile is stored (by one thread that has waited for the warps which did)
  __device__ __forceinline__ void done(const Tile& t) const {
    if (t.product == NEXT && t.step + 1 == steps) return;
    asm volatile("fence.proxy.async;" ::: "memory");  // TMA reads it
    __threadfence();
    asm volatile("red.release.gpu.global.add.s32 [%0], 1;" ::"l"(finished + t.z) : "memory");
  }
};

struct ChainEpi : NsEpi<false> {
  struct Step {
    float ca, cc, diag;
    int e_down, e_down_next;
  };
  struct Args {
    NsArgs part[4];  // GRAM, POLY, NEXT, LAST
    Step step[MAX_STEPS];
    __half* x[2];
    int steps;
  };
  const Args& all;
  __device__ explicit ChainEpi(const Args& args) : NsEpi<false>(args.part[0]), all(args) {}
  __device__ __forceinline__ void enter(const Tile& t, const Spot& sp) {
    const bool last = t.product == NEXT && t.step + 1 == all.steps;
    a = &all.part[last ? LAST : t.product];
    dst = t.product == NEXT ? all.x[(t.step + 1) & 1] : a->dst;
    scale = a->cc;
    const Step& st = all.step[t.step];
    if (t.product == POLY) ca = st.ca, scale = st.cc, diag = st.diag;
    shrunk(a->e0[sp.z], st.e_down, st.e_down_next);
  }
};

template <bool SPLIT>
__global__ void __launch_bounds__(THREADS, 1) chain_kernel(const __grid_constant__ Chain chain, const __grid_constant__ ChainEpi::Args args) {
  ChainEpi epi(args);
  run_tiles<256, true, SPLIT, false>(chain, 1, false, epi);
}

// 8 values from element i on (the first n of them; the rest zeros): 16-byte loads where all 8
// are there and aligned
__device__ __forceinline__ void load8(const void* g, int bf16, int64_t i, int64_t n, float (&v)[8]) {
  if (bf16) {
    const __nv_bfloat16* p = reinterpret_cast<const __nv_bfloat16*>(g) + i;
    if (n >= 8 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
      const uint4 u = *reinterpret_cast<const uint4*>(p);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = __uint_as_float(w[j] << 16);
        v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = j < n ? __bfloat162float(p[j]) : 0.f;
    }
  } else {
    const float* p = reinterpret_cast<const float*>(g) + i;
    if (n >= 8 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
      const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = j < n ? p[j] : 0.f;
    }
  }
}

// Sums of squares of each matrix, a part per block. With a momentum: m' = mu m + g is
// written and G = g + mu m' (nesterov) or m' is what is summed.
__global__ void __launch_bounds__(NT) square_kernel(const void* g, int bf16, const float* mom, float* mom_out, float mu, int nesterov,
                                                    double* part, int64_t n) {
  __shared__ double red[NT / 32];
  const int64_t base = (int64_t)blockIdx.y * n;
  double s = 0.0;
  for (int64_t i = ((int64_t)blockIdx.x * NT + threadIdx.x) * 8; i < n; i += (int64_t)gridDim.x * NT * 8) {
    const int64_t left = n - i;
    float v[8];
    load8(g, bf16, base + i, left, v);
    if (mom) {
      float m[8];
      load8(mom, 0, base + i, left, m);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        m[j] = mu * m[j] + v[j];
        v[j] = nesterov ? v[j] + mu * m[j] : m[j];
      }
      float* p = mom_out + base + i;
      if (left >= 8 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
        *reinterpret_cast<float4*>(p) = make_float4(m[0], m[1], m[2], m[3]);
        *reinterpret_cast<float4*>(p + 4) = make_float4(m[4], m[5], m[6], m[7]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j < left) p[j] = m[j];
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) s += (double)v[j] * (double)v[j];
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

// X0 = 2^8 t G / (|G| + eps) as fp16 planes with rows padded to 8 elements; t's exponent
__global__ void __launch_bounds__(NT) start_kernel(const void* g, int bf16, const float* mom, float mu, int nesterov, const double* part,
                                                   int parts, float eps, int* e0, int* done, __half* x, int64_t ld, int64_t plane, int64_t batch,
                                                   int planes, int64_t rows, int64_t cols) {
  __shared__ double red[NT / 32];
  double s = 0.0;
  for (int i = threadIdx.x; i < parts; i += NT) s += part[(int64_t)blockIdx.y * parts + i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __shared__ float factors[2];
  __syncthreads();
  if (threadIdx.x == 0) {  // (some hundred instructions: as many as a thread's 16 elements)
    s = red[0];
    for (int i = 1; i < NT / 32; ++i) s += red[i];
    const double norm = sqrt(s), share = norm / (norm + (double)eps);
    const int e = share > 0.0 && share < 0.5 ? min(96, -1 - ilogb(share)) : 0;  // t share in [1/2, 1)
    if (blockIdx.x == 0) e0[blockIdx.y] = e, done[blockIdx.y] = 0, done[gridDim.y] = 0;
    // the factor as two, each within fp32's normal range for any norm of fp32 values
    const double full = ldexp((double)SCALE, e) / (norm + (double)eps);
    const int lg = full > 0.0 && full < 1e300 ? ilogb(full) / 2 : 0;
    factors[0] = ldexpf(1.f, lg), factors[1] = (float)ldexp(full, -lg);
  }
  __syncthreads();
  const float lift = factors[0], scale = factors[1];
  const int64_t base = (int64_t)blockIdx.y * rows * cols, per = ld / 8;
  // two pieces of 8 at a time, both loaded before either is worked on
  const int64_t total = rows * per, stride = (int64_t)gridDim.x * NT;
  for (int64_t i = (int64_t)blockIdx.x * NT + threadIdx.x; i < total; i += 2 * stride) {
    float v[2][8], m[2][8];
    __half* d[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int64_t u = i + k * stride, r = u / per, c = u % per * 8, at = base + r * cols + c;
      const int64_t n = u < total ? cols - c : 0;
      d[k] = x + (int64_t)blockIdx.y * batch + r * ld + c;
      if (!mom || nesterov) load8(g, bf16, at, n, v[k]);
      if (mom) load8(mom, 0, at, n, m[k]);  // the new momentum
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (i + k * stride >= total) break;
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float f = !mom ? v[k][j] : (nesterov ? v[k][j] + mu * m[k][j] : m[k][j]);
        v[k][j] = f * lift * scale;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = pack_f16(v[k][2 * j], v[k][2 * j + 1]);
      *reinterpret_cast<uint4*>(d[k]) = make_uint4(w[0], w[1], w[2], w[3]);
      if (planes > 1) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float a, b;
          unpack_f16(w[j], a, b);
          w[j] = pack_f16(v[k][2 * j] - a, v[k][2 * j + 1] - b);
        }
        *reinterpret_cast<uint4*>(d[k] + plane) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
}

static int64_t up8(int64_t v) { return (v + 7) / 8 * 8; }
static size_t align256(size_t v) { return (v + 255) & ~size_t(255); }

struct Plan {
  int planes;
  int64_t side, ldx, ldg, xn, gn;  // shorter side; row strides and sizes of one X and one Gram plane
  size_t x0, x1, s, p, part, e0, done, bytes;
};

static Plan plan(int dtype, int64_t batch, int64_t rows, int64_t cols) {
  Plan q = {};
  q.side = std::min(rows, cols);
  q.planes = dtype == B200_F32 || q.side <= NARROW ? 2 : 1;
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
  q.done = take((size_t)(batch + 1) * 4);
  q.bytes = at;
  return q;
}

// One product, on CTA pairs (256 x 256 tiles) when those fill two thirds of them, else on
// 128 x 128 tiles of single CTAs or teams: a 1024 x 1024 product has 16 of the former (10 reach
// the diagonal) for 74 pairs, 64 (36) of the latter for 148 CTAs.
static int product(const Operand& A, const Operand& B, int64_t M, int64_t N, int64_t K, int64_t batch, int planes, bool triangle,
                   const NsArgs& a, cudaStream_t s, const char* what) {
  Loop lp = {};
  lp.group_m = 16;
  lp.walk = triangle ? WALK_TRIANGLE : WALK_GROUPED;
  const int64_t tm = ceil_div(M, 256), tn = ceil_div(N, 256);
  const int64_t tiles = (triangle ? tn * (tn + 1) / 2 : tm * tn) * batch;
  const bool pair = M > 128 && N > 128 && tiles * 3 >= num_sms();
  return launch<NsEpi<true>>(A, B, M, N, K, batch, planes, pair, lp, a, s, what);
}

// One launch where the Gram product (the one with the fewest tiles) fills two thirds of the pairs.
// Measured, in one launch / as launches (us): fp32 8 x 1024 x 1024 505 / 781, 80 x 256 x 256 285 /
// 408, 8 x 768 x 3000 1004 / 1126, bf16 8 x 1024 x 1024 288 / 383; even, and left to the rule: fp32
// 17 x 512 x 2048 612 - 688 / 665 (51 Gram tiles, just past two thirds), one bf16 4096 x 4096 1219 / 1195
// (large products lose little between launches). Below two thirds the launches' smaller tiles win: fp32
// 4 x 1024 x 1024 422 / 380, 12 x 512 x 512 310 / 259, one 2048 x 2048 649 / 618.
static bool chained(int64_t batch, int64_t rows, int64_t cols, int steps) {
  const int64_t side = std::min(rows, cols), t = ceil_div(side, 256), tri = t * (t + 1) / 2;
  const int64_t all = (2 * tri + ceil_div(rows, 256) * ceil_div(cols, 256)) * batch * steps;
  return side > 128 && tri * batch * 3 >= num_sms() && all < (1ll << 26);
}

template <bool SPLIT>
static int launch_chain(const Chain& c, const ChainEpi::Args& args, cudaStream_t s, const char* what) {
  using G = Geo<256, true, SPLIT>;
  const int units = std::min(resident<G, chain_kernel<SPLIT>>(2), c.batch * c.one[NEXT].per);
  if (units < 1) {
    set_error("%s: the kernel cannot be resident (registers)", what);
    return B200_ERR_CUDA;
  }
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
  cudaLaunchKernelEx(&cfg, chain_kernel<SPLIT>, c, args);
  return check_launch(what);
}

static int run_chain(const ChainEpi::Args& args, int* finished, const Operand (&X)[2], const Operand& S, const Operand& P, int64_t batch,
                     int64_t rows, int64_t cols, int planes, cudaStream_t s, const char* what) {
  const int64_t side = std::min(rows, cols), K = std::max(rows, cols);
  const int tall = rows > cols;
  Chain c = {};
  c.finished = finished, c.batch = (int)batch, c.steps = args.steps, c.tall = tall;
  auto fill = [&](int which, int64_t M, int64_t N, int64_t k, int walk) {
    const int nk = (int)ceil_div(k, BK), tm = (int)ceil_div(M, 256), tn = (int)ceil_div(N, 256);
    c.one[which] = {M, N, nk, planes > 1 ? CHUNK : nk, tm, tn, walk, walk == WALK_TRIANGLE ? tn * (tn + 1) / 2 : tm * tn};
  };
  fill(GRAM, side, side, K, WALK_TRIANGLE);
  fill(POLY, side, side, side, WALK_TRIANGLE);
  fill(NEXT, rows, cols, side, WALK_GROUPED);
  int rc = 0;
  for (int mn = 0; mn < 2 && !rc; ++mn) {
    Operand So = S, Po = P;
    So.mn = Po.mn = mn;
    rc = operand_map(&c.s[mn], So, side, side, planes, batch, BM);
    if (!rc) rc = operand_map(&c.p[mn], Po, side, side, planes, batch, BM);
  }
  for (int i = 0; i < 2 && !rc; ++i) {
    Operand Xo = X[i];
    Xo.mn = !tall;
    rc = operand_map(&c.x_gram[i], X[i], side, K, planes, batch, BM);
    if (!rc) rc = operand_map(&c.x_next[i], Xo, K, side, planes, batch, BM);
  }
  if (rc) return rc;
  return planes > 1 ? launch_chain<true>(c, args, s, what) : launch_chain<false>(c, args, s, what);
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
  int *e0 = reinterpret_cast<int*>(ws + q.e0), *done = reinterpret_cast<int*>(ws + q.done);
  const int64_t n = rows * cols;
  const int parts = (int)std::min<int64_t>(NORM_BLOCKS, ceil_div(n, NT * 8));
  const int bf16 = dtype == B200_BF16;
  square_kernel<<<dim3((unsigned)parts, (unsigned)batch), NT, 0, s>>>(g, bf16, mom, mom_out, mu, nesterov, part, n);
  int rc = check_launch(what);
  if (rc) return rc;
  const int64_t xb = q.planes * q.xn, gb = q.planes * q.gn;
  const unsigned gx = (unsigned)std::min<int64_t>(ceil_div(rows * (q.ldx / 8), NT), ceil_div(8 * (int64_t)num_sms(), batch));
  start_kernel<<<dim3(gx, (unsigned)batch), NT, 0, s>>>(g, bf16, mom ? mom_out : nullptr, mu, nesterov, part, parts, eps, e0, done, x[0], q.ldx, q.xn,
                                                        xb, q.planes, rows, cols);
  if ((rc = check_launch(what))) return rc;
  const bool tall = rows > cols;
  Operand X[2], Sm, Pm;  // by products: X as the Gram product reads it
  X[0].ld = X[1].ld = q.ldx, X[0].plane_stride = X[1].plane_stride = q.xn, X[0].batch_stride = X[1].batch_stride = xb;
  X[0].mn = X[1].mn = tall, X[0].base = x[0], X[1].base = x[1];
  Sm.ld = q.ldg, Sm.plane_stride = q.gn, Sm.batch_stride = gb;
  Pm = Sm;
  Sm.base = S, Pm.base = P;
  ChainEpi::Args all = {};
  NsArgs &gram = all.part[GRAM], &poly = all.part[POLY], &next = all.part[NEXT], &out = all.part[LAST];
  gram.e0 = e0, gram.planes = q.planes, gram.M = gram.N = q.side, gram.ld = q.ldg, gram.plane = q.gn, gram.batch = gb;
  gram.mirror = 1;
  poly = gram;
  gram.which = GRAM, gram.dst = S, gram.cc = 1.f / SCALE;
  poly.which = POLY, poly.src = S, poly.dst = P;
  next.which = NEXT, next.e0 = e0, next.planes = q.planes, next.M = rows, next.N = cols;
  next.ld = q.ldx, next.plane = q.xn, next.batch = xb, next.cc = 1.f / SCALE;
  out = next;
  out.which = LAST, out.cc = f.fb / (SCALE * SCALE);
  out.out = f.out, out.add = f.add, out.fa = f.fa, out.bf16 = f.bf16;
  double grown = 0.0;  // log2 of how far a has made the smallest X grow
  for (int i = 0; i < steps; ++i) {
    const float a = coef[3 * i], b = coef[3 * i + 1], c = coef[3 * i + 2];
    ChainEpi::Step& st = all.step[i];
    st.ca = b, st.cc = c / SCALE, st.diag = a * SCALE;
    st.e_down = st.e_down_next = (int)std::floor(grown);
    grown += std::max(0.0, std::log2((double)std::fabs(a)));
    if (i + 1 < steps) st.e_down_next = (int)std::floor(grown);
  }
  all.x[0] = x[0], all.x[1] = x[1], all.steps = steps;
  const int64_t K = tall ? rows : cols;  // of the Gram product
  if (chained(batch, rows, cols, steps)) return run_chain(all, done, X, Sm, Pm, batch, rows, cols, q.planes, s, what);
  for (int i = 0; i < steps; ++i) {
    const Operand& Xi = X[i & 1];
    if ((rc = product(Xi, Xi, q.side, q.side, K, batch, q.planes, true, gram, s, what))) return rc;
    const ChainEpi::Step& st = all.step[i];
    poly.ca = st.ca, poly.cc = st.cc, poly.diag = st.diag, poly.e_down = st.e_down, poly.e_down_next = st.e_down_next;
    if ((rc = product(Sm, Sm, q.side, q.side, q.side, batch, q.planes, true, poly, s, what))) return rc;
    NsArgs& r = i + 1 < steps ? next : out;
    r.e_down = st.e_down;
    if (i + 1 < steps) r.dst = x[(i + 1) & 1];
    // P X (wide: X's columns are the result's) or X P (tall); P's rows serve as its columns
    Operand Xo = Xi;
    Xo.mn = !tall;
    rc = tall ? product(Xo, Pm, rows, cols, q.side, batch, q.planes, false, r, s, what)
              : product(Pm, Xo, rows, cols, q.side, batch, q.planes, false, r, s, what);
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
  for (int i = 0; i < steps; ++i) {
    // a stands on P's diagonal, in fp16 times 2^8: from 256 on it would be infinite
    const float a = coef[3 * i], b = coef[3 * i + 1], c = coef[3 * i + 2];
    B200_REQUIRE(std::fabs(a) < MOST_A && std::isfinite(b) && std::isfinite(c),
                 "%s: coefficients (%g, %g, %g) of step %d: want finite numbers, the first within %g", what, (double)a, (double)b, (double)c, i,
                 (double)MOST_A);
  }
  B200_REQUIRE(eps >= 0.f, "%s: eps %g is negative", what, (double)eps);
  B200_REQUIRE(need == 0 || (ws && bytes >= need && (reinterpret_cast<uintptr_t>(ws) & 255) == 0),
               "%s: workspace of %zu bytes, %zu needed (256-byte aligned)", what, bytes, need);
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
