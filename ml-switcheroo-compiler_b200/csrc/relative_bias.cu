// The learned position bias of scores that are held in memory, and its table's gradient.
//
//   bias[h, i, j] = table[bucket(j - i - shift), h]
//   dtable[b, h] = sum of dbias[:, h, i, j] over the i, j of bucket b
//
// Both are bound by HBM: the bias is written once, the gradient read once.
// Forward: a block writes a flat piece of one head's plane in 16-byte vectors, whatever the row
// length; a vector outside (-far, far) is one value, the rest looks its elements up in shared memory.
// Gradient: within a run of rows a thread owns one diagonal rel and walks down it, so neighbouring
// threads read neighbouring elements and every element is added in a register, without atomics.
// A diagonal's sum goes to the block's own [-far, far] array, that to buckets, those to the
// workspace, and a second launch adds the blocks up in order.
// Measured: 16 x 1023 x 2047 bf16 in 21 us (29 with a division by the row length an element), the gradient of 4 x 16 x 777 x 1000 fp32
// in 44 to 50 us (67 with 8 loads a thread under way instead of 32). The bias is at half of HBM's rate while HBM is
// all but idle (the L2 takes the writes): its 1024 blocks of 32768 elements are under two waves of 592, so an SM has work for 72 %
// of the launch, and 61 % of its issue slots are taken then.
#include <algorithm>

#include "ew_common.cuh"
#include "relative.cuh"

namespace b200 {
namespace relative {

constexpr int THREADS = 256, PIECE = 32768;  // elements a block writes

template <typename T>
__global__ void __launch_bounds__(THREADS) bias_kernel(const __grid_constant__ b200_relative r, const T* table, T* out, int heads, int64_t plane, int keys,
                                                       int shift, uint32_t mul, uint32_t shr) {
  extern __shared__ __align__(16) uint8_t smem[];
  T* lut = reinterpret_cast<T*>(smem);  // by rel + far
  const int far = far_of(r), h = blockIdx.y;
  for (int i = threadIdx.x; i <= 2 * far; i += THREADS) lut[i] = table[(int64_t)bucket_of(r, i - far) * heads + h];
  __syncthreads();
  constexpr int VEC = 16 / sizeof(T);
  T* base = out + (int64_t)h * plane;
  // the first element of the plane on a 16-byte boundary; pieces start there, the first one takes what is before it
  const int64_t lead = min(plane, (int64_t)((16 - (reinterpret_cast<uintptr_t>(base) & 15)) & 15) / (int64_t)sizeof(T));
  const int64_t begin = lead + (int64_t)blockIdx.x * PIECE, end = min(plane, begin + PIECE);
  auto value = [&](int rel) { return lut[max(-far, min(far, rel)) + far]; };
  if (blockIdx.x == 0 && threadIdx.x < lead) base[threadIdx.x] = value((int)(threadIdx.x % keys) - (int)(threadIdx.x / keys) - shift);
  if (begin >= end) return;
  const int row0 = (int)(begin / keys), col0 = (int)(begin - (int64_t)row0 * keys);
  const int n = (int)(end - begin);
  for (int o = threadIdx.x * VEC; o < n; o += THREADS * VEC) {
    const uint32_t at = (uint32_t)(col0 + o);  // < keys + PIECE
    const uint32_t down = fast_div(at, mul, shr);
    int j = (int)(at - down * (uint32_t)keys);
    int rel = j - (row0 + (int)down) - shift;
    union {
      uint4 v;
      T t[VEC];
    } u;
    if (j + VEC <= keys) {
      if (rel >= far || rel + VEC - 1 <= -far) {
        const T c = lut[rel >= far ? 2 * far : 0];
#pragma unroll
        for (int k = 0; k < VEC; ++k) u.t[k] = c;
      } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k) u.t[k] = value(rel + k);
      }
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        u.t[k] = value(rel);
        ++rel;
        if (++j == keys) j = 0, rel -= keys + 1;
      }
    }
    if (o + VEC <= n) {
      *reinterpret_cast<uint4*>(base + begin + o) = u.v;
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k)
        if (o + k < n) base[begin + o + k] = u.t[k];
    }
  }
}

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }

struct GradShape {
  int rows, runs, pieces;  // rows a run, runs, pieces of WIDE diagonals
};
constexpr int WIDE = 2048;
static GradShape grad_shape(int64_t heads, int64_t queries, int64_t keys) {
  GradShape g;
  // 16 rows a run (its ragged ends cost 15 diagonals of keys + 15); longer ones where that leaves 8 blocks an SM
  int64_t rows = 16;
  while (rows < 64 && heads * ceil_div(queries, 2 * rows) >= 8 * (int64_t)num_sms()) rows *= 2;
  g.rows = (int)std::min<int64_t>(rows, queries);
  g.runs = (int)ceil_div(queries, g.rows);
  g.pieces = (int)ceil_div(keys + g.rows - 1, WIDE);
  return g;
}

template <typename T>
__global__ void __launch_bounds__(THREADS) bias_grad_kernel(const __grid_constant__ b200_relative r, const T* d, float* part, int64_t batch,
                                                            int heads, int queries, int keys, int shift, int rows) {
  extern __shared__ float near[];  // [2 far + 1], by rel + far
  __shared__ float edge[2][THREADS / 32];
  const int far = far_of(r), h = blockIdx.z;
  for (int i = threadIdx.x; i <= 2 * far; i += THREADS) near[i] = 0.f;
  __syncthreads();
  const int i0 = blockIdx.y * rows, n = min(rows, queries - i0);
  const int64_t plane = (int64_t)queries * keys;
  float before = 0.f, after = 0.f;  // rel <= -far, rel >= far
  // diagonal c: column c - (n - 1) + k in row i0 + k
  const int first = blockIdx.x * WIDE, last = min(first + WIDE, keys + n - 1);
  constexpr int WAYS = 2;  // diagonals of a thread at once
  for (int c = first + (int)threadIdx.x; c < last; c += WAYS * THREADS) {
    float s[WAYS] = {};
    for (int64_t b = 0; b < batch; ++b) {
      const T* p = d + (b * heads + h) * plane + (int64_t)i0 * keys + (c - (n - 1));
      for (int k = 0; k < n; k += 16) {  // 32 loads under way
        float v[WAYS][16];
#pragma unroll
        for (int w = 0; w < WAYS; ++w) {
          const int j = c + w * THREADS - (n - 1) + k;  // the column of row k
          const bool in = c + w * THREADS < last;
          const T* q = p + w * THREADS + (int64_t)k * (keys + 1);
#pragma unroll
          for (int u = 0; u < 16; ++u) {
            v[w][u] = in && k + u < n && j + u >= 0 && j + u < keys ? as_float(*q) : 0.f;
            q += keys + 1;
          }
        }
#pragma unroll
        for (int w = 0; w < WAYS; ++w) {
          float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int u = 0; u < 16; ++u) t[u & 3] += v[w][u];
          s[w] += (t[0] + t[1]) + (t[2] + t[3]);
        }
      }
    }
#pragma unroll
    for (int w = 0; w < WAYS; ++w) {
      if (c + w * THREADS >= last) break;
      const int rel = c + w * THREADS - (n - 1) - i0 - shift;  // |.| < 2^31: checked on the host
      if (rel >= far) after += s[w];
      else if (rel <= -far) before += s[w];
      else near[rel + far] = s[w];  // this thread's alone
    }
  }
  before = warp_sum(before), after = warp_sum(after);
  if ((threadIdx.x & 31) == 0) edge[0][threadIdx.x >> 5] = before, edge[1][threadIdx.x >> 5] = after;
  __syncthreads();
  if (threadIdx.x < 2) {
    float s = 0.f;
    for (int w = 0; w < THREADS / 32; ++w) s += edge[threadIdx.x][w];
    near[threadIdx.x ? 2 * far : 0] = s;
  }
  __syncthreads();
  const int nb = buckets_of(r);
  for (int b = threadIdx.x; b < nb; b += THREADS)
    part[(((int64_t)h * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x) * nb + b] = bucket_sum(r, far, near, b);
}

template <typename T>
__global__ void bias_grad_sum_kernel(const float* part, T* dtable, int heads, int64_t blocks, int nb) {
  // 32 lanes a value
  const int64_t at = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (at >= (int64_t)heads * nb) return;
  const int b = (int)(at / heads), h = (int)(at % heads);
  float s = 0.f;
  for (int64_t i = lane; i < blocks; i += 32) s += part[((int64_t)h * blocks + i) * nb + b];
  s = warp_sum(s);
  if (lane == 0) dtable[at] = (T)s;
}

static int check_sizes(const char* what, int64_t heads, int64_t queries, int64_t keys, int64_t shift) {
  B200_REQUIRE(heads >= 0 && heads <= 65535 && queries >= 0 && keys >= 0, "%s: %lld heads, %lld queries, %lld keys", what, (long long)heads,
               (long long)queries, (long long)keys);
  B200_REQUIRE(queries < (1 << 30) && keys < (1 << 30) && shift > -(1ll << 29) && shift < (1ll << 29), "%s: %lld queries, %lld keys, shift %lld",
               what, (long long)queries, (long long)keys, (long long)shift);
  return B200_OK;
}

}  // namespace relative
}  // namespace b200

using namespace b200;
using namespace b200::relative;

extern "C" int b200_relative_bias(const b200_relative* r, int dtype, const void* table, void* out, int64_t heads, int64_t queries,
                                  int64_t keys, int64_t shift, void* stream) {
  if (int rc = relative::check("relative_bias", r)) return rc;
  if (int rc = check_sizes("relative_bias", heads, queries, keys, shift)) return rc;
  if (dtype != B200_F32 && dtype != B200_BF16) {
    set_error("relative_bias: dtype %d (F32 and BF16)", dtype);
    return B200_ERR_DTYPE;
  }
  if (heads == 0 || queries == 0 || keys == 0) return B200_OK;
  B200_REQUIRE(table && out, "relative_bias: null operand");
  const int64_t plane = queries * keys;
  B200_REQUIRE(plane < (1ll << 45), "relative_bias: %lld queries times %lld keys", (long long)queries, (long long)keys);
  const dim3 grid((unsigned)std::max<int64_t>(1, ceil_div(plane, PIECE)), (unsigned)heads);
  const size_t shared = (size_t)(2 * far_of(*r) + 1) * (dtype == B200_F32 ? 4 : 2);
  uint32_t mul, shr;
  fastdiv_params((uint32_t)keys, mul, shr);
  if (dtype == B200_F32)
    bias_kernel<float><<<grid, relative::THREADS, shared, as_stream(stream)>>>(*r, (const float*)table, (float*)out, (int)heads, plane, (int)keys,
                                                                     (int)shift, mul, shr);
  else
    bias_kernel<__nv_bfloat16><<<grid, relative::THREADS, shared, as_stream(stream)>>>(*r, (const __nv_bfloat16*)table, (__nv_bfloat16*)out,
                                                                             (int)heads, plane, (int)keys, (int)shift, mul, shr);
  return check_launch("relative_bias");
}

extern "C" size_t b200_relative_bias_grad_workspace_bytes(const b200_relative* r, int64_t heads, int64_t queries, int64_t keys) {
  if (!r || r->side < 1 || heads <= 0 || queries <= 0 || keys <= 0) return 0;
  const GradShape g = grad_shape(heads, queries, keys);
  return (size_t)heads * g.runs * g.pieces * buckets_of(*r) * sizeof(float);
}

extern "C" int b200_relative_bias_grad(const b200_relative* r, int dtype, const void* dbias, void* dtable, int64_t batch, int64_t heads,
                                       int64_t queries, int64_t keys, int64_t shift, void* workspace, size_t workspace_bytes,
                                       void* stream) {
  if (int rc = relative::check("relative_bias_grad", r)) return rc;
  if (int rc = check_sizes("relative_bias_grad", heads, queries, keys, shift)) return rc;
  B200_REQUIRE(batch >= 0, "relative_bias_grad: batch %lld", (long long)batch);
  if (dtype != B200_F32 && dtype != B200_BF16) {
    set_error("relative_bias_grad: dtype %d (F32 and BF16)", dtype);
    return B200_ERR_DTYPE;
  }
  if (heads == 0) return B200_OK;
  B200_REQUIRE(dtable, "relative_bias_grad: null operand");
  cudaStream_t st = as_stream(stream);
  const int nb = buckets_of(*r);
  const size_t size = dtype == B200_F32 ? 4 : 2;
  if (batch == 0 || queries == 0 || keys == 0) {
    cudaMemsetAsync(dtable, 0, (size_t)heads * nb * size, st);
    return check_launch("relative_bias_grad");
  }
  B200_REQUIRE(dbias, "relative_bias_grad: null operand");
  const GradShape g = grad_shape(heads, queries, keys);
  B200_REQUIRE(g.runs <= 65535, "relative_bias_grad: %lld queries", (long long)queries);
  const size_t need = b200_relative_bias_grad_workspace_bytes(r, heads, queries, keys);
  B200_REQUIRE(workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 3) == 0,
               "relative_bias_grad: workspace of %zu bytes, %zu needed on a 4-byte boundary", workspace_bytes, need);
  float* part = reinterpret_cast<float*>(workspace);
  const dim3 grid((unsigned)g.pieces, (unsigned)g.runs, (unsigned)heads);
  const size_t shared = (size_t)(2 * far_of(*r) + 1) * sizeof(float);
  const int64_t blocks = (int64_t)g.runs * g.pieces;
  const unsigned sum_grid = (unsigned)ceil_div(heads * nb * 32, 256);
  if (dtype == B200_F32) {
    bias_grad_kernel<float><<<grid, relative::THREADS, shared, st>>>(*r, (const float*)dbias, part, batch, (int)heads, (int)queries, (int)keys,
                                                           (int)shift, g.rows);
    bias_grad_sum_kernel<float><<<sum_grid, 256, 0, st>>>(part, (float*)dtable, (int)heads, blocks, nb);
  } else {
    bias_grad_kernel<__nv_bfloat16><<<grid, relative::THREADS, shared, st>>>(*r, (const __nv_bfloat16*)dbias, part, batch, (int)heads, (int)queries,
                                                                   (int)keys, (int)shift, g.rows);
    bias_grad_sum_kernel<__nv_bfloat16><<<sum_grid, 256, 0, st>>>(part, (__nv_bfloat16*)dtable, (int)heads, blocks, nb);
  }
  count_launch();  // the sums' launch; check_launch counts the other
  return check_launch("relative_bias_grad");
}
