// The residual sum's entry points (residual_norm.cuh: the mathematics and the kernels), and the sums of the weights' gradients
// over blocks.
#include "residual_norm.cuh"

namespace b200 {
namespace rnorm {

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
static void shape(int64_t cols, bool vec, bool grad, int* threads, int* nv) {
  *nv = cols <= (grad && vec ? 512 : 256 * 8) ? 1 : (cols <= 512 * 16 && vec ? 2 : 4);
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
// blocks that the SMs hold at once (by the registers that the kernels are capped at)
static int64_t fill_of(int threads, int nv, bool grad) {
  const int most = nv == 1 ? 256 : 512;
  const int blocks = nv == 1 ? (grad ? Bounds<1>::GRADIENT : Bounds<1>::FORWARD)
                             : (nv == 2 ? (grad ? Bounds<2>::GRADIENT : Bounds<2>::FORWARD) : (grad ? Bounds<4>::GRADIENT : Bounds<4>::FORWARD));
  return (int64_t)num_sms() * std::min(32, blocks * most / threads);
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
  a.w_bf16 = (weights ? n->weight_dtype : n->x_dtype) == B200_BF16, a.gate_bf16 = (n->gate ? n->gate_dtype : n->x_dtype) == B200_BF16;
  a.scale = n->scale, a.eps = n->eps, a.inv_cols = (float)(1.0 / (double)n->cols);
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

// the launch's shape, and how the kernel gets its weights
static Launch plan(const b200_residual_norm* n, Args& a, bool vec, bool grad) {
  Launch l = {};
  shape(n->cols, vec, grad, &l.threads, &l.nv);
  const Split s = split(a.rows, a.groups, fill_of(l.threads, l.nv, grad));
  a.chunks = s.chunks, a.per_chunk = s.per_chunk;
  l.blocks = s.blocks, l.vec = vec, l.layer = n->kind == B200_NORM_LAYER, l.post = n->post != 0, l.gate = n->groups > 0;
  a.gate_kept = a.has_gate && a.per_group >= 4;  // read from shared memory thrice at least for one store there
  const int slots = a.has_gamma + a.has_beta + a.has_post_gamma + a.has_post_beta + a.gate_kept;
  l.shared = (size_t)slots * 8 * l.nv * l.threads * sizeof(float);
  // beyond 46 KB (wide rows) the weights are read again: the L1 holds them as well
  a.shared = l.shared <= 46 * 1024;
  if (!a.shared) l.shared = 0;
  return l;
}
static int run(const b200_residual_norm* n, const Args& a, const Launch& l, bool grad, cudaStream_t st) {
  using B = __nv_bfloat16;
  const bool xb = n->x_dtype == B200_BF16, fb = n->f_dtype == B200_BF16;
  if (grad)
    return xb ? (fb ? run_gradient<B, B>(a, l, st) : run_gradient<B, float>(a, l, st)) : (fb ? run_gradient<float, B>(a, l, st) : run_gradient<float, float>(a, l, st));
  return xb ? (fb ? run_forward<B, B>(a, l, st) : run_forward<B, float>(a, l, st)) : (fb ? run_forward<float, B>(a, l, st) : run_forward<float, float>(a, l, st));
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
  return run(n, a, plan(n, a, vectors(n, {x, f, sum, normed}), false), false, as_stream(stream));
}

static int kept_of(int kind, int post) { return (post ? 2 : 1) * (kind == B200_NORM_LAYER ? 2 : 1); }

extern "C" size_t b200_residual_norm_grad_workspace_bytes(const b200_residual_norm* n) {
  if (!n || n->rows <= 0 || n->cols < 1 || n->cols > MAX_COLS || n->groups < 0 || (n->groups && n->rows % n->groups)) return 0;
  int64_t most = 0;
  for (bool vec : {false, true}) {  // which of the two depends on the pointers
    int threads, nv;
    shape(n->cols, vec, true, &threads, &nv);
    const Split s = split(n->rows, n->groups ? n->groups : 1, fill_of(threads, nv, true));
    const int64_t gate = n->groups && s.chunks > 1 ? s.blocks : 0;
    most = std::max(most, s.blocks * kept_of(n->kind, n->post) + gate);
  }
  return (size_t)(most * n->cols) * sizeof(float);
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
  const Launch l = plan(n, a, vectors(n, {dsum, dnormed, x, f, dx, df, g->dgate}), true);
  const int kept = kept_of(n->kind, n->post);
  a.part = reinterpret_cast<float*>(workspace);
  a.gate_part = a.part + l.blocks * kept * n->cols;
  if (int rc = run(n, a, l, true, st)) return rc;
  // the sums over blocks of the weights that are asked for
  Fold fold = {};
  fold.part = a.part, fold.count = l.blocks, fold.pitch = kept * n->cols, fold.cols = a.cols;
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
  if (gate && a.chunks > 1) {
    Fold fg = {};
    fg.part = a.gate_part, fg.count = a.chunks, fg.pitch = n->cols, fg.cols = a.cols;
    fg.out[0] = {g->dgate, 0, a.gate_bf16};
    fold_kernel<<<dim3(wide, 1, (unsigned)a.groups), 256, 0, st>>>(fg);
    return check_launch("residual_norm_grad");
  }
  return B200_OK;
}
