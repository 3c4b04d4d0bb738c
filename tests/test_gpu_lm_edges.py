"""Edges of the language-model operators that the tests by operator leave out. Definitions in 64
bits: ``lm_reference``."""

import threading

import pytest
import torch

import lm_reference as R

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _policy(cuda):
    from b200 import ops

    ops.Config.matmul_dtype = "f32"
    yield
    ops.Config.matmul_dtype = "f32"


def op(name, *args, **kw):
    from b200.backend import B200Backend

    return B200Backend.execute_op(name, *args, **kw)


def rand(*shape, dtype=F32, seed=0):
    g = torch.Generator().manual_seed(seed + sum(shape))
    return torch.randn(*shape, generator=g).to(dtype)


# ---- heads ----
# A rotated element is within 6e-7 (|a| + |b|): three roundings of an angle within pi / 4 (1.4e-7),
# the polynomials (2^-28) and their last roundings (2^-23), then four of 2^-24 for the factor, the
# products and the sum. The norm adds the fp32 sum of 512 squares (16 a lane, a tree of 5: 21
# roundings, halved by the root) and 5 roundings of its products: 1e-6. Held to 2e-6 of the
# terms and half a step of the result's type.
TERMS = 2e-6


def close(got, ref, mag):
    got = got.cpu()
    assert ((got.double() - ref).abs() <= R.HALF_STEP[got.dtype] * ref.abs() + TERMS * mag).all()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("part", [4, 12, 244, 252, 260, 500, 508])
def test_512_wide_interleaved_heads_of_any_rotated_part(part, dtype):
    """Both parts end inside a unit of two vectors: one unit more than 64."""
    b, n, h, hk, d = 2, 5, 3, 1, 512
    pos = torch.arange(n)[None] + 100 * torch.arange(b)[:, None]
    kw = {"rotary_dim": part, "interleaved": True}
    x, k = rand(b, n, h, d, dtype=dtype), rand(b, n, hk, d, dtype=dtype, seed=1)
    for name, sign in (("RotaryEmbedding", 1), ("RotaryEmbeddingGrad", -1)):
        close(op(name, x.cuda(), pos.cuda(), **kw), *R.rotate(x.double(), pos, part, interleaved=True, sign=sign))
    gq, gk = 1 + 0.2 * rand(d, seed=2), 1 + 0.2 * rand(d, seed=3)
    for y, t, g in zip(op("QKNormRotary", x.cuda(), k.cuda(), gq.cuda(), gk.cuda(), pos.cuda(), **kw), (x, k), (gq, gk)):
        close(y, *R.rotate(R.rms_unit(t.double(), 1e-6)[0] * g.double(), pos, part, interleaved=True))
    dy, dk = rand(b, n, h, d, dtype=dtype, seed=8), rand(b, n, hk, d, dtype=dtype, seed=9)
    got = op("QKNormRotaryGrad", dy.cuda(), dk.cuda(), x.cuda(), k.cuda(), gq.cuda(), gk.cuda(), pos.cuda(), **kw)
    for dx, dg, t, g, up in zip(got[:2], got[2:], (x, k), (gq, gk), (dy, dk)):
        gr, mag = R.rotate(up.double(), pos, part, interleaved=True, sign=-1)
        u, rstd = R.rms_unit(t.double(), 1e-6)
        ref = rstd * (gr * g.double() - u * (gr * g.double() * u).mean(-1, keepdim=True))
        m = mag * g.abs().double()
        close(dx, ref, rstd * (m + u.abs() * (m * u.abs()).mean(-1, keepdim=True)) * 2)
        # a sum of at most 30 terms in fp32
        assert ((dg.cpu().double() - (gr * u).sum((0, 1, 2))).abs() <= (mag * u.abs()).sum((0, 1, 2)) * (TERMS + 30 * 2.0**-24)).all()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("heads,dim", [((1, 1), 32), ((3, 1), 32), ((9, 2), 32), ((1, 3), 64), ((5, 1), 64), ((3, 1), 128), ((2, 1), 33)])
def test_norm_gradient_without_eps_and_idle_lanes(heads, dim, dtype):
    """Head counts that are no multiple of what a warp takes; eps = 0 is 1e-30 where no row is zero."""
    q, k = rand(2, 7, heads[0], dim, dtype=dtype), rand(2, 7, heads[1], dim, dtype=dtype, seed=1)
    dq, dk = rand(*q.shape, dtype=dtype, seed=2), rand(*k.shape, dtype=dtype, seed=3)
    g = (1 + 0.2 * rand(dim, seed=4)).cuda()
    args = [t.cuda() for t in (dq, dk, q, k)] + [g, g]
    got, want = op("QKNormRotaryGrad", *args, eps=0.0, rotary_dim=0), op("QKNormRotaryGrad", *args, eps=1e-30, rotary_dim=0)
    for a, b in zip(got, want):
        assert torch.isfinite(a).all() and torch.equal(a, b)
    got, want = op("QKNormRotary", *args[2:], eps=0.0, rotary_dim=0), op("QKNormRotary", *args[2:], eps=1e-30, rotary_dim=0)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---- the head's loss ----


def inputs(n, d, v, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + n + d + v)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return (r(n, d).to(dtype), (r(d, v) / d**0.5).to(dtype), torch.randint(0, v, (n,), generator=g, device="cuda"),
            (0.5 + torch.rand(n, generator=g, device="cuda")) / n)


@pytest.mark.parametrize("tied", [False, True])
def test_threads_with_few_tokens_of_different_widths(tied):
    """Threads that launch the same kernels with different amounts of shared memory above 48 KB: straight
    through the entry points, so that the calls meet."""
    from b200 import _lib as L

    lib, calls, results, keep = L.lib(), [], [], []
    for d in (1508, 1536):
        x, w, labels, dloss = inputs(8, d, 128, F32)
        w = w.t().contiguous() if tied else w
        loss, lse = op("LinearCrossEntropy", x, w.t() if tied else w, labels)
        dx, dw = op("LinearCrossEntropyGrad", dloss, x, w.t() if tied else w, labels, lse)
        for _ in range(2):  # two threads each, on streams, workspaces and results of their own
            s = torch.cuda.Stream()
            got = [torch.zeros_like(t) for t in (loss, lse, dx, w)]
            head = (x.data_ptr(), d, w.data_ptr(), w.stride(0), int(not tied))
            sizes = (8, d, 128)
            nf, nb = (f(L.F32, *head, *sizes) for f in (lib.b200_linear_xent_workspace_bytes, lib.b200_linear_xent_grad_workspace_bytes))
            wf, wb = (torch.empty(n, dtype=torch.uint8, device="cuda") for n in (nf, nb))
            fwd = (L.F32, *head, labels.data_ptr(), L.I64, -100, got[0].data_ptr(), got[1].data_ptr(), *sizes, wf.data_ptr(), nf, s.cuda_stream)
            bwd = (L.F32, dloss.data_ptr(), *head, labels.data_ptr(), L.I64, -100, lse.data_ptr(), got[2].data_ptr(), got[3].data_ptr(), *sizes,
                   wb.data_ptr(), nb, s.cuda_stream)
            calls.append((fwd, bwd))
            results.append((got, (loss, lse, dx, dw.t() if tied else dw)))
            keep.append((x, w, labels, dloss, lse, s, wf, wb))
    torch.cuda.synchronize()
    start, bad = threading.Barrier(len(calls)), []

    def run(fwd, bwd):
        start.wait()
        for _ in range(2000):
            rc = lib.b200_linear_xent(*fwd) or lib.b200_linear_xent_grad(*bwd)
            if rc != L.OK:
                bad.append(rc)

    threads = [threading.Thread(target=run, args=c) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not bad, f"{len(bad)} calls failed, the first with status {bad[0]}"
    assert all(torch.equal(a, b) for got, want in results for a, b in zip(got, want))
    assert keep


@pytest.mark.parametrize("n", [3, 40])
@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("policy,x_type,w_type", [("bf16", F32, F32), ("bf16", BF, F32), ("bf16", F32, BF), ("f32", F32, BF), ("f32", BF, F32)])
def test_gradient_of_a_cast_weight_is_stored_as_the_weight(policy, x_type, w_type, tied, n):
    from b200 import ops

    ops.Config.matmul_dtype = policy
    x, w, labels, dloss = inputs(n, 64, 200, BF)
    x, w = x.to(x_type), w.to(w_type)
    if tied:
        w = w.t().contiguous().t()
    _, lse = op("LinearCrossEntropy", x, w, labels)
    dx, dw = op("LinearCrossEntropyGrad", dloss, x, w, labels, lse)
    assert dw.stride() == w.stride() and dw.dtype == w_type and dx.dtype == x_type and dx.is_contiguous()
    dense = op("LinearCrossEntropyGrad", dloss, x, w.contiguous(), labels, lse)
    for a, b in zip((dx, dw), dense):
        # bf16 values of d and of the operands: each a half step of 2^-8 off, in sums of other orders
        torch.testing.assert_close(a.float(), b.float(), rtol=2.0**-6, atol=2.0**-6 * float(b.float().abs().max()))


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n", [1, 6, 40, 300])
def test_labels_outside_give_no_gradient_whatever_x_holds(n, dtype, tied):
    """As rows of ignore_index do: nothing of a not finite x reaches dw."""
    from b200 import _lib as L
    from b200 import ops

    x, w, labels, dloss = inputs(n, 72, 300, dtype)
    w = w.t().contiguous().t() if tied else w
    labels[0], labels[-1] = 300, -7
    _, lse = op("LinearCrossEntropy", x, w, labels)
    want = op("LinearCrossEntropyGrad", dloss, x, w, labels, lse)
    x[0], x[-1] = float("nan"), float("inf")
    loss, lse = op("LinearCrossEntropy", x, w, labels)
    got = op("LinearCrossEntropyGrad", dloss, x, w, labels, lse)
    assert L.lib().b200_check_device_error(ops.stream_ptr()) == L.ERR_ARG
    assert loss[0] == 0 and loss[-1] == 0 and not got[0][0].any() and not got[0][-1].any()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("n,d,v", [(1, 64, 200), (1, 7, 64), (5, 64, 201), (140, 64, 333), (20000, 64, 16001)])
def test_gradients_are_rounded_to_the_callers_types_only(n, d, v, tied):
    """fp32 x and w under the bf16 policy: bf16 operands and fp32 gradients. Tolerance: that of bf16
    operands (d half a step of 2^-8 off, fp32 sums cut by 2^-23 an addition of 16 products) without a
    bf16 rounding of the result."""
    from b200 import ops

    x, w, labels, dloss = inputs(n, d, v, BF)
    if tied:
        w = w.t().contiguous().t()
    ops.Config.matmul_dtype = "bf16"
    _, lse = op("LinearCrossEntropy", x.float(), w.float(), labels)
    dx, dw = op("LinearCrossEntropyGrad", dloss, x.float(), w.float(), labels, lse)
    narrow = op("LinearCrossEntropyGrad", dloss, x, w, labels, lse)
    assert dx.dtype == dw.dtype == F32 and torch.equal(dx.to(BF), narrow[0]) and torch.equal(dw.to(BF), narrow[1])
    assert float((dx != narrow[0].float()).float().mean()) > 0.5 and float((dw != narrow[1].float()).float().mean()) > 0.5
    half = op("LinearCrossEntropyGrad", dloss, x.float(), w, labels, lse)
    assert torch.equal(half[0], dx) and torch.equal(half[1], narrow[1]) and half[1].dtype == BF
    if n > 1000:
        return
    x64, w64 = x.double(), w.double()
    *_, rdx, rdw, dl = R.linear_xent(x64, w64, labels, dloss=dloss.double())
    cut = lambda k: (k / 16 + 4) * 2.0**-23  # noqa: E731
    er = (x64.abs() @ w64.abs()).max(-1).values * cut(d) + 2.0**-21
    ed = torch.softmax(x64 @ w64, -1) * dloss.double()[:, None] * (2 * er[:, None] + 2.0**-20) + dl.abs() * 2.0**-8 + 2.0**-126
    for got, ref, tol in ((dx, rdx, ed @ w64.abs().t() + (dl.abs() @ w64.abs().t()) * cut(v)),
                          (dw, rdw, x64.abs().t() @ ed + (x64.abs().t() @ dl.abs()) * cut(n))):
        assert ((got.double() - ref).abs() <= tol + R.HALF_STEP[F32] * ref.abs()).all()


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("n", [65537, 2**18 + 77])
def test_weight_gradient_of_many_tokens_is_not_cut_short(n, tied):
    """Sums over all tokens of terms of one sign, in fp32 from bf16 operands. The tensor cores cut a sum
    towards zero by up to 2^-23 of it in each of at most two additions per 16 products, half of
    that on average and of half the final sum: 2^-24 of it per 16. Over the 32768 tokens of one
    accumulator that is 2048 2^-24 = 2^-13, and the same of the whole for sums of several (131072 at once:
    2^-11). d's rounding to bf16 is to either side: 2^-9 a term, 2^-17 of such sums. A logit's
    error, 2^-21 as in the operator's tests, moves p by as much. So the mean over the sums is held to
    2^-12, twice the cut."""
    from b200 import ops

    d, v = 4096, 1000  # tiles enough that the tokens are not shared out for the SMs' sake
    g = torch.Generator(device="cuda").manual_seed(n)
    x = (0.5 + torch.rand(n, d, generator=g, device="cuda")).to(BF)
    w = (torch.randn(d, v, generator=g, device="cuda") / d**0.5).to(BF)
    if tied:
        w = w.t().contiguous().t()
    labels = torch.zeros(n, dtype=torch.int64, device="cuda")  # the other words' sums have positive terms only
    dloss = (0.5 + torch.rand(n, generator=g, device="cuda")) / n
    ops.Config.matmul_dtype = "bf16"
    _, lse = op("LinearCrossEntropy", x.float(), w.float(), labels)
    dx, dw = op("LinearCrossEntropyGrad", dloss, x.float(), w.float(), labels, lse)
    ref = torch.zeros(d, v, dtype=torch.float64, device="cuda")
    for i in range(0, n, 2**16):
        xc, lc = x[i : i + 2**16].double(), slice(i, i + 2**16)
        ref += xc.t() @ (torch.softmax(xc @ w.double(), -1) * dloss[lc].double()[:, None])
    off = ((dw.double() - ref) / ref)[:, 1:]
    assert abs(float(off.mean())) <= 2.0**-12 and float(off.abs().max()) <= 2.0**-10
    narrow = op("LinearCrossEntropyGrad", dloss, x, w, labels, lse)
    assert torch.equal(narrow[1], dw.to(BF)) and torch.equal(narrow[0], dx.to(BF)) and narrow[1].stride() == w.stride()


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("v", [33000, 2**18 + 100])
def test_input_gradient_of_many_words_is_not_cut_short(v, tied):
    """The same of sums over the vocabulary: positive weights, but for the label's own, which are zero. The
    tolerance is that of the sums over tokens."""
    from b200 import ops

    n, d = 1280, 2048  # tiles enough that the words are not shared out for the SMs' sake
    g = torch.Generator(device="cuda").manual_seed(v)
    x = (torch.randn(n, d, generator=g, device="cuda") / d**0.5).to(BF)
    w = (0.5 + torch.rand(d, v, generator=g, device="cuda")).to(BF)
    w[:, 0] = 0
    if tied:
        w = w.t().contiguous().t()
    labels = torch.zeros(n, dtype=torch.int64, device="cuda")
    dloss = (0.5 + torch.rand(n, generator=g, device="cuda")) / n
    ops.Config.matmul_dtype = "bf16"
    _, lse = op("LinearCrossEntropy", x.float(), w, labels)
    dx, dw = op("LinearCrossEntropyGrad", dloss, x.float(), w, labels, lse)
    ref, all_of = torch.zeros(n, d, dtype=torch.float64, device="cuda"), []
    for i in range(0, v, 2**15):
        all_of.append(x.double() @ w[:, i : i + 2**15].double())
    p = torch.softmax(torch.cat(all_of, 1), -1) * dloss.double()[:, None]
    for i in range(0, v, 2**15):
        ref += p[:, i : i + 2**15] @ w[:, i : i + 2**15].double().t()
    off = (dx.double() - ref) / ref
    assert abs(float(off.mean())) <= 2.0**-12 and float(off.abs().max()) <= 2.0**-9
    narrow = op("LinearCrossEntropyGrad", dloss, x, w, labels, lse)
    assert torch.equal(narrow[0], dx.to(BF)) and torch.equal(narrow[1], dw) and dw.stride() == w.stride()


# ---- orthogonalisation ----


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 9), (2, 2), (2, 3), (500, 2), (3, 3), (4, 4), (5, 5), (8, 8), (8, 64), (12, 12), (16, 16), (16, 200)])
def test_narrow_bf16_matrices_one_by_one(rows, cols):
    """Each of 1600 matrices: at most half a step of bf16, and the products' 3e-6 grown by a = 3.4445 in each of five
    steps, which a small singular value may do."""
    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    m = (torch.randn(1600, rows, cols, generator=g, device="cuda") * 1e-3).to(BF)
    ref = R.newton_schulz(m.double())
    off = (op("NewtonSchulz", m).double() - ref).flatten(1).norm(dim=1) / ref.flatten(1).norm(dim=1)
    assert float(off.max()) <= R.HALF_STEP[BF] + 3e-6 * 3.4445**5


# ---- updates ----


@pytest.mark.parametrize("weight_decay", [0.0, 0.1])
@pytest.mark.parametrize("shape", [(24, 40), (40, 24), (33, 33), (3, 64, 256), (3, 256, 64), (20, 300, 270)])
def test_apply_muon_scales_by_the_axis_of_the_outputs(shape, weight_decay):
    """Matmul weights [inputs, outputs]: sqrt(max(1, cols / rows)), and the transpose of the default on
    the transposed weights. Tolerance: the products' 3e-5 of the step (its derivation stands with
    the operator's own tests), and four roundings of 2^-24 of what is added."""
    p, m, g = (rand(*shape, seed=i).cuda() * 0.02 for i in (1, 2, 3))
    kw = {"lr": 0.05, "momentum": 0.9, "weight_decay": weight_decay}
    p2, m2 = op("ApplyMuon", p, m, g, output_axis=-1, **kw)
    rm = 0.9 * m.double() + g.double()
    step = 0.05 * max(1.0, shape[-1] / shape[-2]) ** 0.5 * R.newton_schulz(g.double() + 0.9 * rm)
    err = p2.double() - (p.double() * (1 - 0.05 * weight_decay) - step)
    assert float(err.norm()) <= 3e-5 * float(step.norm()) + 2.0**-22 * float(p.double().norm() + step.norm())
    turned = op("ApplyMuon", p.mT.contiguous(), m.mT.contiguous(), g.mT.contiguous(), output_axis=len(shape) - 2, **kw)
    assert float((turned[0].mT.double() - p2.double()).norm()) <= 6e-5 * float(step.norm()) + 2.0**-21 * float(p.double().norm() + step.norm())
    assert torch.equal(m2, turned[1].mT) and torch.equal(m2, op("ApplyMuon", p, m, g, **kw)[1])
    pc, mc = p.clone(), m.clone()
    op("ApplyMuon", pc, mc, g, out=(pc, mc), output_axis=len(shape) - 1, **kw)
    assert torch.equal(pc, p2) and torch.equal(mc, m2)
    assert torch.equal(op("ApplyMuon", p, m, g, output_axis=-2, **kw)[0], op("ApplyMuon", p, m, g, **kw)[0])
