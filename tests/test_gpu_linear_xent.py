"""The head's cross entropy without logits against its definition in 64 bits.

Tolerances, from T = |x| |w| per logit (and the like for the gradients' sums):
* a logit: few tokens' logits are K / 8 + 8 fp32 additions at most, each off by 2^-24 of the
  terms so far. Above, the tensor cores add 16 products at a time to an fp32 accumulator, each addition
  off by at most 2^-23 of the terms so far: (D / 16 + 2) 2^-23 T (so (D / 16 + 4) 2^-23 T covers both). fp32 operands come as
  hi + lo in bf16 (each rounding at most 2^-8 of its value): lo is off by 2^-16, lo . lo is
  left out: 3 * 2^-16 T more, and three times the additions.
* lse and loss: at most the largest logit's error (twice for the loss), plus 2^-21 for the
  exponentials (2^-22 each) and the sum, plus a rounding of the result (2^-22 relative).
* d = dloss (p - onehot): p off by p (twice the logit's error + 2^-20); rounded to bf16
  (2^-8), or to two planes (2^-16).
* dx, dw: those of d times |w|, |x| summed; the additions as above; a rounding of the result.
* Below the smallest normal fp32 number an exponential is zero: p is off by 2^-126 at most
  besides, d by that times dloss (and by 2^-126 where it falls below that itself), and a
  sum's terms and the sum by 2^-126 each."""

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


def no_device_error():
    from b200 import _lib as L
    from b200 import ops

    return L.lib().b200_check_device_error(ops.stream_ptr()) == L.OK


def inputs(n, d, v, dtype, seed=0, scale=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + n * 31 + d * 7 + v)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x, w = r(n, d).to(dtype), (r(d, v) * scale / d**0.5).to(dtype)
    labels = torch.randint(0, v, (n,), generator=g, device="cuda")
    labels[torch.rand(n, generator=g, device="cuda") < 0.2] = -100
    return x, w, labels, (0.5 + torch.rand(n, generator=g, device="cuda")) / n


def additions(k, dtype):
    return ((k / 16 + 4) * (3 if dtype == F32 else 1)) * 2.0**-23


def check(x, w, labels, dloss, got, ignore=-100):
    loss, lse, dx, dw = got
    x64, w64 = x.double(), w.double()
    rloss, rlse, rdx, rdw, d = R.linear_xent(x64, w64, labels, ignore, dloss.double())
    dtype = x.dtype
    D, V, N = w.shape[0], w.shape[1], x.shape[0]
    split = 3 * 2.0**-16 if dtype == F32 else 0.0
    ez = (x64.abs() @ w64.abs()) * (additions(D, dtype) + split)
    er = ez.max(-1).values + 2.0**-21
    assert ((lse.double() - rlse).abs() <= er + 2.0**-22 * rlse.abs()).all()
    assert ((loss.double() - rloss).abs() <= 2 * er + 2.0**-22 * (rloss.abs() + rlse.abs())).all()
    p = d.abs()  # |d| >= the part of p that errs where the label is not; at the label p dloss <= |d| + dloss
    kept = (labels != ignore).double()
    soft = torch.softmax(x64 @ w64, -1) * (dloss.double() * kept)[:, None]
    ed = soft * (2 * er[:, None] + 2.0**-20) + p * (2.0**-16 + split if dtype == F32 else 2.0**-8)
    ed = ed + 2.0**-126 * (dloss.double() * kept + 1)[:, None]
    xk = x64.abs() * kept[:, None]
    tx = ed @ w64.abs().t() + (p @ w64.abs().t()) * (additions(V, dtype) + split) + (V + 1) * 2.0**-126
    tw = xk.t() @ ed + (xk.t() @ p) * (additions(N, dtype) + split) + (N + 1) * 2.0**-126
    assert ((dx.double() - rdx).abs() <= tx + R.HALF_STEP[dtype] * rdx.abs()).all(), "dx"
    assert ((dw.double() - rdw).abs() <= tw + R.HALF_STEP[dtype] * rdw.abs()).all(), "dw"


# up to 8 tokens of fp32 (one of bf16) in kernels of their own, fp32 products and sums, and just beyond them
FEW = [(8, 1536, 333), (8, 1537, 77), (1, 12288, 40), (1, 12289, 40), (7, 100, 4001), (2, 173, 5000), (3, 64, 129), (4, 96, 128), (9, 96, 128),
       (6, 40, 31), (1, 1024, 32000), (1, 172, 4097), (1, 7, 64), (1, 12292, 36)]
SIZES = [(1, 8, 1), (1, 1, 5), (3, 16, 7), (5, 64, 300), (2, 1000, 129), (130, 72, 513), (257, 40, 1000), (128, 128, 256), (129, 33, 257),
         (600, 256, 3001), (4, 64, 20000)]


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("size", SIZES + FEW)
def test_loss_and_gradients(size, dtype, tied):
    x, w, labels, dloss = inputs(*size, dtype)
    if tied:
        w = w.t().contiguous().t()
    loss, lse = op("LinearCrossEntropy", x, w, labels)
    dx, dw = op("LinearCrossEntropyGrad", dloss, x, w, labels, lse)
    assert dx.dtype == dtype and dw.dtype == dtype and dw.shape == w.shape and (dw.stride() == w.stride() or min(w.shape) == 1)
    check(x, w, labels, dloss, (loss, lse, dx, dw))
    assert no_device_error()


def test_several_pieces_of_the_vocabulary():
    n, d, v = 20000, 64, 16001  # 640 MB of logit gradients: two pieces, the last one ragged
    for dtype, tied in ((BF, False), (F32, True)):
        x, w, labels, dloss = inputs(n, d, v, dtype)
        w = w.t().contiguous().t() if tied else w
        loss, lse = op("LinearCrossEntropy", x, w, labels)
        check(x, w, labels, dloss, (loss, lse, *op("LinearCrossEntropyGrad", dloss, x, w, labels, lse)))


def test_layouts_shapes_and_label_types():
    x, w, labels, dloss = inputs(48, 56, 300, BF)
    loss, lse = op("LinearCrossEntropy", x, w, labels)
    grads = op("LinearCrossEntropyGrad", dloss, x, w, labels, lse)
    wide = torch.zeros(48, 200, dtype=BF, device="cuda")
    wide[:, 64:120] = x
    off = torch.zeros(48 * 56 + 1, dtype=BF, device="cuda")[1:].view(48, 56)
    off.copy_(x)
    cols = torch.zeros(56, 600, dtype=BF, device="cuda")[:, ::2]
    cols.copy_(w)
    big = torch.zeros(57, 304, dtype=BF, device="cuda")
    big[1:, 3:303] = w
    for xv, wv, lv in ((wide[:, 64:120], w, labels), (off, cols, labels.int()), (x, big[1:, 3:303], labels[:, None]),
                       (x.t().contiguous().t(), w, labels)):
        l2, e2 = op("LinearCrossEntropy", xv, wv, lv)
        assert torch.equal(l2, loss) and torch.equal(e2, lse)
        g2 = op("LinearCrossEntropyGrad", dloss, xv, wv, lv, e2)
        assert torch.equal(g2[0], grads[0]) and torch.equal(g2[1], grads[1])
    l3, e3 = op("LinearCrossEntropy", x.view(4, 12, 56), w, labels.view(4, 12))
    assert l3.shape == (4, 12) and torch.equal(l3.view(-1), loss)
    g3 = op("LinearCrossEntropyGrad", dloss.view(4, 12), x.view(4, 12, 56), w, labels.view(4, 12, 1), e3)
    assert g3[0].shape == (4, 12, 56) and torch.equal(g3[0].view(48, 56), grads[0]) and torch.equal(g3[1], grads[1])
    same = x[:1].expand(48, 56)  # a broadcast input
    l4, _ = op("LinearCrossEntropy", same, w, labels)
    l5, _ = op("LinearCrossEntropy", same.contiguous(), w, labels)
    assert torch.equal(l4, l5)


def test_contraction_policy_and_mixed_types():
    from b200 import ops

    x, w, labels, dloss = inputs(40, 64, 200, BF)
    want = op("LinearCrossEntropy", x, w, labels)
    wg = op("LinearCrossEntropyGrad", dloss, x, w, labels, want[1])
    ops.Config.matmul_dtype = "bf16"
    got = op("LinearCrossEntropy", x.float(), w.float(), labels)
    gg = op("LinearCrossEntropyGrad", dloss, x.float(), w.float(), labels, got[1])
    assert torch.equal(got[0], want[0]) and gg[0].dtype == gg[1].dtype == F32
    assert torch.equal(gg[0].to(BF), wg[0]) and torch.equal(gg[1].to(BF), wg[1])
    ops.Config.matmul_dtype = "f32"
    mixed = op("LinearCrossEntropyGrad", dloss, x, w.float(), labels, want[1])
    full = op("LinearCrossEntropyGrad", dloss, x.float(), w.float(), labels, want[1])
    assert mixed[0].dtype == BF and torch.equal(mixed[0], full[0].to(BF)) and torch.equal(mixed[1], full[1])


def test_ignored_rows_stay_out():
    x, w, labels, dloss = inputs(70, 64, 500, BF)
    labels[::3] = -1
    _, lse = op("LinearCrossEntropy", x, w, labels, ignore_index=-1)
    labels[labels == -100] = 3
    loss, lse = op("LinearCrossEntropy", x, w, labels, ignore_index=-1)
    dx, dw = op("LinearCrossEntropyGrad", dloss, x, w, labels, lse, ignore_index=-1)
    check(x, w, labels, dloss, (loss, lse, dx, dw), ignore=-1)
    x2 = x.clone()
    x2[0], x2[3], x2[6, 1] = float("nan"), float("inf"), float("-inf")
    loss2, lse2 = op("LinearCrossEntropy", x2, w, labels, ignore_index=-1)
    dx2, dw2 = op("LinearCrossEntropyGrad", dloss, x2, w, labels, lse2, ignore_index=-1)
    assert torch.equal(loss2, loss) and torch.equal(dx2, dx) and torch.equal(dw2, dw)
    labels[:] = -100
    loss, lse = op("LinearCrossEntropy", x, w, labels)
    dx, dw = op("LinearCrossEntropyGrad", dloss, x, w, labels, lse)
    assert not loss.any() and not dx.any() and not dw.any() and torch.isfinite(lse).all()


def test_labels_outside_set_the_device_error():
    x, w, labels, dloss = inputs(9, 32, 50, BF)
    labels[:] = 5
    labels[4] = 50
    loss, lse = op("LinearCrossEntropy", x, w, labels)
    assert not no_device_error() and loss[4] == 0 and no_device_error()
    dx, dw = op("LinearCrossEntropyGrad", dloss, x, w, labels, lse)
    assert not dx[4].any() and dx[3].any() and no_device_error()


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_few_tokens_ignored_invalid_and_not_finite(dtype, tied):
    x, w, labels, dloss = inputs(6, 72, 300, dtype)
    w = w.t().contiguous().t() if tied else w
    labels[:] = torch.tensor([3, -100, 299, 300, -100, 0], device="cuda")
    x[1], x[4, 0] = float("nan"), float("inf")
    loss, lse = op("LinearCrossEntropy", x, w, labels)
    assert not no_device_error() and loss[1] == loss[3] == loss[4] == 0
    dx, dw = op("LinearCrossEntropyGrad", dloss, x, w, labels, lse)
    assert no_device_error() and not dx[1].any() and not dx[3].any() and not dx[4].any()
    kept = [0, 2, 5]
    l2, e2 = op("LinearCrossEntropy", x[kept], w, labels[kept])
    g2 = op("LinearCrossEntropyGrad", dloss[kept], x[kept], w, labels[kept], e2)
    check(x[kept], w, labels[kept], dloss[kept], (l2, e2, *g2))
    # alone or among others: the same tokens, in sums of other lengths
    torch.testing.assert_close(loss[kept], l2, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(dx[kept].float(), g2[0].float(), rtol=2e-2, atol=1e-6)
    torch.testing.assert_close(dw.float(), g2[1].float(), rtol=2e-2, atol=1e-6)
    x[0, 5] = float("nan")
    loss, lse = op("LinearCrossEntropy", x[kept], w, labels[kept])
    assert torch.isnan(lse[0]) and torch.isfinite(lse[1:]).all() and torch.isnan(loss[0])


def test_large_logits_and_nan_rows():
    x, w, labels, dloss = inputs(33, 64, 700, F32, scale=300.0)
    loss, lse = op("LinearCrossEntropy", x, w, labels)
    check(x, w, labels, dloss, (loss, lse, *op("LinearCrossEntropyGrad", dloss, x, w, labels, lse)))
    labels[:] = 1
    x[7, 3] = float("nan")
    l2, e2 = op("LinearCrossEntropy", x, w, labels)
    assert torch.isnan(l2[7]) and torch.isnan(e2[7]) and torch.isfinite(torch.cat([l2[:7], l2[8:]])).all()


def test_empty_and_same_results_again():
    w = torch.randn(64, 30, device="cuda").to(BF)
    x, labels = torch.zeros(0, 64, dtype=BF, device="cuda"), torch.zeros(0, dtype=torch.int64, device="cuda")
    loss, lse = op("LinearCrossEntropy", x, w, labels)
    dx, dw = op("LinearCrossEntropyGrad", loss, x, w, labels, lse)
    assert loss.shape == (0,) and dx.shape == (0, 64) and not dw.any()
    x, w, labels, dloss = inputs(300, 64, 5000, BF)
    a = [*op("LinearCrossEntropy", x, w, labels)]
    for _ in range(2):
        b = [*op("LinearCrossEntropy", x, w, labels)]
        assert all(torch.equal(s, t) for s, t in zip(a, b))
        ga, gb = (op("LinearCrossEntropyGrad", dloss, x, w, labels, a[1]) for _ in range(2))
        assert all(torch.equal(s, t) for s, t in zip(ga, gb))


def test_gradients_against_differences():
    """Directional derivatives by central differences of the 64-bit forward."""
    x, w, labels, dloss = inputs(12, 24, 40, F32)
    _, lse = op("LinearCrossEntropy", x, w, labels)
    dx, dw = op("LinearCrossEntropyGrad", dloss, x, w, labels, lse)
    x64, w64 = x.double(), w.double()
    vx, vw = torch.randn_like(x64), torch.randn_like(w64)
    value = lambda a, b: float((R.linear_xent(a, b, labels)[0] * dloss.double()).sum())  # noqa: E731
    h = 1e-5
    num = (value(x64 + h * vx, w64) - value(x64 - h * vx, w64)) / (2 * h)
    assert abs(num - float((dx.double() * vx).sum())) <= 3e-4 * float((dx.double() * vx).abs().sum())
    num = (value(x64, w64 + h * vw) - value(x64, w64 - h * vw)) / (2 * h)
    assert abs(num - float((dw.double() * vw).sum())) <= 3e-4 * float((dw.double() * vw).abs().sum())


def test_graph_capture_and_other_streams():
    x, w, labels, dloss = inputs(200, 64, 1000, BF)

    def step():
        loss, lse = op("LinearCrossEntropy", x, w, labels)
        return (loss, lse, *op("LinearCrossEntropyGrad", dloss, x, w, labels, lse))

    want = step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cap = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = step()
    graph.replay()  # while the other stream's call may still run: the two share nothing
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, other, cap))
    x.copy_((x.float() * 0.5).to(BF))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(step(), cap))
