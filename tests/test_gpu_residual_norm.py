"""The residual sum with its norms, and its gradients, against the 64-bit forms on the CPU.

Tolerances: a mean is a tree over at most 32 elements a thread, 5 steps in a warp and 16 warps (53
roundings of 2^-24 at most of its terms), the rest of a value at most 10 roundings; the gradient makes two
such means of products. With mag the terms' magnitudes: 63 x 2^-24 = 4e-6, twice that where a norm reads
the other's result, thrice in the gradients; a weight's gradient adds up to 64 rows in a thread and 1000
blocks in eight slices (200 roundings, 1.2e-5 of the terms). Results of fewer bits: half a step besides."""

import pytest
import torch

import block_reference as R

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
GRADS = ("dx", "df", "dgamma", "dbeta", "dpost_gamma", "dpost_beta", "dgate")


@pytest.fixture(autouse=True)
def _device(cuda):
    yield


def op(name, *args, **kw):
    from b200.backend import B200Backend

    return B200Backend.execute_op(name, *args, **kw)


def rand(*shape, dtype=F32, seed=0, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed + sum(shape))
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype)


def close(got, ref, mag, terms, what):
    got = got.cpu()
    assert tuple(got.shape) == tuple(ref.shape), what
    off, tol = (got.double() - ref).abs(), R.HALF_STEP[got.dtype] * ref.abs() + terms * mag + 1e-37
    assert not (off > tol).any(), f"{what}: {int((off > tol).sum())} of {off.numel()} off, most {float((off / tol).max()):.3g} x"


def check(shape, xt=F32, ft=BF, wt=F32, norm="rms", post=True, gate=None, gt=F32, betas=True, scale=0.75, eps=1e-5, weights=True):
    c = shape[-1]
    x, f = rand(*shape, dtype=xt, shift=0.3), rand(*shape, dtype=ft, seed=1)
    w = {}
    if weights:
        w["gamma"] = rand(c, dtype=wt, seed=2, scale=0.2, shift=1)
        if post:
            w["post_gamma"] = rand(c, dtype=wt, seed=3, scale=0.2, shift=1)
        if norm == "layer" and betas:
            w["beta"] = rand(c, dtype=wt, seed=4)
            if post:
                w["post_beta"] = rand(c, dtype=wt, seed=5)
    if gate is not None:
        w["gate"] = rand(*gate, dtype=gt, seed=6, scale=0.3, shift=0.5)
    ds, dh = rand(*shape, dtype=xt, seed=7), rand(*shape, dtype=ft, seed=8)
    ref, mag = R.residual_norm(x, f, **w, scale=scale, norm=norm, post=post, eps=eps, dsum=ds, dnormed=dh)
    kw = {**{n: t.cuda() for n, t in w.items()}, "residual_scale": scale, "norm": norm, "post_norm": post, "eps": eps}
    total, normed = op("ResidualNorm", x.cuda(), f.cuda(), **kw)
    assert total.dtype == xt and normed.dtype == ft
    close(total, ref["sum"], mag["sum"], 4e-6, "sum")
    close(normed, ref["normed"], mag["normed"], 8e-6, "normed")
    for name, got in zip(GRADS, op("ResidualNormGrad", ds.cuda(), dh.cuda(), x.cuda(), f.cuda(), **kw)):
        given = name in ("dx", "df") or name[1:] in w
        assert (got is not None) == given, name
        if given:
            assert got.dtype == {"dx": xt, "df": ft, "dgate": gt}.get(name, wt)
            close(got, ref[name], mag[name], 2.4e-5, name)


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("width", [1, 7, 8, 64, 100, 256, 257, 1000, 1024, 1032, 2048, 4096, 4099, 8192, 8200, 16384])
def test_widths(width, post, norm):
    check((5, width), norm=norm, post=post, gate=(width,))


@pytest.mark.parametrize("xt", [F32, BF])
@pytest.mark.parametrize("ft", [F32, BF])
@pytest.mark.parametrize("wt", [F32, BF])
def test_types(xt, ft, wt):
    check((3, 50, 72), xt, ft, wt, norm="layer", gate=(3, 1, 72), gt=wt)
    check((3, 50, 75), xt, ft, wt, post=False, gate=(3, 50, 75), gt=ft)


@pytest.mark.parametrize("gate", [(96,), (1, 96), (1, 1, 96), (4, 1, 96), (4, 37, 96), None])
@pytest.mark.parametrize("shape", [(4, 37, 96)])
def test_gates(shape, gate):
    check(shape, gate=gate)
    check(shape, gate=gate, post=False, norm="layer", betas=False)


def test_many_groups_and_rows():
    check((5000, 3, 64), gate=(5000, 1, 64), gt=BF)  # more groups than blocks
    check((2, 9000, 40), gate=(2, 1, 40))
    check((30000, 24), gate=(24,))
    check((64, 1, 512), gate=(64, 1, 512))
    check((2, 3, 5, 64), gate=(2, 3, 1, 64))
    check((2, 3, 5, 64), gate=(2, 1, 1, 64))


def test_without_weights():
    check((3, 20, 128), weights=False, scale=1.0)
    check((3, 20, 128), weights=False, post=False, norm="layer", scale=-2.0)
    check((1, 1, 1024), gate=(1024,))


def test_one_step_of_each_type_and_mixed_weights():
    x, f = rand(4, 64), rand(4, 64, dtype=BF, seed=1)
    g, p = rand(64, dtype=BF, seed=2, shift=1), rand(64, seed=3, shift=1)
    ref, mag = R.residual_norm(x, f, gamma=g, post_gamma=p, dsum=x, dnormed=f)
    kw = {"gamma": g.cuda(), "post_gamma": p.cuda()}
    close(op("ResidualNorm", x.cuda(), f.cuda(), **kw)[1], ref["normed"], mag["normed"], 8e-6, "normed")
    got = op("ResidualNormGrad", x.cuda(), f.cuda(), x.cuda(), f.cuda(), **kw)
    assert got[2].dtype == BF and got[4].dtype == F32
    close(got[2], ref["dgamma"], mag["dgamma"], 2.4e-5, "dgamma")
    close(got[4], ref["dpost_gamma"], mag["dpost_gamma"], 2.4e-5, "dpost_gamma")


def test_layouts_and_empty():
    x, f = rand(3, 10, 64), rand(3, 10, 64, dtype=BF, seed=1)
    want = op("ResidualNorm", x.cuda(), f.cuda(), gamma=torch.ones(64).cuda())
    flat = torch.zeros(x.numel() + 1, device="cuda")
    off = flat[1:].view(x.shape)
    off.copy_(x)
    for a, b in ((off, f.cuda()), (x.cuda().transpose(0, 1).contiguous().transpose(0, 1), f.cuda())):
        got = op("ResidualNorm", a, b)
        assert (got[0] - want[0]).abs().max() < 1e-6 and (got[1].float() - want[1].float()).abs().max() < 2.0**-6
    e = torch.zeros(0, 64, device="cuda")
    gate, gamma = torch.ones(64, device="cuda"), torch.ones(64, device="cuda")
    s, h = op("ResidualNorm", e, e, gamma=gamma, gate=gate)
    assert s.shape == e.shape and h.shape == e.shape
    got = op("ResidualNormGrad", e, e, e, e, gamma=gamma, gate=gate)
    assert got[0].shape == e.shape and not got[2].any() and got[2].shape == (64,) and not got[6].any() and got[6].shape == (64,)


def test_rows_without_eps():
    """A row of zeros under eps 0 is not finite; its neighbours are untouched, idle threads too."""
    x, f = rand(3, 36), rand(3, 36, seed=1)
    x[1], f[1] = 0, 0
    for norm in ("rms", "layer"):
        s, h = op("ResidualNorm", x.cuda(), f.cuda(), eps=0.0, norm=norm, post_norm=True)
        assert s[[0, 2]].isfinite().all() and h[[0, 2]].isfinite().all() and h[1].isnan().all()
        dx, df = op("ResidualNormGrad", x.cuda(), f.cuda(), x.cuda(), f.cuda(), eps=0.0, norm=norm, post_norm=True)[:2]
        assert dx[[0, 2]].isfinite().all() and df[[0, 2]].isfinite().all()


def test_gradient_against_differences():
    shape, u = (2, 7, 40), 1e-5
    t = {"x": rand(*shape), "f": rand(*shape, seed=1), "gamma": rand(40, seed=2, shift=1), "beta": rand(40, seed=3),
         "post_gamma": rand(40, seed=4, shift=1), "post_beta": rand(40, seed=5), "gate": rand(2, 1, 40, seed=6, shift=1)}
    ds, dh = rand(*shape, seed=7), rand(*shape, seed=8)

    def value(v):
        r, _ = R.residual_norm(**v, scale=0.5, norm="layer")
        return float((r["sum"] * ds.double()).sum() + (r["normed"] * dh.double()).sum())

    on = {n: v.cuda() for n, v in t.items()}
    got = op("ResidualNormGrad", ds.cuda(), dh.cuda(), on.pop("x"), on.pop("f"), **on, residual_scale=0.5, norm="layer")
    for name, g in zip(GRADS, got):
        n = name[1:]
        way = rand(*t[n].shape, seed=99).double()
        slope = (value({**t, n: t[n].double() + u * way}) - value({**t, n: t[n].double() - u * way})) / (2 * u)
        terms = g.cpu().double() * way
        assert abs(float(terms.sum()) - slope) < 1e-4 * float(terms.abs().sum()) + 1e-6, name


def test_same_from_run_to_run_and_in_graphs():
    x, f = rand(4, 300, 256).cuda(), rand(4, 300, 256, dtype=BF, seed=1).cuda()
    kw = {"gamma": rand(256, seed=2).cuda(), "post_gamma": rand(256, seed=3).cuda(), "gate": rand(4, 1, 256, seed=4).cuda()}

    def step():
        return (*op("ResidualNorm", x, f, **kw), *[t for t in op("ResidualNormGrad", x, f, x, f, **kw) if t is not None])

    first = step()
    assert all(torch.equal(a, b) for a, b in zip(first, step()))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        res = step()
    x.neg_()
    want = step()
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, res))
