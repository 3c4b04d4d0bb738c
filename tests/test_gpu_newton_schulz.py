"""Newton-Schulz products and the optimizer step that uses them against 64 bits.

Tolerances, in the norm of a whole result (a step's products mix all entries). One step maps
a relative error e of X to at most |a| e |X| plus its own roundings. Measured in units of the
entries' size, an error of a small singular direction grows with the direction itself (by a
each step), so it keeps its share; only where |X| is carried by a few directions that have
stopped growing does its share grow, by at most a = 3.4445 a step for 5 steps. The inputs
below (noise over a part of rank min / 4) start within a factor 8 of a flat spectrum, so at
most the last two of the five steps are of that kind: a growth of a^2 < 12.
* fp32: a product of two-plane operands is off by 3 * 2^-22 of its terms and K / 16 + 2
  additions of 2^-23 each at most, of random sign (their square root counts): with K <= 4096
  16 * 2^-23 + 2^-20 = 3e-6 a product; three products a step, five steps, random sign:
  3e-6 sqrt(15) < 1.2e-5, times 12: 1.5e-4 at most; held to 3e-5 (an fp32 evaluation by
  elementary products measures 1e-6 to 5e-6 on these).
* bf16: fp16 iterates round by at most 2^-11, 2^-11 / sqrt(3) on average: 15 products of two
  such operands and the result's own rounding: 2.8e-4 sqrt(30) = 1.5e-3, times 12 at most;
  held to 6e-3, with 2^-8 / sqrt(3) for the bf16 result in it."""

import math

import pytest
import torch

import lm_reference as R

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
BOUND = {F32: 3e-5, BF: 6e-3}


@pytest.fixture(autouse=True)
def _device(cuda):
    yield


def op(name, *args, **kw):
    from b200.backend import B200Backend

    return B200Backend.execute_op(name, *args, **kw)


def grads(*shape, dtype=F32, seed=0, scale=1e-3):
    g = torch.Generator(device="cuda").manual_seed(seed + sum(shape))
    r = max(1, min(shape[-2:]) // 4)
    a = torch.randn(*shape[:-1], r, generator=g, device="cuda") @ torch.randn(*shape[:-2], r, shape[-1], generator=g, device="cuda")
    return ((a / r**0.5 + torch.randn(*shape, generator=g, device="cuda")) * scale).to(dtype)


def off(got, ref):
    return float((got.double() - ref).norm() / ref.norm())


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("shape", [(1, 1), (1, 7), (5, 1), (3, 3), (48, 48), (33, 130), (130, 33), (128, 128), (129, 257), (300, 77), (256, 1024),
                                   (1000, 520), (3, 64, 64), (2, 3, 40, 72), (5, 200, 136), (16, 256, 512), (2, 1024, 1024), (700, 4096)])
def test_newton_schulz(shape, dtype):
    g = grads(*shape, dtype=dtype)
    got = op("NewtonSchulz", g)
    assert got.shape == g.shape and got.dtype == dtype and torch.isfinite(got).all()
    assert off(got, R.newton_schulz(g.double())) <= BOUND[dtype]


def test_large_enough_for_cta_pairs():
    for shape in ((4, 1500, 1500), (2304, 2560), (2560, 2304), (12, 700, 900)):
        g = grads(*shape)
        assert off(op("NewtonSchulz", g), R.newton_schulz(g.double())) <= BOUND[F32]


def test_each_matrix_of_a_stack_is_its_own():
    g = grads(6, 96, 200)
    g[2] *= 1e6
    g[4] = 0
    got = op("NewtonSchulz", g)
    for i in range(6):
        assert torch.equal(got[i], op("NewtonSchulz", g[i]))
    assert not got[4].any()
    g[1, 5, 5] = float("nan")
    again = op("NewtonSchulz", g)
    assert torch.isnan(again[1]).all() and torch.equal(again[0], got[0]) and torch.equal(again[2:], got[2:])


def test_scale_layout_steps_and_coefficients():
    g = grads(64, 160)
    ref = R.newton_schulz(g.double())
    assert off(op("NewtonSchulz", g * 2.0**60), R.newton_schulz((g * 2.0**60).double())) <= BOUND[F32]
    tiny = g * 2.0**-60
    assert off(op("NewtonSchulz", tiny), R.newton_schulz(tiny.double())) <= BOUND[F32]
    assert off(op("NewtonSchulz", tiny, eps=0.0), ref) <= BOUND[F32]
    assert torch.equal(op("NewtonSchulz", g.t().contiguous().t()), op("NewtonSchulz", g))
    wide = torch.zeros(64, 321, device="cuda")
    wide[:, 1:161] = g
    assert torch.equal(op("NewtonSchulz", wide[:, 1:161]), op("NewtonSchulz", g))
    for steps in (1, 2, 8):
        assert off(op("NewtonSchulz", g, steps=steps), R.newton_schulz(g.double(), steps)) <= BOUND[F32]
    each = [[4.0, -6.9, 2.9], [3.9, -6.3, 2.6], [3.2, -4.4, 1.7], [1.5, -0.5, 0.0]]
    assert off(op("NewtonSchulz", g, steps=4, coefficients=each), R.newton_schulz(g.double(), 4, each)) <= BOUND[F32]
    # the cubic (c = 0) converges to the orthogonal factor itself
    q = op("NewtonSchulz", grads(32, 90), steps=40, coefficients=(1.5, -0.5, 0.0)).double()
    assert float((q @ q.mT - torch.eye(32, device="cuda")).abs().max()) <= 1e-5


@pytest.mark.parametrize("coef", [(2.0, -1.2, 0.01), (1.9, -1.0, 0.1), (1.2, 0.0, -0.2), (3.0, -3.2, 1.2), (1.0, 0.0, 0.0), (2.0, -1.5, 0.5)])
@pytest.mark.parametrize("shape", [(96, 150), (260, 200), (4, 520, 700)])
def test_small_missing_and_negative_coefficients(shape, coef):
    g = grads(*shape)
    got = op("NewtonSchulz", g, coefficients=coef)
    assert off(got, R.newton_schulz(g.double(), 5, coef)) <= BOUND[F32]
    tiny = (g * 2.0**-40).contiguous()
    assert off(op("NewtonSchulz", tiny, coefficients=coef), R.newton_schulz(tiny.double(), 5, coef)) <= BOUND[F32]


def test_extreme_spectra_stay_finite_and_near():
    """One direction far above the rest, equal directions, a rank of one."""
    u, v = torch.linalg.qr(torch.randn(64, 64, device="cuda"))[0], torch.linalg.qr(torch.randn(160, 64, device="cuda"))[0]
    for s in (torch.ones(64), torch.cat([torch.ones(1), torch.full((63,), 1e-3)]), torch.cat([torch.ones(1), torch.zeros(63)])):
        g = u * s.cuda() @ v.t()
        # the share of the small directions' errors may grow by a^5 here
        assert off(op("NewtonSchulz", g), R.newton_schulz(g.double())) <= 3e-6 * 3.4445**5
        assert off(op("NewtonSchulz", g.to(BF)), R.newton_schulz(g.to(BF).double())) <= 5e-2


@pytest.mark.parametrize("dtype,power", [(F32, -140), (F32, -126), (F32, -100), (F32, 100), (F32, 124), (BF, -120), (BF, -100), (BF, 124)])
def test_norms_beyond_fp32s_reciprocals(power, dtype):
    """1 / |g| or |g| itself outside fp32's normal range, eps = 0: the answer is g's times a power of two."""
    g = grads(70, 90)
    g = (g.double() / g.abs().max() * 2.0 ** (power + 3)).to(dtype)
    got = op("NewtonSchulz", g, eps=0.0)
    assert off(got, R.newton_schulz(g.double(), eps=0.0)) <= BOUND[dtype]


STACKS = [(50, 129, 200), (50, 200, 129), (20, 300, 520), (20, 520, 300), (50, 256, 256), (17, 257, 1030), (9, 770, 600)]


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("shape", STACKS)
@pytest.mark.parametrize("steps", [1, 2, 5])
def test_stacks_that_fill_the_gpu(shape, dtype, steps):
    """Every matrix of a stack, each of its own scale, against 64 bits and against the call of that matrix alone."""
    g = grads(*shape, dtype=dtype)
    g = (g * (2.0 ** (torch.arange(shape[0]) % 7 - 3).double()).to(dtype).cuda().view(-1, 1, 1)).contiguous()
    got = op("NewtonSchulz", g, steps=steps)
    ref = R.newton_schulz(g.double(), steps)
    assert max(off(got[i], ref[i]) for i in range(shape[0])) <= BOUND[dtype]
    for i in (0, shape[0] - 1):
        assert off(op("NewtonSchulz", g[i], steps=steps), got[i].double()) <= 2 * BOUND[dtype]
    assert torch.equal(op("NewtonSchulz", g, steps=steps), got)


def test_stacks_with_vanishing_matrices_and_own_coefficients():
    g = grads(20, 300, 520)
    g[3] *= 2.0**-60
    g[7] = 0
    g[11, 5, 9] = float("nan")
    coef = [(2.0, -1.5, 0.5), (3.0, -3.2, 1.2), (1.9, -1.0, 0.1)]
    got = op("NewtonSchulz", g, steps=3, coefficients=coef)
    ref = g.double() / (g.double().flatten(1).norm(dim=1).view(-1, 1, 1) + 1e-7)
    for a, b, c in coef:
        s = ref @ ref.transpose(1, 2)
        ref = a * ref + (b * s + c * s @ s) @ ref
    assert not got[7].any() and got[11].isnan().any()
    assert max(off(got[i], ref[i]) for i in range(20) if i not in (7, 11)) <= BOUND[F32]


@pytest.mark.parametrize("shape", [(20, 300, 520), (20, 520, 300)])
def test_stacks_on_two_streams_and_replayed(shape):
    """Two calls at once, an eager one beside a captured one; the counters start anew each time."""
    a, b = grads(*shape), grads(*shape, seed=4)
    wa, wb = op("NewtonSchulz", a), op("NewtonSchulz", b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cap = op("NewtonSchulz", a)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    outs = []
    for _ in range(4):
        graph.replay()
        with torch.cuda.stream(s):
            outs.append(op("NewtonSchulz", b))
    torch.cuda.synchronize()
    assert torch.equal(cap, wa) and all(torch.equal(o, wb) for o in outs)
    p, m = grads(*shape, seed=7, scale=0.02), grads(*shape, seed=8)
    want = op("ApplyMuon", p, m, a, lr=0.05, weight_decay=0.1)
    op("ApplyMuon", p, m, a, lr=0.05, weight_decay=0.1, out=(p, m))
    assert torch.equal(p, want[0]) and torch.equal(m, want[1])


def test_stacks_beside_each_other_and_a_loss():
    """Calls on six streams at once: each list of tiles advances with whatever CTAs it gets."""
    gs = [grads(*s) for s in ((16, 512, 700), (50, 256, 256), (7, 1024, 600), (20, 300, 520), (300, 200))]
    x, w = torch.randn(700, 512, device="cuda").to(BF), torch.randn(512, 9000, device="cuda").to(BF)
    labels = torch.arange(700, device="cuda") * 11
    want = [op("NewtonSchulz", g) for g in gs] + [op("LinearCrossEntropy", x, w, labels)[0]]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(6)]
    for turn in range(6):
        got = []
        for k, g in enumerate(gs):
            with torch.cuda.stream(streams[(k + turn) % 6]):
                got.append(op("NewtonSchulz", g))
        with torch.cuda.stream(streams[(5 + turn) % 6]):
            got.append(op("LinearCrossEntropy", x, w, labels)[0])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("shape", [(40, 24), (24, 40), (4, 256, 256), (1, 130), (1100, 300), (20, 300, 270)])
def test_apply_muon(shape, nesterov):
    g, m, p = grads(*shape), grads(*shape, seed=3), grads(*shape, seed=5, scale=0.02)
    kw = {"lr": 0.05, "momentum": 0.9, "nesterov": nesterov, "weight_decay": 0.1}
    p2, m2 = op("ApplyMuon", p, m, g, **kw)
    rm = 0.9 * m.double() + g.double()
    # two roundings of 2^-24 relative to the terms
    assert ((m2.double() - rm).abs() <= 2.0**-23 * (m.abs() + g.abs()).double()).all()
    o = R.newton_schulz(g.double() + 0.9 * rm if nesterov else rm)
    step = 0.05 * math.sqrt(max(1.0, shape[-2] / shape[-1])) * o
    err = p2.double() - (p.double() * (1 - 0.05 * 0.1) - step)
    # the products' error, and three roundings of 2^-24 of the terms
    assert float(err.norm()) <= BOUND[F32] * float(step.norm()) + 2.0**-22 * float(p.double().norm() + step.norm())
    # in place
    pc, mc = p.clone(), m.clone()
    op("ApplyMuon", pc, mc, g, out=(pc, mc), **kw)
    assert torch.equal(pc, p2) and torch.equal(mc, m2)


def test_apply_muon_refuses_results_over_other_inputs():
    p, m, g = (grads(16, 24, seed=i) for i in range(3))
    for out in ((m, p), (g, m), (p, g), (p, p), (p, torch.empty(24, 16, device="cuda")), (p.half(), m), (p, torch.empty(24, 16, device="cuda").t())):
        with pytest.raises(ValueError, match="ApplyMuon"):
            op("ApplyMuon", p, m, g, out=out)


def test_apply_muon_refuses_partial_overlaps():
    both = torch.zeros(3, 16, 24, device="cuda")
    flat = both.view(-1)
    g = grads(16, 24)
    n = 16 * 24
    ahead = flat[24 : 24 + n].view(16, 24)
    for out in ((ahead, both[2]), (both[0], flat[2 * n - 24 : 3 * n - 24].view(16, 24)), (both[2], ahead)):
        with pytest.raises(ValueError, match="own input only"):
            op("ApplyMuon", both[0], both[2], g, out=out)
    p, m = op("ApplyMuon", both[0], both[2], g, out=(both[0], both[1]))
    assert p.data_ptr() == both[0].data_ptr() and torch.equal(both[1], g) and m is not None


def test_muon_defaults_and_empty():
    p, m, g = torch.ones(8, 16, device="cuda"), torch.zeros(8, 16, device="cuda"), grads(8, 16)
    a = op("ApplyMuon", p, m, g)
    assert torch.equal(a[0], op("ApplyMuon", p, m, g, lr=0.02, momentum=0.95, nesterov=True)[0]) and torch.equal(a[1], g)
    for shape in ((0, 5), (5, 0), (0, 3, 4)):
        assert tuple(op("NewtonSchulz", torch.zeros(shape, device="cuda")).shape) == shape


def test_graph_capture_and_repeat():
    g = grads(2, 300, 520)
    want = op("NewtonSchulz", g)
    assert torch.equal(op("NewtonSchulz", g), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cap = op("NewtonSchulz", g)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = op("NewtonSchulz", g)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(cap, want) and torch.equal(other, want)
    g.copy_(grads(2, 300, 520, seed=9))
    graph.replay()
    assert torch.equal(cap, op("NewtonSchulz", g))
