"""Rotary positions and query / key norms on the GPU against their definitions in 64 bits.

Tolerances. The angle past the nearest quarter turn is a 32-bit integer turned into a float
and multiplied by 2 pi 2^-32: three roundings (integer, constant, product) of 2^-24 of at most
pi / 4, 1.4e-7. The Taylor polynomials are off by less than 2^-28 there, and by 2^-23 for their
last roundings, so cosine and sine are within 2.7e-7 and a rotated element within (|a| + |b|)
(2.7e-7 + 4 2^-24 for the factor, the products and the sum) < 6e-7 (|a| + |b|). The norm adds the fp32 sum of at most 512 squares over at most 16
elements a lane and a tree of 5 (21 roundings of 2^-24, halved by the root) and 5 roundings
of rsqrt and products: 1e-6 relative in all. So fp32 values are held to 2e-6 of their
terms' magnitude, and a result of fewer bits to half a step of its own value besides."""

import numpy as np
import pytest
import torch

import lm_reference as R

pytestmark = pytest.mark.gpu

TERMS = 2e-6
BF, F32 = torch.bfloat16, torch.float32
SCALINGS = [
    None,
    {"kind": "linear", "factor": 4.0},
    {"kind": "ntk", "factor": 4.0},
    {"kind": "yarn", "factor": 16.0, "original_length": 4096},
    {"kind": "yarn", "factor": 8.0, "original_length": 512, "beta_fast": 16.0, "beta_slow": 2.0, "attention_factor": 0.9},
    {"kind": "wavelength", "factor": 8.0, "original_length": 8192, "low_factor": 1.0, "high_factor": 4.0},
]


@pytest.fixture(autouse=True)
def _device(cuda):
    yield


def op(name, *args, **kw):
    from b200.backend import B200Backend

    return B200Backend.execute_op(name, *args, **kw)


def rand(*shape, dtype=F32, seed=0):
    g = torch.Generator().manual_seed(seed + sum(shape))
    return torch.randn(*shape, generator=g).to(dtype)


def close(got, ref, mag, what=""):
    got = got.cpu()
    tol = R.HALF_STEP[got.dtype] * ref.abs() + TERMS * mag
    bad = (got.double() - ref).abs() > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, most {float(((got.double() - ref).abs() / tol).max()):.3g} x"


@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape,part", [
    ((1, 1, 1, 2), 2), ((1, 1, 32, 128), 128), ((2, 37, 3, 64), 64), ((2, 5, 7, 80), 32), ((3, 33, 16, 96), 46),
    ((1, 17, 5, 512), 512), ((2, 9, 2, 256), 62), ((1, 300, 1, 33), 8), ((2, 4, 3, 48), 0), ((5, 1, 9, 81), 34),
    ((2, 70, 11, 128), 62), ((1, 9, 5, 32), 14), ((1, 6, 3, 511), 510), ((2, 3, 4, 512), 254), ((1, 5, 2, 4), 2), ((1, 4, 2, 512), 510), ((1, 3, 2, 512), 506),
])
def test_rotary_shapes(shape, part, dtype, interleaved, inverse):
    x = rand(*shape, dtype=dtype)
    pos = torch.arange(shape[1])[None] + torch.arange(shape[0])[:, None] * 1000
    kw = {"rotary_dim": part, "interleaved": interleaved}
    got = op("RotaryEmbeddingGrad" if inverse else "RotaryEmbedding", x.cuda(), pos.cuda(), **kw)
    assert got.dtype == dtype and tuple(got.shape) == shape
    close(got, *R.rotate(x.double(), pos, part, interleaved=interleaved, sign=-1 if inverse else 1))


@pytest.mark.parametrize("scaling", SCALINGS)
def test_rotary_scalings_and_far_positions(scaling):
    x = rand(1, 64, 4, 128)
    pos = torch.tensor([0, 1, -1, 7, 4095, 65536, 999_983, -123_456_789, 2**31 - 1, 2**40 + 3] + list(range(1000, 1054)))[None]
    got = op("RotaryEmbedding", x.cuda(), pos.cuda(), scaling=scaling, base=500000.0)
    # 64-bit angles of the farthest positions are themselves off by position * 2^-53: 2e-4 rad at 2^40
    near = (pos.abs() < 2**31)[0]
    ref, mag = R.rotate(x.double(), pos, 128, base=500000.0, scaling=scaling)
    close(got[:, near], ref[:, near], mag[:, near])


def test_rotary_layouts_positions_and_offset():
    x = rand(2, 12, 6, 64, dtype=BF)
    pos = torch.randint(0, 5000, (2, 12))
    want = op("RotaryEmbedding", x.cuda(), pos.cuda())
    # head-major storage, an unaligned slice, a strided slice, adjacent elements not adjacent in memory
    hm = x.cuda().transpose(1, 2).contiguous().transpose(1, 2)
    got = op("RotaryEmbedding", hm, pos.cuda())
    assert got.stride() == hm.stride()
    buf = torch.zeros(2 * 12 * 6 * 64 + 1, dtype=BF, device="cuda")
    off = buf[1:].view(2, 12, 6, 64)
    off.copy_(x)
    wide = torch.zeros(2, 12, 18, 64, dtype=BF, device="cuda")
    wide[:, :, 6:12] = x.cuda()
    turned = x.cuda().permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0)
    for y in (got, op("RotaryEmbedding", off, pos.cuda()), op("RotaryEmbedding", wide[:, :, 6:12], pos.cuda()),
              op("RotaryEmbedding", turned, pos.cuda()), op("RotaryEmbedding", x.numpy() if x.dtype != BF else x, pos),
              op("RotaryEmbedding", x.cuda(), pos.int().cuda()), op("RotaryEmbedding", x.cuda(), pos.cuda().t().contiguous().t())):
        assert torch.equal(y, want)
    # one position row for all sequences, positions by offset, no batch axis, a broadcast input
    row = op("RotaryEmbedding", x.cuda(), torch.arange(12).cuda() + 77)
    assert torch.equal(row, op("RotaryEmbedding", x.cuda(), offset=77))
    assert torch.equal(row, op("RotaryEmbedding", x.cuda(), (torch.arange(12) + 77)[None].cuda()))
    assert torch.equal(row[1], op("RotaryEmbedding", x[1].cuda(), offset=77))
    same = x[:1].cuda().expand(2, -1, -1, -1)
    assert torch.equal(op("RotaryEmbedding", same, offset=77)[1], row[0])


def test_rotary_gradient_is_the_transpose():
    """<R x, y> = <x, R^T y>, with the attention factor."""
    kw = {"scaling": SCALINGS[3], "rotary_dim": 32}
    x, y = rand(2, 40, 3, 48), rand(2, 40, 3, 48, seed=5)
    a = (op("RotaryEmbedding", x.cuda(), **kw).double().cpu() * y.double()).sum()
    b = (x.double() * op("RotaryEmbeddingGrad", y.cuda(), **kw).double().cpu()).sum()
    terms = float((x.abs().double() * y.abs().double()).sum())
    assert abs(float(a - b)) <= 4 * TERMS * terms


def test_rotary_empty():
    for shape in ((0, 4, 2, 64), (2, 0, 2, 64), (2, 4, 0, 64)):
        assert tuple(op("RotaryEmbedding", torch.zeros(shape, device="cuda")).shape) == shape
    q, k = torch.zeros(2, 0, 4, 64, device="cuda"), torch.zeros(2, 0, 1, 64, device="cuda")
    g = op("QKNormRotaryGrad", q, k, q, k)
    assert not g[2].any() and not g[3].any()


QK = [  # batch, seq, heads, kv_heads, dim, rotary_dim
    (1, 1, 1, 1, 64, 64), (32, 1, 32, 8, 128, 128), (2, 65, 4, 1, 128, 64), (3, 7, 5, 2, 80, 32), (1, 19, 3, 3, 46, 46),
    (2, 11, 2, 2, 512, 512), (4, 3, 6, 2, 33, 0), (1, 700, 8, 2, 64, 64), (2, 5, 3, 1, 256, 130),
    (2, 30, 11, 3, 96, 46), (1, 9, 7, 2, 128, 62), (3, 5, 4, 4, 32, 14), (1, 4, 9, 2, 512, 254), (1, 3, 2, 1, 511, 510), (1, 4, 2, 1, 512, 510), (1, 2, 3, 2, 509, 508),
]


def qk_inputs(b, n, h, hk, d, dtype, seed=1):
    q, k = rand(b, n, h, d, dtype=dtype, seed=seed), rand(b, n, hk, d, dtype=dtype, seed=seed + 1) * 3
    gq, gk = 1 + 0.2 * rand(d, seed=seed + 2), 1 + 0.2 * rand(d, seed=seed + 3)
    pos = torch.arange(n)[None] + 100 * torch.arange(b)[:, None]
    return q, k, gq, gk, pos


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("size", QK)
def test_qk_norm_rotary(size, dtype, interleaved):
    *shape, part = size
    q, k, gq, gk, pos = qk_inputs(*shape, dtype)
    got = op("QKNormRotary", q.cuda(), k.cuda(), gq.cuda(), gk.cuda(), pos.cuda(), rotary_dim=part, interleaved=interleaved)
    for y, x, g in zip(got, (q, k), (gq, gk)):
        u = R.rms_unit(x.double(), 1e-6)[0] * g.double()
        close(y, *R.rotate(u, pos, part, interleaved=interleaved))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("size", QK)
def test_qk_norm_rotary_grad(size, dtype, interleaved):
    *shape, part = size
    b, n, h, hk, d = shape
    q, k, gq, gk, pos = qk_inputs(*shape, dtype)
    dq, dk = rand(b, n, h, d, dtype=dtype, seed=8), rand(b, n, hk, d, dtype=dtype, seed=9)
    kw = {"rotary_dim": part, "interleaved": interleaved, "scaling": SCALINGS[3] if part else None}
    got = op("QKNormRotaryGrad", dq.cuda(), dk.cuda(), q.cuda(), k.cuda(), gq.cuda(), gk.cuda(), pos.cuda(), **kw)
    for dx, dg, x, g, dy in zip(got[:2], got[2:], (q, k), (gq, gk), (dq, dk)):
        gr, mag = R.rotate(dy.double(), pos, part, interleaved=interleaved, scaling=kw["scaling"], sign=-1)
        u, rstd = R.rms_unit(x.double(), 1e-6)
        hgr = gr * g.double()
        ref = rstd * (hgr - u * (hgr * u).mean(-1, keepdim=True))
        # the terms of the difference, each within TERMS of its magnitude
        m = mag * g.abs().double()
        close(dx, ref, rstd * (m + u.abs() * (m * u.abs()).mean(-1, keepdim=True)) * 2, "dx")
        # a sum of b n heads terms in fp32: a lane adds at most all of them in order
        terms = (mag * u.abs()).sum((0, 1, 2))
        count = x.shape[0] * x.shape[1] * x.shape[2]
        tol = terms * (TERMS + 2.0**-24 * min(count, 4096))
        assert ((dg.cpu().double() - (gr * u).sum((0, 1, 2))).abs() <= tol).all()


def test_qk_grad_against_differences():
    """Directional derivatives by central differences of the 64-bit forward."""
    b, n, h, hk, d = 1, 6, 2, 1, 32
    q, k, gq, gk, pos = qk_inputs(b, n, h, hk, d, F32)
    dq, dk = rand(b, n, h, d, seed=8), rand(b, n, hk, d, seed=9)

    def value(x, g, dy):
        return float((R.rotate(R.rms_unit(x, 1e-6)[0] * g, pos, d)[0] * dy.double()).sum())

    got = [t.cpu().double() for t in op("QKNormRotaryGrad", dq.cuda(), dk.cuda(), q.cuda(), k.cuda(), gq.cuda(), gk.cuda(), pos.cuda())]
    step = 1e-5
    for x, g, dy, dx, dg in ((q, gq, dq, got[0], got[2]), (k, gk, dk, got[1], got[3])):
        v, w = rand(*x.shape, seed=20).double(), rand(d, seed=21).double()
        num = (value(x.double() + step * v, g.double(), dy) - value(x.double() - step * v, g.double(), dy)) / (2 * step)
        # differences are exact to step^2 and 2^-53 / step: 1e-8 of the terms
        assert abs(num - float((dx * v).sum())) <= 1e-5 * float((dx.abs() * v.abs()).sum())
        num = (value(x.double(), g.double() + step * w, dy) - value(x.double(), g.double() - step * w, dy)) / (2 * step)
        assert abs(num - float((dg * w).sum())) <= 1e-5 * float((dg.abs() * w.abs()).sum())


def test_qk_packed_projection_bf16_weights_and_defaults():
    qkv = rand(2, 30, 12, 64, dtype=BF).cuda()
    q, k = qkv[:, :, :8], qkv[:, :, 8:10]
    gq, gk = (1 + 0.1 * rand(64)).to(BF).cuda(), (1 + 0.1 * rand(64, seed=3)).cuda()
    a = op("QKNormRotary", q, k, gq, gk)
    b = op("QKNormRotary", q.contiguous(), k.contiguous(), gq.float(), gk)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    one = torch.ones(64, device="cuda")
    a, b = op("QKNormRotary", q, k), op("QKNormRotary", q, k, one, one)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    only = op("QKNormRotary", q, k, gq, None, rotary_dim=0)
    assert torch.equal(only[0], op("QKNormRotary", q, k, gq, gk, torch.zeros(30, dtype=torch.int64).cuda())[0])
    dq, dk = torch.ones_like(q), torch.ones_like(k)
    g1 = op("QKNormRotaryGrad", dq, dk, q, k, gq, gk)
    g2 = op("QKNormRotaryGrad", dq, dk, q, k, gq, gk)
    assert all(torch.equal(x, y) for x, y in zip(g1, g2))


def test_qk_zero_rows_and_nan_rows_stay_apart():
    q, k, gq, gk, pos = qk_inputs(1, 8, 4, 2, 64, F32)
    q[0, 3, 2] = 0
    clean = op("QKNormRotary", q.cuda(), k.cuda(), gq.cuda(), gk.cuda())
    assert not clean[0][0, 3, 2].any()
    q[0, 5, 1, 7] = float("nan")
    y = op("QKNormRotary", q.cuda(), k.cuda(), gq.cuda(), gk.cuda())
    hit = torch.isnan(y[0]).any(-1).cpu()
    assert hit[0, 5, 1] and int(hit.sum()) == 1
    y[0][0, 5, 1] = clean[0][0, 5, 1]
    assert torch.equal(y[0], clean[0]) and torch.equal(y[1], clean[1])


def test_rotary_stream_and_graph_capture():
    q, k, gq, gk, pos = (t.cuda() for t in qk_inputs(2, 50, 4, 2, 128, BF))
    want = op("QKNormRotary", q, k, gq, gk, pos)
    grads = op("QKNormRotaryGrad", *want, q, k, gq, gk, pos)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = op("QKNormRotary", q, k, gq, gk, pos)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(other[0], want[0]) and torch.equal(other[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cap = op("QKNormRotary", q, k, gq, gk, pos)
        cgr = op("QKNormRotaryGrad", *cap, q, k, gq, gk, pos)
    for scale in (1.0, 0.5):
        q2 = (q.float() * scale).to(BF)
        q.copy_(q2)
        graph.replay()
        torch.cuda.synchronize()
        now = op("QKNormRotary", q, k, gq, gk, pos)
        now_g = op("QKNormRotaryGrad", *now, q, k, gq, gk, pos)
        assert all(torch.equal(x, y) for x, y in zip((*cap, *cgr), (*now, *now_g)))
    assert len(grads) == 4


def test_rotary_long_tensor_passes_32_bit_offsets():
    """2^31 elements and more behind one stride: the last token of the second sequence."""
    far = torch.empty(2**31 + 4096, dtype=BF, device="cuda")
    x = far.as_strided((2, 2, 4, 64), (2**31, 256, 64, 1))
    small = rand(2, 2, 4, 64, dtype=BF).cuda()
    x.copy_(small)
    assert torch.equal(op("RotaryEmbedding", x, offset=9), op("RotaryEmbedding", small, offset=9))
