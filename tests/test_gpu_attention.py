"""Attention without the scores in memory, and its gradient, against the 64-bit forms on the CPU.

Tolerances. A score is a sum of up to 256 products in fp32 (a tree over 32 lanes of 8 at most, or
tensor-core sums of 16: below 20 roundings or cuts of 2^-23) and four more roundings up to its
exponential, so with mag the terms' magnitudes (a score's error moves its probability by as much) a
result is off by 24 x 2^-23 = 3e-6 of its terms, doubled in the gradients, whose factor is a difference of two
such sums, and doubled again for sums over up to 2^12 tokens: 1e-5. bf16 heads may round the
probabilities (out, dv), the output (so delta = dout . out) and dz before their products: two half
steps of 2^-8 of the terms, and the result's own. Those roundings are independent and of 2^-8 / sqrt(3) at
most in the mean square, so over a whole result the error is below sqrt(3 (2^-8)^2 / 3) = 2^-8
of the norm of the terms."""

import math

import pytest
import torch

import block_reference as R

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
TERMS = 1e-5


@pytest.fixture(autouse=True)
def _device(cuda):
    yield


def op(name, *args, **kw):
    from b200.backend import B200Backend

    return B200Backend.execute_op(name, *args, **kw)


def rand(*shape, dtype=F32, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed + sum(shape))
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def close(got, ref, mag, heads, what=""):
    """heads: the heads' type, whose roundings inside are allowed for."""
    got = got.cpu()
    assert torch.equal(got.isinf(), ref.isinf()) and not got.isnan().any(), what
    fine = ~ref.isinf()
    inner = 2 * R.HALF_STEP[BF] if heads == BF and what != "lse" else 0.0
    tol = R.HALF_STEP[got.dtype] * ref.abs() + (TERMS + inner) * mag + 1e-30
    off = (got.double() - ref).abs()
    bad = (off > tol) & fine
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, most {float((off / tol)[fine].max()):.3g} x"
    if heads == BF and what != "lse" and ref.numel() > 256:
        norm = float(off[fine].norm() / (mag[fine].norm() + 1e-30))
        assert norm < 2.0**-8, f"{what}: {norm:.3g} of the terms' norm"


def check(q, k, v, dout=None, table=None, **kw):
    on = {n: t.cuda() if isinstance(t, torch.Tensor) else t for n, t in kw.items() if n not in ("scale_of",)}
    tc = None if table is None else table.cuda()
    out, lse = op("Attention", q.cuda(), k.cuda(), v.cuda(), relative_bias=tc, **on)
    far = kw.get("max_distance", 128)
    ref_kw = {n: t for n, t in kw.items() if n != "max_distance"}
    ref, mag = R.attention(q, k, v, dout, table=table, far=far, **ref_kw)
    assert out.dtype == q.dtype and lse.dtype == F32 and out.is_contiguous()
    close(out, ref["out"], mag["out"], q.dtype, "out")
    close(lse, ref["lse"], mag["lse"], q.dtype, "lse")
    if dout is None:
        return out, lse
    grads = op("AttentionGrad", dout.cuda(), q.cuda(), k.cuda(), v.cuda(), out, lse, relative_bias=tc, **on)
    for got, name in zip(grads, ("dq", "dk", "dv", "dtable")):
        if name == "dtable" and table is None:
            assert got is None
            continue
        close(got, ref[name], mag[name], q.dtype, name)
    return out, lse, *grads


def inputs(b, nq, nk, h, hk, d, dtype, seed=0):
    return (rand(b, nq, h, d, dtype=dtype, seed=seed), rand(b, nk, hk, d, dtype=dtype, seed=seed + 1), rand(b, nk, hk, d, dtype=dtype, seed=seed + 2),
            rand(b, nq, h, d, dtype=dtype, seed=seed + 3))


SHAPES = [  # batch, queries, keys, heads, key heads, dim
    (1, 1, 1, 1, 1, 1), (1, 1, 1, 2, 1, 8), (2, 3, 5, 3, 3, 16), (1, 17, 33, 4, 2, 33), (2, 64, 64, 2, 2, 64), (1, 129, 257, 2, 1, 64),
    (1, 200, 131, 4, 1, 80), (2, 128, 128, 2, 1, 128), (1, 300, 300, 1, 1, 96), (1, 70, 190, 5, 5, 127), (1, 33, 65, 2, 1, 130),
    (1, 40, 70, 2, 2, 256), (3, 1, 700, 8, 2, 64), (1, 2, 1500, 6, 1, 128), (1, 5, 900, 3, 1, 200), (2, 1, 300, 1, 1, 40),
    (1, 385, 513, 2, 2, 32), (1, 259, 4, 2, 1, 64), (1, 40, 40, 2, 1, 1), (1, 50, 50, 2, 2, 8), (1, 33, 47, 2, 1, 65), (1, 16, 1, 1, 1, 64),
]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape", SHAPES)
def test_shapes(shape, dtype, causal):
    check(*inputs(*shape, dtype), causal=causal)


@pytest.mark.parametrize("causal,window,lengths", [(True, None, None), (False, 1500, [2100, 40]), (True, 700, [0, 1999]), (False, None, None)])
@pytest.mark.parametrize("nq,h,hk,dim", [(16, 4, 1, 128), (33, 8, 8, 64), (100, 2, 1, 40), (292, 2, 1, 64), (293, 2, 1, 64)])
def test_few_queries_of_long_keys(nq, h, hk, dim, causal, window, lengths):
    q, k, v, do = inputs(2, nq, 2100, h, hk, dim, BF)
    lengths = lengths and torch.tensor(lengths)
    check(q, k, v, do, lengths=lengths, causal=causal, window=window)
    check(q, k, v, do, table=rand(32, h, dtype=BF, seed=9), lengths=lengths, causal=causal, window=window, max_distance=300)


@pytest.mark.parametrize("table_type", [BF, F32])
@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("causal,window", [(True, None), (False, 90), (True, 33)])
def test_everything_at_once(causal, window, dim, table_type):
    """Bias of either type, padding of both sides, shared heads, windows; forward and gradients on the tensor cores."""
    b, nq, nk = 6, 190, 270
    q, k, v, do = inputs(b, nq, nk, 4, 2, dim, BF)
    lengths, queries = torch.tensor([0, 70, 128, 270, 200, 64]), torch.tensor([190, 1, 64, 190, 0, 128])
    for e in range(b):
        k[e, lengths[e]:] = v[e, lengths[e]:] = math.nan
        q[e, queries[e]:] = do[e, queries[e]:] = math.nan
    check(q, k, v, do, table=rand(32, 4, dtype=table_type, seed=9), lengths=lengths, query_lengths=queries, causal=causal, window=window,
          max_distance=60)


@pytest.mark.parametrize("causal,window", [(True, 1), (True, 40), (False, 1), (False, 33), (True, 5000), (False, 5000)])
@pytest.mark.parametrize("dtype,dim", [(BF, 64), (BF, 128), (F32, 64), (BF, 192)])
@pytest.mark.parametrize("nq,nk", [(150, 150), (20, 300), (260, 100), (1, 77)])
def test_windows(nq, nk, dtype, dim, causal, window):
    check(*inputs(1, nq, nk, 2, 1, dim, dtype), causal=causal, window=window)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype,dim", [(BF, 64), (BF, 128), (F32, 80), (F32, 144)])
def test_padded_batch(dtype, dim, causal):
    """Lengths of zero, one, a tile and all; what lies behind them is NaN and is never read."""
    b, nq, nk = 7, 190, 270
    q, k, v, do = inputs(b, nq, nk, 4, 2, dim, dtype)
    lengths, queries = torch.tensor([0, 1, 128, 270, 200, 64, 129]), torch.tensor([190, 1, 64, 190, 0, 128, 65])
    for e in range(b):
        k[e, lengths[e]:] = v[e, lengths[e]:] = math.nan
        q[e, queries[e]:] = do[e, queries[e]:] = math.nan
    got = check(q, k, v, do, lengths=lengths, query_lengths=queries, causal=causal)
    out, lse, dq, dk, dv, _ = got
    for e in range(b):
        assert not out[e, queries[e]:].any() and (lse[e, :, queries[e]:] == -math.inf).all() and not dq[e, queries[e]:].any()
        assert not dk[e, lengths[e]:].any() and not dv[e, lengths[e]:].any()
    # 32-bit lengths, lengths of one side alone
    again = op("Attention", q.cuda(), k.cuda(), v.cuda(), lengths=lengths.int().cuda(), query_lengths=queries.cuda(), causal=causal)
    assert torch.equal(again[0], out)
    check(*inputs(b, nq, nk, 4, 2, dim, dtype), lengths=lengths, causal=causal)
    check(*inputs(b, nq, nk, 4, 2, dim, dtype), query_lengths=queries, causal=causal)


def test_decode_from_caches():
    q, k, v, _ = inputs(5, 1, 3000, 8, 2, 128, BF)
    lengths = torch.tensor([1, 2999, 3000, 17, 0])
    for e in range(5):
        k[e, lengths[e]:] = v[e, lengths[e]:] = math.inf
    out, lse = check(q, k, v, lengths=lengths, causal=True)
    assert not out[4].any() and (lse[4] == -math.inf).all()
    # the same token as the last of its own prompt
    qa, ka, va, _ = inputs(1, 300, 300, 8, 2, 128, BF, seed=5)
    whole, l0 = op("Attention", qa.cuda(), ka.cuda(), va.cuda(), causal=True)
    one, l1 = op("Attention", qa[:, -1:].cuda(), ka.cuda(), va.cuda(), causal=True)
    ref, mag = R.attention(qa, ka, va, causal=True)
    close(whole, ref["out"], mag["out"], BF, "out")
    close(one, ref["out"][:, -1:], mag["out"][:, -1:], BF, "out")
    assert (l0[:, :, -1:] - l1).abs().max() < 1e-5


@pytest.mark.parametrize("buckets,far,bidirectional", [(32, 128, True), (32, 128, False), (4, 3, True), (256, 1024, True), (8, 20, False)])
@pytest.mark.parametrize("dtype,dim,h,hk", [(BF, 64, 4, 4), (BF, 128, 4, 2), (F32, 40, 2, 1)])
@pytest.mark.parametrize("nq,nk,causal", [(200, 200, True), (150, 390, False), (1, 500, True)])
def test_position_bias(nq, nk, causal, dtype, dim, h, hk, buckets, far, bidirectional):
    table = rand(buckets, h, dtype=dtype, seed=9)
    check(*inputs(2, nq, nk, h, hk, dim, dtype), table=table, causal=causal, max_distance=far, bidirectional=bidirectional)


def test_position_bias_that_hides_and_padding():
    table = rand(16, 4, dtype=BF, seed=9)
    table[3] = -math.inf  # hides some distances, and for one head all
    table[:, 1] = -math.inf
    table[5, 0] = 40.0
    q, k, v, do = inputs(3, 100, 140, 4, 2, 64, BF)
    lengths, queries = torch.tensor([140, 90, 5]), torch.tensor([100, 50, 5])
    out = check(q, k, v, do, table=table, lengths=lengths, query_lengths=queries, max_distance=30)
    assert not out[0][:, :, 1].any() and not out[2][:, :, 1].any()
    # the type's lowest value is a number: a row of nothing else is a plain mean
    low = torch.full((16, 4), torch.finfo(BF).min, dtype=BF)
    got, _ = op("Attention", q.cuda(), k.cuda(), v.cuda(), relative_bias=low.cuda(), max_distance=30)
    mean = v.double().mean(1, keepdim=True).repeat_interleave(2, 2).expand(3, 100, 4, 64)
    assert (got.cpu().double() - mean).abs().max() < 2.0**-8 * 4


@pytest.mark.parametrize("dtype", [BF, F32])
def test_layouts(dtype):
    q, k, v, do = inputs(2, 70, 90, 4, 2, 64, dtype)
    ref = op("Attention", q.cuda(), k.cuda(), v.cuda(), causal=True)
    gref = op("AttentionGrad", do.cuda(), q.cuda(), k.cuda(), v.cuda(), *ref, causal=True)

    def head_major(t):
        return t.cuda().transpose(1, 2).contiguous().transpose(1, 2)

    def sliced(t):
        wide = torch.full((*t.shape[:2], t.shape[2] + 3, t.shape[3]), math.nan, dtype=dtype, device="cuda")
        wide[:, :, 2 : 2 + t.shape[2]] = t.cuda()
        return wide[:, :, 2 : 2 + t.shape[2]]

    def unaligned(t):
        flat = torch.zeros(t.numel() + 1, dtype=dtype, device="cuda")
        flat[1:].view(t.shape).copy_(t)
        return flat[1:].view(t.shape)

    def odd_rows(t):
        wide = torch.full((*t.shape[:3], t.shape[3] + 1), math.nan, dtype=dtype, device="cuda")
        wide[..., : t.shape[3]] = t.cuda()
        return wide[..., : t.shape[3]]

    def turned(t):
        return t.cuda().permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0)

    for way in (head_major, sliced, unaligned, odd_rows, turned):
        got = op("Attention", way(q), way(k), way(v), causal=True)
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1]), way.__name__
        grads = op("AttentionGrad", way(do), way(q), way(k), way(v), *got, causal=True)
        assert all(torch.equal(x, y) for x, y in zip(grads[:3], gref[:3])), way.__name__
    # without the batch axis; one key and value for every sequence
    one = op("Attention", q[0].cuda(), k[0].cuda(), v[0].cuda(), causal=True)
    assert torch.equal(one[0], ref[0][0]) and torch.equal(one[1], ref[1][0])
    gone = op("AttentionGrad", do[0].cuda(), q[0].cuda(), k[0].cuda(), v[0].cuda(), *one, causal=True)
    assert all(torch.equal(x, y[0]) for x, y in zip(gone[:3], gref[:3])) and gone[3] is None
    ks, vs = k[:1].cuda().expand(2, -1, -1, -1), v[:1].cuda().expand(2, -1, -1, -1)
    shared = op("Attention", q.cuda(), ks, vs, causal=True)
    assert torch.equal(shared[0][0], ref[0][0])
    close(shared[0], *(t["out"] for t in R.attention(q, k[:1].expand(2, -1, -1, -1), v[:1].expand(2, -1, -1, -1), causal=True)), dtype, "out")


@pytest.mark.parametrize("dtype", [BF, F32])
def test_large_scores_and_scale(dtype):
    """Scores of some hundreds: the running maximum moves and most probabilities are zero."""
    q, k, v, do = inputs(1, 150, 300, 2, 1, 64, dtype)
    k = k * torch.linspace(0.1, 12, 300)[None, :, None, None].to(dtype)
    check(q, k, v, scale=1.0)
    check(q, k, v, scale=1e-3)
    check(*inputs(1, 150, 300, 2, 1, 64, dtype), scale=0.5)


def test_nothing_to_do():
    q, k, v, do = inputs(2, 5, 0, 2, 1, 64, BF)
    out, lse = op("Attention", q.cuda(), k.cuda(), v.cuda())
    assert not out.any() and (lse == -math.inf).all()
    table = rand(8, 2, dtype=BF).cuda()
    dq, dk, dv, dt = op("AttentionGrad", do.cuda(), q.cuda(), k.cuda(), v.cuda(), out, lse, relative_bias=table)
    assert not dq.any() and dk.numel() == 0 and dv.numel() == 0 and not dt.any() and dt.shape == table.shape
    q, k, v, do = inputs(2, 0, 5, 2, 1, 64, BF)
    out, lse = op("Attention", q.cuda(), k.cuda(), v.cuda())
    dq, dk, dv, _ = op("AttentionGrad", do.cuda(), q.cuda(), k.cuda(), v.cuda(), out, lse)
    assert out.numel() == 0 and not dk.any() and not dv.any() and dk.shape == k.shape
    q, k, v, do = inputs(0, 4, 5, 2, 1, 64, BF)
    out, lse = op("Attention", q.cuda(), k.cuda(), v.cuda())
    assert out.numel() == 0 and all(t.numel() == 0 for t in op("AttentionGrad", do.cuda(), q.cuda(), k.cuda(), v.cuda(), out, lse)[:3])


def test_gradient_against_differences():
    """The gradients of sum(out dout) by central differences of the 64-bit forward, along one direction an input."""
    q, k, v, do = inputs(1, 40, 50, 4, 2, 32, F32)
    table = rand(16, 4, seed=9)
    out = check(q, k, v, do, table=table, causal=True, max_distance=20)
    grads = dict(zip("qkvt", out[2:]))
    named = {"q": q, "k": k, "v": v, "t": table}

    def value(**moved):
        x = {**named, **moved}
        r, _ = R.attention(x["q"], x["k"], x["v"], table=x["t"], causal=True, far=20)
        return float((r["out"] * do.double()).sum())

    for n, t in named.items():
        u = rand(*t.shape, seed=77).double()
        step = 1e-5
        slope = (value(**{n: t.double() + step * u}) - value(**{n: t.double() - step * u})) / (2 * step)
        got = float((grads[n].cpu().double() * u).sum())
        # fp32 gradients: TERMS of every term; the differences themselves 1e-8 of the value's
        assert abs(got - slope) < 1e-4 * float((grads[n].cpu().double() * u).abs().sum()) + 1e-6


@pytest.mark.parametrize("dtype,dim", [(BF, 64), (BF, 128), (F32, 64)])
def test_same_from_run_to_run_and_in_graphs(dtype, dim):
    q, k, v, do = (t.cuda() for t in inputs(2, 300, 300, 4, 2, dim, dtype))
    table = rand(32, 4, dtype=dtype).cuda()

    def step(x):
        out, lse = op("Attention", x, k, v, causal=True, relative_bias=table)
        return (out, lse, *op("AttentionGrad", do, x, k, v, out, lse, causal=True, relative_bias=table))

    first = step(q)
    assert all(torch.equal(x, y) for x, y in zip(first, step(q)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(q)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(first, other))
    still = q.clone()
    graphs = []
    for _ in range(2):  # two captured steps that replay in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = step(still)
        graphs.append((g, res))
    still.copy_(q.flip(1))
    want = step(still)
    for g, _ in graphs:
        g.replay()
    torch.cuda.synchronize()
    for _, res in graphs:
        assert all(torch.equal(x, y) for x, y in zip(want, res))


def test_lengths_outside_are_clamped_and_flagged():
    from b200 import _lib as L

    q, k, v, _ = (t.cuda() for t in inputs(2, 30, 40, 2, 1, 64, BF))
    L.lib().b200_check_device_error(None)
    want = op("Attention", q, k, v)
    assert L.lib().b200_check_device_error(None) == 0
    got = op("Attention", q, k, v, lengths=torch.tensor([41, 2**31 - 1]).cuda())
    assert torch.equal(got[0], want[0]) and L.lib().b200_check_device_error(None) != 0
    empty = op("Attention", q, k, v, lengths=torch.tensor([-1, -(2**31)]).cuda())
    assert not empty[0].any() and L.lib().b200_check_device_error(None) != 0
    assert L.lib().b200_check_device_error(None) == 0


@pytest.mark.parametrize("b,n,h,hk,d,causal,bias,window", [
    (8, 1000, 16, 16, 64, False, True, None), (16, 512, 16, 16, 64, False, False, None), (4, 2048, 16, 4, 128, True, False, None),
    (2, 3001, 8, 8, 128, False, True, None), (4, 1537, 8, 2, 64, True, False, 300), (2, 1200, 8, 8, 80, True, True, None),
])
def test_many_tiles_on_a_full_gpu(b, n, h, hk, d, causal, bias, window):
    """Thousands of blocks whose warps drift apart: the same bits every time, no wait given up, and within a half step (2^-8) of the
    64-bit results' terms in the mean square (made here, on the GPU)."""
    from b200 import _lib as L

    g = torch.Generator(device="cuda").manual_seed(n)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(BF)  # noqa: E731
    q, k, v, do, table = r(b, n, h, d), r(b, n, hk, d), r(b, n, hk, d), r(b, n, h, d), r(32, h)
    kw = {"causal": causal, "relative_bias": table if bias else None, "window": window}
    L.lib().b200_check_device_error(None)
    out, lse = op("Attention", q, k, v, **kw)
    grads = op("AttentionGrad", do, q, k, v, out, lse, **kw)
    for _ in range(8):
        again = op("Attention", q, k, v, **kw)
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)
        assert all(x is None or torch.equal(x, y) for x, y in zip(op("AttentionGrad", do, q, k, v, out, lse, **kw), grads))
    assert L.lib().b200_check_device_error(None) == 0
    where = R.bias_buckets(n, n, 0, 32, 128, not causal).cuda() if bias else None
    seen = R.seen_keys(n, n, causal, window).cuda()
    e, dk, dv = b - 1, torch.zeros(n, d, dtype=torch.float64, device="cuda"), torch.zeros(n, d, dtype=torch.float64, device="cuda")
    kv = hk - 1

    def near(got, ref):
        assert float((got.double() - ref).norm() / ref.norm()) < 2.0**-8

    for a in range(kv * (h // hk), h):  # the last key head of the last sequence
        Q, K, V, D = q[e, :, a].double(), k[e, :, kv].double(), v[e, :, kv].double(), do[e, :, a].double()
        z = Q @ K.t() / math.sqrt(d)
        if bias:
            z = z + table[:, a].double()[where]
        z = z.masked_fill(~seen, -math.inf)
        p = z.softmax(-1)
        o = p @ V
        near(out[e, :, a], o)
        assert (lse[e, a] - z.logsumexp(-1)).abs().max() < 1e-4
        dz = p * (D @ V.t() - (D * o).sum(-1, keepdim=True))
        near(grads[0][e, :, a], dz @ K / math.sqrt(d))
        dk += dz.t() @ Q / math.sqrt(d)
        dv += p.t() @ D
    near(grads[1][e, :, kv], dk)
    near(grads[2][e, :, kv], dv)
