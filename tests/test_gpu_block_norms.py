"""The attention kernels (both families) and the residual norms against 64 bits in the mean square: results, gradients and the bias
table's gradient within the roundings that the kernels make (rounding_norms.py), for each head and each row of it."""

import math

import pytest
import torch

import block_reference as R
import rounding_norms as N

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _device(cuda):
    yield


def op(name, *args, **kw):
    from b200.backend import B200Backend

    return B200Backend.execute_op(name, *args, **kw)


def rand(*shape, dtype=F32, seed=0, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed + sum(shape))
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype)


def check(q, k, v, do, **kw):
    ref, var = N.attention_noise(q, k, v, do, **kw)
    table, far = kw.pop("table", None), kw.pop("far", 128)
    on = {n: t.cuda() if isinstance(t, torch.Tensor) else t for n, t in kw.items()}
    on.update(relative_bias=None if table is None else table.cuda(), max_distance=far)
    out, lse = op("Attention", q.cuda(), k.cuda(), v.cuda(), **on)
    grads = op("AttentionGrad", do.cuda(), q.cuda(), k.cuda(), v.cuda(), out, lse, **on)
    wrong = []
    for name, got in zip(("out", "dq", "dk", "dv", "dtable"), (out, *grads)):
        if got is not None:
            off = N.attention_off(name, got, ref, var)
            wrong += [f"{name}: {off}"] if off else []
    assert not wrong, wrong


def inputs(b, nq, nk, h, hk, d, dtype, seed=0):
    return (rand(b, nq, h, d, dtype=dtype, seed=seed), rand(b, nk, hk, d, dtype=dtype, seed=seed + 1), rand(b, nk, hk, d, dtype=dtype, seed=seed + 2),
            rand(b, nq, h, d, dtype=dtype, seed=seed + 3))


@pytest.mark.parametrize("table_type", [None, F32])
@pytest.mark.parametrize("causal,window", [(True, None), (False, 90), (True, 33)])
@pytest.mark.parametrize("dtype,dim", [(BF, 40), (BF, 64), (BF, 128), (BF, 250), (F32, 64), (F32, 200)])
def test_padded_sequences(dtype, dim, causal, window, table_type):
    """Padding of both sides, shared heads, masks and a bias of either type; what lies behind the lengths is NaN."""
    b, nq, nk = 5, 190, 270
    q, k, v, do = inputs(b, nq, nk, 4, 2, dim, dtype)
    lengths, queries = torch.tensor([0, 70, 270, 200, 64]), torch.tensor([190, 1, 190, 0, 128])
    for e in range(b):
        k[e, lengths[e]:] = v[e, lengths[e]:] = math.nan
        q[e, queries[e]:] = do[e, queries[e]:] = math.nan
    table = None if table_type is None else rand(32, 4, dtype=table_type, seed=9)
    check(q, k, v, do, lengths=lengths, query_lengths=queries, table=table, causal=causal, window=window, far=60)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("b,nq,nk,h,hk,dim", [(1, 129, 257, 2, 1, 64), (2, 7, 900, 6, 1, 128), (1, 15, 640, 4, 4, 64), (3, 1, 700, 8, 2, 64), (1, 385, 513, 2, 2, 32),
                                              (1, 259, 64, 2, 1, 64), (1, 70, 190, 5, 5, 127), (1, 33, 2100, 8, 8, 64), (1, 300, 300, 8, 1, 128)])
def test_shapes(b, nq, nk, h, hk, dim, causal, dtype):
    check(*inputs(b, nq, nk, h, hk, dim, dtype), causal=causal)


@pytest.mark.parametrize("buckets,far,bidirectional", [(32, 128, True), (256, 1024, True), (8, 20, False)])
@pytest.mark.parametrize("dtype,dim,h,hk", [(BF, 64, 4, 4), (BF, 128, 4, 2), (BF, 200, 2, 1), (F32, 40, 2, 1)])
@pytest.mark.parametrize("nq,nk,causal", [(150, 390, False), (9, 500, True)])
def test_position_bias(nq, nk, causal, dtype, dim, h, hk, buckets, far, bidirectional):
    check(*inputs(2, nq, nk, h, hk, dim, dtype), table=rand(buckets, h, dtype=dtype, seed=9), causal=causal, far=far, bidirectional=bidirectional)


@pytest.mark.parametrize("b,n,h,hk,d,causal,table_type", [(8, 1000, 16, 16, 64, False, BF), (2, 3001, 8, 8, 128, False, F32), (4, 1537, 8, 2, 64, True, F32)])
def test_table_gradient_at_full_size(b, n, h, hk, d, causal, table_type):
    """Thousands of tiles, in 64 bits on the GPU. An entry is off by its own rounding, the rounding of each query's delta (of out, and
    of the probabilities in it: U sqrt(sum D^2 (out^2 + P^2 V^2)), P V <= out's terms) times the query's probability in
    the bucket, and what is fp32; six times their mean square."""
    g = torch.Generator(device="cuda").manual_seed(n)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(BF)  # noqa: E731
    q, k, v, do, table = r(b, n, h, d), r(b, n, hk, d), r(b, n, hk, d), r(b, n, h, d), r(32, h).to(table_type)
    kw = {"causal": causal, "relative_bias": table}
    out, lse = op("Attention", q, k, v, **kw)
    got = op("AttentionGrad", do, q, k, v, out, lse, **kw)[3]
    where, seen = R.bias_buckets(n, n, 0, 32, 128, not causal).cuda(), R.seen_keys(n, n, causal, None).cuda()
    ref, var = (torch.zeros(32, h, dtype=torch.float64, device="cuda") for _ in range(2))
    for a in range(h):
        for e in range(b):
            Q, K, V, D = q[e, :, a].double(), k[e, :, a // (h // hk)].double(), v[e, :, a // (h // hk)].double(), do[e, :, a].double()
            p = (Q @ K.t() / math.sqrt(d) + table[:, a].double()[where]).masked_fill(~seen, -math.inf).softmax(-1)
            o, dp = p @ V, D @ V.t()
            dz = p * (dp - (D * o).sum(-1, keepdim=True))
            vdelta = N.U[BF] ** 2 * ((D * D) * (o * o + (p * p) @ (V * V))).sum(-1, keepdim=True)
            share = torch.zeros(n, 32, dtype=torch.float64, device="cuda").scatter_add_(1, where, p)
            ref[:, a].index_add_(0, where.flatten(), dz.flatten())
            var[:, a] += (vdelta * share**2).sum(0)
            # |q| |k| / sqrt(d) = sqrt(d) and |dout| |v| = d for unit heads, the bias below 5: of that 10 x 2^-24 each (lse once more)
            var[:, a].index_add_(0, where.flatten(), (N.E32**2 * (2 * (math.sqrt(d) + 5) ** 2 * dz * dz + d * d * p * p)).flatten())
    var += (N.U[table_type] * ref) ** 2
    # (the bucket of later keys at no distance has no positions: its gradient is 0)
    off, tol = (got.double() - ref).abs(), 6 * var.sqrt()
    assert got.dtype == table_type and not (off > tol).any(), (off / tol).nan_to_num().max()
    # and the entries stand out of that: one wrong in its first digits would not pass
    assert float((ref.abs() / tol)[var > 0].median()) > 5


GRADS = ("dx", "df", "dgamma", "dbeta", "dpost_gamma", "dpost_beta", "dgate")


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("xt,ft", [(F32, F32), (BF, BF)])
@pytest.mark.parametrize("shape,gate,post", [
    ((5, 64), (64,), True), ((5, 7), (7,), True), ((5, 100), None, True), ((7, 257), (257,), True), ((7, 1024), (1024,), True), ((3, 1032), None, False),
    ((9, 2048), (2048,), True), ((5, 4099), (4099,), True), ((3, 8192), (8192,), True), ((3, 8200), (8200,), True), ((2, 16384), None, True),
    ((2, 16381), (16381,), False), ((2000, 3, 64), (2000, 1, 64), True), ((2, 3000, 40), (2, 1, 40), True), ((9000, 24), (24,), True),
    ((64, 1, 512), (64, 1, 512), True), ((3, 50, 75), (3, 50, 75), True), ((4, 300, 1024), (4, 1, 1024), True),
])
def test_residual_norm_and_gradients(shape, gate, post, xt, ft, norm):
    c = shape[-1]
    x, f = rand(*shape, dtype=xt, shift=0.3), rand(*shape, dtype=ft, seed=1)
    w = {"gamma": rand(c, seed=2, scale=0.2, shift=1)}
    if post:
        w["post_gamma"] = rand(c, seed=3, scale=0.2, shift=1)
    if norm == "layer":
        w["beta"] = rand(c, seed=4)
        if post:
            w["post_beta"] = rand(c, seed=5)
    if gate is not None:
        w["gate"] = rand(*gate, seed=6, scale=0.3, shift=0.5)
    ds, dh = rand(*shape, dtype=xt, seed=7), rand(*shape, dtype=ft, seed=8)
    ref, _ = R.residual_norm(x, f, **w, scale=0.75, norm=norm, post=post, eps=1e-5, dsum=ds, dnormed=dh)
    kw = {**{n: t.cuda() for n, t in w.items()}, "residual_scale": 0.75, "norm": norm, "post_norm": post, "eps": 1e-5}
    results = dict(zip(("sum", "normed"), op("ResidualNorm", x.cuda(), f.cuda(), **kw)))
    results.update(zip(GRADS, op("ResidualNormGrad", ds.cuda(), dh.cuda(), x.cuda(), f.cuda(), **kw)))
    wrong = [N.residual_off(n, t, ref[n], n in ("sum", "normed", "dx", "df") or (n == "dgate" and gate == shape)) for n, t in results.items() if t is not None]
    assert not any(wrong), wrong
