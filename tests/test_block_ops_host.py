"""The block operators' host side: buckets, refusals of the Python operators and of the C entry points (no
kernel runs)."""

import ctypes as C

import pytest
import torch

import block_reference as R
from b200 import _lib as L
from b200 import block_ops, ops
from b200.errors import BackendNotSupportedError

BF = torch.bfloat16


@pytest.mark.parametrize("side,far", [(16, 128), (32, 128), (2, 2), (2, 1024), (3, 7), (128, 1024), (16, 9), (8, 512)])
def test_bucket_starts(side, far):
    starts = block_ops.relative_bucket_starts(side, far)
    assert starts[0] == 0 and len(starts) == side and starts == sorted(starts) and starts[-1] <= far
    for n in range(far + 3):
        assert sum(s <= n for s in starts) - 1 == R.bucket(-n, side, far, True)


def test_names_are_registered():
    from b200 import fused_nodes, lm_ops

    names, others = {}, {}
    block_ops.register(names)
    fused_nodes.register(others)
    lm_ops.register(others)
    assert set(names) == {"Attention", "AttentionGrad", "RelativePositionBias", "RelativePositionBiasGrad", "ResidualNorm", "ResidualNormGrad"}
    assert not set(names) & set(others) and not set(names) & set(ops.ALIASES)
    assert all(ops.OPS[n] is f for n, f in names.items())


def qkv(b=2, nq=5, nk=7, h=4, hk=2, d=16, dtype=torch.float32):
    return torch.zeros(b, nq, h, d, dtype=dtype), torch.zeros(b, nk, hk, d, dtype=dtype), torch.zeros(b, nk, hk, d, dtype=dtype)


def test_attention_refusals():
    q, k, v = qkv()
    f = block_ops.op_attention
    for bad in ((q, k[:1], v), (q, k, v[:, :3]), (q, k[..., :8], v[..., :8]), (q[:, :, :3], k, v), (q[0], k, v), (q[0], k[0], v), (q[0], k, v[0]),
                (q, k[0], v[0]), (q[0], k[:1], v[:1]), (q[0], k[0], v[:1]), (q[0, 0], k[0, 0], v[0, 0]),
                (torch.zeros(1, 2, 2, 257),) * 3, (torch.zeros(1, 2, 2, 0),) * 3, (q, k[:, :, :0], v[:, :, :0])):
        with pytest.raises(ValueError):
            f(*bad)
    for bad in ((q.half(), k.half(), v.half()), (q, k.to(BF), v), (q, k, v.to(BF)), (q.double(), k.double(), v.double())):
        with pytest.raises(BackendNotSupportedError):
            f(*bad)
    for kw in ({"scale": 0.0}, {"scale": -1.0}, {"scale": float("nan")}, {"scale": float("inf")}, {"window": 0}, {"window": -3}, {"window": 1.5},
               {"relative_bias": torch.zeros(32, 3)}, {"relative_bias": torch.zeros(33, 4)}, {"relative_bias": torch.zeros(2, 4)},
               {"relative_bias": torch.zeros(4)}, {"relative_bias": torch.zeros(258, 4)}, {"relative_bias": torch.zeros(32, 4), "max_distance": 8},
               {"relative_bias": torch.zeros(32, 4), "max_distance": 1025}):
        with pytest.raises(ValueError):
            f(q, k, v, **kw)
    with pytest.raises(BackendNotSupportedError):
        f(q, k, v, relative_bias=torch.zeros(32, 4).half())
    if not torch.cuda.is_available():
        with pytest.raises(Exception):
            f(q, k, v)  # no CPU fallback


def test_lengths_refusals():
    for bad, err in (([1, 2, 3], ValueError), (torch.zeros(2, 1, dtype=torch.int64), ValueError), (torch.zeros(2), BackendNotSupportedError),
                     (torch.zeros(2, dtype=torch.bool), BackendNotSupportedError)):
        with pytest.raises(err):
            block_ops._lengths("Attention", "lengths", bad, 2)


def test_bias_refusals():
    f, g = block_ops.op_relative_position_bias, block_ops.op_relative_position_bias_grad
    t = torch.zeros(32, 4)
    for kw in ({}, {"queries": 3}, {"queries": -1, "keys": 2}, {"queries": 2.5, "keys": 2}, {"queries": 2, "keys": 2, "max_distance": 8}):
        with pytest.raises(ValueError):
            f(t, **kw)
    for bad in (t[0], torch.zeros(33, 4), torch.zeros(2, 4)):
        with pytest.raises(ValueError):
            f(bad, queries=2, keys=2)
    with pytest.raises(BackendNotSupportedError):
        f(t.half(), queries=2, keys=2)
    with pytest.raises(ValueError):
        g(torch.zeros(3, 4), buckets=32)
    with pytest.raises(ValueError):
        g(torch.zeros(2, 3, 4))
    with pytest.raises(BackendNotSupportedError):
        g(torch.zeros(2, 3, 4).half(), buckets=32)


def test_residual_norm_refusals():
    f = block_ops.op_residual_norm
    x = torch.zeros(2, 3, 8)
    one = torch.ones(8)
    for args, kw in (((x, x[:1]), {}), ((x, x), {"norm": "batch"}), ((x, x), {"gamma": one[:7]}), ((x, x), {"beta": one}),
                     ((x, x), {"post_gamma": one, "post_norm": False}), ((x, x), {"gate": torch.ones(3, 8)}), ((x, x), {"gate": torch.ones(1, 3, 8)}),
                     ((x, x), {"gate": torch.ones(2, 1, 7)}), ((x, x), {"gate": torch.ones(())}), ((x, x), {"residual_scale": float("nan")}),
                     ((torch.zeros(1, 16385),) * 2, {}), ((torch.zeros(()),) * 2, {}), ((torch.zeros(3, 0),) * 2, {})):
        with pytest.raises(ValueError):
            f(*args, **kw)
    for args, kw in (((x.half(), x), {}), ((x, x.double()), {}), ((x, x), {"gamma": one.half()}), ((x, x), {"gate": one.half()})):
        with pytest.raises(BackendNotSupportedError):
            f(*args, **kw)


def _attention():
    a = L.Attention()
    a.batch, a.queries, a.keys, a.heads, a.kv_heads, a.dim, a.scale = 1, 4, 4, 2, 1, 64, 1.0
    a.q = a.k = a.v = 4096
    return a


@pytest.mark.parametrize("field,value,status", [
    ("batch", -1, L.ERR_ARG), ("batch", 65536, L.ERR_ARG), ("queries", -1, L.ERR_ARG), ("keys", 1 << 30, L.ERR_ARG), ("heads", 0, L.ERR_ARG),
    ("kv_heads", 3, L.ERR_ARG), ("dim", 0, L.ERR_ARG), ("dim", 257, L.ERR_ARG), ("window", -1, L.ERR_ARG), ("scale", 0.0, L.ERR_ARG),
    ("scale", float("nan"), L.ERR_ARG), ("dtype", L.F64, L.ERR_DTYPE), ("q", None, L.ERR_ARG), ("v", None, L.ERR_ARG), ("queries", 1 << 29, L.ERR_ARG),
])
def test_attention_entry_points_check(field, value, status):
    lib = L.load()
    a, g = _attention(), L.AttentionGrads()
    setattr(a, field, value)
    assert lib.b200_attention_workspace_bytes(a) == 0
    assert lib.b200_attention_forward(a, 4096, 4096, None, 0, None) == status and L.last_error()
    assert lib.b200_attention_grad(a, g, None, 0, None) == status


def test_attention_entry_points_check_more():
    lib = L.load()
    a = _attention()
    assert lib.b200_attention_forward(None, 4096, 4096, None, 0, None) == L.ERR_ARG
    assert lib.b200_attention_forward(a, None, 4096, None, 0, None) == L.ERR_ARG
    assert lib.b200_attention_grad(a, None, None, 0, None) == L.ERR_ARG
    assert lib.b200_attention_grad(a, L.AttentionGrads(), None, 0, None) == L.ERR_ARG
    a.lengths, a.length_dtype = 4096, L.F32
    assert lib.b200_attention_forward(a, 4096, 4096, None, 0, None) == L.ERR_DTYPE
    a = _attention()
    a.table = 4096
    assert lib.b200_attention_forward(a, 4096, 4096, None, 0, None) == L.ERR_ARG  # no buckets
    a.relative = block_ops._relative(32, 128, True)
    assert lib.b200_attention_grad(a, L.AttentionGrads(), None, 0, None) == L.ERR_ARG  # no dtable
    a.table_dtype = L.I64
    assert lib.b200_attention_forward(a, 4096, 4096, None, 0, None) == L.ERR_DTYPE
    a.batch = 0
    a.table = None
    assert lib.b200_attention_forward(a, None, None, None, 0, None) == L.OK


def test_bias_entry_points_check():
    lib = L.load()
    r = block_ops._relative(32, 128, True)
    call = lambda r, *s, dt=L.F32: lib.b200_relative_bias(r, dt, 4096, 4096, *s, None)  # noqa: E731
    assert call(None, 1, 1, 1, 0) == L.ERR_ARG
    assert call(r, -1, 1, 1, 0) == L.ERR_ARG and call(r, 1, 1 << 30, 1, 0) == L.ERR_ARG and call(r, 1, 1, 1, 1 << 40) == L.ERR_ARG
    assert call(r, 1, 1 << 23, 1 << 22, 0) == L.ERR_ARG  # more pieces than a grid has
    assert call(r, 1, 1, 1, 0, dt=L.I64) == L.ERR_DTYPE and call(r, 0, 1, 1, 0) == L.OK
    bad = L.Relative()
    for side, starts in ((0, []), (129, []), (2, [1, 2]), (3, [0, 5, 4]), (2, [0, 1025])):
        bad.side = side
        for i, s in enumerate(starts):
            bad.start[i] = s
        assert call(bad, 1, 1, 1, 0) == L.ERR_ARG
    assert lib.b200_relative_bias_grad(r, L.F32, 4096, 4096, 1, 1, 4, 4, 0, None, 0, None) == L.ERR_ARG
    assert lib.b200_relative_bias_grad(r, L.F32, None, 4096, 1, 1, 4, 4, 0, 4096, 1 << 20, None) == L.ERR_ARG
    assert lib.b200_relative_bias_grad(r, L.F32, 4096, 4096, -1, 1, 4, 4, 0, 4096, 1 << 20, None) == L.ERR_ARG


def test_residual_norm_entry_points_check():
    lib = L.load()
    p = 4096

    def make(**kw):
        d = L.ResidualNorm()
        d.rows, d.cols, d.scale = 4, 8, 1.0
        for n, v in kw.items():
            setattr(d, n, v)
        return d

    for kw, status in (({"cols": 0}, 1), ({"cols": 16385}, 1), ({"rows": -1}, 1), ({"kind": 2}, 1), ({"groups": 3, "gate": p}, 1), ({"groups": 2}, 1),
                       ({"gate": p}, 1), ({"post_gamma": p}, 1), ({"beta": p}, 1), ({"x_dtype": L.I64}, 2), ({"weight_dtype": L.F64}, 2)):
        assert lib.b200_residual_norm_forward(make(**kw), p, p, p, p, None) == status, kw
        assert lib.b200_residual_norm_grad(make(**kw), p, p, p, p, p, p, L.ResidualNormGrads(), None, 0, None) == status, kw
    assert lib.b200_residual_norm_forward(make(), None, p, p, p, None) == L.ERR_ARG
    assert lib.b200_residual_norm_forward(make(rows=0), None, None, None, None, None) == L.OK
    assert lib.b200_residual_norm_grad(make(), p, p, p, p, p, p, None, None, 0, None) == L.ERR_ARG
    assert lib.b200_residual_norm_grad(make(), p, p, p, p, p, p, L.ResidualNormGrads(), None, 0, None) == L.ERR_ARG
    assert lib.b200_residual_norm_grad(make(groups=1, gate=p), p, p, p, p, p, p, L.ResidualNormGrads(), p, C.c_size_t(1 << 30), None) == L.ERR_ARG
