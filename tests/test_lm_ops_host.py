"""The language-model operators' host side: rotary frequencies and their fixed-point table,
refusals of the Python operators and of the C entry points (no kernel runs)."""

import ctypes as C
import math
from fractions import Fraction

import pytest
import torch

import lm_reference as R
from b200 import _lib as L
from b200 import lm_ops
from b200.errors import BackendNotSupportedError

SCALINGS = [
    None,
    {"kind": "linear", "factor": 4.0},
    {"kind": "ntk", "factor": 8.0},
    {"kind": "yarn", "factor": 16.0, "original_length": 4096},
    {"kind": "yarn", "factor": 4.0, "original_length": 200, "beta_fast": 8, "beta_slow": 0.5, "attention_factor": 1.25},
    {"kind": "wavelength", "factor": 8.0, "original_length": 8192, "low_factor": 1.0, "high_factor": 4.0},
]


@pytest.mark.parametrize("scaling", SCALINGS)
@pytest.mark.parametrize("dim", [2, 32, 46, 128])
def test_frequencies(dim, scaling):
    got, factor = lm_ops.rotary_frequencies(dim, 10000.0, scaling)
    want, f = R.angles(dim, 10000.0, scaling)
    assert factor == pytest.approx(f, rel=1e-15) and got == pytest.approx(want, rel=1e-13)


def test_fixed_point_turns_are_exact_modulo_a_turn():
    inv, _ = lm_ops.rotary_frequencies(64, 500000.0)
    r = lm_ops._rotary_table(64, 64, 500000.0, False, None)
    for j, w in enumerate(inv):
        for pos in (0, 1, 4097, 10**6 + 3, -(10**9), 2**40 + 1):
            phase = Fraction((pos * r.turns[j]) % 2**64, 2**64)
            # the double w / (2 pi) itself is rounded twice: 2^-52 of it, and 2^-65 of a turn in the table
            want = Fraction(w / (2 * math.pi)) * pos
            d = (phase - want) % 1
            assert min(d, 1 - d) <= abs(pos) * (Fraction(1, 2**65) + Fraction(w) / 2**51)


def test_rotary_refusals():
    x = torch.zeros(1, 4, 2, 64)
    rot = lm_ops.op_rotary_embedding
    with pytest.raises(ValueError, match="even"):
        rot(x, rotary_dim=31)
    with pytest.raises(ValueError, match="rotary_dim"):
        rot(x, rotary_dim=66)
    with pytest.raises(ValueError, match="head_dim 514"):
        rot(torch.zeros(1, 1, 1, 514))
    with pytest.raises(ValueError, match="heads must be"):
        rot(torch.zeros(4, 64))
    with pytest.raises(BackendNotSupportedError):
        rot(x.half())
    with pytest.raises(BackendNotSupportedError):
        rot(x.to(torch.int64))
    for base in (1.0, 0.0, -5.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="base"):
            rot(x, base=base)
    for bad in ({"kind": "other", "factor": 2.0}, {"kind": "linear"}, {"kind": "linear", "factor": 0.5}, {"kind": "ntk", "factor": float("nan")},
                {"kind": "yarn", "factor": 2.0}, {"kind": "yarn", "factor": 2.0, "original_length": 0},
                {"kind": "yarn", "factor": 2.0, "original_length": 64, "beta_fast": 1.0, "beta_slow": 2.0},
                {"kind": "linear", "factor": 2.0, "original_length": 64},
                {"kind": "wavelength", "factor": 2.0, "original_length": 64, "low_factor": 4.0, "high_factor": 1.0}):
        with pytest.raises(ValueError, match="scaling"):
            rot(x, scaling=bad)


def test_qk_refusals():
    q, k = torch.zeros(2, 4, 6, 64), torch.zeros(2, 4, 2, 64)
    f, g = lm_ops.op_qk_norm_rotary, lm_ops.op_qk_norm_rotary_grad
    for bad in (torch.zeros(2, 5, 2, 64), torch.zeros(1, 4, 2, 64), torch.zeros(2, 4, 2, 32), torch.zeros(4, 2, 64)):
        with pytest.raises(ValueError, match="differ in more"):
            f(q, bad)
    with pytest.raises(BackendNotSupportedError):
        f(q, k.to(torch.bfloat16))
    with pytest.raises(ValueError, match="norm weight"):
        f(q, k, torch.ones(6, 64))
    with pytest.raises(BackendNotSupportedError):
        f(q, k, torch.ones(64, dtype=torch.float64))
    with pytest.raises(ValueError, match="gradients"):
        g(q[:, :3], k, q, k)
    with pytest.raises(BackendNotSupportedError):
        g(q.to(torch.bfloat16), k, q, k)


def test_head_refusals():
    f = lm_ops.op_linear_cross_entropy
    x, w = torch.zeros(5, 16), torch.zeros(16, 30)
    with pytest.raises(ValueError, match="not aligned"):
        f(x, w.t(), torch.zeros(5, dtype=torch.int64))
    with pytest.raises(ValueError, match="not aligned"):
        f(x, torch.zeros(2, 16, 30), torch.zeros(5, dtype=torch.int64))


def test_newton_schulz_refusals():
    f = lm_ops.op_newton_schulz
    with pytest.raises(ValueError, match="matrix"):
        f(torch.zeros(7))
    with pytest.raises(BackendNotSupportedError):
        f(torch.zeros(4, 4, dtype=torch.float64))
    for kw in ({"steps": 0}, {"steps": 101}, {"coefficients": (1.0, 2.0)}, {"steps": 3, "coefficients": [[1.0, 2.0, 3.0]] * 2}):
        with pytest.raises(ValueError, match="Newton-Schulz"):
            f(torch.zeros(4, 4), **kw)
    with pytest.raises(ValueError, match="one shape"):
        lm_ops.op_apply_muon(torch.zeros(4, 4), torch.zeros(4, 4), torch.zeros(4, 5))


def test_operands_on_another_device_reach_no_kernel(monkeypatch):
    """Host tensors stand in for another GPU's: refused before a cast, a copy or a kernel runs."""
    def launched(*_):
        raise AssertionError("a kernel was launched")

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(L, "call", launched)
    monkeypatch.setattr(lm_ops.ops.Prog, "run", launched)
    monkeypatch.setattr(lm_ops.ops, "to_device", lambda t, *_: t)
    q, k, b16 = torch.zeros(2, 4, 6, 64), torch.zeros(2, 4, 2, 64), torch.bfloat16
    turned = torch.zeros(2, 4, 64, 6).transpose(2, 3)  # needs a dense copy
    x, w, y = torch.zeros(5, 16), torch.zeros(16, 30), torch.zeros(5, dtype=torch.int64)
    m = torch.zeros(8, 12)
    calls = [
        lambda: lm_ops.op_rotary_embedding(q),
        lambda: lm_ops.op_rotary_embedding(turned),
        lambda: lm_ops.op_rotary_embedding(q, torch.zeros(4, dtype=torch.int16)),
        lambda: lm_ops.op_rotary_embedding(q, torch.zeros(4, dtype=torch.int32)),
        lambda: lm_ops.op_rotary_embedding_grad(turned),
        lambda: lm_ops.op_qk_norm_rotary(q, k),
        lambda: lm_ops.op_qk_norm_rotary(turned, k),
        lambda: lm_ops.op_qk_norm_rotary(q, k, torch.ones(64), torch.ones(64, dtype=b16)),
        lambda: lm_ops.op_qk_norm_rotary(q, k, torch.ones(128)[::2]),
        lambda: lm_ops.op_qk_norm_rotary_grad(turned, k, q, k),
        *[lambda d=d: lm_ops.op_linear_cross_entropy(x, w, y.to(d)) for d in (torch.int64, torch.int32, torch.int16, torch.uint8)],
        lambda: lm_ops.op_linear_cross_entropy(x.to(b16), w, y),
        lambda: lm_ops.op_linear_cross_entropy(x[:, ::2], w[::2], y),
        lambda: lm_ops.op_linear_cross_entropy_grad(torch.zeros(5, dtype=b16), x, w, y, torch.zeros(5)),
        lambda: lm_ops.op_newton_schulz(m),
        lambda: lm_ops.op_newton_schulz(m.t()),
        lambda: lm_ops.op_apply_muon(m, m, m),
        lambda: lm_ops.op_apply_muon(m.to(b16), m, m.to(b16)),
        lambda: lm_ops.op_apply_muon(m, m, m.t().contiguous().t()),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(ValueError, match="current device"):
            call()
            raise AssertionError(i)


P = 256  # a stand-in address: the calls below are refused before anything reads it


def rotary(head_dim=64, rotary_dim=64):
    r = L.Rotary()
    r.head_dim, r.rotary_dim, r.factor = head_dim, rotary_dim, 1.0
    return r


def rotary_heads(r=None, dtype=L.BF16, x=P, batch=1, seq=1, heads=1, pos=None, pos_dtype=L.I64):
    return L.lib().b200_rotary_heads(rotary() if r is None else r, dtype, x, P, batch, seq, heads, *[64] * 6, pos, pos_dtype, 0, 1, 0, 0, None)


def test_c_refusals_rotary():
    for kw in ({"r": rotary(0, 0)}, {"r": rotary(513, 2)}, {"r": rotary(64, 66)}, {"r": rotary(64, 3)}, {"r": rotary(64, -2)}, {"x": None},
               {"batch": -1}, {"batch": 1 << 20, "seq": 1 << 12}, {"heads": 1 << 17}, {"heads": -1}):
        assert rotary_heads(**kw) == L.ERR_ARG, kw
    assert rotary_heads(dtype=L.I32) == L.ERR_DTYPE and rotary_heads(pos=P, pos_dtype=L.F32) == L.ERR_DTYPE
    assert rotary_heads(batch=0, x=None) == L.OK
    n = int(L.lib().b200_qk_norm_rotary_grad_workspace_bytes(64))
    st = L.I64x18(*[64] * 18)

    def grad(ws=P, bytes_=n, eps=1e-6, gamma_dtype=L.F32, strides=st, q=P):
        return L.lib().b200_qk_norm_rotary_grad(rotary(), L.BF16, P, P, q, P, P, P, 1, 1, 1, 1, strides, P, P, gamma_dtype, eps, None, L.I64,
                                                0, 0, 0, P, P, ws, bytes_, None)

    assert grad(ws=None) == grad(bytes_=n - 1) == grad(eps=-1.0) == grad(strides=None) == grad(q=None) == L.ERR_ARG
    assert grad(gamma_dtype=L.I64) == L.ERR_DTYPE


def test_c_refusals_linear_xent():
    def loss(dtype=L.BF16, x=P, w=P, labels=P, ldt=L.I64, N=4, D=64, V=100, ldx=64, ldw=104, ws=P, bytes_=None, loss=P):
        n = int(L.lib().b200_linear_xent_workspace_bytes(dtype, x, ldx, w, ldw, 1, N, D, V))
        return L.lib().b200_linear_xent(dtype, x, ldx, w, ldw, 1, labels, ldt, -100, loss, P, N, D, V, ws, n if bytes_ is None else bytes_, None)

    def grad(dx=P, dw=P, dloss=P, bytes_=None, V=100):
        n = int(L.lib().b200_linear_xent_grad_workspace_bytes(L.F32, P, 64, P, 104, 1, 4, 64, V))
        return L.lib().b200_linear_xent_grad(L.F32, dloss, P, 64, P, 104, 1, P, L.I64, -100, P, dx, dw, 4, 64, V, P,
                                             n if bytes_ is None else bytes_, None)

    for kw in ({"x": None}, {"w": None}, {"labels": None}, {"loss": None}, {"N": -1}, {"D": 0}, {"V": 0}, {"ldx": 63}, {"ldw": 99}, {"ws": None}, {"ws": P + 16},
               {"bytes_": 8}, {"N": 1 << 30}):
        assert loss(**kw) == L.ERR_ARG, kw
    assert loss(dtype=L.I32) == L.ERR_DTYPE and loss(ldt=L.F32) == L.ERR_DTYPE
    assert grad(dx=None, dw=None) == grad(dloss=None) == grad(bytes_=100) == grad(V=0) == L.ERR_ARG
    assert loss(N=0, x=None, labels=None, ws=None) == L.OK


def test_c_refusals_newton_schulz():
    c = (C.c_float * 15)(*[1.0] * 15)

    def ns(dtype=L.F32, g=P, batch=1, rows=64, cols=64, coef=c, steps=5, eps=0.0, ws=P, bytes_=None):
        n = int(L.lib().b200_newton_schulz_workspace_bytes(dtype, batch, rows, cols))
        return L.lib().b200_newton_schulz(dtype, g, P, batch, rows, cols, coef, steps, eps, ws, n if bytes_ is None else bytes_, None)

    for kw in ({"g": None}, {"batch": -1}, {"batch": 1 << 16}, {"rows": 1 << 24}, {"steps": 0}, {"steps": 101}, {"eps": -1.0}, {"coef": None},
               {"ws": None}, {"ws": P + 16}, {"bytes_": 64}):
        assert ns(**kw) == L.ERR_ARG, kw
    assert ns(dtype=L.I32) == L.ERR_DTYPE and ns(rows=0, g=None, ws=None) == L.OK
    assert L.lib().b200_apply_muon_f32(P, None, P, P, P, 1, 64, 64, 0.1, 0.9, 1, 0.0, c, 5, 0.0, P, 1 << 30, None) == L.ERR_ARG
