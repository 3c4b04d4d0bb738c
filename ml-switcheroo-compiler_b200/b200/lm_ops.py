"""Language-model operators: rotary positions, query / key norms, the vocabulary loss and
the orthogonalised update.

They have no counterpart in the reference's op vocabulary. They follow the conventions of
``ops``: values are ``torch.Tensor`` on the current CUDA device, results are fresh tensors,
all arithmetic runs in libb200.so, gradients are separate operators (as the reference's
``LayerNormInputGrad``), ``execute_op`` reaches them by name.
"""

from __future__ import annotations

import ctypes
import functools
import math
from typing import Any, Mapping

import numpy as np
import torch

from . import _lib as L
from . import ops
from .errors import BackendNotSupportedError

_FLOATS = (torch.float32, torch.bfloat16)


def _on_device(name: str, *tensors: torch.Tensor | None) -> None:
    """The kernels run on the current device's stream: operands elsewhere are refused, ahead
    of the first kernel that would read them."""
    dev = torch.cuda.current_device()
    for t in tensors:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"{name}: operand on {t.device}, the current device is cuda:{dev}")


# ----------------------------------------------------------------------------------
# rotary positions
# ----------------------------------------------------------------------------------

_SCALING_KEYS = {
    "linear": ({"factor"}, set()),
    "ntk": ({"factor"}, set()),
    "yarn": ({"factor", "original_length"}, {"beta_fast", "beta_slow", "attention_factor"}),
    "wavelength": ({"factor", "original_length", "low_factor", "high_factor"}, set()),
}


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: Mapping[str, Any] | None = None) -> tuple[list[float], float]:
    """Angle per position (radians) of each of the rotary_dim / 2 pairs, and the factor on
    cosine and sine.

    Pair j turns by ``base ** (-2 j / rotary_dim)`` per position. ``scaling`` stretches
    that to contexts ``factor`` times as long as the angles were made for:

    * ``{"kind": "linear", "factor": f}``: every angle divided by f;
    * ``{"kind": "ntk", "factor": f}``: base times f ** (d / (d - 2)), so the slowest pair
      is divided by f and the fastest keeps its angle;
    * ``{"kind": "yarn", "factor": f, "original_length": n}`` (``beta_fast`` 32,
      ``beta_slow`` 1, ``attention_factor`` 0.1 ln f + 1): pairs that turn less than
      beta_slow times over n positions are divided by f, pairs that turn more than
      beta_fast times are kept, a linear ramp over the pair index between; cosine and sine
      are multiplied by the attention factor;
    * ``{"kind": "wavelength", "factor": f, "original_length": n, "low_factor": a,
      "high_factor": b}``: the same by the turns over n positions themselves, a ramp from a
      (divided) to b (kept).
    """
    inv = [base ** (-2.0 * j / rotary_dim) for j in range(rotary_dim // 2)]
    if scaling is None:
        return inv, 1.0
    kind = scaling.get("kind")
    if kind not in _SCALING_KEYS:
        raise ValueError(f"rotary scaling kind {kind!r} is not one of {sorted(_SCALING_KEYS)}")
    need, may = _SCALING_KEYS[kind]
    given = set(scaling) - {"kind"}
    if not need <= given or not given <= need | may:
        raise ValueError(f"rotary scaling {kind!r} takes {sorted(need)} and optionally {sorted(may)}, got {sorted(given)}")
    f = float(scaling["factor"])
    if not (f >= 1.0 and math.isfinite(f)):
        raise ValueError(f"rotary scaling factor {f} is not a finite number >= 1")
    if kind == "linear":
        return [w / f for w in inv], 1.0
    if kind == "ntk":
        b = base * f ** (rotary_dim / (rotary_dim - 2.0)) if rotary_dim > 2 else base
        return [b ** (-2.0 * j / rotary_dim) for j in range(rotary_dim // 2)], 1.0
    n = float(scaling["original_length"])
    if not (n > 0 and math.isfinite(n)):
        raise ValueError(f"rotary scaling original_length {n} is not a positive number")
    if kind == "yarn":
        fast, slow = float(scaling.get("beta_fast", 32.0)), float(scaling.get("beta_slow", 1.0))
        if not (fast >= slow > 0):
            raise ValueError(f"rotary scaling needs beta_fast >= beta_slow > 0, got {fast} and {slow}")
        pair = [rotary_dim * math.log(n / (b * 2 * math.pi)) / (2 * math.log(base)) for b in (fast, slow)]
        low, high = max(math.floor(pair[0]), 0), min(math.ceil(pair[1]), rotary_dim - 1)
        ramp = [min(1.0, max(0.0, (j - low) / max(high - low, 0.001))) for j in range(rotary_dim // 2)]
        factor = float(scaling.get("attention_factor", 0.1 * math.log(f) + 1.0))
        return [w * (1 - t) + w / f * t for w, t in zip(inv, ramp)], factor
    low, high = float(scaling["low_factor"]), float(scaling["high_factor"])
    if not high > low > 0:
        raise ValueError(f"rotary scaling needs high_factor > low_factor > 0, got {high} and {low}")
    keep = [min(1.0, max(0.0, (n * w / (2 * math.pi) - low) / (high - low))) for w in inv]
    return [w * t + w / f * (1 - t) for w, t in zip(inv, keep)], 1.0


@functools.lru_cache(maxsize=256)
def _rotary_table(head_dim: int, rotary_dim: int, base: float, interleaved: bool, scaling: tuple | None) -> L.Rotary:
    """The kernels' description of a rotation: each pair's fraction of a turn per position in
    64-bit fixed point, so that position * turns is exact modulo one turn."""
    if not 1 <= head_dim <= L.ROTARY_MAX_DIM:
        raise ValueError(f"rotary: head_dim {head_dim} not in [1, {L.ROTARY_MAX_DIM}]")
    if rotary_dim % 2 or not 0 <= rotary_dim <= head_dim:
        raise ValueError(f"rotary: rotary_dim {rotary_dim} must be even and in [0, head_dim = {head_dim}]")
    if not (base > 1.0 and math.isfinite(base)):
        raise ValueError(f"rotary: base {base} is not a finite number > 1")
    inv, factor = rotary_frequencies(rotary_dim, base, None if scaling is None else dict(scaling))
    r = L.Rotary()
    r.head_dim, r.rotary_dim, r.interleaved, r.factor = head_dim, rotary_dim, int(interleaved), factor
    for j, w in enumerate(inv):
        r.turns[j] = round(w / (2 * math.pi) * 2.0**64) % 2**64
    return r


def _rotary(head_dim: int, rotary_dim, base, interleaved, scaling) -> L.Rotary:
    key = None if scaling is None else tuple(sorted(scaling.items()))
    return _rotary_table(head_dim, head_dim if rotary_dim is None else int(rotary_dim), float(base), bool(interleaved), key)


def _heads(name: str, x: torch.Tensor) -> tuple[torch.Tensor, tuple, tuple[int, int, int]]:
    """x [batch, seq, heads, dim] or [seq, heads, dim] -> (x with adjacent head elements,
    (batch, seq, heads, dim), element strides of the first three)."""
    if x.dtype not in _FLOATS:
        raise BackendNotSupportedError(f"{name}: {x.dtype} heads have no b200 kernel (fp32 and bf16)")
    shape, st = tuple(x.shape), x.stride()
    if len(shape) not in (3, 4):
        raise ValueError(f"{name}: heads must be [batch, seq, heads, dim] or [seq, heads, dim], got {shape}")
    if st[-1] != 1 and shape[-1] > 1:
        _on_device(name, x)
        x = ops.contiguous(x)
        st = x.stride()
    return (x, shape, st[:3]) if len(shape) == 4 else (x, (1, *shape), (0, *st[:2]))


def _like(x: torch.Tensor) -> tuple[torch.Tensor, tuple[int, int, int]]:
    """A fresh result for x: dense, its axes in x's storage order, adjacent head elements;
    and its strides."""
    y = torch.empty_like(x)
    st = y.stride()
    if st[-1] != 1 and y.shape[-1] > 1:
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        st = y.stride()
    return y, (st[:3] if len(st) == 4 else (0, *st[:2]))


def _positions(name: str, positions: Any, offset: int, batch: int, seq: int) -> tuple[torch.Tensor | None, tuple]:
    """positions [seq], [1, seq] or [batch, seq] of int32 / int64 -> (tensor kept alive,
    the entry points' position arguments)."""
    if positions is None:
        return None, (None, L.I64, 0, 0, int(offset))
    if offset:
        raise ValueError(f"{name}: give positions or an offset, not both")
    t = positions if isinstance(positions, torch.Tensor) else torch.as_tensor(positions)
    shape = tuple(t.shape)
    if shape not in ((seq,), (1, seq), (batch, seq)):
        raise ValueError(f"{name}: positions {shape} do not match {batch} sequences of {seq} tokens")
    if not t.is_cuda or (t.dtype != torch.int64 and t.dtype != torch.int32):
        t = ops.to_device(t)
        _on_device(name, t)
        t = ops._int_indices(t)
    st = t.stride()
    return t, (t.data_ptr(), L.I64 if t.dtype == torch.int64 else L.I32, st[0] if len(shape) == 2 and shape[0] > 1 else 0, st[-1], 0)


def _rotate(name: str, x: torch.Tensor, positions, base, rotary_dim, interleaved, scaling, offset, inverse: int) -> torch.Tensor:
    x, (batch, seq, heads, dim), xs = _heads(name, x)
    r = _rotary(dim, rotary_dim, base, interleaved, scaling)
    pos, pa = _positions(name, positions, offset, batch, seq)
    _on_device(name, x, pos)
    y, ys = _like(x)
    L.call("b200_rotary_heads", r, ops.code(x), x.data_ptr(), y.data_ptr(), batch, seq, heads, *xs, *ys, *pa, inverse, ops.stream_ptr())
    return y


def op_rotary_embedding(x, positions=None, base=10000.0, rotary_dim=None, interleaved=False, scaling=None, offset=0, **_):
    """Rotary positions: each pair of a head's first ``rotary_dim`` elements (all by default)
    turned by its angle (``rotary_frequencies``) times the token's position.

    x: [batch, seq, heads, dim] or [seq, heads, dim], fp32 or bf16, any strides (a
    head-major tensor is passed as its transposed view); head_dim <= 512. Pairs are (j, j +
    rotary_dim / 2), or neighbours with ``interleaved``. positions: integers [seq], [1, seq]
    or [batch, seq]; None: ``offset`` + 0 .. seq - 1. Computed in fp32, rounded once."""
    return _rotate("RotaryEmbedding", x, positions, base, rotary_dim, interleaved, scaling, offset, 0)


def op_rotary_embedding_grad(dy, positions=None, base=10000.0, rotary_dim=None, interleaved=False, scaling=None, offset=0, **_):
    """The gradient of RotaryEmbedding's input: the rotation turned back."""
    return _rotate("RotaryEmbeddingGrad", dy, positions, base, rotary_dim, interleaved, scaling, offset, 1)


def _pair(name: str, q: torch.Tensor, k: torch.Tensor):
    q, (batch, seq, hq, dim), qs = _heads(name, q)
    k, (kbatch, kseq, hk, kdim), ks = _heads(name, k)
    if q.dim() != k.dim() or (kbatch, kseq, kdim) != (batch, seq, dim):
        raise ValueError(f"{name}: queries {tuple(q.shape)} and keys {tuple(k.shape)} differ in more than their heads")
    if q.dtype != k.dtype:
        raise BackendNotSupportedError(f"{name}: queries of {q.dtype} with keys of {k.dtype}")
    return q, k, batch, seq, hq, hk, dim, qs, ks


def _gammas(name: str, dim: int, gq: torch.Tensor | None, gk: torch.Tensor | None):
    """The norm weights as [dim] tensors of one dtype (fp32 if they differ)."""
    out = []
    for g in (gq, gk):
        if g is not None:
            if tuple(g.shape) != (dim,):
                raise ValueError(f"{name}: norm weight {tuple(g.shape)}, want [{dim}]")
            if g.dtype not in _FLOATS:
                raise BackendNotSupportedError(f"{name}: norm weights of {g.dtype} (fp32 and bf16)")
            _on_device(name, g)
            g = ops.contiguous(g)
        out.append(g)
    if gq is not None and gk is not None and gq.dtype != gk.dtype:
        out = [ops.cast(g, torch.float32) for g in out]
    dt = next((ops.code(g) for g in out if g is not None), L.F32)
    return out[0], out[1], dt


def op_qk_norm_rotary(q, k, gamma_q=None, gamma_k=None, positions=None, eps=1e-6, base=10000.0, rotary_dim=None, interleaved=False,
                      scaling=None, offset=0, **_):
    """RMS norm of each query and key head, times gamma, and the rotary positions of both, in
    one pass: returns (q', k').

    q [batch, seq, heads, dim], k [batch, seq, kv_heads, dim] (or both without the batch) of
    one dtype, any strides, so slices of one projection's result are read in place; gamma_q /
    gamma_k [dim], None: ones. The rest as RotaryEmbedding; ``rotary_dim=0`` norms alone.
    The norm's sum and the rotation are in fp32, rounded once."""
    name = "QKNormRotary"
    q, k, batch, seq, hq, hk, dim, qs, ks = _pair(name, q, k)
    r = _rotary(dim, rotary_dim, base, interleaved, scaling)
    gq, gk, gdt = _gammas(name, dim, gamma_q, gamma_k)
    pos, pa = _positions(name, positions, offset, batch, seq)
    _on_device(name, q, k, gq, gk, pos)
    (yq, yqs), (yk, yks) = _like(q), _like(k)
    L.call("b200_qk_norm_rotary", r, ops.code(q), q.data_ptr(), k.data_ptr(), yq.data_ptr(), yk.data_ptr(), batch, seq, hq, hk, *qs,
           *ks, *yqs, *yks, ops._ptr(gq), ops._ptr(gk), gdt, float(eps), *pa, ops.stream_ptr())
    return yq, yk


def op_qk_norm_rotary_grad(dyq, dyk, q, k, gamma_q=None, gamma_k=None, positions=None, eps=1e-6, base=10000.0, rotary_dim=None,
                           interleaved=False, scaling=None, offset=0, **_):
    """The gradients of QKNormRotary from those of its results and its inputs:
    (dq, dk, dgamma_q, dgamma_k), the weights' in fp32 [dim] (also where a gamma is None),
    summed over tokens and heads in a fixed order."""
    name = "QKNormRotaryGrad"
    q, k, batch, seq, hq, hk, dim, qs, ks = _pair(name, q, k)
    if tuple(dyq.shape) != tuple(q.shape) or tuple(dyk.shape) != tuple(k.shape):
        raise ValueError(f"{name}: gradients {tuple(dyq.shape)}, {tuple(dyk.shape)} of queries {tuple(q.shape)}, keys {tuple(k.shape)}")
    if dyq.dtype != q.dtype or dyk.dtype != q.dtype:
        raise BackendNotSupportedError(f"{name}: gradients of {dyq.dtype}, {dyk.dtype} for {q.dtype} heads")
    dyq, _, dqs = _heads(name, dyq)
    dyk, _, dks = _heads(name, dyk)
    r = _rotary(dim, rotary_dim, base, interleaved, scaling)
    gq, gk, gdt = _gammas(name, dim, gamma_q, gamma_k)
    pos, pa = _positions(name, positions, offset, batch, seq)
    _on_device(name, q, k, dyq, dyk, gq, gk, pos)
    (dq, rqs), (dk, rks) = _like(q), _like(k)
    dgq, dgk = torch.empty(2, dim, dtype=torch.float32, device=q.device).unbind(0)
    wn = L.lib().b200_qk_norm_rotary_grad_workspace_bytes(dim)
    ws = torch.empty(wn, dtype=torch.uint8, device=q.device)
    st = L.I64x18(*qs, *dqs, *rqs, *ks, *dks, *rks)
    L.call("b200_qk_norm_rotary_grad", r, ops.code(q), dyq.data_ptr(), dyk.data_ptr(), q.data_ptr(), k.data_ptr(), dq.data_ptr(),
           dk.data_ptr(), batch, seq, hq, hk, st, ops._ptr(gq), ops._ptr(gk), gdt, float(eps), *pa, dgq.data_ptr(),
           dgk.data_ptr(), ws.data_ptr(), wn, ops.stream_ptr())
    return dq, dk, dgq, dgk


# ----------------------------------------------------------------------------------
# output head and cross entropy
# ----------------------------------------------------------------------------------


def _cast(t: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """A fresh cast (of a transposed matrix in its storage order); t itself if it is of that type."""
    return ops.cast(t.t(), dtype).t() if t.dim() == 2 and t.stride(0) == 1 else ops.cast(t, dtype)


def _head(name: str, x: torch.Tensor, w: torch.Tensor, labels: Any):
    """The operands as the entry points take them: (x [N, D], w, labels [N], row strides,
    whether w is stored [D, V], sizes)."""
    xs, ws = tuple(x.shape), tuple(w.shape)
    if len(ws) != 2 or not xs or xs[-1] != ws[0]:
        raise ValueError(f"{name}: x {xs} and w {ws} not aligned")
    if x.dtype not in _FLOATS or w.dtype not in _FLOATS:
        raise BackendNotSupportedError(f"{name}: x of {x.dtype} and w of {w.dtype} (fp32 and bf16)")
    D, V = ws
    if D < 1 or V < 1:
        raise ValueError(f"{name}: w {ws} has no features or no words")
    if not isinstance(labels, torch.Tensor):
        labels = ops.to_device(labels)
    if tuple(labels.shape) not in (xs[:-1], (*xs[:-1], 1)):
        raise ValueError(f"{name}: labels {tuple(labels.shape)} of x {xs}")
    _on_device(name, x, w, labels)
    if labels.dtype != torch.int32:
        labels = ops._int_indices(labels)
    policy = ops.Config.matmul_dtype
    if x.dtype != w.dtype or (policy == "bf16" and x.dtype == torch.float32):
        # the contraction policy of Matmul: bf16 operands, or fp32 where either is
        dt = torch.bfloat16 if policy == "bf16" else torch.float32
        x, w = _cast(x, dt), _cast(w, dt)
    if len(xs) != 2:
        x = ops.contiguous(x).view(-1, D)
    sn, sd = x.stride()
    if (sd != 1 and D > 1) or sn < D:
        x = ops.contiguous(x)
        sn = D
    N = x.shape[0]
    wr, wc = w.stride()
    dn = wc == 1 and wr >= V
    if not dn and not (wr == 1 and wc >= D):
        w, dn = ops.contiguous(w), True
        wr = V
    labels = ops.contiguous(labels)
    return x, w, labels, max(sn, D), wr if dn else wc, int(dn), N, D, V


def op_linear_cross_entropy(x, w, labels, ignore_index=-100, **_):
    """The head's product and its softmax cross entropy, the logits never in memory:
    (loss, lse) of z = x.w, lse = log sum exp z, loss = lse - z[label], fp32 in x's leading shape.

    x [..., D] and w [D, V], fp32 or bf16 (a tied embedding [V, D] is passed as its
    transposed view), labels integers in x's leading shape (or with a trailing 1). Rows
    labelled ``ignore_index`` have loss 0; another label outside [0, V) sets the device
    error flag. bf16 operands multiply on the tensor cores with fp32 sums; fp32 operands as
    two bf16 planes each (16 bits), or rounded to bf16 where ``Config.matmul_dtype`` is
    "bf16". Keep ``lse`` for LinearCrossEntropyGrad."""
    name = "LinearCrossEntropy"
    shape = x.shape[:-1]
    x, w, labels, ldx, ldw, dn, N, D, V = _head(name, x, w, labels)
    loss, lse = torch.empty(2, *shape, dtype=torch.float32, device=x.device).unbind(0)
    if N:
        dt, xp, wp = ops.code(x), x.data_ptr(), w.data_ptr()
        wn = L.lib().b200_linear_xent_workspace_bytes(dt, xp, ldx, wp, ldw, dn, N, D, V)
        ws = torch.empty(wn, dtype=torch.uint8, device=x.device)
        L.call("b200_linear_xent", dt, xp, ldx, wp, ldw, dn, labels.data_ptr(), ops.code(labels), int(ignore_index), loss.data_ptr(),
               lse.data_ptr(), N, D, V, ws.data_ptr(), wn, ops.stream_ptr())
    return loss, lse


def op_linear_cross_entropy_grad(dloss, x, w, labels, lse, ignore_index=-100, **_):
    """(dx, dw) of LinearCrossEntropy for the losses' gradient ``dloss`` (1 / N for a mean),
    in x's and w's dtype, rounded once to it whatever the operands are multiplied as; dw is
    stored as w is. ``lse`` as the forward returned it. Ignored
    rows give no gradient, whatever x holds there. The logits are made again, one piece of
    the vocabulary at a time: at most 512 MiB of their gradient at once up to 2^20 tokens (2^19
    of fp32 operands), 256 words of it beyond."""
    name = "LinearCrossEntropyGrad"
    x0, w0 = x, w
    x, w, labels, ldx, ldw, dn, N, D, V = _head(name, x, w, labels)
    lead = tuple(x0.shape[:-1])
    for t, what in ((dloss, "dloss"), (lse, "lse")):
        if t.numel() != N or tuple(t.shape) not in (lead, (*lead, 1)):
            raise ValueError(f"{name}: {what} {tuple(t.shape)} of x {tuple(x0.shape)}")
    _on_device(name, dloss, lse)
    dloss, lse = (ops.contiguous(ops.cast(t, torch.float32)) for t in (dloss, lse))
    dx = torch.empty(*lead, D, dtype=x0.dtype, device=x.device)
    dw = torch.empty((D, V) if dn else (V, D), dtype=w0.dtype, device=w.device)
    dt, xp, wp = ops.code(x), x.data_ptr(), w.data_ptr()
    wn = L.lib().b200_linear_xent_grad_workspace_bytes(dt, xp, ldx, wp, ldw, dn, N, D, V)
    ws = torch.empty(wn, dtype=torch.uint8, device=x.device)
    L.call("b200_linear_xent_grad_mixed", dt, dloss.data_ptr(), xp, ldx, wp, ldw, dn, labels.data_ptr(), ops.code(labels), int(ignore_index),
           lse.data_ptr(), dx.data_ptr(), ops.code(dx), dw.data_ptr(), ops.code(dw), N, D, V, ws.data_ptr(), wn, ops.stream_ptr())
    return dx, dw if dn else dw.t()


# ----------------------------------------------------------------------------------
# orthogonalised updates
# ----------------------------------------------------------------------------------

NEWTON_SCHULZ = (3.4445, -4.7750, 2.0315)  # steep at zero: 5 steps bring singular values from 0.01 into 0.7 .. 1.2


@functools.lru_cache(maxsize=64)
def _coefficients(steps: int, coefficients: tuple) -> Any:
    """The steps' (a, b, c) as the entry points take them: one triple for all, or one each."""
    each = any(isinstance(r, tuple) for r in coefficients)
    rows = coefficients if each else (coefficients,) * steps
    if not 1 <= steps <= 100 or len(rows) != steps or any(not isinstance(r, tuple) or len(r) != 3 for r in rows):
        raise ValueError(f"Newton-Schulz: {steps} steps (1 to 100) with coefficients {coefficients}: one (a, b, c), or one per step")
    return (ctypes.c_float * (3 * steps))(*[float(v) for r in rows for v in r])


def _coef(steps: int, coefficients: Any) -> Any:
    def plain(v: Any) -> Any:
        return v.tolist() if isinstance(v, (np.ndarray, torch.Tensor)) else v

    c = tuple(tuple(r) if isinstance(r, (list, tuple)) else r for r in map(plain, plain(coefficients)))
    return _coefficients(int(steps), c)


def _matrices(name: str, t: torch.Tensor) -> tuple[int, int, int]:
    if t.dim() < 2:
        raise ValueError(f"{name}: a matrix or a stack of matrices is wanted, got {tuple(t.shape)}")
    return math.prod(t.shape[:-2]), t.shape[-2], t.shape[-1]


def op_newton_schulz(g, steps=5, coefficients=NEWTON_SCHULZ, eps=1e-7, **_):
    """The nearest (semi-)orthogonal matrix of each g [..., rows, cols], approximately:
    X = g / (|g| + eps), then ``steps`` times X = a X + (b S + c S S) X with S = X X^T.

    fp32 or bf16 in and out. ``coefficients``: one (a, b, c) or one per step, finite, |a| below
    250; they have to keep the entries of X, S and a I + b S + c S S below 250 too (the default
    ones keep them below 4), or the result is infinite or NaN. Sums are fp32; the iterates carry
    22 bits for fp32 matrices, and for bf16 ones of up to 16 rows or columns, else 11."""
    name = "NewtonSchulz"
    if g.dtype not in _FLOATS:
        raise BackendNotSupportedError(f"{name}: matrices of {g.dtype} (fp32 and bf16)")
    batch, rows, cols = _matrices(name, g)
    coef = _coef(steps, coefficients)
    _on_device(name, g)
    gc = ops.contiguous(g)
    out = torch.empty(g.shape, dtype=g.dtype, device=g.device)
    wn = L.lib().b200_newton_schulz_workspace_bytes(ops.code(g), batch, rows, cols)
    ws = torch.empty(wn, dtype=torch.uint8, device=g.device)
    L.call("b200_newton_schulz", ops.code(g), gc.data_ptr(), out.data_ptr(), batch, rows, cols, coef, int(steps), float(eps),
           ws.data_ptr(), wn, ops.stream_ptr())
    return out


def op_apply_muon(param, momentum_buffer, grad, lr=None, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5,
                  coefficients=NEWTON_SCHULZ, eps=1e-7, out=None, output_axis=-2, **_):
    """One step of the orthogonalised momentum update for a matrix or a stack of matrices
    [..., rows, cols], beside ApplyAdam and the others: returns (param', momentum').

    momentum' = momentum * buffer + grad; G = grad + momentum * momentum' (nesterov) or
    momentum'; param' = param (1 - lr weight_decay) - lr sqrt(max(1, outputs / inputs))
    NewtonSchulz(G). ``output_axis``: the axis of the layer's outputs, -2 for matrices
    [outputs, inputs] (so rows / cols), -1 for Matmul weights [inputs, outputs]. fp32; lr 0.02
    unless given. ``out``: the tensors to write (dense; the inputs themselves for a step in
    place)."""
    name = "ApplyMuon"
    lr, weight_decay = 0.02 if lr is None else float(lr), float(weight_decay)
    batch, rows, cols = _matrices(name, param)
    if output_axis not in (-2, -1, param.dim() - 2, param.dim() - 1):
        raise ValueError(f"{name}: output_axis {output_axis} is not one of a matrix's two axes in {tuple(param.shape)}")
    if output_axis in (-1, param.dim() - 1) and rows and cols:
        # the entry point scales by sqrt(max(1, rows / cols)), and decays by lr weight_decay
        turn = math.sqrt(cols / rows)
        lr, weight_decay = lr * turn, weight_decay / turn
    if momentum_buffer.shape != param.shape or grad.shape != param.shape:
        raise ValueError(f"{name}: param, momentum and grad must have one shape, got {tuple(param.shape)}, "
                         f"{tuple(momentum_buffer.shape)}, {tuple(grad.shape)}")
    coef = _coef(steps, coefficients)
    _on_device(name, param, momentum_buffer, grad, *(out or ()))
    p, m, g = (ops.contiguous(ops.cast(t, torch.float32)) for t in (param, momentum_buffer, grad))
    if out is None:
        out = (torch.empty_like(p), torch.empty_like(m))
    po, mo = out
    for t in out:
        if t.shape != p.shape or t.dtype != torch.float32 or not t.is_contiguous():
            raise ValueError(f"{name}: results must be dense fp32 {tuple(p.shape)}")
    apart = [(po, t) for t in (m, g, mo)] + [(mo, t) for t in (p, g)]
    apart += [(o, t) for o, t in ((po, p), (mo, m)) if o.data_ptr() != t.data_ptr()]
    if any(abs(o.data_ptr() - t.data_ptr()) < 4 * p.numel() for o, t in apart):
        raise ValueError(f"{name}: a result may be written over its own input only (param', momentum')")
    wn = L.lib().b200_newton_schulz_workspace_bytes(L.F32, batch, rows, cols)
    ws = torch.empty(wn, dtype=torch.uint8, device=p.device)
    L.call("b200_apply_muon_f32", p.data_ptr(), m.data_ptr(), g.data_ptr(), po.data_ptr(), mo.data_ptr(), batch, rows, cols, lr,
           float(momentum), int(bool(nesterov)), weight_decay, coef, int(steps), float(eps), ws.data_ptr(), wn, ops.stream_ptr())
    return po, mo


def register(table: dict) -> None:
    table.update({
        "RotaryEmbedding": op_rotary_embedding,
        "RotaryEmbeddingGrad": op_rotary_embedding_grad,
        "QKNormRotary": op_qk_norm_rotary,
        "QKNormRotaryGrad": op_qk_norm_rotary_grad,
        "LinearCrossEntropy": op_linear_cross_entropy,
        "LinearCrossEntropyGrad": op_linear_cross_entropy_grad,
        "NewtonSchulz": op_newton_schulz,
        "ApplyMuon": op_apply_muon,
    })
