"""Operators of a transformer block: attention without the scores in memory, the learned position
bias, and the residual sum with its norms.

Like ``lm_ops``: values are ``torch.Tensor`` on the current CUDA device, results are fresh tensors,
all arithmetic runs in libb200.so, gradients are separate operators, ``execute_op`` reaches them by
name. The chain that they replace in a graph is Matmul, Multiply, Softmax, Matmul (attention) and
LayerNorm, Multiply, Add (the residual sum).
"""

from __future__ import annotations

import ctypes
import functools
import math
from typing import Any

import torch

from . import _lib as L
from . import ops
from .errors import BackendNotSupportedError
from .lm_ops import _FLOATS, _on_device

# ----------------------------------------------------------------------------------
# learned position bias
# ----------------------------------------------------------------------------------


def relative_bucket_starts(side: int, max_distance: int) -> list[int]:
    """The smallest distance of each of one side's ``side`` buckets: half of them one distance
    each, the others equal steps of the logarithm from there to ``max_distance``, behind which all
    share the last. Bucket side / 2 + i starts at the first distance n with
    floor(log(n / near) / log(max_distance / near) (side - near)) = i, near = side // 2; compared
    in whole numbers, since the steps may end on one."""
    near = side // 2
    wide = side - near
    starts, d = list(range(near)), near
    for i in range(wide):
        while d**wide < near ** (wide - i) * max_distance**i:
            d += 1
        starts.append(d)
    return starts


@functools.lru_cache(maxsize=64)
def _relative(buckets: int, max_distance: int, bidirectional: bool) -> L.Relative:
    side, odd = divmod(buckets, 2) if bidirectional else (buckets, 0)
    if odd or not 2 <= side <= L.RELATIVE_MAX_SIDE:
        raise ValueError(f"relative bias: {buckets} buckets; want 2 to {L.RELATIVE_MAX_SIDE} a side, as many on both")
    if not side // 2 < max_distance <= L.RELATIVE_MAX_FAR:
        raise ValueError(f"relative bias: max_distance {max_distance} not in ({side // 2}, {L.RELATIVE_MAX_FAR}] for {buckets} buckets")
    r = L.Relative()
    r.side, r.bidirectional = side, int(bidirectional)
    for i, d in enumerate(relative_bucket_starts(side, max_distance)):
        r.start[i] = d
    return r


def _count(name: str, what: str, n: Any) -> int:
    if n is None or int(n) != n or n < 0:
        raise ValueError(f"{name}: {what} {n!r} is not a number of tokens")
    return int(n)


def _shift(name: str, shift: Any, queries: int, keys: int) -> int:
    n = keys - queries if shift is None else int(shift)
    if abs(n) >= L.RELATIVE_MAX_SHIFT:
        raise ValueError(f"{name}: shift {n} of {queries} queries and {keys} keys (below 2^29)")
    return n


def op_relative_position_bias(table, queries=None, keys=None, bidirectional=True, max_distance=128, shift=None, **_):
    """The learned bias of every query and key, [heads, queries, keys] of the table's type, to
    be added to scores: ``table[bucket(rel), head]`` for rel = key - query - shift.

    table [buckets, heads], fp32 or bf16. Half of the buckets (of each side, ``bidirectional``: keys
    behind the query use the second half; else they share the first bucket) hold one distance each,
    the others equal steps of the logarithm up to ``max_distance`` (``relative_bucket_starts``).
    ``shift`` (below 2^29 either way): keys - queries by default, the last query at the last key."""
    name = "RelativePositionBias"
    if table.dim() != 2:
        raise ValueError(f"{name}: table {tuple(table.shape)}, want [buckets, heads]")
    if table.dtype not in _FLOATS:
        raise BackendNotSupportedError(f"{name}: table of {table.dtype} (fp32 and bf16)")
    nq, nk = _count(name, "queries", queries), _count(name, "keys", keys)
    shift = _shift(name, shift, nq, nk)
    r = _relative(table.shape[0], int(max_distance), bool(bidirectional))
    _on_device(name, table)
    table = ops.contiguous(table)
    out = torch.empty(table.shape[1], nq, nk, dtype=table.dtype, device=table.device)
    L.call("b200_relative_bias", r, ops.code(table), table.data_ptr(), out.data_ptr(), table.shape[1], nq, nk, shift,
           ops.stream_ptr())
    return out


def op_relative_position_bias_grad(dscores, buckets=None, bidirectional=True, max_distance=128, shift=None, **_):
    """The gradient of RelativePositionBias's table, [buckets, heads] of the scores' type, from
    that of the scores, [..., heads, queries, keys]: summed over each bucket and all leading axes,
    in fp32 and a fixed order."""
    name = "RelativePositionBiasGrad"
    if dscores.dim() < 3:
        raise ValueError(f"{name}: scores {tuple(dscores.shape)}, want [..., heads, queries, keys]")
    if dscores.dtype not in _FLOATS:
        raise BackendNotSupportedError(f"{name}: scores of {dscores.dtype} (fp32 and bf16)")
    heads, nq, nk = dscores.shape[-3:]
    buckets = _count(name, "buckets", buckets)
    shift = _shift(name, shift, nq, nk)
    r = _relative(buckets, int(max_distance), bool(bidirectional))
    _on_device(name, dscores)
    d = ops.contiguous(dscores)
    out = torch.empty(buckets, heads, dtype=d.dtype, device=d.device)
    wn = L.lib().b200_relative_bias_grad_workspace_bytes(r, heads, nq, nk)
    ws = torch.empty(wn, dtype=torch.uint8, device=d.device)
    L.call("b200_relative_bias_grad", r, ops.code(d), d.data_ptr(), out.data_ptr(), math.prod(d.shape[:-3]), heads, nq, nk, shift,
           ws.data_ptr(), wn, ops.stream_ptr())
    return out


# ----------------------------------------------------------------------------------
# attention
# ----------------------------------------------------------------------------------


def _tokens(name: str, what: str, x: torch.Tensor) -> torch.Tensor:
    """x [batch, tokens, heads, dim] with adjacent head elements."""
    if x.dim() != 4:
        raise ValueError(f"{name}: {what} {tuple(x.shape)}, want [batch, tokens, heads, dim] or [tokens, heads, dim]")
    return ops.contiguous(x) if x.stride(3) != 1 and x.shape[3] > 1 else x


def _window(name: str, window: Any) -> int:
    """The window in tokens, 0 for none; one longer than any sequence is cut, so that it stays itself in C."""
    if window is None:
        return 0
    if not window >= 1 or (window != math.inf and int(window) != window):
        raise ValueError(f"{name}: window {window!r} is not a number of tokens")
    return int(min(window, L.ATTENTION_MAX_WINDOW))


def _lengths(name: str, what: str, n: Any, batch: int) -> torch.Tensor | None:
    if n is None:
        return None
    t = n if isinstance(n, torch.Tensor) else torch.as_tensor(n)
    if tuple(t.shape) != (batch,):
        raise ValueError(f"{name}: {what} {tuple(t.shape)} of {batch} sequences")
    if t.dtype.is_floating_point or t.dtype == torch.bool:
        raise BackendNotSupportedError(f"{name}: {what} of {t.dtype} (integers)")
    t = ops.to_device(t)
    _on_device(name, t)
    if t.dtype not in (torch.int32, torch.int64):
        t = ops._int_indices(t)
    return ops.contiguous(t)


@functools.lru_cache(maxsize=256)
def _attention_plan(name, shapes, dtypes, table, scale, causal, window, max_distance, bidirectional) -> L.Attention:
    """The checks of shapes and types, and what of the description they decide."""
    for s, d, what in zip(shapes, dtypes, ("queries", "keys", "values")):
        if len(s) != 4:
            raise ValueError(f"{name}: {what} {tuple(s)}, want [batch, tokens, heads, dim] or [tokens, heads, dim]")
        if d not in _FLOATS:
            raise BackendNotSupportedError(f"{name}: {what} of {d} (fp32 and bf16)")
    (b, nq, h, d), (kb, nk, hk, kd) = shapes[:2]
    if shapes[1] != shapes[2] or kb != b or kd != d:
        raise ValueError(f"{name}: queries {tuple(shapes[0])}, keys {tuple(shapes[1])} and values {tuple(shapes[2])} do not match")
    if dtypes[1] != dtypes[0] or dtypes[2] != dtypes[0]:
        raise BackendNotSupportedError(f"{name}: queries of {dtypes[0]} with keys of {dtypes[1]} and values of {dtypes[2]}")
    if not 1 <= d <= L.ATTENTION_MAX_DIM:
        raise ValueError(f"{name}: heads of {d} elements (1 to {L.ATTENTION_MAX_DIM})")
    if h < 1 or hk < 1 or h % hk:
        raise ValueError(f"{name}: {h} heads over {hk} key heads")
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"{name}: scale {scale} is not a positive number")
    a = L.Attention()
    if table is not None:
        shape, dtype = table
        if len(shape) != 2 or shape[1] != h:
            raise ValueError(f"{name}: position bias {tuple(shape)}, want [buckets, {h} heads]")
        if dtype not in _FLOATS:
            raise BackendNotSupportedError(f"{name}: position bias of {dtype} (fp32 and bf16)")
        a.relative = _relative(shape[0], int(max_distance), not causal if bidirectional is None else bool(bidirectional))
        a.table_dtype = ops._TORCH2CODE[dtype]
    a.batch, a.queries, a.keys, a.heads, a.kv_heads, a.dim = b, nq, nk, h, hk, d
    a.window, a.causal, a.scale, a.dtype = window, int(bool(causal)), scale, ops._TORCH2CODE[dtypes[0]]
    return a


def _describe(name: str, q, k, v, lengths, query_lengths, table, scale, causal, window, max_distance, bidirectional):
    """(description, the tensors that it points to, whether the batch axis was left out)."""
    flat = q.dim() == 3
    if flat:
        if k.dim() != 3 or v.dim() != 3:
            raise ValueError(f"{name}: queries {tuple(q.shape)}, keys {tuple(k.shape)} and values {tuple(v.shape)}: all with the batch axis or none")
        q, k, v = q.unsqueeze(0), k.unsqueeze(0), v.unsqueeze(0)
    plan = _attention_plan(name, (q.shape, k.shape, v.shape), (q.dtype, k.dtype, v.dtype), None if table is None else (table.shape, table.dtype),
                           None if scale is None else float(scale), bool(causal), _window(name, window), int(max_distance),
                           None if bidirectional is None else bool(bidirectional))
    a = L.Attention.from_buffer_copy(plan)
    _on_device(name, q, k, v, table)
    q, k, v = _tokens(name, "queries", q), _tokens(name, "keys", k), _tokens(name, "values", v)
    if lengths is not None or query_lengths is not None:
        lengths, query_lengths = (_lengths(name, what, n, q.shape[0]) for n, what in ((lengths, "lengths"), (query_lengths, "query_lengths")))
        if lengths is not None and query_lengths is not None and lengths.dtype != query_lengths.dtype:
            lengths, query_lengths = (ops.cast(t, torch.int64) for t in (lengths, query_lengths))
        a.length_dtype = ops.code(query_lengths if lengths is None else lengths)
        a.lengths, a.query_lengths = ops._ptr(lengths), ops._ptr(query_lengths)
    if table is not None:
        table = ops.contiguous(table)
        a.table = table.data_ptr()
    a.q, a.k, a.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    a.q_stride[:], a.k_stride[:], a.v_stride[:] = q.stride()[:3], k.stride()[:3], v.stride()[:3]
    return a, (q, k, v, lengths, query_lengths, table), flat


def op_attention(q, k, v, lengths=None, query_lengths=None, relative_bias=None, scale=None, causal=False, window=None,
                       max_distance=128, bidirectional=None, **_):
    """Attention without the scores in memory: (out, lse), out_i = sum_j softmax_j(z_i) v_j for
    z_ij = scale q_i . k_j (+ the position bias), lse_i = log sum_j exp z_ij.

    q [batch, queries, heads, dim], k and v [batch, keys, kv_heads, dim] (or all without the
    batch), of one type, fp32 or bf16, any strides (slices of one projection are read in place;
    head-major tensors are passed as their transposed views); dim <= 256; heads is a multiple of
    kv_heads, neighbouring heads share a key head. ``scale``: 1 / sqrt(dim). out is dense, in q's
    shape and type; lse fp32 [batch, heads, queries].

    ``lengths`` and ``query_lengths`` (integers [batch]) end each sequence's keys and queries: a padded
    batch, or a cache that is not full. What lies behind them may be anything, NaN too; keys and values inside
    are finite (one that a mask hides is still a factor of zero). The last query is at the last key's
    position: query i at i + keys - queries of its sequence. ``causal`` hides the keys behind a
    query's position, ``window`` w those w or more before it (and, not causal, behind it). A query that
    sees nothing has out 0 and lse -inf. ``relative_bias`` [buckets, heads]: the table of
    RelativePositionBias, added to the scores by the positions' difference (``bidirectional``: not
    causal by default); entries finite or -inf.

    Scores, their maxima and sums are fp32; bf16 heads round the probabilities to bf16 for their
    product with the values, whatever ``Config.matmul_dtype`` is: cast heads to fp32 for fp32 products. Keep
    ``lse`` and ``out`` for AttentionGrad."""
    name = "Attention"
    a, kept, flat = _describe(name, q, k, v, lengths, query_lengths, relative_bias, scale, causal, window, max_distance, bidirectional)
    x = kept[0]
    out = x.new_empty(x.shape)
    lse = x.new_empty((a.batch, a.heads, a.queries), dtype=torch.float32)
    wn = L.lib().b200_attention_workspace_bytes(a)
    ws = x.new_empty(wn, dtype=torch.uint8) if wn else None
    L.call("b200_attention_forward", a, out.data_ptr(), lse.data_ptr(), ops._ptr(ws), wn, ops.stream_ptr())
    return (out[0], lse[0]) if flat else (out, lse)


def op_attention_grad(dout, q, k, v, out, lse, lengths=None, query_lengths=None, relative_bias=None, scale=None, causal=False,
                            window=None, max_distance=128, bidirectional=None, **_):
    """(dq, dk, dv, dtable) of Attention for its output's gradient ``dout``; ``out`` and ``lse`` as
    the forward returned them, the rest as it took it. The probabilities are made again from lse.

    Each is dense, in the shape and type of what it is the gradient of, rounded once; the heads that
    share a key head are summed, dtable (None without ``relative_bias``) over batch and positions.
    Queries and keys behind their sequence's end have zeros. The same from run to run. bf16 heads round the
    probabilities and the scores' gradients to bf16 for their products, and ``out`` is the rounded one (so is
    dout . out of each query, of which an fp32 table's gradient is off as well).

    Probabilities exp(z - lse) are off by the fp32 rounding of lse, up to 2e-7 |lse| of each: hide keys by
    lengths, ``causal``, ``window`` or table entries of -inf rather than by large negative ones. A query whose
    visible scores are all that large (|lse| >= 2^20) gets no gradient, and sets the device error flag where
    its row of dout is not zero; a large negative entry beside others is no harm."""
    name = "AttentionGrad"
    a, kept, flat = _describe(name, q, k, v, lengths, query_lengths, relative_bias, scale, causal, window, max_distance, bidirectional)
    x, y, table = kept[0], kept[1], kept[5]
    if tuple(dout.shape) != tuple(q.shape) or tuple(out.shape) != tuple(q.shape):
        raise ValueError(f"{name}: gradient {tuple(dout.shape)} and output {tuple(out.shape)} of queries {tuple(q.shape)}")
    if dout.dtype != x.dtype or out.dtype != x.dtype:
        raise BackendNotSupportedError(f"{name}: gradient of {dout.dtype} and output of {out.dtype} for {x.dtype} heads")
    want = (a.heads, a.queries) if flat else (a.batch, a.heads, a.queries)
    if tuple(lse.shape) != want or lse.dtype != torch.float32:
        raise ValueError(f"{name}: lse {tuple(lse.shape)} of {lse.dtype}, want fp32 {want}")
    _on_device(name, dout, out, lse)
    dout = _tokens(name, "gradient", dout.unsqueeze(0) if flat else dout)
    out, lse = ops.contiguous(out), ops.contiguous(lse)
    g = L.AttentionGrads()
    dq, dk, dv = x.new_empty(x.shape), y.new_empty(y.shape), y.new_empty(y.shape)
    dtable = None if table is None else table.new_empty(table.shape)
    g.dout, g.out, g.lse, g.dout_stride[:] = dout.data_ptr(), out.data_ptr(), lse.data_ptr(), dout.stride()[:3]
    g.dq, g.dk, g.dv, g.dtable = dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), ops._ptr(dtable)
    wn = L.lib().b200_attention_grad_workspace_bytes_of(a, g)
    ws = x.new_empty(wn, dtype=torch.uint8) if wn else None
    L.call("b200_attention_grad", a, g, ops._ptr(ws), wn, ops.stream_ptr())
    return (dq[0], dk[0], dv[0], dtable) if flat else (dq, dk, dv, dtable)


# ----------------------------------------------------------------------------------
# residual sum and its norms
# ----------------------------------------------------------------------------------

_NORMS = {"rms": 0, "layer": 1}


@functools.lru_cache(maxsize=256)
def _residual_plan(name, shape, f_shape, x_dtype, f_dtype, weights, gate, residual_scale, norm, post_norm, eps) -> L.ResidualNorm:
    """The checks of shapes and types (weights, gate: (shape, dtype) or None), and what of the description they decide."""
    if shape != f_shape or len(shape) < 1:
        raise ValueError(f"{name}: residual stream {tuple(shape)} and block output {tuple(f_shape)} differ")
    for d, what in ((x_dtype, "residual stream"), (f_dtype, "block output")):
        if d not in _FLOATS:
            raise BackendNotSupportedError(f"{name}: {what} of {d} (fp32 and bf16)")
    if norm not in _NORMS:
        raise ValueError(f"{name}: norm {norm!r} is not one of {sorted(_NORMS)}")
    width = shape[-1]
    if not 1 <= width <= L.RESIDUAL_NORM_MAX_COLS:
        raise ValueError(f"{name}: rows of {width} elements (1 to {L.RESIDUAL_NORM_MAX_COLS})")
    given = weights[2] is not None or weights[3] is not None
    post = given if post_norm is None else bool(post_norm)
    if given and not post:
        raise ValueError(f"{name}: post weights without a post norm")
    if norm != "layer" and (weights[1] is not None or weights[3] is not None):
        raise ValueError(f"{name}: an RMS norm has no beta")
    if not math.isfinite(residual_scale):
        raise ValueError(f"{name}: residual_scale {residual_scale} is not finite")
    for w in weights:
        if w is not None:
            if tuple(w[0]) != (width,):
                raise ValueError(f"{name}: norm weight {tuple(w[0])}, want [{width}]")
            if w[1] not in _FLOATS:
                raise BackendNotSupportedError(f"{name}: norm weights of {w[1]} (fp32 and bf16)")
    d = L.ResidualNorm()
    if gate is not None:
        if gate[1] not in _FLOATS:
            raise BackendNotSupportedError(f"{name}: gate of {gate[1]} (fp32 and bf16)")
        lead = tuple(shape[:-1])
        g = (1,) * (len(shape) - len(gate[0])) + tuple(gate[0])
        # leading axes in full, then axes of one: consecutive rows share a gate
        n = next((i for i in range(len(lead)) if len(g) == len(shape) and g[i] != lead[i]), len(lead))
        if len(g) != len(shape) or g[-1] != width or any(s != 1 for s in g[n:-1]):
            raise ValueError(f"{name}: gate {tuple(gate[0])} of {tuple(shape)}: want leading axes in full, then ones, then {width}")
        d.groups, d.gate_dtype = math.prod(g[:n]), ops._TORCH2CODE[gate[1]]
    d.rows, d.cols = math.prod(shape[:-1]), width
    if not d.rows:
        d.groups = 0
    d.kind, d.post, d.scale, d.eps = _NORMS[norm], int(post), float(residual_scale), float(eps)
    d.x_dtype, d.f_dtype = ops._TORCH2CODE[x_dtype], ops._TORCH2CODE[f_dtype]
    kinds = {w[1] for w in weights if w is not None}
    d.weight_dtype = L.BF16 if kinds == {torch.bfloat16} else L.F32  # fp32 where they differ
    return d


def _residual(name: str, x, f, gamma, beta, post_gamma, post_beta, gate, residual_scale, norm, post_norm, eps):
    """(description, x, f, the weights as the kernels take them, the gate)."""
    weights = (gamma, beta, post_gamma, post_beta)
    plan = _residual_plan(name, x.shape, f.shape, x.dtype, f.dtype, tuple([None if w is None else (w.shape, w.dtype) for w in weights]),
                          None if gate is None else (gate.shape, gate.dtype), float(residual_scale), norm, None if post_norm is None else bool(post_norm),
                          float(eps))
    _on_device(name, x, f, gate, *weights)
    d = L.ResidualNorm.from_buffer_copy(plan)
    kind = torch.bfloat16 if d.weight_dtype == L.BF16 else torch.float32
    weights = [None if w is None else ops.contiguous(ops.cast(w, kind)) for w in weights]
    d.gamma, d.beta, d.post_gamma, d.post_beta = [None if w is None else w.data_ptr() for w in weights]
    if gate is not None:
        gate = ops.contiguous(gate)
        d.gate = gate.data_ptr() if d.rows else None
    return d, ops.contiguous(x), ops.contiguous(f), weights, gate


def op_residual_norm(x, f, gamma=None, beta=None, post_gamma=None, post_beta=None, gate=None, residual_scale=1.0, norm="rms",
                     post_norm=None, eps=1e-6, **_):
    """A block's output added to the residual stream, with the norms on both sides of the sum, in
    one pass: (sum, normed), sum = residual_scale x + gate N(f; post_gamma, post_beta), normed =
    N(sum; gamma, beta), which the next block reads.

    x and f [..., width] in one shape, fp32 or bf16 each (an fp32 stream with bf16 blocks too); sum is
    of x's type, normed of f's. ``norm``: "rms" or "layer" (with betas), over the last axis, width <=
    16384; a gamma of None is ones. ``post_norm``: whether f is normed first (by default where it has
    weights). ``gate``: [width], or x's leading axes and then ones ([batch, 1, width], one gate a
    sequence), or x's shape; None: ones. Computed in fp32, rounded once each."""
    name = "ResidualNorm"
    d, x, f, weights, gate = _residual(name, x, f, gamma, beta, post_gamma, post_beta, gate, residual_scale, norm, post_norm, eps)
    total, normed = torch.empty_like(x), torch.empty_like(f)
    L.call("b200_residual_norm_forward", d, x.data_ptr(), f.data_ptr(), total.data_ptr(), normed.data_ptr(), ops.stream_ptr())
    return total, normed


def op_residual_norm_grad(dsum, dnormed, x, f, gamma=None, beta=None, post_gamma=None, post_beta=None, gate=None, residual_scale=1.0,
                          norm="rms", post_norm=None, eps=1e-6, **_):
    """The gradients of ResidualNorm from those of its results and its inputs: (dx, df, dgamma,
    dbeta, dpost_gamma, dpost_beta, dgate), None for weights that were not given, each in the type
    and shape of what it is the gradient of. The sum and its norms are made again; the weights' sums over
    rows are fp32, in a fixed order."""
    name = "ResidualNormGrad"
    given = (gamma, beta, post_gamma, post_beta)
    shape = None if gate is None else gate.shape
    d, x, f, weights, gate = _residual(name, x, f, gamma, beta, post_gamma, post_beta, gate, residual_scale, norm, post_norm, eps)
    if dsum.shape != x.shape or dnormed.shape != x.shape:
        raise ValueError(f"{name}: gradients {tuple(dsum.shape)}, {tuple(dnormed.shape)} of {tuple(x.shape)}")
    if dsum.dtype != x.dtype or dnormed.dtype != f.dtype:
        raise BackendNotSupportedError(f"{name}: gradients of {dsum.dtype}, {dnormed.dtype} for a sum of {x.dtype} and norms of {f.dtype}")
    _on_device(name, dsum, dnormed)
    dsum, dnormed = ops.contiguous(dsum), ops.contiguous(dnormed)
    dx, df = torch.empty_like(x), torch.empty_like(f)
    grads = [None if w is None else torch.empty_like(w) for w in weights]
    dgate = None if gate is None else gate.new_empty(shape)
    g = L.ResidualNormGrads()
    g.dgamma, g.dbeta, g.dpost_gamma, g.dpost_beta = (ops._ptr(t) for t in grads)
    g.dgate = ops._ptr(dgate)
    wn = L.lib().b200_residual_norm_grad_workspace_bytes(d)
    ws = x.new_empty(wn, dtype=torch.uint8) if wn else None
    L.call("b200_residual_norm_grad", d, dsum.data_ptr(), dnormed.data_ptr(), x.data_ptr(), f.data_ptr(), dx.data_ptr(), df.data_ptr(), g,
           ops._ptr(ws), wn, ops.stream_ptr())
    if dgate is not None and not d.rows:
        dgate = ops.full(tuple(shape), 0.0, dgate.dtype) if dgate.numel() else dgate
    grads = [t if t is None else ops.cast(t, w.dtype) for t, w in zip(grads, given)]
    return dx, df, *grads, dgate


def register(table: dict) -> None:
    table.update({
        "Attention": op_attention,
        "AttentionGrad": op_attention_grad,
        "RelativePositionBias": op_relative_position_bias,
        "RelativePositionBiasGrad": op_relative_position_bias_grad,
        "ResidualNorm": op_residual_norm,
        "ResidualNormGrad": op_residual_norm_grad,
    })
