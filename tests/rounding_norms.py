"""How far the attention and residual-norm kernels' results may be off in the mean square, from the roundings that
their arithmetic makes, propagated to first order in 64 bits; and the comparison with it.

A rounding to bf16 is off by at most 2^-8 of the value and uniform over its step, so by U = 2^-8 / sqrt(3) in the mean
square at most, and independent of the others: squares add up. Attention of bf16 heads rounds the probabilities and dz
(as operands of the products), the output (and with it delta = dout . out of each query, one error for its
whole row) and every result. What is fp32: a sum of products has at most 24 roundings or cuts of 2^-23 on a term's
way, each of a partial sum below the product of the norms, so sqrt(24) 2^-23 / sqrt(3) < 6 x 2^-24 of that; with the
scale, bias, maximum and sums behind it 10 x 2^-24 is taken.

A result's error over `n` values then has the norm sqrt(sum of the variances), within a factor that depends on n
alone: 3 is allowed for a head, 6 for each of its rows (thousands of rows, whose common error delta is one number
each)."""

import math

import torch

import block_reference as R

U = {torch.bfloat16: 2.0**-8 / math.sqrt(3), torch.float32: 2.0**-24 / math.sqrt(3)}
E32 = 10 * 2.0**-24


def attention_noise(q, k, v, dout=None, lengths=None, query_lengths=None, table=None, scale=None, causal=False, window=None, far=128,
                    bidirectional=None):
    """Variances of out (and dq, dk, dv, dtable with dout), in their shapes; arguments as block_reference.attention."""
    b, nq, h, d = q.shape
    nk, hk = k.shape[1:3]
    scale = d**-0.5 if scale is None else scale
    bidirectional = not causal if bidirectional is None else bidirectional
    inner, own = (U[q.dtype] if q.dtype == torch.bfloat16 else 0.0), U[q.dtype]
    ref, _ = R.attention(q, k, v, dout, lengths, query_lengths, table, scale, causal, window, far, bidirectional)
    var = {n: (own * t) ** 2 for n, t in ref.items() if n != "lse"}
    if table is not None and dout is not None:
        var["dtable"] = (U[table.dtype] * ref["dtable"]) ** 2
    for e in range(b):
        n = nk if lengths is None else int(lengths[e])
        w = nq if query_lengths is None else int(query_lengths[e])
        if n == 0 or w == 0:
            continue
        seen = R.seen_keys(w, n, causal, window)
        where = None if table is None else R.bias_buckets(w, n, n - w, table.shape[0], far, bidirectional)
        for a in range(h):
            g = a // (h // hk)
            Q, K, V = q[e, :w, a].double(), k[e, :n, g].double(), v[e, :n, g].double()
            z = Q @ K.t() * scale
            ez = E32 * (scale * Q.norm(dim=1)[:, None] * K.norm(dim=1)[None] + 1)
            if table is not None:
                t = table[:, a].double()[where]
                z, ez = z + t, ez + E32 * t.abs().nan_to_num(posinf=0.0)
            z = z.masked_fill(~seen, -math.inf)
            lse = ref["lse"][e, a, :w]
            empty = lse == -math.inf
            p = torch.exp(z - torch.where(empty, torch.zeros_like(lse), lse)[:, None])
            el2 = (p * ez * ez).sum(-1, keepdim=True) + E32**2  # of lse: the scores' weighted errors, and its own
            ez2 = ez * ez
            vp = p * p * (inner**2 + ez2 + el2 + E32**2)
            vout = vp @ (V * V)
            var["out"][e, :w, a] += vout
            if dout is None:
                continue
            D, o = dout[e, :w, a].double(), p @ V
            dp, delta = D @ V.t(), (D * o).sum(-1, keepdim=True)
            vdelta = ((D * D) * (vout + (own * o) ** 2)).sum(-1, keepdim=True) + (E32 * D.norm(dim=1) * o.norm(dim=1))[:, None] ** 2
            dz = p * (dp - delta)
            e_dp = E32 * D.norm(dim=1)[:, None] * V.norm(dim=1)[None]
            v32 = dz * dz * (ez2 + el2 + E32**2) + (p * e_dp) ** 2
            vdz = v32 + (inner * dz) ** 2
            var["dq"][e, :w, a] += scale**2 * (vdz @ (K * K) + vdelta * (p @ K) ** 2)
            var["dk"][e, :n, g] += scale**2 * ((vdz + vdelta * p * p).t() @ (Q * Q))
            var["dv"][e, :n, g] += vp.t() @ (D * D)
            if table is not None:
                # each query's delta moves all of a bucket's dz in it
                in_bucket = torch.zeros(w, table.shape[0], dtype=torch.float64).scatter_add_(1, where, p)
                var["dtable"][:, a] += (vdelta * in_bucket**2).sum(0)
                var["dtable"][:, a].index_add_(0, where.flatten(), v32.flatten())
    return ref, var


def by_head(name, t):
    """A result as [slices, rows, values]: the sequences' heads, or the table's heads (one value a row)."""
    if name == "dtable":
        return t.t()[:, :, None]
    return t.transpose(1, 2).flatten(0, 1)


def off_by_norm(got, ref, var):
    """None, or what of got [slices, rows, values] is off by more than its roundings."""
    off2, var = (got.double() - ref) ** 2, var + 1e-60
    if not off2.isfinite().all():
        return "not finite"
    whole = (off2.sum((1, 2)) / var.sum((1, 2))).sqrt()
    if whole.numel() and float(whole.max()) > 3:
        return f"slice {int(whole.argmax())}: {float(whole.max()):.3g} times its roundings"
    row = (off2.sum(2) / var.sum(2)).sqrt()
    if row.numel() and float(row.max()) > 6:
        return f"row {int(row.argmax())} of {tuple(row.shape)}: {float(row.max()):.3g} times its roundings"
    return None


def attention_off(name, got, ref, var):
    return off_by_norm(by_head(name, got.cpu()), by_head(name, ref[name]), by_head(name, var[name]))


def residual_off(name, got, ref, rows=False):
    """None, or how a result of the residual norm or of its gradient differs from the 64-bit one.

    `rows` (sum, normed, dx, df, an element's gate): their statistics are trees of at most 53 roundings, sqrt(53) 2^-24 / sqrt(3) =
    2.5e-7 in the mean square, six of them in the gradient and 20 roundings of an element's own: below 1e-6; ten times that is
    allowed of a row's norm, or of the rows' mean one where a row's terms cancel. Weights: sums of at most 64 rows in a thread and
    1000 blocks in eight slices, sqrt(200) 2^-24 / sqrt(3) = 5e-7 of terms that grow as their sum does: the same 1e-5 of the
    vector's norm. One value of thousands: ten times the mean one, 1e-4. A result of bf16: 2^-8 of each value at most, so of the
    norm."""
    want = ref.reshape(-1, ref.shape[-1]) if rows else ref.reshape(1, -1)
    off, norm = (got.cpu().double().reshape(want.shape) - want).abs(), want.norm(dim=1)
    if not off.isfinite().all():
        return f"{name}: not finite"
    half, norm32 = R.HALF_STEP[got.dtype], torch.maximum(norm, norm.pow(2).mean().sqrt())
    worst = float((off.norm(dim=1) / (half * norm + 1e-5 * norm32 + 1e-60)).max())
    one = float((off / (half * want.abs() + 1e-4 * norm32[:, None] / math.sqrt(want.shape[1]) + 1e-60)).max())
    return f"{name}: {worst:.3g} times the tolerance of the norm, {one:.3g} of a value" if max(worst, one) > 1 else None
