"""Plain 64-bit forms of the block operators (attention, position bias, residual norms), with the
magnitude of the terms that each result is a sum of."""

import math

import torch

HALF_STEP = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8}  # a rounding's relative size at most


def bucket(rel, side, far, bidirectional):
    """Bucket of one relative position, from the logarithm's definition in whole numbers."""
    n = abs(rel) if bidirectional else max(0, -rel)
    near = side // 2
    if n < near:
        b = n
    else:
        wide, i = side - near, 0
        while i + 1 < wide and n**wide >= near ** (wide - i - 1) * far ** (i + 1):
            i += 1
        b = near + i
    return b + (side if bidirectional and rel > 0 else 0)


def bias_buckets(nq, nk, shift, buckets, far=128, bidirectional=True):
    side = buckets // 2 if bidirectional else buckets
    low = -(nq - 1) - shift
    by_rel = torch.tensor([bucket(r, side, far, bidirectional) for r in range(low, nk - shift)])
    return by_rel[torch.arange(nk)[None] - torch.arange(nq)[:, None] - shift - low]


def seen_keys(nq, nk, causal, window):
    """[nq, nk] of one sequence: query i at i + nk - nq."""
    pos, j = torch.arange(nq)[:, None] + nk - nq, torch.arange(nk)[None]
    seen = torch.ones(nq, nk, dtype=torch.bool)
    if causal:
        seen &= j <= pos
    if window:
        seen &= j > pos - window
        if not causal:
            seen &= j < pos + window
    return seen


def attention(q, k, v, dout=None, lengths=None, query_lengths=None, table=None, scale=None, causal=False, window=None, far=128,
              bidirectional=None):
    """Everything in float64 on the CPU: dicts of results and of their terms' magnitudes."""
    b, nq, h, d = q.shape
    nk, hk = k.shape[1:3]
    scale = d**-0.5 if scale is None else scale
    bidirectional = not causal if bidirectional is None else bidirectional
    zeros = lambda *s: torch.zeros(*s, dtype=torch.float64)  # noqa: E731
    r = {"out": zeros(b, nq, h, d), "lse": torch.full((b, h, nq), -math.inf, dtype=torch.float64)}
    m = {"out": zeros(b, nq, h, d), "lse": zeros(b, h, nq)}
    names = ["dq", "dk", "dv"] + (["dtable"] if table is not None else [])
    if dout is not None:
        for o in (r, m):
            o.update(dq=zeros(b, nq, h, d), dk=zeros(b, nk, hk, d), dv=zeros(b, nk, hk, d))
            if table is not None:
                o["dtable"] = zeros(*table.shape)
    for e in range(b):
        n = nk if lengths is None else int(lengths[e])
        w = nq if query_lengths is None else int(query_lengths[e])
        if n == 0 or w == 0:
            continue
        seen = seen_keys(w, n, causal, window)
        where = None if table is None else bias_buckets(w, n, n - w, table.shape[0], far, bidirectional)
        for a in range(h):
            g = a // (h // hk)
            Q, K, V = q[e, :w, a].double(), k[e, :n, g].double(), v[e, :n, g].double()
            z = Q @ K.t() * scale
            mag = Q.abs() @ K.abs().t() * scale
            if table is not None:
                t = table[:, a].double()[where]
                z, mag = z + t, mag + t.abs().nan_to_num(posinf=0.0)
            z = z.masked_fill(~seen, -math.inf)
            lse = torch.logsumexp(z, -1)
            empty = lse == -math.inf
            p = torch.exp(z - torch.where(empty, torch.zeros_like(lse), lse)[:, None])
            r["lse"][e, a, :w] = lse
            m["lse"][e, a, :w] = torch.where(empty, 0.0, (p * mag).sum(-1) + 1)
            o = p @ V
            # a score off by x of its terms moves its probability by as much
            r["out"][e, :w, a] = o
            p_mag = p * (1 + mag + (p * mag).sum(-1, keepdim=True))
            m["out"][e, :w, a] = p_mag @ V.abs()
            if dout is None:
                continue
            D = dout[e, :w, a].double()
            dz = p * (D @ V.t() - (D * o).sum(-1, keepdim=True))
            dz_mag = p_mag * (D.abs() @ V.abs().t() + (D.abs() * m["out"][e, :w, a]).sum(-1, keepdim=True))
            for out, P, Z, x in ((r, p, dz, lambda t: t), (m, p_mag, dz_mag, torch.abs)):
                out["dq"][e, :w, a] = Z @ x(K) * scale
                out["dk"][e, :n, g] += Z.t() @ x(Q) * scale
                out["dv"][e, :n, g] += P.t() @ x(D)
                if table is not None:
                    out["dtable"][:, a].index_add_(0, where.flatten(), Z.flatten())
    return {n: r[n] for n in ["out", "lse"] + (names if dout is not None else [])}, m


def stats(t, layer, eps):
    mean = t.mean(-1, keepdim=True) if layer else torch.zeros_like(t[..., :1])
    return mean, 1 / ((t - mean).pow(2).mean(-1, keepdim=True) + eps).sqrt()


def residual_norm(x, f, gamma=None, beta=None, post_gamma=None, post_beta=None, gate=None, scale=1.0, norm="rms", post=None, eps=1e-6,
                  dsum=None, dnormed=None):
    """(results, magnitudes) of the residual sum and its norms, float64, gradients with dsum and dnormed."""
    layer = norm == "layer"
    post = post_gamma is not None or post_beta is not None if post is None else post
    one = torch.ones(x.shape[-1], dtype=torch.float64)
    x, f = x.double(), f.double()
    gm, pg = (one if w is None else w.double() for w in (gamma, post_gamma))
    bt, pb = (0 * one if w is None else w.double() for w in (beta, post_beta))
    ga = one if gate is None else gate.double()
    p, pm = f, f.abs()
    if post:
        fm, fr = stats(f, layer, eps)
        fu = (f - fm) * fr
        fu_m = (f.abs() + f.abs().mean(-1, keepdim=True)) * fr
        p, pm = fu * pg + pb, fu_m * pg.abs() + pb.abs()
    s, sm = scale * x + ga * p, abs(scale) * x.abs() + ga.abs() * pm
    mean, rstd = stats(s, layer, eps)
    u = (s - mean) * rstd
    um = (sm + sm.mean(-1, keepdim=True)) * rstd
    um = um + u.abs() * (um * um).mean(-1, keepdim=True)
    r, m = {"sum": s, "normed": u * gm + bt}, {"sum": sm, "normed": um * gm.abs() + bt.abs()}
    if dsum is None:
        return r, m
    ds, dh = dsum.double(), dnormed.double()

    def back(d, dm, u, um, rstd):
        g = d - (d * u).mean(-1, keepdim=True) * u
        gmag = dm + (dm * um).mean(-1, keepdim=True) * um
        if layer:
            g, gmag = g - d.mean(-1, keepdim=True), gmag + dm.mean(-1, keepdim=True)
        # the reciprocal root's own error, from the terms that it is made of
        return rstd * g, rstd * gmag * (1 + (um * um).mean(-1, keepdim=True))

    lead = tuple(range(x.dim() - 1))
    r["dgamma"], m["dgamma"] = (dh * u).sum(lead), (dh.abs() * um).sum(lead)
    r["dbeta"], m["dbeta"] = dh.sum(lead), dh.abs().sum(lead)
    d, dm = back(dh * gm, (dh * gm).abs(), u, um, rstd)
    d, dm = d + ds, dm + ds.abs()
    r["dx"], m["dx"] = scale * d, abs(scale) * dm
    if gate is not None:
        shape = (1,) * (x.dim() - gate.dim()) + tuple(gate.shape)
        over = tuple(i for i in lead if shape[i] == 1)
        r["dgate"] = (d * p).sum(over, keepdim=True).reshape(gate.shape) if over else d * p
        m["dgate"] = (dm * pm).sum(over, keepdim=True).reshape(gate.shape) if over else dm * pm
    d, dm = d * ga, dm * ga.abs()
    if post:
        r["dpost_gamma"], m["dpost_gamma"] = (d * fu).sum(lead), (dm * fu_m).sum(lead)
        r["dpost_beta"], m["dpost_beta"] = d.sum(lead), dm.sum(lead)
        d, dm = back(d * pg, dm * pg.abs(), fu, fu_m, fr)
    r["df"], m["df"] = d, dm
    return r, m
