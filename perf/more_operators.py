"""Cases that measure the attention, position-bias and residual-norm operators of the b200 backend.

The operators of a decoder or encoder block's training step and of its single-token serving form:

* ``Attention`` (and its gradient, which makes the probabilities again from the saved
  log-sum-exp): shared key heads, causal or not, sequences padded at their ends, a cache
  longer than what it holds, a learned bias by relative position;
* ``RelativePositionBias`` (and its gradient): that bias on its own, for scores in memory;
* ``ResidualNorm`` (and its gradient): a block's output normed, gated and added to the scaled
  residual stream, and the norm of the sum that the next block reads.

``run`` computes them in their plain form (elementary torch operations in 32 bits), or through
the backend's public entry point where ``own`` is true. ``exact`` gives the same values from
the definitions in 64 bits.
"""

import math

import torch

own = False

EPS = 1e-5
BUCKETS, FAR = 32, 128  # buckets of a learned position bias, and the distance from which all share the last


def listed():
    """The measured cases."""
    return [
        # one new token of one sequence against its cache
        attention("attn_token", batch=1, queries=1, keys=3001, heads=32, kv_heads=8, dim=128, dtype="bf16", causal=True),
        # a decoding batch: caches of 4096 places, each filled to a length of its own
        attention("attn_decode", batch=32, queries=1, keys=4096, heads=32, kv_heads=8, dim=128, dtype="bf16", causal=True, padded=True),
        # a prompt of two sequences with an odd length, shared key heads
        attention("attn_prompt", batch=2, queries=4099, keys=4099, heads=32, kv_heads=8, dim=128, dtype="bf16", causal=True),
        # the transformer workload's attention (batch 64, 512 tokens, 16 heads of 64), forward and gradients
        attention("attn_train", batch=64, queries=512, keys=512, heads=16, kv_heads=16, dim=64, dtype="bf16", packed=True, grad=True),
        # long sequences of several lengths with shared key heads, forward and gradients
        attention("attn_train_long", batch=4, queries=2048, keys=2048, heads=32, kv_heads=8, dim=128, dtype="bf16", causal=True,
                  padded=True, grad=True),
        # an encoder with a learned position bias, forward and gradients
        attention("attn_train_bias", batch=8, queries=1000, keys=1000, heads=16, kv_heads=16, dim=64, dtype="bf16", bias=True, grad=True),
        # fp32 heads of an odd size with a bias of past positions, forward and gradients
        attention("attn_train_f32", batch=2, queries=777, keys=777, heads=8, kv_heads=4, dim=80, dtype="f32", causal=True, bias=True,
                  grad=True),
        # the bias of every head for scores that are held in memory
        position_bias("bias_scores", batch=1, queries=1023, keys=2047, heads=16, dtype="bf16"),
        # its table's gradient from the scores' gradients of a batch
        position_bias("bias_scores_grad", batch=4, queries=777, keys=1000, heads=16, dtype="f32", grad=True),
        # a decoding batch: one token each of 32 sequences
        norm("norm_token", batch=32, seq=1, width=4096, stream="bf16", kind="rms", post=True, gate="channel"),
        # the transformer workload's residual stream (64 x 512 tokens of 1024) in fp32, bf16 blocks, layer norm
        norm("norm_train", batch=64, seq=512, width=1024, stream="f32", kind="layer", post=False, gate="none"),
        # gradients with norms on both sides and a gate for each sequence
        norm("norm_grad", batch=16, seq=1000, width=2048, stream="bf16", kind="rms", post=True, gate="sequence", grad=True),
    ]


def attention(name, batch, queries, keys, heads, kv_heads, dim, dtype, causal=False, padded=False, bias=False, packed=False, grad=False):
    return {"name": name, "op": "attention", "batch": batch, "queries": queries, "keys": keys, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "dtype": dtype, "causal": causal, "padded": padded, "bias": bias, "packed": packed, "grad": grad}


def position_bias(name, batch, queries, keys, heads, dtype, causal=False, grad=False):
    return {"name": name, "op": "bias", "batch": batch, "queries": queries, "keys": keys, "heads": heads, "dtype": dtype,
            "causal": causal, "grad": grad}


def norm(name, batch, seq, width, stream, kind, post, gate, grad=False):
    return {"name": name, "op": "norm", "batch": batch, "seq": seq, "width": width, "stream": stream, "kind": kind, "post": post,
            "gate": gate, "grad": grad}


def draw(rng):
    """One more case of the ranges that the listed ones stand for."""

    def spread(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["token", "attention", "attention", "bias", "norm"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op in ("token", "attention"):
        kv = rng.choice([1, 2, 4, 8])
        heads, dim = kv * rng.choice([1, 2, 4]), rng.choice([32, 64, 64, 80, 96, 128, 128])
        batch = spread(1, 32)
        if op == "token":
            keys = spread(17, 16384 * 8 // max(8, batch))
            c = attention("", batch, 1, keys, heads, kv, dim, dtype, True, rng.random() < 0.5, rng.random() < 0.25)
        else:
            grad = rng.random() < 0.6
            # scores of all heads at most, so that a case costs no more than the largest listed one
            most = (1 << 28 if dtype == "bf16" else 1 << 25) * 64 // dim
            side = max(16, min(4096, int(math.sqrt(most / (batch * heads)))))
            queries = spread(5, side)
            keys = rng.choice([queries, queries, spread(queries, side)])
            packed = keys == queries and rng.random() < 0.3
            c = attention("", batch, queries, keys, heads, kv, dim, dtype, rng.random() < 0.6, rng.random() < 0.4, rng.random() < 0.4,
                          packed, grad)
    elif op == "bias":
        queries, keys = spread(1, 2048), spread(16, 2048)
        grad = rng.random() < 0.5
        most = max(1, (1 << 26) // (queries * keys * 16))
        c = position_bias("", spread(1, min(16, most)) if grad else 1, queries, keys, rng.choice([4, 12, 16]), dtype, rng.random() < 0.5,
                          grad)
    else:
        width = rng.choice([spread(64, 8192), 768, 1024, 2048, 4096, 8 * spread(8, 1024)])
        batch = spread(1, 64)
        seq = spread(1, max(2, (1 << 25) // (batch * width)))
        c = norm("", batch, seq, width, dtype, rng.choice(["rms", "layer"]), rng.random() < 0.6,
                 rng.choice(["none", "channel", "sequence", "token"]), rng.random() < 0.6)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------

TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def prepare(case, seed):
    """Inputs on the GPU, made from the seed: activations and gradients of unit size, weights
    of a trained size, lengths between a half and all of the places."""
    g = torch.Generator(device="cuda").manual_seed(1000003 * seed + 29)

    def normal(*shape, scale=1.0, dtype="f32"):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(TYPES[dtype])

    s = {"case": dict(case)}
    if case["op"] == "attention":
        b, nq, nk, h, hk, d, dt = (case[k] for k in ("batch", "queries", "keys", "heads", "kv_heads", "dim", "dtype"))
        if case["packed"]:  # queries, keys and values side by side, as one projection writes them
            qkv = normal(b, nq, h + 2 * hk, d, dtype=dt)
            s["q"], s["k"], s["v"] = qkv[:, :, :h], qkv[:, :, h : h + hk], qkv[:, :, h + hk :]
        else:
            s["q"], s["k"], s["v"] = normal(b, nq, h, d, dtype=dt), normal(b, nk, hk, d, dtype=dt), normal(b, nk, hk, d, dtype=dt)
        s["lengths"] = s["query_lengths"] = None
        if case["padded"]:
            s["lengths"] = torch.randint((nk + 1) // 2, nk + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
            if nq > 1:  # as many queries missing as keys
                s["query_lengths"] = (s["lengths"] - (nk - nq)).clamp(min=0)
        s["table"] = normal(BUCKETS, h, dtype=dt) if case["bias"] else None
        if case["grad"]:
            s["dout"] = normal(b, nq, h, d, dtype=dt)
    elif case["op"] == "bias":
        s["table"] = normal(BUCKETS, case["heads"], dtype=case["dtype"])
        if case["grad"]:
            s["dscores"] = normal(case["batch"], case["heads"], case["queries"], case["keys"], dtype=case["dtype"])
    else:
        b, n, c = case["batch"], case["seq"], case["width"]
        s["x"], s["f"] = normal(b, n, c, dtype=case["stream"]), normal(b, n, c, dtype="bf16")
        s["weights"] = {"gamma": 1 + normal(c, scale=0.1)}
        if case["kind"] == "layer":
            s["weights"]["beta"] = normal(c, scale=0.1)
        if case["post"]:
            s["weights"]["post_gamma"] = 1 + normal(c, scale=0.1)
        shape = {"none": None, "channel": (c,), "sequence": (b, 1, c), "token": (b, n, c)}[case["gate"]]
        if shape is not None:
            s["weights"]["gate"] = 0.5 + normal(*shape, scale=0.2, dtype="bf16" if case["gate"] == "token" else "f32")
        if case["grad"]:
            s["dsum"], s["dnormed"] = normal(b, n, c, dtype=case["stream"]), normal(b, n, c, dtype="bf16")
    return s


RESIDUAL = 0.75  # the factor of the residual stream


# ------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------


def run(s):
    """One pass of the case's operator; a training case is the forward and all gradients."""
    c = s["case"]
    if own:
        return _run_own(c, s)
    if c["op"] == "attention":
        return _plain_attention(c, s)
    if c["op"] == "bias":
        return _plain_bias_grad(c, s) if c["grad"] else _plain_bias(c, s["table"].float()).to(s["table"].dtype)
    return _plain_norm_grad(c, s) if c["grad"] else _plain_norm(c, s)


def _run_own(c, s):
    import os
    import sys

    package = os.path.join(os.getcwd(), "ml-switcheroo-compiler_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    from b200 import B200Backend

    op = B200Backend.execute_op
    if c["op"] == "attention":
        kw = {"causal": c["causal"], "lengths": s["lengths"], "query_lengths": s["query_lengths"], "relative_bias": s["table"]}
        out, lse = op("Attention", s["q"], s["k"], s["v"], **kw)
        if not c["grad"]:
            return out, lse
        grads = op("AttentionGrad", s["dout"], s["q"], s["k"], s["v"], out, lse, **kw)
        return (out, *grads) if c["bias"] else (out, *grads[:3])
    if c["op"] == "bias":
        if c["grad"]:
            return op("RelativePositionBiasGrad", s["dscores"], buckets=BUCKETS, bidirectional=not c["causal"])
        return op("RelativePositionBias", s["table"], queries=c["queries"], keys=c["keys"], bidirectional=not c["causal"])
    kw = {"norm": c["kind"], "residual_scale": RESIDUAL, "eps": EPS, **s["weights"]}
    if not c["grad"]:
        return op("ResidualNorm", s["x"], s["f"], **kw)
    return [t for t in op("ResidualNormGrad", s["dsum"], s["dnormed"], s["x"], s["f"], **kw) if t is not None]


def _bucket_starts(buckets, far):
    """The smallest distance of each bucket of one side: one each up to a half, then equal steps
    of the logarithm up to `far`; in whole numbers, as steps may end on one."""
    near = buckets // 2
    wide = buckets - near
    return list(range(near)) + [next(d for d in range(near, far + 1) if d**wide >= near ** (wide - i) * far**i) for i in range(wide)]


def _buckets(c, shift):
    """Buckets [..., queries, keys] of every query and key, query i being at position i + shift."""
    rel = torch.arange(c["keys"], device=shift.device)[None] - torch.arange(c["queries"], device=shift.device)[:, None]
    rel = rel - shift[..., None, None]
    side = BUCKETS if c["causal"] else BUCKETS // 2
    starts = torch.tensor(_bucket_starts(side, FAR), device=shift.device)
    found = torch.bucketize((-rel).clamp(min=0) if c["causal"] else rel.abs(), starts, right=True) - 1
    return found if c["causal"] else found + side * (rel > 0)


def _last_at_last(c, device):
    return torch.tensor(c["keys"] - c["queries"], device=device)


def _plain_bias(c, table):
    return table[_buckets(c, _last_at_last(c, table.device))].permute(2, 0, 1)


def _plain_bias_grad(c, s):
    d = s["dscores"].float().sum(0).flatten(1)
    one_hot = torch.zeros(BUCKETS, d.shape[1], device=d.device).scatter_(0, _buckets(c, _last_at_last(c, d.device)).flatten()[None], 1.0)
    return (one_hot @ d.t()).to(s["dscores"].dtype)


def _seen(c, s):
    """[batch, 1, queries, keys]: which key a query sees."""
    dev = s["q"].device
    i, j = torch.arange(c["queries"], device=dev)[None, :, None], torch.arange(c["keys"], device=dev)[None, None]
    nk = torch.full((c["batch"],), c["keys"], device=dev) if s["lengths"] is None else s["lengths"].long()
    nq = torch.full((c["batch"],), c["queries"], device=dev) if s["query_lengths"] is None else s["query_lengths"].long()
    nk, nq = nk[:, None, None], nq[:, None, None]
    seen = (j < nk) & (i < nq)
    if c["causal"]:
        seen = seen & (j <= i + nk - nq)
    return seen[:, None], (nk - nq)[:, 0, 0]


def _head_major(x, heads):
    """[batch, heads, tokens, dim] in fp32, shared heads repeated."""
    x = x.float().transpose(1, 2)
    return x.repeat_interleave(heads // x.shape[1], 1)


def _plain_attention(c, s):
    h, scale = c["heads"], 1.0 / math.sqrt(c["dim"])
    q, k, v = (_head_major(s[n], h) for n in "qkv")
    seen, shift = _seen(c, s)
    z = (q @ k.transpose(-1, -2)).mul_(scale)
    if c["bias"]:
        bucket = _buckets(c, shift)
        z += s["table"].float()[bucket].permute(0, 3, 1, 2)
    z.masked_fill_(~seen, -math.inf)
    top = z.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = z.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    lse = (top + torch.log(total))[..., 0]
    p = p.div_(torch.where(total == 0, torch.ones_like(total), total))
    out = p @ v
    result = out.transpose(1, 2).to(s["q"].dtype)
    if not c["grad"]:
        return result, lse
    do = _head_major(s["dout"], h)
    dp = do @ v.transpose(-1, -2)
    dz = dp.sub_((do * out).sum(-1, keepdim=True)).mul_(p)
    b, nk, hk, d = s["k"].shape
    dq = (dz @ k).mul_(scale).transpose(1, 2).to(s["q"].dtype)
    dk = (dz.transpose(-1, -2) @ q).mul_(scale).view(b, hk, h // hk, nk, d).sum(2).transpose(1, 2).to(s["k"].dtype)
    dv = (p.transpose(-1, -2) @ do).view(b, hk, h // hk, nk, d).sum(2).transpose(1, 2).to(s["v"].dtype)
    if not c["bias"]:
        return result, dq, dk, dv
    bucket = bucket[:, None]
    dtable = torch.stack([torch.where(bucket == i, dz, 0.0).sum((0, 2, 3)) for i in range(BUCKETS)])
    return result, dq, dk, dv, dtable.to(s["table"].dtype)


def _unit(x, kind):
    """x centred (layer) and over its root mean square, and the reciprocal of that."""
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return x * rstd, rstd


def _unit_grad(d, unit, rstd, kind):
    d = d - unit * (d * unit).mean(-1, keepdim=True)
    return rstd * (d - d.mean(-1, keepdim=True) if kind == "layer" else d)


def _sum_of(c, s):
    """The new residual stream in fp32, with what its gradient needs."""
    w, f = s["weights"], s["f"].float()
    unit, rstd = _unit(f, c["kind"]) if c["post"] else (None, None)
    block = unit * w["post_gamma"] if c["post"] else f
    gated = block * w["gate"].float() if "gate" in w else block
    return RESIDUAL * s["x"].float() + gated, block, unit, rstd


def _plain_norm(c, s):
    total = _sum_of(c, s)[0]
    normed = _unit(total, c["kind"])[0] * s["weights"]["gamma"]
    if "beta" in s["weights"]:
        normed = normed + s["weights"]["beta"]
    return total.to(s["x"].dtype), normed.to(s["f"].dtype)


def _plain_norm_grad(c, s):
    w = s["weights"]
    total, block, post_unit, post_rstd = _sum_of(c, s)
    unit, rstd = _unit(total, c["kind"])
    dn = s["dnormed"].float()
    d = s["dsum"].float() + _unit_grad(dn * w["gamma"], unit, rstd, c["kind"])
    grads = [(RESIDUAL * d).to(s["x"].dtype), None, (dn * unit).sum((0, 1))]
    if "beta" in w:
        grads.append(dn.sum((0, 1)))
    db = d * w["gate"].float() if "gate" in w else d
    df = db
    if c["post"]:
        grads.append((db * post_unit).sum((0, 1)))
        df = _unit_grad(db * w["post_gamma"], post_unit, post_rstd, c["kind"])
    if "gate" in w:
        dg = d * block
        dg = dg.sum((0, 1)) if c["gate"] == "channel" else dg.sum(1, keepdim=True) if c["gate"] == "sequence" else dg
        grads.append(dg.to(w["gate"].dtype))
    grads[1] = df.to(s["f"].dtype)
    return grads


def work(case):
    """What one pass cannot do without."""
    if case["op"] == "attention":
        size = 2 if case["dtype"] == "bf16" else 4
        b, nq, nk, h, hk, d = (case[k] for k in ("batch", "queries", "keys", "heads", "kv_heads", "dim"))
        full = 0.75 if case["padded"] else 1.0  # the mean length
        nq, nk = (nq if nq == 1 else nq * full), nk * full
        pairs = nq * nk - (nq * (nq - 1) / 2 if case["causal"] else 0)
        ins, outs = b * d * (nq * h + 2 * nk * hk), b * d * nq * h
        if case["grad"]:  # queries, keys, values and the output's gradient in; the output and three gradients out
            return {"bytes": int(size * (2 * ins + 2 * outs)), "flops": int(14 * b * h * pairs * d)}
        return {"bytes": int(size * (ins + outs) + 4 * b * h * nq), "flops": int(4 * b * h * pairs * d)}
    if case["op"] == "bias":
        size = 2 if case["dtype"] == "bf16" else 4
        each = case["batch"] * case["heads"] * case["queries"] * case["keys"]
        return {"bytes": each * size, "flops": each}
    rows, c = case["batch"] * case["seq"], case["width"]
    stream, f = (2 if case["stream"] == "bf16" else 4), 2
    gate = 2 if case["gate"] == "token" else 0
    if case["grad"]:
        return {"bytes": rows * c * (3 * stream + 3 * f + 2 * gate), "flops": 30 * rows * c}
    return {"bytes": rows * c * (2 * stream + 2 * f + gate), "flops": 12 * rows * c}


# ------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------


def exact(case, seed):
    """What ``run`` returns, from the definitions in 64 bits."""
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, s)
    if case["op"] == "bias":
        return _exact_bias(case, s)
    return _exact_norm(case, s)


def _side_bucket(n, buckets):
    """The bucket of distance n on one side, by its definition: floor of the logarithm's share."""
    near = buckets // 2
    if n < near:
        return n
    wide, i = buckets - near, 0
    while i + 1 < wide and n**wide >= near ** (wide - i - 1) * FAR ** (i + 1):
        i += 1
    return near + i


def _bucket_of(rel, causal):
    if causal:
        return _side_bucket(max(0, -rel), BUCKETS)
    return _side_bucket(abs(rel), BUCKETS // 2) + (BUCKETS // 2 if rel > 0 else 0)


def _diagonals(low, high, causal, device):
    """Buckets of the relative positions low .. high."""
    return torch.tensor([_bucket_of(r, causal) for r in range(low, high + 1)], device=device)


def _exact_bias(case, s):
    nq, nk, shift = case["queries"], case["keys"], case["keys"] - case["queries"]
    low = -(nq - 1) - shift
    by_rel = _diagonals(low, nk - 1 - shift, case["causal"], s["table"].device)
    place = torch.arange(nk, device=by_rel.device)[None] - torch.arange(nq, device=by_rel.device)[:, None] - shift - low
    bucket = by_rel[place]
    if not case["grad"]:
        return torch.stack([s["table"].double()[:, h][bucket] for h in range(case["heads"])])
    d = s["dscores"].double().sum(0)
    return torch.stack([d[:, bucket == i].sum(-1) for i in range(BUCKETS)])


def _exact_attention(case, s):
    b, nq, nk, h, hk, d = (case[k] for k in ("batch", "queries", "keys", "heads", "kv_heads", "dim"))
    scale, per = d**-0.5, case["heads"] // case["kv_heads"]
    dev = s["q"].device
    out = torch.zeros(b, nq, h, d, dtype=torch.float64, device=dev)
    lse = torch.full((b, h, nq), -math.inf, dtype=torch.float64, device=dev)
    if case["grad"]:
        dq = torch.zeros_like(out)
        dk, dv = (torch.zeros(b, nk, hk, d, dtype=torch.float64, device=dev) for _ in range(2))
        dtable = torch.zeros(BUCKETS, h, dtype=torch.float64, device=dev)
    lengths = [nk] * b if s["lengths"] is None else s["lengths"].tolist()
    queries = [nq] * b if s["query_lengths"] is None else s["query_lengths"].tolist()
    for e in range(b):
        n, m = lengths[e], queries[e]
        if n == 0 or m == 0:
            continue
        i, j = torch.arange(m, device=dev)[:, None], torch.arange(n, device=dev)[None]
        rel = j - i - (n - m)
        hidden = rel > 0 if case["causal"] else torch.zeros_like(rel, dtype=torch.bool)
        if case["bias"]:
            low = int(rel.min())
            bucket = _diagonals(low, int(rel.max()), case["causal"], dev)[rel - low]
        for a in range(h):
            q, k, v = s["q"][e, :m, a].double(), s["k"][e, :n, a // per].double(), s["v"][e, :n, a // per].double()
            z = q @ k.t() * scale
            if case["bias"]:
                z = z + s["table"].double()[:, a][bucket]
            z = z.masked_fill(hidden, -math.inf)
            l = torch.logsumexp(z, -1)
            p = torch.exp(z - l[:, None])
            o = p @ v
            out[e, :m, a], lse[e, a, :m] = o, l
            if not case["grad"]:
                continue
            do = s["dout"][e, :m, a].double()
            dz = p * (do @ v.t() - (do * o).sum(-1, keepdim=True))
            dq[e, :m, a] = dz @ k * scale
            dk[e, :n, a // per] += dz.t() @ q * scale
            dv[e, :n, a // per] += p.t() @ do
            if case["bias"]:
                dtable[:, a].index_add_(0, bucket.flatten(), dz.flatten())
    if not case["grad"]:
        return out, lse
    return (out, dq, dk, dv, dtable) if case["bias"] else (out, dq, dk, dv)


def _exact_norm(case, s):
    layer, w = case["kind"] == "layer", {k: v.double() for k, v in s["weights"].items()}
    x, f = s["x"].double(), s["f"].double()

    def stats(t):
        mean = t.mean(-1, keepdim=True) if layer else torch.zeros_like(t[..., :1])
        return mean, ((t - mean).pow(2).mean(-1, keepdim=True) + EPS).sqrt()

    block = f
    if case["post"]:
        fm, fs = stats(f)
        block = (f - fm) / fs * w["post_gamma"]
    gate = w.get("gate", torch.ones((), dtype=torch.float64, device=x.device))
    total = x * RESIDUAL + gate * block
    tm, ts = stats(total)
    if not case["grad"]:
        return total, (total - tm) / ts * w["gamma"] + w.get("beta", 0.0)
    dn = s["dnormed"].double()
    t = dn * w["gamma"]
    d = s["dsum"].double() + t / ts - (total - tm) * (t * (total - tm)).mean(-1, keepdim=True) / ts**3
    if layer:
        d = d - t.mean(-1, keepdim=True) / ts
    grads = [d * RESIDUAL, None, (dn * (total - tm) / ts).sum((0, 1))]
    if layer:
        grads.append(dn.sum((0, 1)))
    df = d * gate
    if case["post"]:
        grads.append((df * (f - fm) / fs).sum((0, 1)))
        t = df * w["post_gamma"]
        df = t / fs - (f - fm) * (t * (f - fm)).mean(-1, keepdim=True) / fs**3
        if layer:
            df = df - t.mean(-1, keepdim=True) / fs
    if "gate" in w:
        dg = d * block
        grads.append({"channel": dg.sum((0, 1)), "sequence": dg.sum(1, keepdim=True), "token": dg}[case["gate"]])
    grads[1] = df
    return grads
