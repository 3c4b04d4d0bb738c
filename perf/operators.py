"""Cases that measure the language-model operators of the b200 backend.

Four operators of a decoder's training step and of its single-token serving form:

* ``RotaryEmbedding`` (and its gradient): rotary positions of one tensor;
* ``QKNormRotary`` (and its gradient): RMS norm of queries and keys per head and the
  rotation of both in the same pass;
* ``LinearCrossEntropy`` (and its gradient): the head's product and the softmax cross
  entropy over a large vocabulary;
* ``NewtonSchulz`` / ``ApplyMuon``: the orthogonalised update of a weight matrix.

``run`` computes them in their plain form (elementary torch operations in 32 bits, angles
in 64), or through the backend's public entry point where ``own`` is true. ``exact`` gives
the same values from the definitions in 64 bits.
"""

import math

import torch

own = False

COEFFICIENTS = (3.4445, -4.7750, 2.0315)  # the quintic that Newton-Schulz steps iterate
NS_EPS = 1e-7


def listed():
    """The measured cases."""
    return [
        # one new token of one sequence, far into a stretched context
        rotary("rope_token", batch=1, seq=1, heads=32, dim=128, part=128, dtype="bf16", scaling="yarn", start=40000),
        # a long prompt of two sequences with one odd length
        rotary("rope_prompt", batch=2, seq=8191, heads=32, dim=128, part=128, dtype="bf16", scaling="wavelength"),
        # backward over a part of each head, neighbouring pairs, head-major fp32 activations
        rotary("rope_grad_part", batch=8, seq=1000, heads=16, dim=80, part=32, dtype="f32", interleaved=True,
               head_major=True, grad=True),
        # a decoding batch: one token for each of 32 sequences at its own position
        qk_norm("qk_token", batch=32, seq=1, heads=32, kv_heads=8, dim=128, part=128, dtype="bf16", start=3000),
        # the transformer workload's activations (batch 64, 512 tokens, 16 heads of 64), sliced from one projection
        qk_norm("qk_train", batch=64, seq=512, heads=16, kv_heads=16, dim=64, part=64, dtype="bf16", packed=True),
        # backward of 32768 tokens with shared key heads
        qk_norm("qk_grad", batch=16, seq=2048, heads=32, kv_heads=8, dim=128, part=128, dtype="bf16", grad=True),
        # evaluation of a short text: losses alone
        loss("loss_eval", tokens=777, dim=1024, vocab=32000, dtype="bf16"),
        # the transformer workload's head and loss: 64 x 511 next-token targets, both gradients
        loss("loss_train", tokens=32704, dim=1024, vocab=32000, dtype="bf16", grad=True),
        # fp32 activations, a vocabulary that is no multiple of anything, tied embedding layout
        loss("loss_train_f32", tokens=2048, dim=1000, vocab=50001, dtype="f32", grad=True, tied=True),
        # one square projection's update
        muon("ns_one", batch=1, rows=1024, cols=1024, dtype="f32"),
        # the feed-forward matrices of eight layers in bf16, taller than wide
        muon("ns_tall_bf16", batch=8, rows=4096, cols=1024, dtype="bf16"),
        # the whole step for the sixteen attention projections of the transformer workload
        muon("muon_step", batch=16, rows=1024, cols=1024, dtype="f32", step=True),
    ]


def rotary(name, batch, seq, heads, dim, part, dtype, scaling="none", interleaved=False, head_major=False, grad=False, start=0):
    return {"name": name, "op": "rope", "batch": batch, "seq": seq, "heads": heads, "dim": dim, "part": part, "dtype": dtype,
            "scaling": scaling, "interleaved": interleaved, "head_major": head_major, "grad": grad, "start": start}


def qk_norm(name, batch, seq, heads, kv_heads, dim, part, dtype, scaling="none", interleaved=False, packed=False, grad=False,
            start=0):
    return {"name": name, "op": "qk", "batch": batch, "seq": seq, "heads": heads, "kv_heads": kv_heads, "dim": dim, "part": part,
            "dtype": dtype, "scaling": scaling, "interleaved": interleaved, "packed": packed, "grad": grad, "start": start}


def loss(name, tokens, dim, vocab, dtype, grad=False, tied=False):
    return {"name": name, "op": "loss", "tokens": tokens, "dim": dim, "vocab": vocab, "dtype": dtype, "grad": grad, "tied": tied}


def muon(name, batch, rows, cols, dtype, step=False):
    return {"name": name, "op": "muon", "batch": batch, "rows": rows, "cols": cols, "dtype": dtype, "step": step}


def draw(rng):
    """One more case of the ranges that the listed ones stand for."""

    def spread(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["rope", "qk", "loss", "muon"])
    dtype = rng.choice(["bf16", "f32"])
    if op in ("rope", "qk"):
        dim = rng.choice([32, 64, 80, 96, 128, 192, 256])
        part = rng.choice([dim, dim, dim // 2, dim // 4 * 2 - 2])
        tokens = spread(1, 16384)
        batch = min(tokens, spread(1, 64))
        seq = max(1, tokens // batch)
        scaling = rng.choice(["none", "linear", "ntk", "yarn", "wavelength"])
        start = rng.choice([0, rng.randrange(100000)])
        interleaved = rng.random() < 0.5
        grad = rng.random() < 0.5
        if op == "rope":
            c = rotary("", batch, seq, rng.choice([1, 3, 8, 16, 32]), dim, part, dtype, scaling, interleaved,
                       rng.random() < 0.5, grad, start)
        else:
            kv = rng.choice([1, 2, 4, 8])
            c = qk_norm("", batch, seq, kv * rng.choice([1, 2, 4]), kv, dim, part, dtype, scaling, interleaved,
                        rng.random() < 0.5, grad, start)
    elif op == "loss":
        dim, vocab = spread(64, 2048), spread(1000, 100000)
        most = 32704 * 1024 * 32000 / 4 / (dim * vocab)
        c = loss("", spread(1, max(2, min(16384, int(most)))), dim, vocab, dtype, rng.random() < 0.6, rng.random() < 0.5)
    else:
        rows, cols = spread(48, 2048), spread(48, 4096)
        if rng.random() < 0.5:
            rows, cols = cols, rows
        batch = spread(1, max(1, min(16, (1 << 24) // (rows * cols))))
        step = rng.random() < 0.4
        c = muon("", batch, rows, cols, "f32" if step else dtype, step)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------

TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
BASE = 10000.0
SCALINGS = {  # contexts stretched by a factor over the length that the angles were made for
    "none": None,
    "linear": {"kind": "linear", "factor": 4.0},
    "ntk": {"kind": "ntk", "factor": 4.0},
    "yarn": {"kind": "yarn", "factor": 16.0, "original_length": 4096, "beta_fast": 32.0, "beta_slow": 1.0},
    "wavelength": {"kind": "wavelength", "factor": 8.0, "original_length": 8192, "low_factor": 1.0, "high_factor": 4.0},
}


def prepare(case, seed):
    """Inputs on the GPU, made from the seed: activations and gradients of unit size, weights
    of a trained size, labels with one in sixteen ignored."""
    g = torch.Generator(device="cuda").manual_seed(1000003 * seed + 17)

    def normal(*shape, scale=1.0, dtype=None):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype or TYPES[case["dtype"]])

    s = {"case": dict(case)}
    if case["op"] in ("rope", "qk"):
        b, n, d = case["batch"], case["seq"], case["dim"]
        first = torch.randint(0, 16, (b, 1), generator=g, device="cuda") + case["start"]
        s["positions"] = first + torch.arange(n, device="cuda")[None]
        s["rotation"] = {"base": BASE, "rotary_dim": case["part"], "interleaved": case["interleaved"],
                         "scaling": SCALINGS[case["scaling"]]}
        if case["op"] == "rope":
            h = case["heads"]
            s["x"] = normal(b, h, n, d).transpose(1, 2) if case["head_major"] else normal(b, n, h, d)
        else:
            h, hk = case["heads"], case["kv_heads"]
            if case["packed"]:  # queries, keys and values side by side, as one projection writes them
                qkv = normal(b, n, h + 2 * hk, d)
                s["q"], s["k"] = qkv[:, :, :h], qkv[:, :, h : h + hk]
            else:
                s["q"], s["k"] = normal(b, n, h, d), normal(b, n, hk, d)
            s["gamma_q"] = 1 + normal(d, scale=0.1, dtype=torch.float32)
            s["gamma_k"] = 1 + normal(d, scale=0.1, dtype=torch.float32)
            if case["grad"]:
                s["dq"], s["dk"] = normal(b, n, h, d), normal(b, n, hk, d)
    elif case["op"] == "loss":
        n, d, v = case["tokens"], case["dim"], case["vocab"]
        s["x"] = normal(n, d)
        w = normal(v, d, scale=1.5 / math.sqrt(d)) if case["tied"] else normal(d, v, scale=1.5 / math.sqrt(d))
        s["w"] = w.t() if case["tied"] else w
        labels = torch.randint(0, v, (n,), generator=g, device="cuda")
        off = torch.rand(n, generator=g, device="cuda") < 1 / 16
        s["labels"] = torch.where(off, torch.full_like(labels, -100), labels)
        if case["grad"]:  # a weighted mean over the tokens
            s["dloss"] = (0.5 + torch.rand(n, generator=g, device="cuda")) / n
    else:
        z, m, n = case["batch"], case["rows"], case["cols"]
        # a gradient: a part of low rank and noise
        r = max(1, min(m, n) // 4)
        grad = normal(z, m, r, dtype=torch.float32) @ normal(z, r, n, dtype=torch.float32) / math.sqrt(r) + normal(z, m, n, dtype=torch.float32)
        grad = (grad * 1e-3).to(TYPES[case["dtype"]])
        s["grad"] = grad[0] if z == 1 else grad
        if case["step"]:
            s["param"] = normal(*s["grad"].shape, scale=0.02, dtype=torch.float32)
            s["momentum"] = normal(*s["grad"].shape, scale=1e-3, dtype=torch.float32)
    return s


# ------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------


def run(s):
    """One pass of the case's operator."""
    c = s["case"]
    if own:
        return _run_own(c, s)
    if c["op"] == "rope":
        return _rotate(s["x"].float(), s["positions"], s["rotation"], -1.0 if c["grad"] else 1.0).to(s["x"].dtype)
    if c["op"] == "qk":
        return _plain_qk_grad(s) if c["grad"] else _plain_qk(s)
    if c["op"] == "loss":
        return _plain_loss(c, s)
    return _plain_step(s) if c["step"] else _plain_newton_schulz(s["grad"].float()).to(s["grad"].dtype)


def _run_own(c, s):
    import os
    import sys

    package = os.path.join(os.getcwd(), "ml-switcheroo-compiler_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    from b200 import B200Backend

    op = B200Backend.execute_op
    if c["op"] == "rope":
        return op("RotaryEmbeddingGrad" if c["grad"] else "RotaryEmbedding", s["x"], s["positions"], **s["rotation"])
    if c["op"] == "qk":
        if c["grad"]:
            return op("QKNormRotaryGrad", s["dq"], s["dk"], s["q"], s["k"], s["gamma_q"], s["gamma_k"], s["positions"], **s["rotation"])
        return op("QKNormRotary", s["q"], s["k"], s["gamma_q"], s["gamma_k"], s["positions"], **s["rotation"])
    if c["op"] == "loss":
        losses, lse = op("LinearCrossEntropy", s["x"], s["w"], s["labels"])
        if not c["grad"]:
            return losses, lse
        return (losses, *op("LinearCrossEntropyGrad", s["dloss"], s["x"], s["w"], s["labels"], lse))
    if c["step"]:
        return op("ApplyMuon", s["param"], s["momentum"], s["grad"], lr=0.02, momentum=0.95, weight_decay=0.01)
    return op("NewtonSchulz", s["grad"])


def _frequencies(part, rotation, device):
    """Angle per position of each pair (64 bits) and the factor on cosine and sine."""
    i = torch.arange(0, part, 2, dtype=torch.float64, device=device)
    sc = rotation["scaling"]
    base = rotation["base"]
    if sc is not None and sc["kind"] == "ntk" and part > 2:
        base = base * sc["factor"] ** (part / (part - 2))
    inv = base ** (-i / part)
    if sc is None or sc["kind"] == "ntk":
        return inv, 1.0
    if sc["kind"] == "linear":
        return inv / sc["factor"], 1.0
    length = sc["original_length"]
    if sc["kind"] == "yarn":

        def turn(beta):
            return part * math.log(length / (beta * 2 * math.pi)) / (2 * math.log(base))

        low, high = max(math.floor(turn(sc["beta_fast"])), 0), min(math.ceil(turn(sc["beta_slow"])), part - 1)
        ramp = ((i / 2 - low) / max(high - low, 0.001)).clamp(0, 1)
        return inv / sc["factor"] * ramp + inv * (1 - ramp), 0.1 * math.log(sc["factor"]) + 1.0
    turns = length * inv / (2 * math.pi)
    smooth = ((turns - sc["low_factor"]) / (sc["high_factor"] - sc["low_factor"])).clamp(0, 1)
    return inv / sc["factor"] * (1 - smooth) + inv * smooth, 1.0


def _rotate(x, positions, rotation, sign):
    """x [batch, seq, heads, dim] in fp32: the first rotary_dim elements of each head rotated."""
    part = rotation["rotary_dim"]
    inv, factor = _frequencies(part, rotation, x.device)
    angle = positions.double()[..., None] * inv
    cos = (torch.cos(angle) * factor).float()[:, :, None]
    sin = (torch.sin(angle) * (sign * factor)).float()[:, :, None]
    r, rest = x[..., :part], x[..., part:]
    if rotation["interleaved"]:
        a, b = r[..., 0::2], r[..., 1::2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = r[..., : part // 2], r[..., part // 2 :]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([y, rest], -1)


def _unit(x):
    """x over its root mean square, and the reciprocal of that."""
    rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    return x * rstd, rstd


def _plain_qk(s):
    def one(x, gamma):
        return _rotate(_unit(x.float())[0] * gamma, s["positions"], s["rotation"], 1.0).to(x.dtype)

    return one(s["q"], s["gamma_q"]), one(s["k"], s["gamma_k"])


def _plain_qk_grad(s):
    def one(dy, x, gamma):
        g = _rotate(dy.float(), s["positions"], s["rotation"], -1.0)
        u, rstd = _unit(x.float())
        h = g * gamma
        dx = rstd * (h - u * (h * u).mean(-1, keepdim=True))
        return dx.to(x.dtype), (g * u).sum((0, 1, 2))

    dq, dgq = one(s["dq"], s["q"], s["gamma_q"])
    dk, dgk = one(s["dk"], s["k"], s["gamma_k"])
    return dq, dk, dgq, dgk


def _plain_loss(c, s):
    x, w = s["x"].float(), s["w"].float()
    valid = s["labels"] >= 0
    label = s["labels"].clamp(min=0)[:, None]
    z = x @ w
    top = z.max(-1, keepdim=True).values
    picked = z.gather(1, label)
    z = torch.exp(z.sub_(top))
    total = z.sum(-1, keepdim=True)
    lse = top + torch.log(total)
    losses = torch.where(valid, (lse - picked)[:, 0], torch.zeros_like(lse[:, 0]))
    if not c["grad"]:
        return losses, lse[:, 0]
    scale = torch.where(valid, s["dloss"], torch.zeros_like(s["dloss"]))[:, None]
    z = z.mul_(scale / total)
    z = z.scatter_add_(1, label, -scale)
    return losses, (z @ w.t()).to(s["x"].dtype), (x.t() @ z).to(s["w"].dtype)


def _plain_newton_schulz(g):
    a, b, c = COEFFICIENTS
    turned = g.shape[-2] > g.shape[-1]
    x = g.transpose(-1, -2) if turned else g
    x = x / (torch.sqrt((x * x).sum((-2, -1), keepdim=True)) + NS_EPS)
    for _ in range(5):
        gram = x @ x.transpose(-1, -2)
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.transpose(-1, -2).contiguous() if turned else x


def _plain_step(s):
    m = 0.95 * s["momentum"] + s["grad"]
    o = _plain_newton_schulz(s["grad"] + 0.95 * m)
    rows, cols = o.shape[-2:]
    return s["param"] * (1 - 0.02 * 0.01) - 0.02 * math.sqrt(max(1.0, rows / cols)) * o, m


def work(case):
    """What one pass cannot do without."""
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] in ("rope", "qk"):
        rows = case["batch"] * case["seq"]
        each = rows * (case["heads"] + case.get("kv_heads", 0)) * case["dim"]
        arrays = 3 if case["op"] == "qk" and case["grad"] else 2
        return {"bytes": arrays * each * size + 8 * rows, "flops": 3 * each + (6 * each if case["op"] == "qk" else 0)}
    if case["op"] == "loss":
        n, d, v = case["tokens"], case["dim"], case["vocab"]
        both = 2 if case["grad"] else 1
        return {"bytes": both * (n * d + d * v) * size + 16 * n, "flops": (6 if case["grad"] else 2) * n * d * v}
    z, m, n = case["batch"], min(case["rows"], case["cols"]), max(case["rows"], case["cols"])
    # the Gram matrix and its square are symmetric: half of each is enough
    return {"bytes": z * m * n * size * (5 if case["step"] else 2), "flops": 5 * z * (3 * m * m * n + m**3)}


# ------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------


def exact(case, seed):
    """What ``run`` returns, from the definitions in 64 bits."""
    s = prepare(case, seed)
    if case["op"] == "rope":
        return _exact_turn(s["x"].double(), s, -1 if case["grad"] else 1)
    if case["op"] == "qk":
        return _exact_qk(case, s)
    if case["op"] == "loss":
        return _exact_loss(case, s)
    if case["step"]:
        m = s["momentum"].double() * 0.95 + s["grad"].double()
        o = _exact_newton_schulz(m * 0.95 + s["grad"].double())
        tall = max(1.0, case["rows"] / case["cols"])
        return s["param"].double() * (1 - 0.02 * 0.01) - o * (0.02 * tall**0.5), m
    return _exact_newton_schulz(s["grad"].double())


def _exact_angles(case):
    """One angle per pair, from the definition of each scaling, one pair at a time."""
    p, sc, angles = case["part"], SCALINGS[case["scaling"]] or {"kind": "none"}, []
    for j in range(p // 2):
        w = BASE ** (-2.0 * j / p)
        if sc["kind"] == "linear":
            w /= sc["factor"]
        elif sc["kind"] == "ntk" and p > 2:
            w = (BASE * sc["factor"] ** (p / (p - 2.0))) ** (-2.0 * j / p)
        elif sc["kind"] == "yarn":
            edge = [p * math.log(sc["original_length"] / (2 * math.pi * sc[b])) / (2 * math.log(BASE)) for b in ("beta_fast", "beta_slow")]
            lo, hi = max(0, math.floor(edge[0])), min(p - 1, math.ceil(edge[1]))
            t = min(1.0, max(0.0, (j - lo) / max(hi - lo, 0.001)))
            w = w * (1 - t) + w / sc["factor"] * t
        elif sc["kind"] == "wavelength":
            length = 2 * math.pi / w
            if length > sc["original_length"] / sc["low_factor"]:
                w /= sc["factor"]
            elif length >= sc["original_length"] / sc["high_factor"]:
                t = (sc["original_length"] / length - sc["low_factor"]) / (sc["high_factor"] - sc["low_factor"])
                w = (1 - t) * w / sc["factor"] + t * w
        angles.append(w)
    return angles, (0.1 * math.log(sc["factor"]) + 1.0) if sc["kind"] == "yarn" else 1.0


def _exact_turn(x, s, sign):
    """Each pair as a complex number times the unit number of its angle."""
    c = s["case"]
    p = c["part"]
    angles, factor = _exact_angles(c)
    a = s["positions"].double()[:, :, None, None] * torch.tensor(angles, dtype=torch.float64, device=x.device) * sign
    unit = torch.polar(torch.full_like(a, factor), a)
    y = x.clone()
    if c["interleaved"]:
        y[..., :p] = torch.view_as_real(torch.view_as_complex(x[..., :p].contiguous().unflatten(-1, (-1, 2))) * unit).flatten(-2)
    else:
        t = torch.complex(x[..., : p // 2].contiguous(), x[..., p // 2 : p].contiguous()) * unit
        y[..., : p // 2], y[..., p // 2 : p] = t.real, t.imag
    return y


def _exact_qk(case, s):
    out, sums = [], []
    for name in "qk":
        x, gamma = s[name].double(), s["gamma_" + name].double()
        scale = (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt()
        if not case["grad"]:
            out.append(_exact_turn(x / scale * gamma, s, 1))
            continue
        g = _exact_turn(s["d" + name].double(), s, -1)
        sums.append((g * x / scale).sum((0, 1, 2)))
        g = g * gamma
        out.append(g / scale - x * (g * x).mean(-1, keepdim=True) / scale**3)
    return (*out, *sums)


def _exact_loss(case, s):
    n, v = case["tokens"], case["vocab"]
    w = s["w"].double()
    rows = max(1, min(n, (1 << 29) // v))
    losses, lses, dxs, dw = [], [], [], torch.zeros_like(w)
    for i in range(0, n, rows):
        x = s["x"][i : i + rows].double()
        label = s["labels"][i : i + rows]
        kept = (label != -100).double()
        z = x @ w
        lse = torch.logsumexp(z, -1)
        at = (torch.arange(len(x), device=x.device), label.clamp(min=0))
        losses.append((lse - z[at]) * kept)
        lses.append(lse)
        if case["grad"]:
            d = torch.softmax(z, -1)
            d[at] -= 1
            d *= (s["dloss"][i : i + rows].double() * kept)[:, None]
            dxs.append(d @ w.t())
            dw += x.t() @ d
    if not case["grad"]:
        return torch.cat(losses), torch.cat(lses)
    return torch.cat(losses), torch.cat(dxs), dw


def _exact_newton_schulz(g):
    a, b, c = COEFFICIENTS
    x = g / (torch.linalg.vector_norm(g, dim=(-2, -1), keepdim=True) + NS_EPS)
    for _ in range(5):
        if x.shape[-2] <= x.shape[-1]:
            once = (x @ x.mT) @ x
            x = a * x + b * once + c * ((x @ x.mT) @ once)
        else:
            once = x @ (x.mT @ x)
            x = a * x + b * once + c * (once @ (x.mT @ x))
    return x
