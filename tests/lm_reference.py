"""Plain 64-bit forms of the language-model operators, on the CPU with torch.float64."""

import math

import torch

HALF_STEP = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8}  # a rounding's relative size at most


def angles(rotary_dim, base=10000.0, scaling=None):
    """(angle per position of each pair, factor): the definitions, one pair at a time."""
    sc, out = scaling or {"kind": "none"}, []
    for j in range(rotary_dim // 2):
        w = base ** (-2.0 * j / rotary_dim)
        if sc["kind"] == "linear":
            w = w / sc["factor"]
        elif sc["kind"] == "ntk" and rotary_dim > 2:
            w = (base * sc["factor"] ** (rotary_dim / (rotary_dim - 2.0))) ** (-2.0 * j / rotary_dim)
        elif sc["kind"] == "yarn":
            edge = [rotary_dim * math.log(sc["original_length"] / (2 * math.pi * b)) / (2 * math.log(base))
                    for b in (sc.get("beta_fast", 32.0), sc.get("beta_slow", 1.0))]
            lo, hi = max(0, math.floor(edge[0])), min(rotary_dim - 1, math.ceil(edge[1]))
            t = min(1.0, max(0.0, (j - lo) / max(hi - lo, 0.001)))
            w = w * (1 - t) + w / sc["factor"] * t
        elif sc["kind"] == "wavelength":
            length = 2 * math.pi / w
            if length > sc["original_length"] / sc["low_factor"]:
                w = w / sc["factor"]
            elif length >= sc["original_length"] / sc["high_factor"]:
                t = (sc["original_length"] / length - sc["low_factor"]) / (sc["high_factor"] - sc["low_factor"])
                w = (1 - t) * w / sc["factor"] + t * w
        out.append(w)
    factor = sc.get("attention_factor", 0.1 * math.log(sc["factor"]) + 1.0) if sc["kind"] == "yarn" else 1.0
    return out, factor


def rotate(x, positions, rotary_dim, base=10000.0, scaling=None, interleaved=False, sign=1):
    """x float64 [batch, seq, heads, dim], positions int64 [batch, seq] -> (rotated, the
    magnitude |a| + |b| of each element's pair times the factor)."""
    w, factor = angles(rotary_dim, base, scaling)
    t = sign * positions.double()[:, :, None, None] * torch.tensor(w, dtype=torch.float64)
    c, s = torch.cos(t) * factor, torch.sin(t) * factor
    y, mag = x.clone(), x.abs()
    if interleaved:
        ia, ib = slice(0, rotary_dim, 2), slice(1, rotary_dim, 2)
    else:
        ia, ib = slice(0, rotary_dim // 2), slice(rotary_dim // 2, rotary_dim)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    mag[..., ia] = mag[..., ib] = (a.abs() + b.abs()) * factor
    return y, mag


def rms_unit(x, eps):
    rstd = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    return x * rstd, rstd


def linear_xent(x, w, labels, ignore=-100, dloss=None):
    """Losses, lse and (with dloss) dx, dw of the head x [N, D] . w [D, V] in float64, and the
    logits' gradient itself."""
    z = x @ w
    lse = torch.logsumexp(z, -1)
    kept = labels != ignore
    at = (torch.arange(len(x), device=x.device), labels.clamp(min=0))
    loss = torch.where(kept, lse - z[at], torch.zeros_like(lse))
    if dloss is None:
        return loss, lse
    d = torch.softmax(z, -1)
    d[at] -= 1
    d = d * torch.where(kept, dloss, torch.zeros_like(dloss))[:, None]
    return loss, lse, d @ w.t(), x.t() @ d, d


def newton_schulz(g, steps=5, coefficients=(3.4445, -4.7750, 2.0315), eps=1e-7):
    x = g / (torch.linalg.vector_norm(g, dim=(-2, -1), keepdim=True) + eps)
    for i in range(steps):
        a, b, c = coefficients[i] if isinstance(coefficients[0], (list, tuple)) else coefficients
        s = x @ x.mT if x.shape[-2] <= x.shape[-1] else x.mT @ x
        p = b * s + c * (s @ s)
        x = a * x + (p @ x if x.shape[-2] <= x.shape[-1] else x @ p)
    return x
