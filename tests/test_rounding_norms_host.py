"""The comparison of rounding_norms.py itself, on the CPU: attention and residual norms made with the kernels' roundings
pass, results that are wrong in a way that a kernel can be wrong do not."""

import math

import pytest
import torch

import block_reference as R
import rounding_norms as N

BF, F32 = torch.bfloat16, torch.float32


def rand(*shape, dtype=F32, seed=0, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed + sum(shape))
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype)


def rounded_attention(q, k, v, dout, table=None, lengths=None, query_lengths=None, causal=False, window=None, far=128):
    """The operators in fp32 with bf16 heads' roundings where the kernels have them."""
    b, nq, h, d = q.shape
    nk, hk = k.shape[1:3]
    inner = (lambda t: t.to(BF).float()) if q.dtype == BF else (lambda t: t)
    r = {"out": torch.zeros(q.shape), "dq": torch.zeros(q.shape), "dk": torch.zeros(k.shape), "dv": torch.zeros(k.shape)}
    if table is not None:
        r["dtable"] = torch.zeros(table.shape)
    for e in range(b):
        n, w = nk if lengths is None else int(lengths[e]), nq if query_lengths is None else int(query_lengths[e])
        if not n or not w:
            continue
        seen = R.seen_keys(w, n, causal, window)
        for a in range(h):
            g = a // (h // hk)
            Q, K, V, D = q[e, :w, a].float(), k[e, :n, g].float(), v[e, :n, g].float(), dout[e, :w, a].float()
            z = Q @ K.t() * d**-0.5
            if table is not None:
                where = R.bias_buckets(w, n, n - w, table.shape[0], far, not causal)
                z = z + table[:, a].float()[where]
            z = z.masked_fill(~seen, -math.inf)
            top = z.amax(-1, keepdim=True).nan_to_num(neginf=0.0)
            x = torch.exp(z - top)
            total = x.sum(-1, keepdim=True)
            o = (inner(x) @ V / torch.where(total == 0, 1.0, total)).to(q.dtype)
            p = x / torch.where(total == 0, 1.0, total)
            r["out"][e, :w, a] = o.float()
            dz = p * (D @ V.t() - (D * o.float()).sum(-1, keepdim=True))
            r["dq"][e, :w, a] = inner(dz) @ K * d**-0.5
            r["dk"][e, :n, g] += inner(dz).t() @ Q * d**-0.5
            r["dv"][e, :n, g] += inner(p).t() @ D
            if table is not None:
                r["dtable"][:, a].index_add_(0, where.flatten(), dz.flatten())
    return {n: t.to(table.dtype if n == "dtable" else q.dtype) for n, t in r.items()}


CASES = [  # heads' type, dim, causal, window, table's type, padded
    (BF, 64, True, None, None, False), (BF, 64, False, None, F32, True), (BF, 128, False, 33, BF, False), (BF, 40, True, 50, F32, True),
    (BF, 200, True, None, BF, False), (F32, 64, True, None, F32, True), (F32, 80, False, 20, F32, False),
]


@pytest.mark.parametrize("dtype,dim,causal,window,table_type,padded", CASES)
def test_attention_with_its_roundings_passes_and_wrong_ones_do_not(dtype, dim, causal, window, table_type, padded):
    b, nq, nk, h, hk = 3, 70, 90, 4, 2
    q, k, v, do = (rand(b, n, x, dim, dtype=dtype, seed=i) for i, (n, x) in enumerate(((nq, h), (nk, hk), (nk, hk), (nq, h))))
    kw = {"causal": causal, "window": window, "far": 30}
    if padded:
        kw.update(lengths=torch.tensor([90, 31, 64]), query_lengths=torch.tensor([70, 20, 44]))
    if table_type is not None:
        kw["table"] = rand(16, h, dtype=table_type, seed=9)
    ref, var = N.attention_noise(q, k, v, do, **kw)
    got = rounded_attention(q, k, v, do, **kw)
    for name, t in got.items():
        assert N.attention_off(name, t, ref, var) is None, name
        want = ref[name]
        third = max(1, want.shape[1] // 3)
        lost, swapped = want.clone(), want.clone()
        if name == "dtable":
            lost[5] = 0
            swapped[[2, 3]] = want[[3, 2]]
        else:
            lost[0, third] = 0  # one token's row of every head
            swapped[:, :, [0, 1]] = want[:, :, [1, 0]]
        near = 0.02 if dtype == BF else 1e-4
        for how, wrong in {"zeros": 0 * want, "negated": -want, "too large": want * 1.1, "twice": 2 * want, "a little": want * (1 + 2 * near),
                           "lost": lost, "swapped": swapped}.items():
            if how == "swapped" and name in ("dk", "dv") and hk < 2:
                continue
            assert N.attention_off(name, wrong, ref, var) is not None, (name, how)


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("ft", [F32, BF])
@pytest.mark.parametrize("shape,gate", [((5, 64), (64,)), ((5, 1024), (1024,)), ((3, 50, 75), (3, 1, 75)), ((500, 3, 64), (500, 1, 64)), ((4, 9, 7), (4, 9, 7))])
def test_residual_norms_with_roundings_pass_and_wrong_ones_do_not(shape, gate, ft, norm):
    c = shape[-1]
    x, f = rand(*shape, shift=0.3), rand(*shape, dtype=ft, seed=1)
    w = {"gamma": rand(c, seed=2, scale=0.2, shift=1), "post_gamma": rand(c, seed=3, scale=0.2, shift=1), "gate": rand(*gate, seed=6, shift=0.5)}
    ds, dh = rand(*shape, seed=7), rand(*shape, dtype=ft, seed=8)
    ref, _ = R.residual_norm(x, f, **w, scale=0.75, norm=norm, dsum=ds, dnormed=dh, eps=1e-5)

    def unit(t):
        t = t - t.mean(-1, keepdim=True) if norm == "layer" else t
        return t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + 1e-5)

    leaves = {n: t.float().requires_grad_() for n, t in {"x": x, "f": f, **w}.items()}
    total = 0.75 * leaves["x"] + leaves["gate"] * unit(leaves["f"]) * leaves["post_gamma"]
    normed = unit(total) * leaves["gamma"]
    ((total * ds).sum() + (normed * dh.float()).sum()).backward()
    got = {"sum": total, "normed": normed.to(ft), "df": leaves["f"].grad.to(ft), **{"d" + n: t.grad for n, t in leaves.items() if n != "f"}}
    for name, t in got.items():
        rows = name in ("sum", "normed", "dx", "df")
        assert N.residual_off(name, t.detach(), ref[name], rows) is None
        want = ref[name].to(t.dtype)
        lost = want.clone().reshape(-1)
        lost[lost.numel() // 2] = 0
        for how, wrong in {"zeros": 0 * want, "negated": -want, "too large": want * 1.1, "a little": want * 1.02, "lost": lost}.items():
            assert N.residual_off(name, wrong.reshape(want.shape), ref[name], rows) is not None, (name, how)
