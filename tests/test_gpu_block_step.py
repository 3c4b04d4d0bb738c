"""The block operators as they are used together: a decoder block's training step (residual norms on both sides of
attention with a learned position bias), the same through the whole-graph hooks, tokens one at a time from a padded
cache against whole prompts, several threads at once, caches whose offsets pass 32 bits."""

import math

import pytest
import torch

import block_reference as R

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
B, S, C, H, HK, D = 2, 40, 64, 4, 2, 16


@pytest.fixture(autouse=True)
def _policy(cuda):
    from b200 import ops

    ops.Config.matmul_dtype = "f32"
    yield
    ops.Config.matmul_dtype = "f32"


def op(name, *args, **kw):
    from b200.backend import B200Backend

    return B200Backend.execute_op(name, *args, **kw)


def rms(t, eps):
    return t / (t.pow(2).mean(-1, keepdim=True) + eps).sqrt()


def test_decoder_block_training_step_matches_64_bit_gradients():
    """stream -> [sum, norm] -> projections -> attention -> projection -> [sum, norm], fp32. A gradient is a sum of products of
    at most 4 such operators in turn, each within 1e-5 of its terms (their own tests), and of fp32 products over up to 80
    rows: 1e-4 of the gradient's norm."""
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    p = {"x": r(B, S, C), "f": r(B, S, C), "g0": 1 + 0.1 * r(C), "p0": 1 + 0.1 * r(C), "gate": 0.5 + 0.1 * r(B, 1, C),
         "wqkv": r(C, (H + 2 * HK) * D) / 8, "wo": r(H * D, C) / 8, "table": r(8, H), "g1": 1 + 0.1 * r(C)}
    end = r(B, S, C)
    lengths = torch.tensor([S, 23])
    alive = (torch.arange(S)[None] < lengths[:, None])[..., None]
    # by autograd in 64 bits
    w = {k: v.double().requires_grad_() for k, v in p.items()}
    s0 = 0.5 * w["x"] + w["gate"] * rms(w["f"], 1e-6) * w["p0"]
    h0 = rms(s0, 1e-6) * w["g0"]
    q, k, v = (h0 @ w["wqkv"]).view(B, S, H + 2 * HK, D).split([H, HK, HK], 2)
    outs = []
    for e in range(B):
        n = int(lengths[e])
        z = torch.einsum("ihd,jhd->hij", q[e, :n], k[e, :n].repeat_interleave(H // HK, 1)) / math.sqrt(D)
        z = z + w["table"][R.bias_buckets(n, n, 0, 8, 20, False)].permute(2, 0, 1)
        z = z.masked_fill(~R.seen_keys(n, n, True, None), -math.inf)
        o = torch.einsum("hij,jhd->ihd", z.softmax(-1), v[e, :n].repeat_interleave(H // HK, 1))
        outs.append(torch.cat([o, torch.zeros(S - n, H, D, dtype=torch.float64)]))
    a = torch.stack(outs).flatten(2) @ w["wo"]
    s1 = s0 + a
    loss = (rms(s1, 1e-6) * w["g1"] * end.double() * alive).sum()
    loss.backward()
    # by the backend's operators
    c = {k: v.cuda() for k, v in p.items()}
    n0 = {"gamma": c["g0"], "post_gamma": c["p0"], "gate": c["gate"], "residual_scale": 0.5}
    t0, y0 = op("ResidualNorm", c["x"], c["f"], **n0)
    qkv = op("Matmul", y0, c["wqkv"]).view(B, S, H + 2 * HK, D)
    heads = (qkv[:, :, :H], qkv[:, :, H : H + HK], qkv[:, :, H + HK :])
    kw = {"causal": True, "lengths": lengths.cuda(), "query_lengths": lengths.cuda(), "relative_bias": c["table"], "max_distance": 20}
    out, lse = op("Attention", *heads, **kw)
    flat = out.flatten(2)
    f1 = op("Matmul", flat, c["wo"])
    t1, y1 = op("ResidualNorm", t0, f1, gamma=c["g1"])
    got = float((y1.cpu().double() * end.double() * alive).sum())
    assert got == pytest.approx(float(loss), rel=1e-4)
    dy1 = (end * alive).cuda()
    dt0, df1, dg1, *_ = op("ResidualNormGrad", torch.zeros_like(t1), dy1, t0, f1, gamma=c["g1"])
    dflat = op("Matmul", df1, c["wo"].t())
    dwo = op("Matmul", flat.reshape(-1, H * D).t(), df1.reshape(-1, C))
    dq, dk, dv, dtable = op("AttentionGrad", dflat.view(B, S, H, D), *heads, out, lse, **kw)
    dqkv = torch.cat([dq, dk, dv], 2).flatten(2)
    dy0 = op("Matmul", dqkv, c["wqkv"].t())
    dwqkv = op("Matmul", y0.reshape(-1, C).t(), dqkv.reshape(-1, dqkv.shape[-1]))
    dx, df, dg0, _, dp0, _, dgate = op("ResidualNormGrad", dt0, dy0, c["x"], c["f"], **n0)
    for name, grad in {"x": dx, "f": df, "g0": dg0, "p0": dp0, "gate": dgate, "wqkv": dwqkv, "wo": dwo, "table": dtable, "g1": dg1}.items():
        want = w[name].grad
        off = float((grad.cpu().double() - want).norm() / want.norm())
        assert off < 1e-4, (name, off)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_operators_as_graph_nodes(dtype):
    from b200.backend import B200Backend
    from b200.graph import from_json

    def node(i, kind, inputs, **attributes):
        return {"id": i, "op_type": kind, "inputs": inputs, "attributes": attributes}

    inputs = ["q", "k", "v", "len", "table", "do", "x", "f", "gamma"]
    nodes = [{"id": i, "op_type": "Input", "inputs": [], "attributes": {}} for i in inputs] + [
        node("att", "Attention", ["q", "k", "v", "len", "len", "table"], causal=True),
        node("out", "TupleGetItem", ["att"], index=0), node("lse", "TupleGetItem", ["att"], index=1),
        node("ag", "AttentionGrad", ["do", "q", "k", "v", "out", "lse", "len", "len", "table"], causal=True),
        node("dk", "TupleGetItem", ["ag"], index=1), node("dt", "TupleGetItem", ["ag"], index=3),
        node("bias", "RelativePositionBias", ["table"], queries=9, keys=11),
        node("dbias", "RelativePositionBiasGrad", ["bias"], buckets=32),
        node("rn", "ResidualNorm", ["x", "f", "gamma"], residual_scale=0.5),
        node("sum", "TupleGetItem", ["rn"], index=0), node("normed", "TupleGetItem", ["rn"], index=1),
        node("rg", "ResidualNormGrad", ["sum", "normed", "x", "f", "gamma"], residual_scale=0.5),
        node("dx", "TupleGetItem", ["rg"], index=0), node("dgamma", "TupleGetItem", ["rg"], index=2),
    ]
    outs = ["out", "lse", "dk", "dt", "bias", "dbias", "sum", "normed", "dx", "dgamma"]
    graph = from_json({"name": "block", "nodes": nodes, "inputs": inputs, "outputs": outs})
    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)  # noqa: E731

    def values():
        return {"q": r(2, 90, 4, 64), "k": r(2, 90, 2, 64), "v": r(2, 90, 2, 64), "len": torch.randint(1, 91, (2,), generator=g, device="cuda"),
                "table": r(32, 4), "do": r(2, 90, 4, 64), "x": r(30, 72), "f": r(30, 72), "gamma": r(72)}

    def calls(v):
        kw = {"lengths": v["len"], "query_lengths": v["len"], "relative_bias": v["table"], "causal": True}
        out, lse = op("Attention", v["q"], v["k"], v["v"], **kw)
        ag = op("AttentionGrad", v["do"], v["q"], v["k"], v["v"], out, lse, **kw)
        bias = op("RelativePositionBias", v["table"], queries=9, keys=11)
        total, normed = op("ResidualNorm", v["x"], v["f"], v["gamma"], residual_scale=0.5)
        rg = op("ResidualNormGrad", total, normed, v["x"], v["f"], v["gamma"], residual_scale=0.5)
        return [out, lse, ag[1], ag[3], bias, op("RelativePositionBiasGrad", bias, buckets=32), total, normed, rg[0], rg[2]]

    compiled = B200Backend.compile_graph(graph)
    for _ in range(3):
        v = values()
        want = calls(v)
        for got in (B200Backend.execute_graph(graph, v), compiled(v)):
            for name, t in zip(outs, want):
                assert torch.equal(got[name], t), name


@pytest.mark.parametrize("dtype,dim", [(BF, 64), (BF, 128), (F32, 64), (BF, 100)])
def test_tokens_one_at_a_time_equal_the_prompt(dtype, dim):
    """Prompts of several lengths, padded, then the same tokens one by one from a cache of more places, whose rest is left as it
    was and not read. Both are the same sums in another order: 2 half steps of bf16 of the terms, fp32 1e-5."""
    g = torch.Generator().manual_seed(2)
    n, lengths = 30, torch.tensor([30, 7, 19])
    q, k, v = (torch.randn(3, n, h, dim, generator=g).to(dtype) for h in (H, HK, HK))
    table = torch.randn(16, H, generator=g).to(dtype)
    kw = {"causal": True, "relative_bias": table.cuda(), "max_distance": 12}
    whole, lse = op("Attention", q.cuda(), k.cuda(), v.cuda(), lengths=lengths.cuda(), query_lengths=lengths.cuda(), **kw)
    ref, mag = R.attention(q, k, v, lengths=lengths, query_lengths=lengths, causal=True, table=table, far=12)
    caches = [torch.full((3, 64, HK, dim), math.nan, dtype=dtype, device="cuda") for _ in range(2)]
    for t in range(n):
        now = (lengths > t).long()
        for cache, x in zip(caches, (k, v)):
            for e in range(3):
                if now[e]:
                    cache[e, t] = x[e, t].cuda()
        have = torch.minimum(lengths, torch.tensor(t + 1))
        one, one_lse = op("Attention", q[:, t : t + 1].cuda(), *caches, lengths=have.cuda(), **kw)
        for e in range(3):
            if not now[e]:
                continue
            inner = 2 * R.HALF_STEP[BF] if dtype == BF else 0.0
            tol = R.HALF_STEP[dtype] * ref["out"][e, t].abs() + (1e-5 + inner) * mag["out"][e, t]
            assert ((one[e, 0].cpu().double() - ref["out"][e, t]).abs() <= tol).all()
            assert ((whole[e, t].cpu().double() - ref["out"][e, t]).abs() <= tol).all()
            assert (one_lse[e, :, 0] - lse[e, :, t]).abs().max() < 1e-4
    for e in range(3):
        assert caches[0][e, lengths[e]:].isnan().all()


def test_threads_call_at_once():
    import threading

    g = torch.Generator(device="cuda").manual_seed(4)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    sets = [tuple(r(2, 200, h, d).to(t) for h in (4, 2, 2, 4)) for d, t in ((64, BF), (128, BF), (160, BF), (64, F32))]
    table, x = r(256, 4), r(64, 640)
    torch.cuda.synchronize()

    def work():
        res = [op("RelativePositionBias", table, queries=20, keys=70, max_distance=1024), *op("ResidualNorm", x, x, post_norm=True)]
        for q, k, v, do in sets:
            kw = {"relative_bias": table, "max_distance": 1024}
            out, lse = op("Attention", q, k, v, **kw)
            res += [out, lse, *op("AttentionGrad", do, q, k, v, out, lse, **kw)]
        return res

    want = work()
    torch.cuda.synchronize()
    wrong = []

    def run():
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(6):
                got = work()
                s.synchronize()
                wrong.extend(i for i, (a, b) in enumerate(zip(got, want)) if not torch.equal(a, b))

    threads = [threading.Thread(target=run) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("queries", [1, 40])
def test_offsets_beyond_32_bits(queries):
    """A cache whose second sequence, and whose tokens, lie more than 2^31 elements behind the first."""
    g = torch.Generator(device="cuda").manual_seed(5)
    n, step, far = 50, 1 << 20, (1 << 31) + (1 << 26)
    big = torch.empty(far + n * step + 4096, dtype=BF, device="cuda")
    k, v = (big.as_strided((2, n, 2, 64), (far, step, 64, 1), o) for o in (0, 256))
    small = [torch.randn(2, n, 2, 64, generator=g, device="cuda").to(BF) for _ in range(2)]
    k.copy_(small[0])
    v.copy_(small[1])
    q, do = (torch.randn(2, queries, 4, 64, generator=g, device="cuda").to(BF) for _ in range(2))
    want, lse = op("Attention", q, *small, causal=True)
    got, lse2 = op("Attention", q, k, v, causal=True)
    assert torch.equal(got, want) and torch.equal(lse, lse2)
    for a, b in zip(op("AttentionGrad", do, q, *small, want, lse, causal=True)[:3], op("AttentionGrad", do, q, k, v, got, lse, causal=True)[:3]):
        assert torch.equal(a, b)
