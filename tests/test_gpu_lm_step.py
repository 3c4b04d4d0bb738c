"""The language-model operators as they are used together: one decoder layer's training step
(embedding, projections, query / key norm with rotary positions, attention, tied head with
its loss, every gradient, the updates), the same through the whole-graph hooks, and tokens
one at a time against the whole prompt."""

import math

import pytest
import torch

import lm_reference as R

pytestmark = pytest.mark.gpu

B, S, H, HK, D, V = 2, 24, 4, 2, 16, 333
E = 48
KW = {"rotary_dim": 12, "interleaved": True, "scaling": {"kind": "linear", "factor": 2.0}}
SCALE = 1.0 / math.sqrt(D)


@pytest.fixture(autouse=True)
def _policy(cuda):
    from b200 import ops

    ops.Config.matmul_dtype = "f32"
    yield
    ops.Config.matmul_dtype = "f32"


def op(name, *args, **kw):
    from b200.backend import B200Backend

    return B200Backend.execute_op(name, *args, **kw)


def weights():
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    p = {"emb": r(V, E) * 0.3, "wqkv": r(E, (H + 2 * HK) * D) / E**0.5, "wo": r(H * D, E) / (H * D) ** 0.5,
         "gq": 1 + 0.1 * r(D), "gk": 1 + 0.1 * r(D)}
    ids = torch.randint(0, V, (B, S), generator=g)
    labels = torch.roll(ids, -1, 1)
    labels[:, -1] = -100
    return p, ids, labels


def reference(p, ids, labels):
    """Loss and gradients by autograd in 64 bits on the CPU."""
    p = {k: v.double().requires_grad_() for k, v in p.items()}
    h = p["emb"][ids]
    q, k, v = (h @ p["wqkv"]).view(B, S, H + 2 * HK, D).split([H, HK, HK], 2)
    w, f = R.angles(KW["rotary_dim"], 10000.0, KW["scaling"])
    t = torch.arange(S).double()[None, :, None, None] * torch.tensor(w, dtype=torch.float64)

    def norm_rotate(x, gamma):
        x = R.rms_unit(x, 1e-6)[0] * gamma
        a, b, rest = x[..., 0:12:2], x[..., 1:12:2], x[..., 12:]
        turned = torch.stack([a * t.cos() - b * t.sin(), b * t.cos() + a * t.sin()], -1).flatten(-2)
        return torch.cat([turned, rest], -1)

    q, k = norm_rotate(q, p["gq"]), norm_rotate(k, p["gk"])
    k, v = (x.repeat_interleave(H // HK, 2) for x in (k, v))
    a = torch.softmax(torch.einsum("bshd,bthd->bhst", q, k) * SCALE, -1)
    y = torch.einsum("bhst,bthd->bshd", a, v).reshape(B, S, H * D) @ p["wo"] + h
    z = y @ p["emb"].t()
    keep = labels >= 0
    loss = (torch.logsumexp(z, -1) - z.gather(-1, labels.clamp(min=0)[..., None])[..., 0])[keep].mean()
    loss.backward()
    return loss.detach(), {k: v.grad for k, v in p.items()}


def step(p, ids, labels):
    """The same through execute_op."""
    n = int((labels >= 0).sum())
    h = op("Take", p["emb"], ids, axis=0)
    h2 = h.view(B * S, E)
    qkv = op("Matmul", h2, p["wqkv"]).view(B, S, H + 2 * HK, D)
    q0, k0, v0 = qkv.split([H, HK, HK], 2)
    q, k = op("QKNormRotary", q0, k0, p["gq"], p["gk"], **KW)
    group = H // HK
    heads = lambda x: op("Transpose", x, axes=[0, 2, 1, 3])  # noqa: E731
    q4 = op("Reshape", heads(q), shape=[B, HK, group, S, D])
    k4, v4 = (op("Reshape", heads(x), shape=[B, HK, 1, S, D]) for x in (k, v0))
    a = op("Softmax", op("Multiply", op("Matmul", q4, op("Transpose", k4, axes=[0, 1, 2, 4, 3])), SCALE))
    o = op("Reshape", heads(op("Reshape", op("Matmul", a, v4), shape=[B, H, S, D])), shape=[B * S, H * D])
    y = op("Add", op("Matmul", o, p["wo"]), h2)
    head = p["emb"].t()
    losses, lse = op("LinearCrossEntropy", y, head, labels.view(-1))
    dloss = torch.full_like(losses, 1.0 / n)
    dy, dhead = op("LinearCrossEntropyGrad", dloss, y, head, labels.view(-1), lse)
    g = {"wo": op("Matmul", op("Transpose", o), dy)}
    do = op("Reshape", heads(op("Matmul", dy, op("Transpose", p["wo"])).view(B, S, H, D)), shape=[B, HK, group, S, D])
    dv = op("ReduceSum", op("Matmul", op("Transpose", a, axes=[0, 1, 2, 4, 3]), do), axis=2)
    da = op("Matmul", do, op("Transpose", v4, axes=[0, 1, 2, 4, 3]))
    ds = op("Multiply", op("Multiply", a, op("Subtract", da, op("ReduceSum", op("Multiply", da, a), axis=-1, keepdims=True))), SCALE)
    dq = heads(op("Reshape", op("Matmul", ds, k4), shape=[B, H, S, D]))
    dk = heads(op("ReduceSum", op("Matmul", op("Transpose", ds, axes=[0, 1, 2, 4, 3]), q4), axis=2))
    dq0, dk0, g["gq"], g["gk"] = op("QKNormRotaryGrad", dq, dk, q0, k0, p["gq"], p["gk"], **KW)
    dqkv = torch.cat([dq0.reshape(B * S, -1), dk0.reshape(B * S, -1), heads(dv).reshape(B * S, -1)], 1)
    g["wqkv"] = op("Matmul", op("Transpose", h2), dqkv)
    dh = op("Add", op("Matmul", dqkv, op("Transpose", p["wqkv"])), dy)
    g["emb"] = op("TensorScatterAdd", dhead.t(), ids.view(-1, 1), dh)
    return losses, g


def test_decoder_training_step_matches_64_bit_gradients():
    p, ids, labels = weights()
    ref, grads = reference(p, ids, labels)
    dev = {k: v.cuda() for k, v in p.items()}
    losses, g = step(dev, ids.cuda(), labels.cuda())
    # some ten fp32 products and normalisations in a row, each good to 1e-5 in norm
    assert abs(float(losses.sum()) / int((labels >= 0).sum()) - float(ref)) <= 1e-4 * float(ref)
    for k, want in grads.items():
        off = float((g[k].cpu().double() - want).norm() / want.norm())
        assert off <= 1e-4, f"{k}: {off:.2e}"
    # the updates: matrices orthogonalised, the embedding by Adam
    for k in ("wqkv", "wo"):
        new, mom = op("ApplyMuon", dev[k], torch.zeros_like(dev[k]), g[k], lr=0.1)
        o = R.newton_schulz(1.95 * g[k].cpu().double())
        rows, cols = o.shape
        want = p[k].double() - 0.1 * math.sqrt(max(1.0, rows / cols)) * o
        assert float((new.cpu().double() - want).norm() / (new.cpu().double() - p[k].double()).norm()) <= 1e-4
        assert torch.equal(mom, g[k])
    z = torch.zeros_like(dev["emb"])
    assert torch.isfinite(op("ApplyAdam", dev["emb"], z, z, g["emb"])[0]).all()


@pytest.mark.parametrize("policy", ["f32", "bf16"])
def test_operators_as_graph_nodes(policy):
    """Through execute_graph and compile_graph: the same results as one call after the other,
    with inputs changed between replays."""
    from b200 import ops
    from b200.backend import B200Backend
    from b200.graph import from_json

    ops.Config.matmul_dtype = policy
    node = lambda i, t, ins, **a: {"id": i, "op_type": t, "inputs": ins, "attributes": a}  # noqa: E731
    inputs = ["q", "k", "gq", "gk", "pos", "x", "w", "labels", "dloss", "m", "g"]
    nodes = [node(i, "Input", []) for i in inputs] + [
        node("qk", "QKNormRotary", ["q", "k", "gq", "gk", "pos"], **KW),
        node("q1", "TupleGetItem", ["qk"], index=0), node("k1", "TupleGetItem", ["qk"], index=1),
        node("r", "RotaryEmbedding", ["q1", "pos"], rotary_dim=8),
        node("back", "QKNormRotaryGrad", ["r", "k1", "q", "k", "gq", "gk", "pos"], **KW),
        node("dq", "TupleGetItem", ["back"], index=0), node("dgk", "TupleGetItem", ["back"], index=3),
        node("ce", "LinearCrossEntropy", ["x", "w", "labels"]),
        node("loss", "TupleGetItem", ["ce"], index=0), node("lse", "TupleGetItem", ["ce"], index=1),
        node("ceg", "LinearCrossEntropyGrad", ["dloss", "x", "w", "labels", "lse"]),
        node("dx", "TupleGetItem", ["ceg"], index=0), node("dw", "TupleGetItem", ["ceg"], index=1),
        node("total", "Add", ["dw", "w"]),
        node("ns", "NewtonSchulz", ["total"]),
        node("mu", "ApplyMuon", ["w", "m", "g"], lr=0.1), node("w1", "TupleGetItem", ["mu"], index=0),
    ]
    outs = ["q1", "k1", "r", "dq", "dgk", "loss", "lse", "dx", "dw", "ns", "w1"]
    graph = from_json({"name": "lm", "nodes": nodes, "inputs": inputs, "outputs": outs})
    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731

    def values():
        return {"q": r(2, 9, 4, D), "k": r(2, 9, 2, D), "gq": r(D), "gk": r(D), "pos": torch.randint(0, 99, (2, 9), generator=g, device="cuda"),
                "x": r(18, 40), "w": r(40, 120), "labels": torch.randint(0, 120, (18,), generator=g, device="cuda"), "dloss": r(18),
                "m": r(40, 120), "g": r(40, 120)}

    def calls(v):
        q1, k1 = op("QKNormRotary", v["q"], v["k"], v["gq"], v["gk"], v["pos"], **KW)
        rr = op("RotaryEmbedding", q1, v["pos"], rotary_dim=8)
        back = op("QKNormRotaryGrad", rr, k1, v["q"], v["k"], v["gq"], v["gk"], v["pos"], **KW)
        loss, lse = op("LinearCrossEntropy", v["x"], v["w"], v["labels"])
        dx, dw = op("LinearCrossEntropyGrad", v["dloss"], v["x"], v["w"], v["labels"], lse)
        return [q1, k1, rr, back[0], back[3], loss, lse, dx, dw, op("NewtonSchulz", op("Add", dw, v["w"])),
                op("ApplyMuon", v["w"], v["m"], v["g"], lr=0.1)[0]]

    compiled = B200Backend.compile_graph(graph)
    for _ in range(3):
        v = values()
        want = calls(v)
        for got in (B200Backend.execute_graph(graph, v), compiled(v)):
            for name, w in zip(outs, want):
                assert torch.equal(got[name], w), name


def test_tokens_one_at_a_time_equal_the_prompt():
    """A decoding loop: each new token's queries and keys, at its own position, are those of
    the whole prompt bit for bit; keys written into a longer cache leave the rest as it was."""
    g = torch.Generator(device="cuda").manual_seed(2)
    qkv = torch.randn(3, 20, H + 2 * HK, 64, generator=g, device="cuda").to(torch.bfloat16)
    gq, gk = torch.randn(64, generator=g, device="cuda"), torch.randn(64, generator=g, device="cuda")
    kw = {"scaling": {"kind": "yarn", "factor": 4.0, "original_length": 16}}
    q, k = op("QKNormRotary", qkv[:, :, :H], qkv[:, :, H : H + HK], gq, gk, offset=5, **kw)
    cache = torch.full((3, 64, HK, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    for t in range(20):
        one = qkv[:, t : t + 1]
        q1, k1 = op("QKNormRotary", one[:, :, :H], one[:, :, H : H + HK], gq, gk, torch.full((3, 1), 5 + t, device="cuda"), **kw)
        cache[:, t : t + 1] = k1
        assert torch.equal(q1, q[:, t : t + 1]) and torch.equal(k1, k[:, t : t + 1])
    assert torch.equal(cache[:, :20], k) and (cache[:, 20:] == 7).all()


def test_two_threads_call_at_once():
    """Each on its own stream: results of neither depend on the other."""
    import threading

    g = torch.Generator(device="cuda").manual_seed(4)
    x, w = torch.randn(64, 128, generator=g, device="cuda"), torch.randn(128, 700, generator=g, device="cuda")
    labels = torch.randint(0, 700, (64,), generator=g, device="cuda")
    mats = torch.randn(2, 200, 136, generator=g, device="cuda")
    torch.cuda.synchronize()

    def work():
        loss, lse = op("LinearCrossEntropy", x, w, labels)
        return [loss, *op("LinearCrossEntropyGrad", lse, x, w, labels, lse), op("NewtonSchulz", mats), op("RotaryEmbedding", x.view(1, 64, 2, 64))]

    want = work()
    torch.cuda.synchronize()
    wrong = []

    def run():
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(10):
                got = work()
                s.synchronize()
                wrong.extend(i for i, (a, b) in enumerate(zip(got, want)) if not torch.equal(a, b))

    threads = [threading.Thread(target=run) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
