"""Calls of Attention and its gradient at the ends of what their arguments may be."""

import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _device(cuda):
    yield


def op(name, *args, **kw):
    from b200.backend import B200Backend

    return B200Backend.execute_op(name, *args, **kw)


def rand(*shape, dtype=F32, seed=0):
    g = torch.Generator().manual_seed(seed + sum(shape))
    return torch.randn(*shape, generator=g).to(dtype).cuda()


def inputs(b, nq, nk, h, hk, d, dtype, seed=0):
    return (rand(b, nq, h, d, dtype=dtype, seed=seed), rand(b, nk, hk, d, dtype=dtype, seed=seed + 1), rand(b, nk, hk, d, dtype=dtype, seed=seed + 2),
            rand(b, nq, h, d, dtype=dtype, seed=seed + 3))


@pytest.mark.parametrize("dtype,dim", [(BF, 64), (BF, 160), (F32, 64)])
@pytest.mark.parametrize("nq,nk,causal", [(70, 90, True), (70, 90, False), (90, 40, True), (3, 90, True)])
def test_windows_that_hide_nothing(nq, nk, causal, dtype, dim, monkeypatch):
    """Up to the largest number that the C struct holds, and beyond it in Python: as without a window."""
    from b200 import block_ops

    q, k, v, do = inputs(1, nq, nk, 2, 1, dim, dtype)
    want = op("Attention", q, k, v, causal=causal)
    grads = op("AttentionGrad", do, q, k, v, *want, causal=causal)
    describe = block_ops._describe
    for window in (nq + nk, sys.maxsize, 2**63, 2**64 + 3, float("inf"), None):
        if window is None:  # the C struct's largest

            def largest(*args):
                d = describe(*args)
                d[0].window = 2**63 - 1
                return d

            monkeypatch.setattr(block_ops, "_describe", largest)
        got = op("Attention", q, k, v, causal=causal, window=window)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), window
        again = op("AttentionGrad", do, q, k, v, *want, causal=causal, window=window)
        assert all(torch.equal(a, b) for a, b in zip(again[:3], grads[:3])), window


@pytest.mark.parametrize("low", [-1e7, -1e9, torch.finfo(BF).min])
@pytest.mark.parametrize("dtype,dim,nq", [(BF, 64, 70), (BF, 128, 70), (F32, 64, 70), (BF, 160, 70), (BF, 64, 9)])
def test_rows_whose_lse_cannot_tell_their_keys_apart(dtype, dim, nq, low):
    """A bias that leaves the first query nothing but entries of a large negative value: without a gradient of its own the step is
    right and no flag is set; with one its row is left out and the flag says so. Rows that see other keys are not touched."""
    from b200 import _lib as L

    q, k, v, do = inputs(2, nq, nq, 4, 2, dim, dtype)
    table = rand(16, 4, dtype=dtype, seed=9)
    table[0] = low  # distance 0: all that the first query of a causal sequence sees
    kw = {"relative_bias": table, "causal": True, "max_distance": 30}
    out, lse = op("Attention", q, k, v, **kw)
    assert (lse[:, :, 0] < -(2**20)).all() and (lse[:, :, 1:].abs() < 100).all()
    quiet = do.clone()
    quiet[:, 0] = 0
    L.lib().b200_check_device_error(None)
    want = op("AttentionGrad", quiet, q, k, v, out, lse, **kw)
    assert L.lib().b200_check_device_error(None) == L.OK
    wrong = check_gradients(want, (q, k, v, quiet), table)
    assert not wrong, wrong
    got = op("AttentionGrad", do, q, k, v, out, lse, **kw)
    assert L.lib().b200_check_device_error(None) == L.ERR_ARG
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and not got[0][:, 0].any()


def check_gradients(grads, operands, table):
    import rounding_norms as N

    q, k, v, do = (t.cpu() for t in operands)
    ref, var = N.attention_noise(q, k, v, do, table=table.cpu(), causal=True, far=30)
    off = {n: N.attention_off(n, t, ref, var) for n, t in zip(("dq", "dk", "dv", "dtable"), grads)}
    return {n: t for n, t in off.items() if t}


@pytest.mark.parametrize("dtype,dim,nq", [(BF, 64, 70), (F32, 64, 70)])
def test_large_biases_below_that_have_their_gradient(dtype, dim, nq):
    """-65536 for every key: the exponent is off by five roundings, p by 1.2 % at most, and no flag is set."""
    from b200 import _lib as L

    q, k, v, do = inputs(1, nq, nq, 2, 2, dim, dtype)
    q = q * 0  # the scores are the bias alone, so that 64 bits have the same ones
    table = torch.full((16, 2), -65536.0, dtype=dtype, device="cuda")
    kw = {"relative_bias": table, "max_distance": 30}
    L.lib().b200_check_device_error(None)
    out, lse = op("Attention", q, k, v, **kw)
    dv = op("AttentionGrad", do, q, k, v, out, lse, **kw)[2].cpu().double()
    assert L.lib().b200_check_device_error(None) == L.OK
    want = do.cpu().double().mean(1, keepdim=True).expand(-1, nq, -1, -1)
    assert ((dv - want).norm() / want.norm()) < 0.012 + 2.0**-8


@pytest.mark.parametrize("dtype,dim", [(BF, 64), (BF, 100), (F32, 64)])
@pytest.mark.parametrize("shift", [0, 1])
def test_gradient_stays_in_the_workspace_of_its_dout(dtype, dim, shift, monkeypatch):
    """dout aligned (read in place) and not (copied): what lies behind the workspace is left as it was."""
    from b200 import _lib as L

    q, k, v, do = inputs(2, 70, 90, 4, 2, dim, dtype)
    table = rand(32, 4, seed=9)
    kw = {"causal": True, "relative_bias": table}
    out, lse = op("Attention", q, k, v, **kw)
    want = op("AttentionGrad", do, q, k, v, out, lse, **kw)
    flat = torch.zeros(do.numel() + shift, dtype=dtype, device="cuda")
    moved = flat[shift:].view(do.shape).copy_(do)
    spaces, call = [], L.call

    def guarded(name, *args):
        if name == "b200_attention_grad":
            a, g, _, n, stream = args
            spaces.append(torch.full((n + 4096,), 0x5A, dtype=torch.uint8, device="cuda"))
            args = (a, g, spaces[0].data_ptr(), n, stream)
        return call(name, *args)

    monkeypatch.setattr(L, "call", guarded)
    got = op("AttentionGrad", moved, q, k, v, out, lse, **kw)
    assert len(spaces) == 1 and (spaces[0][-4096:] == 0x5A).all()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
