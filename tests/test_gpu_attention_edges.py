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
