"""The learned position bias and its table's gradient. The bias is a copy: equal. The gradient is a sum of
fp32 terms: up to 64 rows a batch entry and thread in four sums, then diagonals, runs and blocks in order; below
200 roundings of 2^-24 of the terms (1.2e-5) for these sizes, and half a step of its type."""

import pytest
import torch

import block_reference as R

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _device(cuda):
    yield


def op(name, *args, **kw):
    from b200.backend import B200Backend

    return B200Backend.execute_op(name, *args, **kw)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("buckets,far,bidirectional", [(32, 128, True), (32, 128, False), (4, 2, True), (256, 1024, True), (128, 1000, False),
                                                       (2, 5, False), (6, 7, True)])
@pytest.mark.parametrize("nq,nk,shift", [(1, 1, None), (1, 300, None), (257, 1, None), (65, 130, None), (130, 65, 0), (33, 2100, 5), (40, 40, -17),
                                         (300, 301, 100)])
def test_bias_and_gradient(nq, nk, shift, buckets, far, bidirectional, dtype):
    heads, batch = 3, 2
    g = torch.Generator().manual_seed(nq + nk + buckets)
    table = torch.randn(buckets, heads, generator=g).to(dtype)
    where = R.bias_buckets(nq, nk, nk - nq if shift is None else shift, buckets, far, bidirectional)
    kw = {"bidirectional": bidirectional, "max_distance": far, "shift": shift}
    got = op("RelativePositionBias", table.cuda(), queries=nq, keys=nk, **kw)
    assert got.dtype == dtype and torch.equal(got.cpu(), table[where].permute(2, 0, 1))
    d = torch.randn(batch, heads, nq, nk, generator=g).to(dtype)
    grad = op("RelativePositionBiasGrad", d.cuda(), buckets=buckets, **kw)
    ref, mag = torch.zeros(2, buckets, heads, dtype=torch.float64)
    for out, t in ((ref, d.double()), (mag, d.double().abs())):
        out.index_add_(0, where.flatten(), t.sum(0).flatten(1).t())
    off, tol = (grad.cpu().double() - ref).abs(), R.HALF_STEP[dtype] * ref.abs() + 1.2e-5 * mag
    assert grad.dtype == dtype and not (off > tol).any()


def test_layouts_and_runs():
    d = torch.randn(3, 4, 2, 50, 70, device="cuda")  # more leading axes, and a transposed view
    want = op("RelativePositionBiasGrad", d, buckets=16)
    assert torch.equal(want, op("RelativePositionBiasGrad", d.flatten(0, 1), buckets=16))
    turned = d.transpose(-1, -2).contiguous().transpose(-1, -2)
    assert torch.equal(want, op("RelativePositionBiasGrad", turned, buckets=16))
    one = op("RelativePositionBiasGrad", d[0, 0], buckets=16)
    assert torch.equal(one, op("RelativePositionBiasGrad", d[:1, :1], buckets=16))
    table = torch.randn(2, 32, device="cuda").t()
    assert torch.equal(op("RelativePositionBias", table, queries=5, keys=9), op("RelativePositionBias", table.contiguous(), queries=5, keys=9))


def test_nothing_to_do():
    table = torch.randn(32, 2, device="cuda")
    assert op("RelativePositionBias", table, queries=0, keys=5).shape == (2, 0, 5)
    assert op("RelativePositionBias", table, queries=3, keys=0).shape == (2, 3, 0)
    got = op("RelativePositionBiasGrad", torch.zeros(0, 2, 4, 4, device="cuda"), buckets=32)
    assert got.shape == (32, 2) and not got.any()
