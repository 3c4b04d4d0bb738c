"""Arguments of the block operators at the ends of their ranges, on the host (no kernel runs)."""

import sys

import pytest
import torch

from b200 import block_ops


@pytest.mark.parametrize("window", [1, 7.0, 2**31, 2**31 + 5, sys.maxsize, 2**63, 2**64 + 2**13, 10**400, float("inf")])
def test_a_window_reaches_the_kernels_as_itself_or_as_more_than_any_length(window):
    got = block_ops._window("Attention", window)
    assert got == (window if window <= 2**31 else 2**31)
    x = torch.Size((1, 4, 2, 64))
    plan = block_ops._attention_plan("Attention", (x,) * 3, (torch.float32,) * 3, None, None, True, got, 128, None)
    assert plan.window == got
    assert block_ops._window("Attention", None) == 0


@pytest.mark.parametrize("window", [0, -1, 0.5, 1.5, float("nan"), -float("inf"), -(2**64) + 5])
def test_no_windows(window):
    x = torch.zeros(1, 4, 2, 64)
    with pytest.raises(ValueError):
        block_ops.op_attention(x, x, x, window=window)


@pytest.mark.parametrize("shift", [2**29, -(2**29), 2**31, 2**63, 2**64, 2**64 + 7, -(2**64) - 7])
def test_a_shift_is_not_taken_for_another_one(shift):
    """Numbers beyond int64 wrap on their way into C."""
    with pytest.raises(ValueError):
        block_ops.op_relative_position_bias(torch.zeros(32, 2), queries=3, keys=4, shift=shift)
    with pytest.raises(ValueError):
        block_ops.op_relative_position_bias_grad(torch.zeros(2, 3, 4), buckets=32, shift=shift)
    assert block_ops._shift("RelativePositionBias", 2**29 - 1, 3, 4) == 2**29 - 1 and block_ops._shift("RelativePositionBias", None, 3, 4) == 1


def test_the_gradients_workspace_has_a_copy_of_dout_only_where_one_is_made():
    from b200 import _lib as L

    lib, a, g = L.load(), L.Attention(), L.AttentionGrads()
    a.batch, a.queries, a.keys, a.heads, a.kv_heads, a.dim, a.scale, a.dtype = 2, 100, 120, 4, 2, 64, 1.0, L.BF16
    a.q = a.k = a.v = 4096
    a.q_stride[:] = 100 * 256, 256, 64
    a.k_stride[:] = a.v_stride[:] = 120 * 128, 128, 64
    copy = 2 * 100 * 4 * 64 * 2
    most = lib.b200_attention_grad_workspace_bytes(a)
    g.dout, g.dout_stride[:] = 4096, (100 * 256, 256, 64)
    assert lib.b200_attention_grad_workspace_bytes_of(a, g) == most - copy
    for pointer, strides in ((4098, (100 * 256, 256, 64)), (4096, (100 * 260, 260, 65)), (4096, (0, 256, 64))):
        g.dout, g.dout_stride[:] = pointer, strides
        assert lib.b200_attention_grad_workspace_bytes_of(a, g) == most
    a.dim = 0
    assert lib.b200_attention_grad_workspace_bytes_of(a, g) == 0 and lib.b200_attention_grad_workspace_bytes_of(None, g) == 0


@pytest.mark.parametrize("scale,fine", [(2.3e38, True), (2.4e38, False), (2.9e38, False), (1e-45, True)])
def test_a_scale_stays_a_number_in_the_log2_domain(scale, fine):
    """Above 2.35e38 scale log2 e is infinite, and a score of zero was not a number."""
    from b200 import _lib as L

    lib, a = L.load(), L.Attention()
    a.batch, a.queries, a.keys, a.heads, a.kv_heads, a.dim, a.scale = 0, 4, 4, 2, 1, 64, scale
    assert lib.b200_attention_forward(a, None, None, None, 0, None) == (L.OK if fine else L.ERR_ARG)
