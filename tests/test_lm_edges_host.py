"""Refusals of the language-model operators that the tests by operator leave out (no kernel runs)."""

import ctypes as C

import numpy as np
import pytest
import torch

from b200 import _lib as L
from b200 import lm_ops

P = 256  # a stand-in address: the calls below are refused before anything reads it


@pytest.mark.parametrize("step", [0, 4])
@pytest.mark.parametrize("bad", [(250.0, 0.0, 0.0), (-300.0, 1.0, 1.0), (float("inf"), 0.0, 0.0), (float("nan"), 0.0, 0.0),
                                 (1.0, float("inf"), 0.0), (1.0, float("nan"), 0.0), (1.0, 0.0, float("-inf")), (1.0, 0.0, float("nan"))])
def test_coefficients_that_cannot_be_kept_are_refused(bad, step):
    rows = [(1.0, 0.0, 0.0)] * 5
    rows[step] = bad
    c = (C.c_float * 15)(*[v for r in rows for v in r])
    n = int(L.lib().b200_newton_schulz_workspace_bytes(L.F32, 1, 64, 64))
    assert L.lib().b200_newton_schulz(L.F32, P, P, 1, 64, 64, c, 5, 0.0, P, n, None) == L.ERR_ARG
    assert "coefficients" in L.last_error()
    assert L.lib().b200_apply_muon_f32(P, P, P, P, P, 1, 64, 64, 0.1, 0.9, 1, 0.0, c, 5, 0.0, P, n, None) == L.ERR_ARG
    good = (C.c_float * 15)(*[249.0, -1000.0, 1000.0] * 5)
    assert L.lib().b200_newton_schulz(L.F32, None, None, 0, 64, 64, good, 5, 0.0, None, 0, None) == L.OK


@pytest.mark.parametrize("axis", [0, 3, -3, None, "rows"])
def test_apply_muon_refuses_an_axis_that_is_not_the_matrix(axis):
    t = torch.zeros(2, 4, 5)
    with pytest.raises(ValueError, match="output_axis"):
        lm_ops.op_apply_muon(t, t, t, output_axis=axis)


def test_coefficients_as_arrays_and_without_any():
    rows = [[4.0, -6.9, 2.9], [3.9, -6.3, 2.6], [1.5, -0.5, 0.25]]
    flat = [v for r in rows for v in r]
    for c in (rows, tuple(map(tuple, rows)), np.array(rows), [np.array(r) for r in rows], torch.tensor(rows, dtype=torch.float64)):
        assert list(lm_ops._coef(3, c)) == [np.float32(v) for v in flat]
    for c in (rows[0], np.array(rows[0]), [np.float32(v) for v in rows[0]]):
        assert list(lm_ops._coef(2, c)) == [np.float32(v) for v in rows[0]] * 2
    for c in ((), [], np.zeros((0, 3)), [1.0, [1.0, 2.0, 3.0], 2.0], np.zeros((3, 2)), np.zeros((2, 3))):
        with pytest.raises(ValueError, match="Newton-Schulz"):
            lm_ops._coef(3, c)


@pytest.mark.parametrize("shift", [1, 2, 3])
def test_norm_gradient_refuses_a_workspace_between_floats(shift):
    r = L.Rotary()
    r.head_dim, r.rotary_dim, r.factor = 64, 64, 1.0
    n = int(L.lib().b200_qk_norm_rotary_grad_workspace_bytes(64))
    rc = L.lib().b200_qk_norm_rotary_grad(r, L.BF16, P, P, P, P, P, P, 1, 1, 1, 1, L.I64x18(*[64] * 18), P, P, L.F32, 1e-6, None, L.I64,
                                          0, 0, 0, P, P, P + shift, n, None)
    assert rc == L.ERR_ARG and "aligned" in L.last_error()


def test_loss_gradient_refuses_other_result_types():
    n = int(L.lib().b200_linear_xent_grad_workspace_bytes(L.BF16, P, 64, P, 104, 1, 4, 64, 100))

    def grad(dx_type, dw_type):
        return L.lib().b200_linear_xent_grad_mixed(L.BF16, P, P, 64, P, 104, 1, P, L.I64, -100, P, P, dx_type, P, dw_type, 4, 64, 100, P, n, None)

    for bad in (L.I32, L.F64, L.BOOL):
        assert grad(bad, L.F32) == grad(L.BF16, bad) == L.ERR_DTYPE
