"""The operators of ssm_ops.py at the edges of what they accept, and in the loops that only larger sizes reach: against their definitions in
float64, with the tolerances that test_gpu_ssm_ops.py derives."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwAD
import torch.nn.functional as F

import ssm_reference as R
from test_gpu_ssm_ops import (DEV, NAN, _check_norm, _close, _gen, _leaves, _norm_case, _poison, _randn, _reference_grads,
                               _scan_case, _three)

pytestmark = pytest.mark.gpu
INF = float("inf")


@pytest.fixture(scope="module")
def ops(pkg):
    return pkg.ssm_ops


# ---- derivatives that are not formed --------------------------------------------------------------------------------------

@pytest.mark.parametrize("name", ["conv", "scan", "norm"])
def test_forward_mode_is_refused_where_gradients_are_recorded(ops, name):
    """A tangent of an input that has a gradient too, and one of the output's gradient."""
    call, t, douts = _three(ops)[name]
    gpu = {k: v.to(DEV).requires_grad_(True) for k, v in t.items()}
    douts = [d.to(DEV) for d in douts]
    with fwAD.dual_level():
        for k in gpu:
            with pytest.raises(RuntimeError):
                call(**{**gpu, k: fwAD.make_dual(gpu[k], torch.ones_like(gpu[k]))})
        outs = call(**gpu)
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(outs, list(gpu.values()), [fwAD.make_dual(d, d) for d in douts])
