"""The Mamba block's operators on the host: sizes near the largest and what forward-mode differentiation gets."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from conftest import load_package


@pytest.fixture(scope="module")
def pkg():
    return load_package()


def _scan_args(pkg, length, channels=1, states=1):
    buf = (ctypes.c_int32 * 160)()
    for i, v in enumerate([pkg._lib.EL_BF16, 1, length, channels, 1, states]):
        buf[i] = v
    return buf


def _calls(o):
    t, w, s = torch.zeros(2, 3, 8), torch.zeros(8, 4), torch.zeros(2, 3, 8)
    return {"causal_conv": (o.causal_conv, dict(x=t, weight=w, bias=t, initial_state=s)),
            "causal_conv_step": (o.causal_conv_step, dict(x=t, state=s, weight=w, bias=t)),
            "selective_scan": (o.selective_scan, dict(u=t, dt=t, A=w, B=t, C=t, D=t, z=t, dt_bias=t, initial_state=s)),
            "selective_scan_step": (o.selective_scan_step, dict(u=t, dt=t, A=w, B=t, C=t, state=s, D=t, z=t, dt_bias=t)),
            "block_norm": (o.block_norm, dict(h=t, y=t, post_weight=w, pre_weight=w, gate=t, scale=w))}


@pytest.mark.parametrize("name", ["causal_conv", "causal_conv_step", "selective_scan", "selective_scan_step", "block_norm"])
@pytest.mark.parametrize("recording", [True, False])
def test_forward_mode_is_refused(pkg, name, recording):
    """A tangent would be lost without a word: any argument that has one is refused, also where no gradient is recorded."""
    call, args = _calls(pkg.ssm_ops)[name]
    with fwAD.dual_level(), torch.set_grad_enabled(recording):
        for k, v in args.items():
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(**{**args, k: fwAD.make_dual(v, torch.ones_like(v))})
        with pytest.raises(RuntimeError, match="must be a CUDA tensor"):      # no tangent: the ordinary checks
            call(**args)
