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


@pytest.mark.parametrize("length", [1 << 20, (1 << 31) - (1 << 27), (1 << 31) - (1 << 26) - 40, 0x7fff0000])
def test_workspaces_of_the_longest_sequences(pkg, length):
    """One channel: 32 chunks, each with a state and a sum of step sizes; backward adds dB and dC of every token and a chunk's dA, dD, dbias."""
    lib = pkg._lib.lib()
    assert lib.el_selective_scan_workspace_bytes(_scan_args(pkg, length)) == 32 * 2 * 4
    assert lib.el_selective_scan_backward_workspace_bytes(_scan_args(pkg, length)) == (2 * length + 32 * 3 + 32 * 2) * 4


def test_longer_sequences_are_refused(pkg):
    lib = pkg._lib
    assert lib.lib().el_selective_scan(_scan_args(pkg, 0x7fff0001), None) == lib.EL_ERR_TOO_LARGE
    assert lib.lib().el_selective_scan_workspace_bytes(_scan_args(pkg, 0x7fff0001)) == 0


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
