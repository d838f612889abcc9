"""The Mamba block's operators on the host: what the C entry points refuse before they touch a device, what the Python functions refuse, and the
reference implementation that the GPU tests compare with against torch's own convolution."""
import ctypes

import pytest
import torch
import torch.nn.functional as F

import ssm_reference as R
from conftest import load_package


@pytest.fixture(scope="module")
def pkg():
    return load_package()


def _struct(first_ints, size=640):
    """A zeroed argument struct whose leading 32-bit fields are given."""
    buf = (ctypes.c_int32 * (size // 4))()
    for i, v in enumerate(first_ints):
        buf[i] = v
    return buf


@pytest.mark.parametrize("name", ["el_causal_conv", "el_causal_conv_backward", "el_causal_conv_step", "el_selective_scan", "el_selective_scan_backward",
                                  "el_selective_scan_step", "el_block_norm", "el_block_norm_backward"])
def test_entry_points_refuse_on_the_host(pkg, name):
    lib, fn = pkg._lib, getattr(pkg._lib.lib(), name)
    assert fn(None, None) == lib.EL_ERR_NULL_PTR
    assert fn(_struct([9]), None) == lib.EL_ERR_INVALID_ARG                                # dtype
    assert fn(_struct([lib.EL_BF16, -1]), None) == lib.EL_ERR_INVALID_ARG                  # a negative size
    if "conv" in name:                   # dtype, batch, length, channels, width
        assert fn(_struct([lib.EL_BF16, 1, 8, 8, 5]), None) == lib.EL_ERR_UNSUPPORTED_SHAPE
    elif "scan" in name:                 # dtype, batch, length, channels, groups, states
        assert fn(_struct([lib.EL_BF16, 1, 8, 8, 3, 16]), None) == lib.EL_ERR_INVALID_ARG
        assert fn(_struct([lib.EL_BF16, 1, 8, 8, 1, 65]), None) == lib.EL_ERR_UNSUPPORTED_SHAPE
    else:                                # dtype, rows, width
        assert fn(_struct([lib.EL_BF16, 1, 16385]), None) == lib.EL_ERR_UNSUPPORTED_SHAPE


def test_workspace_sizes(pkg):
    lib, h = pkg._lib, pkg._lib.lib()
    bad = _struct([9])
    for name in ("el_causal_conv_backward_workspace_bytes", "el_selective_scan_checkpoint_bytes", "el_selective_scan_workspace_bytes",
                 "el_selective_scan_backward_workspace_bytes", "el_block_norm_backward_workspace_bytes"):
        assert getattr(h, name)(bad) == 0
    # one state of every eighth token, float32
    assert h.el_selective_scan_checkpoint_bytes(_struct([lib.EL_BF16, 2, 17, 24, 1, 16])) == 2 * 3 * 24 * 16 * 4


@pytest.mark.parametrize("call,message", [
    (lambda o, t: o.causal_conv(t, t), "x must be a CUDA tensor"),
    (lambda o, t: o.causal_conv_step(t, t, t), "x must be a CUDA tensor"),
    (lambda o, t: o.selective_scan(t, t, t, t, t), "u must be a CUDA tensor"),
    (lambda o, t: o.selective_scan_step(t, t, t, t, t, t), "u must be a CUDA tensor"),
    (lambda o, t: o.block_norm(t, t, t, t), "h must be a CUDA tensor"),
    (lambda o, t: o.causal_conv(t.requires_grad_(True), t), "x must be a CUDA tensor"),
    (lambda o, t: o.causal_conv_step(t.requires_grad_(True), t, t), "no gradient"),
])
def test_python_functions_refuse(pkg, call, message):
    with pytest.raises(RuntimeError, match=message):
        call(pkg.ssm_ops, torch.zeros(2, 3, 8))


def test_reference_convolution_is_torchs():
    g = torch.Generator().manual_seed(0)
    x, w, b = torch.randn(2, 11, 6, generator=g, dtype=torch.float64), torch.randn(6, 4, generator=g, dtype=torch.float64), torch.randn(6, generator=g, dtype=torch.float64)
    y, last = R.causal_conv(x, w, b)
    want = F.silu(F.conv1d(F.pad(x.transpose(1, 2), (3, 0)), w[:, None], b, groups=6)).transpose(1, 2)
    assert torch.allclose(y, want, rtol=0, atol=1e-14) and torch.equal(last, x[:, -3:])
