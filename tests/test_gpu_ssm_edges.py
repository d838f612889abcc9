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


# ---- states that grow ---------------------------------------------------------------------------------------------------

def _growing(L, u_from, dy_to):
    """A state that grows by e^2 per token: e^160 over the 80 tokens of a chunk, which float32 does not hold.  Inputs that are zero before token
    u_from and output gradients that are zero from token dy_to on keep everything that is formed token by token finite."""
    t, _, dy, ds = _scan_case(1, L, 64, 16, 1, torch.float32, state=False, gated=False, bias=False)
    t["A"] = 4.0 + 0.01 * t["A"]
    t["dt"] = torch.full_like(t["dt"], 0.5)
    t["u"][:, :u_from] = 0.0
    dy[:, dy_to:] = 0.0
    return t, dy


def test_scan_of_growing_states_in_chunks_keeps_zeros(ops):
    L = 2500
    t, _ = _growing(L, L - 10, 0)
    d = {k: None if v is None else v.to(DEV) for k, v in t.items()}
    y, s = ops.selective_scan(**d, dt_softplus=False, return_final_state=True)
    yr, sr = R.selective_scan(**{k: None if v is None else v.double() for k, v in t.items()}, softplus=False)
    _close("y", y, yr, 4 * 10 + 16 + 16)                  # ten tokens have a state other than zero
    _close("state", s, sr, 4 * 10 + 16)


def test_scan_gradients_of_growing_states_in_chunks_keep_zeros(ops):
    L = 2500
    t, dy = _growing(L, L - 10, 10)
    gpu, ref = _leaves(t)
    y = ops.selective_scan(**gpu, dt_softplus=False)
    yr, _ = R.selective_scan(**ref, softplus=False)
    names = [k for k, v in gpu.items() if v is not None]
    got = torch.autograd.grad(y, [gpu[k] for k in names], dy.to(DEV))
    want = _reference_grads([yr], [ref[k] for k in names], [dy.double()])
    for k, a, b in zip(names, got, want):
        _close("d" + k, a, b, 8 * 10 + 2 * 16 + 32)
    assert got[0][:, :10].any()


# ---- padding ------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("what", ["initial state", "final state's gradient", "token"])
@pytest.mark.parametrize("N,G", [(16, 1), (12, 2), (64, 1)])
def test_padding_has_zero_gradients_whatever_the_states_hold(ops, what, N, G):
    """Lengths that end inside a tile; a state or a gradient that is not finite in a sequence that has padding."""
    t, lengths, dy, ds = _scan_case(3, 21, 32, N, G, torch.float32)
    lengths = torch.tensor([13, 21, 1])
    for v in (t["u"], t["dt"], t["z"], t["B"], t["C"], dy):
        _poison(v, lengths)
    if what == "initial state":
        t["initial_state"][0, 3], t["initial_state"][2, 5, 1] = INF, NAN
    elif what == "token":
        t["u"][0, 12, 3] = INF
    else:
        ds[0, 3, 2], ds[2, 5] = NAN, INF
    gpu, _ = _leaves(t)
    y, s = ops.selective_scan(**gpu, lengths=lengths.to(DEV), return_final_state=True)
    names = ("u", "dt", "z", "B", "C")
    for k, g in zip(names, torch.autograd.grad((y, s), [gpu[k] for k in names], (dy.to(DEV), ds.to(DEV)))):
        for b, n in enumerate(lengths.tolist()):
            assert not g[b, n:].any(), (k, b)              # a NaN is not zero either
    for b, n in enumerate(lengths.tolist()):
        assert not y[b, n:].any()


# ---- decay rates without bound --------------------------------------------------------------------------------------------

@pytest.mark.parametrize("L,mask", [(21, "full"), (16, "full"), (21, "ragged"), (1500, "full")])
def test_scan_of_states_that_forget_at_once(ops, L, mask):
    """A = -inf: exp(delta A) is 0 for every token, and padding of a tile leaves the state as it is.  (The gradient of the step sizes is
    -inf * 0 in the definition and is not looked at.)"""
    t, lengths, dy, ds = _scan_case(2, L, 32, 16, 1, torch.float32, mask)
    t["A"][3, 2], t["A"][:, 7], t["A"][5] = -INF, -INF, -3e38
    gpu, ref = _leaves(t)
    dev_lengths = None if lengths is None else lengths.to(DEV)
    y, s = ops.selective_scan(**gpu, lengths=dev_lengths, return_final_state=True)
    yr, sr = R.selective_scan(**{k: v if k != "A" else v.detach().masked_fill(t["A"].isinf(), -3.4e38).requires_grad_(True) for k, v in ref.items()}, lengths=lengths)
    _close("y", y, yr, 4 * L + 32)
    _close("state", s, sr, 4 * L + 16)
    names = ("u", "B", "C", "D", "z", "initial_state")
    got = torch.autograd.grad((y, s), [gpu[k] for k in (*names, "A")], (dy.to(DEV), ds.to(DEV)))
    want = _reference_grads((yr, sr), [ref[k] for k in names], (dy.double().nan_to_num(0.0), ds.double()))
    for k, a, b in zip(names, got, want):
        _close("d" + k, a, b, 8 * L + 64 + (2 * L if k == "D" else 32 if k in "BC" else 0))
    assert torch.isfinite(got[-1]).all() and not got[-1][:, 7].any()


# ---- sizes that one launch does not hold ----------------------------------------------------------------------------------

def _conv_reference(x, weight, bias, first=None, lengths=None):
    """(y, final state) of all tokens at once, with SiLU."""
    B, L, D = x.shape
    W = weight.shape[1]
    live = None if lengths is None else (torch.arange(L, device=x.device) < lengths[:, None])[..., None]
    x = x if live is None else torch.where(live, x, 0.0)
    rows = torch.cat([x.new_zeros(B, W - 1, D) if first is None else first, x], 1)
    y = F.silu(bias + sum(weight[:, j] * rows[:, j:j + L] for j in range(W)))
    end = torch.full((B,), L, device=x.device) if lengths is None else lengths.long()
    at = end[:, None] + torch.arange(W - 1, device=x.device)
    return y if live is None else torch.where(live, y, 0.0), rows[torch.arange(B, device=x.device)[:, None], at]


def _check_conv_at_once(ops, B, L, D, W, dtype, ragged):
    g = torch.Generator(device=DEV).manual_seed(B + L + D + W)

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device=DEV).to(dtype)

    lengths = torch.randint(0, L + 1, (B,), generator=g, device=DEV) if ragged else None
    t = dict(x=randn(B, L, D, dtype=dtype), weight=randn(D, W) * 0.5, bias=randn(D), first=randn(B, W - 1, D, dtype=dtype))
    dy, ds = randn(B, L, D, dtype=dtype), randn(B, W - 1, D, dtype=dtype)
    ref = {k: v.double().requires_grad_(True) for k, v in t.items()}
    yr, sr = _conv_reference(**ref, lengths=lengths)
    want = torch.autograd.grad((yr, sr), list(ref.values()), (dy.double(), ds.double()))
    if ragged:
        behind = torch.arange(L, device=DEV) >= lengths[:, None]
        t["x"][behind], dy[behind] = NAN, NAN
    gpu = {k: v.requires_grad_(True) for k, v in t.items()}
    y, s = ops.causal_conv(gpu["x"], gpu["weight"], gpu["bias"], initial_state=gpu["first"], lengths=lengths, return_final_state=True)
    _close("y", y, yr, W + 8)
    assert torch.equal(s.double(), sr)
    for k, a, b in zip(gpu, torch.autograd.grad((y, s), list(gpu.values()), (dy, ds)), want):
        _close("d" + k, a, b, (B * L if k in ("weight", "bias") else W) + 16)


@pytest.mark.parametrize("dtype,D", [(torch.float32, 12), (torch.bfloat16, 8), (torch.float16, 5)])
def test_conv_of_more_sequences_than_a_grid_has_rows(ops, dtype, D):
    B = 2 * 65535 + 3
    _check_conv_at_once(ops, B, 2, D, 3, dtype, True)
    g = torch.Generator(device=DEV).manual_seed(0)
    x, state = (torch.randn(*s, generator=g, device=DEV).to(dtype) for s in ((B, D), (B, 3, D)))
    w = torch.randn(D, 4, generator=g, device=DEV)
    want = torch.cat([state, x[:, None]], 1)
    y = ops.causal_conv_step(x, state, w)
    assert torch.equal(state, want[:, 1:])
    pre = (want.double() * w.double().t()).sum(1)
    _close("y", y, F.silu(pre), 4 + 8)


def test_conv_of_one_sequence_of_millions_of_tokens(ops):
    """More strips than a grid has rows, forward and backward: each output and each gradient of an input is formed from the same few tokens as in
    pieces."""
    L, D = 68_000_000, 4
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn(1, L, D, generator=g, device=DEV, dtype=torch.bfloat16).requires_grad_(True)
    dy = torch.randn(1, L, D, generator=g, device=DEV, dtype=torch.bfloat16)
    w = torch.randn(D, 4, generator=g, device=DEV)
    whole = ops.causal_conv(x, w)
    dx, = torch.autograd.grad(whole, x, dy)
    whole = whole.detach()
    cuts = (0, 16_000_000, 32_000_000, 48_000_000, 64_000_000, L)
    for a, b in zip(cuts, cuts[1:]):
        lead = min(a, 3)                                   # the tokens before a piece, with it, in place of a state
        piece = x.detach()[:, a - lead:b].requires_grad_(True)
        y = ops.causal_conv(piece, w)
        assert torch.equal(y[:, lead:], whole[:, a:b])
        gp, = torch.autograd.grad(y, piece, dy[:, a - lead:b])
        assert torch.equal(gp[:, lead:b - a + lead - 3], dx[:, a:b - 3])


@pytest.mark.parametrize("name", ["conv", "scan"])
def test_lengths_beyond_32_bits_are_clamped(ops, name):
    t, *_ = _scan_case(4, 10, 16, 8, 1, torch.float32)
    d = {k: v.to(DEV) for k, v in t.items()}
    w = _randn(_gen(1), 16, 4).to(DEV)

    def call(lengths):
        if name == "conv":
            return ops.causal_conv(d["u"], w, lengths=lengths, return_final_state=True)
        return ops.selective_scan(**d, lengths=lengths, return_final_state=True)

    got = call(torch.tensor([2 ** 32 + 3, -2 ** 32 + 5, 2 ** 31, -1], device=DEV))
    want = call(torch.tensor([10, 0, 10, 0], device=DEV, dtype=torch.int32))
    for a, b in zip(got, want):
        assert torch.equal(a, b)
