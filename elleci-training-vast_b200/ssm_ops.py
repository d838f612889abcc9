"""The operators between the INT2 projections of a Mamba block, on torch tensors: the short causal convolution, the selective state
space scan (each for training and prompts, and a step form for single tokens) and the norms before and after the block with its gate
and residual scale.

    in_proj -> causal_conv -> x_proj, dt_proj -> selective_scan (gated by z) -> out_proj -> block_norm

The reference's block runs them as tensor operations (core/mamba/mamba2.py:136,149-171); here each is one call of the C-ABI library
(include/elleci_int2.h) per direction, queued on the current CUDA stream.  Activations are float16, bfloat16 or float32, channel-last,
all of one dtype; tensors whose channels are contiguous (slices of a wider projection) are read in place.  Parameters are float32, sums
and states are held in float32, and every output is rounded once.  Gradients do not depend on the order in which blocks run: the same
call gives the same bits.  Derivatives are reverse-mode ones of the first order; a tensor with a forward-mode tangent is refused.
`RuntimeError` on bad arguments.

`lengths` (int32 or int64 [batch], clamped to 0 .. length): sequence b has lengths[b] tokens and padding behind them.  Padding is not read (it may hold
anything, NaN included), its outputs and gradients are zeros and it leaves the state as it is.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from ._lib import host_ops
from .int2_tc_ops import NORM_EPS, _require

_ACTIVATIONS = {"silu": 1, "swish": 1, None: 0}


def _wants_grad(*tensors: Optional[torch.Tensor]) -> bool:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _bits(wanted) -> int:
    return sum(1 << i for i, w in enumerate(wanted) if w)


def _silu(activation: Optional[str]) -> int:
    _require(activation in _ACTIVATIONS, f"activation must be 'silu', 'swish' or None, not {activation!r}")
    return _ACTIVATIONS[activation]


class _CausalConv(Function):
    @staticmethod
    def forward(ctx, x, weight, bias, silu, initial_state, lengths, want_state):
        y, state = host_ops().causal_conv(x, weight, bias, silu, initial_state, lengths, want_state)
        ctx.save_for_backward(x, weight, bias, initial_state, lengths)
        ctx.silu = silu
        ctx.set_materialize_grads(False)
        return y, state

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, d_state):
        x, weight, bias, initial_state, lengths = ctx.saved_tensors
        need = ctx.needs_input_grad
        if dy is None and d_state is None:
            return (None,) * 7
        dx, dw, db, d_first = host_ops().causal_conv_backward(x, weight, bias, ctx.silu, initial_state, lengths, dy, d_state,
                                                              _bits((need[0], need[1], need[2], need[4])))
        return dx, dw, db, None, d_first, None, None


def causal_conv(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: Optional[str] = "silu",
                initial_state: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                return_final_state: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Depthwise causal convolution of x [batch, length, channels] over the last `width` tokens of each channel, with bias [channels] and
    SiLU: y[t] = act(bias + sum_j weight[:, j] * x[t - (width-1) + j]).  weight [channels, width], width 2 to 4.  `initial_state`
    [batch, width-1, channels] in x's dtype holds the inputs before the first token (zeros if None); with `return_final_state` the last
    width-1 inputs of each sequence are returned too: what `causal_conv_step`, or the next piece of the text, goes on from.
    Differentiable in x, weight, bias and initial_state."""
    silu = _silu(activation)
    if _wants_grad(x, weight, bias, initial_state):
        y, state = _CausalConv.apply(x, weight, bias, silu, initial_state, lengths, int(return_final_state))
    else:
        y, state = host_ops().causal_conv(x, weight, bias, silu, initial_state, lengths, int(return_final_state))
    return (y, state) if return_final_state else y


def causal_conv_step(x: torch.Tensor, state: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                     activation: Optional[str] = "silu", state_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token x [batch, channels] of `causal_conv`.  `state` [batch, width-1, channels] becomes the state after the token in place, or,
    with `state_out` (a tensor like it; for callers that may take the token back), is kept and the new state goes there.  Not
    differentiable."""
    return host_ops().causal_conv_step(x, state, weight, bias, _silu(activation), state_out)


class _SelectiveScan(Function):
    @staticmethod
    def forward(ctx, u, dt, A, B, C, D, z, dt_bias, softplus, initial_state, lengths, want_state):
        y, state, kept = host_ops().selective_scan(u, dt, A, B, C, D, z, dt_bias, softplus, initial_state, lengths, want_state, 1)
        ctx.save_for_backward(u, dt, A, B, C, D, z, dt_bias, initial_state, lengths, kept)
        ctx.softplus = softplus
        ctx.set_materialize_grads(False)
        return y, state

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, d_state):
        u, dt, A, B, C, D, z, dt_bias, initial_state, lengths, kept = ctx.saved_tensors
        need = ctx.needs_input_grad
        if dy is None and d_state is None:
            return (None,) * 12
        du, ddt, dA, dB, dC, dD, dz, ddt_bias, d_first = host_ops().selective_scan_backward(
            u, dt, A, B, C, D, z, dt_bias, ctx.softplus, initial_state, lengths, kept, dy, d_state, _bits(need[:8] + (need[9],)))
        return du, ddt, dA, dB, dC, dD, dz, ddt_bias, None, d_first, None, None


def selective_scan(u: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, D: Optional[torch.Tensor] = None,
                   z: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None, dt_softplus: bool = True,
                   initial_state: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                   return_final_state: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Selective state space scan of u [batch, length, channels].  With delta = softplus(dt + dt_bias) (dt_softplus False: dt + dt_bias):

        h[t] = exp(delta[t] A) h[t-1] + delta[t] u[t] B[t],   y[t] = (C[t] . h[t] + D u[t]) * silu(z[t])

    dt and z are like u; A is [channels, states] (1 to 64 states; negative for a state that decays), D and dt_bias [channels]; B and C are
    [batch, length, states], or [batch, length, groups, states] where channels / groups consecutive channels share a group.  `initial_state`
    [batch, channels, states] float32 (zeros if None); with `return_final_state` the state after each sequence's last token is returned too.
    Differentiable in every tensor; the forward pass then keeps the state of every eighth token."""
    if _wants_grad(u, dt, A, B, C, D, z, dt_bias, initial_state):
        y, state = _SelectiveScan.apply(u, dt, A, B, C, D, z, dt_bias, int(dt_softplus), initial_state, lengths, int(return_final_state))
    else:
        y, state, _ = host_ops().selective_scan(u, dt, A, B, C, D, z, dt_bias, int(dt_softplus), initial_state, lengths,
                                                int(return_final_state), 0)
    return (y, state) if return_final_state else y


def selective_scan_step(u: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, state: torch.Tensor,
                        D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None,
                        dt_softplus: bool = True, state_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token of `selective_scan`: u, dt, z [batch, channels], B and C [batch, states] or [batch, groups, states].  `state`
    [batch, channels, states] float32 becomes the state after the token in place, or goes to `state_out` as in `causal_conv_step`.
    Not differentiable."""
    return host_ops().selective_scan_step(u, dt, A, B, C, D, z, dt_bias, int(dt_softplus), state, state_out)


class _BlockNorm(Function):
    @staticmethod
    def forward(ctx, h, y, post_weight, pre_weight, gate, scale, eps):
        h_out, normed, rstd = host_ops().block_norm(h, y, post_weight, pre_weight, gate, scale, eps, 1)
        ctx.save_for_backward(h, y, post_weight, pre_weight, gate, scale, rstd)
        ctx.eps = eps
        ctx.set_materialize_grads(False)
        return h_out, normed

    @staticmethod
    @once_differentiable
    def backward(ctx, dh_out, dnormed):
        h, y, post_weight, pre_weight, gate, scale, rstd = ctx.saved_tensors
        if dh_out is None and dnormed is None:
            return (None,) * 7
        need = ctx.needs_input_grad
        wanted = need[0] | need[1] << 1 | need[2] << 2 | need[3] << 3 | need[4] << 4 | need[5] << 5
        dh, dy, dw1, dw2, dgate, dscale = host_ops().block_norm_backward(h, y, post_weight, pre_weight, gate, scale, ctx.eps, rstd,
                                                                         dh_out, dnormed, wanted)
        return dh, dy, dw1, dw2, dgate, dscale, None


def block_norm(h: torch.Tensor, y: torch.Tensor, post_weight: torch.Tensor, pre_weight: torch.Tensor, gate: Optional[torch.Tensor] = None,
               scale: Optional[torch.Tensor] = None, eps: float = NORM_EPS) -> Tuple[torch.Tensor, torch.Tensor]:
    """Joins a block's output y to the residual stream h and norms the result for the next block:

        h_out  = h + scale * sigmoid(gate) * rmsnorm(y, post_weight)         (gate like y, scale [width]: 1 if None)
        normed = rmsnorm(h_out, pre_weight)                                  (of h_out before it is rounded to the dtype)

    Returns (h_out, normed).  h, y and gate have any leading dimensions and rows of up to 16384 columns.  Differentiable in every tensor."""
    if _wants_grad(h, y, post_weight, pre_weight, gate, scale):
        return _BlockNorm.apply(h, y, post_weight, pre_weight, gate, scale, float(eps))
    h_out, normed, _ = host_ops().block_norm(h, y, post_weight, pre_weight, gate, scale, float(eps), 0)
    return h_out, normed
