"""A Mamba block over INT2 projections: the four projections of the reference's block (core/mamba/mamba2.py:136,149-171) as `BitLinearInt2`
layers, and between them the convolution, the scan and the block norms of `ssm_ops`.

A stack of blocks hands on the residual stream and its norm: a block takes (h, x), x being the normed h, and returns the pair for the
next block, so that the norm behind a block, its gate and scale, the addition and the norm in front of the next one are one pass.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional, Tuple

import torch
import torch.nn as nn

from . import ssm_ops
from .bitnet_int2_optimized import BitLinearInt2
from .int2_tc_ops import NORM_EPS


@dataclass
class MambaState:
    """What generation keeps of a batch of sequences: the last inputs of the convolution, and the scan's states."""
    conv: torch.Tensor         # [batch, d_conv - 1, d_inner]
    ssm: torch.Tensor          # [batch, d_inner, d_state] float32


class MambaBlockInt2(nn.Module):
    """(h, x) -> (h + scale * sigmoid(gate) * norm(mixer(x)), norm of that), x the normed residual stream h.

    mixer: in_proj to 2 d_inner channels; the first half through the causal convolution and SiLU; x_proj to the step sizes' rank and B, C; dt_proj;
    the selective scan, gated by the second half; out_proj.  `gated`: a further projection of x gives the gate of the block's output.
    The projections' pre-linear norms, quantisation and weight update are those of `BitLinearInt2` (`layer_kwargs` go there); all other
    parameters are float32 and get ordinary gradients."""

    def __init__(self, d_model: int, d_inner: Optional[int] = None, d_state: int = 16, d_conv: int = 4, dt_rank: int = 16, gated: bool = False,
                 eps: float = NORM_EPS, **layer_kwargs):
        super().__init__()
        self.d_model, self.d_inner, self.d_state, self.d_conv, self.dt_rank, self.eps = d_model, d_inner or 2 * d_model, d_state, d_conv, dt_rank, eps
        inner = self.d_inner
        self.in_proj = BitLinearInt2(d_model, 2 * inner, **layer_kwargs)
        self.x_proj = BitLinearInt2(inner, dt_rank + 2 * d_state, **layer_kwargs)
        self.dt_proj = BitLinearInt2(dt_rank, inner, **layer_kwargs)
        self.out_proj = BitLinearInt2(inner, d_model, **layer_kwargs)
        self.gate_proj = BitLinearInt2(d_model, d_model, **layer_kwargs) if gated else None
        self.conv_weight = nn.Parameter(torch.empty(inner, d_conv).uniform_(-1, 1) / math.sqrt(d_conv))
        self.conv_bias = nn.Parameter(torch.zeros(inner))
        # step sizes from 0.001 to 0.1 and decay rates 1 .. d_state to start with
        step = torch.exp(torch.rand(inner) * math.log(100.0) + math.log(1e-3))
        self.dt_bias = nn.Parameter(step + torch.log(-torch.expm1(-step)))
        self.A_log = nn.Parameter(torch.log(torch.arange(1, d_state + 1, dtype=torch.float32)).repeat(inner, 1))
        self.D = nn.Parameter(torch.ones(inner))
        self.post_norm = nn.Parameter(torch.ones(d_model))
        self.next_norm = nn.Parameter(torch.ones(d_model))
        self.scale = nn.Parameter(torch.ones(d_model))

    def init_weights(self, std: float = 0.02):
        """Ternarised N(0, std) weights in every projection (they are empty after construction)."""
        for layer in self.children():
            if isinstance(layer, BitLinearInt2):
                device = layer.int2_layer.W_packed.device
                layer.int2_layer.init_from_float(torch.randn(layer.out_features, layer.in_features, device=device) * std)
        return self

    def new_state(self, batch: int, dtype: torch.dtype = torch.bfloat16) -> MambaState:
        """The state before a first token."""
        device = self.D.device
        return MambaState(torch.zeros(batch, self.d_conv - 1, self.d_inner, dtype=dtype, device=device),
                          torch.zeros(batch, self.d_inner, self.d_state, device=device))

    @staticmethod
    def _before(state: Optional[MambaState]) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
        """The state's tensors for a forward pass that then overwrites them.  Where gradients are recorded the operators keep what they start from for
        the backward pass, so they get copies."""
        if state is None:
            return None, None
        if not torch.is_grad_enabled():
            return state.conv, state.ssm
        return state.conv.detach().clone(), state.ssm.detach().clone()

    def _selection(self, u: torch.Tensor):
        """(step sizes, B, C) of the convolved channels; B and C are windows of one projection's output, read in place."""
        p = self.x_proj(u)
        dt, B, C = p.split([self.dt_rank, self.d_state, self.d_state], -1)
        return self.dt_proj(dt.contiguous()), B, C

    def _join(self, h: torch.Tensor, y: torch.Tensor, x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        gate = self.gate_proj(x) if self.gate_proj is not None else None
        return ssm_ops.block_norm(h, self.out_proj(y), self.post_norm, self.next_norm, gate=gate, scale=self.scale, eps=self.eps)

    def forward(self, h: torch.Tensor, x: torch.Tensor, state: Optional[MambaState] = None,
                lengths: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """h, x [batch, length, d_model].  `state` (no gradient goes into it): the text goes on from it, and its tensors become the state after
        each sequence's last token, in place; a backward pass after that is that of the piece that was given.  `lengths` as in ssm_ops: h and x
        may hold anything behind a sequence's end, both outputs and all gradients are zeros there."""
        # the projections and norms run over padding too: zeros on the way in and, for the gradients, on the way out
        live = None if lengths is None else (torch.arange(x.shape[1], device=x.device) < lengths[:, None])[..., None]
        if live is not None:
            h, x = torch.where(live, h, 0.0), torch.where(live, x, 0.0)
        conv_before, ssm_before = self._before(state)
        xz = self.in_proj(x)
        u, z = xz[..., :self.d_inner], xz[..., self.d_inner:]
        u = ssm_ops.causal_conv(u, self.conv_weight, self.conv_bias, initial_state=conv_before, lengths=lengths,
                                return_final_state=state is not None)
        if state is not None:
            u, last = u
            state.conv.copy_(last.detach())
        dt, B, C = self._selection(u)
        y = ssm_ops.selective_scan(u, dt, -torch.exp(self.A_log), B, C, D=self.D, z=z, dt_bias=self.dt_bias,
                                   initial_state=ssm_before, lengths=lengths, return_final_state=state is not None)
        if state is not None:
            y, last = y
            state.ssm.copy_(last.detach())
        out, normed = self._join(h, y, x)
        return (out, normed) if live is None else (torch.where(live, out, 0.0), torch.where(live, normed, 0.0))

    @torch.no_grad()
    def step(self, h: torch.Tensor, x: torch.Tensor, state: MambaState) -> Tuple[torch.Tensor, torch.Tensor]:
        """One token for every sequence: h, x [batch, d_model]; the state is updated in place."""
        xz = self.in_proj(x)
        u = ssm_ops.causal_conv_step(xz[:, :self.d_inner], state.conv, self.conv_weight, self.conv_bias)
        dt, B, C = self._selection(u)
        y = ssm_ops.selective_scan_step(u, dt, -torch.exp(self.A_log), B, C, state.ssm, D=self.D, z=xz[:, self.d_inner:], dt_bias=self.dt_bias)
        return self._join(h, y, x)
