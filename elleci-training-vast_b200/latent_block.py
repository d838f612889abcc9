"""Latent attention over INT2 projections: the projections of the reference's attention block (model/common/mla.py:38-45) as `BitLinearInt2` layers, and
between them the operators of `attention_ops`.

What a served text keeps of a token is the operand of the up projection, an int8 row and its scale, and the rotated part of its key; prompts read it back
and expand it, single tokens attend to it as it is.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch
import torch.nn as nn

from . import attention_ops
from .attention_ops import LatentCache
from .bitnet_int2_optimized import BitLinearInt2
from .int2_tc_ops import NORM_EPS, _require, matmul_rows


@dataclass
class LatentState:
    """What generation keeps of a batch of sequences.  `most`: no sequence has more tokens (the host's count, which needs no look at the device)."""
    cache: LatentCache
    block_table: torch.Tensor      # [batch, pages of a sequence] int32
    lengths: torch.Tensor          # [batch] int32
    most: int = 0

    @property
    def room(self) -> int:
        return self.block_table.shape[1] * self.cache.latents.shape[1]


class LatentAttentionInt2(nn.Module):
    """x -> w_out(attention(w_q(x), w_kv_up(w_kv_down(x)))), causal.

    w_q gives every head's query, head_dim channels, and behind all of them every head's rot_dim channels that are rotated by position; w_kv_down the
    latent vector (kv_rank) and one rotated key part for all heads (rot_dim); w_kv_up every head's key (head_dim), then every head's value (value_dim).  The
    projections' pre-linear norms, quantisation and weight update are those of `BitLinearInt2` (`layer_kwargs` go there; per-token mode)."""

    def __init__(self, d_model: int, heads: int, head_dim: Optional[int] = None, kv_rank: Optional[int] = None, rot_dim: int = 0, value_dim: Optional[int] = None,
                 max_positions: int = 32768, rope_base: float = 10000.0, **layer_kwargs):
        super().__init__()
        self.heads, self.head_dim = heads, head_dim or d_model // heads
        self.kv_rank, self.rot_dim, self.value_dim = kv_rank or min(256, d_model // 4), rot_dim, value_dim or head_dim or d_model // heads
        self.max_positions = max_positions
        _require(layer_kwargs.get("quant_mode", "per_token") == "per_token", "latent attention needs quant_mode='per_token'")
        _require(not layer_kwargs.get("bias", False), "the projections of latent attention have no bias")
        self.w_q = BitLinearInt2(d_model, heads * (self.head_dim + rot_dim), **layer_kwargs)
        self.w_kv_down = BitLinearInt2(d_model, self.kv_rank + rot_dim, **layer_kwargs)
        self.w_kv_up = BitLinearInt2(self.kv_rank, heads * (self.head_dim + self.value_dim), **layer_kwargs)
        self.w_out = BitLinearInt2(heads * self.value_dim, d_model, **layer_kwargs)
        self.register_buffer("table", attention_ops.rotary_table(max_positions, rot_dim, rope_base) if rot_dim else None, persistent=False)

    def init_weights(self, std: float = 0.02):
        """Ternarised N(0, std) weights in every projection (they are empty after construction)."""
        for layer in self.children():
            if isinstance(layer, BitLinearInt2):
                weight = torch.randn(layer.out_features, layer.in_features, device=layer.int2_layer.W_packed.device) * std
                layer.int2_layer.init_from_float(weight, scale=max(float(weight.abs().mean()), 1e-5))
        return self

    def new_state(self, batch: int, tokens: int, page_size: int = 64, dtype: torch.dtype = torch.bfloat16) -> LatentState:
        """An empty state with room for `tokens` tokens of every sequence, on pages of its own.  (A program with a pool of pages makes a LatentState of it.)"""
        per = -(-tokens // page_size)
        device = self.w_q.int2_layer.W_packed.device
        return LatentState(LatentCache.new(batch * per, page_size, self.kv_rank, self.rot_dim, dtype, device),
                           torch.arange(batch * per, device=device, dtype=torch.int32).view(batch, per), torch.zeros(batch, device=device, dtype=torch.int32))

    def _queries(self, x: torch.Tensor):
        q = self.w_q(x)
        content = self.heads * self.head_dim
        return q[..., :content].unflatten(-1, (self.heads, self.head_dim)), q[..., content:].unflatten(-1, (self.heads, self.rot_dim)) if self.rot_dim else None

    def _latent(self, x: torch.Tensor):
        c = self.w_kv_down(x)
        return c[..., :self.kv_rank], c[..., self.kv_rank:] if self.rot_dim else None

    def _up(self):
        """(packed weights, their scale) of the up projection."""
        inner = self.w_kv_up.int2_layer
        if inner._gamma_cached is None:
            inner._gamma_cached = inner.gamma.detach().item()
        return inner.W_packed, inner._gamma_cached

    def _write(self, state: LatentState, latent: torch.Tensor, k_rot: Optional[torch.Tensor], lengths: Optional[torch.Tensor]) -> torch.Tensor:
        """Into the cache; the lengths from before."""
        most = state.most + latent.shape[1]
        _require(most <= min(state.room, self.max_positions if self.rot_dim else state.room), "the state has no room for that many tokens")
        before = state.lengths.clone()
        norm = self.w_kv_up.extra_rmsnorm if self.w_kv_up.use_extra_rmsnorm else None
        attention_ops.latent_cache_write(state.cache, state.block_table, latent, None if norm is None else norm.weight.detach(), k_rot, self.table, before, lengths,
                                         NORM_EPS if norm is None else norm.eps)
        state.most = most
        state.lengths.add_(latent.shape[1] if lengths is None else lengths.clamp(0, latent.shape[1]).to(torch.int32))
        return before

    def forward(self, x: torch.Tensor, state: Optional[LatentState] = None, lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
        """x [batch, length, d_model].  With a `state` the text goes on from it and its tensors are updated in place; such a call records no gradient.
        `lengths` (int32 or int64 [batch]): a sequence's tokens; x may hold anything behind them, outputs and gradients are zeros there."""
        if state is not None:
            with torch.no_grad():
                return self._forward(x, state, lengths)
        return self._forward(x, None, lengths)

    def _forward(self, x: torch.Tensor, state: Optional[LatentState], lengths: Optional[torch.Tensor]) -> torch.Tensor:
        # the projections run over padding too: zeros on the way in and, for the gradients, on the way out
        live = None if lengths is None else (torch.arange(x.shape[1], device=x.device) < lengths[:, None])[..., None]
        if live is not None:
            x = torch.where(live, x, 0.0)
        q, q_rot = self._queries(x)
        latent, k_rot = self._latent(x)
        if state is None:
            _require(self.rot_dim == 0 or x.shape[1] <= self.max_positions, "a text beyond max_positions")
            if self.rot_dim:
                q_rot, k_rot = attention_ops.rotary(q_rot, self.table), attention_ops.rotary(k_rot, self.table)
            out = attention_ops.latent_attention(q, self.w_kv_up(latent), q_rot, k_rot, lengths=lengths)
        else:
            starts = self._write(state, latent, k_rot, lengths)
            if self.rot_dim:
                q_rot = attention_ops.rotary(q_rot, self.table, starts)
            rows, absmax, k_rot = attention_ops.latent_cache_read(state.cache, state.block_table, state.most, lengths=state.lengths)
            W, gamma = self._up()
            kv = matmul_rows(rows, W, absmax, gamma, x.dtype).view(x.shape[0], state.most, -1)
            every = torch.full_like(state.lengths, x.shape[1]) if lengths is None else lengths
            out = attention_ops.latent_attention(q, kv, q_rot, k_rot, lengths=every, key_lengths=state.lengths)
        y = self.w_out(out.flatten(2))
        return y if live is None else torch.where(live, y, 0.0)

    @torch.no_grad()
    def step(self, x: torch.Tensor, state: LatentState) -> torch.Tensor:
        """One token for every sequence: x [batch, d_model]; the state is updated in place."""
        q, q_rot = self._queries(x)
        latent, k_rot = self._latent(x)
        self._write(state, latent[:, None], None if k_rot is None else k_rot[:, None], None)
        W, gamma = self._up()
        out = attention_ops.latent_attention_step(q, W, gamma, state.cache, state.block_table, state.lengths, self.value_dim, q_rot=q_rot, table=self.table)
        return self.w_out(out.flatten(1))
