"""The operators of latent attention, on torch tensors: attention whose keys and values come from one latent vector a token, which an INT2 layer (the
up projection) expands.

    training, prompts    up projection -> latent_attention (the expanded form: every head's keys and values are there)
    cache                latent_cache_write keeps a token as the up projection's quantised operand: an int8 row and its largest magnitude
                         latent_cache_read -> matmul_rows -> latent_attention: a prompt that goes on from cached tokens
    single tokens        latent_attention_step (the absorbed form: the query goes into the latent space, keys and values are never formed)

Part of a key may be rotated by its position instead (`rotary`); that part is one for all heads and is cached beside the row.  The reference's block has
these as tensor operations and torch's attention (model/common/mla.py); here each is one call of the C-ABI library (include/elleci_int2.h) per direction,
queued on the current CUDA stream.  Activations are float16, bfloat16 or float32, all of one dtype; tensors whose last dimension is contiguous (slices of a
projection's output) are read in place.  Sums, softmax statistics and states of a call are float32, and every output is rounded once; on the tensor cores
(16-bit types) probabilities and their gradients are rounded to the dtype as factors of a product.  Gradients do not depend on the order in which blocks run.
Derivatives are reverse-mode ones of the first order.  `RuntimeError` on bad arguments.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple, Union

import torch

from ._lib import host_ops
from .int2_tc_ops import ACT_EPS, NORM_EPS, _require


def rotary_table(positions: int, dim: int, base: float = 10000.0, device: Optional[torch.device] = None) -> torch.Tensor:
    """[positions, dim] float32: row p holds the cosines, then the sines, of p * base^(-2 i / dim), i < dim / 2 (angles in 64 bits: a far position's angle is
    large against its rounding).  Any table of this layout will do."""
    _require(dim % 2 == 0, "the rotated dimension must be even")
    rate = float(base) ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=device) / max(dim, 1))
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * rate
    return torch.cat([angle.cos(), angle.sin()], -1).float()


def rotary(x: torch.Tensor, table: torch.Tensor, positions: Optional[torch.Tensor] = None, neighbours: bool = False) -> torch.Tensor:
    """x [batch, length, heads, dim] or [batch, length, dim] with its pairs (x[i], x[i + dim/2]) (`neighbours`: (x[2i], x[2i+1])) turned by the angles of the
    token's position.  `table` as from `rotary_table`.  `positions` (int32 or int64): [batch] the position of each sequence's first token, or [batch,
    length], or None (token t is at t); positions outside the table are clamped to it.  Differentiable in x."""
    _require(not (isinstance(table, torch.Tensor) and table.requires_grad), "rotary has no gradient of its table")
    return host_ops().rotary(x, table, positions, int(neighbours), 0)


def latent_attention(q: torch.Tensor, kv: torch.Tensor, q_rot: Optional[torch.Tensor] = None, k_rot: Optional[torch.Tensor] = None, causal: bool = True,
                     scale: Optional[float] = None, lengths: Optional[torch.Tensor] = None, key_lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The expanded form, [batch, length, heads, value_dim]: out[i,h] = sum_j softmax_j(scale * (q[i,h] . k[j,h] + q_rot[i,h] . k_rot[j])) v[j,h].

    q [batch, length, heads, key_dim]; kv [batch, keys, heads * (key_dim + value_dim)], the up projection's output: all heads' keys, then all heads' values;
    q_rot [batch, length, heads, rot_dim] and k_rot [batch, keys, rot_dim], both or neither, are rotated already.  key_dim + rot_dim and value_dim up to 256.
    `scale` None: 1 / sqrt(key_dim + rot_dim).  `lengths`, `key_lengths` (int32 or int64 [batch], clamped; `key_lengths` None: `lengths` where there are as many
    keys as queries, else all keys): a sequence's queries and keys, padding behind them.  A sequence's queries are its last tokens: with `causal`, query i of m
    sees the keys up to i + n - m of n.  A query that sees no key has the output 0.  Padding is not read (it may hold anything, NaN included), its
    outputs and gradients are zeros; an infinity or NaN in a token's own key or value reaches other queries of its tile too.  Differentiable in q, kv, q_rot, k_rot."""
    return host_ops().latent_attention(q, kv, q_rot, k_rot, int(causal), scale, lengths, key_lengths)


class LatentCache(NamedTuple):
    """A pool of pages: `latents` int8 [pages, page_size, rank], `absmax` float32 [pages, page_size] (a token's value is row * absmax / 127) and `keys` [pages,
    page_size, rot_dim], the rotated key parts, or None.  A block table (int32 [batch, n]) says which pages hold a sequence: position p is token p % page_size
    of page block_table[b, p // page_size].  Entries outside the pool (-1) are not followed.  rank: a multiple of 16 up to 512; rot_dim up to 64."""
    latents: torch.Tensor
    absmax: torch.Tensor
    keys: Optional[torch.Tensor] = None

    @staticmethod
    def new(pages: int, page_size: int, rank: int, rot_dim: int = 0, dtype: torch.dtype = torch.bfloat16, device: Optional[torch.device] = None) -> "LatentCache":
        """An empty pool on `device` (None: the current CUDA device); dtype is the activations'."""
        device = torch.device("cuda") if device is None else device
        return LatentCache(torch.zeros(pages, page_size, rank, dtype=torch.int8, device=device), torch.zeros(pages, page_size, device=device),
                           torch.zeros(pages, page_size, rot_dim, dtype=dtype, device=device) if rot_dim else None)


def latent_cache_write(cache: LatentCache, block_table: torch.Tensor, latent: torch.Tensor, norm_weight: Optional[torch.Tensor] = None,
                       k_rot: Optional[torch.Tensor] = None, table: Optional[torch.Tensor] = None, starts: Optional[torch.Tensor] = None,
                       lengths: Optional[torch.Tensor] = None, eps: float = NORM_EPS, neighbours: bool = False) -> None:
    """New tokens, latent [batch, length, rank] (the down projection's output), into positions starts[b] + t, t < lengths[b], of the cache, as the up projection's
    operand: through its RMSNorm (norm_weight [rank] float32; None: it has none) and its quantiser, the same bits.  k_rot [batch, length, rot_dim] is
    rotated by the row of `table` for its position (None: it is rotated already).  `starts`, `lengths` int32 or int64 [batch] (None: 0, all).  Two tokens
    of a call must not share a place (two sequences on one page); positions that have no page are dropped.  Not differentiable."""
    host_ops().latent_cache_write(cache.latents, cache.absmax, cache.keys, block_table, latent, norm_weight, k_rot, table, starts, lengths, eps, ACT_EPS,
                                  int(neighbours))


def latent_cache_read(cache: LatentCache, block_table: torch.Tensor, length: int, starts: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                      dtype: Optional[torch.dtype] = None) -> Union[Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]], Tuple[torch.Tensor, Optional[torch.Tensor]]]:
    """Positions starts[b] + t, t < lengths[b] <= length (None: 0, all), of every sequence, zeros behind them.  (rows int8 [batch * length, rank], absmax [batch * length],
    keys [batch, length, rot_dim] or None): what int2_tc_ops.matmul_rows takes; with `dtype` (values [batch, length, rank] of that type, keys)."""
    return host_ops().latent_cache_read(cache.latents, cache.absmax, cache.keys, block_table, length, starts, lengths, dtype)


def latent_attention_step(q: torch.Tensor, W_packed: torch.Tensor, gamma: float, cache: LatentCache, block_table: torch.Tensor, lengths: torch.Tensor, value_dim: int,
                          q_rot: Optional[torch.Tensor] = None, table: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                          neighbours: bool = False) -> torch.Tensor:
    """The absorbed form, [batch, heads, value_dim]: one token of every sequence, q [batch, heads, key_dim], against its lengths[b] cached tokens (int32 or int64,
    clamped), of which it is the last.  W_packed [heads * (key_dim + value_dim), rank / 4] and gamma are the up projection's weights: the result is that of
    expanding the cached rows and attending to them, up to roundings, but keys and values are not formed.  q_rot [batch, heads, rot_dim] is rotated by the
    row of `table` for position lengths[b] - 1 (None: it is rotated already).  A sequence of length 0 gives 0.  Not differentiable."""
    return host_ops().latent_attention_step(cache.latents, cache.absmax, cache.keys, block_table, q, W_packed, gamma, lengths, value_dim, q_rot, table, scale,
                                            int(neighbours))
