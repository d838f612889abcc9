"""The operators of latent attention by their definitions in float64, with bounds of the error that a float32 computation of them may have.

A bound follows the roundings through the formulas, element by element; `unit` is the relative rounding of a factor of a product (2^-8 for
bfloat16, 2^-11 for float16 with 2^-25 absolute, 2^-24 for float32) and e = 2^-24 that of a float32 operation:

  score   a sum of D products: e (D + 4) sum |q| |k| scale, the same relative error in the probability's exponential, whose own is 2^-22, and in its
          row's sum, n e more; together `rel` of a probability
  out     rel and unit of every p v, n e for the sum, the output's own rounding
  dp      e (V + 2) sum |dout| |v|; delta carries out's rounding
  ds      rel and unit of itself, and p times what dp and delta are off
  dq, dk  ds's error times |k| (|q|), n e for the sum, the own rounding"""
import math

import torch

E = 2.0 ** -24
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}


def rotate(x, table, positions, neighbours=False):
    """x [.., dim], positions: rows of the table, one for each leading index."""
    half = x.shape[-1] // 2
    cos, sin = table.double()[positions][..., :half], table.double()[positions][..., half:]
    a, b = (x[..., 0::2], x[..., 1::2]) if neighbours else (x[..., :half], x[..., half:])
    p, q = a * cos - b * sin, b * cos + a * sin
    return torch.stack([p, q], -1).flatten(-2) if neighbours else torch.cat([p, q], -1)


def _largest(x, least):
    """Along the last dimension, which may be empty."""
    return torch.cat([x, x.new_full((*x.shape[:-1], 1), least)], -1).amax(-1, keepdim=True)


def _probabilities(z, seen):
    z = z.masked_fill(~seen, -math.inf)
    top = _largest(z, -math.inf)
    p = torch.exp(z - torch.where(top > -math.inf, top, 0.0))
    return p / p.sum(-1, keepdim=True).clamp_min(1e-300)


def attention(q, kv, q_rot, k_rot, causal, scale, lengths, key_lengths, dtype, dout=None):
    """Tensors as latent_attention takes them, values of `dtype`, padding finite.  ({name: value}, {name: bound})."""
    B, T, H, D = q.shape
    S, V = kv.shape[1], kv.shape[2] // H - D
    R = 0 if q_rot is None else q_rot.shape[-1]
    unit, tiny = UNIT[dtype], TINY[dtype]
    scale = 1 / math.sqrt(D + R) if scale is None else scale
    q, kv, dout = q.double(), kv.double(), None if dout is None else dout.double()
    k, v = kv[..., :H * D].unflatten(-1, (H, D)), kv[..., H * D:].unflatten(-1, (H, V))
    if R:
        q, k = torch.cat([q, q_rot.double()], -1), torch.cat([k, k_rot.double()[:, :, None].expand(-1, -1, H, -1)], -1)
    q, k, v = (x.transpose(1, 2) for x in (q, k, v))                     # [B, H, tokens, channels]
    ln = torch.full((B,), T) if lengths is None else lengths.clamp(0, T)
    kn = (ln if S == T and lengths is not None else torch.full((B,), S)) if key_lengths is None else key_lengths.clamp(0, S)
    i, j = torch.arange(T)[:, None], torch.arange(S)
    seen = (i < ln[:, None, None]) & (j < kn[:, None, None])
    if causal:
        seen = seen & (j <= i + (kn - ln)[:, None, None])
    seen = seen[:, None]
    live, key_live = (torch.arange(T) < ln[:, None])[:, None, :, None], (torch.arange(S) < kn[:, None])[:, None, :, None]
    p = _probabilities(q @ k.transpose(-1, -2) * scale, seen)
    size = (q.abs() @ k.abs().transpose(-1, -2)) * abs(scale)
    size = _largest(torch.where(seen, size, 0.0), 0.0)
    rel = 4 * E * (D + R + 4) * size + 4 * 2.0 ** -22 + 4 * (S + 8) * E
    o = p @ v
    abs_out = p @ v.abs()
    out_bound = abs_out * (rel + unit + S * E) + tiny * v.abs().sum(-2, keepdim=True)
    value = {"out": o.transpose(1, 2)}
    bound = {"out": (out_bound + unit * o.abs() + tiny).transpose(1, 2)}
    if dout is None:
        return value, bound
    g = torch.where(live, dout.transpose(1, 2), 0.0)
    dp = g @ v.transpose(-1, -2)
    ds = p * (dp - (g * o).sum(-1, keepdim=True))
    off = E * (V + 2) * (g.abs() @ v.abs().transpose(-1, -2)) + (g.abs() * (out_bound + unit * o.abs() + tiny)).sum(-1, keepdim=True) \
        + E * (V + 2) * (g.abs() * o.abs()).sum(-1, keepdim=True)
    # the difference dp - delta is formed before it is multiplied: its rounding is that of both terms
    off = off + E * (dp.abs() + (g * o).sum(-1, keepdim=True).abs())
    ds_off = torch.where(seen, ds.abs() * (rel + unit + 4 * E) + p * off * (1 + rel) + tiny, 0.0)

    def product(a_off, a, b, terms, sc):
        """sc * a @ b with a off by a_off."""
        x = (a @ b) * sc
        return x, (a_off @ b.abs() + terms * E * (a.abs() @ b.abs())) * abs(sc) + unit * x.abs() + tiny

    dv, dv_off = product(torch.where(seen, p * (rel + unit) + tiny, 0.0).transpose(-1, -2), p.transpose(-1, -2), g, T + 4, 1.0)
    dq, dq_off = product(ds_off, ds, k, S + 4, scale)
    dk, dk_off = product(ds_off.transpose(-1, -2), ds.transpose(-1, -2), q, T + 4, scale)
    dv, dk, dq = torch.where(key_live, dv, 0.0), torch.where(key_live, dk, 0.0), torch.where(live, dq, 0.0)

    def join(k_part, v_part):
        return torch.cat([k_part[..., :D].transpose(1, 2).flatten(2), v_part.transpose(1, 2).flatten(2)], -1)

    value.update(dq=dq[..., :D].transpose(1, 2), dkv=join(dk, dv))
    bound.update(dq=dq_off[..., :D].transpose(1, 2), dkv=join(dk_off, dv_off))
    if R:
        value.update(dq_rot=dq[..., D:].transpose(1, 2), dk_rot=dk[..., D:].sum(1))
        bound.update(dq_rot=dq_off[..., D:].transpose(1, 2), dk_rot=dk_off[..., D:].sum(1) + H * E * dk[..., D:].abs().sum(1) + unit * dk[..., D:].sum(1).abs() + tiny)
    return value, bound


def cached(latents, absmax, keys, block_table, n):
    """(values [n, rank], keys [n, rot] or None, truth values of what has a page, rows of the pool) of positions 0 .. n - 1 of one sequence; block_table its row."""
    pages, page, rank = latents.shape
    at = torch.arange(n)
    entry = block_table.long()[at // page]
    here = (entry >= 0) & (entry < pages)
    row = torch.where(here, entry, 0) * page + at % page
    value = latents.reshape(-1, rank)[row].double() * (absmax.reshape(-1)[row].double() / 127)[:, None]
    k = None if keys is None else keys.reshape(-1, keys.shape[-1])[row].double()
    return value, k, here, row


def step(q, W, gamma, latents, absmax, keys, block_table, lengths, value_dim, q_rot, table, scale, dtype, neighbours=False):
    """(out, bound): the expanded form.  W [heads * (key_dim + value_dim), rank] holds -1, 0, 1."""
    B, H, D = q.shape
    R = 0 if keys is None else keys.shape[-1]
    unit, tiny, rank = UNIT[dtype], TINY[dtype], latents.shape[-1]
    scale = 1 / math.sqrt(D + R) if scale is None else scale
    most = block_table.shape[1] * latents.shape[1]
    Wk, Wv = W[:H * D].double().view(H, D, rank) * gamma, W[H * D:].double().view(H, value_dim, rank) * gamma
    out, bound = torch.zeros(B, H, value_dim, dtype=torch.float64), torch.zeros(B, H, value_dim, dtype=torch.float64)
    for b in range(B):
        n = int(lengths[b].clamp(0, most))
        c, k, here, rows = cached(latents, absmax, keys, block_table[b], n)
        if not bool(here.any()):
            continue
        u = torch.einsum("hd,hdr->hr", q[b].double(), Wk)
        u_abs = torch.einsum("hd,hdr->hr", q[b].double().abs(), Wk.abs())
        z, size = u @ c.T, u.abs() @ c.abs().T
        # u is rounded as a factor: relative to itself, or to half a 32512th of the sum of |q| that bounds it; it is a sum of D terms before that
        step_of = (q[b].double().abs().sum(-1, keepdim=True) * abs(gamma) / (2 * 32512) if dtype != torch.float32 else 0.0) + unit * u.abs()
        off = (step_of + E * (D + 4) * u_abs) @ c.abs().T + tiny * math.sqrt(rank) * c.abs().sum(-1)
        if R:
            w = q_rot[b].double() if table is None else rotate(q_rot[b].double(), table, torch.full((H,), n - 1).clamp(max=table.shape[0] - 1), neighbours)
            z = z + w @ k.T
            size = size + w.abs() @ k.abs().T
            off = off + (unit + 4 * E) * (w.abs() @ k.abs().T) + tiny * k.abs().sum(-1)
        z = z * scale
        off = ((off + E * (rank + R + 8) * size) * abs(scale)).amax(-1, keepdim=True)
        p = _probabilities(z, here.expand(H, -1))
        rel = 2 * off + 4 * 2.0 ** -22 + 4 * (n + 8) * E + unit
        # probabilities are rounded together with their token's scale, relative to themselves, or to half a 32512th of the largest probability times the
        # largest scale (of the tile; here of all); the parts' sums are float32
        o, o_abs = p @ c, p @ c.abs()
        o_off = o_abs * (rel + n * E) + tiny * c.abs().sum(0)
        if dtype != torch.float32:
            scale_of = absmax.reshape(-1)[rows[here]].double() / 127
            ints = latents.reshape(-1, rank)[rows[here]].double().abs().sum(0)
            o_off = o_off + p.amax(-1, keepdim=True) * float(scale_of.max()) * ints * (1 + 1e-3) / (2 * 32512)
        out[b] = torch.einsum("hr,hvr->hv", o, Wv)
        bound[b] = torch.einsum("hr,hvr->hv", o_off + (rank + 4) * E * o_abs, Wv.abs()) + unit * out[b].abs() + tiny
    return out, bound
