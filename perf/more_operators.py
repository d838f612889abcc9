"""The operators of latent attention, as calls of their own: every token's keys and values come from one latent vector, which an INT2 layer (the up
projection) expands, and which a paged cache holds in 8 bits as that layer's quantised operand; part of a key may be rotated by its position instead,
one rotated part a token for all heads.

A case is a dict of plain values.  `op` and `mode` say which program is measured:

  attention  train    the expanded form, forward and backward: the output and the gradient of every input
             prompt   its forward pass: a prompt, or the next piece of one whose earlier tokens are keys only
  step       token    the absorbed form: one token for every sequence against the cache
  write      tokens   norm, quantisation and rotation of new tokens into the pages of a cache; the values that the pages then stand for
  read       rows     what the pages hold, as the up projection's operand: int8 rows and their scales
             values   the values that they stand for
  rotary     train    rotation by position, and its gradient
             infer    the rotation alone

`run` computes a case either in its plain form (elementary operations on float32 tensors) or, with `own`, through the package.
"""
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_EPS = 1e-6                 # of the norm in front of the up projection
_LEAST = 1e-5               # of a quantised row's largest magnitude
_BASE = 10000.0


def _package():
    """The package; its directory name has a hyphen, so it is loaded by path."""
    name = "elleci_training_vast_b200"
    if name not in sys.modules:
        folder = os.path.join(os.getcwd(), "elleci-training-vast_b200")
        spec = importlib.util.spec_from_file_location(name, os.path.join(folder, "__init__.py"), submodule_search_locations=[folder])
        module = importlib.util.module_from_spec(spec)
        sys.modules[name] = module
        spec.loader.exec_module(module)
    return sys.modules[name]


# ---- cases --------------------------------------------------------------------------------------------------------------

def _attention(mode, batch, length, keys, heads, key_dim=128, rot=64, value_dim=128, dtype="bf16", ragged=False):
    return {"op": "attention", "mode": mode, "batch": batch, "length": length, "keys": keys, "heads": heads, "key_dim": key_dim, "rot": rot,
            "value_dim": value_dim, "dtype": dtype, "ragged": ragged}


def _step(batch, keys, heads, rank=512, key_dim=128, rot=64, value_dim=128, page=64, dtype="bf16", ragged=False):
    return {"op": "step", "mode": "token", "batch": batch, "keys": keys, "heads": heads, "rank": rank, "key_dim": key_dim, "rot": rot,
            "value_dim": value_dim, "page": page, "dtype": dtype, "ragged": ragged}


def _cache(op, mode, batch, length, before=0, rank=512, rot=64, page=64, dtype="bf16", ragged=False):
    return {"op": op, "mode": mode, "batch": batch, "length": length, "before": before, "rank": rank, "rot": rot, "page": page, "dtype": dtype,
            "ragged": ragged}


def _rotary(mode, batch, length, heads, rot=64, dtype="bf16", far=0):
    return {"op": "rotary", "mode": mode, "batch": batch, "length": length, "heads": heads, "rot": rot, "dtype": dtype, "far": far}


def listed():
    return [
        # the 4096-wide model's training batch, 4 x 1024 tokens in 32 heads
        dict(_attention("train", 4, 1024, 1024, 32), name="attention_train"),
        # a small model's, padded sequences of unequal length and sizes that fill no tile, heads without a rotated part, another type
        dict(_attention("train", 3, 777, 777, 12, 96, 0, 64, dtype="fp16", ragged=True), name="attention_train_ragged"),
        # a long prompt of one sequence
        dict(_attention("prompt", 1, 8192, 8192, 32), name="attention_prompt"),
        # the next 250 tokens of two texts, up to 3999 tokens in all
        dict(_attention("prompt", 2, 250, 3999, 32, ragged=True), name="attention_continued"),
        # generation: a full batch of sequences of unequal length, and a single one with a long text behind it
        dict(_step(64, 8192, 32, ragged=True), name="step_64"),
        dict(_step(1, 32768, 32), name="step_1"),
        # a prompt's tokens on their way into the cache, and one token for each of 64 sequences
        dict(_cache("write", "tokens", 4, 1024), name="write_prompt"),
        dict(_cache("write", "tokens", 64, 1, before=1000), name="write_token"),
        # the whole texts of a batch for the next prompt pieces; a small model's in odd pages
        dict(_cache("read", "rows", 8, 8192, ragged=True), name="read_rows"),
        dict(_cache("read", "values", 3, 777, rank=256, rot=32, page=24, dtype="fp16", ragged=True), name="read_values"),
        # the rotated parts of a training batch's queries, and of one token for eight sequences, far into their texts
        dict(_rotary("train", 4, 1024, 32), name="rotary_train"),
        dict(_rotary("infer", 8, 1, 32, far=100000), name="rotary_token"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _odd(rng, lo, hi):
    """From `lo` to `hi`: mostly an odd number, now and then a power of two."""
    n = _log_int(rng, lo, hi)
    return min(n | 1, hi) if rng.random() < 0.7 else max(lo, 1 << (n.bit_length() - 1))


_MOST_PAIRS = 8192 * 8192 * 32 // 2        # query and key pairs of all heads of the largest attention
_MOST_CACHE = 8192 * 64                    # tokens of the largest cache


def draw(rng):
    """Another case of the same ranges: 1 to 64 sequences, 1 to 8192 tokens (generation: up to 32768), 1 to 64 heads, 64 to 128 channels of a key and
    a value, 0 to 64 rotated ones, latent vectors of 128 to 512 values, pages of 8 to 128 tokens, both data types, sequences of equal and unequal length."""
    dtype, ragged = rng.choice(["bf16", "bf16", "fp16"]), rng.random() < 0.5
    rot, page, rank = rng.choice([0, 32, 64, 64]), rng.choice([8, 16, 24, 32, 64, 64, 128]), rng.choice([128, 256, 256, 320, 512, 512])
    key_dim, value_dim = rng.choice([64, 96, 128, 128, 128]), rng.choice([64, 96, 128, 128, 128])
    op = rng.choice(["attention", "attention", "attention", "step", "step", "write", "read", "rotary"])
    if op == "attention":
        mode, batch, heads, length = rng.choice(["train", "prompt"]), _log_int(rng, 1, 16), _log_int(rng, 1, 64), _odd(rng, 1, 8192)
        keys = length if mode == "train" or rng.random() < 0.5 else length + _log_int(rng, 1, 8192)
        most = _MOST_PAIRS // (8 if mode == "train" else 2)
        while batch * heads * length * (keys - length // 2) > most:
            if batch > 1:
                batch //= 2
            elif heads > 4:
                heads //= 2
            else:
                length, keys = length // 2 | 1, keys // 2 + 2
        return _attention(mode, batch, length, keys, heads, key_dim, rot, value_dim, dtype, ragged)
    if op == "step":
        batch, keys = _log_int(rng, 1, 64), _odd(rng, 1, 32768)
        while batch * keys > _MOST_CACHE:
            batch //= 2
        return _step(batch, keys, _log_int(rng, 1, 64), rank, key_dim, rot, value_dim, page, dtype, ragged)
    batch, length = _log_int(rng, 1, 64), _odd(rng, 1, 8192)
    while batch * length > _MOST_CACHE // 8:
        batch //= 2
    if op == "rotary":
        return _rotary(rng.choice(["train", "infer"]), batch, length, _log_int(rng, 1, 32), rng.choice([32, 64, 64, 128]), dtype, rng.choice([0, _log_int(rng, 1, 100000)]))
    before = rng.choice([0, _log_int(rng, 1, 4096)]) if op == "write" else 0
    return _cache(op, "tokens" if op == "write" else rng.choice(["rows", "values"]), batch, length, before, rank, rot, page, dtype, ragged)


def _lengths(case, most):
    """Unequal lengths as a padded batch has them: the first is full, the others anywhere down to an empty one.  The case alone says which."""
    r = np.random.RandomState(case["batch"] * 65537 + most)
    n = r.randint(0, most + 1, case["batch"])
    n[0] = most
    return n if case["ragged"] else np.full(case["batch"], most)


def _key_lengths(case):
    """The keys of an attention's sequences: what a sequence lacks in queries it lacks in keys too."""
    return case["keys"] - case["length"] + _lengths(case, case["length"])


def work(case):
    """Each input read once and each output written once; a multiplication and an addition are an operation each."""
    b = case["batch"]
    if case["op"] == "attention":
        h, d, v = case["heads"], case["key_dim"] + case["rot"], case["value_dim"]
        n = _lengths(case, case["length"]).astype(np.float64)
        m = _key_lengths(case).astype(np.float64)
        pairs = float((n * (m - n) + n * (n + 1) / 2).sum()) * h
        values = b * case["length"] * h * (d + v) + b * case["keys"] * (h * (case["key_dim"] + v) + case["rot"])
        if case["mode"] == "prompt":
            return {"bytes": 2 * values, "flops": 2 * pairs * (d + v)}
        # backward: the scores again (they are too many to keep), and one product for each of dP, dQ, dK and dV
        return {"bytes": 2 * (2 * values), "flops": 2 * pairs * (d + v) + 2 * pairs * (3 * d + 2 * v)}
    if case["op"] == "step":
        h, r, d, v = case["heads"], case["rank"], case["key_dim"], case["value_dim"]
        tokens = int(_lengths(case, case["keys"]).sum())
        weights = h * (d + v) * r
        return {"bytes": tokens * (r + 4 + 2 * case["rot"]) + weights // 4 + b * h * 2 * (d + case["rot"] + v),
                "flops": 2 * tokens * h * (2 * r + case["rot"]) + 2 * b * weights}
    if case["op"] == "rotary":
        values = b * case["length"] * case["heads"] * case["rot"]
        return {"bytes": values * 2 * (4 if case["mode"] == "train" else 2), "flops": values * (6 if case["mode"] == "train" else 3)}
    tokens = int(_lengths(case, case["length"]).sum())
    r, k = case["rank"], case["rot"]
    if case["op"] == "write":           # in, into the pages, out of them, and the values
        return {"bytes": tokens * (2 * (r + k) + 2 * (r + 4 + 2 * k) + 2 * (r + k)), "flops": tokens * (10 * r + 3 * k)}
    each = r + 4 + 2 * k
    return {"bytes": tokens * each + b * case["length"] * (each if case["mode"] == "rows" else 2 * (r + k)), "flops": tokens * r}


# ---- inputs -------------------------------------------------------------------------------------------------------------

def _table(positions, dim):
    """Cosines, then sines, of position * base^(-2 i / dim): float32 values of angles in 64 bits."""
    rate = _BASE ** (-torch.arange(0, dim, 2, dtype=torch.float64, device="cuda") / dim)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * rate
    return torch.cat([angle.cos(), angle.sin()], -1).float()


def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    dt = _DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0, dtype=dt):
        t = torch.randn(*shape, generator=gen, device=dev) * std
        return (t + mean).to(dtype)

    def on_device(lengths):
        return torch.from_numpy(np.asarray(lengths)).to(dev, torch.int32)

    s = {"case": dict(case)}
    b = case["batch"]
    if case["op"] == "rotary":
        s.update(x=normal(b, case["length"], case["heads"], case["rot"]), table=_table(case["far"] + case["length"], case["rot"]),
                 positions=torch.full((b,), case["far"], device=dev, dtype=torch.int32) - torch.arange(b, device=dev, dtype=torch.int32).clamp(max=case["far"]))
        if case["mode"] == "train":
            s.update(x=s["x"].requires_grad_(True), dy=normal(*s["x"].shape, std=1e-2))
        return s
    if case["op"] == "attention":
        t, n, h, d, r, v = (case[k] for k in ("length", "keys", "heads", "key_dim", "rot", "value_dim"))
        # the projections' outputs: queries and keys of some size, so that a few keys count for more than the others
        s["q"] = normal(b, t, h * (d + r), std=1.2)[..., :h * d].unflatten(-1, (h, d))
        s["kv"] = normal(b, n, h * (d + v), std=1.2)
        s["q_rot"], s["k_rot"] = (normal(b, t, h, r, std=1.2), normal(b, n, r, std=1.2)) if r else (None, None)
        s["lengths"] = on_device(_lengths(case, t)) if case["ragged"] else None
        s["key_lengths"] = on_device(_key_lengths(case)) if case["ragged"] else None
        if case["mode"] == "train":
            s["inputs"] = [k for k in ("q", "kv", "q_rot", "k_rot") if s[k] is not None]
            s["dout"] = normal(b, t, h, v, std=1e-2)
            for k in s["inputs"]:
                s[k] = s[k].detach().requires_grad_(True)
        return s
    # a pool whose pages lie in any order, with some that belong to nobody
    page, r, k = case["page"], case["rank"], case["rot"]
    tokens = case["keys"] if case["op"] == "step" else case["before"] + case["length"]
    per = -(-tokens // page)
    pages = b * per + 3
    s["block_table"] = torch.randperm(pages, generator=gen, device=dev)[:b * per].to(torch.int32).view(b, per)
    if case["op"] == "write":
        s["latents"], s["absmax"] = torch.zeros(pages, page, r, device=dev, dtype=torch.int8), torch.zeros(pages, page, device=dev)
        s["keys"] = torch.zeros(pages, page, k, device=dev, dtype=dt) if k else None
        x = normal(b, case["length"], r + k, std=0.8)                  # the down projection's output: the latent vector and the rotated part
        s["latent"], s["k_rot"] = x[..., :r], x[..., r:] if k else None
        s["norm_weight"] = normal(r, std=0.1, mean=1.0, dtype=torch.float32)
        s["table"] = _table(tokens, k) if k else None
        s["starts"] = torch.full((b,), case["before"], device=dev, dtype=torch.int32)
        s["lengths"] = on_device(_lengths(case, case["length"])) if case["ragged"] else None
        return s
    # what a norm and a quantiser leave: the largest of a row is 127
    x = normal(pages, page, r, dtype=torch.float32)
    s["absmax"] = x.abs().amax(-1)
    s["latents"] = torch.round(x * (127.0 / s["absmax"])[..., None]).to(torch.int8)
    del x
    s["keys"] = normal(pages, page, k, std=1.2) if k else None
    if case["op"] == "read":
        s["lengths"] = on_device(_lengths(case, case["length"]))
        return s
    h, d, v = case["heads"], case["key_dim"], case["value_dim"]
    s["lengths"] = on_device(_lengths(case, tokens))
    s["q"], s["q_rot"] = normal(b, h, d, std=1.2), normal(b, h, k, std=1.2) if k else None
    s["table"] = _table(tokens, k) if k else None
    s["W_packed"] = torch.randint(0, 3, (h * (d + v), r // 4, 4), generator=gen, device=dev, dtype=torch.int32).mul_(
        torch.tensor([1, 4, 16, 64], device=dev, dtype=torch.int32)).sum(-1).to(torch.uint8)      # codes 0, 1, 2 stand for -1, 0, 1
    s["gamma"] = 1.2 / math.sqrt(r)
    return s


# ---- the plain forms ----------------------------------------------------------------------------------------------------

def _turn(x, cos, sin):
    """Pairs (x[i], x[i + half]) turned by their angles."""
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _cos_sin(table, at):
    return table[at].chunk(2, -1)


def _softmax(scores, seen):
    """Along the last dimension, over what is seen; zeros where that is nothing."""
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top > -math.inf, top, 0.0))
    return p / p.sum(-1, keepdim=True).clamp_min(1e-30)


def _plain_rotary(s):
    c, x = s["case"], s["x"].float()
    at = s["positions"].long()[:, None] + torch.arange(c["length"], device="cuda")
    cos, sin = (t[:, :, None] for t in _cos_sin(s["table"], at))
    out = {"y": _turn(x, cos, sin).to(s["x"].dtype)}
    if c["mode"] == "train":
        out["dx"] = _turn(s["dy"].float(), cos, -sin).to(s["x"].dtype)
    return out


def _plain_attention(s):
    c = s["case"]
    t, n, h, d, r, v = (c[k] for k in ("length", "keys", "heads", "key_dim", "rot", "value_dim"))
    io, scale = s["q"].dtype, 1.0 / math.sqrt(d + r)
    # heads first: [batch, heads, tokens, channels]
    q = s["q"].float().transpose(1, 2)
    k = s["kv"][..., :h * d].float().unflatten(-1, (h, d)).transpose(1, 2)
    val = s["kv"][..., h * d:].float().unflatten(-1, (h, v)).transpose(1, 2)
    if r:
        q = torch.cat([q, s["q_rot"].float().transpose(1, 2)], -1)
        k = torch.cat([k, s["k_rot"].float()[:, None].expand(-1, h, -1, -1)], -1)
    i, j = torch.arange(t, device="cuda")[:, None], torch.arange(n, device="cuda")
    if s["lengths"] is None:
        seen = (j <= i + (n - t))[None, None]
    else:
        ln, kn = s["lengths"][:, None, None], s["key_lengths"][:, None, None]
        seen = ((i < ln) & (j < kn) & (j <= i + (kn - ln)))[:, None]
        rows, keys = (i < ln)[:, None], (j[:, None] < kn)[:, None]
        q, k, val = (torch.where(live, x, 0.0) for live, x in ((rows, q), (keys, k), (keys, val)))
    p = _softmax(torch.matmul(q, k.transpose(-1, -2)) * scale, seen)
    o = torch.matmul(p, val)
    out = {"out": o.transpose(1, 2).to(io)}
    if c["mode"] == "prompt":
        return out
    do = s["dout"].float().transpose(1, 2)
    if s["lengths"] is not None:
        do = torch.where(rows, do, 0.0)
    dval = torch.matmul(p.transpose(-1, -2), do)
    dp = torch.matmul(do, val.transpose(-1, -2))
    ds = p * (dp - (do * o).sum(-1, keepdim=True)) * scale
    dq, dk = torch.matmul(ds, k), torch.matmul(ds.transpose(-1, -2), q)
    out["dq"] = dq[..., :d].transpose(1, 2).to(io)
    out["dkv"] = torch.cat([dk[..., :d].transpose(1, 2).flatten(2), dval.transpose(1, 2).flatten(2)], -1).to(io)
    if r:
        out["dq_rot"], out["dk_rot"] = dq[..., d:].transpose(1, 2).to(io), dk[..., d:].sum(1).to(io)
    return out


def _slots(s, at):
    """Pages and places in them of the sequences' positions `at` [batch, n]."""
    page = s["case"]["page"]
    return s["block_table"].long().gather(1, at // page), at % page


def _plain_step(s):
    c = s["case"]
    h, r, d, k, v = (c[x] for x in ("heads", "rank", "key_dim", "rot", "value_dim"))
    codes = (s["W_packed"][..., None] >> torch.tensor([0, 2, 4, 6], device="cuda", dtype=torch.uint8)) & 3
    W = ((codes == 2).float() - (codes == 0).float()).flatten(1) * s["gamma"]
    at = torch.arange(c["keys"], device="cuda")
    where = _slots(s, at.expand(c["batch"], -1))
    latent = s["latents"][where].float() * (s["absmax"][where] / 127.0)[..., None]
    # q (W c) = (q W) c: the heads' queries against the latent vectors themselves
    q = torch.einsum("bhd,hdr->bhr", s["q"].float(), W[:h * d].view(h, d, r))
    scores = torch.matmul(q, latent.transpose(1, 2))
    if k:
        cos, sin = (t[:, None] for t in _cos_sin(s["table"], (s["lengths"].long() - 1).clamp_min(0)))
        scores = scores + torch.matmul(_turn(s["q_rot"].float(), cos, sin), s["keys"][where].float().transpose(1, 2))
    p = _softmax(scores / math.sqrt(d + k), (at < s["lengths"][:, None])[:, None])
    o = torch.matmul(p, latent)
    return {"out": torch.einsum("bhr,hvr->bhv", o, W[h * d:].view(h, v, r)).to(s["q"].dtype)}


def _plain_write(s):
    c = s["case"]
    io, w = s["latent"].dtype, s["norm_weight"]
    # the norm of the layer that reads these rows: its definition rounds to the type after the norm and after the weight
    x = s["latent"].float()
    x = (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS)).to(io).float()
    x = (x * w.to(io).float()).to(io).float()
    top = x.abs().amax(-1).clamp_min(_LEAST)
    rows = torch.round(x * (127.0 / top)[..., None]).to(torch.int8)
    at = s["starts"].long()[:, None] + torch.arange(c["length"], device="cuda")
    pages, places = _slots(s, at)
    live = None
    if s["lengths"] is not None:
        live = torch.arange(c["length"], device="cuda") < s["lengths"][:, None]
        pages, places, rows, top = pages[live], places[live], rows[live], top[live]
    s["latents"][pages, places], s["absmax"][pages, places] = rows, top
    if c["rot"]:
        keys = _turn(s["k_rot"].float(), *_cos_sin(s["table"], at)).to(io)
        s["keys"][pages, places] = keys if live is None else keys[live]
    return _plain_values(s, at, live)


def _plain_values(s, at, live):
    io = _DTYPES[s["case"]["dtype"]]
    where = _slots(s, at)
    values = s["latents"][where].float() * (s["absmax"][where] / 127.0)[..., None]
    out = {"values": (values if live is None else torch.where(live[..., None], values, 0.0)).to(io)}
    if s["case"]["rot"]:
        out["keys"] = s["keys"][where] if live is None else torch.where(live[..., None], s["keys"][where], 0.0)
    return out


def _plain_read(s):
    c = s["case"]
    at = torch.arange(c["length"], device="cuda").expand(c["batch"], -1)
    live = at < s["lengths"][:, None]
    if c["mode"] == "values":
        return _plain_values(s, at, live)
    where = _slots(s, at)
    out = {"rows": torch.where(live[..., None], s["latents"][where], 0).flatten(0, 1), "absmax": torch.where(live, s["absmax"][where], 0.0).flatten()}
    if c["rot"]:
        out["keys"] = torch.where(live[..., None], s["keys"][where], 0.0)
    return out


_PLAIN = {"attention": _plain_attention, "step": _plain_step, "write": _plain_write, "read": _plain_read, "rotary": _plain_rotary}


# ---- through the package ------------------------------------------------------------------------------------------------

def _own(s):
    c, ops = s["case"], _package().attention_ops
    if c["op"] == "rotary":
        if c["mode"] == "infer":
            return {"y": ops.rotary(s["x"], s["table"], s["positions"])}
        y = ops.rotary(s["x"], s["table"], s["positions"])
        return {"y": y, "dx": torch.autograd.grad(y, s["x"], s["dy"])[0]}
    if c["op"] == "attention":
        out = ops.latent_attention(s["q"], s["kv"], s["q_rot"], s["k_rot"], lengths=s["lengths"], key_lengths=s["key_lengths"])
        result = {"out": out}
        if c["mode"] == "train":
            result.update(zip(["d" + n for n in s["inputs"]], torch.autograd.grad(out, [s[n] for n in s["inputs"]], s["dout"])))
        return result
    cache = ops.LatentCache(s["latents"], s["absmax"], s["keys"])
    if c["op"] == "step":
        return {"out": ops.latent_attention_step(s["q"], s["W_packed"], s["gamma"], cache, s["block_table"], s["lengths"], c["value_dim"],
                                                 q_rot=s["q_rot"], table=s["table"])}
    if c["op"] == "read" and c["mode"] == "rows":
        rows, absmax, keys = ops.latent_cache_read(cache, s["block_table"], c["length"], lengths=s["lengths"])
        return {"rows": rows, "absmax": absmax, "keys": keys} if c["rot"] else {"rows": rows, "absmax": absmax}
    starts = None
    if c["op"] == "write":
        starts = s["starts"]
        ops.latent_cache_write(cache, s["block_table"], s["latent"], s["norm_weight"], s["k_rot"], s["table"], starts=starts, lengths=s["lengths"])
    values, keys = ops.latent_cache_read(cache, s["block_table"], c["length"], starts=starts, lengths=s["lengths"], dtype=_DTYPES[c["dtype"]])
    return {"values": values, "keys": keys} if c["rot"] else {"values": values}


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _PLAIN[state["case"]["op"]](state)


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------

def _rotated(x, table, first):
    """x [tokens, .., channels] as complex numbers, token t turned by row first + t of the table."""
    half = x.shape[-1] // 2
    turn = torch.complex(table[:, :half].double(), table[:, half:].double())[first:first + x.shape[0]]
    z = torch.complex(x[..., :half], x[..., half:]) * turn.view(x.shape[0], *[1] * (x.dim() - 2), half)
    return torch.cat([z.real, z.imag], -1)


def exact(case, seed):
    """Sequence by sequence and head by head, in float64."""
    s = prepare(case, seed)
    b = case["batch"]
    with torch.no_grad():
        if case["op"] == "rotary":
            first = [int(p) for p in s["positions"]]
            out = {"y": torch.stack([_rotated(s["x"][i].double(), s["table"], first[i]) for i in range(b)])}
            if case["mode"] == "train":
                back = torch.cat([s["table"][:, :case["rot"] // 2], -s["table"][:, case["rot"] // 2:]], -1)
                out["dx"] = torch.stack([_rotated(s["dy"][i].double(), back, first[i]) for i in range(b)])
            return out

        if case["op"] == "attention":
            t, n, h, d, r, v = (case[k] for k in ("length", "keys", "heads", "key_dim", "rot", "value_dim"))
            ends, key_ends = _lengths(case, t), _key_lengths(case)
            train = case["mode"] == "train"

            def zeros(*shape):
                return torch.zeros(*shape, device="cuda", dtype=torch.float64)

            o = zeros(b, t, h, v)
            dq, dkv, dqr, dkr = (zeros(b, t, h, d), zeros(b, n, h * (d + v)), zeros(b, t, h, r), zeros(b, n, r)) if train else [None] * 4
            for i in range(b):
                a, e = int(ends[i]), int(key_ends[i])
                if a == 0:
                    continue
                hidden = torch.ones(a, e, device="cuda", dtype=torch.bool).triu(e - a + 1)
                for j in range(h):
                    key, val = slice(j * d, (j + 1) * d), slice(h * d + j * v, h * d + (j + 1) * v)
                    q, k, x = s["q"][i, :a, j].double(), s["kv"][i, :e, key].double(), s["kv"][i, :e, val].double()
                    z = q @ k.T
                    if r:
                        qr, kr = s["q_rot"][i, :a, j].double(), s["k_rot"][i, :e].double()
                        z += qr @ kr.T
                    p = torch.softmax((z / math.sqrt(d + r)).masked_fill_(hidden, -math.inf), -1)
                    o[i, :a, j] = p @ x
                    if not train:
                        continue
                    g = s["dout"][i, :a, j].double()
                    dkv[i, :e, val] = p.T @ g
                    dz = g @ x.T
                    dz = p * (dz - (p * dz).sum(-1, keepdim=True)) / math.sqrt(d + r)
                    dq[i, :a, j], dkv[i, :e, key] = dz @ k, dz.T @ q
                    if r:
                        dqr[i, :a, j] = dz @ kr
                        dkr[i, :e] += dz.T @ qr
            out = {"out": o}
            if train:
                out.update(dq=dq, dkv=dkv)
                if r:
                    out.update(dq_rot=dqr, dk_rot=dkr)
            return out

        page, r, k = case["page"], case["rank"], case["rot"]

        def token_rows(i, first, count):
            """The pool's rows, counted through its pages, of `count` positions of sequence i."""
            at = torch.arange(first, first + count, device="cuda")
            return s["block_table"][i].long()[at // page] * page + at % page

        latents, absmax = s["latents"].view(-1, r), s["absmax"].view(-1)
        keys = s["keys"].view(-1, k) if k else None
        if case["op"] == "step":
            h, d, v = case["heads"], case["key_dim"], case["value_dim"]
            w = torch.stack([(s["W_packed"] // 4 ** i) % 4 for i in range(4)], -1).flatten(1).double() - 1.0
            o = torch.zeros(b, h, v, device="cuda", dtype=torch.float64)
            for i, e in enumerate(_lengths(case, case["keys"])):
                if e == 0:
                    continue
                rows = token_rows(i, 0, int(e))
                # expanded: every token's keys and values of all heads
                kv = (latents[rows].double() * (absmax[rows].double() / 127)[:, None]) @ w.T * s["gamma"]
                z = torch.einsum("hd,nhd->hn", s["q"][i].double(), kv[:, :h * d].view(-1, h, d))
                if k:
                    z += _rotated(s["q_rot"][i].double()[None], s["table"], int(e) - 1)[0] @ keys[rows].double().T
                o[i] = torch.einsum("hn,nhv->hv", torch.softmax(z / math.sqrt(d + k), -1), kv[:, h * d:].view(-1, h, v))
            return {"out": o}

        l, io = case["length"], _DTYPES[case["dtype"]]
        ends = _lengths(case, l)
        values = torch.zeros(b, l, r, device="cuda", dtype=torch.float64)
        back = torch.zeros(b, l, k, device="cuda", dtype=torch.float64)
        if case["op"] == "write":
            for i in range(b):
                n = int(ends[i])
                x = s["latent"][i, :n].double()
                # the type's two roundings and the 8 bits are part of the definition: the rows are what the layer itself would take
                rate = (1 / (x.pow(2).sum(-1, keepdim=True) / r + _EPS).sqrt()).float().double()
                y = (x * rate).float().to(io).double()
                y = (y * s["norm_weight"].to(io).double()).to(io).double()
                top = y.abs().max(-1, keepdim=True).values.clamp(min=float(np.float32(_LEAST)))
                values[i, :n] = torch.round((y.float() * (127 / top).float())).double() * top / 127
                if k:
                    back[i, :n] = _rotated(s["k_rot"][i, :n].double(), s["table"], case["before"])
            return {"values": values, "keys": back} if k else {"values": values}
        if case["mode"] == "rows":
            held, tops = torch.zeros(b, l, r, device="cuda", dtype=torch.int8), torch.zeros(b, l, device="cuda", dtype=torch.float64)
        for i in range(b):
            n = int(ends[i])
            rows = token_rows(i, 0, n)
            if case["mode"] == "rows":
                held[i, :n], tops[i, :n] = latents[rows], absmax[rows].double()
            else:
                values[i, :n] = latents[rows].double() * (absmax[rows].double() / 127)[:, None]
            if k:
                back[i, :n] = keys[rows].double()
        out = {"rows": held.flatten(0, 1), "absmax": tops.flatten()} if case["mode"] == "rows" else {"values": values}
        if k:
            out["keys"] = back
        return out
