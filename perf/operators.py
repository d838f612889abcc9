"""The operators between the projections of a Mamba block, as calls of their own: the short causal convolution, the selective state
space scan (each for training, for prompts and for single tokens) and the norms before and after the block with its gate and
residual scale.

A case is a dict of plain values.  `op` is conv, scan or norm; `mode` says which program is measured:

  train   forward and backward: the output and the gradient of every input
  prompt  the forward pass of a served prompt: the output and the state after each sequence's last token
  step    one token for every sequence: the output and the state after it
  infer   (norm) the forward pass alone

`run` computes a case either in its plain form (elementary operations on float32 tensors) or, with `own`, through the package.
"""
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_EPS = 1e-6


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

def _conv(mode, batch, length, channels, width=4, dtype="bf16", ragged=False, state=False):
    return {"op": "conv", "mode": mode, "batch": batch, "length": length, "channels": channels, "width": width, "dtype": dtype,
            "ragged": ragged, "state": state}


def _scan(mode, batch, length, channels, states=16, groups=1, dtype="bf16", gated=True, ragged=False, state=False):
    return {"op": "scan", "mode": mode, "batch": batch, "length": length, "channels": channels, "states": states, "groups": groups,
            "dtype": dtype, "gated": gated, "ragged": ragged, "state": state}


def _norm(mode, rows, width, dtype="bf16", gated=True, scaled=True):
    return {"op": "norm", "mode": mode, "rows": rows, "width": width, "dtype": dtype, "gated": gated, "scaled": scaled}


def listed():
    return [
        # the 4096-wide block's inner 8192 channels, batch 4 x 1024 tokens: a training step of each operator
        dict(_conv("train", 4, 1024, 8192), name="conv_train"),
        dict(_scan("train", 4, 1024, 8192), name="scan_train"),
        dict(_norm("train", 4096, 4096), name="norm_train"),
        # the same of a small model, with sizes that fill no tile: another type, shared B and C in two groups, sequences of unequal length
        dict(_scan("train", 2, 777, 1536, groups=2, dtype="fp32", ragged=True), name="scan_train_ragged"),
        dict(_norm("train", 1999, 1536, dtype="fp16"), name="norm_train_small"),
        # prompts: a batch of three unequal ones that continue earlier text, a long one of the large model, a longer one of a narrow model
        dict(_conv("prompt", 3, 1999, 1504, dtype="fp16", ragged=True, state=True), name="conv_prompt_ragged"),
        dict(_scan("prompt", 1, 4096, 8192), name="scan_prompt"),
        dict(_scan("prompt", 1, 16384, 2048, state=True), name="scan_prompt_narrow"),
        # generation: one token for one sequence, for eight and for a full batch
        dict(_scan("step", 1, 1, 8192, state=True), name="scan_step_1"),
        dict(_scan("step", 64, 1, 8192, state=True), name="scan_step_64"),
        dict(_conv("step", 8, 1, 8192, state=True), name="conv_step_8"),
        dict(_norm("infer", 8, 4096), name="norm_infer_8"),
    ]


_MOST_STATES = 4 * 1024 * 8192 * 16        # batch x length x channels x states of the largest scan
_MOST_VALUES = 4 * 1024 * 8192             # batch x length x channels of the largest convolution


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _length(rng, hi):
    """From one token to `hi`: an odd number, or now and then a power of two."""
    n = _log_int(rng, 1, hi)
    return n | 1 if rng.random() < 0.7 else 1 << (n.bit_length() - 1)


def _width(rng):
    """80 to 8200 in steps of 40, and now and then an odd one."""
    w = 40 * _log_int(rng, 2, 205)
    return w + 1 if rng.random() < 0.15 else w


def draw(rng):
    """Another case of the same ranges: 1 to 64 sequences, 1 to 16384 tokens, 80 to 8200 channels, 4 to 64 states (mostly 16), convolutions
    over 2 to 4 tokens, all three data types, with and without gate, initial state and sequences of unequal length."""
    dtype = rng.choice(["bf16"] * 5 + ["fp16"] * 2 + ["fp32"] * 2)
    op = rng.choice(["conv", "scan", "scan", "scan", "norm"])
    width = _width(rng)
    if op == "norm":
        rows = _log_int(rng, 1, 16384) | 1
        while rows * width > 4096 * 4096:
            rows = rows // 4 * 2 + 1
        return _norm(rng.choice(["train", "infer"]), rows, width, dtype, rng.random() < 0.7, rng.random() < 0.7)
    mode = rng.choice(["train", "train", "prompt", "prompt", "step"])
    batch, length = _log_int(rng, 1, 64), 1
    if mode != "step":
        batch = min(batch, 8)
        length = _length(rng, 16384)
    ragged, state = mode != "step" and rng.random() < 0.4, mode == "step" or rng.random() < 0.4
    if op == "conv":
        while batch * length * width > _MOST_VALUES // 2:
            length = length // 4 * 2 + 1
        return _conv(mode, batch, length, width, rng.choice([2, 3, 4, 4]), dtype, ragged, state)
    states, groups = rng.choice([16, 16, 16, 16, 8, 4, 12, 32, 64]), rng.choice([1, 1, 2, 4])
    groups = groups if width % groups == 0 else 1
    while batch * length * width * states > _MOST_STATES // 2:
        length = length // 4 * 2 + 1
    return _scan(mode, batch, length, width, states, groups, dtype, rng.random() < 0.8, ragged, state)


def work(case):
    """Each input read once, each output written once; a multiplication, an addition and an exponential are an operation each."""
    e = _BYTES[case["dtype"]]
    train = case["mode"] == "train"
    if case["op"] == "norm":
        n = case["rows"] * case["width"]
        tensors = (2 + case["gated"]) * (2 if train else 1) + (4 if train else 2)      # h, y, gate and their gradients; both outputs and theirs
        return {"bytes": n * e * tensors + 4 * case["width"] * 3, "flops": n * (40 if train else 14)}
    values = case["batch"] * case["length"] * case["channels"]
    rows = case["batch"] * case["channels"]
    if case["op"] == "conv":
        w = case["width"]
        tensors = 4 if train else 2
        state = (w - 1) * rows * e * ((0 if train else 1) + (2 if train else 1) * case["state"])
        return {"bytes": values * e * tensors + state + 4 * case["channels"] * (w + 1) * (2 if train else 1),
                "flops": values * (2 * w + 5) * (3 if train else 1)}
    n = case["states"]
    shared = case["batch"] * case["length"] * case["groups"] * n * e * 2
    tensors = (2 + case["gated"]) * (2 if train else 1) + (2 if train else 1)
    state = 4 * n * rows * ((0 if train else 1) + (2 if train else 1) * case["state"])
    return {"bytes": values * e * tensors + shared * (2 if train else 1) + state + 4 * case["channels"] * (n + 2) * (2 if train else 1),
            "flops": values * (n * (23 if train else 7) + (30 if train else 12))}


# ---- inputs -------------------------------------------------------------------------------------------------------------

def _lengths(case, seed):
    """Unequal lengths as a padded batch has them: one full, the others anywhere down to an empty one."""
    r = np.random.RandomState(seed & 0x7FFFFFFF)
    n = r.randint(0, case["length"] + 1, case["batch"])
    n[r.randint(case["batch"])] = case["length"]
    return n


def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    dt = _DTYPES[case["dtype"]]
    train = case["mode"] == "train"

    def normal(*shape, std=1.0, mean=0.0, dtype=dt):
        t = torch.randn(*shape, generator=gen, device=dev) * std
        return (t + mean).to(dtype)

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device=dev)

    s = {"case": dict(case)}
    if case["op"] == "norm":
        m, k = case["rows"], case["width"]
        s.update(h=normal(m, k, std=2.0), y=normal(m, k, std=0.5), post_weight=normal(k, std=0.1, mean=1.0, dtype=torch.float32),
                 pre_weight=normal(k, std=0.1, mean=1.0, dtype=torch.float32))
        s["gate"] = normal(m, k) if case["gated"] else None
        s["scale"] = normal(k, std=0.02, mean=0.5, dtype=torch.float32) if case["scaled"] else None
        if train:
            s.update(dh_out=normal(m, k, std=1e-2), dnormed=normal(m, k, std=1e-2))
            s["inputs"] = [n for n in ("h", "y", "post_weight", "pre_weight", "gate", "scale") if s[n] is not None]
    else:
        b, l, d = case["batch"], case["length"], case["channels"]
        shape = (b, d) if case["mode"] == "step" else (b, l, d)
        s["lengths"] = torch.from_numpy(_lengths(case, seed)).to(dev, torch.int32) if case["ragged"] else None
        if case["op"] == "conv":
            w = case["width"]
            # the convolution reads the first half of the input projection's output
            s.update(x=normal(*shape[:-1], 2 * d)[..., :d], weight=normal(d, w, std=0.5 / math.sqrt(w), dtype=torch.float32), bias=normal(d, std=0.1, dtype=torch.float32))
            s["state"] = normal(b, w - 1, d) if case["state"] else None
            if case["mode"] == "step":
                s["state_out"] = torch.empty_like(s["state"])
            if train:
                s["dy"] = normal(b, l, d, std=1e-2)
                s["inputs"] = ["x", "weight", "bias"] + (["state"] if case["state"] else [])
        else:
            n, g = case["states"], case["groups"]
            x = normal(*shape, dtype=torch.float32)
            s["u"] = (x * torch.sigmoid(x)).to(dt)
            # step sizes from 0.001 to 0.1 in the bias, moved by the projection; decay rates around -1 .. -n
            first = torch.exp(uniform(d) * math.log(100.0) + math.log(1e-3))
            s["dt_bias"] = first + torch.log(-torch.expm1(-first))
            s["dt"] = normal(*shape, std=0.5)
            s["A"] = -torch.arange(1, n + 1, device=dev, dtype=torch.float32) * torch.exp(0.1 * normal(d, n, dtype=torch.float32))
            # B and C are parts of one projection's output, behind the step sizes' sixteen
            bc = normal(*shape[:-1], 16 + 2 * g * n)
            s["B"] = bc[..., 16:16 + g * n].unflatten(-1, (g, n))
            s["C"] = bc[..., 16 + g * n:].unflatten(-1, (g, n))
            s["D"] = normal(d, std=0.1, mean=1.0, dtype=torch.float32)
            s["z"] = normal(*shape[:-1], 2 * d)[..., d:] if case["gated"] else None
            s["state"] = normal(b, d, n, std=0.3, dtype=torch.float32) if case["state"] else None
            if case["mode"] == "step":
                s["state_out"] = torch.empty_like(s["state"])
            if train:
                s["dout"] = normal(b, l, d, std=1e-2)
                s["inputs"] = [k for k in ("u", "dt", "A", "B", "C", "D", "z", "dt_bias", "state") if s[k] is not None]
    if train:
        for name in s["inputs"]:
            s[name] = s[name].detach().requires_grad_(True)
    return s


# ---- the plain forms ----------------------------------------------------------------------------------------------------

def _sigmoid(x):
    return 1.0 / (1.0 + torch.exp(-x))


def _softplus(x):
    return torch.clamp(x, min=0.0) + torch.log1p(torch.exp(-x.abs()))


def _recurrence(a, b):
    """h[t] = a[t] h[t-1] + b[t] along dimension 1 by doubling: after a pass with step s, a position holds the last 2 s terms."""
    s = 1
    while s < a.shape[1]:
        b = torch.cat([b[:, :s], torch.addcmul(b[:, s:], a[:, s:], b[:, :-s])], 1)
        a = torch.cat([a[:, :s], a[:, s:] * a[:, :-s]], 1)
        s *= 2
    return b


def _live(s):
    """1 for a token, 0 for padding: [batch, length, 1] truth values, or None."""
    if s["lengths"] is None:
        return None
    return (torch.arange(s["case"]["length"], device="cuda") < s["lengths"][:, None])[..., None]


def _kept(x, live):
    return x if live is None else torch.where(live, x, 0.0)


def _plain_conv(s):
    c = s["case"]
    w, f = c["width"], torch.float32
    io = s["x"].dtype
    weight, bias = s["weight"], s["bias"]
    if c["mode"] == "step":
        rows = torch.cat([s["state"].to(f), s["x"].to(f)[:, None]], 1)
        pre = bias + (rows * weight.t()).sum(1)
        return {"y": (pre * _sigmoid(pre)).to(io), "state": rows[:, 1:].to(io)}
    live, b, l = _live(s), c["batch"], c["length"]
    x = _kept(s["x"].to(f), live)
    first = x.new_zeros(b, w - 1, c["channels"]) if s["state"] is None else s["state"].to(f)
    rows = torch.cat([first, x], 1)
    pre = bias + sum(weight[:, j] * rows[:, j:j + l] for j in range(w))
    sig = _sigmoid(pre)
    y = _kept(pre * sig, live)
    if c["mode"] == "prompt":
        end = torch.full((b,), l, device="cuda") if s["lengths"] is None else s["lengths"].long()
        at = end[:, None] + torch.arange(w - 1, device="cuda")
        return {"y": y.to(io), "state": rows[torch.arange(b, device="cuda")[:, None], at].to(io)}
    dpre = _kept(s["dy"].to(f) * (sig + pre * sig * (1.0 - sig)), live)
    out = {"y": y.to(io), "dbias": dpre.sum((0, 1)), "dweight": torch.stack([(dpre * rows[:, j:j + l]).sum((0, 1)) for j in range(w)], 1)}
    pad = torch.cat([dpre.new_zeros(b, w - 1, c["channels"]), dpre, dpre.new_zeros(b, w - 1, c["channels"])], 1)
    drows = sum(weight[:, j] * pad[:, w - 1 - j:2 * (w - 1) - j + l] for j in range(w))
    out["dx"] = _kept(drows[:, w - 1:], live).to(io)
    if c["state"]:
        out["dstate"] = drows[:, :w - 1].to(io)
    return out


def _plain_scan(s):
    c = s["case"]
    f, g, n = torch.float32, c["groups"], c["states"]
    io = s["u"].dtype
    if c["mode"] == "step":
        u, raw, Bm, Cm = s["u"].to(f), s["dt"].to(f) + s["dt_bias"], s["B"].to(f), s["C"].to(f)
        delta = _softplus(raw)
        b, d = u.shape
        h = torch.exp(delta[..., None] * s["A"]) * s["state"]
        h = h + ((delta * u).view(b, g, d // g, 1) * Bm[:, :, None]).view(b, d, n)
        y = (h.view(b, g, d // g, n) * Cm[:, :, None]).sum(-1).view(b, d) + s["D"] * u
        if c["gated"]:
            z = s["z"].to(f)
            y = y * z * _sigmoid(z)
        return {"y": y.to(io), "state": h}
    b, l, d = c["batch"], c["length"], c["channels"]
    live = _live(s)

    def split(t):                                    # [.., channels] -> [.., groups, channels of a group]
        return t.view(*t.shape[:-1], g, d // g)

    u, raw = _kept(s["u"].to(f), live), s["dt"].to(f) + s["dt_bias"]
    delta = _kept(_softplus(raw), live)
    Bm, Cm = (_kept(s[k].to(f).flatten(2), live).view(b, l, g, 1, n) for k in ("B", "C"))
    A = s["A"].view(g, d // g, n)
    a = torch.exp(split(delta)[..., None] * A)
    first = a.new_zeros(b, g, d // g, n) if s["state"] is None else s["state"].view(b, g, d // g, n)
    du = split(delta * u)[..., None]
    x = du * Bm
    x[:, 0] += a[:, 0] * first
    h = _recurrence(a, x)
    del x
    y = (h * Cm).sum(-1).view(b, l, d) + s["D"] * u
    z = _kept(s["z"].to(f), live) if c["gated"] else None
    sig = _sigmoid(z) if c["gated"] else None
    out = {"y": _kept(y * z * sig if c["gated"] else y, live).to(io)}
    if c["mode"] == "prompt":
        out["state"] = h[:, -1].reshape(b, d, n)
        return out
    dout = _kept(s["dout"].to(f), live)
    dy = dout * z * sig if c["gated"] else dout
    if c["gated"]:
        out["dz"] = (dout * y * (sig + z * sig * (1.0 - sig))).to(io)
    dys = split(dy)[..., None]
    out["dC"] = (dys * h).sum(3).to(io)
    after = torch.cat([a[:, 1:], torch.ones_like(a[:, :1])], 1)
    adj = _recurrence(after.flip(1), (dys * Cm).flip(1)).flip(1)
    del after
    out["dB"] = (adj * du).sum(3).to(io)
    gb = (adj * Bm).sum(-1).view(b, l, d)
    w = adj * a
    if c["state"]:
        out["dstate"] = w[:, 0].reshape(b, d, n)
    w = w * torch.cat([first[:, None], h[:, :-1]], 1)
    out["dA"] = (w * split(delta)[..., None]).sum((0, 1)).view(d, n)
    ddt = _kept(((w * A).sum(-1).view(b, l, d) + u * gb) * _sigmoid(raw), live)
    out.update(du=_kept(s["D"] * dy + delta * gb, live).to(io), ddt=ddt.to(io), dD=(dy * u).sum((0, 1)), ddt_bias=ddt.sum((0, 1)))
    return out


def _plain_norm(s):
    f, io = torch.float32, s["h"].dtype
    h, y = s["h"].to(f), s["y"].to(f)
    r1 = torch.rsqrt((y * y).mean(-1, keepdim=True) + _EPS)
    yn = y * r1
    p = yn * s["post_weight"]
    sig = _sigmoid(s["gate"].to(f)) if s["gate"] is not None else None
    factor = 1.0 if s["scale"] is None else s["scale"]
    q = p * factor * (1.0 if sig is None else sig)
    ho = h + q
    r2 = torch.rsqrt((ho * ho).mean(-1, keepdim=True) + _EPS)
    hn = ho * r2
    out = {"h_out": ho.to(io), "normed": (hn * s["pre_weight"]).to(io)}
    if s["case"]["mode"] == "infer":
        return out
    dn = s["dnormed"].to(f)
    out["dpre_weight"] = (dn * hn).sum(0)
    dn = dn * s["pre_weight"]
    dh = s["dh_out"].to(f) + r2 * (dn - hn * (dn * hn).mean(-1, keepdim=True))
    dp = dh * factor * (1.0 if sig is None else sig)
    if sig is not None:
        out["dgate"] = (dh * factor * p * sig * (1.0 - sig)).to(io)
    if s["scale"] is not None:
        out["dscale"] = (dh * p * (1.0 if sig is None else sig)).sum(0)
    out["dpost_weight"] = (dp * yn).sum(0)
    dp = dp * s["post_weight"]
    out["dy"] = (r1 * (dp - yn * (dp * yn).mean(-1, keepdim=True))).to(io)
    out["dh"] = dh.to(io)
    return out


# ---- the package's operators --------------------------------------------------------------------------------------------

def _own(s):
    ops = _package().ssm_ops
    c = s["case"]
    train, step = c["mode"] == "train", c["mode"] == "step"
    if c["op"] == "norm":
        outs = ops.block_norm(s["h"], s["y"], s["post_weight"], s["pre_weight"], gate=s["gate"], scale=s["scale"], eps=_EPS)
        names, douts = ("h_out", "normed"), (s["dh_out"], s["dnormed"]) if train else None
    elif c["op"] == "conv":
        if step:
            y = ops.causal_conv_step(s["x"], s["state"], s["weight"], s["bias"], activation="silu", state_out=s["state_out"])
            return {"y": y, "state": s["state_out"]}
        outs = ops.causal_conv(s["x"], s["weight"], s["bias"], activation="silu", initial_state=s["state"], lengths=s["lengths"],
                               return_final_state=not train)
        names, douts = ("y", "state"), (s["dy"],) if train else None
    else:
        if step:
            y = ops.selective_scan_step(s["u"], s["dt"], s["A"], s["B"], s["C"], s["state"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"],
                                        state_out=s["state_out"])
            return {"y": y, "state": s["state_out"]}
        outs = ops.selective_scan(s["u"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"],
                                  initial_state=s["state"], lengths=s["lengths"], return_final_state=not train)
        names, douts = ("y", "state"), (s["dout"],) if train else None
    outs = outs if isinstance(outs, tuple) else (outs,)
    result = dict(zip(names, outs))
    if train:
        result.update(zip(["d" + n for n in s["inputs"]], torch.autograd.grad(outs, [s[n] for n in s["inputs"]], douts)))
    return result


_PLAIN = {"conv": _plain_conv, "scan": _plain_scan, "norm": _plain_norm}


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _PLAIN[state["case"]["op"]](state)


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------

def exact(case, seed):
    """Token by token and by the chain rule of each token, in float64."""
    s = prepare(case, seed)
    d64 = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor) and k != "lengths"}
    train = case["mode"] == "train"

    def logistic(x):
        return torch.sigmoid(x)

    def silu_and_slope(x):
        sg = torch.sigmoid(x)
        return x * sg, sg * (1 + x * (1 - sg))

    with torch.no_grad():
        if case["op"] == "norm":
            h, y, w1, w2 = d64["h"], d64["y"], d64["post_weight"], d64["pre_weight"]
            k = case["width"]
            m1 = (y ** 2).sum(-1, keepdim=True) / k + _EPS
            y1 = y / m1.sqrt()
            gate = logistic(d64["gate"]) if case["gated"] else torch.ones_like(y)
            scale = d64["scale"] if case["scaled"] else torch.ones_like(w1)
            ho = h + scale * gate * (w1 * y1)
            m2 = (ho ** 2).sum(-1, keepdim=True) / k + _EPS
            h1 = ho / m2.sqrt()
            out = {"h_out": ho, "normed": w2 * h1}
            if not train:
                return out
            dn = d64["dnormed"]
            out["dpre_weight"] = (dn * h1).sum(0)
            t = dn * w2
            # d(ho / sqrt(m2)): the part along ho is taken out
            dho = d64["dh_out"] + t / m2.sqrt() - ho * (t * ho).sum(-1, keepdim=True) / (k * m2 ** 1.5)
            out["dh"] = dho
            if case["gated"]:
                out["dgate"] = dho * scale * w1 * y1 * gate * (1 - gate)
            if case["scaled"]:
                out["dscale"] = (dho * gate * w1 * y1).sum(0)
            dy1 = dho * scale * gate
            out["dpost_weight"] = (dy1 * y1).sum(0)
            t = dy1 * w1
            out["dy"] = t / m1.sqrt() - y * (t * y).sum(-1, keepdim=True) / (k * m1 ** 1.5)
            return out

        b, l, ch = case["batch"], case["length"], case["channels"]
        step = case["mode"] == "step"
        ends = _lengths(case, seed) if case["ragged"] else np.full(b, l)
        on = [torch.from_numpy(ends > t).cuda() for t in range(l)]

        if case["op"] == "conv":
            w = case["width"]
            x = d64["x"][:, None] if step else d64["x"]
            last = d64["state"] if case["state"] else x.new_zeros(b, w - 1, ch)
            wt, bias = d64["weight"], d64["bias"]
            y, kept = torch.zeros_like(x), last.clone()
            if train:
                dw, db, dx, dfirst = torch.zeros_like(wt), torch.zeros_like(bias), torch.zeros_like(x), torch.zeros_like(last)
            for i in range(b):                            # the sequence with its state in front, without its padding
                n = int(ends[i])
                rows = torch.cat([last[i], x[i, :n]])
                win = rows.unfold(0, w, 1) if n else rows.new_zeros(0, ch, w)      # [n, channels, width]
                val, slope = silu_and_slope((win * wt).sum(-1) + bias)
                y[i, :n] = val
                kept[i] = rows[n:]
                if train and n:
                    dp = d64["dy"][i, :n] * slope
                    db += dp.sum(0)
                    dw += (dp[..., None] * win).sum(0)
                    back = torch.zeros_like(rows)
                    for j in range(w):
                        back[j:j + n] += dp * wt[:, j]
                    dx[i, :n], dfirst[i] = back[w - 1:], back[:w - 1]
            if step:
                return {"y": y[:, 0], "state": kept}
            if not train:
                return {"y": y, "state": kept}
            out = {"y": y, "dbias": db, "dweight": dw, "dx": dx}
            if case["state"]:
                out["dstate"] = dfirst
            return out

        n, g = case["states"], case["groups"]
        u, raw = d64["u"], d64["dt"] + d64["dt_bias"]
        Bm, Cm, z = d64["B"], d64["C"], d64.get("z")
        if step:
            u, raw, Bm, Cm = u[:, None], raw[:, None], Bm[:, None], Cm[:, None]
            z = None if z is None else z[:, None]
        delta = torch.logaddexp(raw, torch.zeros_like(raw))
        A, Dv = d64["A"], d64["D"]
        h = d64["state"] if case["state"] else u.new_zeros(b, ch, n)
        group = torch.arange(ch, device="cuda") // (ch // g)
        hs, y = [h], torch.zeros_like(u)
        for t in range(l):
            new = torch.exp(delta[:, t, :, None] * A) * h + (delta[:, t] * u[:, t])[..., None] * Bm[:, t, group]
            h = torch.where(on[t][:, None, None], new, h) if case["ragged"] else new
            y[:, t] = (h * Cm[:, t, group]).sum(-1) + Dv * u[:, t]
            if train:
                hs.append(h)
        if z is None:
            val, slope = torch.ones_like(y), torch.zeros_like(y)
        else:
            val, slope = silu_and_slope(z)
        live = torch.stack(on, 1)[..., None]
        gated = torch.where(live, y * val, 0.0)
        if step:
            return {"y": gated[:, 0], "state": h}
        if not train:
            return {"y": gated, "state": h}
        out = {"y": gated}
        dout = torch.where(live, d64["dout"], 0.0)
        if z is not None:
            out["dz"] = dout * y * slope
        dy = dout * val
        du, dd = Dv * dy, torch.zeros_like(dy)
        dA, dB, dC = torch.zeros_like(A), torch.zeros_like(Bm), torch.zeros_like(Cm)
        back = torch.zeros_like(h)                         # the gradient of the state after token t
        for t in range(l - 1, -1, -1):
            keep = on[t][:, None, None]
            now = torch.where(keep, back + dy[:, t, :, None] * Cm[:, t, group], 0.0)
            decay = torch.exp(delta[:, t, :, None] * A)
            dC[:, t] = torch.where(keep, dy[:, t, :, None] * hs[t + 1], 0.0).view(b, g, ch // g, n).sum(2)
            dB[:, t] = (now * (delta[:, t] * u[:, t])[..., None]).view(b, g, ch // g, n).sum(2)
            along = (now * Bm[:, t, group]).sum(-1)
            through = now * hs[t] * decay
            dA += (through * delta[:, t, :, None]).sum(0)
            dd[:, t] = (through * A).sum(-1) + u[:, t] * along
            du[:, t] += delta[:, t] * along
            back = torch.where(keep, now * decay, back)
        ddt = dd * logistic(raw)
        out.update(du=torch.where(live, du, 0.0), ddt=ddt, dA=dA, dB=dB, dC=dC, dD=(dy * u).sum((0, 1)), ddt_bias=ddt.sum((0, 1)))
        if case["state"]:
            out["dstate"] = back
        return out
