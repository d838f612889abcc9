"""The convolution, the scan and the block norms against their definitions in float64 (ssm_reference.py), forward and backward, over
types, head layouts, lengths, masks and strides.

Tolerances.  An output is rounded once to its dtype: half a unit in the last place, at most 2^-8 (bfloat16: 8
significant bits), 2^-11 (float16: 11, with 2^-25 absolute for its denormals) or 2^-24 (float32) of the value.  Before that, everything is float32: a value that is a sum of k terms of
magnitude s carries at most k + 8 roundings of 2^-24 s, and a state after t tokens 4 t more, as each token multiplies by an exponential of
relative error 4 * 2^-24.  s is taken as the largest magnitude in the output, times 4 for terms that cancel; for the gradients
of the norms, whose terms cancel completely in rows of one column, as the largest term before that.  A gradient goes through two such chains."""
import pytest
import torch

import ssm_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
NAN = float("nan")


@pytest.fixture(scope="module")
def ops(pkg):
    return pkg.ssm_ops


def _close(name, got, want, terms, top=None):
    assert got.shape == want.shape, name
    want = want.detach().cpu()
    g = got.detach().double().cpu()
    assert torch.isfinite(g).all(), f"{name}: not finite"
    if top is None:
        top = float(want.abs().max()) if want.numel() else 0.0
    bound = HALF_ULP[got.dtype] * want.abs() * 1.0001 + 4 * top * terms * 2.0 ** -24
    if got.dtype == torch.float16:
        bound = bound + 2.0 ** -25
    worst = float(((g - want).abs() - bound).max()) if want.numel() else 0.0
    assert worst <= 0, f"{name}: {float((g - want).abs().max()):.3g} off, {worst:.3g} over the bound; largest value {top:.3g}"


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32, std=1.0, mean=0.0):
    return (torch.randn(*shape, generator=g) * std + mean).to(dtype)


def _wide(t):
    """The same values as a window of a wider tensor: rows that are contiguous but not adjacent, off a 16-byte boundary."""
    big = torch.full((*t.shape[:-1], t.shape[-1] + 5), NAN, dtype=t.dtype, device=t.device)
    big[..., 3:3 + t.shape[-1]] = t
    return big[..., 3:3 + t.shape[-1]]


def _lengths(kind, B, L):
    if kind == "full":
        return None
    return torch.tensor([0, L, (L + 1) // 2, max(L - 1, 0)] * B)[:B] if kind == "ragged" else torch.zeros(B, dtype=torch.int64)


def _poison(t, lengths):
    """NaN behind every sequence's end."""
    if lengths is not None:
        for b in range(t.shape[0]):
            t[b, int(lengths[b]):] = NAN
    return t


def _leaves(tensors, dtype=None):
    """(GPU leaves, float64 CPU leaves) of a dict of tensors, None kept."""
    gpu = {k: None if t is None else t.to(DEV).requires_grad_(True) for k, t in tensors.items()}
    ref = {k: None if t is None else t.detach().double().nan_to_num(0.0).requires_grad_(True) for k, t in tensors.items()}
    return gpu, ref


def _reference_grads(outs, inputs, douts):
    """Zeros where no token leads from an input to an output."""
    used = [(o, d) for o, d in zip(outs, douts) if o.requires_grad]
    got = torch.autograd.grad([o for o, _ in used], inputs, [d for _, d in used], allow_unused=True) if used else [None] * len(inputs)
    return [torch.zeros_like(i) if g is None else g for g, i in zip(got, inputs)]


# ---- convolution --------------------------------------------------------------------------------------------------------

CONV = [(1, 1, 8, 4), (2, 2, 64, 4), (2, 3, 16, 3), (3, 33, 40, 3), (1, 130, 257, 2), (4, 65, 1000, 4), (1, 700, 24, 4)]


def _conv_case(B, L, D, W, dtype, mask, state, bias=True, seed=0):
    g = _gen(B * 1000 + L * 10 + D + W + seed)
    lengths = _lengths(mask, B, L)
    t = dict(x=_poison(_randn(g, B, L, D, dtype=dtype), lengths), weight=_randn(g, D, W, std=0.5), bias=_randn(g, D) if bias else None,
             initial_state=_randn(g, B, W - 1, D, dtype=dtype) if state else None)
    dy, ds = _poison(_randn(g, B, L, D, dtype=dtype), lengths), _randn(g, B, W - 1, D, dtype=dtype)
    return t, lengths, dy, ds


def _check_conv(ops, t, lengths, dy, ds, silu, wide=False):
    B, L, D = t["x"].shape
    W = t["weight"].shape[1]
    gpu, ref = _leaves(t)
    x_in = gpu["x"]
    if wide:
        x_in = _wide(t["x"].to(DEV)).detach().requires_grad_(True)
        gpu["x"] = x_in
    dev_lengths = None if lengths is None else lengths.to(DEV)
    y, s = ops.causal_conv(x_in, gpu["weight"], gpu["bias"], "silu" if silu else None, gpu["initial_state"], dev_lengths, True)
    yr, sr = R.causal_conv(ref["x"], ref["weight"], ref["bias"], silu, ref["initial_state"], lengths)
    _close("y", y, yr, W + 8)
    assert torch.equal(s.double().cpu(), sr.detach()), "the state is a copy of inputs"
    names = [k for k, v in gpu.items() if v is not None]
    got = torch.autograd.grad((y, s), [gpu[k] for k in names], ((_wide if wide else lambda v: v)(dy.to(DEV)), ds.to(DEV)))
    want = _reference_grads((yr, sr), [ref[k] for k in names], (dy.double().nan_to_num(0.0), ds.double()))
    for k, a, b in zip(names, got, want):
        _close("d" + k, a, b, (B * L if k in ("weight", "bias") else W) + 16)
    return y, s, got


@pytest.mark.parametrize("mask", ["full", "ragged"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,L,D,W", CONV)
def test_conv_forward_and_gradients(ops, B, L, D, W, dtype, mask):
    _check_conv(ops, *_conv_case(B, L, D, W, dtype, mask, state=True), silu=True, wide=D % 2 == 0)


@pytest.mark.parametrize("state,bias,silu", [(False, True, True), (True, False, True), (True, True, False), (False, False, False)])
def test_conv_without_state_bias_or_activation(ops, state, bias, silu):
    _check_conv(ops, *_conv_case(2, 19, 48, 4, torch.float32, "ragged", state, bias), silu=silu)


def test_conv_of_empty_sequences_keeps_the_state(ops):
    t, lengths, dy, ds = _conv_case(2, 5, 16, 4, torch.float32, "empty", True)
    y, s, got = _check_conv(ops, t, lengths, dy, ds, True)
    assert not y.any() and torch.equal(s.cpu(), t["initial_state"])
    t, _, dy, ds = _conv_case(2, 0, 16, 4, torch.float32, "full", True)
    y, s = ops.causal_conv(t["x"].to(DEV), t["weight"].to(DEV), initial_state=t["initial_state"].to(DEV), return_final_state=True)
    assert y.shape == (2, 0, 16) and torch.equal(s.cpu(), t["initial_state"])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_conv_tokens_one_by_one_and_in_pieces_equal_the_whole(ops, dtype):
    """Each output is formed from the same inputs in the same order: the same bits."""
    t, *_ = _conv_case(3, 21, 72, 4, dtype, "full", True)
    d = {k: v.to(DEV) for k, v in t.items()}
    whole, last = ops.causal_conv(d["x"], d["weight"], d["bias"], initial_state=d["initial_state"], return_final_state=True)
    y1, s1 = ops.causal_conv(d["x"][:, :2], d["weight"], d["bias"], initial_state=d["initial_state"], return_final_state=True)
    y2, s2 = ops.causal_conv(d["x"][:, 2:], d["weight"], d["bias"], initial_state=s1, return_final_state=True)
    assert torch.equal(torch.cat([y1, y2], 1), whole) and torch.equal(s2, last)
    state, other = d["initial_state"].clone(), torch.empty_like(d["initial_state"])
    for i in range(21):
        kept = state.clone()
        y = ops.causal_conv_step(d["x"][:, i], state, d["weight"], d["bias"], state_out=other)
        assert torch.equal(state, kept)
        again = ops.causal_conv_step(d["x"][:, i], state, d["weight"], d["bias"])
        assert torch.equal(y, whole[:, i]) and torch.equal(y, again) and torch.equal(state, other)
    assert torch.equal(state, last)


# ---- scan ---------------------------------------------------------------------------------------------------------------

SCAN = [(1, 1, 32, 16, 1), (2, 17, 64, 16, 2), (1, 100, 96, 4, 1), (3, 40, 33, 12, 1), (2, 65, 60, 64, 3), (1, 129, 48, 32, 1), (4, 16, 8, 1, 4),
        (1, 300, 200, 16, 1), (2, 48, 40, 8, 2)]


def _scan_case(B, L, D, N, G, dtype, mask="full", state=True, gated=True, skip=True, bias=True, seed=0):
    g = _gen(B * 1000 + L * 10 + D + N + G + seed)
    lengths = _lengths(mask, B, L)
    step = torch.exp(torch.rand(D, generator=g) * 4.6 - 6.9)
    t = dict(u=_poison(_randn(g, B, L, D, dtype=dtype), lengths), dt=_poison(_randn(g, B, L, D, dtype=dtype, std=0.5), lengths),
             A=-torch.arange(1.0, N + 1) * torch.exp(0.1 * _randn(g, D, N)), B=_poison(_randn(g, B, L, G, N, dtype=dtype), lengths),
             C=_poison(_randn(g, B, L, G, N, dtype=dtype), lengths), D=_randn(g, D) if skip else None,
             z=_poison(_randn(g, B, L, D, dtype=dtype), lengths) if gated else None,
             dt_bias=step + torch.log(-torch.expm1(-step)) if bias else None, initial_state=_randn(g, B, D, N) if state else None)
    dy, ds = _poison(_randn(g, B, L, D, dtype=dtype), lengths), _randn(g, B, D, N)
    return t, lengths, dy, ds


def _check_scan(ops, t, lengths, dy, ds, softplus=True, wide=False):
    B, L, D = t["u"].shape
    N, G = t["A"].shape[1], t["B"].shape[2]
    gpu, ref = _leaves(t)
    if wide:
        for k in ("u", "dt", "z", "B", "C"):
            if t[k] is not None:
                gpu[k] = _wide(t[k].to(DEV)).detach().requires_grad_(True)
    dev_lengths = None if lengths is None else lengths.to(DEV, torch.int32)
    y, s = ops.selective_scan(**{k: v for k, v in gpu.items()}, dt_softplus=softplus, lengths=dev_lengths, return_final_state=True)
    yr, sr = R.selective_scan(**{k: v for k, v in ref.items()}, softplus=softplus, lengths=lengths)
    _close("y", y, yr, 4 * L + N + 16)
    _close("state", s, sr, 4 * L + 16)
    names = [k for k, v in gpu.items() if v is not None]
    got = torch.autograd.grad((y, s), [gpu[k] for k in names], ((_wide if wide else lambda v: v)(dy.to(DEV)), ds.to(DEV)))
    want = _reference_grads((yr, sr), [ref[k] for k in names], (dy.double().nan_to_num(0.0), ds.double()))
    terms = dict(A=B * L, D=B * L, dt_bias=B * L, B=D // G, C=D // G)
    for k, a, b in zip(names, got, want):
        _close("d" + k, a, b, 8 * L + 2 * N + 32 + terms.get(k, 0))
    return y, s, got


@pytest.mark.parametrize("mask", ["full", "ragged"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,L,D,N,G", SCAN)
def test_scan_forward_and_gradients(ops, B, L, D, N, G, dtype, mask):
    _check_scan(ops, *_scan_case(B, L, D, N, G, dtype, mask), wide=D % 16 == 0)


@pytest.mark.parametrize("state,gated,skip,bias,softplus", [(False, True, True, True, True), (True, False, True, True, True), (True, True, False, True, True),
                                                            (True, True, True, False, True), (False, False, False, False, True), (True, True, True, True, False)])
def test_scan_without_its_optional_parts(ops, state, gated, skip, bias, softplus):
    t, lengths, dy, ds = _scan_case(2, 37, 40, 16, 2, torch.float32, "ragged", state, gated, skip, bias)
    if not softplus:                      # then the step sizes are given as they are
        t["dt"], t["dt_bias"] = t["dt"].abs() * 0.1, torch.full_like(t["dt_bias"], 0.01)
    _check_scan(ops, t, lengths, dy, ds, softplus)


@pytest.mark.parametrize("B,L,D,N,G,mask", [(1, 2500, 64, 16, 1, "full"), (2, 1601, 24, 16, 2, "ragged"), (1, 1500, 20, 64, 1, "full")])
def test_scan_of_few_channels_over_many_tokens(ops, B, L, D, N, G, mask):
    """Sizes that leave most of the GPU without a channel of its own."""
    _check_scan(ops, *_scan_case(B, L, D, N, G, torch.float32, mask))
    _check_scan(ops, *_scan_case(B, L, D, N, G, torch.bfloat16, mask, state=False))


def test_scan_of_empty_sequences_keeps_the_state(ops):
    t, lengths, dy, ds = _scan_case(2, 5, 32, 16, 1, torch.float32, "empty")
    y, s, got = _check_scan(ops, t, lengths, dy, ds)
    assert not y.any() and torch.equal(s.cpu(), t["initial_state"])
    t, _, dy, ds = _scan_case(2, 0, 32, 16, 1, torch.float32)
    gpu = {k: v.to(DEV).requires_grad_(True) for k, v in t.items()}
    y, s = ops.selective_scan(**gpu, return_final_state=True)
    assert y.shape == (2, 0, 32) and torch.equal(s.detach().cpu(), t["initial_state"])
    grads = torch.autograd.grad(s, [gpu["initial_state"], gpu["A"]], ds.to(DEV))
    assert torch.equal(grads[0].cpu(), ds) and not grads[1].any()


@pytest.mark.parametrize("raw", [-90.0, -20.0, -5.0, 0.0, 19.0, 60.0])
def test_scan_step_sizes_over_the_whole_range(ops, raw):
    """delta from 8e-40 to 60: the logarithm keeps its relative precision, the exponential goes to 0 without a NaN."""
    t, lengths, dy, ds = _scan_case(1, 9, 32, 16, 1, torch.float32)
    t["dt"] = t["dt"] + raw
    t["dt_bias"] = None
    gpu, ref = _leaves(t)
    y, s = ops.selective_scan(**gpu, return_final_state=True)
    yr, sr = R.selective_scan(**ref)
    _close("y", y, yr, 4 * 9 + 32)
    _close("state", s, sr, 4 * 9 + 16)
    got = torch.autograd.grad((y, s), [gpu["dt"], gpu["A"]], (dy.to(DEV), ds.to(DEV)))
    want = torch.autograd.grad((yr, sr), [ref["dt"], ref["A"]], (dy.double(), ds.double()))
    for k, a, b in zip(("ddt", "dA"), got, want):
        _close(k, a, b, 8 * 9 + 64)


def test_scan_keeps_infinities_and_nan_of_real_tokens_where_they_are(ops):
    """A NaN in one channel's input reaches that channel from its token on, and nothing else."""
    t, *_ = _scan_case(2, 40, 64, 16, 1, torch.float32)
    d = {k: v.to(DEV) for k, v in t.items()}
    clean, _ = ops.selective_scan(**d, return_final_state=True)
    d["u"][1, 21, 5] = NAN
    d["dt"][0, 30, 40] = NAN
    y, s = ops.selective_scan(**d, return_final_state=True)
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[1, 21:, 5] = True
    bad[0, 30:, 40] = True
    assert torch.equal(torch.isnan(y), bad) and torch.equal(y[~bad], clean[~bad])
    assert torch.isnan(s).any(-1).sum() == 2


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N,G", [(16, 1), (12, 2), (64, 1), (3, 1)])
def test_scan_tokens_one_by_one_and_in_pieces_equal_the_whole(ops, dtype, N, G):
    t, *_ = _scan_case(3, 25, 72, N, G, dtype)
    d = {k: v.to(DEV) for k, v in t.items()}
    tok = ("u", "dt", "B", "C", "z")
    rest = {k: d[k] for k in ("A", "D", "dt_bias")}
    whole, last = ops.selective_scan(**d, return_final_state=True)
    y1, s1 = ops.selective_scan(**{k: d[k][:, :11] for k in tok}, **rest, initial_state=d["initial_state"], return_final_state=True)
    y2, s2 = ops.selective_scan(**{k: d[k][:, 11:] for k in tok}, **rest, initial_state=s1, return_final_state=True)
    both_rounded = 0 if dtype == torch.float32 else HALF_ULP[dtype] * 2 ** 24
    _close("pieces", torch.cat([y1, y2], 1), whole.double(), 4 * 25 + 32 + both_rounded)
    _close("state", s2, last.double(), 4 * 25 + 32)
    state, other = d["initial_state"].clone(), torch.empty_like(d["initial_state"])
    for i in range(25):
        kept = state.clone()
        y = ops.selective_scan_step(**{k: d[k][:, i] for k in tok}, **rest, state=state, state_out=other)
        assert torch.equal(state, kept)
        again = ops.selective_scan_step(**{k: d[k][:, i] for k in tok}, **rest, state=state)
        assert torch.equal(y, again) and torch.equal(state, other)
        _close("step", y, whole[:, i].double(), 4 * 25 + 32 + both_rounded)
    _close("last", state, last.double(), 4 * 25 + 32)


# ---- norms --------------------------------------------------------------------------------------------------------------

NORM = [(1, 8), (5, 41), (7, 1536), (3, 8200), (2, 16384), (300, 256), (1, 1), (400, 72), (2, 9001)]


def _norm_case(M, K, dtype, gated, scaled):
    g = _gen(M * 100 + K)
    t = dict(h=_randn(g, M, K, dtype=dtype, std=2.0), y=_randn(g, M, K, dtype=dtype, std=0.5), post_weight=_randn(g, K, mean=1.0, std=0.1),
             pre_weight=_randn(g, K, mean=1.0, std=0.1), gate=_randn(g, M, K, dtype=dtype) if gated else None,
             scale=_randn(g, K, std=0.3) if scaled else None)
    return t, _randn(g, M, K, dtype=dtype), _randn(g, M, K, dtype=dtype)


def _norm_terms(ref, da, db, eps=1e-6):
    """The largest term of each gradient, before terms cancel."""
    with torch.no_grad():
        h, y, w1, w2 = (ref[k] for k in ("h", "y", "post_weight", "pre_weight"))
        f = torch.ones_like(y) if ref["gate"] is None else torch.sigmoid(ref["gate"])
        s = torch.ones_like(w1) if ref["scale"] is None else ref["scale"].abs()
        r1 = (y.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
        p = (w1 * y * r1).abs()
        out = h + torch.sign(ref["scale"] if ref["scale"] is not None else s) * s * f * w1 * y * r1
        r2 = (out.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
        d = da.abs() + r2 * (db * w2).abs()
        terms = {"h": d, "y": d * s * f * w1.abs() * r1, "gate": d * s * p, "scale": (d * f * p).sum(0), "post_weight": (d * s * f * (y * r1).abs()).sum(0),
                 "pre_weight": (db * out * r2).abs().sum(0)}
    return {k: float(v.max()) for k, v in terms.items()}


def _check_norm(ops, t, da, db, wide=False):
    M, K = t["h"].shape
    gpu, ref = _leaves(t)
    if wide:
        for k in ("h", "y", "gate"):
            if t[k] is not None:
                gpu[k] = _wide(t[k].to(DEV)).detach().requires_grad_(True)
    out = ops.block_norm(**gpu)
    want_out = R.block_norm(ref["h"], ref["y"], ref["post_weight"], ref["pre_weight"], ref["gate"], ref["scale"])
    for k, a, b in zip(("h_out", "normed"), out, want_out):
        _close(k, a, b, 24)
    names = [k for k, v in gpu.items() if v is not None]
    got = torch.autograd.grad(out, [gpu[k] for k in names], (da.to(DEV), db.to(DEV)), retain_graph=True)
    want = torch.autograd.grad(want_out, [ref[k] for k in names], (da.double(), db.double()), retain_graph=True)
    top = _norm_terms(ref, da.double(), db.double())
    for k, a, b in zip(names, got, want):
        _close("d" + k, a, b, 32 + M + 2 * K ** 0.5, top[k])
    for i in (0, 1):                                     # the gradient of one output alone
        got = torch.autograd.grad(out[i], [gpu[k] for k in names], (da, db)[i].to(DEV), retain_graph=True, allow_unused=True)
        want = torch.autograd.grad(want_out[i], [ref[k] for k in names], (da, db)[i].double(), retain_graph=True, allow_unused=True)
        for k, a, b in zip(names, got, want):
            _close("d" + k, a, torch.zeros(a.shape, dtype=torch.float64) if b is None else b, 32 + M + 2 * K ** 0.5, top[k])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,K", NORM)
def test_norm_forward_and_gradients(ops, M, K, dtype):
    _check_norm(ops, *_norm_case(M, K, dtype, True, True), wide=M == 7)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,K", [(3, 4088), (160, 4096), (3, 4095), (2, 4104), (2, 8192), (1, 8193)])
def test_norm_where_the_kernels_change(ops, M, K, dtype):
    """Rows of up to 4096, 8192 and 16384 columns run differently."""
    _check_norm(ops, *_norm_case(M, K, dtype, True, True))


@pytest.mark.parametrize("gated,scaled", [(False, True), (True, False), (False, False)])
def test_norm_without_gate_or_scale(ops, gated, scaled):
    _check_norm(ops, *_norm_case(33, 200, torch.float32, gated, scaled))


def test_norm_of_no_rows_and_of_zero_rows(ops):
    t, da, db = _norm_case(4, 64, torch.float32, True, True)
    t["y"][1], t["h"][1], t["h"][2] = 0.0, 0.0, 0.0
    _check_norm(ops, t, da, db)
    gpu = {k: (v[:0] if v.dim() == 2 else v).to(DEV).requires_grad_(True) for k, v in t.items()}
    a, b = ops.block_norm(**gpu)
    assert a.shape == b.shape == (0, 64)
    for g in torch.autograd.grad((a, b), [gpu["post_weight"], gpu["pre_weight"], gpu["scale"]], (da[:0].to(DEV), db[:0].to(DEV))):
        assert not g.any()


# ---- what they share ----------------------------------------------------------------------------------------------------

def _three(ops, dtype=torch.float32, seed=0):
    """(call, inputs, output gradients) of each operator on one small case."""
    ct, _, cdy, cds = _conv_case(2, 29, 40, 4, dtype, "full", True, seed=seed)
    st, _, sdy, sds = _scan_case(2, 29, 40, 16, 2, dtype, seed=seed)
    nt, da, db = _norm_case(13, 88, dtype, True, True)
    return {
        "conv": (lambda **k: ops.causal_conv(**k, return_final_state=True), ct, (cdy, cds)),
        "scan": (lambda **k: ops.selective_scan(**k, return_final_state=True), st, (sdy, sds)),
        "norm": (lambda **k: ops.block_norm(**k), nt, (da, db)),
    }


@pytest.mark.parametrize("name", ["conv", "scan", "norm"])
def test_gradients_against_differences(ops, name):
    """Along the gradient's own direction v of unit length, (f(x + e v) - f(x - e v)) / 2 e is |gradient| up to e^2 times a third derivative
    (e = 0.05 spread over all elements: below 1e-3 of it) and the roundings of f, 2^-22 of sum |dy y| each."""
    call, t, douts = _three(ops)[name]
    gpu = {k: v.to(DEV).requires_grad_(True) for k, v in t.items()}
    douts = [d.to(DEV) for d in douts]
    outs = call(**gpu)
    grads = dict(zip(gpu, torch.autograd.grad(outs, list(gpu.values()), douts)))

    def f(inputs):
        with torch.no_grad():
            return sum(float((o.double() * d.double()).sum()) for o, d in zip(call(**inputs), douts))

    rounding = 2.0 ** -22 * sum(float((o.detach().double() * d.double()).abs().sum()) for o, d in zip(outs, douts))
    for k, g in grads.items():
        n = float(g.norm())
        e = 0.05
        at = {j: v.detach() for j, v in gpu.items()}
        v = g / n
        fd = (f({**at, k: at[k] + e * v}) - f({**at, k: at[k] - e * v})) / (2 * e)
        assert abs(fd - n) <= 1e-3 * n + rounding / e, (k, fd, n)


@pytest.mark.parametrize("name", ["conv", "scan", "norm"])
def test_the_same_call_gives_the_same_bits_on_any_stream(ops, name):
    call, t, douts = _three(ops, torch.bfloat16)[name]
    gpu = {k: v.to(DEV).requires_grad_(True) for k, v in t.items()}
    douts = [d.to(DEV) for d in douts]

    def both():
        outs = call(**gpu)
        return [*outs, *torch.autograd.grad(outs, list(gpu.values()), douts)]

    first = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        busy = torch.randn(2048, 2048, device=DEV)
        for _ in range(20):
            busy = busy @ busy * 1e-3
        second = both()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, second):
        assert torch.equal(a, b)


@pytest.mark.parametrize("name", ["conv", "scan", "norm"])
def test_operators_can_be_recorded_in_a_graph(ops, name):
    call, t, _ = _three(ops, torch.bfloat16)[name]
    gpu = {k: v.to(DEV) for k, v in t.items()}
    with torch.no_grad():
        want = call(**gpu)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = call(**gpu)
        graph.replay()
    for a, b in zip(want, got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("name", ["conv", "scan", "norm"])
def test_each_gradient_alone_is_the_one_of_all(ops, name):
    """Whatever else needs no gradient, and whichever output has one."""
    call, t, douts = _three(ops)[name]
    douts = [d.to(DEV) for d in douts]
    gpu = {k: v.to(DEV).requires_grad_(True) for k, v in t.items()}
    whole = dict(zip(gpu, torch.autograd.grad(call(**gpu), list(gpu.values()), douts)))
    for k in gpu:
        alone = {j: v.detach() for j, v in gpu.items()}
        alone[k].requires_grad_(True)
        outs = call(**alone)
        assert torch.equal(torch.autograd.grad(outs, alone[k], douts, retain_graph=True)[0], whole[k]), k
        parts = [torch.autograd.grad(o, alone[k], d, retain_graph=True, allow_unused=True)[0] for o, d in zip(outs, douts)]
        total = sum(p.double() for p in parts if p is not None)
        assert float((total - whole[k].double()).norm()) <= 1e-5 * float(sum(p.double().norm() for p in parts if p is not None)) + 1e-30, k


@pytest.mark.parametrize("name", ["conv", "scan", "norm"])
def test_no_sequences_at_all(ops, name):
    call, t, douts = _three(ops)[name]
    lead = {"conv": ("x", "initial_state"), "scan": ("u", "dt", "B", "C", "z", "initial_state"), "norm": ("h", "y", "gate")}[name]
    gpu = {k: (v[:0] if k in lead else v).to(DEV).requires_grad_(True) for k, v in t.items()}
    outs = call(**gpu)
    assert all(o.numel() == 0 for o in outs)
    for k, g in zip(gpu, torch.autograd.grad(outs, list(gpu.values()), [d[:0].to(DEV) for d in douts])):
        assert g.shape == gpu[k].shape and not g.any(), k


def test_second_derivatives_are_refused(ops):
    call, t, douts = _three(ops)["norm"]
    gpu = {k: v.to(DEV).requires_grad_(True) for k, v in t.items()}
    g = torch.autograd.grad(call(**gpu), gpu["h"], [d.to(DEV) for d in douts], create_graph=True)[0]
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_offsets_beyond_32_bits(ops):
    """Windows of a tensor whose last rows lie more than 2^31 elements behind the first."""
    L, pitch, D = 140000, 16384, 32
    big = torch.empty(L, pitch, dtype=torch.bfloat16, device=DEV)
    g = _gen(3)
    x = _randn(g, 1, L, D, dtype=torch.bfloat16).to(DEV)
    window = big[None, :, 8000:8000 + D]
    window.copy_(x)
    w = _randn(g, D, 4).to(DEV)
    assert torch.equal(ops.causal_conv(window, w), ops.causal_conv(x, w))
    dt = _randn(g, 1, L, D, dtype=torch.bfloat16).to(DEV) - 4
    A = -torch.rand(D, 16, generator=g).to(DEV) - 0.1
    bc = _randn(g, 1, L, 16, dtype=torch.bfloat16).to(DEV)
    assert torch.equal(ops.selective_scan(window, dt, A, bc, bc, z=window), ops.selective_scan(x, dt, A, bc, bc, z=x))
    h = big[:, 8000:8000 + D]
    ones = torch.ones(D, device=DEV)
    for a, b in zip(ops.block_norm(h, h, ones, ones), ops.block_norm(x[0], x[0], ones, ones)):
        assert torch.equal(a, b)


def test_broadcast_inputs_get_summed_gradients(ops):
    """B and C of one group expanded over two batches: autograd adds the gradients of the copies."""
    t, _, dy, _ = _scan_case(2, 20, 32, 16, 1, torch.float32)
    b = t["B"][:1].to(DEV).requires_grad_(True)
    br = t["B"][:1].double().requires_grad_(True)
    d = {k: v.to(DEV) for k, v in t.items() if k != "B"}
    r = {k: v.double() for k, v in t.items() if k != "B"}
    y = ops.selective_scan(**d, B=b.expand(2, -1, -1, -1))
    yr, _ = R.selective_scan(**r, B=br.expand(2, -1, -1, -1))
    _close("dB", torch.autograd.grad(y, b, dy.to(DEV))[0], torch.autograd.grad(yr, br, dy.double())[0], 8 * 20 + 32 + 64)


def _refusals(ops):
    f = torch.zeros
    x, w = f(2, 5, 16, device=DEV), f(16, 4, device=DEV)
    u, A, bc, st = f(2, 5, 16, device=DEV), f(16, 8, device=DEV), f(2, 5, 8, device=DEV), f(2, 16, 8, device=DEV)
    h, k = f(3, 16, device=DEV), f(16, device=DEV)
    cs = f(2, 3, 16, device=DEV)
    return {
        "conv: x on the CPU": (lambda: ops.causal_conv(x.cpu(), w), "x must be a CUDA tensor"),
        "conv: x of two dimensions": (lambda: ops.causal_conv(x[0], w), "x must be"),
        "conv: integers": (lambda: ops.causal_conv(x.int(), w), "float16, bfloat16 or float32"),
        "conv: width 5": (lambda: ops.causal_conv(x, f(16, 5, device=DEV)), "width of 2, 3 or 4"),
        "conv: weight of other channels": (lambda: ops.causal_conv(x, f(15, 4, device=DEV)), "weight must have shape"),
        "conv: half weight": (lambda: ops.causal_conv(x, w.half()), "weight must be Float"),
        "conv: activation": (lambda: ops.causal_conv(x, w, activation="relu"), "activation must be"),
        "conv: state of another dtype": (lambda: ops.causal_conv(x, w, initial_state=cs.half()), "initial_state must be Float"),
        "conv: lengths of another batch": (lambda: ops.causal_conv(x, w, lengths=f(3, dtype=torch.int32, device=DEV)), "one entry per sequence"),
        "conv: float lengths": (lambda: ops.causal_conv(x, w, lengths=f(2, device=DEV)), "int32 or int64"),
        "conv step: state shape": (lambda: ops.causal_conv_step(x[:, 0], f(2, 4, 16, device=DEV), w), "state must have shape"),
        "conv step: state not dense": (lambda: ops.causal_conv_step(x[:, 0], f(2, 16, 3, device=DEV).mT, w), "state must be contiguous"),
        "conv step: overlap": (lambda: _overlapping(ops, x, w), "overlaps"),
        "conv step: gradient": (lambda: ops.causal_conv_step(x[:, 0].clone().requires_grad_(True), cs, w), "no gradient"),
        "scan: dt of another dtype": (lambda: ops.selective_scan(u, u.half(), A, bc, bc), "dt has another dtype"),
        "scan: dt of another shape": (lambda: ops.selective_scan(u, u[:, :4], A, bc, bc), "dt must have shape"),
        "scan: 65 states": (lambda: ops.selective_scan(u, u, f(16, 65, device=DEV), f(2, 5, 65, device=DEV), f(2, 5, 65, device=DEV)), "1 to 64 states"),
        "scan: groups": (lambda: ops.selective_scan(u, u, A, f(2, 5, 3, 8, device=DEV), f(2, 5, 3, 8, device=DEV)), "multiple of B's groups"),
        "scan: C unlike B": (lambda: ops.selective_scan(u, u, A, bc, f(2, 5, 2, 8, device=DEV)), "C must have shape"),
        "scan: A half": (lambda: ops.selective_scan(u, u, A.half(), bc, bc), "A must be Float"),
        "scan: state": (lambda: ops.selective_scan(u, u, A, bc, bc, initial_state=st[:1]), "initial_state must have shape"),
        "scan step: half state": (lambda: ops.selective_scan_step(u[:, 0], u[:, 0], A, bc[:, 0], bc[:, 0], st.half()), "state must be Float"),
        "scan step: state_out": (lambda: ops.selective_scan_step(u[:, 0], u[:, 0], A, bc[:, 0], bc[:, 0], st, state_out=st[:1]), "like state"),
        "norm: y of another shape": (lambda: ops.block_norm(h, h[:2], k, k), "y must have the shape"),
        "norm: gate of another dtype": (lambda: ops.block_norm(h, h, k, k, gate=h.half()), "gate must have the shape and dtype"),
        "norm: weight": (lambda: ops.block_norm(h, h, k[:8], k), "post_weight must have shape"),
        "norm: too wide": (lambda: ops.block_norm(f(1, 16392, device=DEV), f(1, 16392, device=DEV), f(16392, device=DEV), f(16392, device=DEV)), "16384"),
        "norm: eps": (lambda: ops.block_norm(h, h, k, k, eps=-1.0), "eps must not be negative"),
    }


def _overlapping(ops, x, w):
    buf = torch.zeros(64, device=DEV)
    return ops.causal_conv_step(x[:1, 0], buf[:48].view(1, 3, 16), w, state_out=buf[16:64].view(1, 3, 16))


REFUSED = sorted(_refusals(None)) if torch.cuda.is_available() else ["(needs a GPU)"]


@pytest.mark.parametrize("name", REFUSED)
def test_bad_arguments_are_refused(ops, name):
    call, message = _refusals(ops)[name]
    with pytest.raises(RuntimeError, match=message):
        call()
