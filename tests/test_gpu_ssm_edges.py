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


def test_scan_step_of_states_that_forget_at_once(ops):
    t, *_ = _scan_case(2, 1, 32, 16, 1, torch.float32)
    t["A"][3, 2], t["A"][:, 7], t["A"][5] = -INF, -INF, -3e38
    d = {k: v.to(DEV) for k, v in t.items()}
    whole, last = ops.selective_scan(**d, return_final_state=True)
    y = ops.selective_scan_step(**{k: d[k][:, 0] for k in ("u", "dt", "B", "C", "z")}, A=d["A"], D=d["D"], dt_bias=d["dt_bias"], state=d["initial_state"])
    _close("y", y, whole[:, 0].double(), 4 + 32)
    _close("state", d["initial_state"], last.double(), 4 + 16)


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


# ---- loops that only larger sizes reach -----------------------------------------------------------------------------------

def _sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


def _plan(pkg, name, ints):
    """A workspace size, which shows how a call is cut up: leading fields of its struct, all pointers null."""
    buf = (ctypes.c_int32 * 160)()
    for i, v in enumerate(ints):
        buf[i] = v
    return getattr(pkg._lib.lib(), name)(buf)


@pytest.mark.parametrize("B,L,D,W,dtype,ragged,strip", [(1, 517, 7400, 4, torch.bfloat16, False, 16), (3, 1999, 1504, 4, torch.float16, True, 32),
                                                        (2, 1001, 7607, 3, torch.bfloat16, True, 64), (4, 1024, 8192, 4, torch.bfloat16, False, 128),
                                                        (2, 1024, 8192, 2, torch.float32, True, 64)])
def test_conv_where_a_strip_is_longer_than_its_slots(pkg, ops, B, L, D, W, dtype, ragged, strip):
    """A thread's slots hold 8 tokens: strips of 16 to 128 go round them."""
    if _sms() == 148:
        blocks = -(-L // (8 * strip))
        assert _plan(pkg, "el_causal_conv_backward_workspace_bytes", [pkg._lib.EL_BF16, B, L, D, W]) == B * blocks * (W + 1) * D * 4
    _check_conv_at_once(ops, B, L, D, W, dtype, ragged)


def _scan_reference(u, dt, A, B, C, D, z, dt_bias, initial_state, lengths):
    """(y, final state), token by token for all sequences at once."""
    nb, L, ch = u.shape
    G, h, ys = B.shape[2], initial_state, []
    steps = [v.unbind(1) for v in (u, F.softplus(dt + dt_bias, threshold=1e9), B, C, z)]
    for i, (ut, delta, Bt, Ct, zt) in enumerate(zip(*steps)):
        Bt, Ct = (m.repeat_interleave(ch // G, 1) for m in (Bt, Ct))
        new = torch.exp(delta[..., None] * A) * h + (delta * ut)[..., None] * Bt
        on = (i < lengths)[:, None]
        y = (new * Ct).sum(-1) + D * ut
        ys.append(torch.where(on, y * F.silu(zt), 0.0))
        h = torch.where(on[..., None], new, h)
    return torch.stack(ys, 1), h


@pytest.mark.parametrize("B,L,D,N,G,dtype,ragged", [(4, 300, 7168, 16, 1, torch.bfloat16, False), (4, 277, 7184, 16, 2, torch.float32, True),
                                                    (2, 290, 1800, 64, 1, torch.float32, True)])
def test_scan_backward_of_many_tiles_in_one_piece(pkg, ops, B, L, D, N, G, dtype, ragged):
    """So many channels that the sequences are not cut: a warp takes more than the 16 tiles after which its sums over tokens go to memory."""
    lanes = max(N // 4, 1)
    width = 8 * 64 // lanes                                # channels of a block's eight warps
    blocks = -(-(D // G) // width)
    if _sms() == 148:
        assert _plan(pkg, "el_selective_scan_backward_workspace_bytes", [pkg._lib.EL_BF16, B, L, D, G, N]) == 4 * (2 * blocks * B * L * G * N + B * D * (N + 2))
    assert L > 2 * 128
    t, _, dy, ds = _scan_case(B, L, D, N, G, dtype)
    lengths = torch.tensor([L, 0, L - 3, 130][:B]) if ragged else torch.full((B,), L)
    dev = {k: v.to(DEV) for k, v in t.items()}
    dy, ds = dy.to(DEV), ds.to(DEV)
    ref = {k: v.double().requires_grad_(True) for k, v in dev.items()}
    yr, sr = _scan_reference(**ref, lengths=lengths.to(DEV))
    want = torch.autograd.grad((yr, sr), list(ref.values()), (dy.double(), ds.double()))
    yr, sr = yr.detach(), sr.detach()
    for v in [dev[k] for k in ("u", "dt", "z", "B", "C")] + [dy]:
        _poison(v, lengths)
    gpu = {k: v.requires_grad_(True) for k, v in dev.items()}
    y, s = ops.selective_scan(**gpu, lengths=lengths.to(DEV) if ragged else None, return_final_state=True)
    _close("y", y, yr, 4 * L + N + 16)
    _close("state", s, sr, 4 * L + 16)
    got = torch.autograd.grad((y, s), list(gpu.values()), (dy, ds))
    terms = dict(A=B * L, D=B * L, dt_bias=B * L, B=D // G, C=D // G)
    for k, a, b in zip(gpu, got, want):
        _close("d" + k, a, b, 8 * L + 2 * N + 32 + terms.get(k, 0))


@pytest.mark.parametrize("B,D,N,G,dtype", [(64, 8192, 16, 1, torch.bfloat16), (61, 8190, 16, 2, torch.float32), (100, 4100, 12, 1, torch.float16),
                                           (33, 2056, 64, 4, torch.bfloat16)])
def test_scan_step_of_blocks_that_take_several_sequences(ops, B, D, N, G, dtype):
    """In place and beside the old state; a block goes through its sequences with the next one's state under way."""
    lanes = max(1, 1 << (N - 1).bit_length() >> 2)
    assert -(-D * lanes // 128) * B // (16 * _sms()) >= 2
    t, *_ = _scan_case(B, 1, D, N, G, dtype)
    d = {k: v.to(DEV) for k, v in t.items()}
    tok = {k: d[k][:, 0] for k in ("u", "dt", "B", "C", "z")}
    rest = {k: d[k] for k in ("A", "D", "dt_bias")}
    yr, sr = _scan_reference(**{k: v.double() for k, v in d.items()}, lengths=torch.ones(B, device=DEV))
    old, other = d["initial_state"].clone(), torch.full_like(d["initial_state"], NAN)
    y = ops.selective_scan_step(**tok, **rest, state=old, state_out=other)
    assert torch.equal(old, d["initial_state"])
    _close("y", y, yr[:, 0], 4 + N + 16)
    _close("state", other, sr, 4 + 16)
    again = ops.selective_scan_step(**tok, **rest, state=old)
    assert torch.equal(again, y) and torch.equal(old, other)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,K", [(700, 4096), (5000, 256), (400, 4095), (400, 8200), (500, 16384), (600, 8192)])
def test_norm_of_blocks_that_take_several_rows(ops, M, K, dtype):
    """Rows in plenty: the next row fetched while this one is worked on, the sums' buffers in turn, column sums over a block's rows."""
    threads = -(-(-(-K // 8)) // 32) * 32                  # of a row's block, 16-bit types; two blocks an SM where it has 512
    assert M > _sms() * (max(1024 // threads, 1) if K <= 4096 else 1)
    _check_norm(ops, *_norm_case(M, K, dtype, True, True))


# ---- step sizes -----------------------------------------------------------------------------------------------------------

def test_relative_error_of_step_sizes(ops):
    """From a state of zero, with u, B and C of one, the first y is the step size itself.  The exponential: a product with log2(e) rounded to 2^-24 and
    log2(e) to 1.4e-8, both of the exponent, 7.3e-8 |x|, and two units in the last place, 2^-22.  The logarithm's series: its argument e / (2 + e) with an addition, a reciprocal of
    one unit in the last place and a product, 2^-24 + 2^-23 + 2^-24; its sum 2^-24 twice and 1.4e-8 for the terms left out; the largest together 4.1e-7.
    Below 2^-126 two units of 2^-149."""
    x = torch.cat([torch.linspace(-100, 30, 4001), torch.linspace(-8, 1, 4001)])
    one = torch.ones(1, 1, 1, device=DEV)
    y = ops.selective_scan(one.expand(1, 1, len(x)), x[None, None].to(DEV), -torch.ones(len(x), 1, device=DEV), one, one)
    want = F.softplus(x.double(), threshold=1e9)
    off = (y[0, 0].double().cpu() - want).abs()
    assert bool((off <= want * (7.3e-8 * x.double().abs() + 2.0 ** -22 + 4.1e-7) + 2 * 2.0 ** -149).all()), float((off / want).max())


# ---- gradients that nobody asked for ----------------------------------------------------------------------------------------

def _peak(f):
    """Bytes that a call asks for beyond what was there before it."""
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_stats()["requested_bytes.all.current"]
    result = f()
    torch.cuda.synchronize()
    return torch.cuda.memory_stats()["requested_bytes.all.peak"] - before, result


@pytest.mark.parametrize("K", [2048, 8192])
def test_norm_backward_forms_what_is_wanted(ops, K):
    """A frozen norm over one input that has a gradient: one output, no partial sums; and the same bits as beside all others."""
    t, da, db = _norm_case(512, K, torch.bfloat16, True, True)
    gpu = {k: v.to(DEV).requires_grad_(True) for k, v in t.items()}
    douts = (da.to(DEV), db.to(DEV))
    whole = dict(zip(gpu, torch.autograd.grad(ops.block_norm(**gpu), list(gpu.values()), douts)))
    for k in gpu:
        alone = {j: v.detach().requires_grad_(j == k) for j, v in gpu.items()}
        outs = ops.block_norm(**alone)
        bytes_, (g,) = _peak(lambda: torch.autograd.grad(outs, alone[k], douts))
        assert torch.equal(g, whole[k]), k
        if g.dim() == 2:
            assert bytes_ <= g.numel() * 2 + 4096, (k, bytes_)


def test_scan_backward_keeps_no_room_for_what_is_not_wanted(pkg, ops):
    """B and C without a gradient: the partial sums of dB and dC, 2 x 8 blocks of channels x batch x length x states floats here, have no place."""
    t, _, dy, _ = _scan_case(2, 200, 1024, 16, 1, torch.float32)
    gpu = {k: v.to(DEV).requires_grad_(True) for k, v in t.items()}
    dy = dy.to(DEV)
    whole = dict(zip(gpu, torch.autograd.grad(ops.selective_scan(**gpu), list(gpu.values()), dy)))
    partial = 2 * 8 * 2 * 200 * 16 * 4
    sizes = {}
    for k in gpu:
        alone = {j: v.detach().requires_grad_(j == k) for j, v in gpu.items()}
        y = ops.selective_scan(**alone)
        sizes[k], (g,) = _peak(lambda: torch.autograd.grad(y, alone[k], dy))
        assert torch.equal(g, whole[k]), k
        sizes[k] -= g.numel() * 4
    assert abs(sizes["B"] - sizes["A"] - partial) <= 4096 and abs(sizes["C"] - sizes["B"]) <= 4096
    assert all(abs(v - sizes["A"]) <= 4096 for k, v in sizes.items() if k not in "BC"), sizes


# ---- nothing to add up ------------------------------------------------------------------------------------------------------

def test_gradients_of_no_channels_are_zeros(ops):
    """dB and dC are sums over the channels: of none of them, zeros, whatever the memory held before."""
    t, *_ = _scan_case(2, 9, 8, 4, 2, torch.float32)
    gpu = {k: (v[..., :0] if k in ("u", "dt", "z", "D", "dt_bias") else v[:0] if k == "A" else v[:, :0] if k == "initial_state" else v).to(DEV).requires_grad_(True)
           for k, v in t.items()}
    y, s = ops.selective_scan(**gpu, return_final_state=True)
    assert y.shape == (2, 9, 0) and s.shape == (2, 0, 4)
    for _ in range(2):
        junk = [torch.full((2, 9, 2, 4), NAN, device=DEV) for _ in range(8)]
        del junk
        for k, g in zip(gpu, torch.autograd.grad((y, s), list(gpu.values()), (torch.zeros_like(y), torch.zeros_like(s)), retain_graph=True)):
            assert g.shape == gpu[k].shape and not g.any(), k
