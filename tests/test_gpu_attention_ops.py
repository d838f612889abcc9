"""Rotation, latent attention in its expanded and absorbed forms and the cache of latent vectors against their definitions in float64
(attention_reference.py, which also derives the bounds), over types, head sizes, lengths, masks and strides."""
import pytest
import torch

import attention_reference as R
from oracle import int2_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
NAN = float("nan")
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def ops(pkg):
    return pkg.attention_ops


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(g, *shape, dtype=F32, std=1.0):
    return (torch.randn(*shape, generator=g) * std).to(dtype)


def _close(name, got, want, bound):
    assert got.shape == want.shape, f"{name}: {tuple(got.shape)}, not {tuple(want.shape)}"
    g = got.detach().double().cpu()
    assert torch.isfinite(g).all(), f"{name}: not finite"
    over = (g - want).abs() - bound * 1.0001
    assert not over.numel() or float(over.max()) <= 0, f"{name}: {float((g - want).abs().max()):.3g} off, {float(over.max()):.3g} over the bound"


def _wide(t, by=8, at=0):
    """The same values as a window of a wider tensor."""
    big = torch.full((*t.shape[:-1], t.shape[-1] + by), NAN, dtype=t.dtype, device=t.device)
    big[..., at:at + t.shape[-1]] = t
    return big[..., at:at + t.shape[-1]]


# ---- rotation -----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("shape,neighbours,positions", [
    ((2, 5, 3, 64), False, None), ((2, 5, 3, 64), True, "first"), ((3, 7, 16), False, "each"), ((1, 1, 1, 2), False, None), ((2, 3, 2, 10), True, "each"),
    ((1, 300, 4, 128), False, "first"), ((2, 0, 4, 32), False, None)])
def test_rotary(ops, dtype, shape, neighbours, positions):
    g = _gen(1)
    x, dim, B, T = _randn(g, *shape, dtype=dtype), shape[-1], shape[0], shape[1]
    table = ops.rotary_table(900, dim, device=DEV)
    at = torch.arange(T).expand(B, T)
    pos = None
    if positions == "first":
        pos = torch.tensor([500, 0, 7][:B], dtype=torch.int32)
        at = at + pos[:, None]
    elif positions == "each":
        pos = torch.randint(-3, 910, (B, T), generator=g)
        at = pos
    at = at.clamp(0, 899)
    xs = _wide(x.to(DEV)).detach().requires_grad_(True)
    y = ops.rotary(xs, table, None if pos is None else pos.to(DEV), neighbours)
    rows = at if x.dim() == 3 else at[..., None].expand(*shape[:3])
    want = R.rotate(x.double(), table.cpu(), rows, neighbours)
    size = R.rotate(x.double().abs(), torch.cat([table[:, :dim // 2].abs(), -table[:, dim // 2:].abs()], -1).cpu(), rows, neighbours).abs() \
        + R.rotate(x.double().abs(), table.cpu().abs(), rows, neighbours).abs()
    unit, tiny = R.UNIT[dtype], R.TINY[dtype]
    _close("y", y, want, 4 * R.E * size + unit * want.abs() + tiny)
    dy = _randn(g, *shape, dtype=dtype)
    dx, = torch.autograd.grad(y, xs, dy.to(DEV))
    back = torch.cat([table[:, :dim // 2], -table[:, dim // 2:]], -1).cpu()
    want = R.rotate(dy.double(), back, rows, neighbours)
    _close("dx", dx, want, 16 * R.E * dy.double().abs().amax() * torch.ones_like(want) + unit * want.abs() + tiny if want.numel() else want)


def test_rotary_table_of_far_positions(ops):
    t = ops.rotary_table(200001, 64, device=DEV).cpu()
    want = 200000 * 10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    # half a unit of float32, and the angle's own rounding in float64
    assert float((t[-1] - torch.cat([want.cos(), want.sin()])).abs().max()) < 2.0 ** -24 + 1e-9


# ---- the expanded form --------------------------------------------------------------------------------------------------

# batch, length, keys, heads, key_dim, rot_dim, value_dim
SHAPES = [(1, 1, 1, 1, 64, 0, 64), (2, 1, 200, 3, 128, 64, 128), (2, 130, 130, 2, 128, 64, 128), (1, 257, 257, 2, 64, 32, 64), (3, 77, 301, 2, 96, 0, 80),
          (1, 129, 513, 1, 128, 0, 128), (2, 64, 64, 5, 16, 16, 16), (1, 300, 300, 1, 112, 48, 96), (2, 33, 65, 2, 40, 24, 56), (1, 70, 70, 2, 200, 56, 256),
          (1, 20, 20, 3, 7, 1, 5), (1, 640, 640, 1, 128, 64, 64)]


def _inputs(seed, shape, dtype, std=1.2):
    B, T, S, H, D, P, V = shape
    g = _gen(seed)
    q, kv = _randn(g, B, T, H, D, dtype=dtype, std=std), _randn(g, B, S, H * (D + V), dtype=dtype, std=std)
    qr, kr = (_randn(g, B, T, H, P, dtype=dtype, std=std), _randn(g, B, S, P, dtype=dtype, std=std)) if P else (None, None)
    return g, q, kv, qr, kr


def _lengths(kind, B, T, S):
    if kind == "full":
        return None, None
    ln = torch.tensor([T, 0, (T + 1) // 2, 1] * B)[:B]
    return ln, (torch.tensor([S, S - T, max(S - T + (T + 1) // 2 - 1, 0), 1] * B)[:B] if kind == "uneven" else S - T + ln)


def _poison(t, lengths):
    """NaN behind every sequence's end."""
    if t is not None and lengths is not None:
        for b in range(t.shape[0]):
            t[b, int(lengths[b]):] = NAN
    return t


def _check(ops, shape, dtype, lengths="full", causal=True, scale=None, wide=False, seed=0, std=1.2, grad=True):
    B, T, S = shape[:3]
    g, q, kv, qr, kr = _inputs(seed, shape, dtype, std)
    ln, kn = _lengths(lengths, B, T, S)
    dout = _randn(g, B, T, shape[3], shape[6], dtype=dtype, std=0.1)
    want, bound = R.attention(q, kv, qr, kr, causal, scale, ln, kn, dtype, dout if grad else None)
    place = (lambda t, n: None if t is None else _poison(_wide(t.to(DEV)) if wide else t.to(DEV), n).detach().requires_grad_(grad))
    leaves = {"q": place(q, ln), "kv": place(kv, kn), "q_rot": place(qr, ln), "k_rot": place(kr, kn)}
    out = ops.latent_attention(*leaves.values(), causal=causal, scale=scale, lengths=None if ln is None else ln.to(DEV), key_lengths=None if kn is None else kn.to(DEV, torch.int32))
    _close("out", out, want["out"], bound["out"])
    if not grad:
        return
    used = {k: v for k, v in leaves.items() if v is not None}
    d = _poison(dout.to(DEV), ln)
    grads = torch.autograd.grad(out, list(used.values()), _wide(d) if wide else d)
    for name, got in zip(used, grads):
        _close("d" + name, got, want["d" + name], bound["d" + name])


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("shape", SHAPES)
def test_attention(ops, shape, dtype):
    _check(ops, shape, dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lengths", ["ragged", "uneven"])
@pytest.mark.parametrize("shape", [(4, 130, 130, 2, 128, 64, 128), (4, 40, 333, 1, 64, 0, 64), (5, 257, 300, 1, 96, 32, 128), (4, 9, 9, 2, 12, 4, 6)])
def test_attention_of_padded_batches(ops, shape, lengths, dtype):
    _check(ops, shape, dtype, lengths)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape", [(3, 100, 70, 2, 64, 32, 64), (2, 5, 300, 1, 128, 0, 128), (4, 130, 260, 1, 128, 64, 96)])
def test_attention_without_causality(ops, shape, dtype):
    _check(ops, shape, dtype, causal=False)
    _check(ops, shape[:3] + shape[3:], dtype, "ragged" if shape[2] >= shape[1] else "full", causal=False, scale=0.3)


def test_attention_with_more_queries_than_keys(ops):
    # the first queries see nothing
    _check(ops, (2, 200, 70, 2, 64, 0, 64), BF)
    _check(ops, (2, 200, 1, 2, 64, 32, 64), HF)
    _check(ops, (1, 90, 30, 1, 20, 0, 24), F32)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_attention_reads_windows_of_wider_tensors(ops, dtype):
    _check(ops, (2, 150, 150, 2, 64, 32, 64), dtype, wide=True)
    _check(ops, (4, 150, 180, 2, 64, 0, 64), dtype, "ragged", wide=True)


def test_attention_of_large_scores(ops):
    # one key has nearly all of the weight, and which one it is moves along the row: the running maximum grows many times
    _check(ops, (1, 400, 400, 2, 128, 64, 128), BF, std=4.0)
    _check(ops, (1, 300, 900, 1, 64, 0, 64), HF, std=5.0, seed=3)


def test_attention_of_growing_scores(ops):
    """Scores that rise along the keys by more than any float's exponent holds: every tile has a new maximum."""
    T = 700
    q = torch.full((1, T, 1, 64), 1.0, dtype=BF)
    k = (torch.arange(T)[:, None] / 4).expand(T, 64).to(BF)[None]
    v = _randn(_gen(0), 1, T, 64, dtype=BF)
    kv = torch.cat([k, v], -1)
    want, bound = R.attention(q, kv, None, None, True, 1.0, None, None, BF)
    _close("out", ops.latent_attention(q.to(DEV), kv.to(DEV), scale=1.0), want["out"], bound["out"])
    kv = torch.cat([k.flip(1), v], -1)
    want, bound = R.attention(q, kv, None, None, True, 1.0, None, None, BF)
    _close("out", ops.latent_attention(q.to(DEV), kv.to(DEV), scale=1.0), want["out"], bound["out"])


@pytest.mark.parametrize("shape", [(0, 4, 4, 2, 64, 0, 64), (2, 0, 5, 2, 64, 32, 64), (2, 5, 0, 2, 64, 32, 64), (1, 0, 0, 1, 8, 0, 8), (2, 3, 3, 2, 64, 0, 0)])
def test_attention_of_nothing(ops, shape):
    _check(ops, shape, BF)


@pytest.mark.parametrize("wanted", [{"q"}, {"kv"}, {"k_rot"}, {"q_rot", "kv"}])
def test_attention_forms_the_gradients_that_are_wanted(ops, wanted):
    shape = (2, 100, 140, 2, 64, 32, 64)
    g, *tensors = _inputs(5, shape, BF)
    dout = _randn(g, 2, 100, 2, 64, dtype=BF)
    names = ("q", "kv", "q_rot", "k_rot")
    leaves = [t.to(DEV).requires_grad_(n in wanted) for n, t in zip(names, tensors)]
    all_leaves = [t.to(DEV).requires_grad_(True) for t in tensors]
    some = torch.autograd.grad(ops.latent_attention(*leaves), [t for t in leaves if t.requires_grad], dout.to(DEV))
    every = dict(zip(names, torch.autograd.grad(ops.latent_attention(*all_leaves), all_leaves, dout.to(DEV))))
    for name, got in zip([n for n in names if n in wanted], some):
        assert torch.equal(got, every[name]), name


@pytest.mark.parametrize("dtype,shape", [(BF, (2, 300, 300, 4, 128, 64, 128)), (F32, (2, 90, 90, 3, 24, 8, 16))])
def test_attention_gives_the_same_bits(ops, dtype, shape):
    g, *tensors = _inputs(6, shape, dtype)
    leaves = [t.to(DEV).requires_grad_(True) for t in tensors]
    dout = _randn(g, *shape[:2], shape[3], shape[6], dtype=dtype).to(DEV)
    runs = []
    for _ in range(3):
        out = ops.latent_attention(*leaves)
        runs.append((out, *torch.autograd.grad(out, leaves, dout)))
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_attention_gradients_against_differences(ops):
    """float32: the loss along a direction, differences of step h around the point: off by h^2 times the third derivative and by 2^-24 / h of the loss's terms."""
    shape = (2, 20, 31, 2, 24, 8, 16)
    g, *tensors = _inputs(7, shape, F32, std=0.5)
    weight = _randn(g, 2, 20, 2, 16)
    for k in range(4):
        direction = _randn(g, *tensors[k].shape)
        h = 2.0 ** -6
        losses = []
        for sign in (-1, 1):
            moved = [t + sign * h * direction if n == k else t for n, t in enumerate(tensors)]
            losses.append(float((ops.latent_attention(*[t.to(DEV) for t in moved]).cpu().double() * weight).sum()))
        leaves = [t.to(DEV).requires_grad_(True) for t in tensors]
        grad, = torch.autograd.grad(ops.latent_attention(*leaves), leaves[k], weight.to(DEV))
        slope = float((grad.cpu().double() * direction).sum())
        scale = float((grad.cpu().double().abs() * direction.abs()).sum())
        assert abs((losses[1] - losses[0]) / (2 * h) - slope) < 4e-3 * scale, (k, losses, slope)


# ---- the cache ----------------------------------------------------------------------------------------------------------

def _pool(g, pages, page, rank, rot, dtype):
    latents = torch.randint(-128, 128, (pages, page, rank), generator=g, dtype=torch.int32).to(torch.int8)
    return latents, torch.rand(pages, page, generator=g) * 4 + 0.1, _randn(g, pages, page, rot, dtype=dtype) if rot else None


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("B,T,rank,rot,page,norm,wide", [(3, 37, 512, 64, 16, True, False), (2, 1, 256, 0, 64, True, True), (4, 50, 128, 32, 24, False, True), (1, 5, 16, 6, 3, True, False),
                                                        (2, 19, 320, 64, 7, True, True)])
def test_cache_holds_the_up_projections_operand(pkg, ops, dtype, B, T, rank, rot, page, norm, wide):
    g = _gen(rank + T)
    starts, lengths = torch.tensor([0, 5, 11, 2])[:B], torch.tensor([T, T // 2, 0, T - 1])[:B]
    per = -(-(T + 11) // page)
    table, blocks = ops.rotary_table(100, rot, device=DEV) if rot else None, torch.randperm(B * per + 2, generator=g)[:B * per].view(B, per).to(torch.int32)
    cache = ops.LatentCache.new(B * per + 2, page, rank, rot, dtype, DEV)
    for t in cache:
        if t is not None:
            t.fill_(3)
    x = _randn(g, B, T, rank + rot, dtype=dtype, std=0.7)
    x[0, 0, 3] = float("inf")                    # counts as zero, as in the layer's quantiser
    x[0, 1 % T] = 0
    xd = x.to(DEV)
    latent, kr = (_wide(xd[..., :rank], 5, 3), _wide(xd[..., rank:], 5, 3)) if wide else (xd[..., :rank], xd[..., rank:])
    w = (1 + 0.2 * torch.randn(rank, generator=g)).to(DEV) if norm else None
    ops.latent_cache_write(cache, blocks.to(DEV), latent, w, kr if rot else None, table, starts=starts.to(DEV), lengths=lengths.to(DEV))
    flat = x[..., :rank].reshape(-1, rank).to(DEV)
    rows, top = pkg.int2_tc_ops.rmsnorm_quantize_rows(flat, w)[:2] if norm else pkg.int2_tc_ops.quantize_rows(flat)
    keys = ops.rotary(xd[..., rank:], table, starts.to(DEV)) if rot else None
    want = [torch.full_like(t, 3) if t is not None else None for t in cache]
    for b in range(B):
        for t in range(int(lengths[b])):
            p = int(starts[b]) + t
            at = int(blocks[b, p // page]), p % page
            want[0][at], want[1][at] = rows[b * T + t], top[b * T + t]
            if rot:
                want[2][at] = keys[b, t]
    for a, b in zip(cache, want):
        assert a is None and b is None or torch.equal(a, b)
    got = ops.latent_cache_read(cache, blocks.to(DEV), T, starts=starts.to(DEV), lengths=lengths.to(DEV))
    live = (torch.arange(T) < lengths[:, None]).to(DEV)
    assert torch.equal(got[0], torch.where(live.view(-1, 1), rows, torch.zeros_like(rows))) and torch.equal(got[1], torch.where(live.view(-1), top, 0.0))
    if rot:
        assert torch.equal(got[2], torch.where(live[..., None], keys, torch.zeros_like(keys)))


@pytest.mark.parametrize("out", [BF, HF, F32])
def test_cache_reads_values(ops, out):
    g = _gen(9)
    latents, absmax, keys = _pool(g, 9, 10, 48, 6, HF)
    blocks = torch.tensor([[3, 8, -1, 0], [9, 2, 1, 5], [6, 7, 4, 100]], dtype=torch.int32)
    starts, lengths, L = torch.tensor([0, 4, -3]), torch.tensor([40, 20, 33]), 41
    values, back = ops.latent_cache_read(ops.LatentCache(latents.to(DEV), absmax.to(DEV), keys.to(DEV)), blocks.to(DEV), L, starts.to(DEV, torch.int32), lengths.to(DEV), out)
    want, want_keys = torch.zeros(3, L, 48, dtype=torch.float64), torch.zeros(3, L, 6, dtype=HF)
    for b in range(3):
        for t in range(int(lengths[b])):
            # int64 positions below 0 are clamped to -1, int32 ones are taken as they are; neither has a page
            p = int(starts[b]) + t
            if not 0 <= p < 40 or not 0 <= int(blocks[b, p // 10]) < 9:
                continue
            at = int(blocks[b, p // 10]), p % 10
            want[b, t], want_keys[b, t] = latents[at].double() * (absmax[at].double() / 127), keys[at]
    assert torch.equal(back.cpu(), want_keys)
    _close("values", values, want, (R.UNIT[out] + 4 * R.E) * want.abs() + R.TINY[out])


@pytest.mark.parametrize("rank, rot, page", [(16, 2, 7), (48, 0, 64), (272, 64, 33), (512, 64, 64)])
def test_cache_reads_many_tokens(ops, rank, rot, page):
    """So many that a warp takes several; the last warp's are not all there."""
    g = _gen(rank)
    B, L = 5, 5003
    per = -(-L // page)
    latents, absmax, keys = _pool(g, 300, page, rank, rot, BF)
    blocks = torch.randint(-2, 302, (B, per), generator=g, dtype=torch.int32)
    starts, lengths = torch.tensor([0, 5, 0, 4000, 17]), torch.tensor([L, 1, 0, L, 2500])
    at = torch.arange(L)[None] + starts[:, None]
    page_of = torch.where(at < per * page, torch.gather(blocks.long(), 1, (at // page).clamp(max=per - 1)), -1)
    there = (torch.arange(L)[None] < lengths[:, None]) & (page_of >= 0) & (page_of < 300)
    row = torch.where(there, page_of * page + at % page, 0).flatten()
    there = there.flatten()
    want, want_max = latents.view(-1, rank)[row] * there[:, None], absmax.flatten()[row] * there
    cache = ops.LatentCache(latents.to(DEV), absmax.to(DEV), keys.to(DEV) if rot else None)
    rows, most, back = ops.latent_cache_read(cache, blocks.to(DEV), L, starts.to(DEV), lengths.to(DEV))
    assert torch.equal(rows.cpu(), want.to(torch.int8)) and torch.equal(most.cpu(), want_max)
    values, again = ops.latent_cache_read(cache, blocks.to(DEV), L, starts.to(DEV), lengths.to(DEV), BF)
    true = want.double() * (want_max.double() / 127)[:, None]
    _close("values", values.view(-1, rank), true, (R.UNIT[BF] + 4 * R.E) * true.abs() + R.TINY[BF])
    if rot:
        want_keys = keys.view(-1, rot)[row] * there[:, None]
        assert torch.equal(back.cpu().view(-1, rot), want_keys) and torch.equal(again, back)


def test_cache_drops_what_has_no_page(ops):
    cache = ops.LatentCache.new(4, 8, 64, 32, BF, DEV)
    blocks = torch.tensor([[1, -1], [4, 2]], dtype=torch.int32, device=DEV)
    x = torch.ones(2, 30, 96, dtype=BF, device=DEV)
    ops.latent_cache_write(cache, blocks, x[..., :64], None, x[..., 64:])
    wrote = cache.absmax.cpu() > 0
    assert wrote[1].all() and wrote[2].all() and not wrote[0].any() and not wrote[3].any()


# ---- the absorbed form --------------------------------------------------------------------------------------------------

def _step_case(g, B, H, D, P, V, rank, page, tokens, dtype, std=1.2):
    per = -(-tokens // page)
    latents, absmax, keys = _pool(g, B * per + 1, page, rank, P, dtype)
    absmax = absmax * 0.5
    blocks = torch.randperm(B * per + 1, generator=g)[:B * per].view(B, per).to(torch.int32)
    W = torch.randint(-1, 2, (H * (D + V), rank), generator=g, dtype=torch.int8)
    return latents, absmax, keys, blocks, W, _randn(g, B, H, D, dtype=dtype, std=std), _randn(g, B, H, P, dtype=dtype, std=std) if P else None


def _check_step(ops, B, H, D, P, V, rank, page, tokens, dtype, lengths, table=True, neighbours=False, bad=False, wide=False, seed=0, scale=None, std=1.2):
    g = _gen(seed)
    latents, absmax, keys, blocks, W, q, qr = _step_case(g, B, H, D, P, V, rank, page, tokens, dtype, std)
    if bad:
        blocks[0, 0], blocks[-1, -1] = -1, latents.shape[0]
    gamma = 0.7 / rank ** 0.5
    lengths = torch.tensor(lengths)
    tab = ops.rotary_table(tokens, P, device=DEV) if table and P else None
    want, bound = R.step(q, W, gamma, latents, absmax, keys, blocks, lengths, V, qr, None if tab is None else tab.cpu(), scale, dtype, neighbours)
    # what lies behind a sequence's end belongs to nobody
    used = torch.zeros(latents.shape[:2], dtype=torch.bool)
    for b in range(B):
        for p in range(int(lengths[b].clamp(0, blocks.shape[1] * page))):
            e = int(blocks[b, p // page])
            if 0 <= e < latents.shape[0]:
                used[e, p % page] = True
    absmax = torch.where(used, absmax, NAN)
    if keys is not None:
        keys = torch.where(used[..., None], keys, NAN)
    packed = torch.from_numpy(O.pack_ternary(W.numpy(), pad_code=1)).to(DEV)
    cache = ops.LatentCache(latents.to(DEV), absmax.to(DEV), None if keys is None else keys.to(DEV))
    place = lambda t: None if t is None else _wide(t.to(DEV), 5, 1) if wide else t.to(DEV)  # noqa: E731
    out = ops.latent_attention_step(place(q), packed, gamma, cache, blocks.to(DEV), lengths.to(DEV), V, q_rot=place(qr), table=tab, scale=scale, neighbours=neighbours)
    _close("out", out, want, bound)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("B,H,D,P,V,rank,page,lengths", [
    (1, 1, 64, 0, 64, 64, 16, [1]), (3, 32, 128, 64, 128, 512, 64, [700, 1, 513]), (4, 5, 96, 32, 80, 256, 24, [0, 65, 64, 63]), (2, 40, 64, 64, 64, 128, 8, [300, 129]),
    (2, 3, 20, 6, 24, 48, 7, [100, 31]), (1, 64, 128, 64, 128, 512, 128, [1000]), (2, 16, 128, 0, 256, 320, 64, [90, 1200]), (5, 12, 128, 64, 128, 512, 32, [0, 0, 5, 0, 33]),
    (1, 130, 16, 16, 16, 64, 16, [200]), (3, 8, 256, 8, 16, 16, 1, [64, 65, 200])])
def test_step(ops, B, H, D, P, V, rank, page, lengths, dtype):
    _check_step(ops, B, H, D, P, V, rank, page, max(max(lengths), 1), dtype, lengths, seed=B + H)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_step_variants(ops, dtype):
    _check_step(ops, 2, 6, 64, 32, 64, 128, 16, 200, dtype, [200, 77], table=False)
    _check_step(ops, 2, 6, 64, 32, 64, 128, 16, 200, dtype, [200, 77], neighbours=True, wide=True)
    _check_step(ops, 2, 6, 64, 32, 64, 128, 16, 200, dtype, [200, 200], bad=True)
    _check_step(ops, 3, 6, 64, 0, 64, 128, 32, 300, dtype, [-5, 1000, 300], scale=0.02)
    _check_step(ops, 1, 6, 64, 0, 64, 128, 16, 16, dtype, [16], bad=True)                  # no token has a page
    _check_step(ops, 1, 8, 128, 64, 128, 512, 64, 900, dtype, [900], std=6.0)
    _check_step(ops, 70, 2, 32, 16, 32, 64, 16, 100, dtype, [(i * 37) % 101 for i in range(70)])


def test_step_of_nothing(ops):
    _check_step(ops, 2, 3, 64, 32, 64, 128, 16, 40, BF, [0, 0])
    cache = ops.LatentCache.new(2, 16, 128, 0, BF, DEV)
    W = torch.zeros(4 * 128, 32, dtype=torch.uint8, device=DEV)
    out = ops.latent_attention_step(torch.ones(0, 4, 64, dtype=BF, device=DEV), W, 1.0, cache, torch.zeros(0, 1, dtype=torch.int32, device=DEV), torch.zeros(0, dtype=torch.int32, device=DEV), 64)
    assert out.shape == (0, 4, 64)
    out = ops.latent_attention_step(torch.ones(3, 4, 64, dtype=BF, device=DEV), W, 1.0, cache, torch.zeros(3, 0, dtype=torch.int32, device=DEV), torch.ones(3, dtype=torch.int32, device=DEV), 64)
    assert out.shape == (3, 4, 64) and not out.any()


# ---- streams, graphs, refusals ------------------------------------------------------------------------------------------

def test_captured_training_step(ops):
    shape = (2, 200, 200, 2, 128, 64, 128)
    g, *tensors = _inputs(11, shape, BF)
    leaves = [t.to(DEV).requires_grad_(True) for t in tensors]
    dout = _randn(g, 2, 200, 2, 128, dtype=BF).to(DEV)

    def pass_():
        out = ops.latent_attention(*leaves)
        return (out, *torch.autograd.grad(out, leaves, dout))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pass_()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = pass_()
    with torch.no_grad():
        for t in leaves:
            t.mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(captured, pass_()):
        assert torch.equal(a, b)


def test_step_on_another_stream_and_in_two_graphs(ops):
    g = _gen(12)
    latents, absmax, keys, blocks, W, q, qr = _step_case(g, 3, 8, 128, 64, 128, 512, 64, 600, BF)
    cache = ops.LatentCache(latents.to(DEV), absmax.to(DEV), keys.to(DEV))
    packed, blocks, table = torch.from_numpy(O.pack_ternary(W.numpy(), pad_code=1)).to(DEV), blocks.to(DEV), ops.rotary_table(600, 64, device=DEV)
    lengths, q, qr = torch.tensor([600, 33, 0], device=DEV, dtype=torch.int32), q.to(DEV), qr.to(DEV)

    def pass_():
        return ops.latent_attention_step(q, packed, 0.05, cache, blocks, lengths, 128, q_rot=qr, table=table)

    want = pass_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = pass_()
    torch.cuda.synchronize()
    assert torch.equal(want, other)
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(pass_())
    lengths.copy_(torch.tensor([100, 599, 1]))
    want = pass_()
    for graph, stream in zip(graphs, (torch.cuda.Stream(), torch.cuda.Stream())):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_refusals(ops):
    t = lambda *s, dtype=BF: torch.zeros(*s, dtype=dtype, device=DEV)  # noqa: E731
    q, kv = t(2, 3, 4, 64), t(2, 5, 4 * 128)
    cache, blocks, lengths = ops.LatentCache.new(3, 16, 128, 32, BF, DEV), t(2, 1, dtype=torch.int32), t(2, dtype=torch.int32)
    W = t(4 * 128, 32, dtype=torch.uint8)
    for call, message in [
        (lambda: ops.latent_attention(q, kv[..., :-1]), "channels"),
        (lambda: ops.latent_attention(q, kv.float()), "another dtype"),
        (lambda: ops.latent_attention(q, kv[:1]), "shape"),
        (lambda: ops.latent_attention(q, kv, t(2, 3, 4, 32)), "come together"),
        (lambda: ops.latent_attention(t(2, 3, 4, 300), t(2, 5, 4 * 310)), "channels"),
        (lambda: ops.latent_attention(q, kv, lengths=t(3, dtype=torch.int32)), "one entry"),
        (lambda: ops.latent_attention(q, kv, key_lengths=t(2)), "int32 or int64"),
        (lambda: ops.latent_attention(q.int(), kv), "float16"),
        (lambda: ops.rotary(q, ops.rotary_table(4, 32, device=DEV)), "table must have shape"),
        (lambda: ops.rotary(t(2, 3, 7), ops.rotary_table(4, 6, device=DEV)), "even"),
        (lambda: ops.rotary(q, ops.rotary_table(4, 64, device=DEV), t(3, dtype=torch.int32)), "positions must have shape"),
        (lambda: ops.latent_cache_write(cache, blocks, t(2, 4, 64)), "shape"),
        (lambda: ops.latent_cache_write(cache, blocks, t(2, 4, 128)), "come together"),
        (lambda: ops.latent_cache_write(cache, blocks, t(2, 4, 128, dtype=HF), None, t(2, 4, 32, dtype=HF)), "another dtype"),
        (lambda: ops.latent_cache_write(cache, blocks[:1], t(2, 4, 128), None, t(2, 4, 32)), "one row"),
        (lambda: ops.latent_cache_write(cache, blocks.long(), t(2, 4, 128), None, t(2, 4, 32)), "int32"),
        (lambda: ops.latent_cache_write(cache, blocks, t(2, 4, 128).requires_grad_(True), None, t(2, 4, 32)), "no gradient"),
        (lambda: ops.latent_cache_read(cache, blocks, -1), "negative"),
        (lambda: ops.latent_cache_read(cache, blocks, 4, dtype=torch.int8), "dtype must be"),
        (lambda: ops.latent_cache_read(ops.LatentCache(cache.latents[:, :, ::2], cache.absmax), blocks, 4), "contiguous"),
        (lambda: ops.latent_cache_read(ops.LatentCache.new(3, 16, 24, 0, BF, DEV), blocks, 4), "multiples of 16"),
        (lambda: ops.latent_attention_step(t(2, 4, 64), W, 1.0, cache, blocks, lengths, 64), "come together"),
        (lambda: ops.latent_attention_step(t(2, 4, 64), W[:-1], 1.0, cache, blocks, lengths, 64, q_rot=t(2, 4, 32)), "W_packed must have shape"),
        (lambda: ops.latent_attention_step(t(2, 4, 64), W, 1.0, cache, blocks, None, 64, q_rot=t(2, 4, 32)), "lengths"),
        (lambda: ops.latent_attention_step(t(2, 4, 64).requires_grad_(True), W, 1.0, cache, blocks, lengths, 64, q_rot=t(2, 4, 32)), "no gradient"),
        (lambda: ops.latent_attention_step(t(2, 4, 64, dtype=HF), W, 1.0, cache, blocks, lengths, 64, q_rot=t(2, 4, 32, dtype=HF)), "another dtype"),
    ]:
        with pytest.raises(RuntimeError, match=message):
            call()


# ---- recorded calls -----------------------------------------------------------------------------------------------------

def _leaves(rot=True):
    g = _gen(77)
    q, kv = _randn(g, 2, 70, 2, 64, dtype=BF).to(DEV), _randn(g, 2, 70, 2 * 128, dtype=BF).to(DEV)
    qr, kr = (_randn(g, 2, 70, 2, 32, dtype=BF).to(DEV), _randn(g, 2, 70, 32, dtype=BF).to(DEV)) if rot else (None, None)
    return [t.requires_grad_(True) for t in (q, kv, qr, kr) if t is not None]


def test_second_derivatives_are_refused(ops):
    leaves = _leaves()
    table = ops.rotary_table(70, 32, device=DEV)
    for out, leaf in ((ops.latent_attention(*leaves), leaves[0]), (ops.rotary(leaves[2], table), leaves[2])):
        (d,) = torch.autograd.grad(out.float().square().sum(), leaf, create_graph=True)
        assert d.requires_grad
        with pytest.raises(RuntimeError, match="first order"):
            torch.autograd.grad(d.float().sum(), leaf)


def test_recorded_calls_keep_autograds_rules(ops):
    from torch.utils.checkpoint import checkpoint
    leaves = _leaves()
    table = ops.rotary_table(70, 32, device=DEV)

    def f(q, kv, qr, kr):
        return ops.latent_attention(q, kv, ops.rotary(qr, table), ops.rotary(kr, table))

    dout = torch.randn(2, 70, 2, 64, device=DEV).to(BF)
    want = torch.autograd.grad(f(*leaves), leaves, dout)
    for a, b in zip(want, torch.autograd.grad(checkpoint(f, *leaves, use_reentrant=False), leaves, dout)):
        assert torch.equal(a, b)
    # two graphs of the same leaves, walked twice and out of order; gradients that are views
    one, two = f(*leaves), f(*leaves)
    wide = torch.empty(2, 70, 2, 80, device=DEV, dtype=BF)
    wide[..., 8:72] = dout
    for out in (two, one):
        for _ in range(2):
            for a, b in zip(want, torch.autograd.grad(out, leaves, wide[..., 8:72], retain_graph=True)):
                assert torch.equal(a, b)
    # leaves without a gradient, and a graph without the rotated parts
    q, kv = _leaves(False)
    (only,) = torch.autograd.grad(ops.latent_attention(q.detach(), kv), [kv], dout)
    both = torch.autograd.grad(ops.latent_attention(q, kv), [q, kv], dout)
    assert torch.equal(only, both[1])
    with torch.no_grad():
        assert not ops.latent_attention(q, kv).requires_grad
    # what a graph needs and has changed since
    x = leaves[2].detach() * 1
    out = ops.latent_attention(leaves[0], leaves[1], x, leaves[3])
    x.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward(dout)
    out = ops.latent_attention(*leaves)
    out.backward(dout)
    with pytest.raises(RuntimeError, match="second time"):
        out.backward(dout)


def test_errors_of_a_backward_pass_reach_its_caller(ops):
    leaves = _leaves()
    out = ops.latent_attention(*leaves)

    class Wrong(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return x.clone()

        @staticmethod
        def backward(ctx, dy):
            raise ValueError("from a node in front")

    with pytest.raises(ValueError, match="in front"):
        Wrong.apply(out).sum().backward()
    with pytest.raises(RuntimeError):
        ops.latent_attention(leaves[0], leaves[1][:, :, :100], *leaves[2:])
    # an error of the call itself, in the engine's thread: what was kept comes back with another dtype
    table = ops.rotary_table(70, 32, device=DEV)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.half() if t.is_floating_point() else t):
        attended, turned = ops.latent_attention(*leaves), ops.rotary(leaves[2], table)
    for out, message in ((attended, "lse must be Float"), (turned, "table must be Float")):
        with pytest.raises(RuntimeError, match=message):
            out.sum().backward()
    ops.latent_attention(*leaves).sum().backward()
    assert all(t.grad is not None for t in leaves)


def test_gradients_do_not_take_the_outputs_rounding(ops):
    """An element of dq is rounded itself and is a sum over rounded factors ds: two independent errors whose root mean square, relative to a value whose mantissa
    is spread evenly over its logarithm, is 2^-7 sqrt(E[1/m^2] / 12), E = 0.75 / (2 ln 2): 1.66e-3 each, 2.35e-3 together.  dout . out formed of the rounded
    output would add 0.8e-3 (one error for all keys of a row, found for these sizes in 64 bits): 2.48e-3."""
    g = _gen(5)
    H, T = 4, 1024
    q, kv, dout = _randn(g, 1, T, H, 128, dtype=BF), _randn(g, 1, T, H * 256, dtype=BF), _randn(g, 1, T, H, 128, dtype=BF)
    leaf = q.to(DEV).requires_grad_(True)
    (dq,) = torch.autograd.grad(ops.latent_attention(leaf, kv.to(DEV)), [leaf], dout.to(DEV))
    k, v = kv[..., :H * 128].unflatten(-1, (H, 128)).double().movedim(2, 1), kv[..., H * 128:].unflatten(-1, (H, 128)).double().movedim(2, 1)
    x, d = q.double().movedim(2, 1), dout.double().movedim(2, 1)
    p = (x @ k.mT * 128 ** -0.5).masked_fill(torch.ones(T, T).triu(1).bool(), -torch.inf).softmax(-1)
    dp = d @ v.mT
    want = (p * (dp - (p * dp).sum(-1, keepdim=True))) @ k * 128 ** -0.5
    assert (dq.cpu().double().movedim(2, 1) - want).norm() < 2.42e-3 * want.norm()
