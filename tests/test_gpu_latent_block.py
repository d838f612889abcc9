"""Latent attention over INT2 projections: the block against its definition, prompts in pieces and single tokens against the whole text, unequal lengths, and
a training step.

Tolerance of the comparisons.  The projections quantise their inputs to 8 bits per token.  Where two computations of the same values differ by roundings of the
16-bit type, single int8 values behind them move by one step of 1/127 of a row's maximum, about 1/40 of its root mean square for normal values.  Were all values of
a row so moved, an output would differ by 1/40 of its norm per projection; few are, and 2 % of the output's norm is asked for."""
import math

import pytest
import torch


pytestmark = pytest.mark.gpu
DEV = "cuda"


def _block(pkg, width=256, heads=4, rank=64, rot=32, **kw):
    torch.manual_seed(3)
    block = pkg.LatentAttentionInt2(width, heads, head_dim=64, kv_rank=rank, rot_dim=rot, max_positions=512, threshold=3, **kw).to(DEV).init_weights()
    with torch.no_grad():
        block.w_kv_up.extra_rmsnorm.weight.add_(torch.randn(rank, device=DEV) * 0.1)
    return block


def _input(B, L, width=256, seed=0, dtype=torch.bfloat16):
    return torch.randn(B, L, width, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def _near(a, b, name):
    off = float((a.float() - b.float()).norm() / b.float().norm())
    assert off <= 0.02, (name, off)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rot", [0, 32])
def test_forward_against_the_definition(pkg, rot, dtype):
    block = _block(pkg, rot=rot).eval()
    x = _input(2, 90, dtype=dtype)
    with torch.no_grad():
        out = block(x)
        H, D = 4, 64
        q, c = block.w_q(x).double(), block.w_kv_down(x)
        kv = block.w_kv_up(c[..., :64].contiguous()).double()
        qc, kc, v = q[..., :H * D].unflatten(-1, (H, D)), kv[..., :H * D].unflatten(-1, (H, D)), kv[..., H * D:].unflatten(-1, (H, D))
        if rot:
            table = block.table.double()[:90]

            def turn(t):
                cos, sin = (s.view(90, *[1] * (t.dim() - 3), rot // 2) for s in table.chunk(2, -1))
                a, b = t.chunk(2, -1)
                return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

            qc = torch.cat([qc, turn(q[..., H * D:].unflatten(-1, (H, rot)))], -1)
            kc = torch.cat([kc, turn(c[..., 64:].double())[:, :, None].expand(-1, -1, H, -1)], -1)
        z = torch.einsum("bihd,bjhd->bhij", qc, kc) / math.sqrt(D + rot)
        p = torch.softmax(z.masked_fill(torch.ones(90, 90, device=DEV, dtype=torch.bool).triu(1), -math.inf), -1)
        want = block.w_out(torch.einsum("bhij,bjhd->bihd", p, v).flatten(2).to(dtype))
    _near(out, want, "output")


@pytest.mark.parametrize("rot", [0, 32])
def test_pieces_and_single_tokens_equal_the_whole_text(pkg, rot):
    block = _block(pkg, rot=rot).eval()
    x = _input(3, 150)
    with torch.no_grad():
        whole = block(x)
        state = block.new_state(3, 160, page_size=24)
        parts = [block(x[:, :70], state), block(x[:, 70:71], state), block(x[:, 71:140], state)]
        parts += [block.step(x[:, t], state)[:, None] for t in range(140, 150)]
    assert state.lengths.tolist() == [150] * 3 and state.most == 150
    _near(torch.cat(parts, 1), whole, "output")


def test_a_state_records_no_gradient(pkg):
    block = _block(pkg).train()
    x = _input(1, 9).requires_grad_(True)
    assert not block(x, block.new_state(1, 16)).requires_grad


def test_sequences_of_unequal_length_equal_each_by_itself(pkg):
    block = _block(pkg).eval()
    lengths = torch.tensor([50, 1, 0, 33], device=DEV)
    x = _input(4, 50)
    more = _input(4, 20, seed=1)
    for b in range(4):
        x[b, int(lengths[b]):] = float("nan")
    with torch.no_grad():
        plain = block(x, lengths=lengths)
        state = block.new_state(4, 80)
        out = block(x, state, lengths)
        second = block(more, state, torch.tensor([20, 0, 7, 1], device=DEV))
        tokens = block.step(more[:, 0], state)
        for b, n in enumerate(lengths.tolist()):
            own = block.new_state(1, 80)
            assert not out[b, n:].any() and not plain[b, n:].any()
            if n:
                alone = block(x[b:b + 1, :n], own)
                _near(out[b, :n], alone[0], f"sequence {b}")
                _near(plain[b, :n], alone[0], f"sequence {b} without a state")
            m = [20, 0, 7, 1][b]
            if m:
                _near(second[b, :m], block(more[b:b + 1, :m], own)[0], f"second piece of sequence {b}")
            _near(tokens[b], block.step(more[b:b + 1, 0], own)[0], f"token of sequence {b}")


def test_a_full_state_refuses(pkg):
    block = _block(pkg).eval()
    state = block.new_state(1, 16, page_size=16)
    with torch.no_grad():
        block(_input(1, 16), state)
        with pytest.raises(RuntimeError, match="no room"):
            block.step(_input(1, 1)[:, 0], state)


def test_a_training_step_reaches_every_parameter(pkg):
    block = _block(pkg).train()
    before = {n: m.int2_layer.H_packed.clone() for n, m in block.named_children() if isinstance(m, pkg.BitLinearInt2)}
    pkg.set_all_int2_lr(block, 1.0)
    x = _input(2, 96)
    x.requires_grad_(True)
    lengths = torch.tensor([96, 40], device=DEV)
    out = block(x, lengths=lengths)
    out.backward(torch.randn(out.shape, generator=torch.Generator().manual_seed(1)).to(out))
    for name, p in block.named_parameters():
        if name.endswith("gamma"):
            continue
        assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.any(), name
    assert torch.isfinite(x.grad).all() and x.grad[0].any() and not x.grad[1, 40:].any()
    for name, old in before.items():
        assert not torch.equal(getattr(block, name).int2_layer.H_packed, old), name


def test_gradients_against_the_definition(pkg):
    """The gradient of the output's projection with a fixed weight, against the definition of the attention between the same projections."""
    pkg.disable_hysteresis()
    try:
        block = _block(pkg, rot=0).train()
        weight = torch.randn(2, 70, 4, 64, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(DEV)
        q = (torch.randn(2, 70, 4, 64, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(DEV)).requires_grad_(True)
        latent = _input(2, 70, 64, seed=4).requires_grad_(True)
        grads = []
        for own in (True, False):
            kv = block.w_kv_up(latent)
            if own:
                out = pkg.attention_ops.latent_attention(q, kv)
            else:
                k, v = (t.unflatten(-1, (4, 64)).float().transpose(1, 2) for t in kv.chunk(2, -1))
                z = q.float().transpose(1, 2) @ k.transpose(-1, -2) / 8
                out = (torch.softmax(z.masked_fill(torch.ones(70, 70, device=DEV, dtype=torch.bool).triu(1), -math.inf), -1) @ v).transpose(1, 2)
            grads.append(torch.autograd.grad(out, (q, latent), weight.to(out.dtype)))
        for name, a, b in zip(("q", "latent"), *grads):
            _near(a, b, name)
    finally:
        pkg.enable_hysteresis()


def test_the_cache_holds_the_layers_own_operand(pkg):
    """Expanding what the cache holds gives the up projection's own output, bit for bit."""
    block = _block(pkg).eval()
    x = _input(2, 40)
    with torch.no_grad():
        latent, k_rot = block._latent(x)
        state = block.new_state(2, 64, page_size=16)
        block._write(state, latent, k_rot, None)
        rows, absmax, _ = pkg.attention_ops.latent_cache_read(state.cache, state.block_table, 40)
        W, gamma = block._up()
        kv = pkg.int2_tc_ops.matmul_rows(rows, W, absmax, gamma, torch.bfloat16)
        assert torch.equal(kv.view(2, 40, -1), block.w_kv_up(latent.contiguous()))


def test_refusals(pkg):
    with pytest.raises(RuntimeError, match="per_token"):
        pkg.LatentAttentionInt2(256, 4, quant_mode="per_tensor")
    with pytest.raises(RuntimeError, match="no bias"):
        pkg.LatentAttentionInt2(256, 4, bias=True)
