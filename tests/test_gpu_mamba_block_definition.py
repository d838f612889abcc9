"""The Mamba block against a composition of its own: the projections as they are, everything between them from its formula in float64, rounded to the
activations' type where the operators round.

Tolerance: test_gpu_mamba_block.py derives 2 % of the norm for what goes through four projections' quantisers with single bfloat16 values moved by
a unit in the last place; a gradient goes through the four projections and their four backward quantisers, so 4 % are asked for."""
import copy

import pytest
import torch
import torch.nn.functional as F

from test_gpu_mamba_block import DEV, _block, _inputs

pytestmark = pytest.mark.gpu


def _near(a, b, name, tolerance):
    off = float((a.detach().double() - b.detach().double()).norm() / b.detach().double().norm())
    assert off <= tolerance, (name, off)


def _composed(block, h, x):
    """The block's definition on full sequences."""
    io, inner, rank, N = x.dtype, block.d_inner, block.dt_rank, block.d_state
    L = x.shape[1]
    xz = block.in_proj(x)
    first, z = xz[..., :inner].double(), xz[..., inner:].double()
    rows = F.pad(first, (0, 0, block.d_conv - 1, 0))
    u = F.silu(block.conv_bias.double() + sum(block.conv_weight[:, j].double() * rows[:, j:j + L] for j in range(block.d_conv))).to(io)
    p = block.x_proj(u)
    raw = block.dt_proj(p[..., :rank].contiguous()).double() + block.dt_bias.double()
    B, C = p[..., rank:rank + N].double(), p[..., rank + N:].double()
    delta, A, state, ys = F.softplus(raw, threshold=1e9), -torch.exp(block.A_log.double()), 0.0, []
    for ut, dt, Bt, Ct in zip(u.double().unbind(1), delta.unbind(1), B.unbind(1), C.unbind(1)):
        state = torch.exp(dt[..., None] * A) * state + (dt * ut)[..., None] * Bt[:, None]
        ys.append((state * Ct[:, None]).sum(-1) + block.D.double() * ut)
    y = (torch.stack(ys, 1) * F.silu(z)).to(io)

    def norm(v, w):
        return w.double() * v / torch.sqrt(v.pow(2).mean(-1, keepdim=True) + block.eps)

    out = norm(block.out_proj(y).double(), block.post_norm) * block.scale.double()
    if block.gate_proj is not None:
        out = out * torch.sigmoid(block.gate_proj(x).double())
    out = h.double() + out
    return out.to(io), norm(out, block.next_norm).to(io)


@pytest.mark.parametrize("gated", [True, False])
def test_block_equals_its_definition(pkg, gated):
    block = _block(pkg, gated=gated).train()
    with torch.no_grad():                                  # nothing that could be exchanged without being seen
        block.A_log.add_(torch.randn_like(block.A_log) * 0.3)
        block.D.mul_(torch.randn_like(block.D))
        block.next_norm.add_(torch.randn_like(block.next_norm) * 0.1)
    twin = copy.deepcopy(block)
    g = torch.Generator().manual_seed(5)
    grads = [torch.randn(2, 48, 256, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2)]
    results = []
    for model, call in ((block, block), (twin, lambda h, x: _composed(twin, h, x))):
        h, x = _inputs(2, 48, 256)
        h.requires_grad_(True)
        x.requires_grad_(True)
        out = call(h, x)
        torch.autograd.backward(out, grads)
        results.append((out, {"h": h.grad, "x": x.grad, **{n: p.grad for n, p in model.named_parameters() if not n.endswith("gamma")}}))
    (out, got), (want_out, want) = results
    for name, a, b in zip(("h", "normed"), out, want_out):
        _near(a, b, name, 0.02)
    for name in want:
        _near(got[name], want[name], name, 0.04)


def _piecewise(pkg, block, h, x, state):
    """The block's forward pass from its operators, the state's tensors replaced instead of written."""
    ops, inner = pkg.ssm_ops, block.d_inner
    xz = block.in_proj(x)
    u, conv = ops.causal_conv(xz[..., :inner], block.conv_weight, block.conv_bias, initial_state=state[0], return_final_state=True)
    dt, B, C = block._selection(u)
    y, ssm = ops.selective_scan(u, dt, -torch.exp(block.A_log), B, C, D=block.D, z=xz[..., inner:], dt_bias=block.dt_bias, initial_state=state[1],
                                return_final_state=True)
    return block._join(h, y, x), (conv.detach(), ssm.detach())


def test_training_on_a_text_in_pieces(pkg):
    """Backward after each piece, the state going on from one to the next: the gradients are those of the operators on each piece, bit for bit."""
    block = _block(pkg).train()
    pkg.set_all_int2_lr(block, 0.0)
    twin = copy.deepcopy(block)
    h, x = _inputs(2, 75, 256)
    g = torch.Generator().manual_seed(1)
    grads = [torch.randn(2, 75, 256, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2)]
    state = block.new_state(2)
    conv, ssm = state.conv, state.ssm
    own = (conv.clone(), ssm.clone())
    for a, b in ((0, 33), (33, 34), (34, 75)):
        torch.autograd.backward(block(h[:, a:b], x[:, a:b], state), [v[:, a:b] for v in grads])
        out, own = _piecewise(pkg, twin, h[:, a:b], x[:, a:b], own)
        torch.autograd.backward(out, [v[:, a:b] for v in grads])
        assert torch.equal(state.conv, own[0]) and torch.equal(state.ssm, own[1])
        assert state.conv is conv and state.ssm is ssm, "the state's tensors are updated in place"
    for (name, p), q in zip(block.named_parameters(), twin.parameters()):
        assert (p.grad is None) == (q.grad is None) and (p.grad is None or torch.equal(p.grad, q.grad)), name


def test_padding_of_the_block_may_hold_anything(pkg):
    """Outputs and gradients of padding are zeros, and no parameter's gradient has seen it, whatever lies in the padding of the inputs and of the outputs'
    gradients."""
    lengths = torch.tensor([40, 0, 7, 1], device=DEV)
    behind = torch.arange(40, device=DEV) >= lengths[:, None]
    results = []
    for fill in (0.0, float("nan"), float("inf")):
        block = _block(pkg).train()
        h, x = _inputs(4, 40, 256)
        g = torch.Generator().manual_seed(1)
        grads = [torch.randn(4, 40, 256, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2)]
        for t in (h, x, *grads):
            t[behind] = fill
        h.requires_grad_(True)
        x.requires_grad_(True)
        out = block(h, x, lengths=lengths)
        torch.autograd.backward(out, grads)
        for t in (*out, h.grad, x.grad):
            assert not t[behind].any() and torch.isfinite(t).all()
        results.append([*out, h.grad, x.grad, *(p.grad for n, p in block.named_parameters() if not n.endswith("gamma"))])
    for other in results[1:]:
        for a, b in zip(results[0], other):
            assert torch.isfinite(a).all() and torch.equal(a, b)
