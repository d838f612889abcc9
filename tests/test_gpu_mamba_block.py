"""The Mamba block over INT2 projections: prompts and single tokens against the whole sequence, unequal lengths, and a training step.

Tolerance of the comparisons: the same arithmetic in another grouping of tokens moves a bfloat16 value by a unit in its last place here and there, and
the projections behind it quantise to 8 bits per token, so such a move can shift single int8 values by one step of 1/127 of a row's maximum
(about 1/40 of its root mean square for normal values).  Were all values of a row so moved, the outputs would differ by 1/40 of their norm per
projection, four of them in a row; few are, and 2 % of the output's norm is asked for."""
import os
import subprocess
import sys

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _block(pkg, width=256, gated=True, **kw):
    torch.manual_seed(3)
    block = pkg.MambaBlockInt2(width, gated=gated, threshold=3, **kw).to(DEV).init_weights()
    with torch.no_grad():
        block.conv_bias.normal_(std=0.1)
        block.post_norm.add_(torch.randn_like(block.post_norm) * 0.1)
        block.scale.mul_(0.5)
    return block


def _inputs(B, L, width, seed=0):
    g = torch.Generator().manual_seed(seed)
    h, x = (torch.randn(B, L, width, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
    return h, x


def _near(a, b, name):
    off = float((a.float() - b.float()).norm() / b.float().norm())
    assert off <= 0.02, (name, off)


@pytest.mark.parametrize("gated", [True, False])
def test_prompt_and_single_tokens_equal_the_whole_sequence(pkg, gated):
    block = _block(pkg, gated=gated).eval()
    h, x = _inputs(3, 70, 256)
    with torch.no_grad():
        whole = block(h, x)
        state = block.new_state(3)
        first = block(h[:, :64], x[:, :64], state)
        rest = [block.step(h[:, t], x[:, t], state) for t in range(64, 70)]
        for i, name in enumerate(("h", "normed")):
            _near(torch.cat([first[i], torch.stack([r[i] for r in rest], 1)], 1), whole[i], name)
        full = block.new_state(3)
        block(h, x, full)
    _near(state.conv, full.conv, "convolution state")
    _near(state.ssm, full.ssm, "scan state")


def test_sequences_of_unequal_length_equal_each_by_itself(pkg):
    block = _block(pkg).eval()
    lengths = [50, 1, 0, 33]
    h, x = _inputs(4, 50, 256)
    with torch.no_grad():
        state = block.new_state(4)
        out = block(h, x, state, torch.tensor(lengths, device=DEV))
        for b, n in enumerate(lengths):
            own = block.new_state(1)
            if n:
                alone = block(h[b:b + 1, :n], x[b:b + 1, :n], own)
                for i in (0, 1):
                    _near(out[i][b, :n], alone[i][0], f"sequence {b}")
                _near(state.ssm[b], own.ssm[0], "scan state")
            else:
                assert not state.ssm[b].any() and not state.conv[b].any()


def test_a_training_step_reaches_every_parameter(pkg):
    block = _block(pkg).train()
    before = {n: m.int2_layer.H_packed.clone() for n, m in block.named_children() if isinstance(m, pkg.BitLinearInt2)}
    pkg.set_all_int2_lr(block, 1.0)
    h, x = _inputs(2, 96, 256)
    h.requires_grad_(True)
    x.requires_grad_(True)
    out, normed = block(h, x)
    g = torch.Generator().manual_seed(1)
    torch.autograd.backward((out, normed), [torch.randn(out.shape, generator=g).to(out) for _ in range(2)])
    for name, p in block.named_parameters():
        if name.endswith("gamma"):
            continue
        assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.any(), name
    for t in (h, x):
        assert torch.isfinite(t.grad).all() and t.grad.any()
    for name, old in before.items():
        assert not torch.equal(getattr(block, name).int2_layer.H_packed, old), name


def test_the_example_learns_and_generates():
    r = subprocess.run([sys.executable, os.path.join(ROOT, "examples", "mamba_block.py"), "--width", "256", "--steps", "30"], capture_output=True, text=True,
                       timeout=600)
    assert r.returncode == 0, r.stderr[-2000:]
    first, last = (float(v) for v in r.stdout.split("loss ")[1].split(" over")[0].split(" -> "))
    assert last < first, r.stdout
