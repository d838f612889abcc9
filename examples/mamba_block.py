"""Two Mamba blocks over INT2 projections, trained for a few steps on a synthetic task and then run as a generator.

    python examples/mamba_block.py [--width 512] [--steps 30]

The task: the next token is a fixed permutation of this one, and which of two permutations the sequence's first token says.  The projections'
ternary weights move by their own hysteresis rule in the backward pass; everything else takes AdamW steps.  Generation takes a batch of
prompts of unequal length through `forward` with a state, then goes on token by token with `step`.
"""
import argparse
import importlib.util
import os
import sys

import torch

TOKENS = 34
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def load_package():
    """The package; its directory name has a hyphen, so it is loaded by path."""
    name = "elleci_training_vast_b200"
    if name not in sys.modules:
        folder = os.path.join(ROOT, "elleci-training-vast_b200")
        spec = importlib.util.spec_from_file_location(name, os.path.join(folder, "__init__.py"), submodule_search_locations=[folder])
        module = importlib.util.module_from_spec(spec)
        sys.modules[name] = module
        spec.loader.exec_module(module)
    return sys.modules[name]


class Blocks(torch.nn.Module):
    def __init__(self, pkg, width, depth):
        super().__init__()
        self.embed = torch.nn.Embedding(TOKENS, width)
        self.head = torch.nn.Linear(width, TOKENS)
        self.first_norm = torch.nn.Parameter(torch.ones(width))
        self.blocks = torch.nn.ModuleList(pkg.MambaBlockInt2(width, gated=True, threshold=3) for _ in range(depth))

    def _start(self, ids):
        h = self.embed(ids)
        x = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6) * self.first_norm
        return h.to(torch.bfloat16), x.to(torch.bfloat16)

    def forward(self, ids, states=None, lengths=None):
        h, x = self._start(ids)
        for i, block in enumerate(self.blocks):
            h, x = block(h, x, None if states is None else states[i], lengths)
        return self.head(x.float())

    def step(self, ids, states):
        h, x = self._start(ids)
        for block, state in zip(self.blocks, states):
            h, x = block.step(h, x, state)
        return self.head(x.float())


def walks(rules, batch, length, generator):
    """Sequences whose first token is 0 or 1 and says which of the two permutations the rest follows."""
    dev = rules.device
    rule = torch.randint(0, 2, (batch,), generator=generator, device=dev)
    ids = [rule, torch.randint(2, TOKENS, (batch,), generator=generator, device=dev)]
    while len(ids) < length:
        ids.append(rules[rule, ids[-1]])
    return torch.stack(ids, 1)


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--width", type=int, default=512)
    ap.add_argument("--steps", type=int, default=30)
    args = ap.parse_args()
    pkg = load_package()
    torch.manual_seed(0)
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(0)
    rules = torch.stack([torch.cat([torch.arange(2, device=dev), 2 + torch.randperm(TOKENS - 2, generator=gen, device=dev)]) for _ in range(2)])
    model = Blocks(pkg, args.width, 2).to(dev)
    for block in model.blocks:
        block.init_weights()
    opt = torch.optim.AdamW(pkg.get_non_int2_params(model), lr=1e-2)
    pkg.set_all_int2_lr(model, 1e-2)
    losses = []
    for step in range(args.steps):
        ids = walks(rules, 16, 65, gen)
        loss = torch.nn.functional.cross_entropy(model(ids[:, :-1]).flatten(0, 1), ids[:, 1:].flatten())
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        losses.append(loss.item())
    print(f"loss {losses[0]:.3f} -> {losses[-1]:.3f} over {args.steps} steps")

    model.eval()
    with torch.no_grad():
        lengths = torch.tensor([64, 40, 7, 23], device=dev)
        ids, at = walks(rules, 4, 80, gen), torch.arange(4, device=dev)
        states = [b.new_state(4) for b in model.blocks]
        out = model(ids[:, :64], states, lengths)[at, lengths - 1]
        right = 0
        for i in range(16):
            token = out.argmax(-1)
            right += int((token == ids[at, lengths + i]).sum())
            out = model.step(token, states)
    print(f"{right} of 64 generated tokens follow their sequence's rule")


if __name__ == "__main__":
    main()
