"""Train a small language model, then distil it into a smaller one.

Both models end in a head whose logits are never formed: the teacher trains
with ops.linear_cross_entropy (padding ignored, a penalty on the squared
log-partition), the student with ops.linear_distillation on the teacher's top
logits plus a share of the cross entropy, and both are scored by the losses of
single tokens. Muon takes the matrices of the blocks, AdamW the rest. The data
is a seeded random Markov chain.

    python pytorch-opt_amd/examples/distill_lm.py            # a GPU, under bfloat16 autocast
    python pytorch-opt_amd/examples/distill_lm.py --device cpu --steps 5
"""

from __future__ import annotations

import argparse
import os
import sys

import torch
from torch import nn
from torch.nn import functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from pytorch_opt import Muon, matrix_param_groups, ops  # noqa: E402

IGNORE = -100


class Block(nn.Module):
    """Causal self-attention in plain products, then a two-layer MLP."""

    def __init__(self, d, heads):
        super().__init__()
        self.heads = heads
        self.norm1, self.norm2 = nn.LayerNorm(d), nn.LayerNorm(d)
        self.qkv, self.out = nn.Linear(d, 3 * d, bias=False), nn.Linear(d, d, bias=False)
        self.up, self.down = nn.Linear(d, 4 * d, bias=False), nn.Linear(4 * d, d, bias=False)

    def forward(self, x):
        b, t, d = x.shape
        q, k, v = (y.view(b, t, self.heads, -1).transpose(1, 2).float() for y in self.qkv(self.norm1(x)).chunk(3, -1))
        score = (q @ k.transpose(2, 3).contiguous()) * q.shape[-1] ** -0.5
        later = torch.ones(t, t, dtype=torch.bool, device=x.device).triu(1)
        mixed = score.masked_fill(later, float("-inf")).softmax(-1) @ v
        x = x + self.out(mixed.to(x.dtype).transpose(1, 2).reshape(b, t, d))
        return x + self.down(F.gelu(self.up(self.norm2(x))))


class Model(nn.Module):
    """Hidden states of a small decoder; `head` is the output weight."""

    def __init__(self, vocab, d, layers, heads=4):
        super().__init__()
        self.embed = nn.Embedding(vocab, d)
        self.blocks = nn.ModuleList(Block(d, heads) for _ in range(layers))
        self.norm = nn.LayerNorm(d)
        self.head = nn.Parameter(torch.randn(vocab, d) * d ** -0.5)

    def forward(self, tokens):
        x = self.embed(tokens)
        for block in self.blocks:
            x = block(x)
        return self.norm(x)


def batch(chain, rows, length, generator):
    """Sequences of the chain and their next tokens; the last quarter of every
    other one is padding, which the losses leave out."""
    tokens = torch.randint(0, chain.shape[0], (rows, 1), generator=generator)
    for _ in range(length):
        pick = torch.randint(0, chain.shape[1], (rows, 1), generator=generator)
        tokens = torch.cat([tokens, chain[tokens[:, -1:]].gather(2, pick[..., None])[..., 0]], 1)
    targets = tokens[:, 1:].clone()
    targets[::2, -(length // 4):] = IGNORE
    return tokens[:, :-1], targets


def optimizer(model, lr):
    matrices = [name for name, m in model.named_modules() if isinstance(m, nn.Linear)]
    return Muon(matrix_param_groups(model, matrices, lr=lr, adamw_lr=lr / 5))


def top_logits(model, tokens, k):
    """The teacher's k largest logits and their tokens."""
    with torch.no_grad():
        logits = model(tokens).float() @ model.head.float().T
        values, index = logits.topk(k, -1)
        return values, index


def autocast(device):
    return torch.autocast("cuda", dtype=torch.bfloat16, enabled=device.startswith("cuda"))


def train(model, steps, data, lr, loss_of):
    opt, seen = optimizer(model, lr), []
    for _ in range(steps):
        tokens, targets = data()
        with autocast(tokens.device.type):
            loss = loss_of(model, tokens, targets)
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        seen.append(loss.detach())
    return torch.stack(seen).tolist()


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--device", default="cuda")
    ap.add_argument("--vocab", type=int, default=2000)
    ap.add_argument("--d", type=int, default=256)
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--rows", type=int, default=16)
    ap.add_argument("--length", type=int, default=128)
    ap.add_argument("--top", type=int, default=16)
    ap.add_argument("--temperature", type=float, default=2.0)
    a = ap.parse_args(argv)
    if a.device.startswith("cuda") and not ops.load_native():
        raise SystemExit("the HIP library did not load")
    torch.manual_seed(0)
    g = torch.Generator().manual_seed(1)
    chain = torch.randint(0, a.vocab, (a.vocab, 4), generator=g)  # four successors each

    def data():
        tokens, targets = batch(chain, a.rows, a.length, g)
        return tokens.to(a.device), targets.to(a.device)

    def hard(model, tokens, targets):
        return ops.linear_cross_entropy(model(tokens), model.head, targets, ignore_index=IGNORE, z_loss=1e-4)

    teacher = Model(a.vocab, a.d, 2).to(a.device)
    taught = train(teacher, a.steps, data, 0.02, hard)

    def soft(model, tokens, targets):
        values, index = top_logits(teacher, tokens, a.top)
        index = index.masked_fill(targets[..., None] == IGNORE, -1)
        hidden = model(tokens)
        return 0.9 * ops.linear_distillation(hidden, model.head, values, index, temperature=a.temperature) \
            + 0.1 * ops.linear_cross_entropy(hidden, model.head, targets, ignore_index=IGNORE)

    student = Model(a.vocab, a.d // 2, 1).to(a.device)
    learned = train(student, a.steps, data, 0.02, soft)

    tokens, targets = data()
    with torch.no_grad(), autocast(a.device):
        scores = {name: ops.linear_cross_entropy(m(tokens), m.head, targets, ignore_index=IGNORE, reduction="none")
                  for name, m in (("teacher", teacher), ("student", student))}
    kept = targets != IGNORE
    result = {"teacher": taught, "student": learned,
              **{f"{n}_held_out": float(s[kept].mean()) for n, s in scores.items()}}
    print(f"teacher: loss {taught[0]:.3f} -> {taught[-1]:.3f}, student: {learned[0]:.3f} -> {learned[-1]:.3f}; "
          f"held out, nats per token: teacher {result['teacher_held_out']:.3f}, student "
          f"{result['student_held_out']:.3f}")
    return result


if __name__ == "__main__":
    main()
