"""A small recurrent language model trained on labels and on a teacher's top logits.

    python examples/train_head.py [--steps 60] [--vocab 2000] [--width 256]

Embedding -> layer norm -> gated RG-LRU -> residual -> layer norm -> output head, whose losses
(cross entropy on the next token, distillation from a teacher's top 16 logits) come straight
from the hidden states.  The data are a random Markov chain and the
teacher is the chain itself, so both losses have a known floor and fall towards it.  Needs an
MI355X and the built library.
"""
from __future__ import annotations

import argparse
import math
import pathlib
import sys

import torch

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1] / "mlx-recurrence_amd"))
import mlx_recurrence_amd as mr  # noqa: E402

TOP = 16        # teacher entries a token
PROMPT = 8      # first tokens of a sequence, which are read but not trained on
IGNORE = -100


class Model:
    def __init__(self, vocab, width, device, seed=0):
        g = torch.Generator(device=device).manual_seed(seed)

        def p(*shape, scale):
            return (torch.randn(shape, generator=g, device=device) * scale).requires_grad_(True)

        def const(value):
            return torch.full((width,), value, device=device).requires_grad_(True)

        self.embed = p(vocab, width, scale=1.0)
        self.gates = p(width, 3 * width, scale=width ** -0.5)
        self.out = p(width, width, scale=width ** -0.5)
        self.lam = const(-4.0)
        self.norm1, self.bias1, self.norm2, self.bias2 = const(1.0), const(0.0), const(1.0), const(0.0)
        self.head = p(vocab, width, scale=width ** -0.5)

    def parameters(self):
        return [t for t in vars(self).values() if isinstance(t, torch.Tensor)]

    def hidden(self, tokens):
        """[B, L, width] bf16, what the head reads."""
        x = self.embed[tokens]
        h = mr.layer_norm(x, self.norm1, self.bias1, out_dtype=torch.bfloat16)
        r, i, u = (h @ self.gates.to(torch.bfloat16)).chunk(3, dim=-1)
        y = mr.rglru_gated_scan(r, torch.sigmoid(i), u, self.lam)
        x = x + y @ self.out
        return mr.layer_norm(x, self.norm2, self.bias2, out_dtype=torch.bfloat16)


def chain(vocab, device, seed=1):
    """A Markov chain: for each token its TOP successors and their logits."""
    g = torch.Generator(device=device).manual_seed(seed)
    ids = torch.randint(0, vocab, (vocab, 1), generator=g, device=device)
    steps = torch.randperm(vocab, generator=g, device=device)[:TOP]
    return (ids + steps) % vocab, 2 * torch.randn((vocab, TOP), generator=g, device=device)


def sample(ids, logits, batch, length, g):
    p = torch.softmax(logits, -1)
    tokens = [torch.randint(0, len(ids), (batch,), generator=g, device=ids.device)]
    for _ in range(length):
        pick = torch.multinomial(p[tokens[-1]], 1, generator=g)[:, 0]
        tokens.append(ids[tokens[-1], pick])
    return torch.stack(tokens, 1)


def train(steps=60, vocab=2000, width=256, batch=16, length=128, temperature=2.0, report=print):
    device = torch.device("cuda:0")
    ids, logits = chain(vocab, device)
    g = torch.Generator(device=device).manual_seed(2)
    model = Model(vocab, width, device)
    optimiser = torch.optim.Adam(model.parameters(), lr=5e-3)
    history = []
    for step in range(steps):
        tokens = sample(ids, logits, batch, length, g)
        inputs, labels = tokens[:, :-1], tokens[:, 1:].clone()
        labels[:, :PROMPT] = IGNORE
        t_ids = ids[inputs].masked_fill((labels == IGNORE)[..., None], -1)
        hidden = model.hidden(inputs)
        head = model.head.to(torch.bfloat16)
        ce = mr.linear_cross_entropy(hidden, head, labels, ignore_index=IGNORE, z_loss=1e-4)
        kd = mr.linear_distillation(hidden, head, logits[inputs], t_ids, temperature=temperature)
        optimiser.zero_grad(set_to_none=True)
        (ce + kd).backward()
        optimiser.step()
        history.append((ce.detach(), kd.detach()))
        if step % 10 == 0 or step == steps - 1:
            report(f"step {step:4d}  cross entropy {float(ce.detach()):.3f}  distillation {float(kd.detach()):.3f}")
    p = torch.softmax(logits, -1)
    report(f"floor      cross entropy {float(-(p * p.log()).sum(-1).mean()):.3f}  distillation 0; "
           f"an untrained head: {math.log(vocab):.3f}")
    return [(float(a), float(b)) for a, b in history]


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--vocab", type=int, default=2000)
    ap.add_argument("--width", type=int, default=256)
    a = ap.parse_args()
    train(a.steps, a.vocab, a.width)
