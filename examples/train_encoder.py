"""Trains a small text encoder and its fixed-fan-in output layer end to end on made-up data.

A text is a few tokens; a label is right for it if the label's own token is among them.
The encoder (token embedding, two pre-norm feed-forward layers, mean over the text) takes
haste_amd's LayerNorm with the residual sum joined in, the output layer is a GroupFixedFanIn.
The encoder's bf16 weights are stepped by AdamW with 8-bit states, clipped by the norm of all
their gradients, which stays on the device; the output layer's by SRSgd.

    python examples/train_encoder.py [--steps 200] [--state-bits 8]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from haste_amd.layer_norm import LayerNorm  # noqa: E402
from haste_amd.optim_adamw import AdamW, grad_norm  # noqa: E402
from haste_amd.optim_sr import SRSgd  # noqa: E402
from haste_amd.rewire import GroupFixedFanIn  # noqa: E402

TOKENS, LABELS, WIDTH, HIDDEN, LENGTH, BATCH = 256, 4096, 256, 512, 8, 256


class FeedForward(torch.nn.Module):
    def __init__(self, width, hidden, **kw):
        super().__init__()
        self.norm = LayerNorm(width, **kw)
        self.up = torch.nn.Linear(width, hidden, **kw)
        self.down = torch.nn.Linear(hidden, width, **kw)

    def forward(self, delta, stream):
        """What the layer adds to the stream, and the stream with `delta` added to it."""
        x, stream = self.norm(delta, stream)
        return self.down(torch.nn.functional.gelu(self.up(x))), stream


class Encoder(torch.nn.Module):
    def __init__(self, **kw):
        super().__init__()
        self.tokens = torch.nn.Embedding(TOKENS, WIDTH, **kw)
        self.places = torch.nn.Parameter(0.02 * torch.randn(LENGTH, WIDTH, **kw))
        self.layers = torch.nn.ModuleList(FeedForward(WIDTH, HIDDEN, **kw) for _ in range(2))
        self.norm = LayerNorm(WIDTH, **kw)

    def forward(self, ids):
        delta, stream = self.tokens(ids), self.places.expand(ids.shape[0], -1, -1)
        for layer in self.layers:
            delta, stream = layer(delta, stream)
        return self.norm(delta, stream)[0].mean(1)


def batch(owner, g, device):
    """Token ids [BATCH, LENGTH] and the 0/1 labels [BATCH, LABELS] they make right."""
    ids = torch.randint(0, TOKENS, (BATCH, LENGTH), generator=g, device=device)
    has = torch.zeros(BATCH, TOKENS, device=device).scatter_(1, ids, 1.0)
    return ids, has[:, owner]


def train(steps=200, state_bits=8, seed=0, device="cuda"):
    """The loss (binary cross entropy, summed over the labels of a text) of every tenth step."""
    torch.manual_seed(seed)
    g = torch.Generator(device=device).manual_seed(seed)
    kw = dict(device=device, dtype=torch.bfloat16)
    owner = torch.randint(0, TOKENS, (LABELS,), generator=g, device=device)
    encoder = Encoder(**kw)
    output = GroupFixedFanIn(WIDTH, LABELS, 64, group_size=32, prune_mode="fraction",
                             rewire_fraction=0.15, **kw).to(device)
    adamw = AdamW(encoder.parameters(), lr=3e-3, weight_decay=0.01, state_bits=state_bits)
    sgd = SRSgd(output.parameters(), lr=0.02, momentum=0.9)
    losses = []
    for step in range(steps):
        ids, right = batch(owner, g, device)
        logits = output(encoder(ids))
        loss = torch.nn.functional.binary_cross_entropy_with_logits(
            logits.float(), right, reduction="sum") / BATCH
        adamw.zero_grad()
        sgd.zero_grad()
        loss.backward()
        _, coef = grad_norm([p.grad for p in encoder.parameters()], max_norm=1.0)
        adamw.step(grad_scale=coef)
        sgd.step()
        if step % 10 == 0 or step == steps - 1:
            losses.append(loss.detach())
    return [float(x) for x in losses]


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--state-bits", type=int, default=8, choices=(8, 32))
    a = ap.parse_args()
    for k, x in enumerate(train(a.steps, a.state_bits)):
        print(f"step {min(10 * k, a.steps - 1):4d}  loss {x:.4f}")
