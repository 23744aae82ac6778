"""Trains a gated encoder and its fixed-fan-in output layer under a softmax loss, and answers.

A text is a few tokens, and the one with the largest number makes its label right.  Every operator of the encoder and of the loss is haste_amd's: the token embedding scaled
by the root of its width, LayerNorm with the residual sum joined in, the gated feed-forward block,
the grouped fixed-fan-in layer, and the log probabilities of the right labels.  AdamW steps the
encoder, SRSgd the output layer; the answers are the layer's likeliest labels.

    python examples/train_softmax.py [--steps 200]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from haste_amd import ops  # noqa: E402
from haste_amd.embedding import Embedding  # noqa: E402
from haste_amd.gated_mlp import GatedMLP  # noqa: E402
from haste_amd.layer_norm import LayerNorm  # noqa: E402
from haste_amd.optim_adamw import AdamW, grad_norm  # noqa: E402
from haste_amd.optim_sr import SRSgd  # noqa: E402
from haste_amd.rewire import GroupFixedFanIn  # noqa: E402

TOKENS, LABELS, WIDTH, HIDDEN, LENGTH, BATCH = 250, 4100, 256, 384, 8, 256


class Encoder(torch.nn.Module):
    def __init__(self, layers=2, **kw):
        super().__init__()
        self.tokens = Embedding(TOKENS, WIDTH, padding_idx=0, scale=WIDTH ** 0.5, **kw)
        torch.nn.init.normal_(self.tokens.weight, std=WIDTH ** -0.5)
        self.norms = torch.nn.ModuleList(LayerNorm(WIDTH, **kw) for _ in range(layers + 1))
        self.blocks = torch.nn.ModuleList(GatedMLP(WIDTH, HIDDEN, **kw) for _ in range(layers))

    def forward(self, ids):
        stream = self.tokens(ids)
        x = self.norms[0](stream)
        for norm, block in zip(self.norms[1:], self.blocks):
            x, stream = norm(block(x), stream)
        return x.mean(1)


class Model(torch.nn.Module):
    def __init__(self, **kw):
        super().__init__()
        self.encoder = Encoder(**kw)
        self.output = GroupFixedFanIn(WIDTH, LABELS, 64, group_size=32, prune_mode="fraction",
                                      rewire_fraction=0.15, **kw)

    def forward(self, ids):
        return self.output(self.encoder(ids))


def batch(g, device):
    """Token ids [BATCH, LENGTH], 0 where a text has ended, and the right label [BATCH, 1]."""
    ids = torch.randint(1, TOKENS, (BATCH, LENGTH), generator=g, device=device)
    ends = torch.randint(1, LENGTH + 1, (BATCH, 1), generator=g, device=device)
    ids = torch.where(torch.arange(LENGTH, device=device) < ends, ids, 0)
    return ids, ids.amax(1, keepdim=True) * 16


def train(steps=200, seed=0, device="cuda"):
    """The model, the mean loss of every tenth step, and how many of the last batch's answers are
    right."""
    torch.manual_seed(seed)
    g = torch.Generator(device=device).manual_seed(seed)
    model = Model(device=device, dtype=torch.bfloat16).to(device)
    weights = list(model.encoder.parameters())
    adamw = AdamW(weights, lr=2e-3, weight_decay=0.01)
    sgd = SRSgd(model.output.parameters(), lr=1.0, momentum=0.9)
    losses = []
    for step in range(steps):
        ids, right = batch(g, device)
        loss = -ops.label_log_probs(model(ids), right).log_probs.mean()
        adamw.zero_grad()
        sgd.zero_grad()
        loss.backward()
        _, coef = grad_norm([p.grad for p in weights], max_norm=1.0)
        adamw.step(grad_scale=coef)
        sgd.step()
        if step % 10 == 0 or step == steps - 1:
            losses.append(loss.detach())
    with torch.no_grad():
        answers = ops.label_log_probs(model(ids), top=5).top_labels
    return model, [float(x) for x in losses], float((answers[:, :1] == right).float().mean())


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=200)
    a = ap.parse_args()
    _, losses, share = train(a.steps)
    for k, x in enumerate(losses):
        print(f"step {min(10 * k, a.steps - 1):4d}  loss {x:.4f}")
    print(f"right answers: {100 * share:.1f} %")
