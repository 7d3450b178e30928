"""Trains a small gated-delta model on associative recall, then serves it.

A sequence holds pairs (key, value) of symbols and then asks for the values of
some of its keys; the model has to answer from its state.  Training runs the
layer norm, the gated delta rule with its backward and the clipping of the
global gradient norm; serving reads prompts of different lengths with one call
and answers token by token from a pool of states.

    python examples/delta_training.py [--steps 300] [--width 128] [--layers 2]
"""
import argparse
import os
import sys

import torch
import torch.nn as nn
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from orthossm_amd import GatedDeltaLayer, clip_grad_norm, layer_norm  # noqa: E402

SYMBOLS = 32
PAIRS, ASKED = 8, 8


class RecallModel(nn.Module):
    def __init__(self, width: int, layers: int, heads: int = 4):
        super().__init__()
        # a token is a pair: a key and its value, or a key and the blank that asks
        self.key, self.value = nn.Embedding(SYMBOLS, width), nn.Embedding(SYMBOLS + 1, width)
        self.layers = nn.ModuleList(GatedDeltaLayer(width, heads) for _ in range(layers))
        self.norm_weight, self.norm_bias = nn.Parameter(torch.ones(width)), nn.Parameter(torch.zeros(width))
        self.head = nn.Linear(width, SYMBOLS)

    def _finish(self, x):
        return self.head(layer_norm(x, self.norm_weight, self.norm_bias))

    def forward(self, keys, values, lengths=None):
        """Scores of every position, and the layers' states."""
        x, states = self.key(keys) + self.value(values), []
        for layer in self.layers:
            x, state = layer(x, lengths=lengths)
            states.append(state)
        return self._finish(x), states

    @torch.no_grad()
    def step(self, keys, values, pools, slots):
        x = self.key(keys) + self.value(values)
        for layer, pool in zip(self.layers, pools):
            x = layer.step(x, pool, slots)
        return self._finish(x)


def batch(gen, rows, device):
    """(keys, values with blanks where asked, answers) of ``rows`` sequences."""
    keys = torch.stack([torch.randperm(SYMBOLS, generator=gen)[:PAIRS] for _ in range(rows)])
    values = torch.randint(SYMBOLS, (rows, PAIRS), generator=gen)
    asked = torch.randint(PAIRS, (rows, ASKED), generator=gen)
    blanks = torch.full((rows, ASKED), SYMBOLS)
    return tuple(t.to(device) for t in (torch.cat([keys, keys.gather(1, asked)], 1), torch.cat([values, blanks], 1),
                                        values.gather(1, asked)))


def train(model, steps, gen, rows=64, lr=3e-3, limit=1.0, report=None):
    """Losses and gradient norms of every step, on the device."""
    device = model.head.weight.device
    opt = torch.optim.AdamW(model.parameters(), lr=lr)
    losses, norms = [], []
    for i in range(steps):
        keys, values, answers = batch(gen, rows, device)
        scores, _ = model(keys, values)
        loss = F.cross_entropy(scores[:, PAIRS:].flatten(0, 1), answers.flatten())
        opt.zero_grad(set_to_none=True)
        loss.backward()
        norms.append(clip_grad_norm([p.grad for p in model.parameters() if p.grad is not None], limit))
        opt.step()
        losses.append(loss.detach())
        if report and (i + 1) % report == 0:
            print(f"step {i + 1}: loss {loss.item():.4f}, gradient norm {norms[-1].item():.3f}", flush=True)
    return torch.stack(losses), torch.stack(norms)


@torch.no_grad()
def serve(model, gen, rows=8):
    """Share of right answers, one token at a time after prompts of different
    lengths, and the largest difference from scores of whole sequences."""
    device = model.head.weight.device
    keys, values, answers = batch(gen, rows, device)
    whole, _ = model(keys, values)
    lengths = PAIRS + torch.arange(rows, device=device) % ASKED       # some of the questions are in the prompt
    _, states = model(keys, values, lengths=lengths)
    # the states move into the slots of a larger pool, in another order
    slots = torch.randperm(rows + 3, generator=gen)[:rows].to(device)
    pools = []
    for layer, state in zip(model.layers, states):
        pool = layer.new_state(rows + 3)
        pool[slots] = state
        pools.append(pool)
    right, worst, asked = 0, 0.0, 0
    at = torch.arange(rows, device=device)
    for t in range(ASKED):
        pos = lengths + t
        live = pos < PAIRS + ASKED
        pos = pos.clamp(max=PAIRS + ASKED - 1)
        scores = model.step(keys[at, pos], values[at, pos], pools, torch.where(live, slots, -1))
        right += ((scores.argmax(-1) == answers[at, pos - PAIRS]) & live).sum().item()
        worst = max(worst, (scores - whole[at, pos])[live].abs().max().item() if live.any() else 0.0)
        asked += live.sum().item()
    return right / asked, worst


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--steps", type=int, default=300)
    ap.add_argument("--width", type=int, default=128)
    ap.add_argument("--layers", type=int, default=2)
    a = ap.parse_args()
    torch.manual_seed(0)
    gen = torch.Generator().manual_seed(0)
    model = RecallModel(a.width, a.layers).to("cuda")
    train(model, a.steps, gen, report=max(1, a.steps // 10))
    share, worst = serve(model, gen, rows=64)
    print(f"served token by token: {share:.3f} of the answers right; scores within {worst:.1e} of whole sequences")


if __name__ == "__main__":
    main()
