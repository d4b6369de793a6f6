#!/usr/bin/env python3
"""The next item of a history, among all items, on synthetic clicks: the pulled rows of a history's last items are normalised, go through a gated
feed-forward block, and score every item by a softmax cross entropy that holds no matrix of logits.  The gradients, those of
the rows among them, are clipped together; the rows' go back into the table.

    python examples/train_next_item.py [--steps 200] [--samples 2048]
"""
import argparse
import os
import sys

import numpy as np
import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
from hetuctr_amd import capi, nn  # noqa: E402

ITEMS, WIDTH, HIDDEN, HISTORY = 50_000, 64, 256, 4


class Model(torch.nn.Module):
    """Weights in float32; the products run in bfloat16."""

    def __init__(self):
        super().__init__()
        make = lambda *shape: torch.nn.Parameter(torch.randn(*shape) / shape[-1] ** 0.5)
        self.scale, self.shift = torch.nn.Parameter(torch.ones(WIDTH)), torch.nn.Parameter(torch.zeros(WIDTH))
        self.gate, self.up, self.down = make(HIDDEN, HISTORY * WIDTH), make(HIDDEN, HISTORY * WIDTH), make(WIDTH, HIDDEN)
        self.items, self.popular = make(ITEMS, WIDTH), torch.nn.Parameter(torch.zeros(ITEMS))

    def forward(self, rows, samples, target):
        """The loss of each sample; rows: float32 [samples * HISTORY, WIDTH]"""
        h = nn.layer_norm(rows, self.scale, self.shift, dtype=torch.bfloat16).view(samples, -1)
        h = nn.gated_linear(h, self.gate.bfloat16(), self.up.bfloat16())
        return nn.linear_cross_entropy(F.linear(h, self.down.bfloat16()), self.items.bfloat16(), target, self.popular)


def clicks(samples, rng):
    """Histories and what comes next: item i is followed by one of a few that hang on i; some samples end before that (-100)"""
    history = rng.zipf(1.2, size=(samples, HISTORY)) % ITEMS
    following = (history[:, -1] * 7919 + rng.integers(0, 4, samples)) % ITEMS
    following[rng.random(samples) < 0.1] = -100
    return history.astype(np.int64), following.astype(np.int64)


def train(steps=200, samples=2048, report=None, seed=0, max_norm=1.0):
    """(loss, norm of the gradients before they were clipped) of every step."""
    rng = np.random.default_rng(seed)
    n = samples * HISTORY
    capi.seed(seed)
    torch.manual_seed(seed)
    table = capi.Table(0, 1, 0, "127.0.0.1", 23456, ITEMS, WIDTH, 0, 0, np.zeros(ITEMS, np.uint8), np.arange(ITEMS, dtype=np.int64),
                       ("Normal", 0.0, 0.1), 0.5)
    model = Model().cuda()
    parameters = list(model.parameters())
    optimizer = torch.optim.Adam(parameters, lr=1e-3)
    gradient, said = None, []
    for step in range(steps):
        history, following = clicks(samples, rng)
        keys, target = torch.from_numpy(history).cuda().flatten(), torch.from_numpy(following).cuda()
        rows = torch.empty((n, WIDTH), device="cuda")
        table.preprocess(keys.data_ptr(), n)
        # the gradient of the batch before, the rows of this one
        table.push_pull(0 if gradient is None else gradient.data_ptr(), rows.data_ptr())
        rows.requires_grad_()
        loss = model(rows, samples, target).sum() / (target != -100).sum()
        optimizer.zero_grad()
        loss.backward()
        norm = nn.clip_gradients([p.grad for p in parameters] + [rows.grad], max_norm)
        optimizer.step()
        gradient = rows.grad
        said.append((loss.item(), norm.item()))
        if report and step % report == 0:
            print("step %4d  loss %.4f  norm %.4f" % (step, *said[-1]), flush=True)
    table.close()
    return said


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--samples", type=int, default=2048)
    a = ap.parse_args()
    train(a.steps, a.samples, report=max(1, a.steps // 10))
