#!/usr/bin/env python3
"""A click model around the embedding table, on synthetic ids: the pulled rows are normalised and dropped out on their way to
bfloat16, go through two layers joined by residual + dropout + layer norm, and their gradient goes back into the table.

    python examples/train_dense.py [--steps 200] [--samples 2048]
"""
import argparse
import os
import sys

import numpy as np
import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
from hetuctr_amd import capi, nn, workloads  # noqa: E402

WIDTH, HIDDEN = 32, 512


class Model(torch.nn.Module):
    """Weights in float32; the products run in bfloat16, the stream between the layers stays in float32."""

    def __init__(self, fields):
        super().__init__()
        make = lambda *shape: torch.nn.Parameter(torch.randn(*shape) / shape[-1] ** 0.5)
        self.norms = torch.nn.ParameterList([torch.nn.Parameter(torch.full((n,), v)) for n in (WIDTH, HIDDEN) for v in (1.0, 0.0)])
        self.first, self.second, self.last = make(HIDDEN, fields * WIDTH), make(HIDDEN, HIDDEN), make(1, HIDDEN)

    def forward(self, rows, samples, step):
        """rows: float32 [samples * fields, WIDTH]; step None: inference, nothing is dropped"""
        drop = lambda layer, p: None if step is None else nn.Drop(p, seed=layer, step=step)
        h = nn.layer_norm(rows, self.norms[0], self.norms[1], drop=drop(1, 0.05), dtype=torch.bfloat16)
        stream = F.linear(h.view(samples, -1), self.first.bfloat16()).float()
        branch = F.linear(F.gelu(stream).bfloat16(), self.second.bfloat16())
        y, _ = nn.dropout_add_layer_norm(branch, stream, self.norms[2], self.norms[3], drop=drop(2, 0.1))
        return F.linear(nn.dropout(y, drop(3, 0.1)), self.last.bfloat16()).float().view(-1)


def train(steps=200, samples=2048, report=None, seed=0):
    """The loss of every step."""
    ids = workloads.KeyStream(dict(workloads.CONFIGS["cfg2"], rows=200_000, samples=samples), seed=seed)
    n = ids.n
    capi.seed(seed)
    torch.manual_seed(seed)
    table = capi.Table(0, 1, 0, "127.0.0.1", 23456, ids.rows, WIDTH, 0, 0, np.zeros(ids.rows, np.uint8),
                       np.arange(ids.rows, dtype=np.int64), ("Normal", 0.0, 0.1), 0.5)
    model = Model(ids.fields).cuda()
    optimizer = torch.optim.Adam(model.parameters(), lr=1e-3)
    # whether a sample is clicked hangs on its ids alone: the sign of the sum of a number per id
    taste = torch.randn(ids.rows, device="cuda")
    rows, gradient, losses = None, None, []
    for step in range(steps):
        keys = torch.from_numpy(ids.batch()).cuda()
        clicked = (taste[keys].view(samples, -1).sum(1) > 0).float()
        rows = torch.empty((n, WIDTH), device="cuda")
        table.preprocess(keys.data_ptr(), n)
        # the gradient of the batch before, the rows of this one
        table.push_pull(0 if gradient is None else gradient.data_ptr(), rows.data_ptr())
        rows.requires_grad_()
        loss = F.binary_cross_entropy_with_logits(model(rows, samples, step), clicked)
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        gradient = rows.grad
        losses.append(loss.item())
        if report and step % report == 0:
            print("step %4d  loss %.4f" % (step, losses[-1]), flush=True)
    table.close()
    return losses


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--samples", type=int, default=2048)
    a = ap.parse_args()
    train(a.steps, a.samples, report=max(1, a.steps // 10))
