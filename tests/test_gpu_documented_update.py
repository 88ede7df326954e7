"""The update loop that the documents show, run as it is written: lists made
once, design steps whose gradients the lists take."""
import glob
import os
import re

import pytest
import torch

from tests.conftest import ROOT
from tests.test_gpu_loss_and_update import _design

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -24


def documented():
    """The one Python block of the documents that makes an Adam list."""
    text = "".join(open(p, encoding="utf-8").read() for p in sorted(glob.glob(os.path.join(ROOT, "*.md"))))
    blocks = re.findall(r"```python\n(from bindcraft2_amd import ops\n.*?)```", text, re.S)
    blocks = [b for b in blocks if "ops.Adam(" in b]
    assert len(blocks) == 1
    return blocks[0]


class Recorded:
    """A design step that keeps what each backward was given and gave."""

    def __init__(self, step):
        self.step, self.calls = step, []

    def forward(self, logits, *args, **kwargs):
        return self.step.forward(logits, *args, **kwargs)

    def backward(self, cts, logits, *args, **kwargs):
        d = self.step.backward(cts, logits, *args, **kwargs)
        self.calls.append((logits.clone(), d.clone()))
        return d


def test_documented_loop(cuda):
    """Three steps of two states.  Every step's states are held to the update in
    64 bits by the gradients that this step's backward gave: the moments' and
    the move's roundings (18 half steps of a move, and 5 of the terms of the
    first moment at its rate), the norm's and the clipping's among them, summed
    over the steps, and two roundings of the state a step."""
    n, steps = 32, 3
    step, gen = Recorded(_design(n)), torch.Generator("cuda").manual_seed(9)
    states = [torch.randn(n, 20, generator=gen, device="cuda") for _ in range(2)]
    start = [s.double() for s in states]
    at, one = torch.arange(n, device="cuda", dtype=torch.float32), torch.ones(n, device="cuda")
    names = {
        "torch": torch, "step": step, "states": states, "steps": steps,
        "exp_avg": [torch.zeros_like(s) for s in states],
        "exp_avg_sq": [torch.zeros_like(s) for s in states],
        "flags": torch.ones(n, dtype=torch.uint8, device="cuda"),
        "scalars": torch.tensor([1.0, 0.0, 1.0, 1.0], device="cuda"), "ids": [at, one, one, one],
        "seq_mask": one, "seeds": torch.arange(12, dtype=torch.int64).to(torch.uint32).to("cuda"),
        "bins": torch.randint(-1, 64, (n, n), generator=gen, device="cuda", dtype=torch.int32),
        "weight": torch.full((n, n), -100.0 / n, device="cuda")}
    exec(documented(), names)
    torch.cuda.synchronize()
    assert len(step.calls) == steps * len(states)
    m = [torch.zeros_like(s) for s in start]
    v, terms, tol = ([torch.zeros_like(s) for s in start] for _ in range(3))
    now = start
    for t in range(1, steps + 1):
        calls = step.calls[(t - 1) * len(states):t * len(states)]
        for (x, _), s, bound in zip(calls, now, tol):
            assert ((x.double() - s).abs() <= bound).all(), f"states before step {t}"
        grads = [d.double() for _, d in calls]
        norm = torch.sqrt(sum(g.square().sum() for g in grads)).item()
        assert norm > 1.0  # it clips
        for k, g in enumerate(grads):
            g = g / norm
            m[k] = 0.9 * m[k] + 0.1 * g
            v[k] = 0.999 * v[k] + 0.001 * g * g
            terms[k] = 0.9 * terms[k] + 0.1 * g.abs()
            scale = 0.1 / (1 - 0.9 ** t) / ((v[k] / (1 - 0.999 ** t)).sqrt() + 1e-8)
            now[k] = now[k] - scale * m[k]
            # t: the moments carry their roundings from step to step
            tol[k] = tol[k] + HALF * (t * scale * (18 * m[k].abs() + 5 * terms[k]) + 2 * now[k].abs()
                                      + 2 * (scale * m[k]).abs())
    assert abs(names["norm"].item() - norm) <= 3 * HALF * norm
    for s, want, bound in zip(states, now, tol):
        assert ((s.double() - want).abs() <= bound).all()
