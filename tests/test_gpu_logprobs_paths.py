"""Log-probabilities where a path's own steps matter: f32 rows that a whole
wave holds with alternatives from its list, by ties, -inf, NaN and rows left
out and for every way of bounding the list; gradients in place where a row is
divided among workgroups."""
import math

import pytest
import torch

from tests.test_gpu_logprobs import TYPES, logits, special, verify
from bindcraft2_amd import ops

pytestmark = pytest.mark.gpu
HELD = [257, 300, 509, 512]  # f32 classes that a wave's lanes hold, two vectors each


@pytest.mark.parametrize("v", HELD)
def test_special_rows_of_a_wave(cuda, v):
    print(f"special rows of a wave v={v}", flush=True)
    x, at, g = special(v, torch.float32)
    de, dl = (torch.randn(16, generator=g, device="cuda") for _ in range(2))
    for top in (1, 5, 7, 32):
        op = ops.LogProbs(top)
        dt = torch.randn(16, top, generator=g, device="cuda")
        for targets in (at, None):
            out, save = op.forward(x, targets)
            verify(x, targets, top, out)
        out, save = op.forward(x, at)
        verify(x, at, top, out, op.backward((dl, de, dt), x, at, out[3], save), (dl, de, dt))


@pytest.mark.parametrize("v", HELD)
def test_ties_and_orders_of_a_wave(cuda, v):
    print(f"ties of a wave v={v}", flush=True)
    x, g = logits(7, v, torch.float32, v)
    x[0] = torch.arange(v, device="cuda")
    x[1] = -torch.arange(v, device="cuda").float()
    x[2] = torch.randint(3, (v,), generator=g, device="cuda").float()
    x[3] = 7.0
    x[4] = (torch.arange(v, device="cuda") % 17).float()
    x[5] = -math.inf
    x[5, ::37] = 2.0  # fewer than alternatives above -inf
    for top in (1, 2, 6, 7, 20, 32):
        out, _ = ops.LogProbs(top).forward(x)
        verify(x, None, top, out)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("top", [0, 1, 2, 6, 7, 20, 32])
@pytest.mark.parametrize("rows,v", [(9, 32), (5, 300), (2, 5000), (600, 5000), (3, 40001)])
def test_number_of_alternatives_by_type(cuda, top, rows, v, dtype):
    print(f"top={top} rows={rows} v={v} {dtype}", flush=True)
    x, g = logits(rows, v, TYPES[dtype], top + v)
    t = torch.randint(v, (rows,), generator=g, device="cuda")
    dl, de = (torch.randn(rows, generator=g, device="cuda") for _ in range(2))
    dt = torch.randn(rows, top, generator=g, device="cuda") if top else None
    op = ops.LogProbs(top)
    out, save = op.forward(x, t)
    verify(x, t, top, out, op.backward((dl, de, dt), x, t, out[3], save), (dl, de, dt))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [40003, 70001])
def test_in_place_in_parts(cuda, v, dtype):
    """Rows that start at any element; the target before the first vector, in
    the first part, in a later one and behind the last vector, among the
    alternatives and not; a row left out and one without a logit above -inf."""
    print(f"in place in parts v={v} {dtype}", flush=True)
    rows, t = 8, TYPES[dtype]
    wide, g = logits(rows, v + 5, t, v)
    inside = lambda buf: buf[:, 3:3 + v]  # noqa: E731
    x = inside(wide)
    at = torch.tensor([0, 1, 5, v // 2, v - 9, v - 1, -1, 7], device="cuda")
    x[3, v // 2], x[5, v - 1], x[0, 0] = 20.0, 21.0, 22.0
    x[6], x[7] = math.nan, -math.inf
    dl, de = (torch.randn(rows, generator=g, device="cuda") for _ in range(2))
    dt = torch.randn(rows, 5, generator=g, device="cuda")
    op = ops.LogProbs(5)
    out, save = op.forward(x, at)
    want = op.backward((dl, de, dt), x, at, out[3], save)
    verify(x.clone(), at, 5, out, want, (dl, de, dt))
    y = wide.clone()
    op.backward((dl, de, dt), inside(y), at, out[3], save, out=inside(y))
    assert torch.equal(inside(y), want)
    (logp, entropy), one = op.value_and_grad(x, at, dl, de)
    verify(x.clone(), at, 0, (logp, entropy, None, None), one, (dl, de, None))
    z = wide.clone()
    (logp2, entropy2), _ = op.value_and_grad(inside(z), at, dl, de, out=inside(z))
    assert torch.equal(inside(z), one) and torch.equal(logp2, logp) and torch.equal(entropy2, entropy)
    for buf in (y, z):
        assert torch.equal(buf[:, :3], wide[:, :3]) and torch.equal(buf[:, 3 + v:], wide[:, 3 + v:])
