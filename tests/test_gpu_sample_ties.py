"""Classes of the same logit under top-p: the first of them by index stay."""
import pytest
import torch

from tests.sampling_check import verify

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [20, 64, 100, 300, 1000, 5000, 70_000])
def test_ties_under_top_p(cuda, v, dtype):
    g = torch.Generator("cuda").manual_seed(v)
    u = torch.tensor([0.0, 0.2173, 0.6111, 0.9987], device="cuda")
    few = torch.randint(0, 3, (4, v), generator=g, device="cuda").to(dtype)
    for s in (dict(top_p=0.3137), dict(top_p=0.9113), dict(top_k=v // 2 + 1, top_p=0.5537),
              dict(top_p=0.7131, min_p=0.2), dict(temperature=2.7, top_p=0.6137), dict(top_p=0.3137219),
              dict(top_p=0.9113241, min_p=0.2), dict(temperature=2.7, top_p=0.6137531)):
        # a whole number of equal classes (0.3137 of 70 000 = 21 959) ends on a border
        kept = s.get("top_k", v) * s["top_p"]
        verify(torch.zeros(4, v, device="cuda", dtype=dtype), u, most=float(abs(kept - round(kept)) > 1e-6), **s)
        # of 70 000 classes' row 1 top_p = 0.9113 ends 1.13e-9 of the sum beside a class,
        # within the 70 000 units of 2^-44 = 3.98e-9 that a sum of masses may be off
        verify(few, u, most=0.75, **s)


@pytest.mark.parametrize("v", [20, 100, 5000, 70_000])
def test_ties_at_a_border(cuda, v):
    """A cut that falls on a class: one of the two answers beside it."""
    u = torch.tensor([0.0, 0.3, 0.6, 0.999], device="cuda")
    for s in (dict(top_p=0.3), dict(top_p=0.5), dict(top_k=v // 2, top_p=0.5)):
        verify(torch.zeros(4, v, device="cuda"), u, most=0.0, **s)
