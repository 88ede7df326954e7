"""Rows whose largest logit is a type's lowest value: masked throughout with it,
with -infinity beside it or alone left of the row."""
import math

import pytest
import torch

from tests.sampling_check import verify

pytestmark = pytest.mark.gpu
SETTINGS = [dict(), dict(temperature=0.3), dict(temperature=7.0), dict(top_k=1), dict(top_k=7), dict(top_p=0.3137),
            dict(min_p=0.1), dict(temperature=0.0), dict(temperature=0.9, top_k=11, top_p=0.7713, min_p=0.01),
            dict(top_p=0.3137219)]
# the kernels for up to 64 and up to 1024 classes, and for longer rows
WIDTHS = [20, 64, 65, 100, 129, 300, 600, 1000, 1024, 1025, 40_000, 131_072]


def sure(v, top_p=1.0, **_):
    """The part of the rows without a border on a class: none where v equal classes
    are cut after a whole number of them, as 0.3137 of 40 000 = 12 548."""
    return 0.0 if top_p < 1 and abs(v * top_p - round(v * top_p)) < 1e-6 else 0.5


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("v", WIDTHS)
def test_rows_of_the_lowest_value(cuda, v, dtype):
    low = torch.finfo(dtype).min
    u = torch.tensor([0.0, 0.3051, 0.6173, 0.9991], device="cuda")
    for s in SETTINGS:
        x = torch.full((4, v), low, device="cuda", dtype=dtype)
        # what the allocator hands out for the results next
        torch.full((4,), 1 << 20, device="cuda", dtype=torch.int32)
        verify(x, u, sure(v, **s), **s)
        x[:, ::3] = -math.inf
        verify(x, u, **s)
        x[:] = -math.inf
        x[:, v // 2] = low
        verify(x, u, **s)


@pytest.mark.parametrize("v", [20, 300, 40_000])
def test_rows_a_little_above_the_lowest_value(cuda, v):
    """Far below -3e38, and steps of 2^104 apart: the largest alone has a mass."""
    low = torch.finfo(torch.float32).min
    g = torch.Generator("cuda").manual_seed(v)
    x = low * (1 - 2.0 ** -20 * torch.randint(0, 16, (6, v), generator=g, device="cuda"))
    u = torch.rand(6, generator=g, device="cuda")
    for s in SETTINGS:
        verify(x, u, **s)
