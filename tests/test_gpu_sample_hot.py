"""Temperatures at which a difference of 1e38 is small: every finite logit has its
share, the types' lowest values too."""
import math

import pytest
import torch

from tests.sampling_check import verify

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [20, 64, 65, 300, 1000, 5000, 40_000])
def test_hot(cuda, v, dtype):
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    g = torch.Generator("cuda").manual_seed(v)
    u = torch.rand(4, generator=g, device="cuda")
    for t in (3e37, 1e38, 3e39, 1e300):
        for s in (dict(), dict(top_k=v // 3), dict(top_k=5), dict(top_p=0.9137), dict(min_p=1e-3),
                  dict(top_k=v // 2, top_p=0.6137, min_p=1e-4), dict(top_k=v // 2, top_p=0.6137219),
                  dict(top_p=0.9137219)):
            # what is alike to 1e-37 (at 1e300 all classes) weighs the same: 0.6137 of 20 000
            # of them = 12 274 and 0.9137 of 40 000 = 36 548 end on a border
            kept = s.get("top_k", v) * s.get("top_p", 0.5)
            most = 0.5 if abs(kept - round(kept)) > 1e-6 or "top_p" not in s else 0.0
            x = torch.randn(4, v, generator=g, device="cuda").to(dtype)
            x[:, v // 2:] = low
            verify(x, u, most, temperature=t, **s)
            x[:, :v // 4] = high
            x[:, v // 4] = -math.inf
            verify(x, u, most, temperature=t, **s)
            x = ((torch.rand(4, v, generator=g, device="cuda") * 2 - 1) * 3.3e38).to(dtype)
            verify(x, u, most, temperature=t, **s)
