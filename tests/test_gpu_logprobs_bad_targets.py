"""A target at or past the classes makes its row's log-probability and its
gradient NaN: whichever cotangents are given, and in rows without a logit above
-inf too; by each kernel's widths."""
import math

import pytest
import torch

from tests.test_gpu_logprobs import logits, verify
from bindcraft2_amd import ops

pytestmark = pytest.mark.gpu
# lanes of a group; a list (f32) or keys; a workgroup's registers; parts
WIDTHS = [(6, 3), (6, 20), (6, 300), (6, 700), (6, 3001), (6, 20000), (6, 70001), (260, 33100)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,v", WIDTHS)
def test_target_past_the_classes(cuda, rows, v, dtype):
    print(f"bad targets rows={rows} v={v} {dtype}", flush=True)
    x, g = logits(rows, v, dtype, v)
    t = torch.randint(v, (rows,), generator=g, device="cuda")
    x[1:4] = -math.inf
    t[0], t[1], t[2] = v, v, 2 ** 40
    x[4, 1] = math.nan
    t[4] = v + 1
    dl, de = (torch.randn(rows, generator=g, device="cuda") for _ in range(2))
    dt = torch.randn(rows, 2, generator=g, device="cuda")
    op = ops.LogProbs(2)
    out, save = op.forward(x, t)
    for cts in ((dl, de, dt), (None, de, None), (None, None, dt), (dl, None, None), (None, None, None)):
        verify(x, t, 2, out, op.backward(cts, x, t, out[3], save), cts)
    for cts in ((dl, de), (dl, None), (None, de), (None, None)):
        (logp, entropy), d = op.value_and_grad(x, t, *cts)
        verify(x, t, 0, (logp, entropy, None, None), d, (*cts, None))
