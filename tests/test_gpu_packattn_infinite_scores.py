"""Keys whose scores are -infinity: beside others they weigh nothing; rows that
see no others have, by softmax of -infinities, NaN, and lse -infinity."""
import math

import pytest
import torch

from tests import sequence_ref as R
from bindcraft2_amd import ops

pytestmark = pytest.mark.gpu
# few rows of few keys, rows that fill the card, stretches of long caches
SHAPES = [(3, 40, 2, 1, 64), (70, 70, 4, 2, 128), (200, 200, 64, 64, 32), (1, 9000, 8, 2, 64), (1, 20_000, 2, 2, 128)]


def problem(m, n, heads, kv, d, dtype):
    g = torch.Generator("cuda").manual_seed(m + n)
    rand = lambda a, h: torch.randn(a, h, d, generator=g, device="cuda").to(dtype)  # noqa: E731
    q, k, v = rand(m, heads), rand(n, kv), rand(n, kv)
    q[..., 0] = q[..., 0].abs() + 0.5
    offsets = [torch.tensor([0, x], device="cuda", dtype=torch.int32) for x in (m, n)]
    return q, k, v, rand(m, heads), offsets


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,heads,kv,d", SHAPES)
@pytest.mark.parametrize("causal", [True, False])
def test_alone(cuda, causal, m, n, heads, kv, d, dtype):
    q, k, v, g, (qo, ko) = problem(m, n, heads, kv, d, dtype)
    k[..., 0] = -math.inf
    op = ops.PackedAttention(causal)
    out, lse = op.forward(q, k, v, qo, ko)
    assert out.isnan().all() and (lse == -math.inf).all()
    d_q, d_k, d_v = op.backward(g, q, k, v, out, lse, qo, ko)
    assert d_q.isnan().all() and d_k.isnan().all() and d_v.isnan().all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,heads,kv,d", SHAPES)
def test_beside_others(cuda, m, n, heads, kv, d, dtype):
    """Every third key of the last two thirds, and the whole first third."""
    q, k, v, g, (qo, ko) = problem(m, n, heads, kv, d, dtype)
    gone = torch.arange(n, device="cuda") % 3 == 1
    gone[:n // 3] = True
    k[gone, :, 0] = -math.inf
    out, lse = ops.PackedAttention(False).forward(q, k, v, qo, ko)
    want = R.attention(q, k[~gone], v[~gone], False, d ** -0.5)
    R.check("out", out, *want["out"])
    R.check("lse", lse, *want["lse"])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_first_rows_alone(cuda, dtype):
    """Causal rows that see such keys alone, and rows that see others too."""
    q, k, v, g, (qo, ko) = problem(100, 100, 2, 1, 64, dtype)
    k[:10, :, 0] = -math.inf
    out, lse = ops.PackedAttention().forward(q, k, v, qo, ko)
    assert out[:10].isnan().all() and (lse[:, :10] == -math.inf).all()
    assert out[10:].isfinite().all() and lse[:, 10:].isfinite().all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_no_key_is_another_matter(cuda, dtype):
    q, k, v, g, (qo, ko) = problem(50, 20, 2, 1, 64, dtype)
    op = ops.PackedAttention()
    out, lse = op.forward(q, k, v, qo, ko)
    assert (out[:30] == 0).all() and (lse[:, :30] == -math.inf).all() and out[30:].isfinite().all()
    d_q, d_k, d_v = op.backward(g, q, k, v, out, lse, qo, ko)
    assert (d_q[:30] == 0).all() and all(t.isfinite().all() for t in (d_q, d_k, d_v))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_no_key_beside_scores_of_minus_infinity_in_stretches(cuda, dtype):
    """6001 queries of 5000 keys, which are joined from stretches: 1001 rows see none, the
    next 300 see keys of -infinity alone."""
    q, k, v, g, (qo, ko) = problem(6001, 5000, 2, 2, 40, dtype)
    k[:300, :, 0] = -math.inf
    out, lse = ops.PackedAttention().forward(q, k, v, qo, ko)
    assert (out[:1001] == 0).all() and (lse[:, :1301] == -math.inf).all()
    assert out[1001:1301].isnan().all() and out[1301:].isfinite().all() and lse[:, 1301:].isfinite().all()
