"""A causal query's results hang on the keys that it sees alone, and a key's gradients
on the queries that see it, whatever later and earlier tokens of the sequence hold."""
import math

import pytest
import torch

from tests import sequence_ref as R
from bindcraft2_amd import ops

pytestmark = pytest.mark.gpu
INF, NAN = math.inf, math.nan
# few rows of few keys, rows that fill the card, few rows of long caches, long rows in
# stretches, fewer keys than queries
SHAPES = [(70, 70, 4, 2, 128), (9, 40, 6, 2, 32), (200, 200, 64, 64, 32), (300, 300, 64, 32, 128), (130, 200, 192, 64, 16),
          (16, 5000, 2, 1, 64), (3, 9000, 8, 2, 128), (6001, 6001, 2, 2, 40), (330, 260, 64, 64, 64), (40, 20, 2, 1, 64)]


def problem(m, n, heads, kv, d, dtype):
    g = torch.Generator("cuda").manual_seed(m + n)
    rand = lambda a, h: torch.randn(a, h, d, generator=g, device="cuda").to(dtype)  # noqa: E731
    offsets = [torch.tensor([0, x], device="cuda", dtype=torch.int32) for x in (m, n)]
    return [rand(m, heads), rand(n, kv), rand(n, kv), rand(m, heads)], offsets


def same(a, b):
    """The same numbers, NaN for NaN."""
    return torch.equal(a.nan_to_num(1.25e4, 2.5e4, -2.5e4), b.nan_to_num(1.25e4, 2.5e4, -2.5e4))


def run(x, offsets, causal=True):
    q, k, v, g = x
    op = ops.PackedAttention(causal)
    out, lse = op.forward(q, k, v, *offsets)
    return (out, lse, *op.backward(g, q, k, v, out, lse, *offsets))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,heads,kv,d", SHAPES)
@pytest.mark.parametrize("what", [INF, -INF, NAN])
def test_values(cuda, what, m, n, heads, kv, d, dtype):
    """One element of one head of a late key's value, then all of the last keys'."""
    x, offsets = problem(m, n, heads, kv, d, dtype)
    out, lse, *_ = run(x, offsets)
    for key, at, element in ((n - 1 - min(m, n) // 3, slice(0, 1), slice(3, 4)), (n - 2, slice(None), slice(None))):
        v = x[2].clone()
        v[key if element != slice(None) else slice(key, None), at, element] = what
        got, got_lse = ops.PackedAttention().forward(x[0], x[1], v, *offsets)
        sees = key - (n - m)  # the first query that sees it
        assert same(got[:sees], out[:sees]) and torch.equal(got_lse, lse), key
        hit = got[sees:].view(-1, kv, heads // kv, d)[:, at, :, element]
        assert (hit.isnan() if math.isnan(what) else hit == what).all()
        rest = got[sees:].view(-1, kv, heads // kv, d)[..., :3]
        assert element == slice(None) or same(rest, out[sees:].view(-1, kv, heads // kv, d)[..., :3])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,heads,kv,d", SHAPES)
@pytest.mark.parametrize("which", [1, 2])
def test_gradients_of_earlier_queries(cuda, which, m, n, heads, kv, d, dtype):
    """NaN in a late key (1) or value (2): what comes of the queries before it is right.  Not to
    the bit: the rows of a wave raise their references together, and so round apart."""
    x, offsets = problem(m, n, heads, kv, d, dtype)
    want = R.attention(*x[:3], True, d ** -0.5, x[3])
    for bad in (NAN, INF):
        key = n - 1 - min(m, n) // 3
        x[which] = x[which].clone()
        x[which][key, :, 5] = bad
        got = run(x, offsets)
        sees = key - (n - m)
        for name, t in (("out", got[0][:sees]), ("lse", got[1][:, :sees]), ("d_q", got[2][:sees])):
            R.check(name, t, *((w[:, :sees] if name == "lse" else w[:sees]) for w in want[name]))
        assert got[2][sees:].isnan().any(-1).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,heads,kv,d", SHAPES)
@pytest.mark.parametrize("which", [0, 3])
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
def test_gradients_of_later_keys(cuda, bad, which, m, n, heads, kv, d, dtype):
    """In an early query (0) or cotangent (3): gradients of the keys that it does not see."""
    x, offsets = problem(m, n, heads, kv, d, dtype)
    want = R.attention(*x[:3], True, d ** -0.5, x[3])
    query = max(m - n, 0) + min(m, n) // 3
    x[which][query, :, 5] = bad
    got = run(x, offsets)
    last = query + n - m  # the last key that it sees
    for name, t in (("d_k", got[3]), ("d_v", got[4])):
        R.check(name, t[last + 1:], *(w[last + 1:] for w in want[name]))
    d_k, d_v = (~t[:last + 1].isfinite() for t in got[3:])  # of the keys that it sees
    assert d_k.any(-1).all() and (d_v.all() if which == 0 else d_v[..., 5].all())
    keep = torch.arange(m, device="cuda") != query
    assert got[2][keep].isfinite().all() and got[0][keep].isfinite().all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_whole_sequences_and_caches(cuda, dtype):
    """Where nothing is masked within a sequence an infinity reaches every row as it is."""
    x, offsets = problem(70, 90, 4, 2, 64, dtype)
    x[2][33, 1, 7] = -INF
    out = run(x, offsets, False)[0]
    assert (out[:, 2:, 7] == -INF).all() and out[..., :7].isfinite().all() and out[:, :2].isfinite().all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_captured(cuda, dtype):
    """Replayed with and without a NaN."""
    x, offsets = problem(300, 300, 4, 2, 64, dtype)
    run(x, offsets)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run(x, offsets)
    for bad in (0.5, NAN, 0.25, INF):
        x[2][200, 0, 3] = bad
        want = run(x, offsets)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(same(a, b) for a, b in zip(held, want)), bad
        assert held[0][:200].isfinite().all()
