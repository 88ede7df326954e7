"""Classes drawn by given uniform numbers against the definition in 64 bits:
types, widths on both sides of each kernel's range, ties, omitted classes, every
setting by itself and together, rows' own settings, rows nothing can be drawn from."""
import math

import pytest
import torch

from tests import sequence_ref as R
from bindcraft2_amd import ops

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SETTINGS = [dict(), dict(temperature=0.3), dict(top_k=1), dict(top_k=2), dict(top_k=7), dict(top_k=300),
            dict(top_p=0.5), dict(top_p=0.95), dict(top_p=0.0), dict(min_p=0.1), dict(min_p=1.0),
            dict(temperature=0.0), dict(temperature=5.0, top_k=40, top_p=0.8, min_p=0.01),
            dict(temperature=100.0, top_p=0.9), dict(temperature=1e-6), dict(top_p=1e-9, top_k=5)]


def logits(rows, v, dtype, seed, scale=3.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return (scale * torch.randn(rows, v, generator=g, device="cuda")).to(dtype), \
        torch.rand(rows, generator=g, device="cuda")


def verify(x, u, of_row=None, **settings):
    """of_row(r): the row's own settings, as numbers."""
    index, logp = ops.Sampler(**settings).sample(x, u)
    xs, us = x.cpu(), u.tolist()
    unit = x.shape[-1] * 2.0 ** -44  # masses are whole numbers of 2^-44 and less
    for r in range(x.shape[0]):
        at, lp, near = R.draw(xs[r], us[r], **(of_row(r) if of_row else settings))
        if near < unit:  # a border closer than the masses' unit decides nothing
            continue
        assert index[r].item() == at, (r, settings, index[r].item(), at, near)
        # f32's half step of the result, and the sum of masses in their units
        assert abs(logp[r].item() - lp) <= R.E * abs(lp) + unit + 1e-12, (r, settings, logp[r].item(), lp)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [1, 2, 3, 15, 16, 17, 20, 31, 32, 33, 63, 64, 65, 100, 255, 256, 1000, 1023, 1025, 2048,
                               4095, 4096, 4097, 8191, 8193])
def test_widths(cuda, v, dtype):
    for i, s in enumerate(SETTINGS):
        print(f"widths {v} {dtype} {s}", flush=True)
        verify(*logits(5, v, TYPES[dtype], 100 * v + i), **s)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [32771, 131072, 300_001])
def test_long_rows(cuda, v, dtype):
    for i, s in enumerate(SETTINGS):
        print(f"long rows {v} {dtype} {s}", flush=True)
        verify(*logits(2, v, TYPES[dtype], v + i), **s)


@pytest.mark.parametrize("v", [20, 64, 100, 5000, 70_000])
def test_ties(cuda, v):
    """All alike, two values, a few values: the lowest indexes first."""
    u = torch.tensor([0.0, 0.3, 0.6, 0.999], device="cuda")
    for s in (dict(), dict(top_k=3), dict(top_k=v // 2 + 1), dict(top_p=0.3), dict(min_p=0.9), dict(temperature=0.0),
              dict(top_k=v // 2 + 1, top_p=0.55)):
        print(f"ties {v} {s}", flush=True)
        verify(torch.zeros(4, v, device="cuda"), u, **s)
        verify(torch.full((4, v), -7.5, device="cuda", dtype=torch.bfloat16), u, **s)
        x = logits(4, v, torch.float32, v)[0]
        verify(x.sign(), u, **s)
        verify((x * 2).round().half(), u, **s)
        x = torch.zeros(4, v, device="cuda")
        x[:, ::2] = -0.0
        verify(x, u, **s)


@pytest.mark.parametrize("v", [20, 64, 300, 40_000])
def test_omitted_classes(cuda, v):
    """-infinity, the lowest value and -1e4 beside live classes; one class left."""
    for low in (-math.inf, torch.finfo(torch.float32).min, -1e4):
        for s in SETTINGS:
            x, u = logits(4, v, torch.float32, v)
            x[:, v // 3:] = low
            x[3, 1:] = low
            verify(x, u, **s)
    index, _ = ops.Sampler().sample(x, torch.full((4,), 0.9999999, device="cuda"))
    assert (index < v // 3).all()


@pytest.mark.parametrize("v", [2, 20, 64, 300, 9000])
def test_uniforms_at_the_ends(cuda, v):
    x, _ = logits(6, v, torch.float32, v)
    u = torch.tensor([0.0, 1.0, 2.0, -3.0, 1 - 2.0 ** -24, math.inf], device="cuda")
    for s in (dict(), dict(top_k=2), dict(top_p=0.6), dict(min_p=0.2)):
        verify(x, u, **s)


@pytest.mark.parametrize("v", [20, 64, 300, 9000])
def test_rows_of_nothing(cuda, v):
    x, u = logits(8, v, torch.float32, v)
    x[0, v // 2] = math.nan
    x[1, 0] = math.inf
    x[2] = -math.inf
    u[3] = math.nan
    t = torch.ones(8, device="cuda")
    t[4], t[5], t[6] = math.nan, math.inf, -1.0
    for s in SETTINGS:
        s = {k: w for k, w in s.items() if k != "temperature"}
        index, logp = ops.Sampler(temperature=t, **s).sample(x, u)
        for r in (0, 1, 2, 3, 4, 5):
            assert index[r] == -1 and logp[r].isnan(), (r, s)
        assert index[6] == x[6].argmax() and logp[6] == 0  # not positive: the first class
        assert 0 <= index[7] < v and logp[7] <= 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [20, 1000, 20_000])
def test_settings_of_each_row(cuda, v, dtype):
    rows = 40
    x, u = logits(rows, v, TYPES[dtype], v)
    g = torch.Generator("cuda").manual_seed(v)
    one = lambda: torch.rand(rows, generator=g, device="cuda")  # noqa: E731
    s = dict(temperature=one() * 2, top_k=(one() * v / 4).int() - 1, top_p=one() * 1.2, min_p=one() * 0.2)
    verify(x, u, lambda r: {k: w[r].item() for k, w in s.items()}, **s)


def test_shapes_and_strides(cuda):
    x, u = logits(12, 700, torch.float32, 1)
    want = ops.Sampler(top_k=50).sample(x, u)
    got = ops.Sampler(top_k=50).sample(x.view(3, 4, 700), u.view(3, 4))
    assert got[0].shape == (3, 4) and torch.equal(got[0].flatten(), want[0])
    wide = torch.zeros(12, 703, device="cuda")
    wide[:, 1:701] = x
    got = ops.Sampler(top_k=50).sample(wide[:, 1:701], u)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    empty = ops.Sampler().sample(x[:0], u[:0])
    assert empty[0].shape == (0,) and empty[1].shape == (0,)


def test_frequencies(cuda):
    """Evenly spread numbers draw every class by its share."""
    x, _ = logits(1, 50, torch.float32, 3)
    n = 100_000
    u = (torch.arange(n, device="cuda") + 0.5) / n
    index, _ = ops.Sampler(temperature=1.3).sample(x.expand(n, 50).contiguous(), u)
    share = torch.bincount(index.long(), minlength=50).double() / n
    # a class's count is off by one at each end of its stretch
    assert ((share - torch.softmax(x[0].double() / 1.3, 0)).abs() <= 2.1 / n).all()


def test_beyond_2_to_31_elements(cuda):
    rows, v = 33, 1 << 26
    x = torch.zeros(rows, v, device="cuda", dtype=torch.bfloat16)
    x[-1, v - 5] = 30.0
    index, logp = ops.Sampler(top_k=3).sample(x, torch.full((rows,), 0.5, device="cuda"))
    assert index[-1] == v - 5 and (index[:-1] == 1).all()
    assert abs(logp[0].item() + math.log(3)) < 1e-6


def test_same_bits_and_graph(cuda):
    x, u = logits(30, 20_000, torch.bfloat16, 2)
    op = ops.Sampler(0.9, 100, 0.9, 0.001)
    graph = torch.cuda.CUDAGraph()
    op.sample(x, u)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        held = op.sample(x, u)
    for i in range(4):
        u.copy_((u * 7.1) % 1)
        want = [t.clone() for t in op.sample(x, u)]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, held)), i
