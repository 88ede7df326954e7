"""Log-probabilities, entropies and alternatives of rows of logits and their
gradient against their definition in 64 bits: every type, widths on both sides
of each kernel's range, rows left out, without a finite logit, with NaN and
infinities, ties, strides, in place, on another stream and in a graph."""
import math

import pytest
import torch

from tests import logprobs_ref as R
from bindcraft2_amd import NativeError, ops

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def logits(rows, v, dtype, seed, scale=3.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return (scale * torch.randn(rows, v, generator=g, device="cuda")).to(dtype), g


def verify(x, t, top, out, grads=None, cts=(None, None, None)):
    logp, entropy, top_logp, top_index = out
    ref = R.reference(x, t, top)
    of_logp, of_entropy = R.tolerances(x, ref)
    if t is not None:
        at = of_logp.gather(1, t.long().clamp(0, x.shape[1] - 1)[:, None])[:, 0]
        R.check("logp", logp, ref[0], at)
    R.check("entropy", entropy, ref[1], of_entropy)
    if top:
        assert torch.equal(top_index.long(), ref[3])
        R.check("top_logp", top_logp, ref[2], of_logp.gather(1, ref[3].clamp_min(0)))
    if grads is not None:
        d, terms = R.gradient(x, t, ref, *cts)
        R.check("d_logits", grads, d, R.gradient_tolerance(x, d, terms, ref, cts[1]))


def through(x, t, top, g, seed=5):
    """Forward, backward of everything, and the one call, all verified."""
    rows = x.shape[0]
    gen = torch.Generator("cuda").manual_seed(seed)
    cot = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    dl = cot(rows) if t is not None else None
    de, dt = cot(rows), cot(rows, top) if top else None
    op = ops.LogProbs(top)
    out, save = op.forward(x, t)
    d = op.backward((dl, de, dt), x, t, out[3], save)
    verify(x, t, top, out, d, (dl, de, dt))
    (logp, entropy), d1 = ops.LogProbs().value_and_grad(x, t, dl, de)
    verify(x, t, 0, (logp, entropy, None, None), d1, (dl, de, None))
    return out, d


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [1, 2, 3, 4, 5, 7, 8, 9, 16, 17, 20, 31, 32, 33, 37, 50, 63, 64, 65,
                               127, 128, 129, 255, 256, 257, 500, 511, 512, 513, 1000, 1023, 1024])
def test_short_rows(cuda, v, dtype):
    print(f"short rows v={v} {dtype}", flush=True)
    for rows in (1, 3, 70):
        x, g = logits(rows, v, TYPES[dtype], v * 100 + rows)
        t = torch.randint(v, (rows,), generator=g, device="cuda", dtype=torch.int32)
        through(x, t, min(v, 4), g)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [1025, 2047, 4096, 4099, 8192, 8193, 33003, 131073])
def test_long_rows(cuda, v, dtype):
    """A few rows are read in parts by several workgroups."""
    print(f"long rows v={v} {dtype}", flush=True)
    for rows in (1, 5):
        x, g = logits(rows, v, TYPES[dtype], v + rows)
        t = torch.randint(v, (rows,), generator=g, device="cuda")
        through(x, t, 8, g)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [1025, 9001])
def test_many_long_rows(cuda, v, dtype):
    """Enough rows for a workgroup each."""
    print(f"many long rows v={v} {dtype}", flush=True)
    x, g = logits(1100, v, TYPES[dtype], v)
    t = torch.randint(-1, v, (1100,), generator=g, device="cuda")
    t[::7] = -1
    x[t < 0] = math.nan
    through(x, t, 3, g)


@pytest.mark.parametrize("top", [0, 1, 2, 20, 32])
@pytest.mark.parametrize("rows,v", [(9, 32), (5, 300), (2, 5000), (600, 5000)])
def test_number_of_alternatives(cuda, top, rows, v):
    print(f"top={top} rows={rows} v={v}", flush=True)
    x, g = logits(rows, v, torch.bfloat16, top + v)
    t = torch.randint(v, (rows,), generator=g, device="cuda")
    through(x, t, top, g)


def special(v, t):
    f = torch.finfo(t)
    x, g = logits(16, v, t, v)
    at = torch.randint(v, (16,), generator=g, device="cuda", dtype=torch.int32)
    x[0] = -math.inf
    x[1] = -math.inf
    x[1, v // 2] = 1.5
    x[2] = -math.inf
    x[2, v - 1] = f.min
    at[2] = v - 1
    x[3] = f.min
    x[4] = f.min
    x[4, 3] = 0.25
    at[4] = 3
    x[5] = f.max
    x[6, v - 2] = math.nan
    x[7, 1] = math.inf
    x[8] = math.nan
    at[8] = -1
    x[9] = -math.inf
    at[9] = -7
    x[10, : v // 2] = -math.inf  # a target without probability
    at[10] = 0
    x[11, v // 2:] = -math.inf
    at[11] = 2 ** 31 - 1
    x[12] = 0.0
    x[12, ::2] = -0.0  # all alike
    x[13] = f.max
    x[13, 0] = f.min
    x[14, 0] = -math.inf
    return x, at, g


WIDTHS = [20, 64, 700, 3001, 20000]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", WIDTHS)
def test_special_rows(cuda, v, dtype):
    """Rows with nothing allowed, one class allowed, the type's lowest and
    largest values, NaN, infinities; the target on each side; left out."""
    print(f"special rows v={v} {dtype}", flush=True)
    x, at, g = special(v, TYPES[dtype])
    for targets in (at, at.long(), None):
        op = ops.LogProbs(5)
        out, save = op.forward(x, targets)
        verify(x, targets, 5, out)
    de, dl = (torch.randn(16, generator=g, device="cuda") for _ in range(2))
    dt = torch.randn(16, 5, generator=g, device="cuda")
    out, save = op.forward(x, at)
    verify(x, at, 5, out, op.backward((dl, de, dt), x, at, out[3], save), (dl, de, dt))
    verify(x, at, 5, out, op.backward((dl, None, None), x, at, out[3], save), (dl, None, None))
    (logp, entropy), d = op.value_and_grad(x, at, dl, de)
    verify(x, at, 0, (logp, entropy, None, None), d, (dl, de, None))


@pytest.mark.parametrize("rows,v,dtype", [(272, 33003, "f32"), (272, 66001, "bf16"), (256, 65544, "f16"),
                                          (600, 33100, "f32"), (2500, 9001, "f32"), (3000, 700, "f32")])
def test_rows_beyond_a_workgroup_and_the_caches(cuda, rows, v, dtype):
    """Rows of which a workgroup holds a part, every sixteenth a special one;
    logits and gradient of more than the caches keep; in place."""
    print(f"large rows={rows} v={v} {dtype}", flush=True)
    t = TYPES[dtype]
    x, g = logits(rows, v, t, v)
    at = torch.randint(v, (rows,), generator=g, device="cuda", dtype=torch.int32)
    odd, odd_at, _ = special(v, t)
    x[:16], at[:16] = odd, odd_at
    x[rows - 16:], at[rows - 16:] = odd, odd_at
    dl, de = (torch.randn(rows, generator=g, device="cuda") for _ in range(2))
    dt = torch.randn(rows, 3, generator=g, device="cuda")
    op = ops.LogProbs(3)
    out, save = op.forward(x, at)
    verify(x, at, 3, out, op.backward((dl, de, dt), x, at, out[3], save), (dl, de, dt))
    (logp, entropy), d = op.value_and_grad(x, at, dl, de)
    verify(x, at, 0, (logp, entropy, None, None), d, (dl, de, None))
    y = x.clone()
    op.value_and_grad(y, at, dl, de, out=y)
    assert torch.equal(y.nan_to_num(nan=3.0), d.nan_to_num(nan=3.0))


@pytest.mark.parametrize("v", [33, 3001, 70000])
def test_without_targets(cuda, v):
    """Entropies and alternatives alone, and their gradients."""
    x, g = logits(5, v, torch.float32, v)
    de, dt = torch.randn(5, generator=g, device="cuda"), torch.randn(5, 6, generator=g, device="cuda")
    op = ops.LogProbs(6)
    out, save = op.forward(x)
    assert out[0] is None
    verify(x, None, 6, out, op.backward((None, de, dt), x, None, out[3], save), (None, de, dt))
    verify(x, None, 6, out, op.backward((None, de, None), x, None, None, save), (None, de, None))
    verify(x, None, 6, out, op.backward((None, None, dt), x, None, out[3], save), (None, None, dt))
    (logp, entropy), d = op.value_and_grad(x, None, None, de)
    assert logp is None
    verify(x, None, 0, (None, entropy, None, None), d, (None, de, None))
    assert (op.value_and_grad(x, None)[1] == 0).all()


@pytest.mark.parametrize("v", WIDTHS)
def test_ties_and_orders(cuda, v):
    """Alternatives of rows in ascending and descending order, of few distinct
    values, and all alike: ties go to the lowest class."""
    print(f"ties v={v}", flush=True)
    x, g = logits(6, v, torch.float32, v)
    x[0] = torch.arange(v, device="cuda")
    x[1] = -torch.arange(v, device="cuda").float()
    x[2] = torch.randint(3, (v,), generator=g, device="cuda").float()
    x[3] = 7.0
    x[4] = (torch.arange(v, device="cuda") % 17).float()
    for top in (1, 6, 20):
        out, _ = ops.LogProbs(top).forward(x)
        verify(x, None, top, out)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [5, 50, 64, 999, 4001])
def test_strides_and_what_lies_between(cuda, v, dtype):
    """Rows apart and starting at any element; the gaps stay as they were, in
    place and out of it."""
    print(f"strides v={v} {dtype}", flush=True)
    t, rows = TYPES[dtype], 37
    wide, g = logits(rows + 2, v + 9, t, v)
    x = wide[1:-1, 3:3 + v]
    at = torch.randint(-1, v, (rows,), generator=g, device="cuda")
    op = ops.LogProbs(2)
    out, save = op.forward(x, at)
    verify(x.clone(), at, 2, out)
    dl, de = (torch.randn(rows, generator=g, device="cuda") for _ in range(2))
    dt = torch.randn(rows, 2, generator=g, device="cuda")
    want = op.backward((dl, de, dt), x.clone(), at, out[3], save)
    verify(x.clone(), at, 2, out, want, (dl, de, dt))
    canvas = torch.full_like(wide, 11.0)
    op.backward((dl, de, dt), x, at, out[3], save, out=canvas[1:-1, 3:3 + v])
    both = torch.full_like(wide, 11.0)
    _, one = ops.LogProbs().value_and_grad(x, at, dl, de, out=both[1:-1, 3:3 + v])
    again = wide.clone()
    inside = again[1:-1, 3:3 + v]
    assert op.backward((dl, de, dt), inside, at, out[3], save, out=inside) is inside
    third = wide.clone()
    ops.LogProbs().value_and_grad(third[1:-1, 3:3 + v], at, dl, de, out=third[1:-1, 3:3 + v])
    gap = torch.ones_like(wide, dtype=torch.bool)
    gap[1:-1, 3:3 + v] = False
    assert torch.equal(canvas[~gap], want.flatten()) and (canvas[gap] == 11).all()
    assert torch.equal(inside, want) and torch.equal(again[gap], wide[gap])
    assert (both[gap] == 11).all() and torch.equal(third[gap], wide[gap])
    assert torch.equal(third[~gap], one.flatten())


@pytest.mark.parametrize("v", [20, 999, 4001])
def test_gradient_beside_the_logits(cuda, v):
    """Logits and gradient as columns of one buffer."""
    x, g = logits(9, v, torch.float32, v)
    buf = torch.full((9, 2 * v + 3), 11.0, device="cuda")
    buf[:, :v] = x
    t = torch.randint(v, (9,), generator=g, device="cuda")
    dl = torch.randn(9, generator=g, device="cuda")
    (lp, en), d = ops.LogProbs().value_and_grad(buf[:, :v], t, dl, out=buf[:, v + 1:2 * v + 1])
    assert torch.equal(buf[:, :v], x)
    # (not the bits of the same rows elsewhere: a sum's order goes by a row's
    # alignment to 16 bytes)
    verify(x, t, 0, (lp, en, None, None), d, (dl, None, None))
    assert (buf[:, v] == 11).all() and (buf[:, 2 * v + 1:] == 11).all()
    with pytest.raises(NativeError, match="overlaps"):
        ops.LogProbs().value_and_grad(buf[:, :v], t, dl, out=buf[:, 1:v + 1])


def test_leading_dimensions_and_empty(cuda):
    x = torch.randn(4, 5, 64, device="cuda")
    t = torch.randint(64, (4, 5), device="cuda")
    (logp, entropy, tl, ti), save = ops.LogProbs(3).forward(x, t)
    assert logp.shape == entropy.shape == (4, 5) and tl.shape == ti.shape == (4, 5, 3)
    verify(x.view(20, 64), t.view(20), 3, (logp.view(20), entropy.view(20), tl.view(20, 3), ti.view(20, 3)))
    (logp, entropy, _, _), _ = ops.LogProbs().forward(x[0, 0], t[0, 0])
    assert logp.shape == () and abs(logp.item() - torch.log_softmax(x[0, 0], -1)[t[0, 0]].item()) < 1e-5
    (logp, _, _, ti), save = ops.LogProbs(2).forward(x[:, :0], t[:, :0])
    assert logp.shape == (4, 0) and ti.shape == (4, 0, 2)
    assert ops.LogProbs(2).backward((logp, None, None), x[:, :0].contiguous(), t[:, :0], ti, save).shape == (4, 0, 64)


def test_rows_far_apart(cuda):
    """Elements past 2^31 of the buffer."""
    ld, v = 2 ** 30 + 5, 1500
    buf = torch.zeros(2 * ld + v, dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((3, v), (ld, 1))
    x.copy_(torch.randn(3, v, device="cuda"))
    t = torch.tensor([3, 1499, 700], device="cuda")
    op = ops.LogProbs(4)
    out, save = op.forward(x, t)
    dl = torch.randn(3, device="cuda")
    d = op.backward((dl, None, None), x, t, out[3], save)
    verify(x.contiguous(), t, 4, out, d, (dl, None, None))
    y = buf.as_strided((3, 40), (ld, 1))
    (out, _), t = ops.LogProbs(4).forward(y), None
    verify(y.contiguous(), None, 4, out)


@pytest.mark.parametrize("v,dtype", [(8, "f32"), (1100, "bf16")])
def test_more_rows_than_one_launch_takes(cuda, v, dtype):
    """2^21 rows and a few: each row as the same row in a call of few."""
    print(f"many rows v={v} {dtype}", flush=True)
    rows = 2 ** 21 + 5
    x, g = logits(64, v, TYPES[dtype], v)
    x = x.repeat(rows // 64 + 1, 1)[:rows]
    t = torch.randint(v, (64,), generator=g, device="cuda").repeat(rows // 64 + 1)[:rows]
    dl, de = (torch.randn(64, generator=g, device="cuda").repeat(rows // 64 + 1)[:rows] for _ in range(2))
    op = ops.LogProbs(3)
    out, save = op.forward(x, t)
    d = op.backward((dl, de, out[2]), x, t, out[3], save)
    verify(x[:64], t[:64], 3, [o[:64] for o in out], d[:64], (dl[:64], de[:64], out[2][:64]))
    period = lambda o: torch.equal(o[64:], o[:-64])  # noqa: E731
    assert all(period(o) for o in (*out, d))
    del d
    (lp, en), d = ops.LogProbs().value_and_grad(x, t, dl, de)
    verify(x[:64], t[:64], 0, (lp[:64], en[:64], None, None), d[:64], (dl[:64], de[:64], None))
    assert period(d) and period(lp) and period(en)


@pytest.mark.parametrize("rows,v", [(300, 64), (2, 40000), (700, 4000)])
def test_same_bits_streams_and_graphs(cuda, rows, v):
    """The same bits every time, on another stream, and from a captured graph
    replayed with other inputs and eager work between."""
    print(f"graphs rows={rows} v={v}", flush=True)
    x, g = logits(rows, v, torch.float16, v)
    y, _ = logits(rows, v, torch.float16, v + 1)
    t = torch.randint(v, (rows,), generator=g, device="cuda")
    dl, de = (torch.randn(rows, generator=g, device="cuda") for _ in range(2))
    dt = torch.randn(rows, 3, generator=g, device="cuda")
    op = ops.LogProbs(3)

    def go(z):
        out, save = op.forward(z, t)
        d = op.backward((dl, de, dt), z, t, out[3], save)
        (lp, en), d1 = op.value_and_grad(z, t, dl, de)
        return [*out, d, lp, en, d1]

    want_x, want_y = go(x), go(y)
    same = lambda a, b: all(torch.equal(i, j) for i, j in zip(a, b))  # noqa: E731
    assert same(go(x), want_x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = go(x)
    torch.cuda.synchronize()
    assert same(other, want_x)
    z = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = go(z)
    for source, want in ((x, want_x), (y, want_y), (x, want_x), (y, want_y)):
        z.copy_(source)
        graph.replay()
        torch.cuda.synchronize()
        assert same(got, want)
        assert same(go(y), want_y)


@pytest.mark.parametrize("rows,v,dtype", [(5, 64, "f32"), (3, 2000, "f32")])
def test_gradient_against_differences(cuda, rows, v, dtype):
    """The gradient along a direction against the outputs' own central
    difference.  h = 2^-5: the third derivative of a log-probability along a
    direction of size at most 1 is at most 2, and of an entropy at most 8 (1 +
    log v): h^2 / 6 times that; the outputs' 32-bit errors over h."""
    x, g = logits(rows, v, TYPES[dtype], v, 1.5)
    t = torch.randint(v, (rows,), generator=g, device="cuda")
    dl, de = (torch.randn(rows, generator=g, device="cuda") for _ in range(2))
    way = 2 * torch.rand(rows, v, generator=g, device="cuda") - 1
    (_, _), d = ops.LogProbs().value_and_grad(x, t, dl, de)
    h = 2.0 ** -5
    value = lambda z: [o.double() for o in ops.LogProbs().forward(z, t)[0][:2]]  # noqa: E731
    (l1, e1), (l0, e0) = value(x + h * way), value(x - h * way)
    num = ((l1 - l0) * dl + (e1 - e0) * de) / (2 * h)
    got = (d.double() * way.double()).sum(1)
    of_logp, of_entropy = R.tolerances(x, R.reference(x, t, 0))
    round_off = (of_logp.amax(1) * dl.abs() + of_entropy * de.abs()) / h
    shift = 2 * R.HALF * x.abs().amax(1) * (dl.abs() + de.abs() * 2 * math.log(v)) / h
    cut = h * h / 6 * (2 * dl.abs() + 8 * (1 + math.log(v)) * de.abs())
    assert ((num - got).abs() <= round_off + shift + cut).all()


def test_bad_calls(cuda):
    x = torch.randn(4, 32, device="cuda")
    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    op = ops.LogProbs(2)
    out, save = op.forward(x, t)
    bad = [lambda: ops.LogProbs(33), lambda: ops.LogProbs(-1), lambda: op.forward(x.double(), t),
           lambda: op.forward(x, t[:3]), lambda: op.forward(x, t.float()), lambda: op.forward(x.t()),
           lambda: op.forward(x.cpu(), t), lambda: op.forward(x, t.cpu()),
           lambda: op.forward(torch.tensor(1.0, device="cuda")),
           lambda: op.backward((t.float()[:2], None, None), x, t, out[3], save),
           lambda: op.backward((None, None, None), x, t, out[3], save[:2]),
           lambda: op.backward((None, None, None), x, t, out[3].long(), save),
           lambda: op.backward((None, None, None), x, t, out[3], save, out=x.half()),
           lambda: op.value_and_grad(x, t, out=x[:2])]
    for k, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {k} was taken")
    for call in (lambda: ops.LogProbs(3).forward(x[:, :2].contiguous()),
                 lambda: op.forward(x[:1].expand(4, 32)),
                 lambda: op.forward(x[:, :0]),
                 lambda: op.backward((t.float(), None, None), x, None, out[3], save),
                 lambda: op.backward((None, None, out[2]), x, t, None, save)):
        with pytest.raises(NativeError):
            call()
    assert torch.isfinite(op.forward(x, t)[0][0]).all()
