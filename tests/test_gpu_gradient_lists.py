"""The global norm of a list of gradients, clipping and the Adam step against
their definitions in 64 bits: types mixed in a list, lists on both sides of
each path (one workgroup, entries with the launch, a device table), odd sizes
and starts, empty tensors, in place, streams and graphs."""
import math

import pytest
import torch

from bindcraft2_amd import NativeError, ops

pytestmark = pytest.mark.gpu
D = torch.float64
HALF = 2.0 ** -24
TYPES = (torch.float32, torch.float16, torch.bfloat16)
# (sizes; types by turns): one workgroup; entries with the launch; the table
LISTS = {
    "one": [1],
    "states": [480, 480, 4480],
    "odd": [1, 2, 3, 5, 7, 63, 64, 65, 1021, 0, 8191],
    "edge": [16384],
    "over": [16385],
    "chunks": [8192 * 3 + 1, 8191, 8192, 8193, 0, 5],
    "large": [3_000_001, 17, 1_000_000],
    "table_small": [k % 7 for k in range(60)],
    "table": [(k * 7919) % 20011 for k in range(500)],
}


def make(sizes, seed, types=TYPES, scale=0.1):
    """Tensors that start at odd elements of one buffer a type, and the buffers."""
    g = torch.Generator("cuda").manual_seed(seed)
    out, buffers = [], []
    for k, n in enumerate(sizes):
        b = torch.full((n + 16,), 3.0, device="cuda", dtype=types[k % len(types)])
        at = (5 * k) % 8
        b[at:at + n] = scale * torch.randn(n, generator=g, device="cuda")
        buffers.append((b, at, n))
        out.append(b[at:at + n])
    return out, buffers


def untouched(buffers):
    return all((b[:at] == 3).all() and (b[at + n:] == 3).all() for b, at, n in buffers)


def exact_norm(grads):
    return math.sqrt(sum(g.double().square().sum().item() for g in grads))


def rounded(got, want, what):
    """One rounding to the type, of a value with three half steps of f32 behind it."""
    f = torch.finfo(got.dtype)
    tol = (f.eps / 2 + 4 * HALF) * want.abs() + f.smallest_normal * f.eps
    over = ((got.double() - want).abs() - tol)
    assert over.numel() == 0 or over.max().item() <= 0, f"{what}: {over.max().item()}"


@pytest.mark.parametrize("name", LISTS)
@pytest.mark.parametrize("max_norm", [0.5, 1e6])
def test_norm_and_clip(cuda, name, max_norm):
    print(f"clip {name} {max_norm}", flush=True)
    grads, buffers = make(LISTS[name], 3)
    outs, out_buffers = make(LISTS[name], 4)
    norm = exact_norm(grads)
    h = ops.GradientClip(grads, out=outs)
    kept = [g.clone() for g in grads]
    for got in (h.norm(), h.clip(max_norm)):
        assert got.shape == (1,) and abs(got.item() - norm) <= 3 * HALF * norm
    c = 1.0 if norm < max_norm else max_norm / norm
    for o, g, k in zip(outs, grads, kept):
        assert torch.equal(g, k)
        rounded(o, g.double() * c, name)
        if c == 1.0:
            assert torch.equal(o, g)
    assert untouched(buffers) and untouched(out_buffers)
    got = ops.GradientClip(grads).clip(max_norm)  # in place: the same bits
    assert abs(got.item() - norm) <= 3 * HALF * norm
    assert all(torch.equal(g, o) for g, o in zip(grads, outs)) and untouched(buffers)


def test_norms_beyond_32_bits_and_not_finite(cuda):
    big = torch.full((40000,), 3e38, device="cuda")
    h = ops.GradientClip([big], out=[torch.empty_like(big)])
    assert h.norm().item() == math.inf  # 6e40
    h.clip(1.0)
    rounded(h.tensors[1], torch.full_like(big, 1 / 200, dtype=D), "large")
    tiny = torch.full((100,), 1e-30, device="cuda")
    assert abs(ops.GradientClip([tiny]).norm().item() - 1e-29) <= 1e-35
    for n in (100, 40000):
        g = torch.randn(n, device="cuda")
        g[n // 2] = math.nan
        h = ops.GradientClip([g], out=[torch.empty_like(g)])
        assert math.isnan(h.clip(1.0).item()) and torch.isnan(h.tensors[1]).all()
        g[n // 2] = math.inf
        assert h.clip(1.0).item() == math.inf
        want = torch.zeros(n, device="cuda")
        want[n // 2] = math.nan
        assert torch.equal(h.tensors[1].nan_to_num(nan=9.0).abs(), want.nan_to_num(nan=9.0))
        g.zero_()
        assert h.clip(1.0).item() == 0 and (h.tensors[1] == 0).all()


def test_empty_lists(cuda):
    e = torch.empty(0, device="cuda")
    for grads in ([], [e], [e] * 40):
        h = ops.GradientClip(grads)
        assert h.norm().item() == 0 and h.clip(1.0).item() == 0
    a = ops.Adam([], [], [], [])
    assert a.step(1, 0.1) is None and a.step(1, 0.1, max_norm=1.0).item() == 0


def adam_state(sizes, seed, p_types, g_types):
    p, pb = make(sizes, seed, p_types, 1.0)
    g, gb = make(sizes, seed + 1, g_types)
    m, mb = make(sizes, seed + 2, (torch.float32,), 0.01)
    v, vb = make(sizes, seed + 3, (torch.float32,), 0.05)
    for t in v:
        t.square_()
    return (p, g, m, v), (pb, gb, mb, vb)


def adam_exact(p, g, m, v, c, t, lr, b1, b2, eps, wd):
    """The step in 64 bits, and the size of what is added to p."""
    g = g.double() * c
    m1 = b1 * m.double() + (1 - b1) * g
    v1 = b2 * v.double() + (1 - b2) * g * g
    move = (m1 / (1 - b1 ** t)) / ((v1 / (1 - b2 ** t)).sqrt() + eps)
    p1 = p.double() - lr * (move + wd * p.double())
    return p1, m1, v1, lr * move.abs(), ((b1 * m.double()).abs() + ((1 - b1) * g).abs())


def check_adam(state, out, c, t, lr, b1, b2, eps, wd):
    """The moments: two products and a sum, the factor's rounding.  The move:
    the moments' errors, relative to the larger of m's terms, and eight more
    roundings; p: its own rounding, to its type, and two of the decay's."""
    for p, g, m, v, p2, m2, v2 in zip(*state, *out):
        p1, m1, v1, size, terms = adam_exact(p, g, m, v, c, t, lr, b1, b2, eps, wd)
        assert ((m2.double() - m1).abs() <= 5 * HALF * terms + 1e-44).all()
        assert ((v2.double() - v1).abs() <= 7 * HALF * v1 + 1e-44).all()
        scale = lr / (1 - b1 ** t) / ((v1 / (1 - b2 ** t)).sqrt() + eps)
        f = torch.finfo(p2.dtype)
        tol = HALF * (18 * size + 5 * scale * terms + 4 * lr * wd * p.double().abs() + 2 * p1.abs())
        tol = tol + f.eps / 2 * (p1.abs() + tol) + f.smallest_normal * f.eps
        assert ((p2.double() - p1).abs() <= tol).all()


@pytest.mark.parametrize("name", LISTS)
@pytest.mark.parametrize("types", [((torch.float32,), (torch.float32,)), (TYPES, TYPES[1:] + TYPES[:1]),
                                   ((torch.bfloat16,), (torch.bfloat16,))], ids=["f32", "mixed", "bf16"])
def test_adam(cuda, name, types):
    print(f"adam {name} {types}", flush=True)
    for t, max_norm, wd in ((1, None, 0.0), (7, 0.5, 0.01), (100_000, 1e6, 0.1)):
        state, buffers = adam_state(LISTS[name], 11, *types)
        norm = exact_norm(state[1])
        c = 1.0 if max_norm is None or norm < max_norm else max_norm / norm
        kept = [[x.clone() for x in s] for s in state]
        outs, out_buffers = adam_state(LISTS[name], 31, *types)
        h = ops.Adam(*state, out=(outs[0], outs[2], outs[3]), betas=(0.9, 0.999), weight_decay=wd)
        got = h.step(t, 0.01, max_norm=max_norm)
        assert (got is None) == (max_norm is None)
        if got is not None:
            assert abs(got.item() - norm) <= 3 * HALF * norm
        check_adam(state, (outs[0], outs[2], outs[3]), c, t, 0.01, 0.9, 0.999, 1e-8, wd)
        assert all(torch.equal(a, b) for s, k in zip(state, kept) for a, b in zip(s, k))
        assert all(untouched(b) for b in (*buffers, *out_buffers))
        sched = torch.tensor([0.01, t], dtype=torch.float32, device="cuda")
        other = [[torch.empty_like(x) for x in s] for s in (state[0], state[2], state[3])]
        ops.Adam(*state, out=other, weight_decay=wd).step(1, 99.0, max_norm, scalars=sched)
        check_adam(state, other, c, t, float(sched[0]), 0.9, 0.999, 1e-8, wd)
        ops.Adam(*state, weight_decay=wd).step(t, 0.01, max_norm)  # in place: the same bits
        for a, b in zip((state[0], state[2], state[3]), (outs[0], outs[2], outs[3])):
            assert all(torch.equal(i, j) for i, j in zip(a, b))
        assert all(untouched(b) for b in buffers)


def test_adam_without_momentum(cuda):
    """beta1 = 0 and beta2 = 0, where log beta has no value."""
    state, _ = adam_state([33, 20000], 5, (torch.float32,), (torch.float32,))
    out = [[torch.empty_like(x) for x in s] for s in (state[0], state[2], state[3])]
    ops.Adam(*state, out=out, betas=(0.0, 0.0), eps=1e-3).step(3, 0.5)
    check_adam(state, out, 1.0, 3, 0.5, 0.0, 0.0, 1e-3, 0.0)


@pytest.mark.parametrize("name", ["states", "chunks", "table"])
def test_lists_streams_and_graphs(cuda, name):
    """The same bits every time, on another stream, and from a graph whose
    schedule is on the device, replayed with eager work between; a list freed
    and another made while the graph lives."""
    print(f"list graphs {name}", flush=True)
    f = (torch.float32,)
    grads, _ = make(LISTS[name], 3)
    outs = [torch.zeros_like(g) for g in grads]
    state, _ = adam_state(LISTS[name], 11, f, f)
    start = [[x.clone() for x in s] for s in state]
    clip, adam = ops.GradientClip(grads, out=outs), ops.Adam(*state)
    sched = torch.tensor([0.01, 1.0], device="cuda")

    def back():
        for s, k in zip(state, start):
            for a, b in zip(s, k):
                a.copy_(b)
        sched.copy_(torch.tensor([0.01, 1.0]))

    def go():
        n = clip.clip(0.25)
        n2 = adam.step(1, 0.0, max_norm=0.5, scalars=sched)
        sched[1] += 1
        return n, n2

    def now():
        return [x.clone() for x in (*outs, *state[0], *state[2], *state[3])]

    same = lambda a, b: all(torch.equal(i, j) for i, j in zip(a, b))  # noqa: E731
    steps = []
    for _ in range(3):
        n = go()
        steps.append((*n, *now()))
    back()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        n = go()
    torch.cuda.synchronize()
    assert same((*n, *now()), steps[0])
    back()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        n = go()
    back()
    for k in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert same((*n, *now()), steps[k])
        other = ops.GradientClip([torch.randn(50, device="cuda") for _ in range(40 + k)])
        other.clip(0.1)
        del other
        torch.cuda.synchronize()


@pytest.mark.parametrize("count", [3, 50])
def test_lists_beyond_the_caches(cuda, count):
    """Operands of more than 256 MiB, entries with the launch and in the table."""
    print(f"large lists {count}", flush=True)
    sizes = [36_000_000 // count + 7 * k for k in range(count)]
    grads, buffers = make(sizes, 3, (torch.float32,))
    outs, out_buffers = make(sizes, 4, (torch.float32,))
    norm = exact_norm(grads)
    assert abs(ops.GradientClip(grads, out=outs).clip(0.5).item() - norm) <= 3 * HALF * norm
    for o, g in zip(outs, grads):
        rounded(o, g.double() * (0.5 / norm), "large")
    assert untouched(buffers) and untouched(out_buffers)
    sizes = [12_000_000 // count + 7 * k for k in range(count)]
    for types in (((torch.float32,), (torch.float32,)), (TYPES, TYPES[1:] + TYPES[:1])):
        state, buffers = adam_state(sizes, 11, *types)
        outs, out_buffers = adam_state(sizes, 31, *types)
        norm = exact_norm(state[1])
        h = ops.Adam(*state, out=(outs[0], outs[2], outs[3]), weight_decay=0.01)
        assert abs(h.step(5, 0.01, max_norm=0.5).item() - norm) <= 3 * HALF * norm
        check_adam(state, (outs[0], outs[2], outs[3]), 0.5 / norm, 5, 0.01, 0.9, 0.999, 1e-8, 0.01)
        assert all(untouched(b) for b in (*buffers, *out_buffers))


def test_graph_of_a_list_that_is_gone(cuda):
    """A captured call's table is not given to a later list."""
    grads, _ = make(LISTS["table"], 3)
    outs = [torch.zeros_like(g) for g in grads]
    h = ops.GradientClip(grads, out=outs)
    norm = h.clip(0.25)
    want = [o.clone() for o in outs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = h.clip(0.25)
    del h
    others = [ops.GradientClip([torch.ones(7, device="cuda") for _ in range(k)]) for k in (40, 500)]
    for _ in range(3):
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(again, norm) and all(torch.equal(o, w) for o, w in zip(outs, want))
        assert [o.norm().item() for o in others] == pytest.approx([(7 * k) ** 0.5 for k in (40, 500)])


def test_bad_lists(cuda):
    f = lambda n: torch.randn(n, device="cuda")  # noqa: E731
    a, b = f(64), f(64)
    for call in (lambda: ops.GradientClip([a.double()]), lambda: ops.GradientClip([a.cpu()]),
                 lambda: ops.GradientClip([a[::2]]), lambda: ops.GradientClip([a], out=[b, b]),
                 lambda: ops.GradientClip([a], out=[b[:32]]), lambda: ops.GradientClip([a], out=[b.half()]),
                 lambda: ops.Adam([a], [b], [a.half()], [b]), lambda: ops.Adam([a], [], [a], [b]),
                 lambda: ops.Adam([a], [b], [f(64)], [f(64)], out=([f(64).half()], [f(64)], [f(64)]))):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: ops.GradientClip([a, a]), lambda: ops.GradientClip([a, a[8:]]),
                 lambda: ops.GradientClip([a, b], out=[b, f(64)]),
                 lambda: ops.Adam([a], [b], [f(64)], [b]), lambda: ops.Adam([a], [a], [f(64)], [f(64)])):
        with pytest.raises(NativeError, match="shares memory"):
            call()
    shared = ops.GradientClip([a, a], out=[f(64), f(64)])  # inputs may be the same
    assert abs(shared.norm().item() - math.sqrt(2) * a.double().norm().item()) < 1e-4
    h, s = ops.GradientClip([a]), ops.Adam([a], [b], [f(64)], [f(64).square()])
    for call in (lambda: h.clip(0.0), lambda: h.clip(-1.0), lambda: h.clip(math.nan),
                 lambda: s.step(0, 0.1), lambda: s.step(1, math.nan)):
        with pytest.raises(NativeError):
            call()
    with pytest.raises(ValueError):
        s.step(1, 0.1, max_norm=0.0)
    for betas in ((1.0, 0.9), (0.9, -0.1)):
        with pytest.raises(NativeError):
            ops.Adam([a], [b], [f(64)], [f(64)], betas=betas).step(1, 0.1)
