"""Attention of packed sequences and its gradient against the definition in 64
bits: types, widths, grouped heads, lengths on both sides of the tiles, empty
sequences and rows without a key, padded batches and caches with garbage,
strides, offsets past 32 bits, streams and graphs."""
import math

import pytest
import torch

from tests import sequence_ref as R
from bindcraft2_amd import ops

pytestmark = pytest.mark.gpu
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
NAN = float("nan")


def rand(g, *shape, dtype, scale=1.2):
    return (scale * torch.randn(*shape, generator=g, device="cuda")).to(dtype)


def offsets(lengths):
    return torch.tensor([0, *lengths], device="cuda").cumsum(0).int()


class Problem:
    """Sequences of (queries, keys); q_cap and k_cap: each in so many tokens."""

    def __init__(self, lengths, heads=2, kv=1, d=64, dtype=torch.bfloat16, causal=True, seed=0, scale=None,
                 q_cap=None, k_cap=None, spare=0):
        g = torch.Generator("cuda").manual_seed(seed)
        self.lengths, self.causal, self.scale = lengths, causal, scale
        self.lq, self.lk = [m for m, _ in lengths], [n for _, n in lengths]
        have_q = [q_cap] * len(lengths) if q_cap else self.lq
        have_k = [k_cap] * len(lengths) if k_cap else self.lk
        self.qo, self.ko = offsets(have_q), offsets(have_k)
        i32 = lambda v: torch.tensor(v, device="cuda", dtype=torch.int32)  # noqa: E731
        self.ql = i32(self.lq) if q_cap else None
        self.kl = i32(self.lk) if k_cap else None
        nq, nk = sum(have_q) + spare, sum(have_k) + spare
        # what belongs to no sequence is NaN
        self.q, self.d_out = (torch.full((nq, heads, d), NAN, device="cuda", dtype=dtype) for _ in range(2))
        self.k, self.v = (torch.full((nk, kv, d), NAN, device="cuda", dtype=dtype) for _ in range(2))
        for b, (m, n) in enumerate(lengths):
            i, j = int(self.qo[b]), int(self.ko[b])
            self.q[i:i + m] = rand(g, m, heads, d, dtype=dtype)
            self.d_out[i:i + m] = rand(g, m, heads, d, dtype=dtype)
            self.k[j:j + n] = rand(g, n, kv, d, dtype=dtype)
            self.v[j:j + n] = rand(g, n, kv, d, dtype=dtype)
        self.op = ops.PackedAttention(causal, scale)

    def where(self):
        return self.qo, self.ko, self.kl, self.ql

    def run(self):
        out, lse = self.op.forward(self.q, self.k, self.v, *self.where())
        grads = self.op.backward(self.d_out, self.q, self.k, self.v, out, lse, *self.where())
        return dict(zip(("out", "lse", "d_q", "d_k", "d_v"), (out, lse, *grads)))

    def verify(self, got=None, rest=0.0):
        got = got or self.run()
        scale = self.q.shape[2] ** -0.5 if self.scale is None else self.scale
        free_q = torch.ones(self.q.shape[0], dtype=torch.bool, device="cuda")
        free_k = torch.ones(self.k.shape[0], dtype=torch.bool, device="cuda")
        for b, (m, n) in enumerate(self.lengths):
            at_q = slice(int(self.qo[b]), int(self.qo[b]) + m)
            at_k = slice(int(self.ko[b]), int(self.ko[b]) + n)
            free_q[at_q], free_k[at_k] = False, False
            want = R.attention(self.q[at_q], self.k[at_k], self.v[at_k], self.causal, scale, self.d_out[at_q])
            for name, (value, tol) in want.items():
                if name not in got:
                    continue
                x = got[name][:, at_q] if name == "lse" else got[name][at_k if name in ("d_k", "d_v") else at_q]
                R.check(f"{name} of sequence {b} {(m, n)}", x, value, tol)
        for name, x in got.items():  # rows of no sequence
            x = x[:, free_q] if name == "lse" else x[free_k if name in ("d_k", "d_v") else free_q]
            if name == "lse":
                assert (x == (-math.inf if rest == 0 else rest)).all(), name
            else:
                assert (x == rest).all(), name
        return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [8, 16, 24, 32, 40, 64, 72, 80, 96, 104, 128])
def test_widths(cuda, d, dtype):
    for causal in (True, False):
        print(f"widths {d} {dtype} {causal}", flush=True)
        Problem([(70, 70), (5, 33)], 4, 2, d, TYPES[dtype], causal, d).verify()


@pytest.mark.parametrize("heads,kv", [(1, 1), (4, 4), (6, 2), (8, 1), (5, 5), (12, 3), (9, 3), (7, 1), (16, 8), (64, 2)])
@pytest.mark.parametrize("causal", [True, False])
def test_heads(cuda, heads, kv, causal):
    print(f"heads {heads} {kv} {causal}", flush=True)
    Problem([(37, 37), (1, 90), (130, 130)], heads, kv, 32, torch.float16, causal, heads).verify()
    Problem([(37, 37), (1, 90)], heads, kv, 128, torch.bfloat16, causal, heads).verify()


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 191, 192, 193, 255, 256, 257, 700])
@pytest.mark.parametrize("causal", [True, False])
def test_lengths(cuda, n, causal):
    print(f"lengths {n} {causal}", flush=True)
    Problem([(n, n)], 2, 1, 64, torch.bfloat16, causal, n).verify()
    Problem([(n, n + 77), (n, 1)], 2, 2, 128, torch.float16, causal, n).verify()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_empty_and_unequal_sequences(cuda, causal, dtype):
    """No queries, no keys, neither, fewer keys than queries."""
    Problem([(0, 5), (3, 0), (0, 0), (7, 7), (100, 40), (1, 1), (2, 300), (0, 0)], 4, 2, 64, TYPES[dtype],
            causal).verify()
    Problem([(200, 3)], 4, 2, 128, TYPES[dtype], causal).verify()


def test_no_tokens_and_no_sequences(cuda):
    Problem([], 2, 1, 64).verify()
    Problem([(0, 0)], 2, 1, 64).verify()
    Problem([(0, 0), (0, 9)], 2, 1, 64).verify()
    Problem([(4, 0)], 2, 1, 64).verify()
    Problem([], 2, 1, 64, spare=70).verify()


WIDE = [(300, 300), (0, 7), (130, 130), (70, 200), (90, 30), (3, 0)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [16, 40, 64, 72, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_rows_that_fill_the_card(cuda, causal, d, dtype):
    """128-row workgroups: with as many heads as here, from a few hundred tokens."""
    print(f"rows {d} {dtype} {causal}", flush=True)
    Problem(WIDE, 64, 64, d, TYPES[dtype], causal, d).verify()
    Problem(WIDE[:4], 192, 64, d, TYPES[dtype], causal, d).verify()


def test_rows_that_fill_the_card_padded(cuda):
    lengths = [(200, 200), (0, 0), (64, 40), (17, 40), (0, 30), (12, 0), (300, 301)]
    for fill in (True, False):
        p = Problem(lengths, 64, 64, 32, torch.bfloat16, True, q_cap=300, k_cap=301, spare=150)
        if fill:
            p.verify()
            continue
        out = torch.full_like(p.q, 7.0)
        _, lse = p.op.forward(p.q, p.k, p.v, *p.where(), out=out)
        grads = tuple(torch.full_like(t, 7.0) for t in (p.q, p.k, p.v))
        p.op.backward(p.d_out, p.q, p.k, p.v, out, lse, *p.where(), grads=grads)
        p.verify(dict(zip(("out", "d_q", "d_k", "d_v"), (out, *grads))), rest=7.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv,d", [(8, 1, 64), (2, 2, 128), (12, 3, 32), (64, 64, 16), (40, 1, 24), (1, 1, 104)])
@pytest.mark.parametrize("causal", [True, False])
def test_long_caches(cuda, causal, heads, kv, d, dtype):
    """Keys in stretches over workgroups, joined: few and many of them a row."""
    print(f"caches {heads} {kv} {d} {dtype} {causal}", flush=True)
    Problem([(1, 20000)], heads, kv, d, TYPES[dtype], causal, 1).verify()
    Problem([(1, 5000), (3, 70), (0, 9), (2, 0), (1, 1), (5, 4097), (1, 300)], heads, kv, d, TYPES[dtype], causal,
            2).verify()


def test_long_caches_of_fixed_capacity(cuda):
    lengths = [(1, n) for n in (1, 0, 700, 2048, 31, 33, 257, 2047)]
    p = Problem(lengths, 8, 2, 64, torch.bfloat16, True, k_cap=2048, spare=40)
    p.verify()
    out = torch.full_like(p.q, 7.0)
    p.op.forward(p.q, p.k, p.v, *p.where(), out=out)
    p.verify({"out": out}, rest=7.0)


@pytest.mark.parametrize("count", [61, 62, 63, 200, 300, 1000])
def test_many_caches(cuda, count):
    """One query each: held in a wave's lanes to 256 entries, read again beyond."""
    g = torch.Generator().manual_seed(count)
    lengths = [(1, n) for n in torch.randint(0, 90000 // count, (count,), generator=g).tolist()]
    p = Problem(lengths, 4, 2, 32, torch.float16, True)
    out, lse = p.op.forward(p.q, p.k, p.v, *p.where())
    assert not out.isnan().any()
    for b in sorted({0, 1, 60, count // 2, count - 2, count - 1}):
        i, j, n = b, int(p.ko[b]), lengths[b][1]
        want = R.attention(p.q[i:i + 1], p.k[j:j + n], p.v[j:j + n], True, 32 ** -0.5)
        R.check(f"out of sequence {b}", out[i:i + 1], *want["out"])
        R.check(f"lse of sequence {b}", lse[:, i:i + 1], *want["lse"])


def test_a_wide_row_among_caches(cuda):
    """More than 32 rows in a sequence beside single tokens."""
    Problem([(1, 3000), (50, 3000), (1, 10), (1, 1)], 8, 2, 64, torch.bfloat16, True).verify()


@pytest.mark.parametrize("count", [63, 64, 65, 300, 5000])
def test_many_sequences(cuda, count):
    """Searched 64 at a time: one, two and three levels of them."""
    g = torch.Generator().manual_seed(count)
    lengths = [(m, m + e) for m, e in zip(torch.randint(4, (count,), generator=g).tolist(),
                                          torch.randint(3, (count,), generator=g).tolist())]
    p = Problem(lengths, 2, 1, 16, torch.bfloat16)
    got = p.run()
    for b in sorted({0, 1, 61, 62, min(63, count - 1), count // 2, count - 2, count - 1}):
        m, n = lengths[b]
        i, j = int(p.qo[b]), int(p.ko[b])
        want = R.attention(p.q[i:i + m], p.k[j:j + n], p.v[j:j + n], True, 0.25, p.d_out[i:i + m])
        for name, (value, tol) in want.items():
            x = got[name][:, i:i + m] if name == "lse" else got[name][j:j + n] if name in ("d_k", "d_v") else \
                got[name][i:i + m]
            R.check(f"{name} of sequence {b}", x, value, tol)
    assert not any(x.isnan().any() for x in got.values())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_padded_batch_of_garbage(cuda, causal, dtype):
    """A capacity for each sequence, NaN behind its length and behind the last."""
    lengths = [(5, 5), (0, 0), (40, 40), (64, 64), (17, 40), (0, 30), (12, 0)]
    Problem(lengths, 4, 2, 64, TYPES[dtype], causal, q_cap=64, k_cap=70, spare=130).verify()
    Problem(lengths, 2, 1, 128, TYPES[dtype], causal, q_cap=150, k_cap=64).verify()


def test_given_results_keep_rows_of_no_sequence(cuda):
    p = Problem([(5, 9), (40, 40)], 4, 2, 64, q_cap=64, k_cap=70, spare=200)
    out = torch.full_like(p.q, 7.0)
    _, lse = p.op.forward(p.q, p.k, p.v, *p.where(), out=out)
    grads = tuple(torch.full_like(t, 7.0) for t in (p.q, p.k, p.v))
    r = p.op.backward(p.d_out, p.q, p.k, p.v, out, lse, *p.where(), grads=grads)
    assert all(a is b for a, b in zip(r, grads))
    p.verify(dict(zip(("out", "d_q", "d_k", "d_v"), (out, *grads))), rest=7.0)


def test_offsets_that_do_not_start_at_zero(cuda):
    p = Problem([(30, 30), (50, 50)], 4, 2, 64)
    whole = p.run()
    part = slice(30, 80)
    out, lse = p.op.forward(p.q, p.k, p.v, p.qo[1:], p.ko[1:])
    grads = p.op.backward(p.d_out, p.q, p.k, p.v, out, lse, p.qo[1:], p.ko[1:])
    for name, x in zip(("out", "d_q", "d_k", "d_v"), (out, *grads)):
        assert torch.equal(x[part], whole[name][part]) and not x[:30].any(), name
    assert torch.equal(lse[:, part], whole["lse"][:, part]) and (lse[:, :30] == -math.inf).all()


def test_offsets_past_the_tokens_are_cut(cuda):
    """What the device finds in the offsets reaches no memory outside."""
    p = Problem([(30, 30), (50, 50)], 4, 2, 64)
    want = p.run()
    far = p.qo.clone()
    far[-1] = 2 ** 31 - 1
    out, lse = p.op.forward(p.q, p.k, p.v, far, far)
    grads = p.op.backward(p.d_out, p.q, p.k, p.v, out, lse, far, far)
    for name, x in zip(("out", "lse", "d_q", "d_k", "d_v"), (out, lse, *grads)):
        assert torch.equal(x, want[name]), name
    for bad in ([50, 30, 80], [0, -5, 80], [80, 80, 0], [-9, -9, -9], [90, 95, 99]):  # no answer, and no fault
        o = torch.tensor(bad, device="cuda", dtype=torch.int32)
        out, lse = p.op.forward(p.q, p.k, p.v, o, o)
        p.op.backward(p.d_out, p.q, p.k, p.v, out, lse, o, o)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", TYPES)
def test_layouts(cuda, dtype):
    """Slices of one projection and of one gradient; heads first."""
    t = TYPES[dtype]
    p = Problem([(70, 70), (9, 9), (140, 140)], 6, 2, 64, t)
    want = p.run()
    fused = torch.cat((p.q, p.k, p.v), 1)
    p.q, p.k, p.v = fused[:, :6], fused[:, 6:8], fused[:, 8:]
    grad = torch.empty_like(fused)
    out, lse = p.op.forward(p.q, p.k, p.v, p.qo)
    p.op.backward(p.d_out, p.q, p.k, p.v, out, lse, p.qo, grads=(grad[:, :6], grad[:, 6:8], grad[:, 8:]))
    assert torch.equal(out, want["out"]) and torch.equal(lse, want["lse"])
    assert torch.equal(grad, torch.cat((want["d_q"], want["d_k"], want["d_v"]), 1))
    first = lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    p.q, p.k, p.v, p.d_out = map(first, (p.q, p.k, p.v, p.d_out))
    got = p.run()
    for name, x in got.items():
        assert torch.equal(x, want[name]), name


def test_scores_of_a_wide_range(cuda):
    """Rows whose maximum rises from key to key, and scores far apart."""
    for dtype in TYPES.values():
        p = Problem([(130, 300)], 2, 1, 64, dtype, False, scale=1.0)
        ramp = torch.linspace(0, 1, 300, device="cuda")[:, None, None]
        p.k.copy_((p.q[:1, :1].float() * ramp * 2).to(dtype))
        p.q.copy_(p.q[:1].expand_as(p.q))
        p.verify()
        p.k.copy_(p.k.flip(0))
        p.verify()


def test_large_and_small_cotangents(cuda):
    """A binary16 dS far below its normal numbers, beside one far above."""
    for scale in (1e-4, 1.0, 300.0):
        p = Problem([(65, 700)], 2, 1, 64, torch.float16, False)
        p.d_out.copy_((p.d_out.float() * scale).half())
        p.verify()


def test_keys_of_infinities_and_nan(cuda):
    """What a masked place holds stays there: NaN in keys that no row sees."""
    p = Problem([(64, 64)], 2, 1, 64, torch.bfloat16, True)
    p.k[40:, :, :] = NAN
    out, lse = p.op.forward(p.q, p.k, p.v, p.qo)
    assert not out[:40].isnan().any() and out[40:].isnan().all() and lse[:, 40:].isnan().all()
    want = R.attention(p.q[:40], p.k[:40], p.v[:40], True, 0.125)
    R.check("out", out[:40], *want["out"])


def test_offsets_past_32_bits(cuda):
    """A sequence whose tokens lie beyond 2^31 elements of its buffer."""
    tokens, d = 40_000_000, 64
    k = torch.empty(tokens, 1, d, device="cuda", dtype=torch.bfloat16)
    v = torch.empty(tokens, 1, d, device="cuda", dtype=torch.bfloat16)
    p = Problem([(3, 500)], 2, 1, d, torch.bfloat16, True)
    at = tokens - 500
    k[at:], v[at:] = p.k, p.v
    ko = torch.tensor([at, tokens], device="cuda", dtype=torch.int32)
    out, lse = p.op.forward(p.q, k, v, p.qo, ko)
    dk, dv = torch.zeros_like(k), torch.zeros_like(v)
    dq = torch.zeros_like(p.q)
    p.op.backward(p.d_out, p.q, k, v, out, lse, p.qo, ko, grads=(dq, dk, dv))
    p.verify({"out": out, "lse": lse, "d_q": dq, "d_k": dk[at:], "d_v": dv[at:]})


@pytest.mark.parametrize("dtype", TYPES)
def test_same_bits_and_graph(cuda, dtype):
    """Replayed after the offsets and the values have changed."""
    p = Problem([(70, 70), (130, 130)], 4, 2, 64, TYPES[dtype], spare=60)
    p.qo[2:], p.ko[2:] = 200, 200
    for t in (p.q, p.k, p.v, p.d_out):
        t.nan_to_num_(0.5)
    want = {k: v.clone() for k, v in p.run().items()}
    assert all(torch.equal(v, want[k]) for k, v in p.run().items())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = p.run()
    for cut in (70, 3, 129, 200):
        p.qo[1], p.ko[1] = cut, cut
        for t in (p.q, p.k, p.v, p.d_out):
            t.mul_(0.9)
        want = {k: v.clone() for k, v in p.run().items()}
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(v, want[k]) for k, v in held.items()), cut


def test_two_streams_at_once(cuda):
    ps = [Problem([(300, 300), (5, 400)], 4, 2, 64, torch.float16, seed=i) for i in range(2)]
    want = [{k: v.clone() for k, v in p.run().items()} for p in ps]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [None, None]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = ps[i].run()
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(g[k], w[k]) for k in w)


def test_differences(cuda):
    """The gradient formulas against differences of the 64-bit definition."""
    p = Problem([(5, 9)], 4, 2, 16, torch.float16)
    got = p.run()
    x, h = [t.double() for t in (p.q, p.k, p.v)], 1e-4
    # the definition reads the type for its tolerances alone, and f32 holds the steps
    loss32 = lambda xs: (R.attention(*[t.float() for t in xs], True, 0.25)["out"][0] * p.d_out.double()).sum()  # noqa: E731
    for i, name in enumerate(("d_q", "d_k", "d_v")):
        for at in [(0, 0, 0), (3, 1, 7), (4, 0, 15)]:
            up, down = [t.clone() for t in x], [t.clone() for t in x]
            up[i][at] = (up[i][at] + h).float().double()
            down[i][at] = (down[i][at] - h).float().double()
            slope = (loss32(up) - loss32(down)) / (up[i][at] - down[i][at])
            # binary16's roundings of P, dS, out and the result: 4 half steps of the
            # terms' size, and h^2
            assert abs(slope - got[name][at].double()) < 4 * 2 ** -11 * 4 + 1e-4, (name, at)
