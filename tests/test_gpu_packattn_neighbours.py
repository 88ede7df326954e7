"""Sequences, groups of heads and rows of one call whose cotangents differ by
many powers of two, or are infinite: each has the accuracy that it has alone."""
import math

import pytest
import torch

from tests import sequence_ref as R
from bindcraft2_amd import ops

pytestmark = pytest.mark.gpu


class Packed:
    def __init__(self, lengths, heads, kv, d, dtype, causal, seed=0):
        g = torch.Generator("cuda").manual_seed(seed)
        rand = lambda n, h: (1.2 * torch.randn(n, h, d, generator=g, device="cuda")).to(dtype)  # noqa: E731
        self.lengths, self.causal, self.heads, self.kv, self.d = lengths, causal, heads, kv, d
        ends = lambda i: torch.tensor([0] + [x[i] for x in lengths], device="cuda").cumsum(0).int()  # noqa: E731
        self.qo, self.ko = ends(0), ends(1)
        nq, nk = int(self.qo[-1]), int(self.ko[-1])
        self.q, self.g, self.k, self.v = rand(nq, heads), rand(nq, heads), rand(nk, kv), rand(nk, kv)

    def span(self, b):
        return (slice(int(self.qo[b]), int(self.qo[b + 1])), slice(int(self.ko[b]), int(self.ko[b + 1])))

    def times(self, rows, heads, by):
        self.g[rows, heads] = (self.g[rows, heads].float() * by).to(self.g.dtype)

    def run(self):
        op = ops.PackedAttention(self.causal)
        out, lse = op.forward(self.q, self.k, self.v, self.qo, self.ko)
        self.got = dict(zip(("d_q", "d_k", "d_v"), op.backward(self.g, self.q, self.k, self.v, out, lse, self.qo,
                                                               self.ko)))

    def verify(self, b, group=None):
        """One sequence's gradients, or those of one group of heads, by themselves."""
        rows, keys = self.span(b)
        n = self.heads // self.kv
        hq, hk = (slice(None),) * 2 if group is None else (slice(group * n, group * n + n), slice(group, group + 1))
        want = R.attention(self.q[rows, hq], self.k[keys, hk], self.v[keys, hk], self.causal, self.d ** -0.5,
                           self.g[rows, hq])
        for name, x in self.got.items():
            x = x[rows, hq] if name == "d_q" else x[keys, hk]
            R.check(f"{name} of sequence {b}, group {group}", x, *want[name])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,d", [(2, 1, 64), (6, 2, 32), (8, 8, 128)])
@pytest.mark.parametrize("causal", [True, False])
def test_sequences(cuda, causal, heads, kv, d, dtype):
    p = Packed([(65, 700), (65, 700), (40, 40), (65, 700), (200, 200)], heads, kv, d, dtype, causal)
    for b, by in enumerate((1e-4, 300.0, 1.0, 1e-3, 1e-2)):
        p.times(p.span(b)[0], slice(None), by)
    p.g[p.span(2)[0].start + 3, 0, 5] = math.inf
    p.run()
    for b in (0, 1, 3, 4):
        p.verify(b)


@pytest.mark.parametrize("heads,kv,d", [(4, 2, 64), (9, 3, 16), (64, 64, 32)])
@pytest.mark.parametrize("causal", [True, False])
def test_groups_of_heads(cuda, causal, heads, kv, d):
    p = Packed([(65, 900), (300, 300)], heads, kv, d, torch.float16, causal, 1)
    n = heads // kv
    p.times(slice(None), slice(0, n), 300.0)
    p.times(slice(None), slice(n, 2 * n), 1e-4)
    p.run()
    for b in range(2):
        p.verify(b, 0)
        p.verify(b, 1)


def test_infinite_values_of_another_sequence(cuda):
    p = Packed([(65, 900), (30, 30), (0, 50), (65, 900)], 2, 1, 64, torch.float16, False, 2)
    p.times(slice(None), slice(None), 1e-4)
    p.v[p.span(1)[1]] = math.inf
    p.v[p.span(2)[1]] = -60000.0  # of keys without a query
    p.run()
    p.verify(0)
    p.verify(3)


@pytest.mark.parametrize("what", [math.inf, -math.inf, math.nan, 60000.0])
@pytest.mark.parametrize("m,n", [(700, 600), (400, 330), (40, 0)])
def test_cotangents_of_rows_without_a_key(cuda, m, n, what):
    p = Packed([(m, n), (65, 700)], 4, 2, 64, torch.float16, True, 3)
    p.times(slice(None), slice(None), 1e-4)
    p.g[:m - n] = what
    p.run()
    p.g[:m - n] = 0  # the definition multiplies them by P = 0
    p.verify(0)
    p.verify(1)


def test_rows_of_one_sequence(cuda):
    """d_q of each row by its own cotangent."""
    p = Packed([(300, 900)], 4, 2, 64, torch.float16, False, 4)
    small = torch.arange(300, device="cuda") % 3 == 0
    p.times(small, slice(None), 1e-4)
    p.times(~small, slice(None), 300.0)
    p.run()
    for rows in (small, ~small):
        want = R.attention(p.q[rows], p.k, p.v, False, 0.125, p.g[rows])
        R.check("d_q", p.got["d_q"][rows], *want["d_q"])


def test_parts_of_long_sequences(cuda):
    """Few workgroups, whose rows and keys are cut into parts."""
    p = Packed([(2600, 2600), (2600, 2600)], 2, 1, 64, torch.float16, True, 5)
    p.times(p.span(0)[0], slice(None), 300.0)
    p.times(p.span(1)[0], slice(None), 1e-4)
    p.run()
    p.verify(0)
    p.verify(1)
