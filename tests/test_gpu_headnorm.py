"""Norm and rotation of heads and their gradient against the definition in 64
bits: types, widths on both sides of each layout, strides, far positions, in
place, one token and many, without keys, streams and graphs."""
import pytest
import torch

from tests import sequence_ref as R
from bindcraft2_amd import NativeError, ops

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def inputs(n, hq, hk, d, r, dtype, seed=0, far=0, wide=torch.int32, layout="fused"):
    g = torch.Generator("cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    if layout == "fused":  # slices of one projection
        qkv = rand(n, hq + 2 * hk + 1, d).to(dtype)
        q, k = qkv[:, :hq], qkv[:, hq:hq + hk]
    elif layout == "heads":  # heads first
        q, k = rand(hq, n, d).to(dtype).transpose(0, 1), rand(hk, n, d).to(dtype).transpose(0, 1)
    else:  # a column more, so that rows lie on odd addresses
        q, k = rand(n, hq, d + 1).to(dtype)[..., 1:], rand(n, hk, d + 1).to(dtype)[..., :-1]
    pos = torch.randint(far, (n,), generator=g, device="cuda") if far else torch.arange(n, device="cuda") % 97
    freq = (10000.0 ** (-torch.arange(0, r, 2, device="cuda").double() / max(r, 1))).float()
    return q, k, pos.to(wide), freq, 1 + 0.3 * rand(d), 1 + 0.3 * rand(d), rand(n, hq, d).to(dtype), rand(n, hk, d).to(dtype)


def verify(t, eps=1e-5, interleaved=False, wt=None, where=None):
    q, k, pos, freq, qw, kw, dq, dk = t
    if wt is not None:
        qw, kw = qw.to(wt), kw.to(wt)
    op = ops.HeadNormRotate(freq, eps, interleaved)
    out = op.forward(q, k, pos, qw, kw)
    grads = op.backward((dq, dk), q, k, pos, qw, kw)
    for i, (x, w, d) in enumerate(((q, qw, dq), (k, kw, dk))):
        y, tol = R.head_norm(x, pos, freq, w, eps, interleaved)
        R.check("qk"[i], out[i], y, tol + R.rounding(y, q.dtype))
        dx, tol, dw, tol_w = R.head_norm_grad(d, x, pos, freq, w, eps, interleaved)
        R.check("d_" + "qk"[i], grads[i], dx, tol + R.rounding(dx, q.dtype))
        R.check("d_weight", grads[2 + i], dw, tol_w)
    return out, grads


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,r", [(2, 2), (2, 0), (6, 4), (10, 10), (16, 8), (16, 16), (20, 12), (34, 2), (64, 32),
                                 (64, 64), (80, 80), (96, 24), (126, 126), (128, 128), (128, 64), (256, 256),
                                 (512, 128)])
def test_widths(cuda, d, r, dtype):
    for interleaved in (False, True):
        print(f"widths {d} {r} {dtype} {interleaved}", flush=True)
        verify(inputs(5, 3, 2, d, r, TYPES[dtype], d + r), interleaved=interleaved)


@pytest.mark.parametrize("n,hq,hk", [(1, 1, 1), (1, 32, 8), (3, 9, 1), (4, 5, 7), (33, 1, 2), (517, 8, 2), (3000, 4, 4)])
@pytest.mark.parametrize("dtype", TYPES)
def test_tokens_and_heads(cuda, n, hq, hk, dtype):
    verify(inputs(n, hq, hk, 128, 128, TYPES[dtype], n))
    verify(inputs(n, hq, hk, 48, 16, TYPES[dtype], n), interleaved=True)


@pytest.mark.parametrize("layout", ["heads", "odd"])
@pytest.mark.parametrize("dtype", TYPES)
def test_layouts(cuda, layout, dtype):
    verify(inputs(21, 4, 2, 64, 64, TYPES[dtype], 3, layout=layout))
    verify(inputs(21, 4, 2, 64, 32, TYPES[dtype], 3, layout=layout), interleaved=True)


@pytest.mark.parametrize("far,wide", [(1_000_000, torch.int32), (2 ** 31 - 1, torch.int32), (2 ** 40, torch.int64)])
def test_far_positions(cuda, far, wide):
    verify(inputs(64, 3, 2, 64, 64, torch.float32, 5, far, wide))


def test_negative_positions(cuda):
    q, k, pos, *rest = inputs(64, 3, 2, 64, 64, torch.float32, 5)
    verify((q, k, -pos, *rest))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_weights_of_the_operands_type(cuda, dtype):
    verify(inputs(9, 4, 2, 64, 64, dtype, 6), wt=dtype)


def test_without_keys_and_without_tokens(cuda):
    q, k, pos, freq, qw, kw, dq, dk = inputs(7, 4, 2, 64, 64, torch.bfloat16)
    op = ops.HeadNormRotate(freq, 1e-5)
    both = op.forward(q, k, pos, qw, kw)
    alone = op.forward(q, None, pos, qw)
    assert alone[1] is None and torch.equal(alone[0], both[0])
    g = op.backward((dq, None), q, None, pos, qw)
    assert g[1] is None and g[3] is None
    assert torch.equal(g[0], op.backward((dq, dk), q, k, pos, qw, kw)[0])
    z = op.backward((dq[:0], dk[:0]), q[:0], k[:0], pos[:0], qw, kw)
    assert z[0].shape == (0, 4, 64) and not z[2].any() and not z[3].any()


def test_zero_rows_and_nan_rows(cuda):
    t = list(inputs(8, 4, 2, 64, 32, torch.float32))
    t[0] = t[0].clone()
    t[0][3] = 0.0
    verify(t)
    t[0][5, 1] = float("nan")
    out, grads = ops.HeadNormRotate(t[3], 1e-5).forward(*t[:3], *t[4:6]), None
    assert out[0][5, 1].isnan().all() and not out[0][:5].isnan().any() and not out[0][5, 2:].isnan().any()


def test_in_place(cuda):
    q, k, pos, freq, qw, kw, dq, dk = inputs(33, 4, 2, 64, 64, torch.bfloat16)
    op = ops.HeadNormRotate(freq)
    want, grads = op.forward(q, k, pos, qw, kw), op.backward((dq, dk), q, k, pos, qw, kw)
    dq2, dk2 = dq.clone(), dk.clone()
    g = op.backward((dq2, dk2), q, k, pos, qw, kw, out=(dq2, dk2))
    assert g[0] is dq2 and all(torch.equal(a, b) for a, b in zip(g, grads))
    got = op.forward(q, k, pos, qw, kw, out=(q, k))  # slices of one projection
    assert got[0] is q and torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_overlaps_are_refused(cuda):
    q, k, pos, freq, qw, kw, dq, dk = inputs(8, 4, 2, 64, 64, torch.bfloat16)
    op = ops.HeadNormRotate(freq)
    whole = torch.zeros(8 * 7 * 64 + 8, device="cuda", dtype=q.dtype)
    shifted = whole[8:8 + 8 * 4 * 64].view(8, 4, 64)
    with pytest.raises(NativeError, match="overlaps"):
        op.forward(whole[:8 * 4 * 64].view(8, 4, 64), k, pos, qw, kw, out=(shifted, torch.empty_like(dk)))
    with pytest.raises(NativeError, match="elements overlap"):
        op.forward(q, k, pos, qw, kw, out=(k.expand(8, 2, 64).repeat(1, 2, 1), k[:, :1].expand(8, 2, 64)))


def test_same_bits_and_graph(cuda):
    t = inputs(700, 8, 2, 64, 64, torch.float32, 4)
    q, k, pos, freq, qw, kw, dq, dk = t
    op = ops.HeadNormRotate(freq)
    call = lambda: (*op.forward(q, k, pos, qw, kw), *op.backward((dq, dk), q, k, pos, qw, kw))  # noqa: E731
    want = [x.clone() for x in call()]
    assert all(torch.equal(a, b) for a, b in zip(want, call()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    for i in range(3):
        for x in (q, k, dq, dk):
            x.mul_(1.0 + 0.5 * i)
        want = [x.clone() for x in call()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, held)), i


def test_other_stream(cuda):
    q, k, pos, freq, qw, kw, dq, dk = inputs(300, 8, 2, 64, 64, torch.float32, 4)
    op = ops.HeadNormRotate(freq)
    want = op.forward(q, k, pos, qw, kw)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = op.forward(q, k, pos, qw, kw)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_differences(cuda):
    """The gradient against differences of the 64-bit definition."""
    q, k, pos, freq, qw, kw, dq, dk = inputs(3, 2, 1, 16, 8, torch.float32, 9)
    grads = ops.HeadNormRotate(freq, 1e-3).backward((dq, dk), q, k, pos, qw, kw)
    loss = lambda x, w: (R.head_norm(x, pos, freq, w, 1e-3, False)[0] * dq.double()).sum()  # noqa: E731
    x, w, h = q.double().contiguous(), qw.double(), 1e-5
    for at in [(0, 0, 0), (1, 1, 5), (2, 0, 15), (0, 1, 9)]:
        step = torch.zeros_like(x)
        step[at] = h
        slope = (loss(x + step, w) - loss(x - step, w)) / (2 * h)
        assert abs(slope - grads[0][at].double()) < 1e-5 * (1 + abs(slope))  # h^2 and f32's own
    for i in (0, 7, 15):
        step = torch.zeros_like(w)
        step[i] = h
        slope = (loss(x, w + step) - loss(x, w - step)) / (2 * h)
        assert abs(slope - grads[2][i].double()) < 1e-5 * (1 + abs(slope))
