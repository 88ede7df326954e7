"""What the sequence operators' documentation allows at its borders: no heads,
rows without a key whose cotangents are NaN, results given beside new ones, one
token of any stride, more rows than a launch takes, and refused tensors."""
import math

import pytest
import torch

from tests import sequence_ref as R
from bindcraft2_amd import NativeError, ops

pytestmark = pytest.mark.gpu
NAN = float("nan")


def rand(seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda").to(dtype)


def i32(*v):
    return torch.tensor(v, device="cuda", dtype=torch.int32)


def test_headnorm_of_no_queries(cuda):
    """Weights of no heads have gradients of zero."""
    freq, w = torch.ones(16, device="cuda"), 1 + 0.1 * rand(1, 32)
    q, k, pos = rand(2, 9, 0, 32), rand(3, 9, 2, 32), torch.arange(9, device="cuda")
    op = ops.HeadNormRotate(freq)
    out = op.forward(q, k, pos, w, w)
    y, tol = R.head_norm(k, pos, freq, w, 1e-6, False)
    R.check("k", out[1], y, tol + R.rounding(y, k.dtype))
    torch.full((2, 32), NAN, device="cuda")  # what the allocator may hand out next
    d = op.backward((q, k), q, k, pos, w, w)
    assert d[0].shape == q.shape and (d[2] == 0).all() and d[3].isfinite().all()


def test_headnorm_of_one_token_of_any_stride(cuda):
    w, freq = 1 + 0.1 * rand(1, 64), torch.ones(32, device="cuda")
    base = rand(2, 4, 64, dtype=torch.float16)
    pos = i32(7)
    op = ops.HeadNormRotate(freq)
    want = op.forward(base[None].contiguous(), None, pos, w)[0]
    for stride in (0, 3, 1 << 41):
        q = base.as_strided((1, 4, 64), (stride, 64, 1))
        assert torch.equal(op.forward(q, None, pos, w)[0], want), stride


def test_attention_of_one_token_of_any_stride(cuda):
    base = [rand(i, 2, 64, dtype=torch.bfloat16) for i in range(4)]
    off, op = i32(0, 1), ops.PackedAttention()

    def run(s):
        q, k, v, g = (t.as_strided((1, 2, 64), (s, 64, 1)) for t in base)
        out, lse = op.forward(q, k, v, off)
        return out, lse, *op.backward(g, q, k, v, out, lse, off)
    want = run(128)
    for stride in (0, 3, 1 << 41):
        assert all(torch.equal(a, b) for a, b in zip(run(stride), want)), stride


def test_lse_beside_a_given_out(cuda):
    """out keeps its rows of no sequence; lse, which the call makes, has -inf."""
    q, k = rand(1, 40, 2, 64, dtype=torch.bfloat16), rand(2, 40, 1, 64, dtype=torch.bfloat16)
    out = torch.full_like(q, 3.0)
    torch.full((2, 40), NAN, device="cuda")
    _, lse = ops.PackedAttention().forward(q, k, k, i32(5, 9, 30), out=out)
    assert (lse[:, :5] == -math.inf).all() and (lse[:, 30:] == -math.inf).all() and lse[:, 5:30].isfinite().all()
    assert (out[:5] == 3).all() and (out[30:] == 3).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n", [(5, 3), (70, 40), (400, 330), (40, 0)])
def test_rows_without_a_key_hold_anything(cuda, m, n, dtype):
    """The first m - n queries see no key: NaN there, and in their cotangents,
    reaches nothing."""
    q, g = rand(1, m, 4, 64, dtype=dtype), rand(2, m, 4, 64, dtype=dtype)
    k, v = rand(3, n, 2, 64, dtype=dtype), rand(4, n, 2, 64, dtype=dtype)
    want = R.attention(q, k, v, True, 0.125, g)
    q[:m - n], g[:m - n] = NAN, NAN
    op, qo, ko = ops.PackedAttention(), i32(0, m), i32(0, n)
    out, lse = op.forward(q, k, v, qo, ko)
    grads = op.backward(g, q, k, v, out, lse, qo, ko)
    for name, got in zip(("out", "lse", "d_q", "d_k", "d_v"), (out, lse, *grads)):
        R.check(name, got, *want[name])


@pytest.mark.parametrize("v", [2, 70])
def test_more_rows_than_a_launch_takes(cuda, v):
    rows = (1 << 21) * 2 + 5
    x = torch.full((rows, v), -math.inf, device="cuda", dtype=torch.float16)
    want = torch.arange(rows, device="cuda") % v
    x.scatter_(1, want[:, None], 1.0)
    index, logp = ops.Sampler(top_p=0.9).sample(x, torch.full((rows,), 0.5, device="cuda"))
    assert torch.equal(index, want.int()) and logp.abs().max() < 1e-12


def test_refused_tensors(cuda):
    q, k = rand(1, 8, 4, 64, dtype=torch.float16), rand(2, 8, 2, 64, dtype=torch.float16)
    w, pos, freq = torch.ones(64, device="cuda"), torch.arange(8, device="cuda"), torch.ones(32, device="cuda")
    norm, attn, off = ops.HeadNormRotate(freq), ops.PackedAttention(), i32(0, 8)
    for what, args in {
        "q": (q[0], k, pos, w, w), "q:": (q.double(), k, pos, w, w), "k:": (q, k[:4], pos, w, w),
        "k: ": (q, k.float(), pos, w, w), "positions": (q, k, pos.float(), w, w), "positions:": (q, k, pos[:4], w, w),
        "q_weight": (q, k, pos, w[:32], w), "k_weight": (q, k, pos, w, w.half()), "k_weight: missing": (q, k, pos, w),
        "current device": (q, k, pos.cpu(), w, w), "contiguous": (q[..., ::2], None, pos, w[:32]),
        "contiguous tensor": (q, k, pos, torch.ones(128, device="cuda")[::2], w),
    }.items():
        with pytest.raises(ValueError, match=what):
            norm.forward(*args)
    with pytest.raises(ValueError, match="out: expected"):
        norm.forward(q, k, pos, w, w, out=(q[:4], k))
    with pytest.raises(ValueError, match="d_k: missing"):
        norm.backward((q, None), q, k, pos, w, w)
    other = q.clone()  # k of as many heads is no place for what comes of q
    with pytest.raises(NativeError, match="q_out overlaps k"):
        norm.forward(q, other, pos, w, w, out=(other, torch.empty_like(q)))
    for what, args in {
        "q:": (q.float(), k, k, off), "k:": (q, k[:, :, :32], k, off), "v:": (q, k, k[:4], off),
        "v: ": (q, k, k.bfloat16(), off), "q_offsets": (q, k, k, off.long()), "q_offsets:": (q, k, k, off[:0]),
        "k_offsets: needed": (q, k[:4], k[:4], off), "k_offsets: ": (q, k, k, off, i32(0, 4, 8)),
        "k_lengths": (q, k, k, off, off, i32(1, 2)), "q_lengths": (q, k, k, off, off, None, i32(1, 2)),
        "a divisor": (q, rand(1, 8, 3, 64, dtype=torch.float16), k, off), "current device": (q.cpu(), k, k, off),
    }.items():
        with pytest.raises(ValueError, match=what):
            attn.forward(*args)
    with pytest.raises(NativeError, match="unaligned"):
        attn.forward(torch.empty(8 * 256 + 1, device="cuda", dtype=q.dtype)[1:].view(8, 4, 64), k, k, off)
    with pytest.raises(NativeError, match="width"):
        attn.forward(q[..., :20], k[..., :20], k[..., :20], off)
    out, lse = attn.forward(q, k, k, off)
    with pytest.raises(ValueError, match="lse"):
        attn.backward(q, q, k, k, out, lse[:, :4], off)
    with pytest.raises(ValueError, match="d_out"):
        attn.backward(q.bfloat16(), q, k, k, out, lse, off)
    v = k.clone()
    with pytest.raises(NativeError, match="d_k overlaps v"):
        attn.backward(q, q, k, v, out, lse, off, grads=(torch.empty_like(q), v, torch.empty_like(k)))
    x, u = rand(5, 6, 50), torch.rand(6, device="cuda")
    for what, args in {
        "logits": (x.double(), u), "logits: ": (x[:, :0], u), "uniforms": (x, u[:5]), "uniforms:": (x, u.double()),
        "contiguous": (x, torch.rand(12, device="cuda")[::2]), "current device": (x, u.cpu()),
    }.items():
        with pytest.raises(ValueError, match=what):
            ops.Sampler().sample(*args)
    with pytest.raises(ValueError, match="top_p: expected a value for each of 6 rows"):
        ops.Sampler(top_p=u[:5]).sample(x, u)
    with pytest.raises(NativeError, match="row stride"):
        ops.Sampler().sample(x[:1].expand(6, 50), u)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,heads,kv,d,causal", [(700, 9000, 2, 1, 64, True), (1200, 5000, 3, 1, 128, False),
                                                   (2600, 2600, 2, 2, 32, True), (5100, 5100, 1, 1, 64, True),
                                                   (6001, 6001, 2, 2, 40, True)])
def test_few_long_sequences(cuda, m, n, heads, kv, d, causal, dtype):
    """On both sides of the rules by which few workgroups of rows share the keys."""
    q, g = rand(1, m, heads, d, dtype=dtype), rand(2, m, heads, d, dtype=dtype)
    k, v = rand(3, n, kv, d, dtype=dtype), rand(4, n, kv, d, dtype=dtype)
    op, qo, ko = ops.PackedAttention(causal), i32(0, m), i32(0, n)
    out, lse = op.forward(q, k, v, qo, ko)
    grads = op.backward(g, q, k, v, out, lse, qo, ko)
    want = R.attention(q, k, v, causal, d ** -0.5, g)
    for name, got in zip(("out", "lse", "d_q", "d_k", "d_v"), (out, lse, *grads)):
        R.check(name, got, *want[name])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_graph_of_the_widest(cuda, dtype):
    """Forward and gradient of heads of 128, captured where no call has been before."""
    q, g = rand(1, 300, 4, 128, dtype=dtype), rand(2, 300, 4, 128, dtype=dtype)
    k, v = rand(3, 300, 2, 128, dtype=dtype), rand(4, 300, 2, 128, dtype=dtype)
    op, off = ops.PackedAttention(), i32(0, 120, 300)

    def run():
        out, lse = op.forward(q, k, v, off)
        return out, lse, *op.backward(g, q, k, v, out, lse, off)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for _ in range(3):
        q.mul_(0.9)
        want = run()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
