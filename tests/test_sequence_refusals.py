"""The refusals of the sequence operators' entry points, which are made on the
host before any GPU call."""
import math

import pytest
import torch

import bindcraft2_amd as b
from bindcraft2_amd import ops

F32, F16, BF16 = 0, 1, 2
P = 1 << 20  # addresses that no refused call reads
STEP = 1 << 20


def refused(status, text):
    assert status != 0 and text in b.lib().bc2n_last_error(), (status, b.lib().bc2n_last_error())


def heads(i, st, sh):
    """The i-th operand: address, token stride, head stride."""
    return [None if i is None else P + i * STEP, st, sh]


NORM = dict(dtype=BF16, tokens=8, heads=4, kv_heads=2, width=64, rotated=64, interleaved=0, q=heads(0, 256, 64),
            k=heads(1, 128, 64), pos=P, bits=32, freq=P, qw=P, kw=P, wtype=F32, eps=1e-6, qo=heads(2, 256, 64),
            ko=heads(3, 128, 64), dq=heads(4, 256, 64), dk=heads(5, 128, 64), dqw=P, dkw=P, work=P)


def norm(**change):
    o = {**NORM, **change}
    return b.lib().bc2n_headnorm_fwd(None, *(o[k] for k in ("dtype", "tokens", "heads", "kv_heads", "width", "rotated",
                                                            "interleaved")), *o["q"], *o["k"], o["pos"], o["bits"],
                                     o["freq"], o["qw"], o["kw"], o["wtype"], o["eps"], *o["qo"], *o["ko"])


def norm_bwd(**change):
    o = {**NORM, **change}
    return b.lib().bc2n_headnorm_bwd(None, *(o[k] for k in ("dtype", "tokens", "heads", "kv_heads", "width", "rotated",
                                                            "interleaved")), *o["dq"], *o["dk"], *o["q"], *o["k"],
                                     o["pos"], o["bits"], o["freq"], o["qw"], o["kw"], o["wtype"], o["eps"], *o["qo"],
                                     *o["ko"], o["dqw"], o["dkw"], o["work"])


@pytest.mark.parametrize("call", [norm, norm_bwd])
def test_headnorm_refusals(call):
    refused(call(dtype=3), b"dtype")
    refused(call(wtype=F16), b"weights")
    refused(call(tokens=-1), b"tokens")
    refused(call(tokens=1 << 26), b"tokens")
    refused(call(heads=-1), b"heads")
    refused(call(heads=0, kv_heads=0), b"heads")
    refused(call(heads=1 << 17), b"heads")
    for width in (0, 3, -2):
        refused(call(width=width, rotated=0), b"width")
    for rotated in (-2, 3, 66):
        refused(call(rotated=rotated), b"rotated")
    refused(call(width=1026, rotated=1026), b"no layout")
    refused(call(width=1008, rotated=504), b"no layout")  # vectors of 4 at most, 252 of them
    refused(call(pos=None), b"null positions")
    refused(call(freq=None), b"null positions")
    refused(call(bits=16), b"i32 or i64")
    refused(call(qw=None), b"null q_weight")
    refused(call(kw=None), b"null k_weight")
    for eps in (-1e-6, math.inf, math.nan):
        refused(call(eps=eps), b"eps")
    refused(call(pos=P + 4, bits=64), b"unaligned")
    refused(call(qw=P + 2), b"unaligned")
    refused(call(q=heads(None, 256, 64)), b"q: null")
    refused(call(ko=heads(None, 128, 64)), b"null operand")
    refused(call(q=[P + 1, 256, 64]), b"unaligned")
    refused(call(q=heads(0, -256, 64)), b"negative stride")
    refused(call(q=heads(0, 256, -64)), b"negative stride")
    refused(call(q=heads(0, 1 << 40, 64)), b"stride too large")
    refused(call(tokens=1 << 25, q=heads(0, 1 << 39, 64)), b"stride too large")  # beyond every address
    refused(call(qo=heads(2, 255, 64)), b"elements overlap")
    refused(call(qo=heads(2, 256, 63)), b"elements overlap")
    refused(call(qo=heads(2, 256, 0)), b"elements overlap")


def test_headnorm_places():
    """A result may lie in its own operand, and in nothing else."""
    refused(norm(qo=[P + 2, 256, 64]), b"q_out overlaps q")
    refused(norm(qo=heads(1, 256, 64)), b"q_out overlaps k")
    refused(norm(qo=heads(2, 256, 64), ko=heads(2, 128, 64)), b"overlaps")
    # of as many heads, k is still no place for what comes of q
    alike = dict(kv_heads=4, k=heads(1, 256, 64), ko=heads(3, 256, 64), dk=heads(5, 256, 64))
    refused(norm(**{**alike, "qo": heads(1, 256, 64)}), b"q_out overlaps k")
    refused(norm(**{**alike, "qo": heads(1, 256, 64), "ko": heads(0, 256, 64)}), b"overlaps")
    refused(norm_bwd(**{**alike, "qo": heads(5, 256, 64)}), b"q_grad overlaps d_k")
    refused(norm_bwd(**{**alike, "ko": heads(0, 256, 64)}), b"k_grad overlaps q")
    # one token, whose stride says nothing
    refused(norm(tokens=1, q=heads(0, 0, 64), qo=[P + 128, 0, 64]), b"q_out overlaps q")
    refused(norm_bwd(work=None), b"null work")
    refused(norm_bwd(work=P + 8), b"unaligned")


ATTN = dict(dtype=BF16, causal=1, sequences=2, q_tokens=16, k_tokens=16, heads=4, kv_heads=2, width=64, scale=0.125,
            qof=P, kof=P, ql=None, kl=None, g=heads(0, 256, 64), q=heads(1, 256, 64), k=heads(2, 128, 64),
            v=heads(3, 128, 64), out=heads(4, 256, 64), lse=P, fill=0, dq=heads(5, 256, 64), dk=heads(6, 128, 64),
            dv=heads(7, 128, 64), work=P)
SIZES = ("dtype", "causal", "sequences", "q_tokens", "k_tokens", "heads", "kv_heads", "width", "scale", "qof", "kof",
         "ql", "kl")


def attn(**change):
    o = {**ATTN, **change}
    return b.lib().bc2n_attention_fwd(None, *(o[k] for k in SIZES), *o["q"], *o["k"], *o["v"], o["fill"], *o["out"],
                                      o["lse"], o["work"])


def attn_bwd(**change):
    o = {**ATTN, **change}
    return b.lib().bc2n_attention_bwd(None, *(o[k] for k in SIZES), *o["g"], *o["q"], *o["k"], *o["v"], *o["out"],
                                      o["lse"], o["fill"], *o["dq"], *o["dk"], *o["dv"], o["work"])


@pytest.mark.parametrize("call", [attn, attn_bwd])
def test_attention_refusals(call):
    refused(call(dtype=F32), b"f16 or bf16")
    refused(call(dtype=7), b"f16 or bf16")
    refused(call(sequences=-1), b"sequences")
    refused(call(sequences=(1 << 24) + 1), b"sequences")
    for h, kv in ((0, 1), (4, 0), (4, 3), (-4, 2), (65536, 2)):
        refused(call(heads=h, kv_heads=kv), b"heads")
    for width in (0, 4, 60, 136, -8):
        refused(call(width=width), b"width")
    refused(call(q_tokens=-1), b"tokens")
    refused(call(k_tokens=-1), b"tokens")
    refused(call(q_tokens=1 << 30), b"tokens")  # times two heads a group
    for scale in (0.0, -1.0, math.inf, math.nan):
        refused(call(scale=scale), b"scale")
    refused(call(qof=None), b"null offsets")
    refused(call(kof=None), b"null offsets")
    refused(call(qof=P + 2), b"unaligned")
    refused(call(kl=P + 2), b"unaligned")
    refused(call(q=heads(None, 256, 64)), b"q: null")
    refused(call(q=[P + 8, 256, 64]), b"unaligned")
    refused(call(q=heads(1, 260, 64)), b"keep the alignment")
    refused(call(k=heads(2, 128, 68)), b"keep the alignment")
    refused(call(k=heads(2, 32, 2048)), b"k: tokens overlap")
    refused(call(v=heads(3, 0, 64)), b"v: tokens overlap")
    refused(call(k=heads(2, 1 << 25, 64)), b"k: stride too large")
    refused(call(v=heads(3, 128, 1 << 30)), b"v: stride too large")
    refused(call(lse=None), b"null lse")
    refused(call(lse=P + 2), b"unaligned")
    refused(call(work=P + 8), b"unaligned")


def test_attention_places():
    refused(attn(out=heads(1, 256, 64)), b"out overlaps q")
    refused(attn(out=heads(2, 256, 64)), b"out overlaps k")
    refused(attn(out=heads(4, 128, 64)), b"out: elements overlap")
    refused(attn_bwd(dq=heads(1, 256, 64)), b"d_q overlaps q")
    refused(attn_bwd(dk=heads(7, 128, 64)), b"overlaps")
    refused(attn_bwd(dv=heads(0, 128, 64)), b"d_v overlaps d_out")
    refused(attn_bwd(dv=heads(4, 128, 64)), b"d_v overlaps out")
    refused(attn_bwd(dk=heads(6, 64, 64)), b"d_k: elements overlap")
    refused(attn_bwd(q=heads(1, 1 << 25, 64)), b"q: stride too large")
    refused(attn_bwd(g=heads(0, 256, 1 << 29)), b"d_out: stride too large")
    # one token, whose stride says nothing
    refused(attn(q_tokens=1, q=heads(1, 0, 64), out=[P + STEP + 128, 0, 64]), b"out overlaps q")


SAMPLE = dict(dtype=F32, x=P, ld=100, rows=4, v=100, u=P, t=1.0, ts=None, k=0, ks=None, p=1.0, ps=None, m=0.0, ms=None,
              index=P, logp=P)


def sample(**change):
    return b.lib().bc2n_sample(None, *{**SAMPLE, **change}.values())


def test_sample_refusals():
    refused(sample(dtype=3), b"dtype")
    refused(sample(rows=-1), b"rows")
    refused(sample(rows=1 << 31), b"rows")
    refused(sample(v=0, ld=0), b"classes")
    refused(sample(v=(1 << 28) + 1, ld=1 << 29), b"classes")
    refused(sample(ld=99), b"stride")
    refused(sample(x=None), b"null operand")
    refused(sample(u=None), b"null operand")
    refused(sample(index=None), b"null output")
    for t in (-0.5, math.inf, math.nan):
        refused(sample(t=t), b"temperature")
    refused(sample(k=-1), b"top_k")
    refused(sample(p=math.nan), b"top_p")
    refused(sample(m=math.nan), b"min_p")
    for name in ("x", "u", "ts", "ks", "ps", "ms", "index", "logp"):
        refused(sample(**{name: P + 2}), b"unaligned")


def test_sampler_settings():
    for kw in (dict(temperature=-1), dict(temperature=math.inf), dict(temperature=math.nan), dict(top_k=-1),
               dict(top_p=-0.1), dict(top_p=math.nan), dict(min_p=math.nan), dict(min_p=-1)):
        with pytest.raises(ValueError):
            ops.Sampler(**kw)
    with pytest.raises(ValueError, match="int32"):
        ops.Sampler(top_k=torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="float32"):
        ops.Sampler(top_p=torch.zeros(3, dtype=torch.float64))
    assert ops.Sampler(top_k=1 << 64).numbers[2] == 1 << 31  # all classes, in 64 bits too


def test_settings_of_the_others():
    for freq in (torch.ones(4, dtype=torch.float64), torch.ones(2, 2), torch.ones(8)[::2]):
        with pytest.raises(ValueError, match="freq"):
            ops.HeadNormRotate(freq)
    for eps in (-1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="eps"):
            ops.HeadNormRotate(torch.ones(4), eps)
    for scale in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="scale"):
            ops.PackedAttention(scale=scale)
