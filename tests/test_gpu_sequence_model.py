"""The sequence operators as a model runs them together.  Serving: prompts
through norm and rotation, attention against a cache and a drawn class, then
token by token from a captured graph.  Training: the same with the classes'
likelihood, its gradient back to the projection and both norms' weights, clipped
and taken by Adam.  Every stage is held to its definition in 64 bits on the
tensors that the run itself gives it."""
import pytest
import torch

from tests import sequence_ref as R
from bindcraft2_amd import ops

pytestmark = pytest.mark.gpu
H, KV, D, C, V, EPS = 6, 2, 32, 48, 1500, 1e-6


class Model:
    """One layer: x -> queries, keys and values as one projection -> classes."""

    def __init__(self, dtype):
        g = torch.Generator("cuda").manual_seed(11)
        rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        self.dtype, self.gen = dtype, g
        self.w_in, self.w_out = rnd(C, (H + 2 * KV) * D) / C ** 0.5, 2 * rnd(H * D, V) / (H * D) ** 0.5
        self.norms = [1 + 0.2 * rnd(D) for _ in range(2)]
        freq = (10000.0 ** (-torch.arange(0, D, 2, device="cuda").double() / D)).float()
        self.norm, self.attn = ops.HeadNormRotate(freq, EPS), ops.PackedAttention(causal=True)
        self.freq = freq

    def project(self, x):
        return (x @ self.w_in).to(self.dtype).view(x.shape[0], H + 2 * KV, D)

    @staticmethod
    def split(p):
        return p[:, :H], p[:, H:H + KV], p[:, H + KV:]

    def rnd(self, *s):
        return torch.randn(*s, generator=self.gen, device="cuda")

    def check_norm(self, raw, got, pos):
        for i, (x, y) in enumerate(zip(self.split(raw)[:2], got)):
            want, tol = R.head_norm(x, pos, self.freq, self.norms[i], EPS, False)
            R.check("qk"[i], y, want, tol + R.rounding(want, self.dtype))


def starts(lengths):
    return torch.tensor([0, *lengths], device="cuda").cumsum(0).int()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prompts_then_tokens(cuda, dtype):
    m, lengths, room = Model(dtype), [37, 1, 130], 160
    n = len(lengths)
    qo, ko = starts(lengths), starts([room] * n)
    have = torch.tensor(lengths, device="cuda", dtype=torch.int32)
    cache = [torch.full((n * room, KV, D), float("nan"), device="cuda", dtype=dtype) for _ in range(2)]
    sampler = ops.Sampler(0.8, top_k=200, top_p=0.95)

    def layer(x, pos, slots, q_off):
        """-> (raw projection, queries, logits); keys and values go to their slots"""
        p = m.project(x)
        raw = p.clone()
        q, k, v = m.split(p)
        m.norm.forward(q, k, pos, *m.norms, out=(q, k))  # in place
        cache[0][slots], cache[1][slots] = k, v
        out, _ = m.attn.forward(q, *cache, q_off, ko, have)
        return raw, q, k, out, out.flatten(1).float() @ m.w_out

    def check_layer(raw, q, k, out, pos, q_len):
        m.check_norm(raw, (q, k), pos)
        at = 0
        for b, c in enumerate(q_len):
            keys = slice(b * room, b * room + int(have[b]))
            want = R.attention(q[at:at + c], cache[0][keys], cache[1][keys], True, D ** -0.5)["out"]
            R.check(f"out of sequence {b}", out[at:at + c], *want)
            at += c

    def check_draw(logits, u, index, logp):
        unit = V * 2.0 ** -44  # masses are whole numbers of 2^-44 and less
        for r in range(n):
            at, lp, near = R.draw(logits[r].cpu(), u[r].item(), 0.8, 200, 0.95)
            if near >= unit:
                assert index[r].item() == at and abs(logp[r].item() - lp) <= R.E * abs(lp) + unit + 1e-12

    x = m.rnd(sum(lengths), C)
    pos = torch.cat([torch.arange(c, device="cuda") for c in lengths])
    slots = torch.cat([b * room + torch.arange(c, device="cuda") for b, c in enumerate(lengths)])
    raw, q, k, out, logits = layer(x, pos, slots, qo)
    check_layer(raw, q, k, out, pos, lengths)
    last = logits[(qo[1:] - 1).long()]
    u = torch.rand(n, generator=m.gen, device="cuda")
    index, logp = sampler.sample(last, u)
    check_draw(last, u, index, logp)

    # a token of each sequence at a time: written once, captured, replayed
    embed, base = m.rnd(V, C), torch.arange(n, device="cuda") * room
    token, ones = index.clone(), starts([1] * n)

    def step():
        at = have.long()
        have.add_(1)
        r = layer(embed[token.long()], at, base + at, ones)
        i, lp = sampler.sample(r[-1], u)
        token.copy_(i)
        return *r, at, i, lp

    def state():
        return [t.clone() for t in (*cache, have, token)]

    def restore(s):
        for t, v in zip((*cache, have, token), s):
            t.copy_(v)
    begin = state()
    step()
    restore(begin)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    restore(begin)
    for i in range(6):
        u.copy_(torch.rand(n, generator=m.gen, device="cuda"))
        before = state()
        want = [t.clone() for t in step()]
        after = state()
        restore(before)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), i
        assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip(state(), after)), i
        raw, q, k, out, logits, at, index, logp = held
        check_layer(raw, q, k, out, at, [1] * n)
        check_draw(logits, u, index, logp)
    assert have.tolist() == [c + 6 for c in lengths]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_training_step(cuda, dtype):
    m, lengths = Model(dtype), [65, 3, 0, 100]
    n, off = sum(lengths), starts(lengths)
    pos = torch.cat([torch.arange(c, device="cuda") for c in lengths])
    x, targets = m.rnd(n, C), torch.randint(V, (n,), generator=m.gen, device="cuda")
    weight = torch.full((n,), -1.0 / n, device="cuda")
    params = [m.w_in, m.w_out, *m.norms]
    grads = [torch.zeros_like(p) for p in params]
    avg, avg_sq = [torch.zeros_like(p) for p in params], [torch.zeros_like(p) for p in params]
    clip, adam = ops.GradientClip(grads), ops.Adam(params, grads, avg, avg_sq)

    def run():
        """Forward and backward; the gradients go to `grads`."""
        raw = m.project(x)
        q, k, v = m.split(raw)
        qn, kn = m.norm.forward(q, k, pos, *m.norms)
        out, lse = m.attn.forward(qn, kn, v, off)
        y = out.flatten(1).float()
        (logp, _), d_logits = ops.LogProbs().value_and_grad(y @ m.w_out, targets, weight)
        d_out = (d_logits @ m.w_out.t()).to(dtype).view(n, H, D)
        d_raw = torch.empty_like(raw)  # its slices take the three gradients
        dq, dk, dv = m.split(d_raw)
        m.attn.backward(d_out, qn, kn, v, out, lse, off, grads=(dq, dk, dv))
        cts = dq.clone(), dk.clone()
        d = m.norm.backward((dq, dk), q, k, pos, *m.norms, out=(dq, dk))  # in place
        grads[0].copy_(x.t() @ d_raw.flatten(1).float())
        grads[1].copy_(y.t() @ d_logits)
        grads[2].copy_(d[2])
        grads[3].copy_(d[3])
        return raw, qn, kn, out, lse, logp, d_out, d_raw, *cts
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for i in range(4):
        x.copy_(m.rnd(n, C))
        want = [t.clone() for t in (*run(), *grads)]
        for g in grads:
            g.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((*held, *grads), want)), i
        raw, qn, kn, out, lse, logp, d_out, d_raw, cq, ck = held
        q, k, v = m.split(raw)
        dq, dk, dv = m.split(d_raw)
        m.check_norm(raw, (qn, kn), pos)
        at = 0
        for b, c in enumerate(lengths):
            s = slice(at, at + c)
            want = R.attention(qn[s], kn[s], v[s], True, D ** -0.5, d_out[s])
            for name, got in {"out": out[s], "lse": lse[:, s], "d_q": cq[s], "d_k": ck[s], "d_v": dv[s]}.items():
                R.check(f"{name} of sequence {b}", got, *want[name])
            at += c
        for what, a, d, got, w, g in (("q", q, cq, dq, m.norms[0], grads[2]), ("k", k, ck, dk, m.norms[1], grads[3])):
            dx, tol, dw, tol_w = R.head_norm_grad(d, a, pos, m.freq, w, EPS, False)
            R.check("d_" + what, got, dx, tol + R.rounding(dx, dtype))
            R.check("d_weight of " + what, g, dw, tol_w)
        before = [p.clone() for p in params]
        total = torch.sqrt(sum(g.double().square().sum() for g in grads)).item()
        norm = clip.clip(1.0)
        assert abs(norm.item() - total) <= 1e-6 * total
        adam.step(i + 1, 1e-3)
        assert all(p.isfinite().all() and not torch.equal(p, q_) for p, q_ in zip(params, before))


def test_gradient_of_the_whole_by_differences(cuda):
    """d loss / d(norms' weights) of the run in binary16 against differences of the
    64-bit definition of the same run.  Each of q, k, P, dS, dq and dk is rounded
    once, at most 2^-11 of its size; a rotated q or k moves a score of at most
    |q| |k| / sqrt(32) < 16 by 2^-10 of it, so P by 2^-6 of itself in the worst of
    cases.  With signs at random over the 32 terms of a score and the
    thousands of a weight's sum that is below 2^-8; 2% is five times as much, and
    a wrong term, factor or sign is a multiple of it."""
    m, lengths = Model(torch.float16), [33, 20]
    n, off = sum(lengths), starts(lengths)
    pos = torch.cat([torch.arange(c, device="cuda") for c in lengths])
    raw = m.project(m.rnd(n, C))
    w = m.rnd(n, H, D).half()  # the loss: sum of w out
    q, k, v = m.split(raw)
    qn, kn = m.norm.forward(q, k, pos, *m.norms)
    out, lse = m.attn.forward(qn, kn, v, off)
    dq, dk, _ = m.attn.backward(w, qn, kn, v, out, lse, off)
    got = torch.cat(m.norm.backward((dq, dk), q, k, pos, *m.norms)[2:])

    def loss(a, b):
        x, _ = R.head_norm(q, pos, m.freq, a, EPS, False)
        y, _ = R.head_norm(k, pos, m.freq, b, EPS, False)
        at, total = 0, 0.0
        for c in lengths:
            s = slice(at, at + c)
            r = R.attention(x[s], y[s], v[s].double(), True, D ** -0.5)["out"][0]
            total += (r * w[s].double()).sum().item()
            at += c
        return total
    norms, h = [t.double() for t in m.norms], 1e-4
    want = torch.zeros(2 * D, dtype=torch.float64, device="cuda")
    for i in range(2 * D):
        e = torch.zeros(D, dtype=torch.float64, device="cuda")
        e[i % D] = h
        up, down = ((norms[0] + t, norms[1]) if i < D else (norms[0], norms[1] + t) for t in (e, -e))
        want[i] = (loss(*up) - loss(*down)) / (2 * h)
    assert (got.double() - want).norm() <= 0.02 * want.norm()
