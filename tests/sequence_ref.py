"""Definitions in 64 bits of the sequence operators -- norm and rotation of
heads, attention of packed sequences, drawing a class -- and how far a kernel's
results may be off them, from the roundings that the operators state.

U is half a step of a type relative to a value; E = 2^-24 that of f32."""
import math

import torch

E = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rounding(value, dtype):
    """How far a value rounded to a type may be off: half a step, which below the
    smallest normal number is the same as at it (binary16: multiples of 2^-24)."""
    return half_step(dtype) * value.abs().clamp_min(torch.finfo(dtype).smallest_normal)


def check(what, got, want, tol):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    got = got.double()
    same = (got == want) | (got.isnan() & want.isnan())
    off = torch.where(same, 0.0, (got - want).abs() - tol)
    bad = ~(off <= 0)  # a NaN is bad
    if bad.any():
        i = torch.where(bad, torch.where(off.isnan(), math.inf, off), -math.inf).argmax().item()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, the worst at {i}: got "
                             f"{got.flatten()[i].item()!r}, want {want.flatten()[i].item()!r} +- "
                             f"{tol.expand(want.shape).flatten()[i].item():.3g}")


# --------------------------------------------------------------- norm and rotation
def pairs_of(x, r, interleaved):
    if interleaved:
        return x[..., 0:r:2], x[..., 1:r:2]
    return x[..., :r // 2], x[..., r // 2:r]


def joined(a, b, rest, interleaved):
    if interleaved:
        return torch.cat((torch.stack((a, b), -1).flatten(-2), rest), -1)
    return torch.cat((a, b, rest), -1)


def turn(x, angle, r, interleaved):
    a, b = pairs_of(x, r, interleaved)
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    return joined(a * c - b * s, b * c + a * s, x[..., r:], interleaved)


def partner_sum(x, r, interleaved):
    """|x| of an element and of the one that it turns into: bounds a rotated
    element and the error of one."""
    a, b = pairs_of(x.abs(), r, interleaved)
    return joined(a + b, a + b, x[..., r:].abs(), interleaved)


def far(angle):
    """An angle itself is good to 64 bits: the product (of 53 bits where the
    position has more than 29), the one with 1 / pi and that number's own
    rounding, and the product here, half a step of 2^-53 each."""
    return 4 * 2.0 ** -53 * angle.abs().amax(-1)[:, None, None] if angle.shape[-1] else 0.0


def head_norm(x, pos, freq, w, eps, interleaved):
    """-> (y, tolerance of an f32 result).  Factors' errors in E: a sum of squares
    of N <= 8 pairs a lane over 64 lanes at most 22 additions, so 11 of its
    root; the root 2, two products 2, the angle (2^-25 of half a turn) 2, its
    cosine 2, the rotation 3: 22, and 32 taken."""
    x, w, r = x.double(), w.double(), 2 * freq.shape[0]
    n = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w
    angle = pos.double()[:, None] * freq.double()
    return turn(n, angle, r, interleaved), (32 * E + far(angle)) * partner_sum(n, r, interleaved)


def head_norm_grad(d, x, pos, freq, w, eps, interleaved):
    """-> (dx, its tolerance, dw, its tolerance)."""
    d, x, w, r = d.double(), x.double(), w.double(), 2 * freq.shape[0]
    angle = pos.double()[:, None] * freq.double()
    g = turn(d, -angle, r, interleaved)
    scale = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    n = x * scale
    mean = (g * w * n).mean(-1, keepdim=True)
    dx = scale * (g * w - n * mean)
    # the turned cotangent 7 E, the norm 15 (once in scale, once in n), the mean's
    # own sum 22 more of its absolute terms
    turned = partner_sum(g, r, interleaved) * w.abs()
    terms = turned + n.abs() * (turned * n.abs()).mean(-1, keepdim=True)
    # a weight's sum has a term a token and head, added in some order
    dw_terms = (partner_sum(g, r, interleaved) * n.abs()).sum((0, 1))
    count = x.shape[0] * x.shape[1]
    return dx, (64 * E + far(angle)) * scale * terms, (g * n).sum((0, 1)), (count + 64) * E * dw_terms + (
        far(angle) * partner_sum(g, r, interleaved) * n.abs()).sum((0, 1))


# ------------------------------------------------------------------------ attention
def attention(q, k, v, causal, scale, d_out=None):
    """One sequence: q [m, heads, d], k and v [n, kv_heads, d] -> a dict of out, lse and
    the gradients, each with its tolerance for results of q's type."""
    U, dt = half_step(q.dtype), q.dtype
    m, heads, d = q.shape
    n, kv = k.shape[0], k.shape[1]
    G = heads // kv
    q, k, v = q.double(), k.double(), v.double()
    kk, vv = (t.repeat_interleave(G, 1).transpose(0, 1) for t in (k, v))  # [heads, n, d]
    qq = q.transpose(0, 1)
    s = qq @ kk.transpose(1, 2) * scale
    seen = torch.ones(m, n, dtype=torch.bool, device=q.device)
    if causal:
        seen = seen.tril(n - m)
    live = seen.any(1)
    s = torch.where(seen, s, -math.inf)
    lse = torch.logsumexp(s, -1) if n else torch.full((heads, m), -math.inf, device=q.device).double()
    p = torch.where(seen, torch.exp(s - torch.where(live, lse, 0.0)[..., None]), 0.0)
    o = p @ vv
    # a score's error, absolute: d products and sums in f32, the scaling and the
    # exponent's own rounding at its size in log 2
    size = torch.where(seen, qq.abs() @ kk.abs().transpose(1, 2) * scale, 0.0)
    top = size.amax(-1, keepdim=True) if n else size.sum(-1, keepdim=True)
    es = (d + 8) * E * top + 4 * E
    flat = 2.0 ** -31 if dt == torch.float16 else 0.0  # binary16's smallest step beside a shifted P
    pv = p @ vv.abs()
    rows = lambda t: t.transpose(0, 1)  # noqa: E731
    tol_o = rounding(o, dt) + pv * (U + 2 * es + n * E) + flat * vv.abs().sum(1, keepdim=True)
    r = {"out": (rows(o), rows(tol_o)),
         "lse": (lse, (es[..., 0] + (n + 16) * E + 4 * E * torch.where(live, lse, 0.0).abs()).clamp_min(0))}
    if d_out is None:
        return r
    g = d_out.double().transpose(0, 1)
    dp = g @ vv.transpose(1, 2)
    delta = (g * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    # D comes from the rounded out; dP and D are sums of d products
    e_delta = (g.abs() * tol_o).sum(-1, keepdim=True) + d * E * (g.abs() * o.abs()).sum(-1, keepdim=True)
    e_dp = d * E * (g.abs() @ vv.abs().transpose(1, 2))
    norms = g.norm(dim=-1).max() * vv.norm(dim=-1).max() if m and n else torch.tensor(0.0)
    flat_ds = 2.0 ** -36 * norms if dt == torch.float16 else 0.0
    e_lse = r["lse"][1][..., None]
    e_ds = ds.abs() * (U + 2 * es + e_lse) + p * (e_delta + e_dp + 4 * E * (dp.abs() + delta.abs()))
    e_ds = torch.where(seen, e_ds + flat_ds, 0.0)
    flat_p = 2.0 ** -39 if dt == torch.float16 else 0.0
    e_p = torch.where(seen, p * (U + 2 * es + e_lse) + flat_p, 0.0)
    shared = lambda t: t.view(kv, G, n, d).sum(1).transpose(0, 1)  # noqa: E731

    def one(value, tol, terms, count):
        return value, rounding(value, dt) + tol + count * E * terms
    r["d_q"] = one(rows(scale * ds @ kk), rows(scale * e_ds @ kk.abs()), rows(scale * ds.abs() @ kk.abs()), n + 8)
    t = lambda x: x.transpose(1, 2)  # noqa: E731
    r["d_k"] = one(shared(scale * t(ds) @ qq), shared(scale * t(e_ds) @ qq.abs()),
                   shared(scale * t(ds.abs()) @ qq.abs()), m * G + 8)
    r["d_v"] = one(shared(t(p) @ g), shared(t(e_p) @ g.abs()), shared(t(p) @ g.abs()), m * G + 8)
    return r


# --------------------------------------------------------------------------- drawing
def draw(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row, 64 bits -> (index, log-probability, the distance of u to the
    borders of its class in the distribution, of the cuts to theirs)."""
    x = x.double()
    v = x.shape[0]
    order = torch.sort(x, descending=True, stable=True)[1]
    if temperature == 0:
        return int(order[0]), 0.0, 1.0
    e = torch.exp((x[order] - x[order[0]]) / temperature)
    if 0 < top_k < v:
        e[top_k:] = 0
    near = 1.0
    if top_p < 1:
        before = e.cumsum(0) - e
        end = max(top_p, 0.0) * e.sum()
        keep = before < end
        keep[0] = True
        near = min(near, ((before[1:] - end).abs() / e.sum()).min().item() if v > 1 else 1.0)
        e = torch.where(keep, e, 0.0)
    e = torch.where(e >= min(min_p, 1.0), e, 0.0)
    mass = torch.zeros_like(e).scatter_(0, order, e)
    run = mass.cumsum(0) / mass.sum()
    at = min(max(u, 0.0), 1.0)
    index = int((run <= at).sum())
    if index >= v or mass[index] == 0:
        index = int(torch.nonzero(mass)[-1])
    near = min(near, (run - at).abs()[mass > 0][:-1].min().item() if (mass > 0).sum() > 1 else 1.0)
    return index, math.log(mass[index] / mass.sum()), near
