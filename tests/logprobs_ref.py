"""The log-probability operator in 64 bits from its definition, row by row of
what counts, and how far 32-bit sums may be from it."""
import math

import torch

D = torch.float64
HALF = 2.0 ** -24  # half a step of f32, relative


def reference(x, targets=None, top=0):
    """logp, entropy, top_logp, top_index, p, log p of rows x [R, V] (any type)."""
    x = x.double()
    r, v = x.shape
    t = torch.zeros(r, dtype=torch.long, device=x.device) if targets is None else targets.long()
    left_out = t < 0
    empty = (x == -math.inf).all(1)
    bad = (torch.isnan(x) | (x == math.inf)).any(1) & ~left_out
    live = ~(left_out | empty | bad)
    z = torch.where(live[:, None], x, 0.0)
    z = z - z.amax(1, keepdim=True)  # first: log s is lost beside 1e38
    lp = z - torch.log(torch.exp(z).sum(1, keepdim=True))
    p = torch.exp(lp)
    h = -torch.where(p > 0, p * lp, 0.0).sum(1)
    out = t >= v
    logp = lp.gather(1, t.clamp(0, v - 1)[:, None])[:, 0]
    logp[empty] = -math.inf
    logp[bad | out] = math.nan
    logp[left_out] = 0.0
    h[empty | left_out] = 0.0
    h[bad] = math.nan
    index = torch.where(live[:, None], x, 0.0).sort(dim=1, descending=True, stable=True)[1][:, :top]
    values = lp.gather(1, index)
    values[empty], values[bad], values[left_out] = -math.inf, math.nan, 0.0
    index[bad | left_out] = -1
    return logp, h, values, index, p, lp, live


def gradient(x, targets, ref, g=None, e=None, h=None):
    """d_logits from the definition, and the sum of the magnitudes of its terms."""
    logp, ent, _, index, p, lp, live = ref
    r, v = x.shape
    zero = torch.zeros(r, dtype=D, device=x.device)
    g = zero if g is None else g.double()
    e = zero if e is None else e.double()
    own = torch.zeros_like(p)
    total, size = g.clone(), g.abs()
    if targets is not None:
        own.scatter_add_(1, targets.long().clamp(0, v - 1)[:, None], g[:, None])
    if h is not None:
        own.scatter_add_(1, index.clamp_min(0), h.double())
        total = total + h.double().sum(1)
        size = size + h.double().abs().sum(1)
    slope = torch.where(p > 0, lp + ent[:, None], 0.0)
    d = own - p * total[:, None] - p * slope * e[:, None]
    terms = own.abs() + p * (size[:, None] + slope.abs() * e.abs()[:, None])
    keep = live if targets is None else live & (targets < v)
    d[~keep] = 0.0
    bad = torch.isnan(ent)
    if targets is not None:
        bad = bad | (targets >= v)
    d[bad] = math.nan
    return d, terms


def chain(v):
    """Additions that one of the sums' addends can pass through: a lane's own
    elements (at least 4 lanes, then 256), and the joining of lanes, waves and
    parts."""
    return (v / 4 if v <= 64 else v / 16 if v <= 256 else v / 64 if v <= 1024 else v / 256 + 32) + 16


def tolerances(x, ref):
    """(of a log-probability [R, V], of an entropy [R]): x - m and log s are
    rounded once each; every addend of s has the product d log2(e) rounded (at
    most |d| e^d <= 1/e of a half step), exp2 (one step) and its additions."""
    lp, h, live = ref[5], ref[1], ref[6]
    v = x.shape[1]
    m = torch.where(live[:, None], x.double(), 0.0).amax(1, keepdim=True)
    spread = torch.where(torch.isfinite(lp), (m - torch.where(live[:, None], x.double(), 0.0)).abs(), 0.0)
    s = HALF * (chain(v) + 6)
    of_logp = s + 2 * HALF * (spread + lp.abs().nan_to_num(posinf=0.0) + math.log(v) + 1)
    # u / s has the relative error of u and s, and log s the absolute one of s
    of_entropy = (s + 6 * HALF) * (2 + 2 * math.log(v) + h.nan_to_num().abs())
    return of_logp, of_entropy


def gradient_tolerance(x, d, terms, ref, e):
    """Each term has p's relative error (that of log p, and exp2's two half
    steps and its product's) and four roundings; then the rounding to the
    type (and to its smallest steps)."""
    of_logp, of_entropy = tolerances(x, ref)
    f = torch.finfo(x.dtype)
    lp = ref[5].abs().nan_to_num(posinf=0.0)
    rel = of_logp + HALF * (2 * lp + 12)
    tol = terms * rel + f.eps / 2 * (d.abs() + terms * rel) + f.smallest_normal * f.eps
    if e is not None:
        tol = tol + ref[4] * e.double().abs()[:, None] * (of_logp + of_entropy[:, None])
    return tol


def check(name, got, want, tol):
    """Not further than tol, elementwise; infinities and NaN in the same places."""
    got = got.double()
    nan = torch.isnan(want)
    inf = torch.isinf(want)
    assert torch.equal(torch.isnan(got), nan), name
    assert torch.equal(got[inf], want[inf]), name
    fine = ~(nan | inf)
    over = ((got - want).abs() - tol)[fine]
    assert over.numel() == 0 or over.max().item() <= 0, (
        f"{name}: {over.max().item():.3e} over its tolerance")
