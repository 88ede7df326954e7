"""d(queries) of rows of up to 1024 keys, whose D is summed from the keys: the
definition in 64 bits and a bound that leaves no room for the rounding of `out`."""
import torch

from tests import sequence_ref as R

E = R.E


def problem(m, n, heads, kv, d, dtype, device, seed=0):
    """Rows that lean on one key: dS is far below dP and D there."""
    g = torch.Generator(device).manual_seed(seed + 100 * n + d)
    rand = lambda a, h: torch.randn(a, h, d, generator=g, device=device)  # noqa: E731
    k, v, d_out = rand(n, kv), rand(n, kv), rand(m, heads)
    near = torch.arange(m, device=device) * 7 % n
    q = 4 * (16 / d) * k[near].repeat_interleave(heads // kv, 1) * d ** -0.5 * 4 ** 0.5 + 0.1 * rand(m, heads)
    return [t.to(dtype) for t in (q, k, v, d_out)]


def d_q(q, k, v, d_out, scale, rounded_out=False):
    """-> (d_q [m, heads, d], tolerance).  Errors: of a score's products and of lse as in
    sequence_ref.attention; P and dP in f32, D a sum of n of their products; dS
    rounded to the type once.  rounded_out: D from `out` rounded to the type instead."""
    dt, U = q.dtype, R.half_step(q.dtype)
    m, heads, d = q.shape
    n, kv = k.shape[0], k.shape[1]
    q, k, v, g = (t.double().transpose(0, 1) for t in (q, k, v, d_out))
    k, v = (t.repeat_interleave(heads // kv, 0) for t in (k, v))
    s = q @ k.transpose(1, 2) * scale
    lse = torch.logsumexp(s, -1, keepdim=True)
    p = torch.exp(s - lse)
    dp = g @ v.transpose(1, 2)
    delta = (p * dp).sum(-1, keepdim=True)
    if rounded_out:
        delta = (g * (p @ v).to(dt).double()).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    top = (q.abs() @ k.abs().transpose(1, 2) * scale).amax(-1, keepdim=True)
    es = (d + 8) * E * top + 4 * E
    e_p = 2 * es + es + (n + 16) * E + 4 * E * lse.abs()
    e_dp = d * E * (g.abs() @ v.abs().transpose(1, 2))
    e_delta = (p * (dp.abs() * e_p + e_dp)).sum(-1, keepdim=True) + n * E * (p * dp.abs()).sum(-1, keepdim=True)
    # a scale a row: binary16's smallest step beside dS, from the row's own norm
    flat = 2.0 ** -36 * g.norm(dim=-1, keepdim=True) * v.norm(dim=-1).amax() if dt == torch.float16 else 0.0
    e_ds = ds.abs() * (U + e_p) + p * (e_delta + e_dp + 4 * E * (dp.abs() + delta.abs())) + flat
    value = scale * ds @ k
    tol = R.rounding(value, dt) + scale * e_ds @ k.abs() + (n + 8) * E * scale * ds.abs() @ k.abs()
    return value.transpose(0, 1), tol.transpose(0, 1)
