"""What a sequence model beside the trunk does from its projections to its
next token, as timed cases: the norm and rotation of queries and keys, the
attention of packed sequences with its gradient and over a cache, and the
choice of a class from logits.

  norm            root-mean-square norm of every head of queries and keys,
                  and their rotation by position in the same pass
  norm_grad       its gradient: queries, keys and both weights
  attention       attention of sequences packed one after another, grouped
                  heads, causal or whole
  attention_grad  the same with d(queries), d(keys) and d(values): a training
                  step's forward and backward
  tokens          one query a sequence against its keys in a cache of a fixed
                  capacity, of which the sequence's length counts
  sample          a class a row from given uniform numbers, with temperature,
                  top-k, top-p and min-p

Queries, keys and values are slices of one projection [tokens, heads, width].
A causal query i of a sequence of m queries and n keys sees keys 0 .. i + n - m.
Classes are ranked by logit, ties to the lowest index; top-k keeps the first k
of them, top-p those whose forerunners hold less than top_p of what top-k
kept, min-p those of at least min_p times the largest probability; the class is
the first, by index, at which the kept ones' running sum exceeds u times their
sum.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6
BASE = 10000.0


# ------------------------------------------------------------------- the cases
def listed():
    return [
        # the next tokens of four running sequences, far along: launch and latency count
        {"name": "norm_tokens", "kind": "norm", "tokens": 4, "heads": 32, "kv_heads": 8, "width": 128,
         "rotated": 128, "type": "bf16", "far": 130_000, "interleaved": False},
        # a batch of prompts through one layer
        {"name": "norm_prompt", "kind": "norm", "tokens": 16384, "heads": 32, "kv_heads": 8, "width": 128,
         "rotated": 128, "type": "bf16", "far": 0, "interleaved": False},
        # a training batch with half of each head rotated in pairs
        {"name": "norm_grad", "kind": "norm_grad", "tokens": 8191, "heads": 16, "kv_heads": 4, "width": 64,
         "rotated": 32, "type": "f32", "far": 0, "interleaved": True},
        # chains of a few complexes, whole attention at the width of the trunk's MSA rows
        {"name": "attention_chains", "kind": "attention", "sequences": 8, "tokens": 896, "heads": 8,
         "kv_heads": 8, "width": 32, "causal": False, "type": "f16", "mix": 3, "prefix": 0},
        # prompts of very different lengths, packed
        {"name": "attention_prompt", "kind": "attention", "sequences": 11, "tokens": 16384, "heads": 32,
         "kv_heads": 8, "width": 128, "causal": True, "type": "bf16", "mix": 1, "prefix": 0},
        # the trunk's headline length, four states: forward and backward, launches count
        {"name": "attention_grad_states", "kind": "attention_grad", "sequences": 4, "tokens": 4 * 224,
         "heads": 8, "kv_heads": 8, "width": 32, "causal": False, "type": "f16", "mix": -1, "prefix": 0},
        # a training batch of packed sequences
        {"name": "attention_grad_prompt", "kind": "attention_grad", "sequences": 6, "tokens": 10007,
         "heads": 32, "kv_heads": 8, "width": 128, "causal": True, "type": "bf16", "mix": 2, "prefix": 0},
        # a served batch: one token each against what its sequence has so far
        {"name": "tokens_batch", "kind": "tokens", "sequences": 64, "capacity": 8192, "heads": 32,
         "kv_heads": 8, "width": 128, "type": "bf16", "mix": 5},
        # one long sequence alone
        {"name": "tokens_long", "kind": "tokens", "sequences": 1, "capacity": 131072, "heads": 32,
         "kv_heads": 4, "width": 64, "type": "f16", "mix": -1},
        # acids for the designed positions of many short binders
        {"name": "sample_acids", "kind": "sample", "rows": 5000, "classes": 20, "type": "f32", "omitted": 0.05,
         "temperature": 0.3, "top_k": 0, "top_p": 1.0, "min_p": 0.02, "by_row": False},
        # the next token of a served batch over a large vocabulary
        {"name": "sample_tokens", "kind": "sample", "rows": 64, "classes": 131072, "type": "bf16",
         "omitted": 0.0, "temperature": 0.8, "top_k": 50, "top_p": 0.95, "min_p": 0.0, "by_row": False},
        # many rows of an odd width, every row with settings of its own
        {"name": "sample_rows", "kind": "sample", "rows": 1021, "classes": 50001, "type": "f32",
         "omitted": 0.01, "temperature": 1.0, "top_k": 200, "top_p": 0.9, "min_p": 0.01, "by_row": True},
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], spread over the logarithm."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(("norm", "norm_grad", "attention", "attention", "attention_grad", "attention_grad",
                       "tokens", "tokens", "sample", "sample"))
    if kind == "sample":
        classes = _spread(rng, 2, 200_000)
        return {"kind": kind, "rows": _spread(rng, 1, min(20_000, max(1, 50_000_000 // classes))),
                "classes": classes, "type": rng.choice(tuple(TYPES)),
                "omitted": round(rng.choice((0.0, rng.uniform(0.0, 0.3))), 3),
                "temperature": round(rng.uniform(0.2, 1.5), 3),
                "top_k": rng.choice((0, 1, _spread(rng, 1, classes))),
                "top_p": round(rng.choice((1.0, rng.uniform(0.2, 0.99))), 3),
                "min_p": round(rng.choice((0.0, rng.uniform(0.001, 0.2))), 4),
                "by_row": rng.random() < 0.5}
    kv_heads = rng.choice((1, 2, 3, 4, 8))
    heads = kv_heads * rng.choice((1, 1, 2, 3, 4, 6, 8))
    heads = min(heads, 32) // kv_heads * kv_heads
    if kind in ("norm", "norm_grad"):
        width = rng.choice((16, 32, 64, 80, 96, 128, 256))
        rotated = rng.choice((width, width, width // 2, width // 4))
        top = min(16384, 60_000_000 // ((heads + kv_heads) * width))
        return {"kind": kind, "tokens": _spread(rng, 1, top), "heads": heads, "kv_heads": kv_heads,
                "width": width, "rotated": rotated, "type": rng.choice(tuple(TYPES)),
                "far": rng.choice((0, 0, _spread(rng, 100, 1_000_000))), "interleaved": rng.random() < 0.5}
    width = rng.choice((16, 32, 48, 64, 64, 80, 96, 128, 128))
    case = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "width": width,
            "type": rng.choice(("f16", "bf16"))}
    if kind == "tokens":
        # keys of the whole cache: at most those of the largest listed one
        cells = min(64 * 8192, 500_000_000 // (kv_heads * width))
        capacity = _spread(rng, 16, min(131072, cells))
        return case | {"sequences": _spread(rng, 1, min(256, cells // capacity)), "capacity": capacity,
                       "mix": rng.randrange(1 << 20)}
    # pairs of positions times heads times width: at most a quarter of the largest listed one
    tokens = _spread(rng, 1, int(min(8192, math.sqrt(1.0e11 / (heads * width)))))
    return case | {"sequences": min(tokens, _spread(rng, 1, 40)), "tokens": tokens,
                   "causal": rng.random() < 0.7, "mix": rng.randrange(1 << 20),
                   "prefix": rng.choice((0, 0, 0, _spread(rng, 1, 500)))}


# ---------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator("cuda").manual_seed(1_000_003 * int(seed) + 29)


def _lengths(case):
    """(queries, keys) of each sequence: the case's alone, no seed's."""
    n = case["sequences"]
    g = torch.Generator().manual_seed(max(0, case["mix"]))
    if case["kind"] == "tokens":
        share = torch.rand(n, generator=g, dtype=torch.float64) if case["mix"] >= 0 else torch.ones(n)
        # from a few tokens to the whole capacity
        return [1] * n, [max(1, int(case["capacity"] ** v)) for v in (0.3 + 0.7 * share).tolist()]
    if case["mix"] < 0:
        q = [case["tokens"] // n] * n
    else:  # shares over a factor of 50, cut to whole tokens that add up to `tokens`
        share = torch.exp(3.9 * torch.rand(n, generator=g, dtype=torch.float64)).cumsum(0)
        ends = (share / share[-1] * case["tokens"]).round().int().tolist()
        q = [b - a for a, b in zip([0] + ends, ends)]
    return q, [v + case["prefix"] for v in q]


def _offsets(lengths):
    return torch.tensor([0] + lengths, device="cuda").cumsum(0).int()


def _projection(gen, tokens, heads, width, t, scale=1.0):
    return (torch.randn(tokens, heads, width, generator=gen, device="cuda") * scale).to(t)


def _in_norm(case, seed):
    gen, t = _generator(seed), TYPES[case["type"]]
    n, hq, hk, d = case["tokens"], case["heads"], case["kv_heads"], case["width"]
    # one projection's queries, keys and values; token scales spread over a factor of e^2
    qkv = torch.randn(n, hq + 2 * hk, d, generator=gen, device="cuda")
    qkv = (qkv * torch.exp(torch.randn(n, 1, 1, generator=gen, device="cuda"))).to(t)
    # sequences packed one after another: positions start again
    pos = torch.arange(n, device="cuda") % 4099
    if case["far"]:
        pos = torch.randint(case["far"], (n,), generator=gen, device="cuda")
    r = case["rotated"]
    freq = BASE ** (-torch.arange(0, r, 2, device="cuda", dtype=torch.float64) / r)
    s = {"case": case, "q": qkv[:, :hq], "k": qkv[:, hq:hq + hk], "pos": pos.int(), "freq": freq.float()}
    for name in ("q_weight", "k_weight"):
        s[name] = 1 + 0.2 * torch.randn(d, generator=gen, device="cuda")
    if case["kind"] == "norm_grad":
        s["d_q"] = _projection(gen, n, hq, d, t)
        s["d_k"] = _projection(gen, n, hk, d, t)
    return s


def _in_attention(case, seed):
    gen, t = _generator(seed), TYPES[case["type"]]
    lq, lk = _lengths(case)
    nq, nk, hq, hk, d = sum(lq), sum(lk), case["heads"], case["kv_heads"], case["width"]
    s = {"case": case, "lq": lq, "lk": lk, "q_offsets": _offsets(lq), "k_offsets": _offsets(lk)}
    if nq == nk:  # slices of one projection
        qkv = _projection(gen, nq, hq + 2 * hk, d, t, 1.2)
        s |= {"q": qkv[:, :hq], "k": qkv[:, hq:hq + hk], "v": qkv[:, hq + hk:]}
    else:
        kv = _projection(gen, nk, 2 * hk, d, t, 1.2)
        s |= {"q": _projection(gen, nq, hq, d, t, 1.2), "k": kv[:, :hk], "v": kv[:, hk:]}
    if case["kind"] == "attention_grad":
        s["d_out"] = _projection(gen, nq, hq, d, t)
    return s


def _in_tokens(case, seed):
    gen, t = _generator(seed), TYPES[case["type"]]
    n, cap, hq, hk, d = (case[x] for x in ("sequences", "capacity", "heads", "kv_heads", "width"))
    lq, lk = _lengths(case)
    cache = torch.randn(2, n * cap, hk, d, generator=gen, device="cuda", dtype=t)
    return {"case": case, "lq": lq, "lk": lk, "q": _projection(gen, n, hq, d, t, 1.5),
            "k": cache[0], "v": cache[1], "q_offsets": torch.arange(n + 1, device="cuda").int(),
            "k_offsets": cap * torch.arange(n + 1, device="cuda").int(),
            "k_lengths": torch.tensor(lk, device="cuda").int()}


def _in_sample(case, seed):
    gen, t = _generator(seed), TYPES[case["type"]]
    rows, classes = case["rows"], case["classes"]
    x = 2.5 * torch.randn(rows, classes, generator=gen, device="cuda")
    # what the model is sure of: one class a row stands out
    peak = torch.randint(classes, (rows, 1), generator=gen, device="cuda")
    x.scatter_add_(1, peak, 8 * torch.rand(rows, 1, generator=gen, device="cuda"))
    gone = int(case["omitted"] * classes)
    if gone:  # classes that are not allowed: -infinity, one of them the type's lowest value
        x[:, classes - gone:] = -math.inf
        x[:, classes - 1] = torch.finfo(t).min
    s = {"case": case, "logits": x.to(t), "uniforms": torch.rand(rows, generator=gen, device="cuda")}
    s |= {k: case[k] for k in ("temperature", "top_k", "top_p", "min_p")}
    if case["by_row"]:  # every row's own settings, around the case's
        vary = lambda: torch.rand(rows, generator=gen, device="cuda")  # noqa: E731
        s["temperature"] = case["temperature"] * (0.5 + vary())
        s["top_k"] = (case["top_k"] * (0.01 + 1.5 * vary())).ceil().int()
        s["top_p"] = 1 - (1 - case["top_p"]) * 2 * vary()
        s["min_p"] = case["min_p"] * 2 * vary()
    return s


IN = {"norm": _in_norm, "norm_grad": _in_norm, "attention": _in_attention,
      "attention_grad": _in_attention, "tokens": _in_tokens, "sample": _in_sample}


def prepare(case, seed):
    s = IN[case["kind"]](case, seed)
    if own:  # the modules, as a model keeps them
        from bindcraft2_amd import ops
        if case["kind"] in ("norm", "norm_grad"):
            s["op"] = ops.HeadNormRotate(s["freq"], eps=EPS, interleaved=case["interleaved"])
        elif case["kind"] != "sample":
            s["op"] = ops.PackedAttention(causal=case.get("causal", True))
    return s


# --------------------------------------------------- the operators in plain form
def _halves(x, case):
    """The two members of every rotated pair, and the rest."""
    r = case["rotated"]
    if case["interleaved"]:
        return x[..., 0:r:2], x[..., 1:r:2], x[..., r:]
    return x[..., :r // 2], x[..., r // 2:r], x[..., r:]


def _whole(a, b, rest, case):
    if case["interleaved"]:
        return torch.cat((torch.stack((a, b), -1).flatten(-2), rest), -1)
    return torch.cat((a, b, rest), -1)


def _angles(s):
    # far positions: the product and its cosine in 64 bits
    angle = s["pos"].double()[:, None, None] * s["freq"].double()
    return torch.cos(angle).float(), torch.sin(angle).float()


def _plain_norm(s):
    case, (c, si) = s["case"], _angles(s)
    out = {}
    for name in ("q", "k"):
        x = s[name].float()
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s[name + "_weight"]
        a, b, rest = _halves(y, case)
        out[name] = _whole(a * c - b * si, b * c + a * si, rest, case).to(s[name].dtype)
    return out


def _plain_norm_grad(s):
    case, (c, si) = s["case"], _angles(s)
    out = {}
    for name in ("q", "k"):
        x = s[name].float()
        a, b, rest = _halves(s["d_" + name].float(), case)
        g = _whole(a * c + b * si, b * c - a * si, rest, case)
        scale = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        n = x * scale
        gw = g * s[name + "_weight"]
        out["d_" + name] = (scale * (gw - n * (gw * n).mean(-1, keepdim=True))).to(s[name].dtype)
        # a long sum
        out["d_" + name + "_weight"] = (g * n).sum((0, 1), dtype=torch.float64).float()
    return out


def _plain_sequence(s, b, at_q, at_k):
    """One sequence's outputs: out, lse and, with a cotangent, its gradients."""
    case = s["case"]
    m, n, hk = s["lq"][b], s["lk"][b], case["kv_heads"]
    heads = lambda x, at, l: (x[at:at + l].float().view(l, hk, -1, case["width"])  # noqa: E731
                              .permute(1, 2, 0, 3))
    q, k, v = heads(s["q"], at_q, m), heads(s["k"], at_k, n), heads(s["v"], at_k, n)
    scale = case["width"] ** -0.5
    x = torch.matmul(q, k.transpose(2, 3)) * scale
    if case["causal"]:
        seen = torch.ones(m, n, dtype=torch.bool, device="cuda").tril(n - m)
        x = torch.where(seen, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - top)
    z = p.sum(-1, keepdim=True)
    p = p / z
    o = torch.matmul(p, v)
    rows = lambda t: t.permute(2, 0, 1, 3).reshape(t.shape[2], -1, case["width"]).to(s["q"].dtype)  # noqa: E731
    out = {"out": rows(o), "lse": (top + torch.log(z)).flatten(0, 1)[..., 0]}
    if case["kind"] == "attention_grad":
        g = heads(s["d_out"], at_q, m)
        d = p * (torch.matmul(g, v.transpose(2, 3)) - (g * o).sum(-1, keepdim=True)) * scale
        shared = lambda t: rows(t.sum(1, keepdim=True))  # noqa: E731
        out |= {"d_q": rows(torch.matmul(d, k)), "d_k": shared(torch.matmul(d.transpose(2, 3), q)),
                "d_v": shared(torch.matmul(p.transpose(2, 3), g))}
    return out


def _plain_attention(s):
    starts = lambda lengths: [sum(lengths[:i]) for i in range(len(lengths))]  # noqa: E731
    at_q, at_k = starts(s["lq"]), starts(s["lk"])
    parts = [_plain_sequence(s, b, at_q[b], at_k[b]) for b in range(len(s["lk"])) if s["lk"][b]]
    return {key: torch.cat([p[key] for p in parts], 1 if key == "lse" else 0) for key in parts[0]}


def _plain_tokens(s):
    case = s["case"]
    n, cap, hk, d = (case[x] for x in ("sequences", "capacity", "kv_heads", "width"))
    q = s["q"].float().view(n, hk, -1, d)
    k, v = (s[x].float().view(n, cap, hk, d).transpose(1, 2) for x in ("k", "v"))
    x = torch.matmul(q, k.transpose(2, 3)) * d ** -0.5
    seen = torch.arange(cap, device="cuda") < s["k_lengths"][:, None]
    x = torch.where(seen[:, None, None], x, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - top)
    z = p.sum(-1, keepdim=True)
    out = torch.matmul(p / z, v).reshape(n, -1, d)
    return {"out": out.to(s["q"].dtype), "lse": (top + torch.log(z)).view(n, -1).t().contiguous()}


def _column(v):
    """A setting as a column of 64-bit numbers, or a number."""
    return v.double()[:, None] if torch.is_tensor(v) else v


def _plain_sample(s):
    # sums next to a border decide the class: 64 bits
    x = s["logits"].double()
    classes = x.shape[1]
    e = torch.exp((x - x.amax(1, keepdim=True)) / _column(s["temperature"]))
    order = s["logits"].sort(dim=1, descending=True, stable=True)[1]
    ranked = e.gather(1, order)
    rank = torch.arange(classes, device="cuda")
    k = _column(s["top_k"])
    if not torch.is_tensor(k):
        k = torch.full((1, 1), k, device="cuda", dtype=torch.float64)
    ranked = torch.where((rank < k) | (k < 1), ranked, 0.0)
    before = ranked.cumsum(1) - ranked
    p = _column(s["top_p"])
    kept = before < p * ranked.sum(1, keepdim=True)
    if not torch.is_tensor(p) and p >= 1:
        kept = torch.ones_like(kept)
    kept &= (ranked > 0) & (ranked >= _column(s["min_p"]))
    kept[:, 0] = True
    mass = torch.zeros_like(e).scatter_(1, order, torch.where(kept, ranked, 0.0))
    run = mass.cumsum(1)
    total = run[:, -1:]
    index = torch.searchsorted(run, s["uniforms"].double()[:, None] * total, right=True)
    logp = torch.log(mass.gather(1, index.clamp_max(classes - 1)) / total)
    return {"index": index[:, 0].int(), "logp": logp[:, 0].float()}


PLAIN = {"norm": _plain_norm, "norm_grad": _plain_norm_grad, "attention": _plain_attention,
         "attention_grad": _plain_attention, "tokens": _plain_tokens, "sample": _plain_sample}


# --------------------------------------------------------- the framework's calls
def _own(s):
    kind = s["case"]["kind"]
    if kind == "norm":
        q, k = s["op"].forward(s["q"], s["k"], s["pos"], s["q_weight"], s["k_weight"])
        return {"q": q, "k": k}
    if kind == "norm_grad":
        d_q, d_k, d_qw, d_kw = s["op"].backward((s["d_q"], s["d_k"]), s["q"], s["k"], s["pos"],
                                                s["q_weight"], s["k_weight"])
        return {"d_q": d_q, "d_k": d_k, "d_q_weight": d_qw, "d_k_weight": d_kw}
    if kind == "sample":
        from bindcraft2_amd import ops
        op = ops.Sampler(s["temperature"], s["top_k"], s["top_p"], s["min_p"])
        index, logp = op.sample(s["logits"], s["uniforms"])
        return {"index": index, "logp": logp}
    where = (s["q_offsets"], s["k_offsets"], s.get("k_lengths"))
    out, lse = s["op"].forward(s["q"], s["k"], s["v"], *where)
    r = {"out": out, "lse": lse}
    if kind == "attention_grad":
        r["d_q"], r["d_k"], r["d_v"] = s["op"].backward(s["d_out"], s["q"], s["k"], s["v"], out, lse, *where)
    return r


def run(state):
    return _own(state) if own else PLAIN[state["case"]["kind"]](state)


# ------------------------------------------------------------------------- work
def work(case):
    width = TYPES[case["type"]].itemsize
    if case["kind"] == "sample":
        return {"bytes": case["rows"] * (case["classes"] * width + 12), "flops": 4 * case["rows"] * case["classes"]}
    heads, d = case["heads"] + case["kv_heads"], case["width"]
    if case["kind"] in ("norm", "norm_grad"):
        n = case["tokens"] * heads * d
        grad = case["kind"] == "norm_grad"
        return {"bytes": n * width * (3 if grad else 2), "flops": n * (12 if grad else 7)}
    lq, lk = _lengths(case)
    live = [(m, n) for m, n in zip(lq, lk) if m]
    pairs = sum(m * n - (m * (m - 1) // 2 if case.get("causal", True) else 0) for m, n in live)
    grad = case["kind"] == "attention_grad"
    q, kv = sum(lq) * case["heads"] * d * width, sum(lk) * case["kv_heads"] * d * width
    # the gradient reads all but lse again with d(out) for `out`'s place, and writes d(q), d(k), d(v)
    return {"bytes": (2 * q + 2 * kv) + (4 * q + 4 * kv if grad else 0) + 4 * sum(lq) * case["heads"],
            "flops": (14 if grad else 4) * pairs * case["heads"] * d}


# ----------------------------------------------------- the definitions in 64 bits
def _exact_norm(case, seed):
    s = _in_norm(case, seed)
    r = case["rotated"]
    turn = torch.polar(torch.ones((), device="cuda", dtype=torch.float64),
                       s["pos"].double()[:, None] * s["freq"].double())[:, None]
    out = {}
    for name in ("q", "k"):
        x = s[name].double().requires_grad_()
        w = s[name + "_weight"].double().requires_grad_()
        y = w * x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS)
        if case["interleaved"]:
            pairs = y[..., :r].unflatten(-1, (r // 2, 2))
        else:
            pairs = y[..., :r].unflatten(-1, (2, r // 2)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        z = (z if case["interleaved"] else z.transpose(-1, -2)).flatten(-2)
        y = torch.cat((z, y[..., r:]), -1)
        if case["kind"] == "norm":
            out[name] = y.detach()
        else:
            out["d_" + name], out["d_" + name + "_weight"] = torch.autograd.grad(
                y, (x, w), s["d_" + name].double())
    return out


def _exact_attention(case, seed):
    s = (_in_tokens if case["kind"] == "tokens" else _in_attention)(case, seed)
    grad, d = case["kind"] == "attention_grad", case["width"]
    hq, hk = case["heads"], case["kv_heads"]
    nq, nk = s["q"].shape[0], s["k"].shape[0]
    wide = lambda *shape: torch.zeros(*shape, dtype=torch.float64, device="cuda")  # noqa: E731
    out = {"out": wide(nq, hq, d), "lse": wide(hq, nq)}
    if grad:
        out |= {"d_q": wide(nq, hq, d), "d_k": wide(nk, hk, d), "d_v": wide(nk, hk, d)}
    qs, ks = s["q_offsets"].tolist(), s["k_offsets"].tolist()
    for b, (m, n) in enumerate(zip(s["lq"], s["lk"])):
        here, there = slice(qs[b], qs[b] + m), slice(ks[b], ks[b] + n)
        later = torch.arange(n, device="cuda") > torch.arange(m, device="cuda")[:, None] + (n - m)
        for h in range(hq):  # one head at a time
            j = h * hk // hq
            q, k, v = (t.double().contiguous().requires_grad_(grad) for t in
                       (s["q"][here, h], s["k"][there, j], s["v"][there, j]))
            x = q @ k.t() / math.sqrt(d)
            if case.get("causal", True):
                x = x.masked_fill(later, -math.inf)
            o = torch.softmax(x, -1) @ v
            out["out"][here, h] = o.detach()
            out["lse"][h, here] = torch.logsumexp(x.detach(), -1)
            if grad and m:
                dq, dk, dv = torch.autograd.grad(o, (q, k, v), s["d_out"][here, h].double())
                out["d_q"][here, h] = dq
                out["d_k"][there, j] += dk
                out["d_v"][there, j] += dv
    return out


def _exact_sample(case, seed):
    s = _in_sample(case, seed)
    rows, classes = case["rows"], case["classes"]
    value = lambda v: v.double() if torch.is_tensor(v) else torch.full((rows,), float(v), device="cuda").double()  # noqa: E731
    # settings are numbers of 32 bits where they lie in tensors, and the case's own elsewhere
    t, p, floor = (value(s[x])[:, None] if torch.is_tensor(s[x]) else torch.full(
        (rows, 1), s[x], dtype=torch.float64, device="cuda") for x in ("temperature", "top_p", "min_p"))
    k = value(s["top_k"])[:, None]
    z = s["logits"].double() / t
    ranked, order = torch.sort(z, dim=1, descending=True, stable=True)
    first = torch.arange(classes, device="cuda").expand(rows, classes)
    ranked = torch.where((k >= 1) & (first >= k), -math.inf, ranked)
    share = torch.softmax(ranked, 1)
    head = share.cumsum(1) - share < p
    keep = (head | (p >= 1)) & (share > 0) & (share >= floor * share[:, :1])
    keep[:, 0] = True
    final = torch.softmax(torch.where(keep, ranked, -math.inf), 1)
    by_class = torch.zeros_like(final).scatter_(1, order, final)
    run = by_class.cumsum(1)
    u = s["uniforms"].double()[:, None] * run[:, -1:]
    index = (run <= u).sum(1)
    return {"index": None, "logp": torch.log(by_class.gather(1, index[:, None]))[:, 0]}


def exact(case, seed):
    kind = case["kind"]
    if kind == "sample":
        return _exact_sample(case, seed)
    return _exact_norm(case, seed) if kind in ("norm", "norm_grad") else _exact_attention(case, seed)
