"""What a design or training program does with the model's answers, as timed
cases: log-probabilities of given classes with their gradient, the global
norm of a list of gradients with its clipping, and the Adam update that takes
the clipped gradients.

  logprobs       log-probability of a target class, entropy and the top
                 alternatives of rows of logits
  logprobs_grad  the log-probabilities and entropies with d(logits) in one
                 call, the cotangents known beforehand (a weighted likelihood)
  logprobs_vjp   forward with alternatives, then the backward of all outputs
  clip           global 2-norm of many gradients, and the gradients scaled to
                 at most max_norm
  adam           an Adam step with decoupled weight decay on many parameters,
                 the gradients clipped by their global norm

Rows whose target is negative are left out: they hold padding (NaN here), and
their outputs are zero.  Lists of tensors are views of one buffer, each at a
256-byte boundary, with zeros between; the same buffer is what comes back.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ADAM = {"lr": 1e-2, "betas": (0.9, 0.999), "eps": 1e-8, "weight_decay": 0.01}

# elements of the tensors of one Evoformer block's parameters: the pair
# track's attentions, multiplications and transition at 128 channels, the MSA
# track's at 256, the outer product mean
_ATT = lambda c, h: [c, c] + [c * h] * (h > 0) + [c * c] * 5 + [c, c]  # noqa: E731
_MUL = [128, 128, 128 * 256, 256, 128 * 256, 256, 128, 128, 128 * 128, 128, 128 * 128, 128]
_TRANS = lambda c: [c, c, 4 * c * c, 4 * c, 4 * c * c, c]  # noqa: E731
BLOCK = (_ATT(128, 4) * 2 + _MUL * 2 + _TRANS(128) + _TRANS(256) + _ATT(256, 0) * 2 + [128, 128, 1024]
         + [256, 256, 256 * 32, 32, 256 * 32, 32, 32 * 32 * 128, 128])


# ------------------------------------------------------------------- the cases
def listed():
    return [
        # the acids of a short binder: launches and latency count
        {"name": "logprobs_sequence", "kind": "logprobs", "rows": 64, "classes": 20, "type": "f32",
         "top": 3, "ignored": 0.0, "omitted": 0.05},
        # distance bins of every residue pair at the headline length, padding left out
        {"name": "logprobs_distogram", "kind": "logprobs", "rows": 224 * 224, "classes": 64,
         "type": "f32", "top": 1, "ignored": 0.1, "omitted": 0.0},
        # single tokens of a few running sequences over a large vocabulary
        {"name": "logprobs_tokens", "kind": "logprobs", "rows": 4, "classes": 131072,
         "type": "bf16", "top": 8, "ignored": 0.0, "omitted": 0.0},
        # prompts scored: many rows of an odd width, so that no two rows are aligned alike
        {"name": "logprobs_prompt", "kind": "logprobs", "rows": 2047, "classes": 50001,
         "type": "f16", "top": 5, "ignored": 0.02, "omitted": 0.01},
        # the large complex's distance bins as a loss term with its gradient
        {"name": "grad_distogram", "kind": "logprobs_grad", "rows": 512 * 512, "classes": 64,
         "type": "f32", "ignored": 0.1, "omitted": 0.0, "entropy": True},
        # a training batch over a large vocabulary
        {"name": "grad_vocabulary", "kind": "logprobs_grad", "rows": 2048, "classes": 131072,
         "type": "bf16", "ignored": 0.1, "omitted": 0.0, "entropy": False},
        # a loss whose weights come from the values: forward, then backward
        {"name": "vjp_vocabulary", "kind": "logprobs_vjp", "rows": 1021, "classes": 33003,
         "type": "f32", "top": 4, "ignored": 0.0, "omitted": 0.01},
        # three states of a design: a gradient of designed logits each
        {"name": "clip_states", "kind": "clip", "type": "f32", "sizes": "states", "count": 3,
         "n": 224, "mix": 0},
        # every parameter's gradient of the main stack
        {"name": "clip_blocks", "kind": "clip", "type": "f32", "sizes": "blocks", "count": 48,
         "n": 0, "mix": 0},
        # a few large matrices and small ones of odd sizes
        {"name": "clip_mixed", "kind": "clip", "type": "bf16", "sizes": "mixed", "count": 37,
         "n": 300_000_007, "mix": 5},
        # the update of one state's designed logits
        {"name": "adam_states", "kind": "adam", "type": "f32", "sizes": "states", "count": 1,
         "n": 224, "mix": 0, "step": 1},
        # the update of the main stack's parameters
        {"name": "adam_blocks", "kind": "adam", "type": "f32", "sizes": "blocks", "count": 48,
         "n": 0, "mix": 0, "step": 1000},
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], spread over the logarithm."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(("logprobs", "logprobs", "logprobs_grad", "logprobs_vjp", "clip", "adam"))
    kind_of = rng.choice(tuple(TYPES))
    if kind in ("clip", "adam"):
        case = {"kind": kind, "type": kind_of, "sizes": rng.choice(("states", "blocks", "mixed")),
                "mix": rng.randrange(1 << 20)}
        if case["sizes"] == "states":
            case |= {"count": rng.randint(1, 8), "n": _spread(rng, 5, 768)}
        elif case["sizes"] == "blocks":
            case |= {"count": rng.randint(1, 47), "n": 0}
        else:
            top = 200_000_000 if kind == "clip" else 60_000_000
            case |= {"count": _spread(rng, 2, 300), "n": _spread(rng, 1000, top)}
        return case | ({"step": _spread(rng, 1, 100_000)} if kind == "adam" else {})
    classes = _spread(rng, 2, 200_000)
    rows = _spread(rng, 1, min(300_000, max(1, 200_000_000 // classes)))
    case = {"kind": kind, "rows": rows, "classes": classes, "type": kind_of,
            "ignored": round(rng.choice((0.0, rng.uniform(0.01, 0.3))), 3),
            "omitted": round(rng.choice((0.0, rng.uniform(0.0, 0.3))), 3)}
    if kind == "logprobs_grad":
        return case | {"entropy": rng.random() < 0.5}
    return case | {"top": min(classes, rng.choice((0, 1, 3, 5, 8, 20)))}


# ---------------------------------------------------------------------- inputs
def _sizes(case):
    """Elements of each tensor of the list: the case's alone, no seed's."""
    if case["sizes"] == "states":
        return [20 * case["n"]] * case["count"]
    if case["sizes"] == "blocks":
        return BLOCK * case["count"]
    # sizes over four decades that add up to n
    g = torch.Generator().manual_seed(case["mix"])
    share = torch.exp(9.2 * torch.rand(case["count"], generator=g, dtype=torch.float64))
    return [max(1, int(case["n"] * v)) for v in (share / share.sum()).tolist()]


def _places(sizes, width):
    """(start of each tensor in the buffer, length of the buffer), in elements."""
    step = 256 // width
    starts, at = [], 0
    for n in sizes:
        starts.append(at)
        at += -(-n // step) * step
    return starts, at


def _generator(seed):
    return torch.Generator("cuda").manual_seed(1_000_003 * int(seed) + 17)


def _views(buffer, sizes, starts):
    return [buffer[a:a + n] for a, n in zip(starts, sizes)]


def _in_lists(case, seed):
    gen, t = _generator(seed), TYPES[case["type"]]
    sizes = _sizes(case)
    starts, total = _places(sizes, t.itemsize)
    index = torch.arange(total, device="cuda", dtype=torch.int32)
    ends = torch.tensor([a + n for a, n in zip(starts, sizes)], device="cuda", dtype=torch.int32)
    begin = torch.tensor(starts, device="cuda", dtype=torch.int32)
    at = torch.searchsorted(begin, index, right=True) - 1
    real = index < ends[at]
    del index, at

    def buffer(scale, square=False):
        x = torch.randn(total, generator=gen, device="cuda") * scale
        return torch.where(real, x * x if square else x, 0.0)

    # gradients spread over several orders of magnitude
    grads = buffer(0.05) * torch.exp(1.5 * torch.randn(total, generator=gen, device="cuda"))
    s = {"case": case, "sizes": sizes, "starts": starts, "grads": grads.to(t)}
    if case["kind"] == "adam":
        s |= {"params": buffer(1.0).to(t), "avg": buffer(0.01), "avg_sq": buffer(0.05, True)}
        s |= {"out_params": torch.zeros_like(s["params"]), "out_avg": torch.zeros_like(s["avg"]),
              "out_avg_sq": torch.zeros_like(s["avg_sq"])}
    else:
        s["out"] = torch.zeros_like(s["grads"])
    return s


def _in_rows(case, seed):
    gen, t = _generator(seed), TYPES[case["type"]]
    rows, classes = case["rows"], case["classes"]
    x = torch.randn(rows, classes, generator=gen, device="cuda", dtype=t if t != torch.float16 else torch.float32)
    x.mul_(2.5)
    # what the model is sure of: one class a row stands out
    peak = torch.randint(classes, (rows, 1), generator=gen, device="cuda")
    x.scatter_add_(1, peak, 8 * torch.rand(rows, 1, generator=gen, device="cuda").to(x.dtype))
    gone = int(case["omitted"] * classes)
    if gone:  # classes that are not allowed: -infinity, one of them the type's lowest value
        x[:, classes - gone:] = -math.inf
        x[:, classes - 1] = torch.finfo(t).min
    targets = torch.randint(classes - gone, (rows,), generator=gen, device="cuda")
    if case["ignored"]:
        out = torch.rand(rows, generator=gen, device="cuda") < case["ignored"]
        targets = torch.where(out, -1, targets)
        x[out] = math.nan
    s = {"case": case, "logits": x.to(t), "targets": targets}
    if case["kind"] != "logprobs":
        cot = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
        s["d_logp"] = cot(rows)
        if case["kind"] == "logprobs_vjp" or case["entropy"]:
            s["d_entropy"] = cot(rows)
        if case["kind"] == "logprobs_vjp" and case["top"]:
            s["d_top"] = cot(rows, case["top"])
    return s


def prepare(case, seed):
    if case["kind"] in ("clip", "adam"):
        s = _in_lists(case, seed)
        if own:  # the list's handle, as an optimiser keeps one
            from bindcraft2_amd import ops
            lists = {k: _views(v, s["sizes"], s["starts"]) for k, v in s.items()
                     if torch.is_tensor(v)}
            if case["kind"] == "clip":
                s["handle"] = ops.GradientClip(lists["grads"], out=lists["out"])
            else:
                s["handle"] = ops.Adam(lists["params"], lists["grads"], lists["avg"], lists["avg_sq"],
                                       out=(lists["out_params"], lists["out_avg"], lists["out_avg_sq"]),
                                       betas=ADAM["betas"], eps=ADAM["eps"],
                                       weight_decay=ADAM["weight_decay"])
        return s
    return _in_rows(case, seed)


# --------------------------------------------------- the operators in plain form
def _softmax(s):
    """32-bit log-probabilities and probabilities, entropies, and which rows count."""
    x = s["logits"].float()
    keep = s["targets"] >= 0
    x = torch.where(keep[:, None], x, 0.0)
    x = x - x.amax(1, keepdim=True)
    e = torch.exp(x)
    z = e.sum(1, keepdim=True)
    logp = x - torch.log(z)
    p = e / z
    entropy = -torch.where(p > 0, p * logp, 0.0).sum(1)
    return logp, p, torch.where(keep, entropy, 0.0), keep


def _at_target(s, logp, keep):
    at = logp.gather(1, s["targets"].clamp_min(0)[:, None])[:, 0]
    return torch.where(keep, at, 0.0)


def _tops(s, logp, keep, top):
    """The largest logits of each row, ties to the lowest index: a stable sort."""
    order = torch.where(keep[:, None], s["logits"], 0.0).sort(dim=1, descending=True, stable=True)[1]
    index = order[:, :top]
    values = torch.where(keep[:, None], logp.gather(1, index), 0.0)
    return values, torch.where(keep[:, None], index, -1).int()


def _d_logits(s, logp, p, entropy, keep, top_index):
    g, h = s["d_logp"], s.get("d_top")
    total = g if h is None else g + h.sum(1)
    d = -p * total[:, None]
    if "d_entropy" in s:
        d = d - torch.where(p > 0, p * (logp + entropy[:, None]), 0.0) * s["d_entropy"][:, None]
    d.scatter_add_(1, s["targets"].clamp_min(0)[:, None], g[:, None])
    if h is not None:
        d.scatter_add_(1, top_index.clamp_min(0).long(), h)
    return torch.where(keep[:, None], d, 0.0).to(s["logits"].dtype)


def _plain_rows(s):
    case = s["case"]
    logp, p, entropy, keep = _softmax(s)
    out = {"logp": _at_target(s, logp, keep), "entropy": entropy}
    if case.get("top"):
        out["top_logp"], out["top_index"] = _tops(s, logp, keep, case["top"])
    if case["kind"] != "logprobs":
        out["d_logits"] = _d_logits(s, logp, p, entropy, keep, out.get("top_index"))
    return out


def _plain_lists(s):
    g = s["grads"].float()
    norm = torch.sqrt((g * g).sum(dtype=torch.float64))
    scale = torch.where(norm < 1.0, 1.0, 1.0 / norm).float()
    if s["case"]["kind"] == "clip":
        return {"norm": norm.float().reshape(1), "grads": (g * scale).to(s["grads"].dtype)}
    (b1, b2), t = ADAM["betas"], s["case"]["step"]
    g = g * scale
    avg = b1 * s["avg"] + (1 - b1) * g
    avg_sq = b2 * s["avg_sq"] + (1 - b2) * g * g
    p = s["params"].float()
    move = (avg / (1 - b1 ** t)) / (torch.sqrt(avg_sq / (1 - b2 ** t)) + ADAM["eps"])
    p = p - ADAM["lr"] * (move + ADAM["weight_decay"] * p)
    return {"norm": norm.float().reshape(1), "params": p.to(s["params"].dtype), "avg": avg,
            "avg_sq": avg_sq}


# --------------------------------------------------------- the framework's calls
def _own_rows(s):
    from bindcraft2_amd import ops
    case, x, t = s["case"], s["logits"], s["targets"]
    if case["kind"] == "logprobs_grad":
        (logp, entropy), d = ops.LogProbs().value_and_grad(x, t, s["d_logp"], s.get("d_entropy"))
        return {"logp": logp, "entropy": entropy, "d_logits": d}
    op = ops.LogProbs(top=case["top"])
    (logp, entropy, top_logp, top_index), save = op.forward(x, t)
    out = {"logp": logp, "entropy": entropy}
    if case["top"]:
        out |= {"top_logp": top_logp, "top_index": top_index}
    if case["kind"] == "logprobs_vjp":
        out["d_logits"] = op.backward((s["d_logp"], s["d_entropy"], s.get("d_top")), x, t, top_index,
                                      save)
    return out


def _own_lists(s):
    if s["case"]["kind"] == "clip":
        return {"norm": s["handle"].clip(1.0), "grads": s["out"]}
    norm = s["handle"].step(s["case"]["step"], ADAM["lr"], max_norm=1.0)
    return {"norm": norm, "params": s["out_params"], "avg": s["out_avg"], "avg_sq": s["out_avg_sq"]}


def run(state):
    lists = state["case"]["kind"] in ("clip", "adam")
    if own:
        return _own_lists(state) if lists else _own_rows(state)
    return _plain_lists(state) if lists else _plain_rows(state)


# ------------------------------------------------------------------------- work
def work(case):
    width = TYPES[case["type"]].itemsize
    if case["kind"] in ("clip", "adam"):
        n = sum(_sizes(case))
        if case["kind"] == "clip":
            return {"bytes": 2 * n * width, "flops": 3 * n}
        return {"bytes": n * (3 * width + 16), "flops": 15 * n}
    live = case["rows"] * (1 - case["ignored"])
    cells = case["rows"] * case["classes"]
    out = case["rows"] * (8 + 8 * case.get("top", 0) + 8)
    if case["kind"] == "logprobs":
        return {"bytes": live * case["classes"] * width + out, "flops": 6 * cells}
    return {"bytes": (live * case["classes"] + cells) * width + out, "flops": 14 * cells}


# ----------------------------------------------------- the definitions in 64 bits
def _exact_rows(case, seed):
    s = _in_rows(case, seed)
    keep = s["targets"] >= 0
    x = s["logits"][keep].double()  # the rows that count, and nothing else
    t = s["targets"][keep]
    rows = torch.arange(len(t), device="cuda")

    def whole(v):
        full = torch.zeros(len(keep), *v.shape[1:], dtype=torch.float64, device="cuda")
        full[keep] = v
        return full

    lse = torch.logsumexp(x, 1)
    p = torch.exp(x - lse[:, None])
    finite = torch.where(x == -math.inf, 0.0, x)
    entropy = lse - (p * finite).sum(1)
    out = {"logp": whole(x[rows, t] - lse), "entropy": whole(entropy)}
    if case.get("top"):
        out["top_logp"] = whole(torch.topk(x, case["top"], 1)[0] - lse[:, None])
        out["top_index"] = None
    if case["kind"] == "logprobs":
        return out
    g = s["d_logp"][keep].double()
    weight = torch.zeros_like(x)
    weight[rows, t] = g
    if "d_top" in s:
        # ties in the logits: the lowest index first, by a last significant digit
        order = torch.argsort(x, dim=1, descending=True, stable=True)[:, :case["top"]]
        weight = weight.scatter_add(1, order, s["d_top"][keep].double())
        g = g + s["d_top"][keep].double().sum(1)
    d = weight - p * g[:, None]
    if "d_entropy" in s:
        # dH/dx_j = -p_j (log p_j + H)
        slope = p * (finite - lse[:, None] + entropy[:, None])
        d = d - slope * s["d_entropy"][keep].double()[:, None]
    out["d_logits"] = whole(d)
    return out


def _exact_lists(case, seed):
    s = _in_lists(case, seed)
    g = s["grads"].double()
    norm = torch.linalg.vector_norm(g)
    g = g * min(1.0, 1.0 / norm.item())
    if case["kind"] == "clip":
        return {"norm": norm.reshape(1), "grads": g}
    b1, b2 = ADAM["betas"]
    avg = s["avg"].double().lerp(g, 1 - b1)
    avg_sq = s["avg_sq"].double().lerp(g.square(), 1 - b2)
    hat, hat_sq = avg / (1 - b1 ** case["step"]), avg_sq / (1 - b2 ** case["step"])
    p = s["params"].double()
    p = p * (1 - ADAM["lr"] * ADAM["weight_decay"]) - ADAM["lr"] * hat / (hat_sq.sqrt() + ADAM["eps"])
    return {"norm": norm.reshape(1), "params": p, "avg": avg, "avg_sq": avg_sq}


def exact(case, seed):
    return (_exact_lists if case["kind"] in ("clip", "adam") else _exact_rows)(case, seed)
