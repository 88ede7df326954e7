"""The prompt-to-token program that the documents show, run as it is written."""
import glob
import os
import re

import pytest
import torch

from tests import sequence_ref as R
from tests.conftest import ROOT

pytestmark = pytest.mark.gpu


def documented():
    """The one Python block of the documents that draws classes."""
    text = "".join(open(p, encoding="utf-8").read() for p in sorted(glob.glob(os.path.join(ROOT, "*.md"))))
    blocks = [b for b in re.findall(r"```python\n(from bindcraft2_amd import ops\n.*?)```", text, re.S)
              if "ops.Sampler(" in b]
    assert len(blocks) == 1
    return blocks[0]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_documented_prompts(cuda, dtype):
    gen = torch.Generator("cuda").manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    lengths, capacity, heads, kv, width, channels, classes = [33, 1, 70], 80, 4, 2, 64, 32, 500
    n = len(lengths)
    at = torch.tensor([0, *lengths], device="cuda").cumsum(0).int()
    pos = torch.cat([torch.arange(c, device="cuda") for c in lengths])
    slots = torch.cat([b * capacity + torch.arange(c, device="cuda") for b, c in enumerate(lengths)])
    names = {
        "torch": torch, "freq": 10000.0 ** (-torch.arange(0, width, 2, device="cuda").float() / width),
        "sequences": n, "capacity": capacity, "heads": heads, "kv_heads": kv, "width": width,
        "w_qkv": (rnd(channels, (heads + 2 * kv) * width) / channels ** 0.5).to(dtype),
        "w_out": (3 * rnd(heads * width, classes) / (heads * width) ** 0.5).to(dtype),
        "q_weight": 1 + 0.1 * rnd(width), "k_weight": 1 + 0.1 * rnd(width),
        "cache_k": torch.full((n * capacity, kv, width), float("nan"), device="cuda", dtype=dtype),
        "cache_v": torch.full((n * capacity, kv, width), float("nan"), device="cuda", dtype=dtype),
        "prompts": rnd(sum(lengths), channels).to(dtype), "positions": pos, "slots": slots, "starts": at,
        "lengths": torch.tensor(lengths, device="cuda", dtype=torch.int32)}
    exec(documented(), names)
    torch.cuda.synchronize()
    raw = (names["prompts"] @ names["w_qkv"]).view(-1, heads + 2 * kv, width)
    args = pos, names["freq"]
    q, _ = R.head_norm(raw[:, :heads], *args, names["q_weight"], 1e-6, False)
    k, tol = R.head_norm(raw[:, heads:heads + kv], *args, names["k_weight"], 1e-6, False)
    R.check("keys in the cache", names["cache_k"][slots], k, tol + R.rounding(k, dtype))
    assert torch.equal(names["cache_v"][slots], raw[:, heads + kv:])
    out = []
    for b, c in enumerate(lengths):
        s = slice(int(at[b]), int(at[b]) + c)
        out.append(R.attention(q[s], k[s], raw[s, heads + kv:].double(), True, width ** -0.5)["out"][0][-1].flatten())
    logits = torch.stack(out) @ names["w_out"].double()
    # roundings of q, k, P, out and the logits, 2^-8 at most each and of random signs
    # over 256 terms: held to ten times one of them
    assert (names["logits"].double() - logits).norm() <= 10 * R.half_step(dtype) * logits.norm()
    drawn = names["token"]
    assert drawn.shape == (n,) and drawn.dtype == torch.int32 and ((drawn >= 0) & (drawn < classes)).all()
    x = names["logits"].double() / 0.8
    for r in range(n):  # among the first 50, with its share of them
        kept = x[r].sort(descending=True, stable=True)[1][:50]
        assert drawn[r] in kept and names["logp"][r] >= torch.log_softmax(x[r][kept], 0)[kept == drawn[r]].item() - 1e-6
