"""The operators as a design program runs them together: head logits of a
design step, a loss of their log-probabilities and entropies, its gradient
into the step's backward, and the states' gradients clipped and taken by Adam."""
import numpy as np
import pytest
import torch

from bindcraft2_amd import ops, params as bparams
from tests.helpers import metrics, weights_dir

pytestmark = pytest.mark.gpu
D = torch.float64


def test_loss_of_head_logits_to_updated_logits(cuda):
    """Heads in, gradients out: bins of a distogram [N, N, 64] with padded
    pairs, pLDDT [N, 50] and sequence logits [N, 20] as one loss; the
    sequences' gradients of three states clipped together and stepped.  The
    whole against the same in 64 bits."""
    n, gen = 37, torch.Generator("cuda").manual_seed(1)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    states = [rnd(n, 20) for _ in range(3)]
    avg, avg_sq = [torch.zeros_like(s) for s in states], [torch.zeros_like(s) for s in states]
    native = torch.randint(20, (n,), generator=gen, device="cuda")
    native[30:] = -1
    weight = torch.full((n,), -1.0 / 30, device="cuda")
    grads = [torch.empty_like(s) for s in states]
    clip = ops.GradientClip(grads)
    adam = ops.Adam(states, grads, avg, avg_sq, eps=1e-2)
    ref = [s.double().cpu().requires_grad_() for s in states]
    first, second = [torch.zeros(n, 20, dtype=D) for _ in ref], [torch.zeros(n, 20, dtype=D) for _ in ref]
    for step in (1, 2, 3):
        for s, g in zip(states, grads):
            (logp, entropy), d = ops.LogProbs().value_and_grad(s, native, weight, weight, out=g)
            assert d is g
        norm = clip.clip(0.05)
        adam.step(step, 0.1)
        loss = 0
        for s in ref:
            lp = torch.log_softmax(s[:30], -1)
            picked = lp.gather(1, native[:30].cpu()[:, None])
            loss = loss - (picked.sum() - (lp.exp() * lp).sum()) / 30
        g = torch.autograd.grad(loss, ref)
        total = torch.sqrt(sum((x * x).sum() for x in g))
        assert abs(norm.item() - total.item()) <= 1e-5 * total.item()
        with torch.no_grad():
            for k, s in enumerate(ref):
                c = g[k] * min(1.0, 0.05 / total.item())
                first[k] = 0.9 * first[k] + 0.1 * c
                second[k] = 0.999 * second[k] + 0.001 * c * c
                s -= 0.1 * (first[k] / (1 - 0.9 ** step)) / ((second[k] / (1 - 0.999 ** step)).sqrt() + 1e-2)
    for s, r in zip(states, ref):
        # a gradient's terms are at most (2 + log 20) / 30 with 40 half steps
        # (5e-7); over eps, times 0.1, three times; and three roundings of s
        assert (s.cpu().double() - r).abs().max() < 3e-5
        assert (s[30:].cpu().double() - r[30:].detach()).abs().max() == 0


def _design(n):
    rng = np.random.default_rng(77)
    extra = {}
    for mod, shapes in bparams.module_shapes(c_m=64).items():
        if mod == "msa_column_attention":
            mod, shapes = "msa_column_global_attention", bparams.global_attention_shapes(64)
        for name, arr in bparams.init_module(shapes, rng, gates="random", ln="random").items():
            extra[f"param/block0/{mod}/{name}"] = arr
    post = bparams.init_structure_heads_params(rng, final="random", ln="random")
    post.update({f"const/{k}": v for k, v in bparams.init_residue_tables(rng).items()})
    prm = {"emb": bparams.init_embedder_params(rng),
           "tpl": bparams.init_template_embedding_params(1, rng, gates="random", ln="random"),
           "extra": extra, "main": bparams.init_block_params(0, rng, gates="random", ln="random"),
           "post": post}
    dirs = [weights_dir(v, f"loss_{k}_{n}") for k, v in prm.items()]
    return ops.DesignStepSeq(*dirs, depths=(1, 1, 1, 1))


def test_distogram_likelihood_through_a_design_step(cuda):
    """Designed logits of two states -> design step -> likelihood and entropy of
    distance bins -> the step's backward -> clipped gradients -> Adam.  The
    step's backward is linear in its cotangent, so the loss's gradient is held
    to the 64-bit one through it, and what follows to the definition."""
    n = 32
    step, gen = _design(n), torch.Generator("cuda").manual_seed(3)
    states = [torch.randn(n, 20, generator=gen, device="cuda") for _ in range(2)]
    flags = torch.ones(n, dtype=torch.uint8, device="cuda")
    scalars = torch.tensor([1.0, 0.0, 1.0, 1.0], device="cuda")
    mask = torch.ones(n, device="cuda")
    at = torch.arange(n, device="cuda", dtype=torch.float32)
    ids = [at, torch.ones_like(mask), torch.ones_like(mask), torch.ones_like(mask)]
    bins = torch.randint(-1, 64, (n, n), generator=gen, device="cuda", dtype=torch.int32)
    keep = bins >= 0
    weight = torch.full((n, n), -1.0 / n, device="cuda")
    grads = []
    for s in states:
        outs, save = step.forward(s, flags, scalars, ids, mask, dropout=False)
        (logp, entropy), d = ops.LogProbs().value_and_grad(outs[1], bins, weight, weight)
        x = outs[1].double().requires_grad_()
        lp = torch.log_softmax(x, -1)
        picked = lp.gather(2, bins.clamp_min(0).long()[..., None])[..., 0]
        h = -(lp.exp() * lp).sum(-1)
        want, = torch.autograd.grad((weight * (picked + h) * keep).sum(), x)
        # 80 half steps of f32 of terms of at most weight (2 + log 64)
        assert (d.double() - want).abs().max() <= 80 * 2.0 ** -24 * (2 + np.log(64)) / n
        back = lambda c: step.backward([None, c, None, None, None], s, flags, scalars, mask, save,  # noqa: E731
                                       with_template=False, dropout=False)
        got, ref = back(d), back(want.float())
        assert got.abs().max() > 0 and metrics(got, ref)["rel_l2"] <= 5e-3
        grads.append(got)
    clipped = [torch.empty_like(g) for g in grads]
    norm = ops.GradientClip(grads, out=clipped).clip(1e-3)
    total = torch.sqrt(sum(g.double().square().sum() for g in grads)).item()
    assert abs(norm.item() - total) <= 1e-6 * total
    c = min(1.0, 1e-3 / total)
    assert all(torch.allclose(o.double(), g.double() * c, rtol=1e-6, atol=0)
               for o, g in zip(clipped, grads))
    zeros = lambda: [torch.zeros_like(s) for s in states]  # noqa: E731
    before = [s.clone() for s in states]
    again = [s.clone() for s in states]
    ops.Adam(states, clipped, zeros(), zeros()).step(1, 0.1)
    ops.Adam(again, grads, zeros(), zeros()).step(1, 0.1, max_norm=1e-3)
    for s, t, b, g in zip(states, again, before, clipped):
        g = g.double()
        assert (s.double() - (b.double() - 0.1 * g / (g.abs() + 1e-8))).abs().max() <= 1e-6
        assert (s - t).abs().max() <= 1e-6  # the norm's rounding between the two
