"""The smallest eps that Adam takes, f32's smallest subnormal and normal
values: a parameter whose gradient has always been zero stays where it is."""
import pytest
import torch

from bindcraft2_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [65, 100001])
@pytest.mark.parametrize("eps", [2.0 ** -149, 2.0 ** -126])
def test_smallest_eps(cuda, n, eps):
    p = torch.randn(n, device="cuda")
    kept, zeros = p.clone(), [torch.zeros_like(p) for _ in range(3)]
    adam = ops.Adam([p], [zeros[0]], [zeros[1]], [zeros[2]], eps=eps)
    for step in (1, 2):
        adam.step(step, 0.1)
        assert torch.equal(p, kept) and not any(z.any() for z in zeros)
