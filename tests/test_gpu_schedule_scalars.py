"""A step's learning rate and number on the device have to lie side by side:
a column of a schedule's table is refused, its row is taken."""
import pytest
import torch

from bindcraft2_amd import ops

pytestmark = pytest.mark.gpu


def test_schedule_columns_are_refused(cuda):
    f = lambda: torch.randn(64, device="cuda")  # noqa: E731
    p, g, m, v = f(), f(), f(), f().square()
    table = torch.tensor([[0.1, 0.2, 0.3], [1.0, 2.0, 3.0]], device="cuda")
    adam, kept = ops.Adam([p], [g], [m], [v]), [x.clone() for x in (p, m, v)]
    with pytest.raises(ValueError, match="scalars"):
        adam.step(1, 0.0, scalars=table[:, 1])
    assert all(torch.equal(a, b) for a, b in zip((p, m, v), kept))
    adam.step(1, 0.0, scalars=table.t().contiguous()[1])
    got = [x.clone() for x in (p, m, v)]
    for a, b in zip((p, m, v), kept):
        a.copy_(b)
    adam.step(2, float(table[0, 1]))
    assert all(torch.equal(a, b) for a, b in zip((p, m, v), got))
