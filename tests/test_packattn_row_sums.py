"""The bound on d(queries) of rows of few keys tells D of the keys from D of the
rounded `out`."""
import pytest
import torch

from tests import packattn_row_sums as S


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [2, 5, 33, 200])
def test_bound(n, dtype):
    x = S.problem(40, n, 4, 2, 16, dtype, "cpu")
    want, tol = S.d_q(*x, 0.25)
    other, _ = S.d_q(*x, 0.25, rounded_out=True)
    off = (other - want).abs() > tol
    assert off.double().mean() > 0.02, off.double().mean()
