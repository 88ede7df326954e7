"""d(queries) of rows of up to 1024 keys without the rounding of `out` in them."""
import pytest
import torch

from tests import packattn_row_sums as S
from tests import sequence_ref as R
from bindcraft2_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [2, 5, 31, 64, 65, 200, 700, 1023, 1024])
@pytest.mark.parametrize("heads,kv,d", [(4, 2, 16), (2, 2, 32), (128, 64, 16)])
def test_d_q(cuda, heads, kv, d, n, dtype):
    x = S.problem(40, n, heads, kv, d, dtype, "cuda")
    offsets = [torch.tensor([0, t.shape[0]], device="cuda", dtype=torch.int32) for t in x[:2]]
    op = ops.PackedAttention(False)
    out, lse = op.forward(*x[:3], *offsets)
    got = op.backward(x[3], *x[:3], out, lse, *offsets)[0]
    R.check("d_q", got, *S.d_q(*x, d ** -0.5))
