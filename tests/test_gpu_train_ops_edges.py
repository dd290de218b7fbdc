"""The operators around the blocks of a training step where their plans change: pairs of CTAs, strips and gate groups, columns one by
one, several contexts at once, what a graph keeps, what is refused. The statements in 64 bits and their bounds are those of
test_gpu_train_ops.py."""
import pytest
import torch

from asca_b200 import ops
from test_gpu_train_ops import DTYPES, join_case, rand
from test_gpu_train_ops import test_gated_residual_forward_and_gradients as check_join

pytestmark = pytest.mark.gpu


# Above 4096 columns two CTAs share a row of the backward pass. Up to 74 rows a pair has one row: every value rests on the first
# exchange between its CTAs.
@pytest.mark.parametrize("rows,cols,per", [(1, 4097, None), (1, 8192, None), (2, 4100, 1), (5, 8191, 2), (60, 5001, 7), (74, 8192, None), (73, 6144, 1)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_first_rows_of_a_pair(gpu, rows, cols, per, dtype):
    check_join(gpu, rows, cols, per, True, True, dtype)
    t, kw = join_case(rows, cols, per, True, True, dtype)
    args = dict(gate=t["gate"], w_post=t["w_post"], w_pre=t["w_pre"], **kw)
    d_xn, d_out = rand(7, rows, cols, dtype=dtype), rand(8, rows, cols)
    first = ops.gated_residual_rmsnorm_bwd(gpu, t["y"], t["x"], d_xn, d_out, **args)
    for _ in range(50):   # one behind the other: pairs that start while others leave
        again = ops.gated_residual_rmsnorm_bwd(gpu, t["y"], t["x"], d_xn, d_out, **args)
        assert all(torch.equal(v, again[k]) for k, v in first.items())
