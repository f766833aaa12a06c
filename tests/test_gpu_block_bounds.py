"""The block's operators where their launches change kind: every element against the formulas in 64 bits."""
import pytest

from test_gpu_residual import BF, F32, FP, check, inputs, ops  # noqa: F401 (ops: a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt,out,rows,dim,p", [(BF, BF, 6200, 1536, 0.0), (FP, FP, 6200, 1539, 0.1), (F32, BF, 4104, 2048, 0.0),
                                               (F32, F32, 6151, 1025, 0.1), (BF, BF, 4100, 1024, 0.0), (BF, BF, 4100, 2049, 0.0)])
def test_grids_of_the_residuals_gradient(ops, dt, out, rows, dim, p):  # noqa: F811
    """Widths on both sides of 1025 .. 2048, whose backward pass has half as many work-groups more, over enough rows for all of
    them, and the sums of their partial rows."""
    check(ops, inputs(rows, dim, dt, out, seed=40), p)
