"""The block's operators where their launches change kind: every element against the formulas in 64 bits."""
import importlib

import pytest

import block_ref as R
from test_gpu_residual import BF, F32, FP, check, close, inputs, ops  # noqa: F401 (ops: a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt,out,rows,dim,p", [
    (BF, BF, 6200, 1536, 0.0), (FP, FP, 6200, 1539, 0.1), (F32, BF, 4104, 2048, 0.0), (F32, F32, 6151, 1025, 0.1),
    (BF, BF, 4100, 1024, 0.0), (BF, BF, 4100, 2049, 0.0)])
def test_grids_of_the_residuals_gradient(ops, dt, out, rows, dim, p):  # noqa: F811
    """Widths on both sides of 1025 .. 2048, whose backward pass has half as many work-groups more, over enough rows for all of
    them, and the sums of their partial rows."""
    check(ops, inputs(rows, dim, dt, out, seed=40), p)


@pytest.mark.parametrize("dt,out", [(BF, BF), (F32, BF), (FP, FP), (F32, F32)])
@pytest.mark.parametrize("pdt", [F32, BF, FP])
def test_bias_without_weight_and_gate(pkg, ops, dt, out, pdt):  # noqa: F811
    """The gradient of a bias alone is rounded to the bias's type and to no other."""
    ad = importlib.import_module(pkg.__name__ + ".autograd")
    i = inputs(300, 72, dt, out, seed=41, gate=False)
    bias = i["bias"].to(pdt).to("cuda:0").requires_grad_()
    h, y = ad.residual_norm(i["x"].to("cuda:0"), i["branch"].to("cuda:0"), bias=bias)
    y.backward(i["dy"].to("cuda:0"))
    want = i["dy"].double().sum(0)
    tol = 303 * R.E32 * i["dy"].double().abs().sum(0)
    assert bias.grad.dtype == pdt
    close(bias.grad, want, R.rounded(want, tol, pdt), "dbias")
