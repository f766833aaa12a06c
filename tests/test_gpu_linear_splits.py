"""Split reductions whose last split is a single step of 64, whole or cut off, in each of the three products; every element
against the formulas in 64 bits."""
import importlib

import pytest

from test_gpu_linear import BF, DEV, F32, check, inputs, ops  # noqa: F401 (ops: a fixture)

pytestmark = pytest.mark.gpu

# (rows, columns, steps, splits of them): tiles of 64 x 64 with three and more steps a split, then of 128 x 128
PLANS = [(33, 64, 19, 7), (64, 72, 46, 16), (200, 136, 25, 9), (520, 72, 61, 11), (130, 512, 466, 32), (1536, 72, 181, 16)]


def last_split(pkg, m, n, k):
    """(splits, steps of the last one) of a product [m, k] x [k, n] of more than 32 rows, from its workspace."""
    lib = importlib.import_module(pkg.__name__ + "._lib").load()
    used = lib.saf3r_linear_fwd_workspace_bytes(m, k, n, 0, 0, 0) // (m * -(-n // 8) * 8 * 4)
    steps = -(-k // 64)
    per = {p for p in range(1, steps + 1) if -(-steps // p) == used}
    return used, {steps - p * (used - 1) for p in per}


@pytest.mark.parametrize("cut", [0, 24, 61])
@pytest.mark.parametrize("m,n,steps,splits", PLANS)
def test_a_last_split_of_one_step(pkg, ops, m, n, steps, splits, cut):  # noqa: F811
    k = 64 * steps - cut
    assert last_split(pkg, m, n, k) == (splits, {1}), "other splits than these sizes were chosen for"
    check(ops, inputs(m, k, n, BF, seed=50, residual=F32), "gelu", 0.1, where=DEV)  # forward
    check(ops, inputs(m, n, k, BF, seed=51, gate=False), None, where=DEV)           # dx: out is summed over
    check(ops, inputs(k, n, m, BF, seed=52, gate=False), None, where=DEV)           # dweight: rows are
