"""What the C header promises about the workspaces of the block's operators (CPU: the size functions and refusals)."""
import os
import re
from importlib import import_module

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def L(pkg):
    return import_module(pkg.__name__ + "._lib")


def header():
    with open(os.path.join(ROOT, "include", "saf3r_hip.h")) as f:
        return f.read()


@pytest.mark.parametrize("name", ["saf3r_layer_norm_bwd_workspace_bytes", "saf3r_residual_norm_bwd_workspace_bytes"])
def test_bounds_of_row_workspaces(L, name):
    """The size never passes the documented multiple of the width, and some width reaches it."""
    doc = re.search(rf"Workspace bytes of {name[:-len('_workspace_bytes')]} \(at most (\d+) \* dim\)", header())
    bound = int(doc.group(1))
    size = getattr(L.load(), name)
    dims = (1, 2, 7, 63, 64, 65, 256, 512, 1023, 1024, 1025, 1536, 2047, 2048, 2049, 4096, 8191, 8192)
    sizes = {d: max(size(rows, d) for rows in (0, 1, 8, 4096, 6144, 10408, 1 << 20, 1 << 38)) for d in dims}
    assert all(0 < n <= bound * d for d, n in sizes.items()), (bound, {d: n / d for d, n in sizes.items()})
    assert any(n == bound * d for d, n in sizes.items())


def test_operands_that_are_copied(pkg, L):
    """The header's list, the wrappers' and the entry's: each is refused without the copy's workspace."""
    ops, lib = import_module(pkg.__name__ + ".ops"), L.load()
    limit = int(re.search(r"copies: 1: of x, 2: of w [^*]*\* is less than `in` or more than (\d+)\)", header()).group(1))
    assert not ops._copied(256, limit, 64)
    for ptr, stride, width in ((256, limit + 8, 64), (256, 56, 64), (256, 65, 64), (264, 64, 64), (256, 64, 60)):
        assert ops._copied(ptr, stride, width)
        for x, w in (((ptr, stride), (256, 64)), ((256, 64), (ptr, stride))):
            assert lib.saf3r_linear_fwd_workspace_bytes(3, 64, 32, 0, 0, 0) == 0
            rc = lib.saf3r_linear_fwd(*x, *w, 1, 3, width, 32, None, None, 0, 0, 0, None, None, 0, 256, 32, 1, None, 0, None, 0,
                                      None)
            assert rc == 1 and b"workspace" in lib.saf3r_last_error()
