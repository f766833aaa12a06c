"""Vector accesses of the row kernels, as the compiler sees them (CPU: compiled for gfx950).

``load_vec`` and ``store_vec`` are called where rows, parameters and LDS rows lie at 16-byte alignment. A vector of eight floats
has 32 bytes of its own, and an access that promises as much may be compiled to addresses whose low five bits are taken for
zeros."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "sparse-attention-vggt_amd", "csrc")

SOURCE = """
#include "row_ops.h"
using namespace saf3r;
template <int VE, typename T>
__device__ void copy(const void* from, void* to) {
  float x[VE];
  load_vec<VE>((const T*)from, x);
  store_vec<VE>((T*)to, x);
}
"""


@pytest.mark.parametrize("kind,ve,aligned", [("float", 8, 16), ("float", 4, 16), ("__bf16", 8, 16), ("_Float16", 8, 16),
                                             ("_Float16", 16, 16), ("__bf16", 4, 8), ("float", 2, 8)])
def test_alignment_of_vectors(tmp_path, kind, ve, aligned):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("no hipcc")
    src, out = tmp_path / "copy.hip", tmp_path / "copy.ll"
    src.write_text(SOURCE + f"__global__ void k(const void* from, void* to) {{ copy<{ve}, {kind}>(from, to); }}\n")
    subprocess.run([hipcc, "--offload-arch=gfx950", "-O1", "-std=c++17", "-I../../include", "-I.", "-Xclang", "-target-feature",
                    "-Xclang", "-packed-fp32-ops", "--cuda-device-only", "-S", "-emit-llvm", str(src), "-o", str(out)],
                   cwd=CSRC, check=True, capture_output=True, timeout=300)
    body = re.search(r"define [^\n]*@_Z1kPKvPv\(.*?\n}", out.read_text(), re.S).group(0)
    promised = [int(n) for n in re.findall(r"(?:load|store) <[^\n]*, align (\d+)", body)]
    assert len(promised) == 2 and max(promised) <= aligned, body
