"""The hand-ordered kernel of the attention's backward pass over keys, as the compiler leaves it (CPU: compiled for gfx950).

Its matrix products are inline assembly, for which the compiler keeps no distance to instructions that read their results.
So nothing may touch those registers but the order written down: no spill, no copy between register classes in the loop."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "sparse-attention-vggt_amd", "csrc")
KERNEL = "frame_attn_dkv_long_kernel"


@pytest.fixture(scope="module")
def assembly(tmp_path_factory):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("no hipcc")
    out = str(tmp_path_factory.mktemp("build") / "frame_attn.s")
    flags = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-I../../include", "-I.", "-Xclang", "-target-feature",
             "-Xclang", "-packed-fp32-ops", "-munsafe-fp-atomics"]
    with open(os.path.join(CSRC, "Makefile")) as f:  # the library is built with these
        made = re.search(r"HIPFLAGS = (.*?[^\\])\n", f.read(), re.S).group(1).replace("\\\n", " ")
    made = made.replace("$(ARCH)", "gfx950").replace("$(INC)", "-I../../include -I.").split()
    assert [x for x in made if not x.startswith("-W")] == flags
    subprocess.run([hipcc, *flags, "--cuda-device-only", "-S", "frame_attn.hip", "-o", out], cwd=CSRC, check=True,
                   capture_output=True, timeout=600)
    with open(out) as f:
        text = f.read()
    body = re.search(rf"^_ZN5saf3r\d+{KERNEL}E\S*:.*?\n(.*?)^\s*\.end_amdhsa_kernel", text, re.S | re.M).group(1)
    return body.split("s_endpgm")[0], body


def test_nothing_is_spilled(assembly):
    code, body = assembly
    assert re.search(r"\.amdhsa_private_segment_fixed_size 0\b", body)
    assert not re.search(r"^\s*(scratch|buffer)_(load|store)", code, re.M)


def test_sums_stay_where_they_are(assembly):
    """Between the first and the last product of the loop no accumulation register is read or written but by products."""
    lines = assembly[0].splitlines()
    products = [i for i, x in enumerate(lines) if "v_mfma_f32_32x32x16_bf16" in x]
    assert len(products) == 64
    loop = lines[products[0]:products[-1] + 1]
    assert not [x for x in loop if "v_accvgpr" in x]
    assert not [x for x in loop if re.search(r"\ba\[?\d", x) and "v_mfma" not in x]


def test_distances(assembly):
    """A result in vector registers is read three products later at the earliest; an operand is not written in the two
    instructions before a product reads it unless a product lies between."""
    lines = [x.split(";")[0].strip() for x in assembly[0].splitlines()]
    lines = [x for x in lines if x and not x.startswith(".")]

    def regs(text, kind="v"):
        found = set()
        for lo, hi in re.findall(rf"\b{kind}\[(\d+):(\d+)\]", text):
            found.update(range(int(lo), int(hi) + 1))
        found.update(int(x) for x in re.findall(rf"\b{kind}(\d+)\b", text))
        return found
    fresh = {}  # vector register -> products since the product that wrote it
    checked = 0
    for x in lines:
        op, _, rest = x.partition(" ")
        args = rest.split(",")
        if op.startswith("v_mfma"):
            assert args[0].strip()[0] in "va"
            used = regs(",".join(args[1:3]))
            assert not used & set(fresh), x  # (the third operand may be a result: the pipe forwards it)
            fresh = {r: n + 1 for r, n in fresh.items() if n < 2}
            if args[0].strip()[0] == "v":
                fresh.update(dict.fromkeys(regs(args[0]), 0))
                checked += 1
        elif op.startswith("v_") or op.startswith("ds_") or op.startswith("global_"):
            assert not regs(rest) & set(fresh), x
    assert checked == 32
