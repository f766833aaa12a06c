"""Distances between the inline-assembly products of the hand-ordered kernel and everything around them, on the paths that
the compiled code takes: into the loop, round it twice, past its branches either way, and out of it (CPU: compiled for
gfx950). Texts with a mistake planted show that each rule is looked at."""
import re

import pytest

from test_frame_attn_build import assembly  # noqa: F401 (a fixture)

WAIT = 16  # steps that an instruction other than a product keeps from the last write of the sums it reads


def instructions(text):
    lines = (re.split(r";|//", x)[0].strip() for x in text.splitlines())
    return [x for x in lines if x and (not x.startswith(".") or x.endswith(":"))]


def regs(text):
    """Registers that operands name: ("v" or "a", number)."""
    found = set()
    for kind, lo, hi in re.findall(r"\b([va])\[(\d+):(\d+)\]", text):
        found.update((kind, r) for r in range(int(lo), int(hi) + 1))
    found.update((kind, int(r)) for kind, r in re.findall(r"\b([va])(\d+)\b", text))
    return found


def is_product(x):
    return x.startswith("v_mfma")


def loop_of(lines):
    """(first, last): the label and the backward branch around all products."""
    products = [i for i, x in enumerate(lines) if is_product(x)]
    assert len(products) == 64
    for i in range(products[-1], len(lines)):
        m = re.match(r"s_c?branch\S*\s+(\S+)", lines[i])
        if m and m.group(1) + ":" in lines and lines.index(m.group(1) + ":") < products[0]:
            return lines.index(m.group(1) + ":"), i
    raise AssertionError("no loop around the products")


def path(lines, taken, turns=2, behind=400):
    """The instructions of a run that enters the loop, goes `turns` times round it and leaves it; branches inside it are all
    taken, or none."""
    first, last = loop_of(lines)
    start = max(i for i in range(first) if lines[i].endswith(":") or lines[i].startswith("s_branch")) + 1
    labels = {x[:-1]: i for i, x in enumerate(lines) if x.endswith(":")}
    out, i, left, outside = [], start, turns, 0
    while i < len(lines) and outside < behind:
        x = lines[i]
        m = re.match(r"s_(c?)branch\S*\s+(\S+)", x)
        if first <= i <= last and m:
            to = labels[m.group(2)]
            if i == last:
                left -= 1
                go = left > 0 or not m.group(1)
                assert left > 0 or m.group(1), "the loop is left at its end or by a branch before it"
            elif first < to <= last:
                go = taken
            else:  # out of the loop: where nothing but the rest of the last turn is behind
                go = left == 1 and not any(is_product(y) for y in lines[i:last])
            i = to if go else i + 1
        else:
            if not x.endswith(":"):
                out.append(x)
            outside += i > last
            i += 1
    assert sum(map(is_product, out)) == 64 * turns
    return out


def violations(run):
    """What a run does too early: (rule, instruction)."""
    found = []
    fresh = {}    # vector register -> products since the product that wrote it
    third = {}    # register of a separate third operand -> products since its product
    written = []  # (steps ago, registers) of vector instructions since the last product
    sums = set()  # accumulation registers that products write
    since = 0     # steps since the last product
    for x in run:
        op, _, rest = x.partition(" ")
        args = [a.strip() for a in rest.split(",")]
        if is_product(x):
            dest, c = regs(args[0]), regs(args[3])
            if regs(",".join(args[1:3])) & set(fresh):
                found.append(("a product's result as a factor", x))
            if any(steps < 2 and r & (regs(",".join(args[1:])) | dest) for steps, r in written):
                found.append(("an operand written right ahead of its product", x))
            if dest != c and dest & c:
                found.append(("a third operand that overlaps the result", x))
            if dest & set(third):
                found.append(("a third operand overwritten by a product", x))
            fresh = {r: n + 1 for r, n in fresh.items() if n < 2 and r not in dest}
            third = {r: n + 1 for r, n in third.items() if n < 1}
            if dest != c:
                third.update(dict.fromkeys(c, 0))
            fresh.update({r: 0 for r in dest if r[0] == "v"})
            sums |= {r for r in dest if r[0] == "a"}
            written, since = [], 0
            continue
        if re.match(r"(v_|ds_|global_|buffer_|flat_|scratch_)", op):
            touched = regs(rest)
            if touched & set(fresh):
                found.append(("a product's result too early", x))
            if touched & sums and since < WAIT:
                found.append(("a sum too early", x))
            stores = re.match(r"(ds_write|ds_store|global_store|buffer_store|global_load_lds|v_cmp|v_readlane|v_readfirst)", op)
            wrote = set() if stores else regs(args[0])
            if wrote & set(third):
                found.append(("a third operand overwritten too early", x))
            if op.startswith("v_") and wrote:
                written.append((-1, wrote))
        steps = int(args[0]) + 1 if op == "s_nop" else 1
        written = [(n + steps, r) for n, r in written]
        since += steps
    return found


@pytest.mark.parametrize("taken", [False, True])
def test_distances_on_every_path(assembly, taken):  # noqa: F811
    assert violations(path(instructions(assembly[0] + "\ns_endpgm"), taken)) == []


def test_sums_are_read_behind_their_wait(assembly):  # noqa: F811
    """The kernel's own wait lies between the loop and the first copy that the compiler makes of a sum."""
    lines = instructions(assembly[0])
    run = path(lines, False)
    behind = run[max(i for i, x in enumerate(run) if is_product(x)) + 1:]
    first = next(i for i, x in enumerate(behind) if re.match(r"v_accvgpr_(read|mov)", x))
    assert [x for x in behind[:first] if x.split() == ["s_nop", "15"]], behind[:first + 1]


def at_product(lines, n):
    return [i for i, x in enumerate(lines) if is_product(x)][n]


def operands(x):
    return [a.strip() for a in x.partition(" ")[2].split(",")]


def first_of(text):
    kind, r = re.match(r"([va])\[(\d+)", text).groups()
    return f"{kind}{r}"


def ahead_of_the_last(lines):
    i = at_product(lines, 63)
    return lines[:i] + [f"v_mov_b32_e32 {first_of(operands(lines[i])[1])}, 0"] + lines[i:]


def one_ahead_of_the_last(lines):
    i = at_product(lines, 63)
    return lines[:i] + [f"v_mov_b32_e32 {first_of(operands(lines[i])[2])}, 0", "s_add_i32 s0, s0, 1"] + lines[i:]


def over_a_third_operand(lines):
    i = at_product(lines, 0)
    return lines[:i + 1] + [f"v_mov_b32_e32 {first_of(operands(lines[i])[3])}, 0"] + lines[i + 1:]


def read_over_a_third_operand(lines):
    i = at_product(lines, 1)
    c = operands(lines[at_product(lines, 0)])[3]
    lo = int(re.search(r"\d+", c).group())
    return lines[:i] + [f"ds_read_b128 v[{lo}:{lo + 3}], v0"] + lines[i:]


def over_the_back_edge(lines):
    _, last = loop_of(lines)
    first = at_product(lines, 0)
    kept = [x for x in lines[loop_of(lines)[0] + 1:first] if x.startswith("s_nop")]
    assert not kept
    # (nothing but the label between it and the first product: the instructions there are taken out)
    label = loop_of(lines)[0]
    cut = lines[:label + 1] + lines[first:]
    last -= first - label - 1
    x = f"v_mov_b32_e32 {first_of(operands(lines[first])[1])}, 0"
    return cut[:last] + [x] + cut[last:]


def a_result_too_early(lines):
    i = at_product(lines, 3)  # (the last product of the first score tile)
    return lines[:i + 1] + [f"v_mul_f32_e32 v255, 1.0, {first_of(operands(lines[i])[0])}"] + lines[i + 1:]


def a_sum_right_behind_the_loop(lines):
    _, last = loop_of(lines)
    i = at_product(lines, 63)
    return lines[:i + 1] + [f"v_accvgpr_read_b32 v0, {first_of(operands(lines[i])[0])}"] + lines[i + 1:]


@pytest.mark.parametrize("plant", [ahead_of_the_last, one_ahead_of_the_last, over_a_third_operand,
                                   read_over_a_third_operand, over_the_back_edge, a_result_too_early,
                                   a_sum_right_behind_the_loop])
@pytest.mark.parametrize("taken", [False, True])
def test_planted_mistakes_are_seen(assembly, plant, taken):  # noqa: F811
    assert violations(path(plant(instructions(assembly[0])), taken))
