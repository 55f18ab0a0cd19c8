"""The waits in front of the 8-bit tiles' products, on every way to them: the products are written as instructions, before which the compiler adds no waits, and the
last instructions of a round of the loop come before the first product of the next one."""
import importlib
import os
import re
import subprocess

import pytest


def _operands(text):
    return [x.strip() for x in re.split(r",(?![^\[]*\])", text.split(" op_sel")[0])]


def _registers(name):
    m = re.fullmatch(r"v\[(\d+):(\d+)\]|v(\d+)", name)
    return set() if not m else {int(m[3])} if m[3] else set(range(int(m[1]), int(m[2]) + 1))


def _written(op, rest):
    """The vector registers that an instruction of the vector unit writes (the matrix cores write accumulation registers here)."""
    if not op.startswith("v_") or "mfma" in op or op.startswith("v_cmp"):
        return set()
    ops = _operands(rest)
    return _registers(ops[0]) | (_registers(ops[1]) if "swap" in op else set())


def _ways(body):
    """The instructions of a kernel, and for each those that may come right before it."""
    code, labels = [], {}
    for line in body.splitlines():
        line = line.split(";")[0].strip()
        if line.endswith(":"):
            labels[line[:-1]] = len(code)
        elif line and line[0] != ".":
            code.append(tuple(x.strip() for x in line.partition(" ")[::2]))
    before = [[] for _ in range(len(code) + 1)]
    for at, (op, rest) in enumerate(code):
        if op == "s_branch" or op.startswith("s_cbranch"):
            before[labels[rest]].append(at)
        if op not in ("s_branch", "s_endpgm", "s_setpc_b64"):
            before[at + 1].append(at)
    return code, before


def _unwaited(code, before):
    """(products, pairs of a write by the vector unit and a product that reads it less than two instructions or an s_nop 1 later)"""
    products, found = 0, []
    for at, (op, rest) in enumerate(code):
        if not op.startswith("v_mfma_scale"):
            continue
        products += 1
        _, w, a, _, w_powers, a_powers = _operands(rest)
        read = _registers(w) | _registers(a) | _registers(w_powers) | _registers(a_powers)
        ways = [(p, 0) for p in before[at]]
        while ways:
            p, waits = ways.pop()
            if _written(*code[p]) & read:
                found.append((p, at))
            waits += 1 + (int(code[p][1]) if code[p][0] == "s_nop" else 0)
            if waits < 2:
                ways += [(q, waits) for q in before[p]]
    return products, found


MFMA = "v_mfma_scale_f32_16x16x128_f8f6f4 a[0:3], v[8:15], v[16:23], a[0:3], v1, v2 op_sel:[0,0,0] op_sel_hi:[0,0,0]"


@pytest.mark.parametrize("lines,bad", [
    (["v_mov_b32_e32 v9, v3", MFMA], True),
    (["v_mov_b32_e32 v9, v3", "s_nop 0", MFMA], True),
    (["v_mov_b32_e32 v9, v3", "s_nop 1", MFMA], False),
    (["v_mov_b32_e32 v9, v3", "s_mov_b32 s0, 1", "s_mov_b32 s1, 1", MFMA], False),
    (["v_mov_b32_e32 v24, v3", MFMA], False),
    (["v_mov_b32_e32 v2, v3", MFMA], True),
    (["v_permlane16_swap_b32 v30, v16", MFMA], True),
    ([".LBB0_1:", MFMA, "s_add_i32 s0, s0, 1", "v_add_u32_e32 v1, 1, v1", "s_cbranch_scc1 .LBB0_1", "s_endpgm"], True),        # over the loop's edge only
    ([".LBB0_1:", "s_nop 1", MFMA, "v_add_u32_e32 v1, 1, v1", "s_cbranch_scc1 .LBB0_1", "s_endpgm"], False),
    (["v_add_u32_e32 v1, 1, v1", "s_branch .LBB0_2", ".LBB0_1:", "v_mov_b32_e32 v8, v3", ".LBB0_2:", "s_nop 0", MFMA, "s_endpgm"], True),
    (["s_branch .LBB0_2", "v_mov_b32_e32 v8, v3", ".LBB0_2:", MFMA, "s_endpgm"], True),
    (["s_branch .LBB0_2", "v_mov_b32_e32 v8, v3", "s_endpgm", ".LBB0_2:", MFMA, "s_endpgm"], False),
])
def test_what_the_check_sees(lines, bad):
    products, found = _unwaited(*_ways("\n".join(lines)))
    assert products == 1 and bool(found) == bad


def test_products_wait_on_every_way(tmp_path):
    library = importlib.import_module("daisi-llogos_amd.ops.library")
    try:
        hipcc = library._hipcc()
    except library.KernelLibraryError:
        pytest.skip("no compiler")
    out = tmp_path / "tiles.s"
    subprocess.run([hipcc, *library.HIPCC_FLAGS, "-I", library._CSRC, "--offload-device-only", "-S", os.path.join(library._CSRC, "gemm_blocks_tiles.hip"),
                    "-o", str(out)], check=True, capture_output=True)
    kernels = re.findall(r"^(_Z24gemm_blocks_tiles_kernel\S*):(.*?)^\.Lfunc_end", out.read_text(), re.S | re.M)
    assert kernels
    for name, body in kernels:
        code, before = _ways(body)
        products, found = _unwaited(code, before)
        assert products >= 64 and any(p >= at for at, ways in enumerate(before) for p in ways), name          # (there is a loop to follow)
        assert not found, (name, [(code[p], code[at]) for p, at in found[:3]])
