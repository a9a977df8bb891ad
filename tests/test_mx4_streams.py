"""Waits that the kernels of mx4 products are themselves to keep, read off the assembly of their sources; no GPU.

The tiles' products are written in place (inline assembly), so that the compiler does not know them: a vector
instruction's result needs two waits before a product takes it as an operand, and a sum stands sixteen behind its product.  Loads
that go from memory straight to LDS may land where a wave has read only behind a written wait for its reads."""
import os
import re
import subprocess

import pytest

from karume_amd import build
from test_lds_streams import _functions, _reads_on_their_way


def assembly(tmp_path, source):
    if not os.path.exists(build.HIPCC):
        pytest.skip("no compiler")
    out = tmp_path / "device.s"
    subprocess.run([build.HIPCC, *build.FLAGS, "--offload-device-only", "-S", os.path.join(build.CSRC, source), "-o", str(out)],
                   check=True, capture_output=True)
    return out.read_text()


def registers(operand):
    many = re.match(r"^([va])\[(\d+):(\d+)\]$", operand)
    if many:
        return {(many.group(1), i) for i in range(int(many.group(2)), int(many.group(3)) + 1)}
    one = re.match(r"^([va])(\d+)$", operand)
    return {(one.group(1), int(one.group(2)))} if one else set()


def instructions(lines):
    for line in lines:
        text = line.split(";")[0].strip()
        if text and not text.startswith("."):
            name, _, rest = text.partition(" ")
            yield name, [part.strip().split()[0] for part in rest.split(",")] if rest.strip() else []


def waits(code, at, most):
    """Instructions in front of place `at`, nearest first, while fewer than `most` waits lie between."""
    passed = 0
    while at > 0 and passed < most:
        at -= 1
        name, operands = code[at]
        if name == "s_nop":
            passed += int(operands[0]) + 1
        else:
            yield name, operands
            passed += 1


def test_products_in_place(tmp_path):
    checked = 0
    for name, lines in _functions(assembly(tmp_path, "linear_mx4_tiles.hip")):
        if "linear_mx4_tile_kernel" not in name:
            continue
        code = list(instructions(lines))
        products = 0
        for at, (op, operands) in enumerate(code):
            if op.startswith("v_mfma"):
                products += 1
                assert operands[0] == operands[3], (name, operands)   # the sum in place
                sources = set().union(*(registers(operands[i]) for i in (1, 2, 4, 5)))
                for before, written in waits(code, at, 2):
                    if before.startswith("v_") and not before.startswith("v_mfma"):
                        assert not registers(written[0]) & sources, (name, before, written, operands)
            elif op.startswith(("v_", "global_store", "ds_write")):
                sums = {r for operand in operands for r in registers(operand) if r[0] == "a"}
                for before, written in waits(code, at, 16) if sums else ():
                    if before.startswith("v_mfma"):
                        assert not registers(written[0]) & sums, (name, op, operands)
            # 16 bytes on their way to memory are read a little later than the store is issued
            if op.startswith("v_") and at and code[at - 1][0] == "global_store_dwordx4" and operands:
                assert not registers(operands[0]) & registers(code[at - 1][1][1]), (name, op, operands)
        assert products in (32, 64, 256), name
        checked += 1
    assert checked == 5 * 2 * 2 * 2    # tiles and depths, stored types, pairs, whole words


def test_rings_are_filled_behind_their_reads(tmp_path):
    counted = {"rows": 0, "batch": 0}
    for name, lines in _functions(assembly(tmp_path, "linear_mx4_rows.hip")):
        kind = re.search(r"linear_mx4_(rows|batch)_kernel", name)
        if kind:
            loads = _reads_on_their_way(lines)
            assert len(loads) >= 4 and not any(loads), name
            counted[kind.group(1)] += 1
    assert counted == {"rows": 3 * 4 * 2 * 2 * 2, "batch": 2 * 2 * 2 * 2}
