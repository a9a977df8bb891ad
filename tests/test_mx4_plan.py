"""The form that a product of mx4 rows takes, asked of the plan itself (a header without anything of the device)."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

import test_gpu_mx4
from karume_amd import build

SHIM = """
#include "mx4_plan.h"
extern "C" void form(uint32_t m, uint32_t n, uint32_t k, uint64_t scratch, uint32_t counters, uint32_t* out) {
  const krm::Mx4Form f = krm::mx4_form(m, n, k, 256, scratch, counters);
  out[0] = (uint32_t)f.kernel; out[1] = f.rows; out[2] = f.parts; out[3] = f.deep; out[4] = f.whole;
}
extern "C" uint32_t fits(uint32_t m, uint32_t k) { return krm::mx4_rows_fit(m, k); }
"""
SCRATCH, COUNTERS = 64 << 20, 1 << 16
ROWS, BATCH, TILES = 0, 1, 2


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no compiler")
    at = tmp_path_factory.mktemp("plan")
    (at / "shim.cpp").write_text(SHIM)
    library = os.path.join(at, "shim.so")
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-I", build.CSRC, str(at / "shim.cpp"), "-o", library],
                   check=True)
    return C.CDLL(library)


def form(plan, m, n, k, scratch=SCRATCH, counters=COUNTERS):
    out = (C.c_uint32 * 5)()
    plan.form(m, n, k, C.c_uint64(scratch), counters, out)
    return tuple(out)


def test_every_form_has_a_product_that_the_gpu_tests_run(plan):
    seen = set()
    for m, n, k in test_gpu_mx4.PRODUCTS + test_gpu_mx4.LARGE:
        kernel, rows, parts, deep, whole = form(plan, m, n, k)
        words = k % 128 == 0
        if kernel == ROWS:
            steps = (k + 127) // 128
            seen.add((kernel, 4 if steps > 16 else 2 if steps > 8 else 1, words))
        elif kernel == BATCH:
            seen.add((kernel, 32 if m <= 32 else 64, words))
        else:
            seen.add((kernel, rows, deep, parts > 1, words))
            if parts > 1 and whole:
                seen.add(("last round", rows, parts, words))
    for words in (True, False):
        assert {(ROWS, u, words) for u in (1, 2, 4)} <= seen
        assert {(BATCH, rows, words) for rows in (32, 64)} <= seen
        assert {(TILES, rows, True, shared, words) for rows in (64, 128) for shared in (True, False)} <= seen
        assert {(TILES, rows, False, False, words) for rows in (64, 128, 256)} <= seen
        assert (TILES, 256, False, True, words) in seen
    assert {("last round", 128, 3, words) for words in (True, False)} <= seen
    assert ("last round", 128, 2, True) in seen


def test_few_rows_fit_lds(plan):
    """16 rows of 6144, one of 2^20 / 9 and so on: codes and scales within 64 KiB."""
    for m in range(1, 17):
        k = 32
        while plan.fits(m, k):
            k += 32
        blocks = k // 32
        assert m * (blocks * 16 + 16 + (blocks + 15) // 16 * 16) > 64 * 1024
        assert form(plan, m, 64, k)[0] != ROWS and form(plan, m, 64, k - 32)[0] == ROWS
    assert not plan.fits(17, 32)


def test_parts_have_a_run_and_a_place_each(plan):
    for m in (17, 65, 300, 900, 1700, 5000):
        for n in (16, 130, 2330, 16530, 40000):
            for k in (32, 512, 544, 4096, 8224, 100000):
                kernel, rows, parts, deep, whole = form(plan, m, n, k)
                columns = 256 if rows == 256 else 128
                tiles = -(-m // rows) * -(-n // columns)
                assert deep == (kernel == TILES and rows < 256 and tiles * parts <= 256)
                if kernel == TILES:
                    assert whole == tiles if parts == 1 else whole % 256 == 0 and whole < tiles
                if parts > 1:
                    shared = tiles - whole
                    assert kernel == TILES and parts <= -(-k // 512) and shared <= COUNTERS
                    assert shared * parts * rows * columns * 4 <= SCRATCH
                assert form(plan, m, n, k, 0, 0)[2] == 1   # without scratch nothing is shared
