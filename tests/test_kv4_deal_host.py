"""What counts as a launch's work when the paged attention splits its columns (kv4_plan.h).  Host code; no GPU."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

from karume_amd import _ffi, build

SHIM = """
#include "kv4_plan.h"
extern "C" float tiles(uint32_t rows, int32_t len, const uint32_t* w) {
  return krm::kv4_tiles(rows, len, w[0], w[1], w[2], 16, w[3], 5000, 32);
}
"""


@pytest.fixture(scope="module")
def tiles(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no compiler")
    at = tmp_path_factory.mktemp("deal")
    (at / "shim.cpp").write_text(SHIM)
    library = os.path.join(at, "shim.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-Wno-format-security", "-shared", "-fPIC", "-I",
                    build.CSRC, str(at / "shim.cpp"), "-o", library], check=True)
    call = C.CDLL(library).tiles
    call.restype = C.c_float
    return lambda rows, length, share=4, least=0, most=0xffffffff, window=0: call(
        rows, length, (C.c_uint32 * 4)(share, least, most, window))


@pytest.mark.parametrize("rows,length,share,window,want", [
    (1, 1, 4, 0, 1), (1, 31, 4, 0, 1), (1, 32, 4, 0, 2), (1, 5000, 4, 0, 157), (1, 5000, 16, 0, 157), (1, 5000, 17, 0, 2 * 157),
    (4, 640, 4, 0, 21), (5, 640, 4, 0, 2 * 21), (40, 640, 8, 0, 20 * 21), (1, 5000, 4, 512, 17), (1, 300, 4, 512, 10),
    (1, 300, 4, 0xffffffff, 10), (9, 5000, 4, 1, 3)])
def test_a_sequence_counts_with_the_columns_and_blocks_it_has(tiles, rows, length, share, window, want):
    assert tiles(rows, length, share, window=window) == want


@pytest.mark.parametrize("length", [5000, 0, -1, 2**31 - 1, -2**31])
@pytest.mark.parametrize("least", [0, 33])
def test_entries_without_rows_count_nothing(tiles, length, least):
    assert tiles(0, length, least=least) == 0


@pytest.mark.parametrize("rows,least,most,counts", [(8, 0, 32, True), (9, 0, 32, False), (8, 33, 0xffffffff, False),
                                                    (9, 33, 0xffffffff, True)])
def test_the_other_launch_s_sequences_count_nothing(tiles, rows, least, most, counts):
    assert (tiles(rows, 640, least=least, most=most) > 0) == counts


def test_a_refused_sequence_counts_within_the_limits(tiles):
    assert tiles(1, 2**31 - 1) == 157 and tiles(1, -5) == 1


@pytest.mark.parametrize("depth", [64, 128, 256])
@pytest.mark.parametrize("nseq,rows,share", [(64, 5, 8), (128, 8, 8), (256, 16, 4), (512, 64, 1)])
def test_many_sequences_of_up_to_64_pairs_have_blocks_of_16(depth, nseq, rows, share):
    """They need no workspace then: there are workgroups enough without a split, and the kernel for many rows, which has
    one whatever the step is, would use a quarter of its rows."""
    lib, size = _ffi.load(), C.c_size_t()
    assert lib.krm_kv4_attention_workspace(nseq, rows, 4096, nseq * rows, 8 * share, 8, depth, 0, 0, C.byref(size)) == 0
    assert size.value == 0
    assert lib.krm_kv4_attention_workspace(nseq, 4 * rows, 4096, nseq * 4 * rows, 8 * share, 8, depth, 0, 0, C.byref(size)) == 0
    assert size.value > 0


@pytest.mark.parametrize("rows", [-1, -10, -2**30, -2**31, 2**22 + 1, 2**31 - 1])
def test_rows_that_no_call_takes_count_nothing(tiles, rows):
    assert tiles(rows & 0xffffffff, 5000) == 0
