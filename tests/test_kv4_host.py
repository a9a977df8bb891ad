"""The paged 4-bit cache and the rotary frequencies, as far as no device is needed: the layout and the
checks of kv4_plan.h asked of the header itself, the reference's own two ways of packing, the stretched
frequencies against their definitions."""
import ctypes as C
import math
import os
import shutil
import subprocess

import numpy as np
import pytest

import karume_amd as ka
import kv4_reference as ref
from karume_amd import _ffi, build

SHIM = """
#include "kv4_plan.h"
using namespace krm;
extern "C" void offsets(uint32_t depth, uint32_t group, uint32_t page_rows, uint32_t row, uint32_t word, uint32_t g,
                        uint32_t* out) {
  const Kv4Layout l{depth, group, page_rows, 3};
  out[0] = l.key_word(row, word); out[1] = l.key_param(row, g); out[2] = l.value_word(row, word);
  out[3] = l.value_param(row, g); out[4] = l.block(); out[5] = (uint32_t)l.page();
}
extern "C" int sequence(int32_t cu0, int32_t cu1, int32_t len, const uint32_t* limits, int32_t* rows) {
  const Kv4Sequence s = kv4_sequence(cu0, cu1, len, {limits[0], limits[1], limits[2], limits[3], limits[4]});
  *rows = s.rows;
  return s.ok;
}
extern "C" int32_t first_column(int32_t position, uint32_t window) { return kv4_first_column(position, window); }
extern "C" int shape(const uint32_t* w, char* why) {
  return kv4_shape_ok({w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7], w[8], w[9]}, why, 128);
}
extern "C" void blocks(uint64_t pairs, uint32_t share, uint32_t of, int32_t len, uint32_t window, uint32_t grain,
                       uint32_t* out) {
  const Kv4Blocks b = kv4_blocks(pairs, share, of, len, window, grain);
  out[0] = b.blocks; out[1] = b.first; out[2] = b.step;
}
extern "C" int64_t lost_block(uint32_t blocks, uint32_t first, uint32_t step) {   // the first unit found in a wrong one
  const Kv4Blocks b{blocks, first, step};
  for (uint32_t i = 0; i < blocks; ++i) {
    const uint32_t at = b.before(i), last = at + b.of(i) - 1;
    if (b.block_at(at) != i) return at;
    if (b.block_at(last) != i || b.block_at(at + b.of(i) / 2) != i) return last;
  }
  return b.before(blocks) == b.all() ? -1 : -2;
}
// The pieces of all runs, one after the other: run, block, from, to, parts, first run.
extern "C" int deal(const uint32_t* width, int blocks, uint32_t runs, uint32_t least, uint32_t begin, uint32_t snap,
                    uint32_t* out) {
  uint32_t total = 0, n = 0;
  for (int i = 0; i < blocks; ++i) total += width[i];
  uint32_t per = (total + runs - 1) / runs;
  if (per < least) per = least;
  for (uint32_t g = 0; g < runs; ++g) {
    Kv4Run r{per, g * per < total ? g * per : total, 0, begin, snap, 0, 1};
    r.end = r.at + per < total ? r.at + per : total;
    while (r.at < r.end) {
      uint32_t at = 0, i = 0;
      while (at + width[i] <= r.at) at += width[i++];
      Kv4Cut c;
      const Kv4Dealt dealt = kv4_cut(r, at, width[i], c);
      if (dealt == kRunEnds) break;
      if (dealt == kBlockSkipped) continue;
      const uint32_t piece[6] = {g, i, c.from, c.to, c.parts, c.first};
      for (uint32_t x : piece) out[n++] = x;
    }
  }
  return (int)n / 6;
}
extern "C" uint32_t tile(uint32_t begin, uint32_t even, uint32_t unit, uint32_t width, uint32_t tiles, uint32_t grain,
                         uint32_t of) {
  return kv4_tile({1, 0, 0, begin, 1, even, 0}, unit, width, tiles, grain, of);
}
extern "C" int turn(uint32_t depth, uint32_t rotary, int32_t layout, uint32_t rows, uint32_t width, char* why) {
  return kv4_turn_ok(depth, rotary, layout, rows, width, why, 128);
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no compiler")
    at = tmp_path_factory.mktemp("kv4")
    (at / "shim.cpp").write_text(SHIM)
    library = os.path.join(at, "shim.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-Wno-format-security", "-shared", "-fPIC", "-I",
                    build.CSRC, str(at / "shim.cpp"), "-o", library], check=True)
    return C.CDLL(library)


@pytest.mark.parametrize("depth,group,page", [(64, 32, 16), (128, 32, 64), (128, 128, 256), (256, 64, 32)])
def test_header_places_rows_where_the_layout_says(plan, depth, group, page):
    lay, out = ref.Layout(3, depth, group, page), (C.c_uint32 * 6)()
    raw = np.zeros((1, lay.page_bytes), dtype=np.uint8)
    rng = np.random.default_rng(depth + page)
    for row in {0, 1, 5, page - 1}:
        for word in {0, 3, 4, depth // 8 - 1}:
            g = word * 8 // group
            plan.offsets(depth, group, page, row, word, g, out)
            assert out[4] * 3 == out[5] == lay.page_bytes
            raw[:] = 0
            k, v = (tuple(np.zeros(n, t) for n, t in ((depth, np.uint8), (depth // group, np.float16),
                                                      (depth // group, np.float16))) for _ in range(2))
            codes = rng.integers(1, 16, size=8).astype(np.uint8)
            k[0][8 * word:8 * word + 8] = v[0][8 * word:8 * word + 8] = codes
            k[1][g], k[2][g], v[1][g], v[2][g] = 1.5, -2.5, 3.5, -4.5
            lay.write(raw, 0, row, 1, k, v)
            block = raw[0, out[4]:2 * out[4]]
            word_of = lambda at: int(block[at:at + 4].view(np.uint32)[0])  # noqa: E731
            half = lambda at: float(block[at:at + 2].view(np.float16)[0])  # noqa: E731
            assert [(word_of(out[0]) >> (4 * ((e & 1) * 4 + e // 2))) & 15 for e in range(8)] == codes.tolist()
            assert [(word_of(out[2]) >> (4 * e)) & 15 for e in range(8)] == codes.tolist()
            assert (half(out[1]), half(out[1] + 2)) == (1.5, -2.5)
            assert (half(out[3]), half(out[3] + 8)) == (3.5, -4.5)
            assert np.count_nonzero(raw) == np.count_nonzero(block)


def test_packing_all_rows_equals_packing_them_one_by_one():
    rng = np.random.default_rng(4)
    lay = ref.Layout(2, 64, 32, 16)
    x = rng.normal(size=(2, 2, 2, 16, 64)).astype(np.float32)
    k, v = ref.quantised(x[0], 32), ref.quantised(x[1], 32)
    raw = np.zeros((2, lay.page_bytes), np.uint8)
    ref.pack_all(lay, lay.pages(raw), k, v)
    one = np.zeros_like(raw)
    for p in range(2):
        for h in range(2):
            for r in range(16):
                lay.write(one, p, r, h, *(tuple(a[p, h, r] for a in t) for t in (k, v)))
    assert np.array_equal(raw, one)
    got_k, got_v = lay.values(raw, [0, 1])
    for got, (codes, step, minimum), given in ((got_k, k, x[0]), (got_v, v, x[1])):
        stands = codes * np.repeat(step.astype(np.float64), 32, -1) + np.repeat(minimum.astype(np.float64), 32, -1)
        got = got.reshape(2, 2, 16, 64).transpose(1, 0, 2, 3)
        assert np.array_equal(got, stands)
        # half a step, and the f32 roundings of the difference and the quotient
        assert np.all(np.abs(stands - given) <= np.repeat(step.astype(np.float64), 32, -1) * (0.5 + 16 * 2.0**-23))


def test_quantiser_covers_a_group_from_end_to_end():
    for x in (np.full(32, 0.1), np.linspace(-3, 7.7, 32), np.r_[np.zeros(31), 1e-7], np.r_[np.zeros(31), -1e-9],
              np.r_[np.full(31, -32640.0), 32640.0]):
        x = x.astype(np.float32)[None]
        codes, step, minimum = ref.quantised(x, 32)
        low, s = float(minimum[0, 0]), float(step[0, 0])
        assert low <= x.min() and low + 15 * s >= x.max() and np.isfinite(np.float16(low + 15 * s))
        assert np.all(np.abs(low + s * codes - x) <= s * (0.5 + 16 * 2.0**-23))
    for bad in (np.nan, np.inf, -np.inf, 32641.0):
        codes, step, minimum = ref.quantised(np.r_[np.ones(31), bad].astype(np.float32)[None], 32)
        assert np.isnan(step[0, 0]) and not codes.any()


LIMITS = (100, 20, 500, 10, 64)   # rows in all, rows a sequence, columns, pages a sequence, rows a page


@pytest.mark.parametrize("words,ok,rows", [
    ((0, 1, 1), 1, 1), ((0, 20, 20), 1, 20), ((80, 100, 500), 1, 20), ((5, 5, -7), 1, 0), ((100, 100, 0), 1, 0),
    ((0, 0, 2**31 - 1), 1, 0),
    ((-1, 1, 5), 0, 0), ((3, 2, 5), 0, 0), ((99, 101, 5), 0, 0), ((0, 21, 50), 0, 21), ((0, 2, 1), 0, 2),
    ((0, 1, 501), 0, 1), ((0, 1, 0), 0, 1), ((0, 1, -5), 0, 1), ((-2**31, 2**31 - 1, 5), 0, 0),
    ((0, 1, 2**31 - 1), 0, 1)])
def test_a_sequence_whose_words_break_the_limits_is_refused(plan, words, ok, rows):
    got = C.c_int32(-9)
    assert plan.sequence(*words, (C.c_uint32 * 5)(*LIMITS), C.byref(got)) == ok
    assert got.value == rows


def test_a_sequence_ends_where_its_table_does(plan):
    got = C.c_int32()
    limits = lambda pages: (C.c_uint32 * 5)(100, 20, 2**31 - 1, pages, 64)  # noqa: E731
    assert plan.sequence(0, 1, 640, limits(10), C.byref(got)) == 1
    assert plan.sequence(0, 1, 641, limits(10), C.byref(got)) == 0
    assert plan.sequence(0, 1, 2**31 - 1, limits(2**31 - 1), C.byref(got)) == 1   # the product passes 32 bits


@pytest.mark.parametrize("runs,least,begin,snap", [(256, 1, 0, 1), (256, 32, 32, 48), (8, 32, 32, 48), (5, 3, 2, 3),
                                                   (256, 1, 1, 1), (7, 1, 0, 4)])
@pytest.mark.parametrize("seed", range(12))
def test_runs_of_work_cover_every_block_once(plan, runs, least, begin, snap, seed):
    """Pieces join up to whole blocks, each cut block's in neighbouring runs, one a run; a run begins a cut block with its
    last piece and goes on with one in its first, so that two places a run hold all parts."""
    rng = np.random.default_rng(seed)
    most = (3, 40, 900, 5000)[seed % 4]
    width = (rng.integers(1, most + 1, size=rng.integers(1, 400)) + begin).astype(np.uint32)
    if seed % 3 == 0:
        width[rng.integers(len(width))] = 100000
    out = np.zeros((runs + len(width) + 8, 6), np.uint32)
    n = plan.deal(width.ctypes.data_as(C.c_void_p), len(width), runs, least, begin, snap,
                  out.ctypes.data_as(C.c_void_p))
    pieces, places = [tuple(map(int, p)) for p in out[:n]], set()
    for block, w in enumerate(width):
        mine = [p for p in pieces if p[1] == block]
        assert mine[0][2] == 0 and mine[-1][3] == w and all(a[3] == b[2] for a, b in zip(mine, mine[1:]))
        assert all(p[2] < p[3] and p[4] == len(mine) for p in mine)
        if len(mine) > 1:
            assert [p[0] for p in mine] == list(range(mine[0][5], mine[0][5] + len(mine)))
            assert all(p[5] == mine[0][5] and min(p[3] - p[2], w - p[3] or w) >= min(snap, w) // 2 for p in mine)
            for i, p in enumerate(mine):
                place = 2 * p[0] + (i == 0)
                assert place not in places
                places.add(place)
                of_run = [x for x in pieces if x[0] == p[0]]
                assert of_run[-1 if i == 0 else 0] == p
    # no run has more than its share and what the two ends move
    per = max(-(-int(width.sum()) // runs), least)
    for g in range(runs):
        assert sum(p[3] - p[2] for p in pieces if p[0] == g) <= per + 2 * snap


@pytest.mark.parametrize("blocks,first,step", [(1, 7, 0), (1, 1, 5), (300, 5, 0), (4000, 1, 1), (64, 16, 8),
                                               (20000, 3, 10), (2**15, 1, 3), (46000, 1, 2), (1500, 1400000, 3),
                                               (2, 2**30 - 5, 1)])
def test_every_unit_is_found_in_its_block(plan, blocks, first, step):
    assert blocks * first + step * blocks * (blocks - 1) // 2 < 2**31
    plan.lost_block.restype = C.c_int64
    assert plan.lost_block(blocks, first, step) == -1


@pytest.mark.parametrize("pairs,share,of,length,window,grain", [
    (1, 1, 256, 1, 0, 2), (2048, 4, 256, 1024, 0, 2), (4096, 8, 128, 9000, 0, 2), (700, 7, 256, 150, 0, 2),
    (1040, 4, 256, 700, 100, 2), (4096, 8, 256, 512, 5000, 2), (2**20, 64, 256, 2**20, 0, 4), (640, 1, 128, 640, 1, 2)])
def test_blocks_count_the_columns_that_their_rows_see(plan, pairs, share, of, length, window, grain):
    out = (C.c_uint32 * 3)()
    plan.blocks(C.c_uint64(pairs), share, of, length, window, grain, out)
    blocks, first, step = out
    assert blocks == -(-pairs // of)
    rows = pairs // share
    for b in range(blocks):
        last = min((b + 1) * of, pairs) - 1
        seen = length - rows + last // share + 1
        if window:
            seen = min(seen, window + last // share - b * of // share)
        units = first + b * step
        # at least one; rounding loses less than a unit and a row a block; a window's blocks are all taken for the widest
        assert units >= 1 and units <= ((length + of) >> grain) + 1
        if not window:
            assert (seen - (b + 1) * (1 + (1 << grain))) >> grain <= units <= ((seen + of) >> grain) + 1
        else:
            assert units * 2**grain >= min(seen, window)


def test_tiles_of_the_parts_of_a_block(plan):
    for tiles in (1, 2, 7, 64, 10**6):
        for parts in (1, 2, 3, 8, 256):   # equal parts
            at = [plan.tile(0, 1, u, parts, tiles, 2, 64) for u in range(parts + 1)]
            assert at[0] == 0 and at[-1] == tiles and all(0 <= b - a <= -(-tiles // parts) + 1 for a, b in zip(at, at[1:]))
    for begin in (0, 32):   # units of four columns, 16 a tile, behind what beginning counts as
        width = 16 * 10 + begin + 3
        at = [plan.tile(begin, 0, u, width, 11, 2, 64) for u in range(width + 1)]
        assert at[0] == 0 and at[-1] == 11 and at == sorted(at) and at[begin + 16] == 1 and at[begin + 159] == 9
    assert plan.tile(0, 0, 2**31 - 2, 2**31 - 1, 2**25, 2, 64) == 2**25


def test_first_column_of_a_window(plan):
    assert [plan.first_column(p, w) for p, w in ((0, 0), (9, 0), (9, 1), (9, 4), (9, 10), (9, 11),
                                                 (2**31 - 1, 0xffffffff))] == [0, 0, 9, 6, 0, 0, 0]


GOOD = dict(nseq=2, max_query=3, total_rows=5, heads=8, kv_heads=2, depth=128, group=32, page_rows=16, pages=9,
            table_stride=4)


@pytest.mark.parametrize("change,ok", [
    ({}, 1), ({"depth": 64, "group": 64}, 1), ({"depth": 256, "group": 128, "page_rows": 256}, 1),
    ({"heads": 2}, 1), ({"total_rows": 0, "max_query": 0, "nseq": 0}, 1),
    ({"depth": 96}, 0), ({"depth": 512}, 0), ({"depth": 64, "group": 128}, 0), ({"group": 16}, 0), ({"group": 0}, 0),
    ({"page_rows": 8}, 0), ({"page_rows": 512}, 0), ({"page_rows": 48}, 0), ({"page_rows": 0}, 0),
    ({"heads": 7}, 0), ({"heads": 0}, 0), ({"kv_heads": 0}, 0), ({"heads": 65536, "kv_heads": 1}, 0),
    ({"max_query": 6}, 1), ({"nseq": 65536}, 0), ({"max_query": 0}, 0), ({"total_rows": 2**31}, 0),
    ({"pages": 0}, 0), ({"pages": 2**31}, 0), ({"table_stride": 0}, 0), ({"table_stride": 2**31}, 0)])
def test_shapes_are_checked(plan, change, ok):
    words = (C.c_uint32 * 10)(*{**GOOD, **change}.values())
    why = C.create_string_buffer(128)
    assert plan.shape(words, why) == ok, why.value
    assert bool(why.value) != bool(ok)


@pytest.mark.parametrize("words,ok", [((128, 128, 0, 1, 64), 1), ((128, 2, 1, 1, 1), 1), ((128, 0, 0, 0, 0), 1),
                                      ((128, 130, 0, 9, 65), 0), ((128, 3, 0, 9, 9), 0), ((128, 64, 2, 9, 32), 0),
                                      ((128, 64, -1, 9, 32), 0), ((128, 64, 0, 0, 32), 0), ((128, 64, 0, 9, 31), 0)])
def test_rotations_are_checked(plan, words, ok):
    assert plan.turn(*words, C.create_string_buffer(128)) == ok


def test_sizes_need_no_device_and_refuse_with_a_reason():
    lib, size = _ffi.load(), C.c_size_t()
    assert lib.krm_kv4_page_bytes(8, 128, 32, 64, C.byref(size)) == 0
    assert size.value == ref.Layout(8, 128, 32, 64).page_bytes == 8 * 64 * 2 * (64 + 16)
    assert lib.krm_kv4_page_bytes(8, 96, 32, 64, C.byref(size)) == -1 and b"depth 96" in lib.krm_last_error(None)
    assert lib.krm_kv4_page_bytes(8, 128, 32, 64, None) == -1
    assert lib.krm_kv4_attention_workspace(4, 1, 4096, 4, 32, 8, 128, 0, ka.F16, C.byref(size)) == 0
    assert lib.krm_kv4_attention_workspace(4, 1, 4096, 4, 30, 8, 128, 0, ka.F16, C.byref(size)) == -1
    assert b"heads 30" in lib.krm_last_error(None)
    assert lib.krm_kv4_attention_workspace(4, 1, 4096, 4, 32, 8, 128, 0, 7, C.byref(size)) == -1


def test_frequencies():
    plain, amplitude = ka.rope_frequencies(64, 10000.0)
    assert amplitude == 1.0 and plain.dtype == np.float64
    np.testing.assert_allclose(plain, [10000.0 ** (-2 * j / 64) for j in range(32)], rtol=1e-14)
    linear, _ = ka.rope_frequencies(64, scaling="linear", factor=4.0)
    np.testing.assert_allclose(linear, plain / 4, rtol=1e-15)
    base, _ = ka.rope_frequencies(64, scaling="base", factor=4.0)
    assert base[0] == 1.0 and base[-1] == pytest.approx(plain[-1] / 4, rel=1e-12)
    assert np.all(np.diff(plain / base) > 0)


def test_frequencies_by_wavelength_and_by_index():
    plain, _ = ka.rope_frequencies(128, 500000.0)
    got, amplitude = ka.rope_frequencies(128, 500000.0, scaling="wavelength", factor=8.0, trained=8192, slow=1.0,
                                         fast=4.0)
    turns = 8192 * plain / (2 * math.pi)
    assert amplitude == 1.0
    assert np.array_equal(got[turns >= 4], plain[turns >= 4])
    np.testing.assert_allclose(got[turns <= 1], plain[turns <= 1] / 8, rtol=1e-15)
    between = (turns > 1) & (turns < 4)
    assert between.any() and np.all((got < plain)[between] & (got > plain / 8)[between])
    assert np.all(np.diff(got) < 0)
    got, amplitude = ka.rope_frequencies(128, 10000.0, scaling="ramp", factor=16.0, trained=4096)
    plain, _ = ka.rope_frequencies(128, 10000.0)
    turns = 4096 * plain / (2 * math.pi)
    assert amplitude == pytest.approx(0.1 * math.log(16) + 1)
    assert np.all(got[:np.argmax(turns < 32) - 1] == plain[:np.argmax(turns < 32) - 1])
    last = np.argmax(turns < 1)
    np.testing.assert_allclose(got[last + 1:], plain[last + 1:] / 16, rtol=1e-15)
    assert np.all(np.diff(got) < 0)


@pytest.mark.parametrize("arguments", [dict(rotary_dim=0), dict(rotary_dim=63), dict(rotary_dim=64, base=1.0),
                                       dict(rotary_dim=64, base=math.nan), dict(rotary_dim=64, factor=0.5),
                                       dict(rotary_dim=64, scaling="ramp"), dict(rotary_dim=64, scaling="other"),
                                       dict(rotary_dim=64, scaling="wavelength", trained=9, slow=4.0, fast=1.0),
                                       dict(rotary_dim=2, scaling="base", factor=2.0)])
def test_frequencies_refuse(arguments):
    with pytest.raises(ValueError):
        ka.rope_frequencies(**arguments)
