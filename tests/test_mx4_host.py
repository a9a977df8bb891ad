"""Packing of rows into blocks of 32 e2m1 numbers on the host; no GPU."""
import numpy as np
import pytest

import karume_amd
import mx4_reference as ref


def rows_of_every_kind():
    """Values next to and at every border, at several scales, with signs, zeros and subnormals."""
    borders = np.array([0.25, 0.5, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.999], dtype=np.float32)
    near = np.concatenate([borders, np.nextafter(borders, np.float32(0)), np.nextafter(borders, np.float32(9))])
    out = []
    for power in (-149, -140, -127, -126, -125, -60, -3, 0, 5, 100, 125):
        for top in (4.0, 5.0, 6.0, 6.5, 7.5):
            block = np.zeros((3, 32), dtype=np.float64)
            block[:, :11] = near.reshape(3, 11) * (1 - 2 * (np.arange(11) % 2))
            block[:, 11] = top
            block = np.where(np.abs(block) > top, top / 2, block)
            with np.errstate(over="ignore"):
                out.append(np.ldexp(block, power).astype(np.float32))
    rng = np.random.default_rng(3)
    out.append((rng.standard_normal((40, 32)) * np.exp(3 * rng.standard_normal((40, 1)))).astype(np.float32))
    out.append(np.zeros((2, 32), dtype=np.float32))
    rows = np.concatenate(out)
    return rows[np.isfinite(rows).all(1)]


@pytest.mark.parametrize("ceil", [False, True])
def test_packing_follows_the_definition(ceil):
    rows = rows_of_every_kind()
    codes, scales = karume_amd.pack_mx4(rows, ceil=ceil)
    want_codes, want_scales = ref.quantised(rows, ceil)
    assert np.array_equal(scales, want_scales) and np.array_equal(codes, want_codes)
    if ceil:   # nothing is clipped: off by half of the largest spacing at most
        v = ref.values(codes, scales)
        assert (np.abs(v - rows) <= np.exp2(scales.astype(np.float64) - 127)).all()


def test_blocks_that_hold_no_number():
    rows = np.ones((4, 96), dtype=np.float32)
    rows[0, 40], rows[1, 0], rows[2, 95] = np.nan, np.inf, -np.inf
    codes, scales = karume_amd.pack_mx4(rows)
    assert scales.tolist() == [[125, 255, 125], [255, 125, 125], [125, 125, 255], [125, 125, 125]]
    assert not codes[0, 16:32].any() and not codes[1, :16].any() and not codes[2, 32:].any()
    assert codes[3].tolist() == [0x66] * 48


def test_a_negative_that_rounds_to_zero_keeps_its_sign():
    rows = np.zeros((1, 32), dtype=np.float32)
    rows[0, :4] = 4.0, -0.25, -0.0, 0.25
    codes, scales = karume_amd.pack_mx4(rows)
    assert scales.tolist() == [[127]] and codes[0, :2].tolist() == [0x86, 0x08]


@pytest.mark.parametrize("shape", [(32,), (2, 31), (2, 0), (1, 2, 32)])
def test_rows_that_are_no_blocks_are_refused(shape):
    with pytest.raises(karume_amd.Mx4Error):
        karume_amd.pack_mx4(np.zeros(shape, dtype=np.float32))


def test_reference_products_see_a_lost_block():
    """The bound that the GPU tests use would not hide a block of 32 that a kernel leaves out."""
    rng = np.random.default_rng(5)
    x, w = rng.standard_normal((4, 4096)), rng.standard_normal((8, 4096)) * 0.02
    xv, wv = ref.values(*ref.quantised(x, False)), ref.values(*ref.quantised(w, False))
    want, off = ref.product(xv, wv, None, None, False, "f32")
    xv[:, 4064:] = 0
    assert (np.abs(xv @ wv.T - want) > off).mean() > 0.9
