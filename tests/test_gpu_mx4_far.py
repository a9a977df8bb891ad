"""Products and rows of mx4 codes whose rows are very long, whose bytes pass 2^32, or whose scales are at their ends."""
import numpy as np
import pytest

import karume_amd as ka
import mx4_reference as ref
from test_gpu_mx4 import CODE, Guarded, guarded

pytestmark = pytest.mark.gpu


def codes(rng, rows, k):
    return rng.integers(0, 256, (rows, k // 2), dtype=np.uint8), rng.integers(120, 127, (rows, k // 32), dtype=np.uint8)


def expected(x, w, k):
    xv, wv = ref.values(*x), ref.values(*w).T
    return xv @ wv, (k / 32 + 64) * 2.0 ** -24 * (np.abs(xv) @ np.abs(wv))


def repeated(gpu, array, times):
    """The array's bytes `times` times over, one behind the other."""
    buf = gpu.alloc(array.nbytes * times)
    buf.upload(array)
    have = 1
    while have < times:
        more = min(have, times - have)
        gpu.copy(buf.offset(have * array.nbytes), int(buf), more * array.nbytes)
        have += more
    return buf


@pytest.mark.parametrize("m,n,k", [(1, 34, 1 << 18), (2, 34, (1 << 20) + 32), (40, 18, (1 << 19) + 32), (70, 34, (1 << 18) + 32),
                                   (300, 18, 1 << 18), (1, 2, 1 << 24), (65, 2, 1 << 21)])
def test_long_rows(gpu_ctx, m, n, k):
    rng = np.random.default_rng(k + m)
    x, w = codes(rng, m, k), codes(rng, n, k)
    want, off = expected(x, w, k)
    args = [int(guarded(gpu_ctx, a)) for a in (*x, *w)]
    for out in ("f32", "f16"):
        held = Guarded(gpu_ctx, m * n * ref.NUMPY[out]().nbytes)
        gpu_ctx.linear_mx4(*args, int(held), m, n, k, out_dtype=CODE[out])
        with np.errstate(over="ignore"):
            most = np.abs(want) < 65000
            got = np.where(most, held.read(ref.NUMPY[out], (m, n)), 0).astype(np.float64)
        ref.check(got, np.where(most, want, 0), off + ref.HALF_STEP[out] * np.abs(want) + ref.TINY_STEP[out], (m, n, k, out))


@pytest.mark.parametrize("m", [3, 40, 130, 600])
def test_weights_past_32_bits(gpu_ctx, m):
    """Rows of w that repeat: so do the results, to the last bit."""
    rng = np.random.default_rng(m)
    k, period, times = 1 << 16, 512, 272                       # 139264 rows, 4.25 GiB
    x, w = codes(rng, m, k), codes(rng, period, k)
    n = period * times
    held = repeated(gpu_ctx, w[0], times), repeated(gpu_ctx, w[1], times)
    out = gpu_ctx.zeros(m * n * 4)
    gpu_ctx.linear_mx4(gpu_ctx.upload(x[0]), gpu_ctx.upload(x[1]), *held, out, m, n, k)
    got = out.download(np.float32, (m, times, period))
    want, off = expected(x, w, k)
    ref.check(got[:, -1], want, off + ref.HALF_STEP["f32"] * np.abs(want), m)
    assert np.array_equal(got, np.broadcast_to(got[:, -1:], got.shape))
    for buf in (*held, out):
        buf.free()


def test_results_past_32_bits(gpu_ctx):
    rng = np.random.default_rng(9)
    k, n, period, times = 64, 16384, 512, 140                  # 71680 rows of 64 KiB
    x, w = codes(rng, period, k), codes(rng, n, k)
    m = period * times
    held = repeated(gpu_ctx, x[0], times), repeated(gpu_ctx, x[1], times)
    dw = gpu_ctx.upload(w[0]), gpu_ctx.upload(w[1])
    want, off = expected(x, w, k)
    for out, pairs in (("f32", False), ("f16", True)):
        width, t = n // (2 if pairs else 1), ref.NUMPY[out]
        result = gpu_ctx.zeros(m * width * t().nbytes)
        gpu_ctx.linear_mx4(*held, *dw, result, m, n, k, out_dtype=CODE[out],
                           epilogue=ka.EPILOGUE_SILU_PAIRS if pairs else ka.EPILOGUE_NONE)
        tail = result.download(np.uint8, (period * width * t().nbytes,), (times - 1) * period * width * t().nbytes)
        first = result.download(np.uint8, tail.shape)
        assert np.array_equal(tail, first)
        if not pairs:
            ref.check(tail.view(t).reshape(period, n), want, off + ref.HALF_STEP[out] * np.abs(want))
        result.free()
    for buf in held:
        buf.free()


def test_rows_past_32_bits_are_quantised_and_read_back(gpu_ctx):
    rng = np.random.default_rng(4)
    dim, period, times = 1 << 15, 256, 144                     # 36864 rows of 128 KiB
    x = rng.standard_normal((period, dim)).astype(np.float32)
    dx = repeated(gpu_ctx, x, times)
    rows = period * times
    dc, ds, back = gpu_ctx.zeros(rows * dim // 2), gpu_ctx.zeros(rows * dim // 32), gpu_ctx.zeros(rows * dim * 4)
    gpu_ctx.quantize_mx4(dx, dc, ds, rows=rows, dim=dim)
    gpu_ctx.dequant_mx4(dc, ds, back, rows=rows, dim=dim)
    want = ka.pack_mx4(x)
    last = (times - 1) * period * dim
    assert np.array_equal(dc.download(np.uint8, want[0].shape, last // 2), want[0])
    assert np.array_equal(ds.download(np.uint8, want[1].shape, last // 32), want[1])
    assert np.array_equal(back.download(np.float32, x.shape, last * 4), ref.values(*want).astype(np.float32))
    weight = gpu_ctx.upload(np.ones(1 << 14, dtype=np.float32))
    gpu_ctx.block_norm(dx, rows=rows * 2, dim=1 << 14, residual=back, pre_weight=weight, sum_out=back, norm_out=dx)
    a, b = x.reshape(-1, 1 << 14).astype(np.float64), ref.values(*want).reshape(-1, 1 << 14)
    first, second = ref.block_norm(a, None, None, False, b, np.ones(1 << 14), np.float64(np.float32(1e-5)), 1.0, 1.0, "f32", "f32")
    ref.check(back.download(np.float32, a.shape, last * 4), *first)
    ref.check(dx.download(np.float32, a.shape, last * 4), *second)
    for buf in (dx, dc, ds, back):
        buf.free()


@pytest.mark.parametrize("m", [1, 40, 300])
@pytest.mark.parametrize("largest", [(254, 254), (254, 0), (200, 200)])
def test_zeros_at_any_scale_add_nothing(gpu_ctx, m, largest):
    """Blocks of zeros whose two scales together pass f32's range, beside blocks of numbers."""
    rng = np.random.default_rng(m)
    n, k = 64, 256
    x, w = codes(rng, m, k), codes(rng, n, k)
    x[0][:, :16], w[0][:, 16:32], x[0][:, 32:48] = 0, 0x80, 0x08      # zeros of either sign
    for block in range(3):
        x[1][:, block], w[1][:, block] = largest
    want, off = expected((x[0], np.where(np.arange(k // 32) < 3, 127, x[1]).astype(np.uint8)),
                         (w[0], np.where(np.arange(k // 32) < 3, 127, w[1]).astype(np.uint8)), k)
    held = Guarded(gpu_ctx, m * n * 4)
    gpu_ctx.linear_mx4(*(int(guarded(gpu_ctx, a)) for a in (*x, *w)), int(held), m, n, k)
    ref.check(held.read(np.float32, (m, n)), want, off + ref.HALF_STEP["f32"] * np.abs(want), (m, largest))
