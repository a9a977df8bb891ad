"""Blocks of 32 e2m1 numbers on the GPU: quantisation, read-back, products; each result held to its own bound."""
import numpy as np
import pytest

import karume_amd as ka
import mx4_reference as ref
from test_mx4_host import rows_of_every_kind

pytestmark = pytest.mark.gpu
CODE = {"f16": ka.F16, "f32": ka.F32}
GUARD = 64   # bytes of a known value in front of and behind what a call may write


class Guarded:
    """A device buffer between two guards, at `shift` bytes past 16-byte alignment."""

    def __init__(self, gpu, nbytes, shift=0):
        self.nbytes, self.at = nbytes, GUARD + shift
        self.buf = gpu.upload(np.full(nbytes + 2 * GUARD + 16, 0xA5, dtype=np.uint8))

    def __int__(self):
        return self.buf.offset(self.at)

    def read(self, dtype, shape):
        raw = self.buf.download(np.uint8, (self.buf.nbytes,))
        assert (raw[:self.at] == 0xA5).all() and (raw[self.at + self.nbytes:] == 0xA5).all()
        return raw[self.at:self.at + self.nbytes].view(dtype).reshape(shape)

    def fill(self, array):
        self.buf.upload(array, self.at)
        return self


def guarded(gpu, array, shift=0):
    return Guarded(gpu, array.nbytes, shift).fill(array)


def activations(rng, rows, k, dtype):
    return (rng.standard_normal((rows, k)) * np.exp(0.8 * rng.standard_normal(k))).astype(dtype)


# ------------------------------------------------------------------------------------ quantisation
def quantise(gpu, x, ceil, stride=None):
    rows, dim = x.shape
    stride = dim if stride is None else stride
    held = np.full((rows, stride), np.nan, dtype=x.dtype)   # what lies between rows is not looked at
    held[:, :dim] = x
    dx = guarded(gpu, held)
    codes, scales = Guarded(gpu, rows * dim // 2), Guarded(gpu, rows * dim // 32, shift=3)
    gpu.quantize_mx4(int(dx), int(codes), int(scales), rows=rows, dim=dim, x_stride=stride,
                     x_dtype=ka.dtype_code(x.dtype), scale_rule=ka.MX4_CEIL if ceil else ka.MX4_FLOOR)
    gpu.sync()
    return codes.read(np.uint8, (rows, dim // 2)), scales.read(np.uint8, (rows, dim // 32))


@pytest.mark.parametrize("ceil", [False, True])
@pytest.mark.parametrize("io", ["f16", "f32"])
def test_borders_of_the_codes(gpu_ctx, io, ceil):
    x = rows_of_every_kind()
    if io == "f16":
        with np.errstate(over="ignore"):
            x = np.concatenate([np.ldexp(x, p).astype(np.float16) for p in (0, -10, -20, 8)])
        x = x[np.isfinite(x).all(1)]
    got = quantise(gpu_ctx, x, ceil)
    want = ref.quantised(x.astype(np.float64), ceil)
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[0], want[0])


SHAPES = [(1, 32), (1, 64), (3, 96), (7, 4096), (2, 2080), (513, 160), (70, 11008), (5, 16416), (2000, 32)]


@pytest.mark.parametrize("rows,dim", SHAPES)
@pytest.mark.parametrize("io", ["f16", "f32"])
def test_rows_are_quantised_and_read_back(gpu_ctx, rows, dim, io):
    rng = np.random.default_rng(rows * 7 + dim)
    x = activations(rng, rows, dim, ref.NUMPY[io])
    ceil = (rows + dim // 32) % 2 == 1
    codes, scales = quantise(gpu_ctx, x, ceil, dim + 8 * (dim % 64 == 0) * (rows % 3))
    want = ref.quantised(x.astype(np.float64), ceil)
    assert np.array_equal(scales, want[1]) and np.array_equal(codes, want[0])
    dc, ds = guarded(gpu_ctx, codes), guarded(gpu_ctx, scales, shift=1)
    for out in ("f32", "f16"):
        values = Guarded(gpu_ctx, rows * dim * ref.NUMPY[out]().nbytes)
        gpu_ctx.dequant_mx4(int(dc), int(ds), int(values), rows=rows, dim=dim, out_dtype=CODE[out])
        got = values.read(ref.NUMPY[out], (rows, dim))
        with np.errstate(over="ignore"):
            stands = ref.values(codes, scales).astype(ref.NUMPY[out])
        assert np.array_equal(got.view(np.uint8), stands.view(np.uint8))   # the signs of zeros among them


def test_blocks_of_no_numbers_spoil_themselves_alone(gpu_ctx):
    rng = np.random.default_rng(2)
    x = rng.standard_normal((6, 256)).astype(np.float32)
    x[0, 33], x[1, 255], x[2, 0], x[3, 128:160] = np.nan, np.inf, -np.inf, np.nan
    x[4, :32] = 0
    for io in ("f32", "f16"):
        codes, scales = quantise(gpu_ctx, x.astype(ref.NUMPY[io]), False)
        want = ref.quantised(x.astype(ref.NUMPY[io]).astype(np.float64), False)
        assert np.array_equal(scales, want[1]) and np.array_equal(codes, want[0])
        assert scales[4, 0] == 0 and (scales == 255).sum() == 4
    values = Guarded(gpu_ctx, 6 * 256 * 4)
    gpu_ctx.dequant_mx4(gpu_ctx.upload(codes), gpu_ctx.upload(scales), int(values), rows=6, dim=256)
    got = values.read(np.float32, (6, 8, 32))
    assert np.array_equal(np.isnan(got).all(-1), scales == 255) and np.isnan(got).sum() == 4 * 32


def test_every_code_at_every_scale_reads_back(gpu_ctx):
    codes = np.tile(np.arange(16, dtype=np.uint8) * 17, (256, 1))
    scales = np.arange(256, dtype=np.uint8)[:, None]
    for out in ("f32", "f16"):
        values = Guarded(gpu_ctx, 256 * 32 * ref.NUMPY[out]().nbytes)
        gpu_ctx.dequant_mx4(gpu_ctx.upload(codes), gpu_ctx.upload(scales), int(values), rows=256, dim=32,
                            out_dtype=CODE[out])
        got = values.read(ref.NUMPY[out], (256, 32))
        with np.errstate(over="ignore", invalid="ignore"):
            want = ref.values(codes, scales).astype(ref.NUMPY[out])
        assert np.array_equal(np.isnan(got), np.isnan(want))
        keep = ~np.isnan(want)
        assert np.array_equal(got[keep], want[keep])


# ---------------------------------------------------------------------------------------- products
def weights(rng, n, k):
    return ref.quantised(rng.standard_normal((n, k)) * 0.02, False)


def run_product(gpu, m, n, k, *, out="f32", io=None, pairs=False, bias=False, residual=False, in_place=False, seed=0,
                stride=None, ceil=False, shift=0, given=True, x=None, w=None):
    """The product of codes (io None) or of rows of floats, held to its bound; the raw result."""
    rng = np.random.default_rng(seed * 1009 + m * 31 + n * 7 + k)
    wq, ws = weights(rng, n, k) if w is None else w
    if x is None:
        x = activations(rng, m, k, ref.NUMPY[io or "f32"])
    xq, xs = ref.quantised(x.astype(np.float64), ceil)
    width = n // 2 if pairs else n
    b = rng.standard_normal(n).astype(np.float32) if bias else None
    r = rng.standard_normal((m, width)).astype(ref.NUMPY[out]) if residual else None
    dw, dws = guarded(gpu, wq), guarded(gpu, ws, shift=shift)
    eb = ref.NUMPY[out]().nbytes
    dout = Guarded(gpu, m * width * eb, shift=shift * eb)
    dres = None
    if r is not None:
        dres = dout.fill(r) if in_place else guarded(gpu, r, shift=shift * eb)
    kw = dict(bias=None if b is None else gpu.upload(b), residual=None if dres is None else int(dres),
              out_dtype=CODE[out], epilogue=ka.EPILOGUE_SILU_PAIRS if pairs else ka.EPILOGUE_NONE)
    if io is None:
        gpu.linear_mx4(int(guarded(gpu, xq)), int(guarded(gpu, xs, shift=shift)), int(dw), int(dws), int(dout), m, n, k,
                       **kw)
    else:
        stride = k if stride is None else stride
        held = np.full((m, stride), np.nan, dtype=x.dtype)
        held[:, :k] = x
        work = [int(Guarded(gpu, xq.nbytes)), int(Guarded(gpu, xs.nbytes, shift=shift))] if given else [None, None]
        gpu.linear_mx4_fused(int(guarded(gpu, held)), int(dw), int(dws), int(dout), m, n, k, xq=work[0], xs=work[1],
                             x_stride=stride, x_dtype=CODE[io], scale_rule=ka.MX4_CEIL if ceil else ka.MX4_FLOOR, **kw)
    got = dout.read(ref.NUMPY[out], (m, width))
    with np.errstate(invalid="ignore"):
        want, off = ref.product(ref.values(xq, xs), ref.values(wq, ws), b, None if r is None else r.astype(np.float64),
                                pairs, out)
    ref.check(got, want, off, (m, n, k, out, io, pairs))
    return got


PRODUCTS = [(1, 1, 32), (1, 16, 32), (1, 17, 64), (2, 2, 96), (1, 130, 128), (3, 33, 160), (16, 16, 512), (17, 48, 544),
            (15, 31, 4096), (1, 4096, 512), (8, 1000, 2048), (31, 257, 1056), (33, 64, 4128), (64, 200, 736),
            (65, 129, 288), (100, 514, 1024), (128, 256, 512), (129, 255, 480), (200, 130, 2080), (256, 512, 256),
            (257, 513, 1184), (300, 1030, 320), (1, 64, 16416), (16, 40, 11008), (50, 130, 1024), (17, 300, 544), (9, 100, 1568),
            (40, 5001, 2048)]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_products_of_codes(gpu_ctx, m, n, k):
    odd = (m + n + k // 32) % 2 == 1
    run_product(gpu_ctx, m, n, k, out="f16" if odd else "f32", bias=m % 3 == 1, residual=n % 3 == 1, shift=n % 2)
    run_product(gpu_ctx, m, n, k, out="f32" if odd else "f16", pairs=n % 2 == 0, residual=m % 2 == 1, in_place=True,
                bias=n % 4 == 0)


@pytest.mark.parametrize("m,n,k", PRODUCTS)
@pytest.mark.parametrize("io", ["f16", "f32"])
def test_products_of_floats_are_those_of_their_codes(gpu_ctx, m, n, k, io):
    kw = dict(out=io, pairs=n % 2 == 0, bias=True, seed=5, ceil=m % 2 == 0)
    rng = np.random.default_rng(m + n + k)
    x = activations(rng, m, k, ref.NUMPY[io])
    got = run_product(gpu_ctx, m, n, k, io=io, x=x, stride=k + 8 * (m % 3), **kw)
    same = run_product(gpu_ctx, m, n, k, x=x, **kw)
    assert np.array_equal(got.view(np.uint8), same.view(np.uint8))


# forms that only larger products take, and the same with scales that are no whole words (see test_mx4_plan.py)
LARGE = [(65, 130, 8192), (70, 130, 8224), (67, 9430, 11008), (67, 9430, 11040), (197, 17830, 11008), (197, 17830, 11040),
         (65, 16530, 64), (65, 16530, 256), (197, 12230, 64), (197, 12230, 256), (272, 20630, 64), (272, 20630, 256),
         (517, 19230, 64), (517, 19230, 256), (16, 500, 8192), (3, 200, 16384), (64, 516, 11008), (31, 300, 11040),
         (131, 22030, 6656), (197, 16430, 6656), (197, 16430, 6688)]


@pytest.mark.parametrize("m,n,k", LARGE)
def test_large_products(gpu_ctx, m, n, k):
    rng = np.random.default_rng(m + n)
    w = (rng.integers(0, 256, (n, k // 2), dtype=np.uint8), rng.integers(112, 122, (n, k // 32), dtype=np.uint8))
    kw = dict(w=w, bias=True, residual=True, out="f16" if k % 128 else "f32")
    a = run_product(gpu_ctx, m, n, k, pairs=m % 2 == 1, **kw)
    b = run_product(gpu_ctx, m, n, k, pairs=m % 2 == 1, io="f32", **kw)
    assert np.array_equal(a.view(np.uint8), b.view(np.uint8))


@pytest.mark.parametrize("m,k", [(1, 32), (1, 2048), (5, 4096), (16, 6144), (7, 544)])
@pytest.mark.parametrize("io", ["f16", "f32"])
def test_few_rows_do_without_work_buffers(gpu_ctx, m, k, io):
    run_product(gpu_ctx, m, 333, k, io=io, given=False, stride=k + 64, bias=True)
    run_product(gpu_ctx, m, 5000, k, io=io, given=False, pairs=True, out="f16")


@pytest.mark.parametrize("m", [1, 5, 40, 300])
def test_what_is_no_number_stays_in_its_row_and_column(gpu_ctx, m):
    rng = np.random.default_rng(m)
    n, k = 70, 416
    w = weights(rng, n, k)
    w[1][3, 12], w[1][69, 0] = 255, 255
    x = activations(rng, m, k, np.float32)
    x[m - 1, 77] = np.inf
    got = run_product(gpu_ctx, m, n, k, w=w, x=x)
    assert np.isnan(got[m - 1]).all() and np.isnan(got[:, [3, 69]]).all()
    assert np.isnan(got).sum() == n + 2 * (m - 1)
    run_product(gpu_ctx, m, n, k, w=w, x=x, io="f32")


@pytest.mark.parametrize("m", [1, 9, 70, 260])
def test_rows_past_the_end_of_k_do_not_reach_a_sum(gpu_ctx, m):
    """The block behind a row's last is the next row's first: here it is NaN."""
    rng = np.random.default_rng(m)
    n, k = 64, 96
    w, x = weights(rng, n, k), activations(rng, m, k, np.float32)
    w[1][1::2, 0] = 255
    x[1::2, 0] = np.nan
    got = run_product(gpu_ctx, m, n, k, w=w, x=x)
    assert not np.isnan(got[0::2, 0::2]).any()


@pytest.mark.parametrize("m", [1, 20, 200])
def test_scales_from_end_to_end(gpu_ctx, m):
    """Scales of x and w far from one whose products are in f32's range, zeros at the lowest scale."""
    rng = np.random.default_rng(m)
    n, k = 50, 512
    w = weights(rng, n, k)
    codes, scales = ref.quantised(activations(rng, m, k, np.float32).astype(np.float64), False)
    x = ref.values(codes, scales)
    w[1][:] = (w[1].astype(np.int64) + 100).clip(0, 254).astype(np.uint8)
    x = (x * 2.0 ** -100).astype(np.float32)
    x[:, 64:96] = 0
    run_product(gpu_ctx, m, n, k, w=w, x=x)
    run_product(gpu_ctx, m, n, k, w=w, x=x, io="f32")


def test_nothing_to_do(gpu_ctx):
    buf = gpu_ctx.upload(np.full(4096, 0x5A, dtype=np.uint8))
    gpu_ctx.linear_mx4(buf, buf, buf, buf, buf, 0, 16, 32)
    gpu_ctx.linear_mx4(buf, buf, buf, buf, buf, 4, 0, 32)
    gpu_ctx.linear_mx4_fused(buf, buf, buf, buf, 0, 16, 32)
    gpu_ctx.quantize_mx4(buf, buf, buf, rows=0, dim=32)
    gpu_ctx.dequant_mx4(buf, buf, buf, rows=0, dim=32)
    assert (buf.download(np.uint8, (4096,)) == 0x5A).all()


# ------------------------------------------------------------------------------- recorded, streams
def test_recorded_products_replay(gpu_ctx):
    """A quantisation and products of few and many rows, recorded once (one on a side branch) and replayed over new
    inputs with eager work between."""
    rng = np.random.default_rng(11)
    k, n = 1024, 320
    w, ws = weights(rng, n, k)
    dw, dws = gpu_ctx.upload(w), gpu_ctx.upload(ws)
    state = []
    for m in (1, 24, 300):
        x = activations(rng, m, k, np.float16)
        state.append((m, gpu_ctx.upload(x), gpu_ctx.zeros(m * k // 2), gpu_ctx.zeros(m * k // 32),
                      gpu_ctx.zeros(m * n * 4), gpu_ctx.zeros(m * n * 4)))

    def step(rec=None):
        for i, (m, x, xq, xs, out, eager) in enumerate(state):
            if rec is not None:
                rec.branch(i % 2)
            gpu_ctx.linear_mx4_fused(x, dw, dws, eager if rec is None else out, m, n, k, xq=xq, xs=xs,
                                     x_dtype=ka.F16)

    step()
    gpu_ctx.sync()
    with gpu_ctx.record() as rec:
        step(rec)
    for turn in range(4):
        for m, x, *_ in state:
            x.upload(activations(rng, m, k, np.float16))
        step()
        gpu_ctx.sync()
        rec.graph.launch()
        gpu_ctx.sync()
        for m, _, _, _, out, eager in state:
            a, b = out.download(np.float32, (m, n)), eager.download(np.float32, (m, n))
            assert np.array_equal(a, b) and np.abs(a).max() > 0, (turn, m)
    rec.graph.destroy()


def test_two_contexts_at_once(gpu_ctx):
    other = ka.acquire_gpu(0)
    try:
        rng = np.random.default_rng(4)
        m, n, k = 300, 512, 2048
        jobs = []
        for gpu in (gpu_ctx, other):
            w, ws = weights(rng, n, k)
            x = activations(rng, m, k, np.float32)
            jobs.append((gpu, w, ws, x, gpu.upload(w), gpu.upload(ws), gpu.upload(x), gpu.zeros(m * k // 2),
                         gpu.zeros(m * k // 32), gpu.zeros(m * n * 4)))
        for _ in range(4):
            for gpu, _, _, _, dw, dws, dx, xq, xs, out in jobs:
                gpu.linear_mx4_fused(dx, dw, dws, out, m, n, k, xq=xq, xs=xs)
        for gpu, w, ws, x, *_, out in jobs:
            want, off = ref.product(ref.values(*ref.quantised(x.astype(np.float64), False)), ref.values(w, ws), None, None,
                                    False, "f32")
            ref.check(out.download(np.float32, (m, n)), want, off)
    finally:
        other.destroy()


# ----------------------------------------------------------------------------------------- refusals
def test_refusals(gpu_ctx):
    buf = gpu_ctx.zeros(1 << 16)
    at = int(buf)

    def refused(call, *args, **kw):
        with pytest.raises(ka.GpuValidationError):
            call(*args, **kw)

    q = gpu_ctx.quantize_mx4
    for kw in (dict(dim=0), dict(dim=31), dict(dim=48), dict(x_dtype=7), dict(scale_rule=2), dict(x_stride=32),
               dict(x_stride=66), dict(x_stride=1 << 62)):
        refused(q, at, at + 4096, at + 8192, **{**dict(rows=2, dim=64, x_dtype=ka.F32), **kw})
    refused(q, at, at + 4096, at + 8192, rows=2, dim=64, x_stride=68, x_dtype=ka.F16)
    for args in ((0, at, at), (at, 0, at), (at, at, 0), (at + 4, at, at), (at, at + 8, at)):
        refused(q, *args, rows=2, dim=64)
    d = gpu_ctx.dequant_mx4
    for kw in (dict(dim=0), dict(dim=40), dict(out_dtype=3)):
        refused(d, at, at + 4096, at + 8192, **{**dict(rows=2, dim=64), **kw})
    for args in ((0, at, at), (at, 0, at), (at, at, 0), (at + 8, at, at), (at, at, at + 8)):
        refused(d, *args, rows=2, dim=64)
    p = gpu_ctx.linear_mx4
    for m, n, k, kw in ((2, 4, 0, {}), (2, 4, 48, {}), (2, 3, 64, dict(epilogue=1)), (2, 4, 64, dict(epilogue=2)),
                        (2, 4, 64, dict(out_dtype=5)), (2, 4, 64, dict(bias=at + 2)), (2, 4, 64, dict(residual=at + 2))):
        refused(p, at, at, at, at, at, m, n, k, **kw)
    for m, n, k in ((2, 4, (1 << 24) + 32), (1 << 31, 4, 64), ((1 << 32) - 1, 4, 64), (2, (1 << 32) - 1, 64), (17, 1 << 31, 64),
                    (1 << 30, 16, 64), (1 << 20, 1 << 17, 64)):
        refused(p, at, at, at, at, at, m, n, k)
    for i in range(5):
        args = [at] * 5
        args[i] = 0
        refused(p, *args, 2, 4, 64)
    refused(p, at + 8, at, at, at, at, 2, 4, 64)
    refused(p, at, at, at + 8, at, at, 2, 4, 64)
    refused(p, at, at, at, at, at + 2, 2, 4, 64)
    f = gpu_ctx.linear_mx4_fused
    for kw in (dict(x_dtype=4), dict(scale_rule=5), dict(x_stride=32), dict(x_stride=65), dict(epilogue=3),
               dict(out_dtype=2), dict(xq=at + 8)):
        refused(f, at, at, at, at, 40, 4, 64, **{**dict(xq=at, xs=at), **kw})
    refused(f, at, at, at, at, 40, 4, 64)              # (two launches: the work buffers are needed)
    refused(f, at, at, at, at, 40, 4, 64, xq=at)
    refused(f, at + 8, at, at, at, 40, 4, 64, xq=at, xs=at)
    refused(f, 0, at, at, at, 40, 4, 64, xq=at, xs=at)
    assert not buf.download(np.uint8, (1 << 16,)).any()


def test_shared_tiles_on_two_streams_and_in_two_graphs(gpu_ctx):
    """Products whose tiles several workgroups share, in two contexts at once (own streams, own scratch) and in two graphs of one
    context that use the same scratch: the bits of a product alone."""
    m, n, k = 65, 130, 8192
    rng = np.random.default_rng(7)
    other = ka.acquire_gpu(0)
    try:
        held = []
        for gpu in (gpu_ctx, other):
            w, ws = weights(rng, n, k)
            xq, xs = ref.quantised(activations(rng, m, k, np.float64), False)
            args = [gpu.upload(a) for a in (xq, xs, w, ws)]
            alone, outs = gpu.zeros(m * n * 4), [gpu.zeros(m * n * 4) for _ in range(12)]
            gpu.linear_mx4(*args, alone, m, n, k)
            gpu.sync()
            held.append((gpu, args, alone.download(np.float32, (m, n)), outs))
        for i in range(12):
            for gpu, args, _, outs in held:
                gpu.linear_mx4(*args, outs[i], m, n, k)
        for gpu, _, want, outs in held:
            gpu.sync()
            assert np.abs(want).max() > 0
            for out in outs:
                assert np.array_equal(out.download(np.float32, (m, n)).view(np.uint32), want.view(np.uint32))
        gpu, args, want, outs = held[0]
        graphs = []
        for i in range(2):
            outs[i].zero()
            with gpu.record() as rec:
                gpu.linear_mx4(*args, outs[i], m, n, k)
            graphs.append(rec.graph)
        for turn in range(3):
            for graph in graphs:
                graph.launch()
            gpu.linear_mx4(*args, outs[2], m, n, k)
            gpu.sync()
            for out in outs[:3]:
                assert np.array_equal(out.download(np.float32, (m, n)).view(np.uint32), want.view(np.uint32)), turn
        for graph in graphs:
            graph.destroy()
    finally:
        other.destroy()
