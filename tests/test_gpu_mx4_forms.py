"""Every form of a product of mx4 rows, plain and with silu pairs, into both types, held to its bound; the plan's choice of
form is checked in test_mx4_plan_forms.py without a GPU."""
import numpy as np
import pytest

import karume_amd as ka
import mx4_reference as ref
from test_gpu_mx4 import CODE, Guarded, activations, guarded

pytestmark = pytest.mark.gpu
OUTS, WAYS = ("f32", "f16"), (False, True)

# Up to 16 rows: turns of one, two and four steps, deep rings and shallow ones, several pieces of 16 columns a workgroup.
ROWS = [(5, 70, 640), (4, 4210, 96), (9, 40, 1536), (6, 50, 4096), (16, 36, 6144), (3, 70, 544), (7, 40, 1568), (3, 50, 4128),
        (16, 36, 4128)]
# 17 to 64 rows: of 32 and of 64.
BATCH = [(20, 70, 1024), (50, 70, 1024), (20, 4130, 256), (20, 70, 1056), (50, 70, 1056), (50, 4130, 288)]
# Tiles of 64, 128 and 256 rows: with a CU to themselves or two on one, one run of scales, several and one that is
# not whole, shared throughout and in the last round, by two and by three.
TILES = [(65, 66, 256), (65, 66, 2048), (65, 66, 6656), (130, 16430, 2048),
         (65, 66, 96), (65, 66, 1056), (65, 66, 4128), (130, 16430, 1056),
         (197, 12230, 256), (65, 16430, 2048), (67, 9430, 11008), (130, 22030, 2048),
         (197, 12230, 64), (65, 16430, 1056), (65, 8200, 8224), (130, 22030, 1056),
         (517, 19230, 256), (260, 22030, 2048), (197, 17830, 11008),
         (517, 19230, 64), (390, 19230, 1056), (390, 20630, 1568), (197, 17830, 11040),
         (130, 22030, 6656), (130, 22030, 6688), (197, 16430, 6656), (197, 16430, 6688)]


class Product:
    """Random codes of both sides on the GPU, their sums and sums of magnitudes in 64 bits."""

    def __init__(self, gpu, m, n, k, io=None, shift=0):
        rng = np.random.default_rng(m * 31 + n * 7 + k)
        self.gpu, self.shape, self.io = gpu, (m, n, k), io
        w = rng.integers(0, 256, (n, k // 2), dtype=np.uint8), rng.integers(112, 119, (n, k // 32), dtype=np.uint8)
        x = activations(rng, m, k, ref.NUMPY[io or "f32"])
        xq = ref.quantised(x.astype(np.float64), False)
        xv, wv = ref.values(*xq), ref.values(*w).T
        self.sums, self.sizes = xv @ wv, np.abs(xv) @ np.abs(wv)
        self.bias = rng.standard_normal(n).astype(np.float32)
        self.residual = rng.standard_normal((m, n))
        self.w = [guarded(gpu, w[0]), guarded(gpu, w[1], shift=shift)]
        self.xq = [guarded(gpu, xq[0]), guarded(gpu, xq[1], shift=shift)]
        self.x = None if io is None else guarded(gpu, x)
        self.device_bias = gpu.upload(self.bias)

    def run(self, out, pairs):
        (m, n, k), t = self.shape, ref.NUMPY[out]
        width = n // 2 if pairs else n
        residual = self.residual[:, :width].astype(t)
        held = Guarded(self.gpu, residual.nbytes)
        kw = dict(bias=self.device_bias, residual=int(guarded(self.gpu, residual)), out_dtype=CODE[out],
                  epilogue=ka.EPILOGUE_SILU_PAIRS if pairs else ka.EPILOGUE_NONE)
        if self.io is None:
            self.gpu.linear_mx4(*map(int, self.xq), *map(int, self.w), int(held), m, n, k, **kw)
        else:
            self.gpu.linear_mx4_fused(int(self.x), *map(int, self.w), int(held), m, n, k, x_dtype=CODE[self.io], **kw)
        got = held.read(t, (m, width))
        ref.check(got, *self.expected(residual, pairs, out), (self.shape, out, pairs, self.io))
        return got

    def expected(self, residual, pairs, out):
        """As mx4_reference.product, with the gate's own error through the largest slope of silu."""
        step = 2.0 ** -24
        sums = self.sums + self.bias
        off = (self.shape[2] / 32 + 64) * step * self.sizes + step * np.abs(sums)
        if pairs:
            g, u, og, ou = sums[:, 0::2], sums[:, 1::2], off[:, 0::2], off[:, 1::2]
            s = ref.silu(g)
            # of silu itself: 15 half steps for f32, 7 and the exponent's for fp16
            own = step * np.abs(s) * (15 if out == "f32" else 7 + 1.25 * np.abs(g))
            sums, off = s * u, (1.1 * og + own) * (np.abs(u) + ou) + np.abs(s) * ou
        sums = sums + residual
        off = off + step * np.abs(sums)
        return sums, off * 1.001 + ref.HALF_STEP[out] * np.abs(sums) + ref.TINY_STEP[out]


@pytest.mark.parametrize("m,n,k", ROWS)
@pytest.mark.parametrize("io", [None, "f32", "f16"])
def test_few_rows(gpu_ctx, m, n, k, io):
    product = Product(gpu_ctx, m, n, k, io)
    for out in OUTS:
        for pairs in WAYS:
            product.run(out, pairs)


@pytest.mark.parametrize("m,n,k", BATCH + TILES)
def test_many_rows(gpu_ctx, m, n, k):
    product = Product(gpu_ctx, m, n, k)
    for out in OUTS:
        for pairs in WAYS:
            product.run(out, pairs)


@pytest.mark.parametrize("m,n,k", [(6, 50, 4096), (50, 70, 1024), (65, 66, 2048), (65, 66, 6656), (130, 22030, 2048),
                                   (260, 22030, 2048), (197, 16430, 6656)])
def test_scales_that_begin_inside_a_word(gpu_ctx, m, n, k):
    """Lengths whose scales are whole words, at addresses that are not: the same bits."""
    aligned, shifted = Product(gpu_ctx, m, n, k), Product(gpu_ctx, m, n, k, shift=3)
    for out in OUTS:
        for pairs in WAYS:
            a, b = aligned.run(out, pairs), shifted.run(out, pairs)
            assert np.array_equal(a.view(np.uint8), b.view(np.uint8))


@pytest.mark.parametrize("m,n,k", [(65, 66, 6656), (67, 9430, 11008), (197, 16430, 6656)])
def test_shared_tiles_on_a_side_branch(gpu_ctx, m, n, k):
    """On a side branch of a graph no tile is shared: within its bound beside a product of the main branch that is."""
    product = Product(gpu_ctx, m, n, k)
    alone = product.run("f32", False)
    outs = [gpu_ctx.zeros(m * n * 4) for _ in range(3)]
    kept = gpu_ctx.upload(product.residual.astype(np.float32))

    def call(out):
        gpu_ctx.linear_mx4(*map(int, product.xq), *map(int, product.w), out, m, n, k, bias=product.device_bias, residual=kept)

    with gpu_ctx.record() as rec:
        for branch in (1, 0, 2):
            rec.branch(branch)
            call(outs[branch])
    want, off = product.expected(product.residual.astype(np.float32), False, "f32")
    for _ in range(3):
        for out in outs:
            out.zero()
        rec.graph.launch()
        gpu_ctx.sync()
        got = [out.download(np.float32, (m, n)) for out in outs]
        assert np.array_equal(got[0].view(np.uint32), alone.view(np.uint32))
        for side in got[1:]:
            ref.check(side, want, off, (m, n, k))
        assert np.array_equal(got[1].view(np.uint32), got[2].view(np.uint32))
        call(outs[1])          # eager work between
        gpu_ctx.sync()
    rec.graph.destroy()
