"""silu(gate) * up of products of mx4 rows at gates of every size: the sums are the bias alone, so that each result has a
bound of its own."""
import numpy as np
import pytest

import karume_amd as ka
import mx4_reference as ref
from test_gpu_mx4 import CODE, Guarded, weights

pytestmark = pytest.mark.gpu

SIZES = [0, 1e-30, 0.3, 1, 5, 10, 20, 40, 63, 64, 80, 86, 87, 87.3, 87.4, 88, 90, 92, 95, 100, 103.5, 104, 110, 120, 150, 170,
         174, 180, 200, 1e3, 1e6, 3e7, 5e7, 1e9, 1e12, 1e30, 2.3e38, 2.4e38, 3e38]
UPS = {"f32": (1.0, -35000.0, 1e30, 1e-30), "f16": (1.0, -35000.0, 1e-4)}


def expected(gates, ups, out):
    """(f64 results, how far one may be off).

    fp16: the exponent -g log2 e is off by half a step for its product and a third for its constant, 1.25 |g| 2^-24 of the
    exponential; an exponential and a reciprocal of a step each, a sum and two products.  f32: two exponentials and the reciprocal of
    a step each, nine more operations of half a step; a subnormal result is rounded twice."""
    g, u = gates.astype(np.float64), ups.astype(np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        want = ref.silu(g) * u
        size = np.abs(want)
        off = size * 2.0 ** -24 * (15 if out == "f32" else 7 + 1.25 * np.minimum(np.abs(g), 1e4))
        off = off * 1.001 + ref.HALF_STEP[out] * size + 2 * ref.TINY_STEP[out]
        most = float(np.finfo(ref.NUMPY[out]).max)
    return np.where(size > most * (1 + ref.HALF_STEP[out]), np.copysign(np.inf, want), want), off


def check(got, want, off, what):
    got = got.astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want)), (what, np.flatnonzero(np.isnan(got) != np.isnan(want)))
    infinite = np.isinf(want)
    assert np.array_equal(got[infinite], want[infinite]), what
    rest = np.isfinite(want)
    over = rest & ~(np.abs(got - np.where(rest, want, 0)) <= off)
    assert not over.any(), (what, int(over.sum()), got[over][:4], want[over][:4], off[over][:4])


def run(gpu, m, gates, ups, out, k=64, io=None):
    n = 2 * len(gates)
    bias = np.stack([gates, ups], 1).reshape(-1).astype(np.float32)
    w, ws = weights(np.random.default_rng(m), n, k)
    dout = Guarded(gpu, m * n // 2 * ref.NUMPY[out]().nbytes)
    kw = dict(bias=gpu.upload(bias), out_dtype=CODE[out], epilogue=ka.EPILOGUE_SILU_PAIRS)
    if io is None:
        gpu.linear_mx4(gpu.zeros(m * k // 2), gpu.zeros(m * k // 32), gpu.upload(w), gpu.upload(ws), int(dout), m, n, k, **kw)
    else:
        gpu.linear_mx4_fused(gpu.zeros(m * k * 4), gpu.upload(w), gpu.upload(ws), int(dout), m, n, k,
                             xq=gpu.zeros(m * k // 2), xs=gpu.zeros(m * k // 32), **kw)
    want, off = expected(bias[0::2], bias[1::2], out)
    got = dout.read(ref.NUMPY[out], (m, n // 2))
    for row in range(m):
        check(got[row], want, off, (m, out, k, row))


@pytest.mark.parametrize("m,k", [(1, 64), (40, 64), (300, 64), (70, 8192)])   # each kernel, tiles that are shared too
@pytest.mark.parametrize("out", ["f32", "f16"])
def test_gates_of_every_size(gpu_ctx, m, k, out):
    gates = np.array([s * g for g in SIZES for s in (1, -1)], dtype=np.float32)
    for up in UPS[out]:
        run(gpu_ctx, m, gates, np.full(len(gates), up, dtype=np.float32), out, k)
    run(gpu_ctx, m, gates, np.ones(len(gates), dtype=np.float32), out, k, io="f32")


@pytest.mark.parametrize("out", ["f32", "f16"])
def test_gates_that_are_no_numbers(gpu_ctx, out):
    """An infinite gate is itself times up; that of the other sign and NaN are no number."""
    for m in (1, 40, 300):
        run(gpu_ctx, m, np.array([np.inf, 1, -np.inf, np.nan, 3e38, 0.0], dtype=np.float32),
            np.array([2, np.inf, 1, 1, np.nan, -np.inf], dtype=np.float32), out)


@pytest.mark.parametrize("out", ["f32", "f16"])
def test_many_gates(gpu_ctx, out):
    rng = np.random.default_rng(8)
    for low, high in ((-1, 1), (-20, 20), (-87, 87), (-110, -80), (-180, -100)):
        gates = rng.uniform(low, high, 8000).astype(np.float32)
        ups = np.exp(rng.uniform(-5, 60 if out == "f32" else 5, 8000)).astype(np.float32) * rng.choice((-1, 1), 8000)
        run(gpu_ctx, 2, gates, ups.astype(np.float32), out)
