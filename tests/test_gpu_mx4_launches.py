"""Rows past what one launch, or one pass of its workgroups, has: quantisation steps by 65535 rows, the norms launch 2^21 at once."""
import numpy as np
import pytest

import karume_amd as ka
import mx4_reference as ref
from test_gpu_block_norm import run
from test_gpu_mx4 import CODE, Guarded, guarded, quantise

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [65534, 65535, 65536, 65537, 131070, 140001])
@pytest.mark.parametrize("io", ["f16", "f32"])
def test_rows_past_a_pass_are_quantised_and_read_back(gpu_ctx, rows, io):
    rng = np.random.default_rng(rows)
    x = rng.standard_normal((rows, 32)).astype(ref.NUMPY[io])
    codes, scales = quantise(gpu_ctx, x, False, 40)
    want = ka.pack_mx4(x.astype(np.float32))
    assert np.array_equal(codes, want[0]) and np.array_equal(scales, want[1])
    back = Guarded(gpu_ctx, x.nbytes)
    gpu_ctx.dequant_mx4(int(guarded(gpu_ctx, codes)), int(guarded(gpu_ctx, scales, shift=1)), int(back), rows=rows, dim=32,
                        out_dtype=CODE[io])
    assert np.array_equal(back.read(x.dtype, x.shape), ref.values(*want).astype(x.dtype))


@pytest.mark.parametrize("rows", [(1 << 21) - 1, 1 << 21, (1 << 21) + 1, (1 << 22) + 3])
def test_norms_of_more_rows_than_a_launch(gpu_ctx, rows):
    run(gpu_ctx, rows, 4, io="f32", gate="plain", span=300007)
    run(gpu_ctx, rows, 8, io="f16", gate="sigmoid", span=1, sum_in="residual", norm_in="y")
