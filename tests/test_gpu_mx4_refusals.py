"""Quantisation and read-back of mx4 rows: calls that are refused before anything is launched."""
import numpy as np
import pytest

import karume_amd as ka

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1 << 31, (1 << 32) - 65536, (1 << 32) - 1])
def test_more_rows_than_a_row_number_and_its_step_hold(gpu_ctx, rows):
    """A launch of 65535 rows at once steps on by as many: past 2^32 - 65536 the next number would wrap round."""
    buf = gpu_ctx.zeros(1 << 14)
    at = int(buf)
    for dtype in (ka.F32, ka.F16):
        with pytest.raises(ka.GpuValidationError):
            gpu_ctx.quantize_mx4(at, at + 4096, at + 8192, rows=rows, dim=32, x_dtype=dtype)
        with pytest.raises(ka.GpuValidationError):
            gpu_ctx.dequant_mx4(at, at + 4096, at + 8192, rows=rows, dim=32, out_dtype=dtype)
    assert not buf.download(np.uint8, (1 << 14,)).any()


def test_results_in_the_place_of_what_is_read(gpu_ctx):
    """Rows are read by other threads than those that write there."""
    buf = gpu_ctx.zeros(1 << 14)
    at = int(buf)
    for args in ((at, at, at + 4096), (at, at + 4096, at), (at, at + 4096, at + 4096)):
        with pytest.raises(ka.GpuValidationError):
            gpu_ctx.quantize_mx4(*args, rows=2, dim=64)
    for args in ((at, at + 4096, at), (at, at + 4096, at + 4096)):
        with pytest.raises(ka.GpuValidationError):
            gpu_ctx.dequant_mx4(*args, rows=2, dim=64)
    assert not buf.download(np.uint8, (1 << 14,)).any()
