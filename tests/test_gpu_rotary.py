"""Rotation tables and the general rotation on the GPU, against 64-bit angles and the f32 operations."""
import numpy as np
import pytest

import karume_amd as ka
import kv4_reference as ref

pytestmark = pytest.mark.gpu

IO = {np.float16: ka.F16, np.float32: ka.F32}


@pytest.mark.parametrize("pairs,rows,first,both,base,amplitude", [
    (1, 1, 0, False, 10000.0, 1.0), (32, 512, 0, True, 10000.0, 1.0), (20, 77, 3, True, 10000.0, 1.25),
    (64, 1000, 131072 - 500, False, 500000.0, 1.2079), (3, 257, 2**31 - 257, False, 10.0, 1.0),
    (128, 9, 1 << 20, True, 1e6, -0.5)])
def test_tables(gpu_ctx, pairs, rows, first, both, base, amplitude):
    ctx, width = gpu_ctx, pairs * (2 if both else 1)
    freq, _ = ka.rope_frequencies(2 * pairs, base)
    bufs = [ctx.upload(freq)] + [ctx.upload(np.full(rows * width + 4, 7.0, np.float32)) for _ in range(2)]
    ctx.rope_tables(*bufs, rows=rows, pairs=pairs, width=width, first=first, amplitude=amplitude)
    got = [b.download(np.float32, (rows * width + 4,)) for b in bufs[1:]]
    angle = (first + np.arange(rows, dtype=np.float64))[:, None] * freq
    # the 64-bit angle is off by half a step of it, and so is this one: 2 * 2^-53 * |angle|; r is rounded to 32
    # bits (|r| < 1: 2^-25), the series, its terms and the amplitude are off by 2^-24 each at most
    tol = abs(amplitude) * (2 * 2.0**-53 * np.abs(angle).max() + 2.0**-25 + 4 * 2.0**-24)
    for g, want in zip(got, (np.cos(angle), np.sin(angle))):
        assert np.all(g[rows * width:] == 7.0)
        g = g[:rows * width].reshape(rows, width)
        assert np.max(np.abs(g[:, :pairs] - want * np.float64(np.float32(amplitude)))) <= tol
        assert not both or np.array_equal(g[:, :pairs], g[:, pairs:])
    for b in bufs:
        b.free()


def test_tables_feed_the_half_split_rotation(gpu_ctx):
    """width = 2 * pairs is the table that rope_half reads, and rope_rows gives its result."""
    ctx, (rows, heads, d) = gpu_ctx, (37, 3, 64)
    rng = np.random.default_rng(1)
    x = rng.normal(size=(rows, heads, d)).astype(np.float32)
    freq, _ = ka.rope_frequencies(d)
    f, cos, sin = ctx.upload(freq), ctx.alloc(128 * d * 4), ctx.alloc(128 * d * 4)
    ctx.rope_tables(f, cos, sin, rows=128, pairs=d // 2, width=d)
    positions = ctx.upload(rng.integers(0, 128, size=rows).astype(np.int32))
    xin, one, two = ctx.upload(x), ctx.alloc(x.nbytes), ctx.alloc(x.nbytes)
    for head_major in (False, True):
        ctx.rope_half(xin, positions, cos, sin, one, rows, heads, d, 128, head_major)
        ctx.rope_rows(xin, positions, cos, sin, two, rows=rows, heads=heads, head_dim=d, rotary_dim=d, table_rows=128,
                      table_width=d, to_head_major=head_major)
        assert one.download(np.float32, x.shape).tobytes() == two.download(np.float32, x.shape).tobytes()
    for b in (f, cos, sin, positions, xin, one, two):
        b.free()


def angles(rng, table_rows, pairs, width):
    table = rng.normal(size=(2, table_rows, width)).astype(np.float32)
    table[:, :, pairs:] = np.nan   # not read
    return table


@pytest.mark.parametrize("io", [np.float16, np.float32])
@pytest.mark.parametrize("layout", [ka.ROPE_HALF, ka.ROPE_INTERLEAVED])
@pytest.mark.parametrize("rows,heads,d,rotary,width,pad,head_major", [
    (1, 1, 2, 2, 1, 0, False), (5, 3, 64, 64, 32, 0, False), (16, 32, 128, 64, 32, 0, True),
    (33, 5, 128, 128, 64, 128, True), (7, 2, 80, 20, 11, 3, False), (9, 1, 7, 6, 3, 0, True), (3, 4, 96, 0, 0, 0, False),
    (130, 2, 256, 48, 24, 8, False), (2, 2, 128, 74, 37, 0, True)])
def test_rows(gpu_ctx, io, layout, rows, heads, d, rotary, width, pad, head_major):
    ctx, rng = gpu_ctx, np.random.default_rng(rows * d + rotary)
    stride, table_rows = heads * d + pad, 50
    x = rng.normal(size=(rows, stride)).astype(io)
    cos, sin = angles(rng, table_rows, rotary // 2, max(width, 1))
    pos = rng.integers(0, table_rows, size=rows).astype(np.int32)
    bufs = [ctx.upload(a) for a in (x, pos, cos, sin)]
    out_stride = heads * d if head_major else stride + 5
    out = ctx.upload(np.full(rows * out_stride, 9, dtype=io))
    ctx.rope_rows(*bufs, out, rows=rows, heads=heads, head_dim=d, rotary_dim=rotary, layout=layout,
                  table_rows=table_rows, table_width=width, x_stride=stride, out_stride=out_stride,
                  to_head_major=head_major, io_dtype=IO[io])
    got = out.download(io, (rows * out_stride,))
    heads_of = x[:, :heads * d].reshape(rows, heads, d).astype(np.float32)
    want = ref.turned(heads_of, cos[pos], sin[pos], rotary, layout).astype(io)
    if head_major:
        assert got.reshape(heads, rows, d).tobytes() == want.swapaxes(0, 1).tobytes()
    else:
        got = got.reshape(rows, out_stride)
        assert got[:, :heads * d].tobytes() == want.tobytes()
        assert np.all(got[:, heads * d:] == 9)
    if not pad and (not head_major or heads == 1):   # in place
        ctx.rope_rows(*bufs, bufs[0], rows=rows, heads=heads, head_dim=d, rotary_dim=rotary, layout=layout,
                      table_rows=table_rows, table_width=width, to_head_major=head_major, io_dtype=IO[io])
        assert bufs[0].download(io, x.shape).tobytes() == want.tobytes()
    for b in bufs + [out]:
        b.free()


def test_a_position_outside_the_table_is_no_rotation(gpu_ctx):
    ctx, rng = gpu_ctx, np.random.default_rng(3)
    x = rng.normal(size=(4, 1, 64)).astype(np.float32)
    cos, sin = angles(rng, 10, 16, 16)
    pos = np.array([0, 10, -1, 9], np.int32)
    bufs = [ctx.upload(a) for a in (x, pos, cos, sin)]
    out = ctx.alloc(x.nbytes)
    ctx.rope_rows(*bufs, out, rows=4, heads=1, head_dim=64, rotary_dim=32, table_rows=10)
    got = out.download(np.float32, x.shape)
    assert np.all(np.isnan(got[1:3, :, :32])) and np.array_equal(got[:, :, 32:], x[:, :, 32:])
    assert np.all(np.isfinite(got[[0, 3]]))
    for b in bufs + [out]:
        b.free()


def test_refusals(gpu_ctx):
    ctx = gpu_ctx
    buf = ctx.alloc(4096)
    rows = dict(rows=2, heads=2, head_dim=64, rotary_dim=64, table_rows=4)
    for change in (dict(rotary_dim=66), dict(rotary_dim=63), dict(layout=2), dict(table_width=31), dict(table_rows=0),
                   dict(x_stride=127), dict(out_stride=127), dict(io_dtype=5), dict(head_dim=0), dict(rows=2**31)):
        with pytest.raises(ka.GpuValidationError):
            ctx.rope_rows(buf, buf, buf, buf, buf.offset(2048), **{**rows, **change})
    for name, change in (("in place", dict(to_head_major=True)), ("in place", dict(out_stride=130))):
        with pytest.raises(ka.GpuValidationError, match=name):
            ctx.rope_rows(buf, buf, buf, buf, buf, **{**rows, **change})
    with pytest.raises(ka.GpuValidationError, match="NULL"):
        ctx.rope_rows(buf, None, buf, buf, buf, **rows)
    with pytest.raises(ka.GpuValidationError, match="misaligned"):
        ctx.rope_rows(buf.offset(2), buf, buf, buf, buf, **rows)
    tables = dict(rows=4, pairs=8)
    for change in (dict(width=9), dict(width=24), dict(pairs=0, width=0), dict(amplitude=np.inf), dict(first=2**31 - 3)):
        with pytest.raises(ka.GpuValidationError):
            ctx.rope_tables(buf, buf, buf, **{**tables, **change})
    with pytest.raises(ka.GpuValidationError, match="NULL"):
        ctx.rope_tables(None, buf, buf, **tables)
    ctx.rope_tables(None, None, None, rows=0, pairs=8)
    ctx.rope_rows(None, None, None, None, None, **{**rows, "rows": 0})
    buf.free()


@pytest.mark.parametrize("pairs,rows,first,base,amplitude", [
    (64, 16384, 2**31 - 16384, 1.5, 1.0), (63, 8000, 2**31 - 8000, 1.5, 1.2079), (64, 8000, 2**30, 1.1, 0.75),
    (32, 20000, 0, 10000.0, 1.0), (64, 8000, 131072, 500000.0, 1.2079)])
def test_tables_are_off_by_a_step_at_most(gpu_ctx, pairs, rows, first, base, amplitude):
    """What is promised for |angle| < 2^31, 2^-23 of the amplitude, against angles in 64 bits of mantissa (off by 2^-33
    there): ones in 53 bits are off by as much as the promise themselves."""
    if np.finfo(np.longdouble).nmant < 63:
        pytest.skip("no longer numbers than 64 bits")
    ctx = gpu_ctx
    freq, _ = ka.rope_frequencies(2 * pairs, base)
    bufs = [ctx.upload(freq)] + [ctx.alloc(rows * pairs * 4) for _ in range(2)]
    ctx.rope_tables(*bufs, rows=rows, pairs=pairs, first=first, amplitude=amplitude)
    angle = (first + np.arange(rows, dtype=np.longdouble))[:, None] * freq.astype(np.longdouble)
    amplitude = np.longdouble(np.float32(amplitude))
    for buf, want in zip(bufs[1:], (np.cos(angle), np.sin(angle))):
        got = buf.download(np.float32, (rows, pairs))
        assert np.abs(got - want * amplitude).max() <= 2.0**-23 * amplitude
    for b in bufs:
        b.free()
