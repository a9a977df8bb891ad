"""The paged 4-bit K/V cache on the GPU: the append against the quantiser's f32 operations, byte for byte, the
attention against 64 bits from the cache's own bytes."""
import numpy as np
import pytest

import karume_amd as ka
import kv4_reference as ref

pytestmark = pytest.mark.gpu

IO = {np.float16: ka.F16, np.float32: ka.F32}


def up(ctx, *arrays):
    return [ctx.upload(np.ascontiguousarray(a)) for a in arrays]


def free(*buffers):
    for b in buffers:
        b.free()


# ------------------------------------------------------------------------------------------------- append
def expected_append(step, raw, q, k, v, cos, sin, rotary, layout, positions, table_rows):
    """(cache bytes, q rows in f32) after an append of f32 rows."""
    lay, raw, cu = step.layout, raw.copy(), step.cu
    at = np.concatenate([np.arange(n - r, n) for r, n in zip(step.rows, step.lens)])
    pos = at if positions is None else positions
    known = (pos >= 0) & (pos < table_rows)
    if rotary:
        c, s = (np.where(known[:, None], t[np.where(known, pos, 0)], np.nan) for t in (cos, sin))
        k = ref.turned(k, c, s, rotary, layout)
        q = ref.turned(q, c, s, rotary, layout) if q is not None else None
    ks, vs = ref.quantised(k, lay.group), ref.quantised(v, lay.group)
    for i in range(len(step.rows)):
        pages, rows = step.columns_of(i)
        for r in range(step.rows[i]):
            c, token = step.lens[i] - step.rows[i] + r, cu[i] + r
            for h in range(lay.kv_heads):
                lay.write(raw, pages[c], rows[c], h, tuple(a[token, h] for a in ks), tuple(a[token, h] for a in vs))
    return raw, q


def rows_of(rng, total, heads, depth, io, edges=True):
    x = rng.normal(size=(total, heads, depth)) * np.exp(rng.normal(size=(heads, depth)))
    if edges and total > 2:   # constant groups, tiny ones, zeros, the largest, one far element
        x[0, :, :32] = 0.1
        x[1, :, 32:64] = 0
        x[0, :, 32:64] *= 1e-6
        x[1, :, :32] = np.linspace(-32640, 32640, 32)
        x[2, :, 0] = 3000.0
    return x.astype(io).astype(np.float32)


@pytest.mark.parametrize("io", [np.float16, np.float32])
@pytest.mark.parametrize("depth,group,page,hkv,heads,rotary,layout,rows,lens", [
    (128, 32, 16, 2, 8, 128, ka.ROPE_HALF, (1, 1, 1), (1, 16, 17)),
    (64, 32, 16, 3, 3, 64, ka.ROPE_INTERLEAVED, (33, 0, 5), (33, 0, 70)),
    (64, 64, 64, 1, 4, 32, ka.ROPE_HALF, (7, 130), (128, 130)),
    (128, 128, 32, 2, 2, 74, ka.ROPE_HALF, (3, 4, 1), (40, 4, 33)),
    (128, 64, 64, 4, 28, 50, ka.ROPE_INTERLEAVED, (65,), (200,)),
    (256, 32, 256, 1, 8, 256, ka.ROPE_HALF, (2, 5), (257, 256)),
    (256, 128, 16, 2, 4, 0, ka.ROPE_HALF, (4, 1, 1, 9), (4, 1, 50, 31)),
])
def test_append_writes_these_bytes_and_no_others(gpu_ctx, io, depth, group, page, hkv, heads, rotary, layout, rows,
                                                 lens):
    ctx, rng = gpu_ctx, np.random.default_rng(depth + page + rotary)
    lay = ref.Layout(hkv, depth, group, page)
    step = ref.Step.make(lay, rows, lens, rng)
    raw = rng.integers(0, 256, size=(step.pages, lay.page_bytes), dtype=np.uint8)
    total, table_rows, width = step.total, max(lens) + 3, max(rotary // 2, 1) + 2
    qkv = rows_of(rng, total, heads + 2 * hkv, depth, io)
    angle = rng.uniform(0, 6, size=(table_rows, width))
    cos, sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    want, want_q = expected_append(step, raw, qkv[:, :heads], qkv[:, heads:heads + hkv], qkv[:, heads + hkv:], cos,
                                   sin, rotary, layout, None, table_rows)
    x, cache, table, cu, n, c, s = up(ctx, qkv.astype(io), raw, step.table, step.cu, np.int32(lens), cos, sin)
    fault, q_out = ctx.zeros(16), ctx.upload(np.full(total * heads * depth + 8, 5, dtype=io))
    eb, row = np.dtype(io).itemsize, (heads + 2 * hkv) * depth
    ctx.kv4_append(x.offset(heads * depth * eb), x.offset((heads + hkv) * depth * eb), cache, table, cu, n,
                   q=x, q_out=q_out, heads=heads, cos_table=c, sin_table=s, rotary_dim=rotary, layout=layout,
                   table_rows=table_rows, table_width=width, q_stride=row, k_stride=row, v_stride=row, fault=fault,
                   io_dtype=IO[io], **step.shape())
    got = cache.download(np.uint8, raw.shape)
    assert got.tobytes() == want.tobytes(), np.argwhere(got != want)[:5]
    got_q = q_out.download(io, (total * heads * depth + 8,))
    assert got_q[:-8].tobytes() == want_q.astype(io).tobytes() and np.all(got_q[-8:] == 5)
    assert not fault.download(np.uint32, (1,))[0]
    # the same rows read back, with the values that they stand for
    for out_dtype in (np.float16, np.float32):
        k_out, v_out = (ctx.upload(np.full((total + 1) * hkv * depth, 7, dtype=out_dtype)) for _ in range(2))
        ctx.kv4_read(cache, table, cu, n, k_out, v_out, fault=fault, out_dtype=IO[out_dtype], **step.shape())
        at = [(i, c) for i in range(len(rows)) for c in range(lens[i] - rows[i], lens[i])]
        for buf, held in zip((k_out, v_out), lay.values(want, np.arange(step.pages))):
            held = held.reshape(hkv, step.pages, page, depth)
            stands = np.stack([held[:, step.table[i, c // page], c % page] for i, c in at])
            back = buf.download(out_dtype, (total + 1, hkv, depth))
            assert back[:total].tobytes() == stands.astype(np.float32).astype(out_dtype).tobytes()
            assert np.all(back[total] == 7)
        free(k_out, v_out)
    free(x, cache, table, cu, n, c, s, fault, q_out)


def test_append_without_queries_with_positions_of_its_own(gpu_ctx):
    ctx, rng = gpu_ctx, np.random.default_rng(8)
    lay = ref.Layout(2, 64, 32, 16)
    step = ref.Step.make(lay, (3, 2), (20, 2), rng)
    raw = np.zeros((step.pages, lay.page_bytes), np.uint8)
    k, v = rows_of(rng, 5, 2, 64, np.float32), rows_of(rng, 5, 2, 64, np.float32)
    positions = np.array([9, 0, 4, 10, -1], np.int32)   # the last two outside the table
    cos, sin = rng.normal(size=(2, 10, 16)).astype(np.float32)
    want, _ = expected_append(step, raw, None, k, v, cos, sin, 32, ka.ROPE_HALF, positions, 10)
    bufs = up(ctx, k, v, raw, step.table, step.cu, np.int32(step.lens))
    pos, c, s = up(ctx, positions, cos, sin)
    ctx.kv4_append(*bufs, positions=pos, cos_table=c, sin_table=s, rotary_dim=32, table_rows=10, **step.shape())
    got = bufs[2].download(np.uint8, raw.shape)
    assert got.tobytes() == want.tobytes()
    page, row = step.columns_of(1)
    assert np.isnan(lay.pages(got)["params"][page[0], :, row[0], 0, 0]).all()   # the turned group, loudly
    assert np.isfinite(lay.pages(got)["params"][page[0], :, row[0], 1, 0]).all()
    free(*bufs, pos, c, s)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, 32648.0, 32656.0, -65504.0])
def test_groups_that_four_bits_cannot_hold_read_as_nan(gpu_ctx, bad):
    ctx, rng = gpu_ctx, np.random.default_rng(2)
    lay = ref.Layout(1, 64, 32, 16)
    step = ref.Step.make(lay, (2,), (2,), rng)
    k, v = rng.normal(size=(2, 2, 1, 64)).astype(np.float16)
    k[0, 0, 40] = v[1, 0, 3] = bad
    bufs = up(ctx, k, v, np.zeros((step.pages, lay.page_bytes), np.uint8), step.table, step.cu, np.int32([2]))
    ctx.kv4_append(*bufs, io_dtype=ka.F16, **step.shape())
    out = [ctx.alloc(2 * 64 * 4) for _ in range(2)]
    ctx.kv4_read(*bufs[2:], *out, **step.shape())
    gk, gv = (o.download(np.float32, (2, 64)) for o in out)
    nan_k, nan_v = np.zeros((2, 64), bool), np.zeros((2, 64), bool)
    # (fp16's step is 16 here: 32648 is a tie and becomes 32640, which is still held)
    nan_k[0, 32:], nan_v[1, :32] = (not abs(np.float16(bad)) <= 32640,) * 2
    assert np.array_equal(np.isnan(gk), nan_k) and np.array_equal(np.isnan(gv), nan_v)
    free(*bufs, *out)


def test_append_turns_queries_in_place(gpu_ctx):
    ctx, rng = gpu_ctx, np.random.default_rng(12)
    lay = ref.Layout(1, 64, 32, 16)
    step = ref.Step.make(lay, (5, 30), (5, 30), rng)
    q = rng.normal(size=(35, 7, 64)).astype(np.float32)
    k = rng.normal(size=(35, 1, 64)).astype(np.float32)
    cos, sin = rng.normal(size=(2, 30, 32)).astype(np.float32)
    bufs = up(ctx, k, k, np.zeros((step.pages, lay.page_bytes), np.uint8), step.table, step.cu, np.int32(step.lens))
    x, c, s = up(ctx, q, cos, sin)
    ctx.kv4_append(*bufs, q=x, q_out=x, heads=7, cos_table=c, sin_table=s, rotary_dim=64, table_rows=30,
                   **step.shape())
    at = np.r_[np.arange(5), np.arange(30)]
    assert x.download(np.float32, q.shape).tobytes() == ref.turned(q, cos[at], sin[at], 64, 0).tobytes()
    free(*bufs, x, c, s)


# ---------------------------------------------------------------------------------------------- attention
class Attention:
    """One step's attention on the device."""

    def __init__(self, ctx, step, raw, q, io, window=0, max_columns=None, half_scale=None, max_query=None):
        self.ctx, self.step, self.q, self.io, self.window = ctx, step, q.astype(io), io, window
        self.half_scale = step.layout.depth ** -0.25 if half_scale is None else half_scale
        self.shape = dict(step.shape(), heads=q.shape[1], window=window,
                          max_columns=max(step.lens + [1]) if max_columns is None else max_columns)
        if max_query:
            self.shape["max_query"] = max_query
        self.buf = dict(zip(("q", "cache", "table", "cu", "lens"),
                            up(ctx, self.q, raw, step.table, step.cu, np.int32(step.lens))))
        self.fault = ctx.zeros(16)
        self.out = ctx.upload(np.full((step.total + 1, *q.shape[1:]), 77, dtype=io))
        need = ctx.kv4_attention_workspace(io_dtype=IO[io], **self.shape)
        self.workspace = ctx.upload(np.full(need // 4 + 4, np.nan, np.float32))
        self.need = need

    def run(self, **change):
        self.ctx.kv4_attention(*self.buf.values(), self.out, fault=self.fault, half_scale=self.half_scale,
                               io_dtype=IO[self.io], workspace=self.workspace, **{**self.shape, **change})

    def result(self):
        out = self.out.download(self.io, (self.step.total + 1, *self.q.shape[1:]))
        assert np.all(out[-1] == 77), "rows behind the last sequence"
        return out[:-1]

    def faulted(self):
        return int(self.fault.download(np.uint32, (1,))[0])

    def free(self):
        free(*self.buf.values(), self.fault, self.out, self.workspace)


def tolerance(io, reach, top, span):
    """Largest error of an output element, and the 2-norm error's share.

    f32: a score is a sum of products that are exact or known to 2^-22, in f32, so it is off by
    16 * 2^-24 * reach at most (sums over groups, their parameters, the scale), the weights by as much and
    2^-22 more, and the sums over columns (blocks of 32, waves, splits, at most 64 + log2 of them in a row)
    by 2^-24 each; an error d of the weights moves an output by 2 d top.
    fp16: keys, values, weights and the result are each rounded once, by 2^-11 of themselves (weights below
    2^-14 by 2^-25): a score is off by 2^-11 reach, the result by 2^-11 top (2 reach + 2 + 1) and what f32
    would be off by.  As the roundings are independent, their 2-norm is 2^-11 each, not their sum: 4 * 2^-11."""
    f32 = top * (2 * 16 * 2.0**-24 * reach + 4 * 2.0**-22 + (64 + np.log2(span + 1)) * 2.0**-24)
    if io == np.float32:
        return f32, 2e-6 * max(1.0, reach / 16)
    return top * 2.0**-11 * (2 * reach + 3) + f32, 4 * 2.0**-11


def check(ctx, step, heads, io, rng, window=0, spread=1.0, **more):
    raw = step.random_cache(rng, spread)
    q = rng.normal(size=(step.total, heads, step.layout.depth)).astype(io)
    a = Attention(ctx, step, raw, q, io, window, **more)
    a.run()
    got = a.result().astype(np.float64)
    want, reach, top = step.attention(raw, a.q, a.half_scale, window)
    most, share = tolerance(io, reach, top, max(step.lens + [1]))
    assert np.all(np.isfinite(got))
    worst = np.abs(got - want).max() if got.size else 0.0
    rel = np.linalg.norm(got - want) / max(np.linalg.norm(want), 1e-30)
    assert worst <= most and rel <= share, (worst, most, rel, share)
    assert not a.faulted()
    a.run()   # the same call again: the same bits
    assert a.result().astype(np.float64).tobytes() == got.tobytes()
    a.free()


LAYOUTS = [(64, 32, 16), (64, 64, 64), (128, 32, 16), (128, 64, 128), (128, 128, 32), (256, 32, 64), (256, 64, 16),
           (256, 128, 256)]


@pytest.mark.parametrize("io", [np.float16, np.float32])
@pytest.mark.parametrize("depth,group,page", LAYOUTS)
def test_single_rows_of_ragged_sequences(gpu_ctx, io, depth, group, page):
    """Lengths of one, around pages and tiles of columns, and past what one workgroup walks."""
    rng = np.random.default_rng(depth + group + page)
    lens = (1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 255, 257, 700, 1300)
    step = ref.Step.make(ref.Layout(2, depth, group, page), (1,) * len(lens), lens, rng)
    check(gpu_ctx, step, 8, io, rng)


@pytest.mark.parametrize("io", [np.float16, np.float32])
@pytest.mark.parametrize("hkv,share", [(1, 1), (3, 1), (2, 7), (1, 8), (1, 16), (2, 17), (1, 64)])
def test_heads_that_share_keys(gpu_ctx, io, hkv, share):
    rng = np.random.default_rng(hkv * 100 + share)
    step = ref.Step.make(ref.Layout(hkv, 128, 32, 16), (1, 1, 2), (40, 333, 90), rng)
    check(gpu_ctx, step, hkv * share, io, rng)


@pytest.mark.parametrize("io", [np.float16, np.float32])
@pytest.mark.parametrize("window", [1, 2, 16, 31, 33, 200, 5000])
def test_windows(gpu_ctx, io, window):
    rng = np.random.default_rng(window)
    step = ref.Step.make(ref.Layout(2, 64, 32, 16), (1, 1, 5, 40, 1), (1, 33, 150, 64, 600), rng)
    check(gpu_ctx, step, 4, io, rng, window=window)


@pytest.mark.parametrize("io", [np.float16, np.float32])
@pytest.mark.parametrize("depth,group,page,hkv,share,rows,lens", [
    (128, 32, 64, 2, 4, (128,), (300,)), (64, 32, 16, 1, 8, (17, 1, 0, 64), (17, 90, 0, 1000)),
    (256, 128, 32, 1, 8, (33, 2), (33, 700)), (128, 64, 128, 2, 1, (200, 37), (200, 411)),
    (64, 64, 256, 1, 5, (9, 8, 7, 31, 3), (100, 8, 500, 31, 257)), (128, 128, 16, 1, 7, (63, 65), (64, 1025))])
def test_chunks_of_rows(gpu_ctx, io, depth, group, page, hkv, share, rows, lens):
    rng = np.random.default_rng(sum(rows) + depth)
    step = ref.Step.make(ref.Layout(hkv, depth, group, page), rows, lens, rng)
    check(gpu_ctx, step, hkv * share, io, rng)
    check(gpu_ctx, step, hkv * share, io, rng, window=50)


@pytest.mark.parametrize("io", [np.float16, np.float32])
@pytest.mark.parametrize("depth,group,page", LAYOUTS)
def test_many_rows_of_many_heads(gpu_ctx, io, depth, group, page):
    """Steps with blocks enough for the kernel that turns a tile's codes once for many rows: with whole and part waves and
    workgroups of rows, columns that are split and joined, and sequences of few rows and of none among them."""
    rng = np.random.default_rng(depth * group + page)
    hkv = 8 if depth < 256 else 4
    rows, lens = (260, 1, 0, 75, 8), (700, 333, 0, 75, 129)
    step = ref.Step.make(ref.Layout(hkv, depth, group, page), rows, lens, rng)
    check(gpu_ctx, step, hkv * 4, io, rng)
    check(gpu_ctx, step, hkv * 4, io, rng, window=100)
    whole = ref.Step.make(ref.Layout(hkv, depth, group, page), (150,), (150,), rng)
    check(gpu_ctx, whole, hkv * 7, io, rng)
    check(gpu_ctx, whole, hkv * 7, io, rng, max_columns=2048)
    more = ref.Step.make(ref.Layout(8, depth, group, page), (300,), (301,), rng)
    check(gpu_ctx, more, 8 * 7, io, rng)


@pytest.mark.parametrize("io", [np.float16, np.float32])
@pytest.mark.parametrize("depth,group", [(64, 32), (128, 128), (256, 64)])
def test_many_sequences_of_many_rows(gpu_ctx, io, depth, group):
    """More sequences than a wave reads at a time, chunks and single rows in one step, and one long sequence among them."""
    rng = np.random.default_rng(depth)
    rows = [(40, 1, 0, 17, 9)[i % 5] for i in range(133)]
    lens = [r + int(rng.integers(0, 90)) if r else 0 for r in rows]
    lens[130] = 1500
    step = ref.Step.make(ref.Layout(2, depth, group, 32), rows, lens, rng)
    check(gpu_ctx, step, 8, io, rng)
    check(gpu_ctx, step, 8, io, rng, window=33)


@pytest.mark.parametrize("io", [np.float16, np.float32])
@pytest.mark.parametrize("depth,rows,lens", [(64, (512,), (512,)), (64, (512, 512), (512, 512)),
                                             (128, (700, 260), (700, 5000)), (256, (300, 300), (300, 1200)),
                                             (256, (300, 300, 1, 77), (300, 1200, 5, 77))])
def test_whole_prompts(gpu_ctx, io, depth, rows, lens):
    """Rows that see nothing but each other: blocks of rows with few columns beside ones with all of them."""
    rng = np.random.default_rng(depth)
    step = ref.Step.make(ref.Layout(4, depth, 64, 64), rows, lens, rng)
    check(gpu_ctx, step, 16, io, rng)


@pytest.mark.parametrize("io", [np.float16, np.float32])
def test_all_rows_of_a_refused_chunk_are_nan(gpu_ctx, io):
    rng = np.random.default_rng(3)
    rows, lens = (70, 90, 1, 64), (70, 300, 40, 500)
    step = ref.Step.make(ref.Layout(8, 64, 32, 16), rows, lens, rng)
    raw = step.random_cache(rng)
    q = rng.normal(size=(step.total, 64, 64))
    a = Attention(gpu_ctx, step, raw, q, io)
    want, reach, top = step.attention(raw, a.q, a.half_scale, 0)
    most, _ = tolerance(io, reach, top, 500)
    refused = np.zeros(step.total, bool)
    refused[70:160] = True
    for change, lengths in ((dict(), (70, 89, 40, 500)), (dict(max_query=70), lens)):
        a.buf["lens"].upload(np.int32(lengths))
        a.fault.zero()
        a.run(**change)
        got = a.result().astype(np.float64)
        assert a.faulted() == 1 and np.all(np.isnan(got[refused]))
        assert np.abs(got[~refused] - want[~refused]).max() <= most
    a.free()


@pytest.mark.parametrize("io", [np.float16, np.float32])
def test_limits_larger_than_the_step_needs(gpu_ctx, io):
    """What a recorded call is made with: more rows and columns than the sequences have yet."""
    rng = np.random.default_rng(6)
    step = ref.Step.make(ref.Layout(2, 128, 32, 16), (1, 0, 3, 1), (5, 0, 40, 900), rng)
    check(gpu_ctx, step, 8, io, rng, max_columns=20000)
    step = ref.Step.make(ref.Layout(2, 64, 32, 16), (1, 2, 0, 30), (5, 9, 0, 333), rng, extra=9)
    check(gpu_ctx, step, 6, io, rng, max_columns=2**31 - 1 if io == np.float16 else 4096, max_query=33)


@pytest.mark.parametrize("io", [np.float16, np.float32])
@pytest.mark.parametrize("spread", [1e-4, 30.0])
def test_small_and_large_values(gpu_ctx, io, spread):
    """Parameters among fp16's subnormals, and scores whose softmax is nearly one column's."""
    rng = np.random.default_rng(int(spread * 1e4))
    step = ref.Step.make(ref.Layout(1, 64, 32, 16), (1, 3, 20), (100, 260, 64), rng)
    check(gpu_ctx, step, 8, io, rng, spread=spread)


@pytest.mark.parametrize("io", [np.float16, np.float32])
def test_queries_of_any_size(gpu_ctx, io):
    """Rows of 1e-3 and of 300 beside each other, and a row of zeros (equal weights)."""
    rng = np.random.default_rng(14)
    step = ref.Step.make(ref.Layout(1, 128, 32, 16), (3, 18), (70, 50), rng)
    raw = step.random_cache(rng)
    q = rng.normal(size=(21, 4, 128)) * np.r_[1e-3, 300.0, 0.0, np.ones(18)][:, None, None]
    a = Attention(gpu_ctx, step, raw, q, io)
    a.run()
    want, reach, top = step.attention(raw, a.q, a.half_scale)
    assert np.abs(a.result() - want).max() <= tolerance(io, reach, top, 70)[0]
    assert np.abs(a.result()[2] - want[2]).max() <= tolerance(io, 0.0, top, 70)[0]
    a.free()


def test_no_rows_at_all(gpu_ctx):
    rng = np.random.default_rng(0)
    step = ref.Step.make(ref.Layout(1, 64, 32, 16), (0, 0), (0, 9), rng)
    a = Attention(gpu_ctx, step, step.random_cache(rng), np.zeros((1, 2, 64)), np.float16, max_query=1)
    a.shape["total_rows"] = 1
    a.run()
    assert np.all(a.out.download(np.float16, (1, 2, 64)) == 77) and not a.faulted()
    a.run(total_rows=0, max_query=0)
    a.run(nseq=0)
    a.free()


REFUSED = {"longer than its table": dict(lens=(40, 97, 8)), "longer than max_columns": dict(lens=(40, 81, 8)),
           "no columns": dict(lens=(40, 0, 8)), "fewer columns than rows": dict(lens=(40, 1, 8)),
           "negative": dict(lens=(40, -2**31, 8))}


@pytest.mark.parametrize("io", [np.float16, np.float32])
@pytest.mark.parametrize("case", REFUSED)
def test_refused_sequences_are_nan_and_the_others_are_not(gpu_ctx, io, case):
    rng = np.random.default_rng(77)
    step = ref.Step.make(ref.Layout(2, 64, 32, 16), (1, 2, 3), (40, 80, 8), rng)
    assert step.table.shape[1] == 6
    raw = step.random_cache(rng)
    q = rng.normal(size=(6, 4, 64))
    a = Attention(gpu_ctx, step, raw, q, io, max_columns=80 if "max_columns" in case else 96)
    a.run()
    good = a.result()
    assert not a.faulted()
    a.buf["lens"].upload(np.int32(REFUSED[case]["lens"]))
    a.run()
    got = a.result()
    assert a.faulted() == 1
    assert np.all(np.isnan(got[1:3])) and got[[0, 3, 4, 5]].tobytes() == good[[0, 3, 4, 5]].tobytes()
    # rows that the offsets do not give to any sequence stay as they were
    a.buf["lens"].upload(np.int32((40, 80, 8)))
    a.out.upload(np.full(a.out.nbytes // np.dtype(io).itemsize, 77, io))
    a.buf["cu"].upload(np.int32((0, 1, 7, 6)))   # past the rows, then descending
    a.fault.zero()
    a.run()
    got = a.out.download(io, (7, 4, 64))
    assert a.faulted() == 1 and np.all(got[1:] == 77) and got[0].tobytes() == good[0].tobytes()
    # an append of the refused sequences writes nothing
    before = a.buf["cache"].download(np.uint8, raw.shape)
    rows = gpu_ctx.upload(rng.normal(size=(6, 2, 64)).astype(io))
    a.fault.zero()
    gpu_ctx.kv4_append(rows, rows, a.buf["cache"], a.buf["table"], a.buf["cu"], a.buf["lens"], fault=a.fault,
                       io_dtype=IO[io], **step.shape())
    after = a.buf["cache"].download(np.uint8, raw.shape)
    changed = np.unique(np.argwhere((before != after).reshape(step.pages, -1))[:, 0])
    assert a.faulted() == 1 and set(changed) <= {step.table[0, 2]}
    free(rows)
    a.free()


@pytest.mark.parametrize("io", [np.float16, np.float32])
@pytest.mark.parametrize("page", [-1, 10**6, -2**31, 2**31 - 1])
@pytest.mark.parametrize("chunk", [False, True])
def test_pages_outside_the_cache(gpu_ctx, io, page, chunk):
    """Rows that see such a page are NaN, rows of a window that does not are as before."""
    rng = np.random.default_rng(78)
    heads = 256 if chunk else 4
    step = ref.Step.make(ref.Layout(2, 64, 32, 16), (1, 40 if chunk else 3, 3), (40, 90, 8), rng)
    raw = step.random_cache(rng)
    q = rng.normal(size=(step.total, heads, 64))
    good = {}
    for window in (0, 20):
        a = Attention(gpu_ctx, step, raw, q, io, window)
        a.run()
        good[window] = a.result()
        table = step.table.copy()
        table[1, 2] = page   # columns 32 .. 47
        a.buf["table"].upload(table)
        a.run()
        got = a.result()
        p = np.arange(90 - step.rows[1], 90)
        sees = (p >= 32) & ((p - (window or 999) + 1) <= 47)
        lost = np.r_[False, sees, [False] * 3]
        assert a.faulted() == lost.any()
        assert np.all(np.isnan(got[lost])) and got[~lost].tobytes() == good[window][~lost].tobytes()
        assert lost.any() == (window == 0 or chunk)
        a.free()


@pytest.mark.parametrize("io", [np.float16, np.float32])
def test_append_and_read_skip_pages_outside_the_cache(gpu_ctx, io):
    ctx, rng = gpu_ctx, np.random.default_rng(79)
    lay = ref.Layout(1, 64, 32, 16)
    step = ref.Step.make(lay, (20,), (20,), rng)
    raw = rng.integers(0, 256, size=(step.pages, lay.page_bytes), dtype=np.uint8)
    k = rng.normal(size=(20, 1, 64)).astype(io).astype(np.float32)
    want, _ = expected_append(step, raw, None, k, k, None, None, 0, 0, None, 0)
    want[step.table[0, 1]] = raw[step.table[0, 1]]
    table = step.table.copy()
    table[0, 1] = step.pages
    x, cache, t, cu, n = up(ctx, k.astype(io), raw, table, step.cu, np.int32([20]))
    fault, out = ctx.zeros(16), [ctx.alloc(20 * 64 * 4) for _ in range(2)]
    ctx.kv4_append(x, x, cache, t, cu, n, fault=fault, io_dtype=IO[io], **step.shape())
    assert fault.download(np.uint32, (1,))[0] == 1
    assert cache.download(np.uint8, raw.shape).tobytes() == want.tobytes()
    fault.zero()
    ctx.kv4_read(cache, t, cu, n, *out, fault=fault, **step.shape())
    assert fault.download(np.uint32, (1,))[0] == 1
    got = out[0].download(np.float32, (20, 64))
    assert np.all(np.isfinite(got[:16])) and np.all(np.isnan(got[16:]))
    free(x, cache, t, cu, n, fault, *out)


@pytest.mark.parametrize("io", [np.float16, np.float32])
@pytest.mark.parametrize("depth,group,share", [(64, 32, 4), (128, 32, 3), (128, 128, 1), (256, 64, 8)])
def test_nan_in_a_seen_column_shows_and_in_an_unseen_one_does_not(gpu_ctx, io, depth, group, share):
    """A key's NaN is its row's, a value's its group's, in the rows that see the column and in no others."""
    rng = np.random.default_rng(80)
    for rows, lens, window in (((1, 1), (50, 70), 0), ((1, 1), (50, 70), 5), ((20, 30), (50, 70), 0),
                               ((40, 30), (50, 70), 7), ((2, 3), (60, 46), 12), ((200, 3), (230, 60), 0),
                               ((200, 300), (230, 300), 9)):
        lay = ref.Layout(2, depth, group, 16)
        step = ref.Step.make(lay, rows, lens, rng)
        raw = step.random_cache(rng)
        share = 8 * share if rows[0] == 200 else share    # (blocks enough for the kernel of many rows)
        q = rng.normal(size=(sum(rows), 2 * share, depth))
        for name in ("params", "vparams"):
            held = raw.copy()
            page, row = step.columns_of(0)
            if name == "params":
                lay.pages(held)["params"][page[45], 1, row[45], 1 % lay.pages(held)["params"].shape[3], 0] = np.nan
            else:
                lay.pages(held)["vparams"][page[45], 1, row[45] // 4, -1, 0, row[45] % 4] = np.nan
            a = Attention(gpu_ctx, step, held, q, io, window)
            a.run()
            p = np.arange(lens[0] - rows[0], lens[0])
            sees = np.r_[(p >= 45) & (p - 45 < (window or 999)), np.zeros(rows[1], bool)]
            want = np.zeros(q.shape, bool)
            want[sees, share:, 0 if name == "params" else depth - group:] = True
            assert np.array_equal(np.isnan(a.result()), want), (rows, window, name)
            a.free()


def test_offsets_past_32_bits(gpu_ctx):
    """Pages that lie more than 4 GiB behind the cache's address."""
    ctx, rng = gpu_ctx, np.random.default_rng(81)
    lay = ref.Layout(8, 128, 32, 256)
    pages = (5 << 30) // lay.page_bytes
    small = ref.Step.make(lay, (1, 20), (300, 290), rng, spare=0)
    raw = small.random_cache(rng)
    q = rng.normal(size=(21, 8, 128)).astype(np.float16)
    cache = ctx.alloc(pages * lay.page_bytes)
    k = rng.normal(size=(21, 8, 128)).astype(np.float16)
    try:
        far = ref.Step(lay, small.rows, small.lens, pages, np.where(small.table < small.pages,
                                                                     pages - 1 - small.table, small.table))
        for i in range(small.pages):
            cache.upload(raw[i], byte_offset=(pages - 1 - i) * lay.page_bytes)
        bufs = up(ctx, q, far.table, far.cu, np.int32(far.lens), k)
        near = Attention(ctx, small, raw, q, np.float16)
        outs = []
        for c, step, table in ((cache, far, bufs[1]), (near.buf["cache"], small, near.buf["table"])):
            ctx.kv4_append(bufs[4], bufs[4], c, table, bufs[2], bufs[3], io_dtype=ka.F16, **step.shape())
            ctx.kv4_attention(bufs[0], c, table, bufs[2], bufs[3], near.out, half_scale=0.3, heads=8,
                              max_columns=300, io_dtype=ka.F16, workspace=near.workspace, **step.shape())
            outs.append(near.result())
        assert outs[0].tobytes() == outs[1].tobytes() and np.all(np.isfinite(outs[0]))
        got = np.stack([cache.download(np.uint8, (lay.page_bytes,), byte_offset=(pages - 1 - i) * lay.page_bytes)
                        for i in range(small.pages)])
        assert got.tobytes() == near.buf["cache"].download(np.uint8, raw.shape).tobytes()
        near.free()
        free(*bufs)
    finally:
        cache.free()


def test_a_recorded_step_replays_while_sequences_grow(gpu_ctx):
    """Tables, append and attention together: a prompt, then decode steps recorded once and replayed, with eager work
    and a synchronisation between replays, against the eager calls and 64 bits."""
    ctx, rng = gpu_ctx, np.random.default_rng(90)
    lay, heads, io = ref.Layout(2, 64, 32, 16), 8, np.float16
    prompts, steps = [37, 1, 16], 5
    final = ref.Step.make(lay, (1, 1, 1), [n + steps for n in prompts], rng)
    freq, amplitude = ka.rope_frequencies(64, 10000.0, scaling="ramp", factor=4.0, trained=16)
    f, cos, sin = ctx.upload(freq), ctx.alloc(64 * 32 * 4), ctx.alloc(64 * 32 * 4)
    ctx.rope_tables(f, cos, sin, rows=64, pairs=32, amplitude=amplitude)
    table, = up(ctx, final.table)
    caches = [ctx.zeros(final.pages * lay.page_bytes) for _ in range(2)]
    turn = dict(cos_table=cos, sin_table=sin, rotary_dim=64, table_rows=64, io_dtype=ka.F16)

    def inputs(rows):
        return [rng.normal(size=(sum(rows), n, 64)).astype(io) for n in (heads, 2, 2)]

    prompt = ref.Step(lay, prompts, prompts, final.pages, final.table)
    x, (cu, n) = inputs(prompts), up(ctx, prompt.cu, np.int32(prompts))
    limits = dict(heads=heads, max_columns=max(prompts) + steps, half_scale=0.4, io_dtype=ka.F16)
    sizes = dict(heads=heads, max_columns=max(prompts) + steps, io_dtype=ka.F16)
    for cache in caches:
        q, k, v = up(ctx, *x)
        ctx.kv4_append(k, v, cache, table, cu, n, q=q, q_out=q, heads=heads, **turn, **prompt.shape())
        ws = ctx.alloc(max(16, ctx.kv4_attention_workspace(**sizes, **prompt.shape())))
        out = ctx.alloc(q.nbytes)
        ctx.kv4_attention(q, cache, table, cu, n, out, workspace=ws, **limits, **prompt.shape())
        got = out.download(io, x[0].shape)
        raw = cache.download(np.uint8, (final.pages, lay.page_bytes))
        want, reach, top = prompt.attention(raw, q.download(io, x[0].shape), 0.4)
        assert np.abs(got - want).max() <= tolerance(io, reach, top, 40)[0]
        free(q, k, v, ws, out)
    free(cu, n)
    one = ref.Step(lay, [1, 1, 1], prompts, final.pages, final.table)
    lens, cu = ctx.alloc(16), ctx.upload(one.cu)
    ws = ctx.alloc(max(16, ctx.kv4_attention_workspace(**sizes, **one.shape())))
    q, k, v = (ctx.alloc(3 * h * 64 * 2) for h in (heads, 2, 2))
    q_out, out = ctx.alloc(3 * heads * 64 * 2), ctx.alloc(3 * heads * 64 * 2)

    def step_on(cache):
        ctx.kv4_append(k, v, cache, table, cu, lens, q=q, q_out=q_out, heads=heads, **turn, **one.shape())
        ctx.kv4_attention(q_out, cache, table, cu, lens, out, workspace=ws, **limits, **one.shape())

    with ctx.record() as rec:
        step_on(caches[0])
    for t in range(steps):
        now = [p + t + 1 for p in prompts]
        x = inputs([1, 1, 1])
        for b, a in zip((q, k, v, lens), x + [np.int32(now)]):
            b.upload(a)
        rec.graph.launch()
        ctx.sync()
        replayed, turned = out.download(io, (3, heads, 64)), q_out.download(io, (3, heads, 64))
        out.zero()
        step_on(caches[1])
        assert out.download(io, (3, heads, 64)).tobytes() == replayed.tobytes(), t
        raw = [c.download(np.uint8, (final.pages, lay.page_bytes)) for c in caches]
        assert raw[0].tobytes() == raw[1].tobytes()
        done = ref.Step(lay, [1, 1, 1], now, final.pages, final.table)
        want, reach, top = done.attention(raw[0], turned, 0.4)
        assert np.abs(replayed - want).max() <= tolerance(io, reach, top, 64)[0]
    rec.graph.destroy()
    free(f, cos, sin, table, *caches, lens, cu, ws, q, k, v, q_out, out)


def test_two_contexts_read_one_cache_at_once(gpu_ctx):
    """Each on its own stream with its own workspace."""
    rng = np.random.default_rng(91)
    step = ref.Step.make(ref.Layout(2, 128, 32, 16), (1,) * 6, (900, 40, 1300, 600, 77, 1), rng)
    raw, q = step.random_cache(rng), rng.normal(size=(6, 8, 128))
    other = ka.acquire_gpu(0)
    try:
        a = Attention(gpu_ctx, step, raw, q, np.float16)
        b = Attention(other, step, raw, q, np.float16)
        for name in ("cache", "table", "cu", "lens"):
            b.buf[name].free()
            b.buf[name] = a.buf[name]
        for _ in range(20):
            a.run()
            b.run()
        gpu_ctx.sync()
        other.sync()
        assert a.result().tobytes() == b.result().tobytes()
        free(b.buf["q"], b.fault, b.out, b.workspace)
        a.free()
    finally:
        other.destroy()


def test_two_recorded_calls_share_a_workspace(gpu_ctx):
    """Two graphs of one context, launched in turn over the same workspace."""
    rng = np.random.default_rng(92)
    lay = ref.Layout(2, 64, 32, 16)
    calls = []
    for lens, rows in (((1500, 700), (1, 1)), ((900, 1100, 64), (1, 1, 1))):
        step = ref.Step.make(lay, rows, lens, rng)
        a = Attention(gpu_ctx, step, step.random_cache(rng), rng.normal(size=(len(rows), 8, 64)), np.float16)
        a.run()
        calls.append((a, a.result().tobytes()))
    big = max((a for a, _ in calls), key=lambda a: a.need)
    graphs = []
    for a, _ in calls:
        with gpu_ctx.record() as rec:
            gpu_ctx.kv4_attention(*a.buf.values(), a.out, fault=a.fault, half_scale=a.half_scale, io_dtype=ka.F16,
                                  workspace=big.workspace, **a.shape)
        graphs.append(rec.graph)
    for replay in range(4):
        for a, _ in calls:
            a.out.upload(np.full(a.out.nbytes // 2, 77, np.float16))
        for g in graphs:
            g.launch()
        gpu_ctx.sync()
        for a, want in calls:
            assert a.result().tobytes() == want, replay
    for g in graphs:
        g.destroy()
    for a, _ in calls:
        a.free()


@pytest.mark.parametrize("io", [np.float16, np.float32])
def test_recorded_chunks_replay_with_other_rows_and_lengths(gpu_ctx, io):
    """One graph with room for 300 rows a sequence: chunks that grow, shrink, end and are refused between replays, which
    changes what every workgroup does; each replay has the bits of the eager call."""
    ctx, rng = gpu_ctx, np.random.default_rng(93)
    lay, heads = ref.Layout(4, 64, 64, 32), 32
    full = ref.Step.make(lay, (300, 300, 300), (1000, 700, 300), rng)
    raw, q = full.random_cache(rng), rng.normal(size=(full.total, heads, 64))
    a = Attention(ctx, full, raw, q, io)
    with ctx.record() as rec:
        a.run()
    for rows, lens, bad in (((300, 300, 300), (1000, 700, 300), False), ((1, 300, 2), (999, 300, 50), False),
                            ((0, 0, 200), (7, 0, 280), False), ((130, 0, 31), (130, 3, 31), False),
                            ((200, 300, 40), (1000, 299, 300), True), ((1, 1, 1), (5, 640, 1), False)):
        step = ref.Step(lay, list(rows), list(lens), full.pages, full.table)
        got = []
        for run in (rec.graph.launch, a.run):
            a.buf["cu"].upload(step.cu)
            a.buf["lens"].upload(np.int32(lens))
            a.out.upload(np.full(a.out.nbytes // np.dtype(io).itemsize, 77, io))
            a.fault.zero()
            run()
            ctx.sync()
            got.append(a.out.download(io, (full.total + 1, heads, 64)))
            assert a.faulted() == bad
        assert got[0].tobytes() == got[1].tobytes(), rows
        assert np.all(got[0][step.total:] == 77)
        if not bad:
            want, reach, top = step.attention(raw, a.q[:step.total], a.half_scale)
            assert np.abs(got[0][:step.total] - want).max() <= tolerance(io, reach, top, 1000)[0]
        else:
            assert np.all(np.isnan(got[0][200:500])) and np.all(np.isfinite(got[0][:200]))
    rec.graph.destroy()
    a.free()


def test_side_branches_have_calls_without_a_workspace_only(gpu_ctx):
    ctx, rng = gpu_ctx, np.random.default_rng(94)
    calls = []
    for lens in ((30, 9), (800, 90)):
        step = ref.Step.make(ref.Layout(2, 64, 32, 16), (1, 1), lens, rng)
        calls.append(Attention(ctx, step, step.random_cache(rng), rng.normal(size=(2, 4, 64)), np.float16))
    short, long = calls
    assert short.need == 0 < long.need
    with ctx.record() as rec:
        rec.branch(1)
        with pytest.raises(ka.GpuValidationError):
            long.run()
        short.run()
        rec.branch(0)
        long.run()
    for _ in range(3):
        rec.graph.launch()
        ctx.sync()
    got = [a.result().tobytes() for a in calls]
    for a, g in zip(calls, got):
        a.run()
        assert a.result().tobytes() == g
    rec.graph.destroy()
    short.free()
    long.free()


def test_refusals(gpu_ctx):
    ctx, rng = gpu_ctx, np.random.default_rng(1)
    step = ref.Step.make(ref.Layout(2, 64, 32, 16), (1, 2), (700, 80), rng)
    a = Attention(ctx, step, step.random_cache(rng), rng.normal(size=(3, 4, 64)), np.float32)
    for change in (dict(depth=96), dict(group=48), dict(page_rows=24), dict(heads=3), dict(max_query=0),
                   dict(max_columns=1), dict(pages=0), dict(table_stride=0), dict(kv_heads=0),
                   dict(max_columns=2**31)):
        with pytest.raises(ka.GpuValidationError):
            a.run(**change)
    b = a.buf
    args = (b["q"], b["cache"], b["table"], b["cu"], b["lens"], a.out)
    call = lambda args, **more: ctx.kv4_attention(*args, **{**dict(half_scale=1.0, workspace=a.workspace),  # noqa: E731
                                                            **a.shape, **more})
    for at in range(6):
        with pytest.raises(ka.GpuValidationError, match="NULL"):
            call(args[:at] + (None,) + args[at + 1:])
    for at in (0, 1, 5):
        with pytest.raises(ka.GpuValidationError, match="misaligned"):
            call(args[:at] + (args[at].offset(4),) + args[at + 1:])
    for more, match in ((dict(half_scale=np.nan), "half_scale"), (dict(half_scale=1e30), "half_scale"),
                        (dict(io_dtype=3), "io_dtype"), (dict(fault=a.fault.offset(2)), "misaligned")):
        with pytest.raises(ka.GpuValidationError, match=match):
            call(args, **more)
    with pytest.raises(ka.GpuValidationError, match="out is q"):
        call(args[:5] + (args[0],))
    if a.need:
        with pytest.raises(ka.GpuValidationError, match="workspace"):
            call(args, workspace=None)
        with pytest.raises(ka.GpuValidationError, match="workspace"):
            call(args, workspace_bytes=a.need - 1)
    rows = (b["q"], b["q"], b["cache"], b["table"], b["cu"], b["lens"])
    append = lambda args, **more: ctx.kv4_append(*args, **{**step.shape(), **more})  # noqa: E731
    for more, match in ((dict(q=b["q"]), "together"), (dict(rotary_dim=64), "tables"),
                        (dict(rotary_dim=64, table_rows=9), "NULL"), (dict(rotary_dim=66), "rotary_dim"),
                        (dict(k_stride=64), "stride"), (dict(v_stride=130), "misaligned"),
                        (dict(io_dtype=9), "io_dtype"), (dict(page_rows=20), "page_rows"),
                        (dict(q=b["q"], q_out=b["q"], heads=2, q_stride=256), "in place"),
                        (dict(q=b["q"], q_out=a.out, heads=5), "heads")):
        with pytest.raises(ka.GpuValidationError, match=match):
            append(rows, **more)
    for at in range(6):
        with pytest.raises(ka.GpuValidationError, match="NULL"):
            append(rows[:at] + (None,) + rows[at + 1:])
    for more, match in ((dict(out_dtype=2), "out_dtype"), (dict(group=256), "group")):
        with pytest.raises(ka.GpuValidationError, match=match):
            ctx.kv4_read(*args[1:5], a.out, a.out, **{**step.shape(), **more})
    with pytest.raises(ka.GpuValidationError, match="NULL"):
        ctx.kv4_read(*args[1:5], None, a.out, **step.shape())
    a.run()
    assert np.all(np.isfinite(a.result()))
    a.free()


@pytest.mark.parametrize("io", [np.float16, np.float32])
@pytest.mark.parametrize("depth,group,hkv,rows,lens,window", [
    (64, 32, 8, (2100,), (2100,), 200), (128, 128, 8, (2100,), (2300,), 90), (256, 64, 8, (1100, 1100), (1100, 1300), 40)])
def test_columns_of_no_numbers_in_most_tiles_of_many_rows(gpu_ctx, io, depth, group, hkv, rows, lens, window):
    """Windows shorter than a block of rows, so that every tile has a column that some row does not see: tiles with marked
    columns and without, in every order one and two tiles apart, call after call."""
    rng = np.random.default_rng(depth + window)
    lay = ref.Layout(hkv, depth, group, 64)
    step = ref.Step.make(lay, rows, lens, rng)
    raw = step.random_cache(rng)
    q = rng.normal(size=(step.total, hkv, depth))
    held, groups, wide = raw.copy(), depth // group, 32 if depth == 256 else 64
    vparams = lay.pages(held)["vparams"]
    want, cu = np.zeros(q.shape, bool), step.cu
    for i, n in enumerate(lens):
        page, row = step.columns_of(i)
        for head, tile in np.argwhere(rng.random((hkv, n // wide)) < 0.4):
            column, g = wide * tile + int(rng.integers(wide)), int(rng.integers(groups))
            vparams[page[column], head, row[column] // 4, g, tile & 1, row[column] % 4] = (np.nan, np.inf)[head & 1]
            p = np.arange(n - rows[i], n)
            sees = np.flatnonzero((p >= column) & (p - column < window))
            want[cu[i] + sees, head, g * group:(g + 1) * group] = True
    assert 0.05 < want.mean() < 0.95
    a = Attention(gpu_ctx, step, held, q, io, window)
    sound, reach, top = step.attention(raw, a.q, a.half_scale, window)
    most, _ = tolerance(io, reach, top, window)
    first = None
    for _ in range(12):
        a.out.upload(np.full(a.out.nbytes // np.dtype(io).itemsize, 77, io))
        a.run()
        got = a.result()
        assert np.array_equal(np.isfinite(got), ~want)
        assert np.abs(got.astype(np.float64) - sound)[~want].max() <= most
        first = got.tobytes() if first is None else first
        assert got.tobytes() == first
    assert not a.faulted()
    a.free()


@pytest.mark.parametrize("out_dtype", [np.float16, np.float32])
@pytest.mark.parametrize("depth,hkv", [(64, 1), (128, 3), (256, 2)])
def test_all_rows_of_a_refused_sequence_read_as_nan(gpu_ctx, out_dtype, depth, hkv):
    """Also those that the call's limit of rows a sequence leaves no workgroup for; others, and rows of no sequence, as
    they would be."""
    ctx, rng = gpu_ctx, np.random.default_rng(depth + hkv)
    rows, lens = (2, 75, 0, 3), (20, 90, 0, 40)
    step = ref.Step.make(ref.Layout(hkv, depth, 32, 16), rows, lens, rng)
    cache, table, cu, n = up(ctx, step.random_cache(rng), step.table, step.cu, np.int32(lens))
    fault, out = ctx.zeros(16), [ctx.alloc((step.total + 1) * hkv * depth * np.dtype(out_dtype).itemsize) for _ in range(2)]

    def read(lengths, offsets=step.cu, **change):
        n.upload(np.int32(lengths))
        cu.upload(np.int32(offsets))
        fault.zero()
        for o in out:
            o.upload(np.full((step.total + 1) * hkv * depth, 7, out_dtype))
        ctx.kv4_read(cache, table, cu, n, *out, fault=fault, out_dtype=IO[out_dtype], **{**step.shape(), **change})
        return [o.download(out_dtype, (step.total + 1, hkv * depth)) for o in out], fault.download(np.uint32, (1,))[0]

    good, faulted = read(lens)
    assert not faulted and all(np.all(np.isfinite(g)) and np.all(g[-1] == 7) for g in good)
    refused = np.r_[np.zeros(2, bool), np.ones(75, bool), np.zeros(4, bool)]
    for lengths, change in (((20, 74, 0, 40), {}), ((20, 16 * step.table.shape[1] + 1, 0, 40), {}), ((20, -1, 0, 40), {}),
                            (lens, dict(max_query=3))):
        got, faulted = read(lengths, **change)
        assert faulted == 1
        for g, whole in zip(got, good):
            assert np.all(np.isnan(g[refused])) and g[~refused].tobytes() == whole[~refused].tobytes(), (lengths, change)
    for offsets in ((0, 2, 99, 77, 80), (0, 2, -1, 77, 80)):   # no rows of its own
        got, faulted = read((20, 90, 0, 40), offsets, max_query=3)
        assert faulted == 1
        for g, whole in zip(got, good):
            assert g[:2].tobytes() == whole[:2].tobytes() and g[77:].tobytes() == whole[77:].tobytes()
            assert np.all(g[2:77] == 7)
    free(cache, table, cu, n, fault, *out)


def check_by_row(step, raw, a, classes):
    """Each row against its own error, and the 2-norm of each class of rows against what independent roundings give.

    fp16 rows: values are rounded to fp16 once, which the reference does too, and so is the result; f32 rows: values are
    known to 2^-22.  Beside what the scores' errors move (attention_by_row), weights are known to 2^-22, exp2 and the scale
    to as much, and at most 64 + log2(columns) sums come in a row, each rounding by 2^-23.
    2-norm: the result's rounding is that of the reference's result, 10 % more for classes of a thousand elements; the rest
    is independent roundings of 2^-25 rms, 8 in a row of a score's size and of as many sums as there are columns, whose
    sizes add up to sqrt(columns) times their sum's.  (A plane of keys or of weights left out, so that they are rounded to
    fp16, is 1.15 to 1.9 times that and more.)"""
    half = a.io == np.float16
    want, moved, size, top = ref.attention_by_row(step, raw, a.q, a.half_scale, a.window, a.io if half else np.float64)
    got = a.result().astype(np.float64)
    span = max(step.lens)
    most = moved + top * (4 * 2.0**-22 + (64 + np.log2(span)) * 2.0**-23)
    if half:
        most = most + 2.0**-11 * (np.abs(want) + most) + 2.0**-25
    assert np.all(np.isfinite(got))
    assert np.all(np.abs(got - want) <= most), np.argwhere(np.abs(got - want) > most)[:5]
    told = 0
    for name in sorted(set(classes)):
        mine = np.array([c == name for c in classes])
        other = 2.0**-22 + 2.0**-25 * (8 * np.sqrt((size[mine] ** 2).mean()) + 16 * np.sqrt(span))
        norm = np.linalg.norm(want[mine])
        if other > 0.01:   # (scores that f32 cannot tell apart: the rows' own limits are all that there is)
            told += np.mean(moved[mine] < 1e-6 * top) > 0.5
            continue
        share = other + (1.1 * np.linalg.norm(want[mine].astype(np.float16) - want[mine]) / norm if half else 0.0)
        told += 1
        assert np.linalg.norm(got[mine] - want[mine]) <= share * norm, (name, share)
    assert told == len(set(classes))
    assert not a.faulted()


# Rows and heads for the kernel of few rows, and blocks enough for that of many.
FEW, MANY = (2, 4, (3, 18), (70, 500)), (2, 32, (260, 9), (300, 120))


@pytest.mark.parametrize("io", [np.float16, np.float32])
@pytest.mark.parametrize("depth,group,page", [(64, 32, 16), (128, 64, 128), (128, 128, 32), (256, 32, 64)])
@pytest.mark.parametrize("rows", ["few", "many"])
def test_each_row_is_within_its_own_error(gpu_ctx, io, depth, group, page, rows):
    """Rows of queries of all sizes beside each other, zeros among them, in both kernels."""
    rng = np.random.default_rng(depth + group + page)
    hkv, share, n, lens = FEW if rows == "few" else MANY
    step = ref.Step.make(ref.Layout(hkv, depth, group, page), n, lens, rng)
    raw = step.random_cache(rng)
    sizes = (1.0, 1e-3, 300.0, 0.0, 8.0) + ((1e4, 1e-6) if io == np.float16 else (1e4, 1e-30))
    classes = [sizes[i % len(sizes)] for i in range(step.total)]
    q = np.clip(rng.normal(size=(step.total, hkv * share, depth)), -4.0, 4.0)   # (fp16 ends at 65504)
    a = Attention(gpu_ctx, step, raw, q * np.array(classes)[:, None, None], io)
    a.run()
    check_by_row(step, raw, a, classes)
    a.free()


@pytest.mark.parametrize("io", [np.float16, np.float32])
@pytest.mark.parametrize("depth,group,page", [(64, 64, 64), (128, 32, 16), (256, 128, 256)])
@pytest.mark.parametrize("rows", ["few", "many"])
@pytest.mark.parametrize("spread,window", [(1e-4, 0), (1.0, 90), (30.0, 0)])
def test_keys_and_values_of_all_sizes_in_both_kernels(gpu_ctx, io, depth, group, page, rows, spread, window):
    """Steps and minima among fp16's subnormals, and in the hundreds."""
    rng = np.random.default_rng(depth + group)
    hkv, share, n, lens = FEW if rows == "few" else MANY
    step = ref.Step.make(ref.Layout(hkv, depth, group, page), n, lens, rng)
    raw = step.random_cache(rng, spread)
    a = Attention(gpu_ctx, step, raw, rng.normal(size=(step.total, hkv * share, depth)), io, window)
    a.run()
    check_by_row(step, raw, a, ["all"] * step.total)
    a.free()


@pytest.mark.parametrize("io", [np.float16, np.float32])
@pytest.mark.parametrize("depth,group,page", [(64, 32, 16), (128, 64, 128), (256, 128, 64)])
@pytest.mark.parametrize("rows", ["few", "many"])
def test_scores_past_what_f32_can_tell_apart(gpu_ctx, io, depth, group, page, rows):
    """Up to f32 queries of 1e33, and fp16 ones of 65504 beside keys of thousands: neighbouring f32 numbers are more than a
    weight's range apart there, and the largest column still has the weight."""
    rng = np.random.default_rng(depth + page)
    hkv, share, n, lens = FEW if rows == "few" else MANY
    step = ref.Step.make(ref.Layout(hkv, depth, group, page), n, lens, rng)
    sizes = (1.0, 30.0, 100.0, 300.0, 1e3, 3e3, 16376.0) if io == np.float16 else (1.0, 100.0, 1e3, 1e5, 1e7, 1e20, 2.5e31)
    for spread, half_scale in ((500.0, 1.0), (1.0, None)):
        raw = step.random_cache(rng, spread)
        if half_scale is None and io == np.float32:
            sizes = tuple(10 * x for x in sizes)
        classes = [sizes[i % len(sizes)] for i in range(step.total)]
        q = np.clip(rng.normal(size=(step.total, hkv * share, depth)), -4.0, 4.0) * np.array(classes)[:, None, None]
        a = Attention(gpu_ctx, step, raw, q, io, half_scale=half_scale)
        a.run()
        check_by_row(step, raw, a, classes)
        a.free()


@pytest.mark.parametrize("io", [np.float16, np.float32])
def test_lengths_that_mean_nothing_change_nothing(gpu_ctx, io):
    """Entries of a padded batch, whatever their lengths say, take no part in how the others' columns are dealt: the same
    bits, and as many workgroups for the sequences that have rows."""
    rng = np.random.default_rng(95)
    rows, lens = (0, 0, 1, 0, 0, 1, 0, 0), (0, 0, 333, 0, 0, 40000, 0, 0)
    step = ref.Step.make(ref.Layout(2, 64, 32, 64), rows, lens, rng)
    a = Attention(gpu_ctx, step, step.random_cache(rng), rng.normal(size=(2, 8, 64)), io)
    a.run()
    good = a.result()
    assert np.all(np.isfinite(good))
    for other in (40000, 2**31 - 1, -7):
        a.buf["lens"].upload(np.int32([n if r else other for r, n in zip(rows, lens)]))
        a.run()
        assert a.result().tobytes() == good.tobytes() and not a.faulted()
    a.free()


@pytest.mark.parametrize("io", [np.float16, np.float32])
def test_single_rows_are_dealt_by_their_own_lengths_beside_prompts(gpu_ctx, io):
    """In a step of both kinds, single rows' bits do not hang on how far the prompts beside them have come."""
    rng = np.random.default_rng(96)
    lay, heads = ref.Layout(8, 64, 32, 64), 32
    rows, full = (1, 200, 1, 200, 1), (2500, 2600, 40, 2600, 900)
    step = ref.Step.make(lay, rows, full, rng)
    raw, q = step.random_cache(rng), rng.normal(size=(step.total, heads, 64))
    a, singles, got = Attention(gpu_ctx, step, raw, q, io), [0, 201, 402], []
    for prompts in (200, 1000, 2600):
        now = ref.Step(lay, rows, [n if r == 1 else prompts for r, n in zip(rows, full)], step.pages, step.table)
        a.buf["lens"].upload(np.int32(now.lens))
        a.run()
        got.append(a.result()[singles])
        want, reach, top = now.attention(raw, a.q, a.half_scale)
        assert np.abs(a.result() - want).max() <= tolerance(io, reach, top, 2600)[0]
        assert got[-1].tobytes() == got[0].tobytes()
    assert not a.faulted()
    a.free()


@pytest.mark.parametrize("io", [np.float16, np.float32])
@pytest.mark.parametrize("cu", [(0, 1, 30, 5), (0, 1, 30, -2**31), (0, 1, 30, 2**31 - 1)])
def test_offsets_that_are_none_leave_the_others_their_rows(gpu_ctx, io, cu):
    """With limits as large as they may be: what the words of such an entry multiply to is no measure of work."""
    rng = np.random.default_rng(97)
    step = ref.Step.make(ref.Layout(2, 64, 32, 16), (1, 29, 0), (1500, 40, 0), rng)
    a = Attention(gpu_ctx, step, step.random_cache(rng), rng.normal(size=(30, 8, 64)), io, max_columns=2**31 - 1)
    a.run()
    good = a.result()
    assert np.all(np.isfinite(good)) and not a.faulted()
    a.buf["cu"].upload(np.int32(cu))
    a.buf["lens"].upload(np.int32((1500, 40, 2**31 - 1)))
    a.out.upload(np.full(a.out.nbytes // np.dtype(io).itemsize, 77, io))
    a.run()
    assert a.result().tobytes() == good.tobytes() and a.faulted()
    a.free()
