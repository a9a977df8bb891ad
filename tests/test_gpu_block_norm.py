"""The norms around a block with gate and scaled residual, and a layer's run of them with products of 4-bit rows."""
import numpy as np
import pytest

import karume_amd as ka
import mx4_reference as ref
from test_gpu_mx4 import CODE, Guarded, activations, guarded, weights

pytestmark = pytest.mark.gpu


def run(gpu, rows, dim, *, io="f32", norm=None, post=True, gate=None, span=0, residual=True, pre=True, total=True,
        eps=1e-5, scales=(0.22, 0.95), shift=0, sum_in=None, norm_in=None, seed=0, size=1.0):
    """One call held to its bounds; sum_in / norm_in: "y" or "residual", whose place the output takes."""
    norm = norm or io
    rng = np.random.default_rng(seed * 77 + rows * 13 + dim)
    t, nt = ref.NUMPY[io], ref.NUMPY[norm]
    eb, nb = t().nbytes, nt().nbytes
    y = (size * rng.standard_normal((rows, dim))).astype(t)
    host = {"y": y, "residual": (3 * activations(rng, rows, dim, np.float32)).astype(t) if residual else None}
    dev = {name: None if a is None else guarded(gpu, a, shift=shift * eb) for name, a in host.items()}
    wpost = (1 + 0.2 * rng.standard_normal(dim)).astype(np.float32) if post else None
    wpre = (1 + 0.2 * rng.standard_normal(dim)).astype(np.float32) if pre else None
    g = None
    if gate:
        g = rng.standard_normal((-(-rows // span) if span else 1, dim)).astype(t)
    out = {"sum": None, "norm": None}
    if total:
        out["sum"] = dev[sum_in] if sum_in else Guarded(gpu, rows * dim * eb, shift=shift * eb)
    if pre:
        out["norm"] = dev[norm_in] if norm_in else Guarded(gpu, rows * dim * nb, shift=shift * nb)
    at = lambda b: None if b is None else int(b)  # noqa: E731
    up = lambda a: None if a is None else int(guarded(gpu, a, shift=shift * a.itemsize))  # noqa: E731
    keep = [guarded(gpu, a, shift=shift * a.itemsize) if a is not None else None for a in (wpost, wpre, g)]
    gpu.block_norm(int(dev["y"]), rows=rows, dim=dim, post_weight=at(keep[0]), gate=at(keep[2]), gate_span=span,
                   gate_kind=ka.GATE_SIGMOID if gate == "sigmoid" else ka.GATE_PLAIN, residual=at(dev["residual"]),
                   pre_weight=at(keep[1]), sum_out=at(out["sum"]), norm_out=at(out["norm"]), eps=eps,
                   block_scale=scales[0], residual_scale=scales[1], io_dtype=CODE[io], norm_dtype=CODE[norm])
    f = lambda a: None if a is None else a.astype(np.float64)  # noqa: E731
    if g is not None:
        g = g[np.arange(rows) // span if span else np.zeros(rows, dtype=int)]
    a, b = (np.float64(np.float32(s)) for s in scales)
    first, second = ref.block_norm(f(y), f(wpost), f(g), gate == "sigmoid", f(host["residual"]), f(wpre),
                                   np.float64(np.float32(eps)), a, b, io, norm)
    if total:
        ref.check(out["sum"].read(t, (rows, dim)), *first, "sum")
    if pre:
        ref.check(out["norm"].read(nt, (rows, dim)), *second, "norm")
    for name, d in dev.items():
        if d is not None and d is not out["sum"] and d is not out["norm"]:
            assert np.array_equal(d.read(t, (rows, dim)), host[name]), name


DIMS = [1, 2, 7, 8, 63, 64, 100, 512, 513, 520, 1000, 1024, 1032, 2048, 2304, 4096, 4100, 5632, 8192, 8200, 11008,
        16383, 16384]


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("io,norm", [("f16", "f16"), ("f32", "f32"), ("f32", "f16")])
def test_rows_of_every_length(gpu_ctx, dim, io, norm):
    run(gpu_ctx, 3, dim, io=io, norm=norm, gate="sigmoid", span=2)
    run(gpu_ctx, 5, dim, io=io, norm=norm, shift=1, gate="plain", span=1, post=False)


@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("gate,span", [(None, 0), ("plain", 0), ("plain", 3), ("sigmoid", 1), ("sigmoid", 100)])
@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("pre,total", [(True, True), (True, False), (False, True)])
def test_what_is_not_given_is_left_out(gpu_ctx, post, gate, span, residual, pre, total):
    for io, dim in (("f16", 264), ("f32", 131)):
        run(gpu_ctx, 7, dim, io=io, post=post, gate=gate, span=span, residual=residual, pre=pre, total=total)


@pytest.mark.parametrize("sum_in,norm_in", [("residual", None), ("y", None), (None, "y"), (None, "residual"),
                                            ("residual", "y"), ("y", "residual")])
@pytest.mark.parametrize("dim", [96, 1001, 9000])
def test_outputs_in_the_place_of_inputs(gpu_ctx, sum_in, norm_in, dim):
    for io in ("f16", "f32"):
        run(gpu_ctx, 9, dim, io=io, sum_in=sum_in, norm_in=norm_in)
    if norm_in is None:
        run(gpu_ctx, 9, dim, io="f32", norm="f16", sum_in=sum_in)


def test_many_rows(gpu_ctx):
    run(gpu_ctx, 3001, 160, io="f16")
    run(gpu_ctx, 70001, 8, io="f32", gate="plain", span=7)


def test_small_and_zero_rows(gpu_ctx):
    """Rows whose squares meet eps, rows of zeros, and an eps of zero."""
    run(gpu_ctx, 4, 512, io="f32", size=1e-4, eps=1e-6)
    run(gpu_ctx, 4, 512, io="f32", size=0.0)
    run(gpu_ctx, 4, 512, io="f32", eps=0.0)


def test_what_is_no_number_stays_in_its_row(gpu_ctx):
    rng = np.random.default_rng(1)
    y = rng.standard_normal((5, 264)).astype(np.float16)
    r = rng.standard_normal((5, 264)).astype(np.float16)
    y[1, 7], r[3, 200] = np.nan, np.inf
    w = gpu_ctx.upload(np.ones(264, dtype=np.float32))
    s, n = gpu_ctx.zeros(y.nbytes), gpu_ctx.zeros(y.nbytes)
    gpu_ctx.block_norm(gpu_ctx.upload(y), rows=5, dim=264, post_weight=w, residual=gpu_ctx.upload(r), pre_weight=w,
                       sum_out=s, norm_out=n, io_dtype=ka.F16)
    s, n = s.download(np.float16, y.shape), n.download(np.float16, y.shape)
    assert np.isnan(s[1]).all() and np.isnan(n[1]).all()
    assert np.isinf(s[3, 200]) and np.isfinite(s[3, :200]).all() and np.isnan(n[3, 200]) and not n[3, :200].any()
    for good in (0, 2, 4):
        assert np.isfinite(s[good]).all() and np.isfinite(n[good]).all()


def test_refusals(gpu_ctx):
    buf = gpu_ctx.zeros(1 << 16)
    at = int(buf)
    good = dict(rows=2, dim=64, residual=at + 4096, pre_weight=at + 8192, sum_out=at + 12288, norm_out=at + 16384)
    for kw in (dict(dim=0), dict(dim=16385), dict(io_dtype=2), dict(norm_dtype=9), dict(io_dtype=ka.F16, norm_dtype=ka.F32),
               dict(gate_kind=2), dict(norm_out=None), dict(pre_weight=None), dict(sum_out=None, norm_out=None, pre_weight=None),
               dict(sum_out=at + 12289), dict(residual=at + 2), dict(pre_weight=at + 2), dict(post_weight=at + 1),
               dict(gate=at + 3), dict(norm_out=at + 12288), dict(norm_dtype=ka.F16, norm_out=at),
               dict(norm_dtype=ka.F16, norm_out=at + 4096), dict(norm_out=at + 16385), dict(gate=at + 12288),
               dict(gate=at + 16384, gate_span=1)):
        with pytest.raises(ka.GpuValidationError):
            gpu_ctx.block_norm(at, **{**good, **kw})
    with pytest.raises(ka.GpuValidationError):
        gpu_ctx.block_norm(None, **good)
    gpu_ctx.block_norm(at, **{**good, "rows": 0})
    assert not buf.download(np.uint8, (1 << 16,)).any()


@pytest.mark.parametrize("m", [1, 6, 70])
def test_a_layers_feed_forward(gpu_ctx, m):
    """The norm behind the attention and in front of the feed-forward block, gate and up, the product down, and the norm
    behind it, recorded and replayed: each step against the definition over what the step before it left."""
    rng = np.random.default_rng(m)
    dim, inner = 416, 1056
    w1, s1 = weights(rng, 2 * inner, dim)
    w2, s2 = weights(rng, dim, inner)
    post, pre, last = ((1 + 0.2 * rng.standard_normal(dim)).astype(np.float32) for _ in range(3))
    d = {name: gpu_ctx.upload(a) for name, a in dict(w1=w1, s1=s1, w2=w2, s2=s2, post=post, pre=pre, last=last).items()}
    wide = max(dim, inner)
    for name, width in (("y", dim), ("stream", dim), ("normed", dim), ("act", inner), ("down", dim), ("out", dim),
                        ("next", dim)):
        d[name] = gpu_ctx.zeros(m * width * 2)
    d["xq"], d["xs"] = gpu_ctx.zeros(m * wide // 2), gpu_ctx.zeros(m * wide // 32)
    f16 = dict(io_dtype=ka.F16)

    def layer():
        g = gpu_ctx
        g.block_norm(d["y"], rows=m, dim=dim, post_weight=d["post"], residual=d["stream"], pre_weight=d["pre"],
                     sum_out=d["stream"], norm_out=d["normed"], **f16)
        g.linear_mx4_fused(d["normed"], d["w1"], d["s1"], d["act"], m, 2 * inner, dim, xq=d["xq"], xs=d["xs"],
                           x_dtype=ka.F16, out_dtype=ka.F16, epilogue=ka.EPILOGUE_SILU_PAIRS)
        g.linear_mx4_fused(d["act"], d["w2"], d["s2"], d["down"], m, dim, inner, xq=d["xq"], xs=d["xs"],
                           x_dtype=ka.F16, out_dtype=ka.F16, scale_rule=ka.MX4_CEIL)
        g.block_norm(d["down"], rows=m, dim=dim, post_weight=d["last"], residual=d["stream"], pre_weight=d["pre"],
                     sum_out=d["out"], norm_out=d["next"], block_scale=0.5, residual_scale=0.5, **f16)

    layer()
    gpu_ctx.sync()
    with gpu_ctx.record() as rec:
        layer()
    for _ in range(3):
        y, stream = (rng.standard_normal((m, dim)).astype(np.float16) for _ in range(2))
        d["y"].upload(y)
        d["stream"].upload(stream)
        rec.graph.launch()
        gpu_ctx.sync()
        got = {n: d[n].download(np.float16, (m, inner if n == "act" else dim)) for n in
               ("stream", "normed", "act", "down", "out", "next")}
        v = {n: a.astype(np.float64) for n, a in got.items()}
        first, second = ref.block_norm(y.astype(np.float64), post, None, False, stream.astype(np.float64), pre,
                                       np.float64(np.float32(1e-5)), 1.0, 1.0, "f16", "f16")
        ref.check(got["stream"], *first)
        ref.check(got["normed"], *second)
        ref.check(got["act"], *ref.product(ref.values(*ref.quantised(v["normed"], False)), ref.values(w1, s1), None, None,
                                           True, "f16"))
        ref.check(got["down"], *ref.product(ref.values(*ref.quantised(v["act"], True)), ref.values(w2, s2), None, None,
                                            False, "f16"))
        first, second = ref.block_norm(v["down"], last, None, False, v["stream"], pre, np.float64(np.float32(1e-5)), 0.5, 0.5,
                                       "f16", "f16")
        ref.check(got["out"], *first)
        ref.check(got["next"], *second)
    rec.graph.destroy()
