"""Blocks of 32 e2m1 numbers with a power of two each, their products and the norms around a block, in 64 bits and
from the definitions alone."""
import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
HALF_STEP = {"f16": 2.0 ** -11, "f32": 2.0 ** -24}
NUMPY = {"f16": np.float16, "f32": np.float32}
# a number below the smallest normal one is off by at most half of the smallest subnormal
TINY_STEP = {"f16": 2.0 ** -25, "f32": 2.0 ** -150}


def unpack(codes):
    """[..., k/2] bytes -> [..., k] codes."""
    return np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1)


def values(codes, scales):
    """f64 values of packed codes and scale bytes."""
    c = unpack(codes)
    v = np.where(c & 8, -GRID[c & 7], GRID[c & 7])
    scale = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return (v.reshape(*scales.shape, 32) * scale[..., None]).reshape(v.shape)


def quantised(x, ceil):
    """(packed codes, scale bytes) of f64 rows, element by element from the nearest code."""
    blocks = np.asarray(x, dtype=np.float64).reshape(x.shape[0], -1, 32)
    top = np.abs(blocks).max(-1)
    bad = ~np.isfinite(blocks).all(-1)
    _, exponent = np.frexp(np.where(bad, 1.0, top))          # top = m 2^exponent, 0.5 <= m < 1
    power = exponent - 3
    if ceil:
        power = np.where(top > 6 * np.exp2(power.astype(np.float64)), power + 1, power)
    power = np.where(top == 0, -127, np.maximum(power, -127))
    v = np.where(bad[..., None], 0.0, blocks) / np.exp2(power.astype(np.float64))[..., None]
    away = np.abs(np.abs(v)[..., None] - GRID)
    least = away.min(-1, keepdims=True)
    near = away == least                                     # one code, or two at a tie
    even = near & (np.arange(8) % 2 == 0)
    code = np.where(even.any(-1), even.argmax(-1), near.argmax(-1))
    code = (code | np.where(np.signbit(v), 8, 0)).astype(np.uint8)
    code[bad] = 0
    code = code.reshape(x.shape)
    return code[:, 0::2] | (code[:, 1::2] << 4), np.where(bad, 255, power + 127).astype(np.uint8)


def silu(g):
    t = np.exp(-np.abs(g))
    return g * np.where(g < 0, t / (1 + t), 1 / (1 + t))


def product(xv, wv, bias, residual, pairs, out):
    """(f64 result, how far a result in `out` may be off).

    A block's 32 products are multiples of a quarter of its two scales, 36 at most: 14 bits, so that their sum is exact
    in f32.  The k / 32 sums of blocks and the joining of up to 64 parts round by 2^-24 of what they have so far, which
    the sum of magnitudes bounds."""
    sums, sizes = xv @ wv.T, np.abs(xv) @ np.abs(wv).T
    off = (xv.shape[1] / 32 + 64) * 2.0 ** -24 * sizes
    if bias is not None:
        sums = sums + bias
        off = off + 2.0 ** -24 * np.abs(sums)
    if pairs:
        g, u, og, ou = sums[:, 0::2], sums[:, 1::2], off[:, 0::2], off[:, 1::2]
        s = silu(g)
        # |silu'| <= 1.1; the exponential is off by two steps, the four operations by half a step each
        off = (1.1 * og + 6 * 2.0 ** -24 * np.abs(s)) * (np.abs(u) + ou) + np.abs(s) * ou
        sums = s * u
        off = off + 2.0 ** -24 * np.abs(sums)
    if residual is not None:
        sums = sums + residual
        off = off + 2.0 ** -24 * np.abs(sums)
    return sums, off * 1.001 + HALF_STEP[out] * np.abs(sums) + TINY_STEP[out]


def block_norm(y, post, gate, sigmoid, residual, pre, eps, block_scale, residual_scale, io, norm):
    """((sum, off), (norm, off)) in 64 bits; `gate` has a row for each of y's."""
    dim, u = y.shape[1], 2.0 ** -24
    t, rel = y, 0.0
    # a mean of squares: 16 sums in a thread, 6 over the lanes, 16 over the waves, a quotient and eps; its root halves
    # that, and the root, the reciprocal and two products follow
    rms_rel = (40 / 2 + 5) * u
    if post is not None:
        t = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * post
        rel = rms_rel
    if gate is not None:
        # the logistic: an exponential of two steps and two operations
        t = t * (1 / (1 + np.exp(-gate)) if sigmoid else gate)
        rel = rel + (6 if sigmoid else 1) * u
    part = block_scale * t
    total = part + (0 if residual is None else residual_scale * residual)
    off = np.abs(part) * (rel + 2 * u) + u * np.abs(total)
    if residual is not None:
        off = off + u * np.abs(residual_scale * residual)
    off = off * 1.001
    first = total, off + HALF_STEP[io] * np.abs(total) + TINY_STEP[io]
    if pre is None:
        return first, None
    root = np.sqrt((total * total).mean(-1, keepdims=True) + eps)
    # the root's own change with what the sums are off by
    shift = np.sqrt((off * off).mean(-1, keepdims=True)) / root
    out = total / root * pre
    off = off / root * np.abs(pre) + np.abs(out) * (rms_rel + shift)
    return first, (out, off * 1.001 + HALF_STEP[norm] * np.abs(out) + TINY_STEP[norm])


def check(got, want, off, what=""):
    """Every number within its own bound; NaN where the definition has NaN."""
    got = got.astype(np.float64)
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan), what
    over = ~nan & (np.abs(got - want) > off)
    assert not over.any(), (what, int(over.sum()), got[over][:4], want[over][:4], off[over][:4])
