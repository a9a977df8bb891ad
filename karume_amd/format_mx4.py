"""Blocks of 32 e2m1 numbers that share a power of two — host-side packing of weights.

Layout (that of the device entry points): an element is a nibble (sign, two bits of exponent, one of
mantissa: 0, 0.5, 1, 1.5, 2, 3, 4, 6), element 2j of a row in the low nibble of its byte j; scale byte
E of each 32 elements stands for 2^(E - 127), 255 for NaN.  ``pack_mx4`` gives the bytes that
``GpuContext.quantize_mx4`` gives for the same f32 rows.
"""
from __future__ import annotations

from typing import Tuple

import numpy as np

MX4_BLOCK = 32
_EDGES = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=np.float32)


class Mx4Error(ValueError):
    """The rows cannot be stored in blocks of 32."""


def pack_mx4(values: np.ndarray, *, ceil: bool = False) -> Tuple[np.ndarray, np.ndarray]:
    """(codes uint8 [rows, k / 2], scales uint8 [rows, k / 32]) of f32 rows [rows, k].

    A block's largest magnitude comes to stand in [4, 8) and is clipped above 6, or with ``ceil`` in
    (3, 6]; a block that holds an infinity or a NaN has scale 255 and codes 0.
    """
    rows = np.ascontiguousarray(values, dtype=np.float32)
    if rows.ndim != 2 or rows.shape[1] == 0 or rows.shape[1] % MX4_BLOCK:
        raise Mx4Error(f"rows of shape {rows.shape} are not [rows, a multiple of {MX4_BLOCK}]")
    blocks = rows.reshape(rows.shape[0], -1, MX4_BLOCK)
    top = np.ascontiguousarray(np.abs(blocks)).view(np.uint32).max(-1)   # NaN and infinity are the largest
    bad = top >= 0x7F800000
    byte = (top >> 23).astype(np.int64) - 2
    if ceil:
        byte += (top & 0x7FFFFF) > 0x400000
    byte = np.where(bad, 127, np.maximum(byte, 0))
    with np.errstate(invalid="ignore", over="ignore"):
        # (exact: a power of two, and the quotient is below 8)
        size = np.ldexp(blocks, (127 - byte).astype(np.int32)[..., None])
    code = np.zeros(size.shape, dtype=np.uint8)
    for i, edge in enumerate(_EDGES):       # a tie goes to the even code
        code += np.abs(size) >= edge if i % 2 else np.abs(size) > edge
    code |= np.signbit(size).astype(np.uint8) << 3
    code[bad] = 0
    code = code.reshape(rows.shape)
    scales = np.where(bad, 255, byte).astype(np.uint8)
    return code[:, 0::2] | (code[:, 1::2] << 4), scales
