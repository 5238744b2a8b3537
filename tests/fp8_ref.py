"""Plain restatements of the FP8 operators (include/litemind_fp8.h) in numpy: blocks bit for bit in fp32, products in
64 bits with a bound of what fp32 sums may be off by."""
import numpy as np

BLOCK = 128
NAN = 0x7F


def _table():
    code = np.arange(256)
    exponent, mantissa = (code >> 3) & 15, code & 7
    value = np.where(exponent == 0, mantissa * 2.0 ** -9, (8 + mantissa) * 2.0 ** (exponent - 10.0))
    value[(code & 127) == 127] = np.nan
    return np.where(code & 128, -value, value)


VALUES = _table()
POSITIVE = VALUES[:127]  # 0 .. 448, rising


def blocks(n):
    return -(-n // BLOCK)


def widen(x):
    """fp32 values of fp32, fp16 or BF16 bits (uint16)."""
    return (x.astype(np.uint32) << 16).view(np.float32) if x.dtype == np.uint16 else x.astype(np.float32)


def encode(v):
    """Nearest e4m3 code of each value of magnitude under 464, ties to the even code; NaN is 0x7f."""
    m = np.abs(v).astype(np.float64)
    above = np.clip(np.searchsorted(POSITIVE, m), 0, 126)
    below = np.maximum(above - 1, 0)
    up, down = POSITIVE[above] - m, m - POSITIVE[below]
    code = np.where((up < down) | ((up == down) & (above % 2 == 0)), above, below).astype(np.uint8)
    code |= np.where(np.signbit(v), 0x80, 0).astype(np.uint8)
    return np.where(np.isnan(v), NAN, code).astype(np.uint8)


def quantize(x, block_rows=1):
    """Codes and scales of x [rows][width]: the scales in fp32; 448 x / m in 64 bits is a middle between two codes where
    it is one, and else, 2^-29 of itself away, on the right side of it."""
    x = widen(x)
    rows, width = x.shape
    tall, wide = -(-rows // block_rows), blocks(width)
    padded = np.zeros((tall * block_rows, wide * BLOCK), np.float32)
    padded[:rows, :width] = x
    padded = padded.reshape(tall, block_rows, wide, BLOCK)
    finite = np.isfinite(padded)
    most = np.where(finite, np.abs(padded), np.float32(0)).max((1, 3))
    scale = np.maximum(most / np.float32(448), np.float32(2.0 ** -126))
    least = most < np.float32(448 * 2.0 ** -126)
    m = np.where(least, 448 * 2.0 ** -126, most.astype(np.float64))[:, None, :, None]
    v = np.where(finite, padded, np.float32(0)).astype(np.float64) * 448 / m
    q = np.where(finite, encode(v), NAN).astype(np.uint8)
    return q.reshape(tall * block_rows, wide * BLOCK)[:rows, :width].copy(), scale


def dequantize(q, scale, block_rows=1):
    rows, width = q.shape
    return VALUES[q] * scale.astype(np.float64)[np.arange(rows) // block_rows][:, np.arange(width) // BLOCK]


def product(a, a_scale, w, w_scale, dtype="f32"):
    """a . w^T in 64 bits, and the most that its sums may be off by: a block's 128 additions and the blocks' sums (one
    product of scales and one addition each, and at most 32 joins) each lose at most a step, 2^-23, of the sum of
    magnitudes, whether the matrix cores round or cut. For outputs of 16 bits the FP8 matrix cores cut the products of
    eight neighbouring channels 13 bits under their largest exponent: seven of them lose less than 2^-13 of the eighth."""
    x, y = dequantize(a, a_scale), dequantize(w, w_scale, BLOCK)
    steps = BLOCK + 2 * blocks(a.shape[1]) + 32 + (0 if dtype == "f32" else 7 * 2 ** 10)
    with np.errstate(invalid="ignore"):
        return x @ y.T, np.nan_to_num(np.abs(x), nan=0.0) @ np.nan_to_num(np.abs(y), nan=0.0).T * steps * 2.0 ** -23


def swiglu(a, a_scale, gate, gate_scale, up, up_scale):
    """gate / (1 + e^-gate) up in 64 bits, and the most that fp32 may be off by."""
    g, dg = product(a, a_scale, gate, gate_scale)
    u, du = product(a, a_scale, up, up_scale)
    with np.errstate(over="ignore", invalid="ignore"):
        sigmoid = 1.0 / (1.0 + np.exp(-g))
        act = g * sigmoid * u
        # the exponential is off by 2^-23 (2 + |g|) of itself, of which 1 - sigmoid reaches the quotient, the quotient
        # and the two products by 4 steps more; quotients under 2^-126 may be 0; |d silu / dg| <= 1.1
        own = np.abs(act) * 2.0 ** -23 * ((2 + np.abs(g)) * (1 - sigmoid) + 6) + np.abs(g * u) * 2.0 ** -125
        return act, own + 1.1 * dg * np.abs(u) + np.abs(g * sigmoid) * du + 1.1 * dg * du + 2.0 ** -126


def check_blocks(q, scale, value, off, what=""):
    """Codes and scales of rows [rows][width] whose exact values are `value`, computed to within `off`."""
    rows, width = value.shape
    for b in range(blocks(width)):
        at = slice(b * BLOCK, min(width, (b + 1) * BLOCK))
        v, d, s = value[:, at], off[:, at], scale[:, b].astype(np.float64)
        good = np.isfinite(v)
        most = np.where(good, np.abs(v), 0).max(1)
        slack = np.where(good, d, 0).max(1) / 448 + most / 448 * 2.0 ** -23
        assert (np.abs(s - np.maximum(most / 448, 2.0 ** -126)) <= slack).all(), (what, b)
        got = VALUES[q[:, at]] * s[:, None]
        # half an e4m3 step of the value: 2^-4 of it, at least 2^-10 scales; and two fp32 roundings before it
        room = np.maximum(np.abs(v) * 2.0 ** -4, s[:, None] * 2.0 ** -10) * (1 + 2.0 ** -20) + d + np.abs(v) * 2.0 ** -22
        # the largest value may lie past 448 scales by what the scale is off by
        room = room + 448 * slack[:, None]
        bad = good & ~(np.abs(got - v) <= room)
        assert not bad.any(), (what, b, np.argwhere(bad)[:3], got[bad][:3], v[bad][:3])
        assert (np.isnan(got) == ~good).all(), (what, b)


def bf16(x):
    """BF16 bits of fp32 values, rounded to nearest even."""
    u = np.asarray(x, np.float32).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
LEAST_STEP = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}  # half the least subnormal


def check_product(got, want, off, dtype, what=""):
    """An output of `dtype` against want +- off."""
    y = widen(got).astype(np.float64)
    bad = np.isnan(want)
    assert (np.isnan(y) == bad).all(), what
    room = off + (np.abs(want) + off) * HALF_STEP[dtype] + LEAST_STEP[dtype]
    d = np.abs(y - want)
    assert (d[~bad] <= room[~bad]).all(), (what, float(np.max((d - room)[~bad])), float(np.max(d[~bad])))
