"""The plain restatements that the FP8 operators' GPU tests compare with (no GPU calls)."""
import numpy as np
import pytest

import fp8_ref as ref


def test_codes_are_e4m3():
    assert ref.VALUES[0x7E] == 448 and ref.VALUES[0xFE] == -448 and ref.VALUES[0x01] == 2.0 ** -9
    assert ref.VALUES[0x38] == 1.0 and ref.VALUES[0x08] == 2.0 ** -6
    assert np.isnan(ref.VALUES[0x7F]) and np.isnan(ref.VALUES[0xFF])
    assert (np.diff(ref.POSITIVE) > 0).all()


def test_codes_round_to_nearest_even():
    codes = np.arange(126)
    middle = ((ref.VALUES[codes] + ref.VALUES[codes + 1]) / 2).astype(np.float32)
    assert (ref.encode(middle) == codes + codes % 2).all()
    assert (ref.encode(np.nextafter(middle, np.float32(0))) == codes).all()
    assert (ref.encode(np.nextafter(middle, np.float32(500))) == codes + 1).all()
    assert (ref.encode(ref.VALUES[codes].astype(np.float32)) == codes).all()
    assert (ref.encode(-middle) == (codes + codes % 2) | 0x80).all()


@pytest.mark.parametrize("block_rows", [1, 128])
def test_blocks(block_rows):
    x = np.random.default_rng(1).standard_normal((300, 200)).astype(np.float32)
    x[3, :128] = 0
    q, s = ref.quantize(x, block_rows)
    assert s.shape == (-(-300 // block_rows), 2)
    assert np.abs(ref.dequantize(q, s, block_rows) - x).max() <= np.abs(x).max() * 2.0 ** -4 * 1.0001
    if block_rows == 1:
        assert s[3, 0] == np.float32(2.0 ** -126) and (q[3, :128] == 0).all()


def test_not_finite():
    x = np.ones((1, 128), np.float32)
    x[0, :3] = [np.nan, np.inf, -np.inf]
    q, s = ref.quantize(x)
    assert (q[0, :3] & 0x7F == 0x7F).all() and (q[0, 3:] == 0x7E).all() and s[0, 0] == np.float32(1) / np.float32(448)


def test_checks_see_a_mistake():
    rng = np.random.default_rng(2)
    a, sa = ref.quantize(rng.standard_normal((5, 300)).astype(np.float32))
    w, sw = ref.quantize(rng.standard_normal((130, 300)).astype(np.float32), 128)
    y, off = ref.product(a, sa, w, sw)
    good = y.astype(np.float32)
    ref.check_product(good, y, off, "f32")
    for wrong in (np.roll(good, 1, 1), np.where(np.arange(130) == 129, 0, good).astype(np.float32)):
        with pytest.raises(AssertionError):
            ref.check_product(wrong, y, off, "f32")
    act, d = ref.swiglu(a, sa, w, sw, w[::-1].copy(), sw)
    q, s = ref.quantize(act.astype(np.float32))
    ref.check_blocks(q, s, act, d)
    q[2, 77] += 3
    with pytest.raises(AssertionError):
        ref.check_blocks(q, s, act, d)
