"""FP8 blocks of fp16 and BF16 values at their extremes and where two codes meet: these types find a block's largest
magnitude two to a word, and choose the even of two codes by themselves."""
import numpy as np
import pytest

import fp8_ref as ref
import litemind_amd as lm
from conftest import announce
from litemind_amd import workload as wl
from test_gpu_fp8 import as_type, quantized

pytestmark = pytest.mark.gpu

# widths of 16-byte loads, of scalar ones, and of scalar ones by their stride
LAYOUTS = [(384, 0), (381, 0), (376, 379)]
INFINITY = {"f16": 0x7C00, "bf16": 0x7F80}
NAN = {"f16": 0x7E00, "bf16": 0x7FC0}
LARGEST = {"f16": 0x7BFF, "bf16": 0x7F7F}


@pytest.fixture(scope="module")
def ctx():
    c = lm.Context(wl.V2_LITE.moe_config(num_layers=1))
    yield c
    c.close()


def same(ctx, bits, dtype, block_rows, stride=0):
    """Values given by their bits, [rows][width]."""
    x = bits.view(np.float16) if dtype == "f16" else bits
    q, s = quantized(ctx, x, dtype, block_rows, stride)
    want_q, want_s = ref.quantize(x, block_rows)
    assert (s == want_s).all()
    assert (q == want_q).all(), np.argwhere(q != want_q)[:4]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("width,stride", LAYOUTS)
def test_extremes(ctx, width, stride, block_rows, dtype):
    """Zeros, subnormals, the largest values, and infinities and NaN in either half of a word."""
    announce(f"fp8 quantize extremes {dtype} {width} stride {stride}, blocks of {block_rows}")
    kinds = 14
    rng = np.random.default_rng(3)
    x = as_type(rng.standard_normal((kinds * block_rows, width)).astype(np.float32), dtype).view(np.uint16)
    each = x.reshape(kinds, block_rows, width)
    each[0] = 0
    each[1] = 0x8000
    each[2] = rng.integers(0, 16, each[2].shape) | 0x8000 * rng.integers(0, 2, each[2].shape)  # subnormals
    each[3] = rng.integers(0, 0x90, each[3].shape)  # subnormals and the least normal values
    each[4, 0, :2] = [LARGEST[dtype], 0x8000 | LARGEST[dtype]]
    each[5, -1, 4] = INFINITY[dtype]
    each[6, 0, 131] = 0x8000 | INFINITY[dtype]
    each[7, 0, 6] = NAN[dtype]
    each[8, -1, 135] = 0x8000 | NAN[dtype]
    each[9, 0, 2:6] = [INFINITY[dtype] + 1, LARGEST[dtype], INFINITY[dtype], 0xFFFF]  # a NaN of the least payload, of the largest
    each[10] = INFINITY[dtype]
    each[11] = NAN[dtype]
    each[12, :, ::2] = 0
    each[12, 0, 0] = INFINITY[dtype]
    each[13, 0, 1:128] = 0
    each[13, 0, 0] = 1
    same(ctx, x, dtype, block_rows, stride)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("width,stride", LAYOUTS)
def test_next_to_middles(ctx, width, stride, block_rows, dtype):
    """Values at the middle of two codes, where the type has them, and up to two steps away, for largest magnitudes of all
    kinds: powers of two times 7 (every middle is a value), whole numbers, and any."""
    announce(f"fp8 quantize next to the middles {dtype} {width} stride {stride}, blocks of {block_rows}")
    rng = np.random.default_rng(5)
    low, high = (-6, 7) if dtype == "f16" else (-110, 100)
    most = np.concatenate([7 * 2.0 ** rng.integers(low, high, 40), rng.integers(1, 256, 40) * 2.0 ** rng.integers(low, high - 5, 40),
                           rng.uniform(1, 2, 60) * 2.0 ** rng.integers(low, high, 60)])
    most = ref.widen(as_type(most.astype(np.float32), dtype)).astype(np.float64)
    middle = (ref.POSITIVE[:-1] + ref.POSITIVE[1:]) / 2
    x = np.zeros((len(most), block_rows, width), np.uint16)
    row = as_type((middle * most[:, None] / 448).astype(np.float32), dtype).view(np.uint16).astype(np.int32)
    for b in range(2):  # a block a row: five places from a middle in turn
        step = rng.integers(-2, 3, row.shape)
        value = np.clip(row + step, 0, None) | 0x8000 * rng.integers(0, 2, row.shape)
        at = slice(128 * b + 1, 128 * b + 127)
        x[:, rng.integers(0, block_rows), at] = value.astype(np.uint16)
        x[:, 0, 128 * b] = as_type(most.astype(np.float32), dtype).view(np.uint16)
    same(ctx, x.reshape(-1, width), dtype, block_rows, stride)
