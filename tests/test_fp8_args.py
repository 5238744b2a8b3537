"""What the FP8 operators refuse (no GPU calls: every argument is checked before the context)."""
import ctypes as C

import pytest

import litemind_amd as lm

A, SA, W, SW, OUT, S2, IDX = (0x100000000 * i for i in range(1, 8))  # addresses that are never followed, far apart


def refused(status):
    assert status == -1
    return lm.load_library().lm_last_error().decode()


def quantize(**kw):
    v = dict(x=A, dtype=lm.DT_F32, rows=5, width=300, stride=300, block_rows=1, q=OUT, scale=S2)
    v.update(kw)
    return lm.load_library().lm_fp8_quantize(None, v["x"], v["dtype"], v["rows"], v["width"], v["stride"],
                                             v["block_rows"], v["q"], v["scale"])


def groups(kw):
    g = lm.Fp8Groups(groups=8, rows=100, offsets=IDX)
    for k in list(kw):
        if k in ("groups", "rows_of_groups", "offsets", "source", "divisor", "target"):
            setattr(g, "rows" if k == "rows_of_groups" else k, kw.pop(k))
    return g


def gemm(**kw):
    v = dict(a=A, sa=SA, rows=5, w=W, sw=SW, n=300, k=144, out=OUT, dtype=lm.DT_F32)
    v.update(kw)
    return lm.load_library().lm_fp8_gemm(None, v["a"], v["sa"], v["rows"], v["w"], v["sw"], v["n"], v["k"], v["out"],
                                         v["dtype"])


def grouped(**kw):
    g = C.byref(groups(kw)) if not kw.pop("no_groups", False) else None
    v = dict(a=A, sa=SA, rows=100, w=W, sw=SW, n=300, k=144, out=OUT, out_rows=100, dtype=lm.DT_BF16)
    v.update(kw)
    return lm.load_library().lm_fp8_grouped_gemm(None, g, v["a"], v["sa"], v["rows"], v["w"], v["sw"], v["n"], v["k"],
                                                 v["out"], v["out_rows"], v["dtype"])


def swiglu(**kw):
    g = C.byref(groups(kw)) if not kw.pop("no_groups", False) else None
    v = dict(a=A, sa=SA, rows=100, w=W, sw=SW, n=272, k=144, q=OUT, s=S2)
    v.update(kw)
    return lm.load_library().lm_fp8_grouped_swiglu(None, g, v["a"], v["sa"], v["rows"], v["w"], v["sw"], v["n"],
                                                   v["k"], v["q"], v["s"])


@pytest.mark.parametrize("call", [quantize, gemm, grouped, swiglu])
def test_good_arguments_reach_the_context(call):
    assert "null context" in refused(call())
    empty = {"rows": 0} if call in (quantize, gemm) else {"rows_of_groups": 0}
    assert "null context" in refused(call(**empty))


def test_good_edges():
    for kw in (dict(block_rows=128), dict(width=2 ** 24, stride=2 ** 24, rows=1), dict(rows=2 ** 31 - 1, width=1, stride=1, x=A, q=A + 2 ** 34, scale=A + 2 ** 36),
               dict(dtype=lm.DT_F16, x=A + 2), dict(rows=(2 ** 23) - 128, width=1, stride=1, block_rows=128)):
        assert "null context" in refused(quantize(**kw))
    assert "null context" in refused(gemm(k=2 ** 20, n=1, rows=1))
    assert "null context" in refused(grouped(source=IDX * 2, divisor=6, target=IDX * 3))
    assert "null context" in refused(swiglu(source=IDX * 2, divisor=1, groups=512))


@pytest.mark.parametrize("bad", [
    dict(dtype=0), dict(dtype=lm.DT_I8), dict(block_rows=0), dict(block_rows=64), dict(rows=-1), dict(rows=2 ** 31),
    dict(rows=2 ** 23, block_rows=128), dict(width=0), dict(width=2 ** 24 + 1, stride=2 ** 24 + 1), dict(stride=299),
    dict(stride=2 ** 28 + 1), dict(x=None), dict(x=A + 2), dict(x=A + 1, dtype=lm.DT_BF16), dict(q=None),
    dict(q=OUT + 8), dict(scale=None), dict(scale=S2 + 2), dict(q=A), dict(q=A + 16), dict(scale=A + 5996),
    dict(scale=OUT + 1496), dict(x=A, q=A - 16)], ids=str)
def test_quantize(bad):
    assert "null context" not in refused(quantize(**bad))


PRODUCT = [dict(a=None), dict(a=A + 8), dict(sa=None), dict(sa=SA + 1), dict(w=None), dict(w=W + 4), dict(sw=None),
           dict(sw=SW + 2), dict(n=0), dict(n=2 ** 24 + 16), dict(k=0), dict(k=8), dict(k=24), dict(k=2 ** 20 + 16),
           dict(k=-16), dict(rows=-1), dict(rows=2 ** 31), dict(rows=2 ** 28, k=16), dict(n=2 ** 22, k=1024)]
OUTPUT = [dict(out=None), dict(out=OUT + 4), dict(dtype=0), dict(dtype=lm.DT_F64), dict(out=A), dict(out=W + 16),
          dict(out=SA), dict(out=SW), dict(out=A - 16)]
GROUPS = [dict(no_groups=True), dict(groups=0), dict(groups=513), dict(groups=-1), dict(rows_of_groups=-1),
          dict(rows_of_groups=2 ** 31), dict(offsets=None), dict(offsets=IDX + 1), dict(source=IDX * 2),
          dict(source=IDX * 2, divisor=-1), dict(divisor=1), dict(source=IDX * 2 + 2, divisor=1), dict(target=IDX + 3),
          dict(rows=0)]


@pytest.mark.parametrize("bad", PRODUCT + OUTPUT, ids=str)
def test_gemm(bad):
    assert "null context" not in refused(gemm(**bad))


@pytest.mark.parametrize("bad", PRODUCT + OUTPUT + GROUPS + [dict(out_rows=0), dict(out_rows=-1), dict(out_rows=2 ** 31),
                                                            dict(out=IDX), dict(target=OUT, out_rows=1)], ids=str)
def test_grouped_gemm(bad):
    assert "null context" not in refused(grouped(**bad))


@pytest.mark.parametrize("bad", PRODUCT + GROUPS + [
    dict(q=None), dict(q=OUT + 8), dict(s=None), dict(s=S2 + 2), dict(q=A), dict(q=W), dict(s=SA), dict(s=OUT),
    dict(q=IDX), dict(target=IDX * 2), dict(n=24), dict(n=8), dict(n=2 ** 20 + 16),
    dict(rows_of_groups=2 ** 28, n=16), dict(n=2 ** 19, k=4096)], ids=str)
def test_swiglu(bad):
    assert "null context" not in refused(swiglu(**bad))


def test_messages():
    assert "multiple of 16" in refused(gemm(k=40))
    assert "divisor" in refused(grouped(divisor=2))
    assert "target" in refused(swiglu(target=IDX * 2))
    assert "overlap" in refused(gemm(out=A))
