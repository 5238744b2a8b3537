"""The FP8 products' kernels of tiles, each at sizes that the rule sends to it (asserted by the plan): against 64 bits,
with rows and features that end inside a tile and reduced axes that end inside a block."""
import ctypes as C

import numpy as np
import pytest

import fp8_ref as ref
import litemind_amd as lm
from conftest import announce
from litemind_amd import workload as wl
from test_gpu_fp8 import TYPES, Groups, Out, fp8_matrix, fp8_rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = lm.Context(wl.V2_LITE.moe_config(num_layers=1))
    yield c
    c.close()


def copy_in(ctx, at, host):
    host = np.ascontiguousarray(host)
    ctx._check(ctx.lib.lm_copy_h2d(ctx.handle, C.c_void_p(at), host.ctypes.data_as(C.c_void_p), host.nbytes))


def copy_out(ctx, at, shape, dtype=np.float32):
    host = np.empty(shape, dtype)
    ctx._check(ctx.lib.lm_copy_d2h(ctx.handle, host.ctypes.data_as(C.c_void_p), C.c_void_p(at), host.nbytes))
    return host


def test_larger_tiles_where_small_ones_are_too_many(ctx):
    """512 experts of 2^20 features, a row each: tiles of 32 x 128 would be more than a launch has room for."""
    announce("fp8 grouped gemm, 2^20 features by 512 groups")
    groups, n, k = 512, 2 ** 20, 16
    plan = lm.fp8_plan_gemm(groups, n, k, groups=groups)
    assert (plan.tile_rows, plan.tile_features) == (128, 256)
    rng = np.random.default_rng(90)
    a, sa = fp8_rows(rng, groups, k)
    w, sw = fp8_matrix(rng, 512, k)  # the last rows of two of the matrices
    dw, dsw = ctx.empty((groups, n, k), np.uint8).zero(), ctx.empty((groups, n // 128)).zero()
    y = ctx.empty((groups, n)).zero()
    for e in (3, groups - 1):
        copy_in(ctx, dw.ptr + ((e + 1) * n - 512) * k, w)
        copy_in(ctx, dsw.ptr + 4 * ((e + 1) * n // 128 - 4), sw)
    g = Groups(ctx, np.arange(groups + 1), groups)
    ctx.fp8_grouped_gemm(g.c, ctx.to_device(a), ctx.to_device(sa), groups, dw, dsw, n, k, y, groups)
    ctx.synchronize()
    for e in (3, groups - 1):
        got = copy_out(ctx, y.ptr + 4 * ((e + 1) * n - 600), (1, 600))
        assert (got[0, :88] == 0).all()
        ref.check_product(got[:, 88:], *ref.product(a[e:e + 1], sa[e:e + 1], w, sw), "f32", e)
    for b in (dw, dsw, y):
        b.free()


def test_matrix_in_several_calls(ctx):
    """A matrix quantized from a multiple of 128 rows on: the same codes and scales as in one call."""
    announce("fp8 quantize, a matrix in two calls")
    rows, width, first = 700, 208, 384
    x = np.random.default_rng(91).standard_normal((rows, width)).astype(np.float32)
    dx, q, s = ctx.to_device(x), ctx.empty((rows, width), np.uint8), ctx.empty((6, 2))
    for at, n in ((0, first), (first, rows - first)):
        ctx.fp8_quantize(dx.ptr + 4 * at * width, n, width, q.ptr + at * width, s.ptr + 4 * at // 128 * 2, block_rows=128)
    want_q, want_s = ref.quantize(x, 128)
    assert (q.download() == want_q).all() and (s.download() == want_s).all()
