"""The FP8 products' kernels of tiles, each at sizes that the rule sends to it (asserted by the plan): against 64 bits,
with rows and features that end inside a tile and reduced axes that end inside a block."""
import ctypes as C

import numpy as np
import pytest

import fp8_ref as ref
import litemind_amd as lm
from conftest import announce
from litemind_amd import workload as wl
from test_gpu_fp8 import TYPES, Groups, Out, fp8_matrix, fp8_rows, quantized
from test_gpu_fp8_run import Product
from test_gpu_serving_run import Hip

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


# ---- one matrix ----

def rows_of(ctx, rng, rows, width):
    return quantized(ctx, (rng.standard_normal((rows, width)) * np.exp(rng.uniform(-1, 1, (rows, 1)))).astype(np.float32))


def matrix_of(ctx, rng, rows, width):
    return quantized(ctx, (rng.standard_normal((rows, width)) * 0.05).astype(np.float32), block_rows=128)


def check_norms(got, want, dtype):
    """Outputs of 16 bits: the FP8 matrix cores' sums are off by 4e-5 of their norm, a row's by at most twice that, and
    their rounding by half a step of each. (One scale block less of 65 would be off by an eighth.)"""
    good = np.isfinite(want).all(1)
    y, want = ref.widen(got)[good].astype(np.float64), want[good]
    room = (8e-5 + ref.HALF_STEP[dtype]) * np.linalg.norm(want, axis=1)
    assert (np.linalg.norm(y - want, axis=1) <= room).all()


def gemm(ctx, a, w, dtype):
    (a, sa), (w, sw) = a, w
    y = Out(ctx, (len(a), len(w)), TYPES[dtype][1])
    held = [ctx.to_device(v) for v in (a, sa, w, sw)]
    ctx.fp8_gemm(held[0], held[1], len(a), held[2], held[3], len(w), a.shape[1], y.ptr, dtype=TYPES[dtype][0])
    got = y.read()
    for h in held:
        h.free()
    return got


# rows, features, reduced channels, output, tile, whether the reduced axis is shared
GEMM = [(100, 8200, 144, "f32", (32, 128), False), (65, 4100, 656, "f32", (32, 128), False),
        (33, 2600, 2064, "f32", (32, 128), False), (33, 1290, 4112, "f32", (32, 128), True),
        (400, 5130, 144, "f32", (64, 128), False), (400, 5130, 656, "f32", (64, 128), False),
        (400, 5130, 1520, "f32", (64, 128), False), (300, 2056, 6016, "f32", (64, 128), True),
        (3000, 1290, 144, "f32", (128, 128), False), (3000, 1290, 656, "f32", (128, 128), False),
        (3000, 1030, 1424, "f32", (128, 128), False), (4100, 130, 6016, "f32", (128, 128), True),
        (3000, 5130, 6064, "f32", (128, 256), False),
        (100, 8200, 144, "bf16", (32, 128), False), (65, 4100, 656, "f16", (32, 128), False),
        (33, 2600, 2064, "bf16", (32, 128), False), (33, 1290, 4112, "f16", (32, 128), True),
        (400, 5130, 144, "bf16", (64, 128), False), (400, 5130, 1424, "f16", (64, 128), False),
        (1300, 130, 6016, "bf16", (64, 128), True), (3000, 1290, 656, "bf16", (128, 128), False),
        (3000, 1290, 1424, "f16", (128, 128), False), (1000, 2056, 6016, "bf16", (128, 128), True),
        (1930, 2056, 8208, "bf16", (128, 256), False), (1000, 8200, 272, "bf16", (256, 256), False),
        (1000, 8200, 656, "f16", (256, 256), False), (1000, 8200, 1424, "bf16", (256, 256), False)]


def planned(rows, n, k, dtype, tile, shared=False, groups=0):
    p = lm.fp8_plan_gemm(rows, n, k, TYPES[dtype][0], groups=groups)
    assert (p.tile_rows, p.tile_features) == tile and (p.shares > 1) == shared


@pytest.mark.parametrize("rows,n,k,dtype,tile,shared", GEMM)
def test_gemm(ctx, rows, n, k, dtype, tile, shared):
    announce(f"fp8 gemm {rows} x {n} x {k} {dtype}, tiles of {tile}")
    planned(rows, n, k, dtype, tile, shared)
    rng = np.random.default_rng(rows + 1000 * n + k)
    a, w = rows_of(ctx, rng, rows, k), matrix_of(ctx, rng, n, k)
    got = gemm(ctx, a, w, dtype)
    want, off = ref.product(*a, *w, dtype)
    ref.check_product(got, want, off, dtype, (rows, n, k))
    if dtype != "f32":
        check_norms(got, want, dtype)


def with_nan(rng, q, every):
    """Codes with NaN at the end and at the beginning of some rows: a row's last block is followed in memory by the next
    row's first."""
    q = q.copy()
    at = rng.permutation(len(q))[:max(2, len(q) // every)]
    half = len(at) // 2
    q[at[:half], -1] = 0x7F
    q[at[half:], 0] = 0xFF
    return q


@pytest.mark.parametrize("rows,n,k,dtype,tile,shared", [c for c in GEMM if c[2] % 128 != 0 and c[2] > 500])
def test_gemm_nan(ctx, rows, n, k, dtype, tile, shared):
    announce(f"fp8 gemm with NaN {rows} x {n} x {k} {dtype}, tiles of {tile}")
    planned(rows, n, k, dtype, tile, shared)
    rng = np.random.default_rng(5 + rows)
    (a, sa), (w, sw) = rows_of(ctx, rng, rows, k), matrix_of(ctx, rng, n, k)
    a, w = with_nan(rng, a, 9), with_nan(rng, w, 40)
    got = gemm(ctx, (a, sa), (w, sw), dtype)
    want, off = ref.product(a, sa, w, sw, dtype)
    assert 0 < np.isnan(want).sum() < want.size / 2
    ref.check_product(got, want, off, dtype, (rows, n, k))


@pytest.mark.parametrize("rows,n,k,tile", [(65, 4100, 656, (32, 128)), (400, 5130, 656, (64, 128)), (3000, 1290, 656, (128, 128))])
def test_gemm_extreme_scales(ctx, rows, n, k, tile):
    announce(f"fp8 gemm with extreme scales {rows} x {n} x {k}, tiles of {tile}")
    planned(rows, n, k, "f32", tile)
    rng = np.random.default_rng(6)
    (a, sa), (w, sw) = rows_of(ctx, rng, rows, k), matrix_of(ctx, rng, n, k)
    sa, sw = ((s * 10.0 ** rng.uniform(-15, 15, s.shape)).astype(np.float32) for s in (sa, sw))
    a[7] = 0
    w[100] = 0x80
    got = gemm(ctx, (a, sa), (w, sw), "f32")
    assert (got[7] == 0).all() and (got[:, 100] == 0).all()
    ref.check_product(got, *ref.product(a, sa, w, sw), "f32")


# ---- by groups ----

def ragged(rng, groups, rows):
    """Sizes of groups, some of them empty and one of a single row."""
    share = rng.exponential(size=groups) ** 1.5
    share[rng.permutation(groups)[:max(1, groups // 4)]] = 0
    sizes = rng.multinomial(rows - 1, share / share.sum())
    sizes[np.flatnonzero(sizes == 0)[0]] = 1
    return sizes


class Experts:
    """Groups of ragged sizes whose rows are gathered (three of a row of a) and scattered, with NaN in some rows and in the
    last rows of one expert's matrices."""

    def __init__(self, ctx, groups, rows, n, k, parts=1, extra=3):
        rng = self.rng = np.random.default_rng(rows + n + k)
        self.ctx, self.n, self.k, self.rows, self.parts = ctx, n, k, rows, parts
        self.sizes = ragged(rng, groups, rows - extra)  # rows - extra.. are behind the last group
        self.offsets = np.concatenate([[0], np.cumsum(self.sizes)]).astype(np.int32)
        self.used = int(self.offsets[-1])
        self.source = rng.permutation(rows).astype(np.int32)
        self.target = rng.permutation(rows + 5)[:rows].astype(np.int32)
        self.a, self.sa = rows_of(ctx, rng, -(-rows // 3), k)
        self.a = with_nan(rng, self.a, 50)
        self.w, self.sw = [], []
        for _ in range(groups):
            pair = [matrix_of(ctx, rng, n, k) for _ in range(parts)]
            self.w.append(np.stack([q for q, _ in pair]))
            self.sw.append(np.stack([s for _, s in pair]))
        self.w[groups // 2][-1, -1, 0] = 0x7F
        self.held = [ctx.to_device(v) for v in (self.a, self.sa, np.stack(self.w), np.stack(self.sw))]

    def free(self):
        for h in self.held:
            h.free()

    def each(self):
        for e, size in enumerate(self.sizes):
            if size:
                at = slice(self.offsets[e], self.offsets[e + 1])
                yield e, at, self.source[at] // 3


# groups, rows, features, reduced channels, output, tile
GROUPED = [(4, 1040, 130, 1424, "f32", (32, 128)), (8, 6400, 130, 144, "f32", (32, 128)), (6, 4800, 130, 656, "f32", (64, 128)),
           (6, 4800, 130, 1424, "f32", (64, 128)), (64, 16640, 130, 144, "f32", (128, 128)),
           (20, 8000, 130, 656, "f32", (128, 128)), (20, 8000, 130, 1424, "f32", (128, 128)),
           (16, 1600, 2056, 4112, "f32", (128, 256)), (4, 1040, 130, 1424, "bf16", (32, 128)),
           (6, 4800, 130, 1424, "f16", (64, 128)), (20, 8000, 130, 1424, "bf16", (128, 128)),
           (16, 1600, 2056, 4112, "f16", (128, 256)), (160, 41600, 130, 144, "bf16", (256, 256)),
           (20, 16000, 130, 2064, "bf16", (256, 256))]


@pytest.mark.parametrize("groups,rows,n,k,dtype,tile", GROUPED)
def test_grouped_gemm(ctx, groups, rows, n, k, dtype, tile):
    announce(f"fp8 grouped gemm, {groups} groups, {rows} rows, {n} x {k} {dtype}, tiles of {tile}")
    planned(rows, n, k, dtype, tile, groups=groups)
    x = Experts(ctx, groups, rows, n, k)
    y = Out(ctx, (rows + 5, n), TYPES[dtype][1])
    before = y.host[:y.bytes].view(y.dtype).reshape(y.shape)
    g = Groups(ctx, x.offsets, rows, source=x.source, divisor=3, target=x.target)
    ctx.fp8_grouped_gemm(g.c, x.held[0], x.held[1], len(x.a), x.held[2], x.held[3], n, k, y.ptr, rows + 5,
                         dtype=TYPES[dtype][0])
    ctx.synchronize()
    got = y.read()
    for e, at, src in x.each():
        want, off = ref.product(x.a[src], x.sa[src], x.w[e][0], x.sw[e][0], dtype)
        ref.check_product(got[x.target[at]], want, off, dtype, e)
        if dtype != "f32":
            check_norms(got[x.target[at]], want, dtype)
    rest = np.setdiff1d(np.arange(rows + 5), x.target[:x.used])
    assert (got[rest].view(np.uint8) == before[rest].view(np.uint8)).all()
    x.free()


@pytest.mark.parametrize("what", ["source", "negative source", "target", "offsets", "past rows", "negative offset"])
@pytest.mark.parametrize("groups,rows,n,k,dtype,tile", [GROUPED[0], GROUPED[2], GROUPED[5], GROUPED[12]])
def test_bad_indexes(ctx, groups, rows, n, k, dtype, tile, what):
    """Indexes outside their range in tiles: reported once, the rows of a good group come out right."""
    announce(f"fp8 grouped gemm, bad {what}, tiles of {tile}")
    planned(rows, n, k, dtype, tile, groups=groups)
    x = Experts(ctx, groups, rows, n, k)
    source, target, offsets = x.source.copy(), x.target.copy(), x.offsets.copy()
    first = int(np.flatnonzero(x.sizes)[0])
    row = int(offsets[first])
    if what == "source":
        source[row] = 3 * len(x.a)
    elif what == "negative source":
        source[row] = -2 ** 31
    elif what == "target":
        target[row] = 2 ** 30
    elif what == "offsets":
        offsets[1] = rows + 10 ** 6
    elif what == "past rows":
        offsets[-1] = 2 ** 31 - 1
    else:
        offsets[0] = -5
    y = Out(ctx, (rows + 5, n), TYPES[dtype][1])
    g = Groups(ctx, offsets, rows, source=source, divisor=3, target=target)
    ctx.fp8_grouped_gemm(g.c, x.held[0], x.held[1], len(x.a), x.held[2], x.held[3], n, k, y.ptr, rows + 5,
                         dtype=TYPES[dtype][0])
    with pytest.raises(lm.LmError) as e:
        ctx.synchronize()
    assert e.value.status == -5 and "index" in str(e.value)
    ctx.synchronize()  # once
    got = y.read()
    if what != "offsets":
        middle = [e for e in range(first + 1, groups - 1) if x.sizes[e]]
        for e, at, src in x.each():
            if e in middle:
                want, off = ref.product(x.a[src], x.sa[src], x.w[e][0], x.sw[e][0], dtype)
                ref.check_product(got[x.target[at]], want, off, dtype, (what, e))
    x.free()


@pytest.mark.parametrize("groups,rows,inter,k,kernel", [
    (8, 2080, 144, 656, 1), (8, 2080, 144, 1424, 1), (6, 4800, 144, 656, 2), (6, 4800, 144, 1424, 2), (2, 800, 1408, 656, 2),
    (20, 8000, 144, 656, 3), (6, 4800, 144, 2064, 3), (20, 8000, 144, 144, 3)])
def test_grouped_swiglu(ctx, groups, rows, inter, k, kernel):
    announce(f"fp8 grouped swiglu, {groups} groups, {rows} rows, {inter} x {k}, kernel {kernel}")
    assert lm.fp8_plan_swiglu(groups, rows, inter, k).kernel == kernel
    x = Experts(ctx, groups, rows, inter, k, parts=2)
    q, s = Out(ctx, (rows, inter), np.uint8), Out(ctx, (rows, ref.blocks(inter)), np.float32)
    g = Groups(ctx, x.offsets, rows, source=x.source, divisor=3)
    ctx.fp8_grouped_swiglu(g.c, x.held[0], x.held[1], len(x.a), x.held[2], x.held[3], inter, k, q.ptr, s.ptr)
    ctx.synchronize()
    q, s = q.read(), s.read()
    for e, at, src in x.each():
        act, off = ref.swiglu(x.a[src], x.sa[src], x.w[e][0], x.sw[e][0], x.w[e][1], x.sw[e][1])
        ref.check_blocks(q[at], s[at], act, off, e)
    assert (q[x.used:] == 0xA5).all() and (s[x.used:].view(np.uint8) == 0xA5).all()
    x.free()


# ---- shared sums ----

SHARES = [(200, 512, 6016), (300, 640, 10944), (33, 515, 10944)]  # the last one's rows * features are no multiple of 4


def shared_product(ctx, seed, size):
    assert lm.fp8_plan_gemm(*size).shares > 1
    return Product(ctx, seed, *size)


def test_captured_shares(ctx):
    announce("fp8 gemm: shared sums, captured")
    hip = Hip(ctx)
    runs = [shared_product(ctx, 30 + i, size) for i, size in enumerate(SHARES[:2])]
    other = shared_product(ctx, 40, SHARES[2])
    for r in runs + [other]:
        r.run()
    graphs = [hip.capture(r.run) for r in runs]
    try:
        for _ in range(4):
            for r, (_, runnable) in zip(runs, graphs):
                r.y.upload(np.full((r.rows, r.n), np.nan, np.float32))
                hip.replay(runnable)
                other.run()
            for r in runs + [other]:
                r.check()
    finally:
        for g in graphs:
            hip.free(*g)


def test_two_contexts_share():
    """Two contexts' shared sums at once, each in its own workspace."""
    announce("fp8: shared sums of two contexts at once")
    with lm.Context(wl.V2_LITE.moe_config(num_layers=1)) as c, lm.Context(wl.V2_LITE.moe_config(num_layers=1)) as d:
        products = [shared_product(x, 70 + i, SHARES[i]) for i, x in enumerate((c, d))]
        for p in products:
            p.run()
        for x in (c, d):
            x.synchronize()
        for _ in range(20):
            for p in products:
                p.run()
        for p in products:
            p.check()
