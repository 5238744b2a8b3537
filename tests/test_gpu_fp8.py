"""FP8 blocks and products on the GPU against their restatements in 64 bits."""
import numpy as np
import pytest

import fp8_ref as ref
import litemind_amd as lm
from conftest import announce
from litemind_amd import workload as wl

pytestmark = pytest.mark.gpu

TYPES = {"f32": (lm.DT_F32, np.float32), "f16": (lm.DT_F16, np.float16), "bf16": (lm.DT_BF16, np.uint16)}
GUARD = 64


@pytest.fixture(scope="module")
def ctx():
    c = lm.Context(wl.V2_LITE.moe_config(num_layers=1))
    yield c
    c.close()


def as_type(x, dtype):
    return ref.bf16(x) if dtype == "bf16" else x.astype(TYPES[dtype][1])


class Out:
    """An output on the GPU, filled, with guard bytes behind it."""

    def __init__(self, ctx, shape, dtype, fill=0xA5):
        self.shape, self.dtype = shape, np.dtype(dtype)
        self.bytes = int(np.prod(shape)) * self.dtype.itemsize
        self.host = np.full(self.bytes + GUARD, fill, np.uint8)
        self.dev = ctx.to_device(self.host)
        self.ptr = self.dev.ptr

    def read(self):
        raw = self.dev.download()
        assert (raw[self.bytes:] == self.host[self.bytes:]).all(), "written past the end"
        self.dev.free()
        return raw[:self.bytes].view(self.dtype).reshape(self.shape)


def quantized(ctx, x, dtype="f32", block_rows=1, stride=0):
    rows, width = x.shape
    held = x
    if stride:
        held = np.full((rows, stride), 3e4, x.dtype)  # what lies between the rows does not count
        held[:, :width] = x
    d = ctx.to_device(held)
    q, s = Out(ctx, (rows, width), np.uint8), Out(ctx, (-(-rows // block_rows), ref.blocks(width)), np.float32)
    ctx.fp8_quantize(d, rows, width, q.ptr, s.ptr, dtype=TYPES[dtype][0], row_stride=stride, block_rows=block_rows)
    got = q.read(), s.read()
    d.free()
    return got


# ---- blocks ----

@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,width,stride", [(1, 1, 0), (1, 2048, 0), (3, 128, 0), (2, 7, 0), (5, 129, 0), (17, 200, 208),
                                               (129, 256, 0), (130, 1408, 1411), (257, 136, 0), (64, 10944, 0),
                                               (33, 1000, 1001), (2, 16384, 0)])
def test_quantize(ctx, rows, width, stride, block_rows, dtype):
    announce(f"fp8 quantize {rows} x {width} stride {stride} {dtype}, blocks of {block_rows}")
    rng = np.random.default_rng(rows * 7919 + width + block_rows)
    x = as_type((rng.standard_normal((rows, width)) * 10.0 ** rng.uniform(-3, 3, (rows, 1))).astype(np.float32), dtype)
    q, s = quantized(ctx, x, dtype, block_rows, stride)
    want_q, want_s = ref.quantize(x, block_rows)
    assert (s == want_s).all()
    assert (q == want_q).all()


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_extremes(ctx, block_rows):
    """Zeros, subnormals, the largest values, NaN and infinities, and values halfway between two codes."""
    announce(f"fp8 quantize extremes, blocks of {block_rows}")
    rows = 12 if block_rows == 1 else 12 * 128
    x = np.random.default_rng(3).standard_normal((rows, 384)).astype(np.float32)
    each = x.reshape(12, block_rows, 384)
    each[0] = 0
    each[1, :, :128] = -0.0
    each[2] *= np.float32(1e-42)
    each[3] *= np.float32(1e-38)
    each[4] *= np.float32(1e38)
    each[4].flat[:2] = [np.finfo(np.float32).max, -np.finfo(np.float32).max]
    each[5].flat[5] = np.nan
    each[6].flat[[1, 130]] = [np.inf, -np.inf]
    each[7] = np.nan
    each[8] = np.inf
    halfway = (ref.POSITIVE[:-1] + ref.POSITIVE[1:]) / 2
    each[9, 0, :128] = np.r_[448.0, halfway, 0.0].astype(np.float32)
    each[10, 0, :128] = -each[9, 0, :128]
    each[11].flat[0] = np.float32(2.0 ** -120)
    q, s = quantized(ctx, x, "f32", block_rows)
    want_q, want_s = ref.quantize(x, block_rows)
    assert (s == want_s).all()
    assert (q == want_q).all()


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_next_to_middles(ctx, block_rows):
    """Values a step of fp32 or two from where two codes meet, for largest magnitudes of all kinds."""
    announce(f"fp8 quantize next to the middles, blocks of {block_rows}")
    rng = np.random.default_rng(5)
    most = (rng.uniform(1, 2, 300) * 2.0 ** rng.integers(-110, 100, 300)).astype(np.float32)
    most[:3] = [448, 1, 448 * 2.0 ** -126]
    middle = (ref.POSITIVE[:-1] + ref.POSITIVE[1:]) / 2
    x = np.zeros((len(most), block_rows, 5, 128), np.float32)
    x[:, 0, :, 1:127] = (middle * most[:, None].astype(np.float64) / 448).astype(np.float32)[:, None]
    for b, steps in enumerate((-2, -1, 0, 1, 2)):
        for _ in range(abs(steps)):
            x[:, 0, b] = np.nextafter(x[:, 0, b], np.float32(np.sign(steps) * np.inf))
    x[:, 0, :, 127] = -x[:, 0, :, 64]
    x[:, 0, :, 0] = most[:, None]
    x = x.reshape(-1, 640)
    q, s = quantized(ctx, x, "f32", block_rows)
    want_q, want_s = ref.quantize(x, block_rows)
    assert (s == want_s).all() and (q == want_q).all()


def test_quantize_nothing(ctx):
    announce("fp8 quantize without rows")
    q = Out(ctx, (4,), np.uint8)
    ctx.fp8_quantize(None, 0, 128, q.ptr, None)
    assert (q.read() == 0xA5).all()


# ---- products ----

def fp8_rows(rng, rows, width, spread=1.0):
    x = rng.standard_normal((rows, width)) * np.exp(rng.uniform(-spread, spread, (rows, 1)))
    return ref.quantize(x.astype(np.float32))


def fp8_matrix(rng, rows, width):
    return ref.quantize((rng.standard_normal((rows, width)) * 0.05).astype(np.float32), ref.BLOCK)


GEMM = [(1, 1, 16), (1, 2048, 1408), (2, 129, 128), (3, 5, 144), (16, 256, 2048), (17, 130, 256), (31, 1408, 400),
        (33, 515, 1040), (64, 257, 128), (65, 256, 2816), (100, 1000, 16), (255, 384, 272), (257, 259, 1408),
        (300, 640, 10944), (513, 264, 640), (1, 24576, 64), (40, 2048, 5120), (1, 515, 10944), (5, 64, 32768)]


@pytest.mark.parametrize("rows,n,k", GEMM)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_gemm(ctx, rows, n, k, dtype):
    announce(f"fp8 gemm {rows} x {n} x {k} {dtype}")
    rng = np.random.default_rng(rows + 1000 * n + k)
    a, sa = fp8_rows(rng, rows, k)
    w, sw = fp8_matrix(rng, n, k)
    y = Out(ctx, (rows, n), TYPES[dtype][1])
    held = [ctx.to_device(v) for v in (a, sa, w, sw)]
    ctx.fp8_gemm(held[0], held[1], rows, held[2], held[3], n, k, y.ptr, dtype=TYPES[dtype][0])
    want, off = ref.product(a, sa, w, sw, dtype)
    ref.check_product(y.read(), want, off, dtype, (rows, n, k))
    for h in held:
        h.free()


@pytest.mark.parametrize("rows,n,k", [(1, 70, 16), (3, 300, 144), (40, 300, 400), (300, 300, 272)])
def test_gemm_nan(ctx, rows, n, k):
    """A NaN code reaches its row's or its column's products and no others, the row's neighbour in memory included."""
    announce(f"fp8 gemm with NaN {rows} x {n} x {k}")
    rng = np.random.default_rng(5)
    a, sa = fp8_rows(rng, rows, k)
    w, sw = fp8_matrix(rng, n, k)
    a[rows // 2, k - 1] = 0x7F
    a[rows // 3, 0] = 0xFF
    w[n // 2, 0] = 0x7F
    w[n - 1, k - 1] = 0xFF
    y = Out(ctx, (rows, n), np.float32)
    ctx.fp8_gemm(ctx.to_device(a), ctx.to_device(sa), rows, ctx.to_device(w), ctx.to_device(sw), n, k, y.ptr)
    want, off = ref.product(a, sa, w, sw)
    assert np.isnan(want).any() and (rows < 3 or np.isfinite(want).any())
    ref.check_product(y.read(), want, off, "f32")


def test_gemm_extreme_scales(ctx):
    """Scales far from one another, and codes that are all zeros."""
    announce("fp8 gemm with extreme scales")
    rng = np.random.default_rng(6)
    a, sa = fp8_rows(rng, 20, 640)
    w, sw = fp8_matrix(rng, 200, 640)
    sa *= (10.0 ** rng.uniform(-15, 15, sa.shape)).astype(np.float32)
    sw *= (10.0 ** rng.uniform(-15, 15, sw.shape)).astype(np.float32)
    a[7] = 0
    w[100] = 0x80
    y = Out(ctx, (20, 200), np.float32)
    ctx.fp8_gemm(ctx.to_device(a), ctx.to_device(sa), 20, ctx.to_device(w), ctx.to_device(sw), 200, 640, y.ptr)
    want, off = ref.product(a, sa, w, sw)
    got = y.read()
    assert (got[7] == 0).all() and (got[:, 100] == 0).all()
    ref.check_product(got, want, off, "f32")


# ---- by groups ----

def routing(rng, counts, assignments=None):
    """Offsets of groups of these sizes, and an order of the assignments."""
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    perm = rng.permutation(offsets[-1] if assignments is None else assignments)[:offsets[-1]].astype(np.int32)
    return offsets, perm


class Groups:
    def __init__(self, ctx, offsets, rows, source=None, divisor=0, target=None):
        self.held = [None if v is None else ctx.to_device(np.asarray(v, np.int32)) for v in (offsets, source, target)]
        self.c = lm.Fp8Groups(groups=len(offsets) - 1, divisor=divisor, rows=rows)
        self.c.offsets, self.c.source, self.c.target = [None if h is None else h.ptr for h in self.held]


COUNTS = {"one token": [0, 1, 0, 0, 1, 1, 0, 1], "one group": [37], "empty": [0, 0, 0], "one row": [1],
          "ragged": [0, 1, 15, 16, 17, 0, 33, 64, 65, 2, 0, 127, 129, 0], "long": [3, 300, 0, 5], "last empty": [70, 0],
          "many": [1 + (i * 7) % 5 for i in range(160)], "most groups": [i % 2 for i in range(512)]}
WIDTHS = [(200, 400), (130, 128), (48, 1408)]


@pytest.mark.parametrize("counts", COUNTS, ids=str)
@pytest.mark.parametrize("n,k", WIDTHS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_grouped_gemm(ctx, counts, n, k, dtype):
    """Rows of each group in order, written to their assignments' places; the other rows of the output stay."""
    announce(f"fp8 grouped gemm, {counts}, {n} x {k} {dtype}")
    rng = np.random.default_rng(len(counts) + n)
    sizes = COUNTS[counts]
    rows, E = sum(sizes), len(sizes)
    offsets, target = routing(rng, sizes, rows + 3)
    a, sa = fp8_rows(rng, max(rows, 1), k)
    ws = [fp8_matrix(rng, n, k) for _ in range(E)]
    y = Out(ctx, (rows + 3, n), TYPES[dtype][1])
    before = y.host[:y.bytes].view(y.dtype).reshape(y.shape)
    g = Groups(ctx, offsets, rows, target=target if rows else [0])
    ctx.fp8_grouped_gemm(g.c, ctx.to_device(a), ctx.to_device(sa), len(a), ctx.to_device(np.stack([w for w, _ in ws])),
                         ctx.to_device(np.stack([s for _, s in ws])), n, k, y.ptr, rows + 3, dtype=TYPES[dtype][0])
    ctx.synchronize()
    got = y.read()
    for e in range(E):
        at = slice(offsets[e], offsets[e + 1])
        if sizes[e]:
            want, off = ref.product(a[at], sa[at], *ws[e], dtype)
            ref.check_product(got[target[at]], want, off, dtype, (counts, e))
    rest = np.setdiff1d(np.arange(rows + 3), target)
    assert (got[rest].view(np.uint8) == before[rest].view(np.uint8)).all()


@pytest.mark.parametrize("counts", ["one token", "ragged", "long", "many"])
@pytest.mark.parametrize("top_k", [1, 6])
def test_grouped_gemm_gathered(ctx, counts, top_k):
    """Rows read through an index, several of one row of a; rows of the arrays behind the last group stay."""
    announce(f"fp8 grouped gemm gathered, {counts}, top-{top_k}")
    rng = np.random.default_rng(top_k)
    sizes, n, k = COUNTS[counts], 136, 272
    rows, E = sum(sizes), len(sizes)
    offsets, perm = routing(rng, sizes)
    a, sa = fp8_rows(rng, -(-rows // top_k), k)
    ws = [fp8_matrix(rng, n, k) for _ in range(E)]
    y = Out(ctx, (rows + 5, n), np.float32)
    g = Groups(ctx, offsets, rows + 5, source=np.concatenate([perm, [-1] * 5]), divisor=top_k)
    ctx.fp8_grouped_gemm(g.c, ctx.to_device(a), ctx.to_device(sa), len(a), ctx.to_device(np.stack([w for w, _ in ws])),
                         ctx.to_device(np.stack([s for _, s in ws])), n, k, y.ptr, rows + 5)
    ctx.synchronize()  # the indexes behind the last group are not looked at
    got = y.read()
    for e in range(E):
        at = slice(offsets[e], offsets[e + 1])
        if sizes[e]:
            src = perm[at] // top_k
            want, off = ref.product(a[src], sa[src], *ws[e])
            ref.check_product(got[at], want, off, "f32", (counts, e))
    assert (got[rows:].view(np.uint8) == 0xA5).all()


@pytest.mark.parametrize("counts", COUNTS, ids=str)
@pytest.mark.parametrize("inter,k", [(208, 400), (128, 128), (16, 1408), (1408, 256)])
def test_grouped_swiglu(ctx, counts, inter, k):
    announce(f"fp8 grouped swiglu, {counts}, {inter} x {k}")
    rng = np.random.default_rng(len(counts) + inter)
    sizes, top_k = COUNTS[counts], 3
    if inter * len(sizes) > 200000:
        sizes = sizes[:64]
    rows, E = sum(sizes), len(sizes)
    offsets, perm = routing(rng, sizes)
    a, sa = fp8_rows(rng, max(1, -(-rows // top_k)), k)
    ws = [[fp8_matrix(rng, inter, k) for _ in range(2)] for _ in range(E)]
    q, s = Out(ctx, (rows + 2, inter), np.uint8), Out(ctx, (rows + 2, ref.blocks(inter)), np.float32)
    g = Groups(ctx, offsets, rows + 2, source=np.concatenate([perm, [0, 0]]), divisor=top_k)
    ctx.fp8_grouped_swiglu(g.c, ctx.to_device(a), ctx.to_device(sa), len(a),
                           ctx.to_device(np.stack([[w for w, _ in pair] for pair in ws])),
                           ctx.to_device(np.stack([[v for _, v in pair] for pair in ws])), inter, k, q.ptr, s.ptr)
    ctx.synchronize()
    q, s = q.read(), s.read()
    for e in range(E):
        at = slice(offsets[e], offsets[e + 1])
        if sizes[e]:
            src = perm[at] // top_k
            act, off = ref.swiglu(a[src], sa[src], *ws[e][0], *ws[e][1])
            ref.check_blocks(q[at], s[at], act, off, (counts, e))
    assert (q[rows:] == 0xA5).all() and (s[rows:].view(np.uint8) == 0xA5).all()


@pytest.mark.parametrize("rows", [1, 40])
def test_swiglu_extremes(ctx, rows):
    """Gates far on either side of 0, a row of zeros, a row with NaN, infinite products."""
    announce(f"fp8 swiglu extremes, {rows} rows")
    rng = np.random.default_rng(8)
    inter, k = 272, 256
    kinds = 5
    a, sa = fp8_rows(rng, rows * kinds, k, spread=0.0)
    a, sa = a.reshape(kinds, rows, k), sa.reshape(kinds, rows, 2)
    sa[0] *= 50          # |gate| into the hundreds
    a[1] = 0
    a[2, :, 77] = 0x7F
    sa[3] *= 1e30        # act is far past the largest value, or 0: infinities become NaN codes
    sa[4] *= 1e-20       # act underflows
    a, sa = a.reshape(-1, k), sa.reshape(-1, 2)
    pair = [fp8_matrix(rng, inter, k) for _ in range(2)]
    q, s = Out(ctx, (len(a), inter), np.uint8), Out(ctx, (len(a), 3), np.float32)
    g = Groups(ctx, [0, len(a)], len(a))
    ctx.fp8_grouped_swiglu(g.c, ctx.to_device(a), ctx.to_device(sa), len(a), ctx.to_device(np.stack([w for w, _ in pair])),
                           ctx.to_device(np.stack([v for _, v in pair])), inter, k, q.ptr, s.ptr)
    q, s = q.read(), s.read()
    act, off = ref.swiglu(a, sa, *pair[0], *pair[1])
    assert not ((np.abs(act) > 1e37) & (np.abs(act) < 1e40)).any()  # none where fp32 might go either way
    act = np.where(np.abs(act) > 3.5e38, np.nan, act)
    ref.check_blocks(q, s, act, off)


@pytest.mark.parametrize("what", ["source", "negative source", "target", "offsets", "past rows", "negative offset"])
def test_bad_indexes_are_not_followed(ctx, what):
    """An index outside its range is reported once; good groups' rows come out right, nothing else is written."""
    announce(f"fp8 grouped gemm, bad {what}")
    rng = np.random.default_rng(9)
    n, k, sizes = 64, 144, [20, 0, 5, 9]
    rows = sum(sizes)
    offsets, perm = routing(rng, sizes)
    a, sa = fp8_rows(rng, rows, k)
    ws = [fp8_matrix(rng, n, k) for _ in sizes]
    source, target = perm.copy(), perm.copy()
    if what == "source":
        source[1] = rows
    elif what == "negative source":
        source[1] = -2 ** 31
    elif what == "target":
        target[1] = 2 ** 30
    elif what == "offsets":
        offsets[1] = rows + 10 ** 6  # group 0 past the arrays, group 1 falls
    elif what == "past rows":
        offsets[4] = 2 ** 31 - 1
    else:
        offsets[0] = -5
    y = Out(ctx, (rows, n), np.float32)
    g = Groups(ctx, offsets, rows, source=source, divisor=1, target=target)
    held = [ctx.to_device(v) for v in (a, sa, np.stack([w for w, _ in ws]), np.stack([s for _, s in ws]))]
    ctx.fp8_grouped_gemm(g.c, held[0], held[1], rows, held[2], held[3], n, k, y.ptr, rows)
    with pytest.raises(lm.LmError) as e:
        ctx.synchronize()
    assert e.value.status == -5 and "index" in str(e.value)
    ctx.synchronize()  # once
    got = y.read()
    at = slice(20, 25)  # group 2
    want, off = ref.product(a[perm[at]], sa[perm[at]], *ws[2])
    if what != "offsets":
        ref.check_product(got[perm[at]], want, off, "f32", what)


def test_more_tiles_than_a_launch_takes(ctx):
    """128 groups of 2^24 features: refused before anything runs."""
    announce("fp8 grouped gemm, 2^24 features by 128 groups")
    groups, n, k = 128, 2 ** 24, 16
    w, ws = ctx.empty((groups, n, k), np.uint8), ctx.empty((groups, n // 128))
    a, sa, y = ctx.empty((groups, k), np.uint8), ctx.empty((groups, 1)), ctx.empty((groups, n))
    g = Groups(ctx, np.arange(groups + 1, dtype=np.int32), groups)
    with pytest.raises(lm.LmError) as e:
        ctx.fp8_grouped_gemm(g.c, a, sa, groups, w, ws, n, k, y, groups)
    assert e.value.status == -1 and "tiles" in str(e.value)
    for b in (w, ws, a, sa, y):
        b.free()
    ctx.synchronize()
