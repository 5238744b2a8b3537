"""The FP8 operators together as they are used: a FFN from rows to outputs, captured and replayed, on two contexts at once,
call after call over one workspace, and past 2^31 bytes."""
import ctypes as C

import numpy as np
import pytest

import fp8_ref as ref
import litemind_amd as lm
from conftest import announce
from litemind_amd import workload as wl
from test_gpu_fp8 import Groups, fp8_matrix, fp8_rows, routing
from test_gpu_serving_run import Hip

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = lm.Context(wl.V2_LITE.moe_config(num_layers=1))
    yield c
    c.close()


class Ffn:
    """An expert FFN's operands on a context, and its four calls: blocks, gate/up, down, and back to assignments."""

    def __init__(self, ctx, seed, tokens, sizes, top_k, hidden, inter):
        rng = np.random.default_rng(seed)
        self.ctx, self.T, self.hidden, self.inter, self.sizes = ctx, tokens, hidden, inter, sizes
        self.rows, self.top_k = sum(sizes), top_k
        self.offsets, self.perm = routing(rng, sizes)
        self.x = rng.standard_normal((tokens, hidden)).astype(np.float32)
        self.wide = [[fp8_matrix(rng, inter, hidden) for _ in range(2)] for _ in sizes]
        self.low = [fp8_matrix(rng, hidden, inter) for _ in sizes]
        self.dx = ctx.to_device(self.x)
        self.w = [ctx.to_device(np.stack([[m[i] for m in pair] for pair in self.wide])) for i in (0, 1)]
        self.d = [ctx.to_device(np.stack([m[i] for m in self.low])) for i in (0, 1)]
        self.q, self.s = ctx.empty((tokens, hidden), np.uint8), ctx.empty((tokens, ref.blocks(hidden)))
        self.aq, self.a_s = ctx.empty((self.rows, inter), np.uint8), ctx.empty((self.rows, ref.blocks(inter)))
        self.y = ctx.to_device(np.full((self.rows, hidden), 7, np.float32))
        self.into = Groups(ctx, self.offsets, self.rows, source=self.perm, divisor=top_k)
        self.out = Groups(ctx, self.offsets, self.rows, target=self.perm)

    def run(self):
        c = self.ctx
        c.fp8_quantize(self.dx, self.T, self.hidden, self.q, self.s)
        c.fp8_grouped_swiglu(self.into.c, self.q, self.s, self.T, *self.w, self.inter, self.hidden, self.aq, self.a_s)
        c.fp8_grouped_gemm(self.out.c, self.aq, self.a_s, self.rows, *self.d, self.hidden, self.inter, self.y, self.rows)

    def read(self):
        return self.q.download(), self.s.download(), self.aq.download(), self.a_s.download(), self.y.download()

    def check(self):
        """Each step against the definition, on what the step before it gave."""
        q, s, aq, a_s, y = self.read()
        want_q, want_s = ref.quantize(self.x)
        assert (q == want_q).all() and (s == want_s).all()
        for e, n in enumerate(self.sizes):
            at = slice(self.offsets[e], self.offsets[e + 1])
            if n == 0:
                continue
            src = self.perm[at] // self.top_k
            act, off = ref.swiglu(q[src], s[src], *self.wide[e][0], *self.wide[e][1])
            ref.check_blocks(aq[at], a_s[at], act, off, e)
            want, off = ref.product(aq[at], a_s[at], *self.low[e])
            ref.check_product(y[self.perm[at]], want, off, "f32", e)


SIZES = {"one token": (1, [0, 1, 0, 1, 1, 0], 3), "few": (5, [3, 0, 9, 1, 2, 0], 3),
         "many": (200, [0, 130, 3, 64, 300, 103], 3), "one group": (33, [33], 1)}


@pytest.mark.parametrize("name", SIZES)
def test_ffn(ctx, name):
    announce(f"fp8 ffn, {name}")
    f = Ffn(ctx, 1, *SIZES[name], 272, 208)
    f.run()
    f.check()
    before = f.read()
    f.run()
    for a, b in zip(before, f.read()):
        assert (a.view(np.uint8) == b.view(np.uint8)).all()  # the same bits every time


def test_captured_ffn(ctx):
    """Two captured FFNs and eager ones of other sizes between their replays; inputs are read at the replay."""
    announce("fp8 ffn captured and replayed")
    hip = Hip(ctx)
    runs = [Ffn(ctx, 2, *SIZES["few"], 272, 208), Ffn(ctx, 3, *SIZES["many"], 144, 128)]
    other = Ffn(ctx, 4, *SIZES["one token"], 400, 304)
    for f in runs + [other]:
        f.run()
    ctx.synchronize()
    graphs = [hip.capture(f.run) for f in runs]
    try:
        for turn in range(3):
            for f, (_, runnable) in zip(runs, graphs):
                f.x = np.random.default_rng(10 + turn).standard_normal(f.x.shape).astype(np.float32)
                f.dx.upload(f.x)
                f.y.upload(np.full((f.rows, f.hidden), np.nan, np.float32))
                hip.replay(runnable)
                other.run()
                f.check()
                other.check()
    finally:
        for g in graphs:
            hip.free(*g)


class Product:
    def __init__(self, ctx, seed, rows, n, k):
        rng = np.random.default_rng(seed)
        self.ctx, self.rows, self.n, self.k = ctx, rows, n, k
        self.a, self.w = fp8_rows(rng, rows, k), fp8_matrix(rng, n, k)
        self.held = [ctx.to_device(v) for v in (*self.a, *self.w)]
        self.y = ctx.empty((rows, n))
        self.want = ref.product(*self.a, *self.w)

    def run(self):
        a, s, w, ws = self.held
        self.ctx.fp8_gemm(a, s, self.rows, w, ws, self.n, self.k, self.y)

    def check(self):
        ref.check_product(self.y.download(), *self.want, "f32", (self.rows, self.n, self.k))


# a long reduced axis over few tiles: several workgroups share it, and their sums go through the context's workspace
SHARED = [(48, 256, 8192), (100, 130, 4112), (33, 515, 10944), (200, 512, 6016)]


def test_shares_take_turns(ctx):
    announce("fp8 gemm: shared sums, call after call")
    runs = [Product(ctx, 20 + i, *size) for i, size in enumerate(SHARED)]
    for r in runs:
        r.run()
    for r in reversed(runs):
        r.run()
    for r in runs:
        r.check()


def test_captured_shares(ctx):
    announce("fp8 gemm: shared sums, captured")
    hip = Hip(ctx)
    runs = [Product(ctx, 30 + i, *size) for i, size in enumerate(SHARED[:2])]
    other = Product(ctx, 40, *SHARED[2])
    for r in runs:
        r.run()
    graphs = [hip.capture(r.run) for r in runs]
    try:
        for _ in range(3):
            for r, (_, runnable) in zip(runs, graphs):
                r.y.upload(np.full((r.rows, r.n), np.nan, np.float32))
                hip.replay(runnable)
                other.run()
            for r in runs + [other]:
                r.check()
    finally:
        for g in graphs:
            hip.free(*g)


def test_first_call_cannot_be_captured():
    announce("fp8: a context's first product under capture")
    with lm.Context(wl.V2_LITE.moe_config(num_layers=1)) as c:
        hip, p = Hip(c), Product(c, 50, 3, 64, 128)
        said = []

        def work():
            try:
                p.run()
            except lm.LmError as e:
                said.append(e)

        hip.free(*hip.capture(work))
        assert said and said[0].status == -1 and "captured" in str(said[0])
        p.run()
        p.check()
        q, s = c.empty((4, 128), np.uint8), c.empty((4, 1))
        x = np.random.default_rng(1).standard_normal((4, 128)).astype(np.float32)
        dx = c.to_device(x)
        graph = hip.capture(lambda: c.fp8_quantize(dx, 4, 128, q, s))  # needs nothing of the context
        hip.replay(graph[1])
        c.synchronize()
        assert (q.download() == ref.quantize(x)[0]).all()
        hip.free(*graph)


def test_two_contexts():
    """Two contexts' calls at once, each on its own stream and workspace."""
    announce("fp8: two contexts at once")
    with lm.Context(wl.V2_LITE.moe_config(num_layers=1)) as c, lm.Context(wl.V2_LITE.moe_config(num_layers=1)) as d:
        ffns = [Ffn(x, 60 + i, *SIZES["many"], 272, 208) for i, x in enumerate((c, d))]
        products = [Product(x, 70 + i, *SHARED[i]) for i, x in enumerate((c, d))]
        for _ in range(4):
            for f, p in zip(ffns, products):
                f.run()
                p.run()
        for x in ffns + products:
            x.check()


def test_past_4_gib_of_rows(ctx):
    """Quantized rows, gathered rows and outputs whose byte offsets pass 2^31 and 2^32."""
    announce("fp8: rows past 2^31 and outputs past 2^32 bytes")
    k, n = 2048, 640
    rows = 2 ** 32 // k - 1  # the most that a product takes
    picks = np.array([0, 1, 2 ** 31 // k - 1, 2 ** 31 // k, rows - 2, rows - 1])
    rng = np.random.default_rng(80)
    a, s = fp8_rows(rng, len(picks), k)
    w, sw = fp8_matrix(rng, n, k)
    da, ds = ctx.empty((rows, k), np.uint8).zero(), ctx.empty((rows, k // 128)).zero()
    for i, r in enumerate(picks):
        for dev, host in ((da, a), (ds, s)):
            line = np.ascontiguousarray(host[i])
            ctx._check(ctx.lib.lm_copy_h2d(ctx.handle, C.c_void_p(dev.ptr + int(r) * line.nbytes),
                                           line.ctypes.data_as(C.c_void_p), line.nbytes))
    out = ctx.empty((rows, n), np.uint16)
    ctx.fp8_gemm(da, ds, rows, ctx.to_device(w), ctx.to_device(sw), n, k, out, dtype=lm.DT_BF16)
    ctx.synchronize()
    want, off = ref.product(a, s, w, sw, "bf16")
    for i, r in enumerate(picks):
        line = np.empty(n, np.uint16)
        ctx._check(ctx.lib.lm_copy_d2h(ctx.handle, line.ctypes.data_as(C.c_void_p),
                                       C.c_void_p(out.ptr + int(r) * 2 * n), line.nbytes))
        ref.check_product(line[None], want[i:i + 1], off[i:i + 1], "bf16", int(r))
    y = ctx.empty((len(picks), n))
    g = Groups(ctx, [0, 2, len(picks)], len(picks), source=picks, divisor=1)
    two, scales = np.stack([w, w[::-1]]), np.stack([sw, sw[::-1]])
    ctx.fp8_grouped_gemm(g.c, da, ds, rows, ctx.to_device(two), ctx.to_device(scales), n, k, y, len(picks))
    got = y.download()
    ref.check_product(got[:2], *ref.product(a[:2], s[:2], w, sw), "f32")
    ref.check_product(got[2:], *ref.product(a[2:], s[2:], two[1], scales[1]), "f32")
    x = ctx.empty((2 ** 31 // 8192 + 3, 8192), np.uint16).zero()  # BF16 rows past 2^32 bytes
    line = ref.bf16(rng.standard_normal(8192).astype(np.float32))
    last = x.shape[0] - 1
    ctx._check(ctx.lib.lm_copy_h2d(ctx.handle, C.c_void_p(x.ptr + last * line.nbytes), line.ctypes.data_as(C.c_void_p),
                                   line.nbytes))
    q, qs = ctx.empty(x.shape, np.uint8), ctx.empty((x.shape[0], 64))
    ctx.fp8_quantize(x, x.shape[0], 8192, q, qs, dtype=lm.DT_BF16)
    code = np.empty(8192, np.uint8)
    ctx._check(ctx.lib.lm_copy_d2h(ctx.handle, code.ctypes.data_as(C.c_void_p), C.c_void_p(q.ptr + last * 8192), 8192))
    assert (code == ref.quantize(line[None])[0][0]).all()
    for b in (da, ds, out, x, q, qs):
        b.free()


def test_weights_past_4_gib(ctx):
    """Experts whose matrices lie past 2^32 bytes from the first, and a matrix of nearly 2^32."""
    announce("fp8: weights past 2^32 bytes")
    k, n, E = 4096, 8192, 140
    rng = np.random.default_rng(81)
    a, s = fp8_rows(rng, 5, k)
    w, sw = fp8_matrix(rng, n, k)
    dw, dsw = ctx.empty((E, n, k), np.uint8).zero(), ctx.empty((E, n // 128, k // 128)).zero()
    for dev, host in ((dw, w), (dsw, sw)):
        ctx._check(ctx.lib.lm_copy_h2d(ctx.handle, C.c_void_p(dev.ptr + (E - 1) * host.nbytes),
                                       host.ctypes.data_as(C.c_void_p), host.nbytes))
    y = ctx.empty((5, n))
    g = Groups(ctx, [0] * E + [5], 5)
    ctx.fp8_grouped_gemm(g.c, ctx.to_device(a), ctx.to_device(s), 5, dw, dsw, n, k, y, 5)
    ref.check_product(y.download(), *ref.product(a, s, w, sw), "f32")
    # the same memory as one matrix: its last rows
    rows = 2 ** 32 // k - 1
    top = rows - n
    assert top % 128 != 0
    out = ctx.empty((5, rows))
    ctx._check(ctx.lib.lm_copy_h2d(ctx.handle, C.c_void_p(dw.ptr + top * k), w.ctypes.data_as(C.c_void_p), w.nbytes))
    ones = np.ones((ref.blocks(rows), k // 128), np.float32)
    ctx.fp8_gemm(ctx.to_device(a), ctx.to_device(s), 5, dw, ctx.to_device(ones), rows, k, out)
    want, off = ref.product(a, s, w, np.ones_like(sw))
    got = np.empty((5, n), np.float32)
    for r in range(5):
        ctx._check(ctx.lib.lm_copy_d2h(ctx.handle, got[r].ctypes.data_as(C.c_void_p),
                                       C.c_void_p(out.ptr + 4 * (r * rows + top)), 4 * n))
    ref.check_product(got, want, off, "f32")
    for b in (dw, dsw, out):
        b.free()
