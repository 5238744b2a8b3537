"""LM_PATH_FP8 at DeepSeek-V2-Lite's widths, where the layers' own launches run: the shared experts' tiles beside the
routed experts', SwiGLU and fp32 outputs on the FP8 matrix cores, tiles of up to 256 rows, shared sums of the dense
FFN.  Against the FP8 operators one after another, whose sums are fp32's."""
import dataclasses

import numpy as np
import pytest

import fp8_ref as ref
import litemind_amd as lm
from conftest import announce
from litemind_amd import workload as wl

pytestmark = pytest.mark.gpu

D = wl.V2_LITE


class Ffn:
    """FFNs of [groups] experts in FP8 blocks, quantized matrix by matrix, and their operators."""

    def __init__(self, ctx, gate, up, down):
        self.ctx, self.E, (self.I, self.H) = ctx, len(gate), gate[0].shape
        hb, ib = ref.blocks(self.H), ref.blocks(self.I)
        self.w, self.ws = ctx.empty((self.E, 2, self.I, self.H), np.uint8), ctx.empty((self.E, 2, ib, hb))
        self.d, self.ds = ctx.empty((self.E, self.H, self.I), np.uint8), ctx.empty((self.E, hb, ib))
        for e in range(self.E):
            for part, m in enumerate((gate[e], up[e])):
                at = 2 * e + part
                self.quantize(m, self.w.ptr + at * self.I * self.H, self.ws.ptr + 4 * at * ib * hb)
            self.quantize(down[e], self.d.ptr + e * self.I * self.H, self.ds.ptr + 4 * e * ib * hb)

    def quantize(self, m, q, s):
        x = self.ctx.to_device(m)
        self.ctx.fp8_quantize(x, *m.shape, q, s, dtype=lm.DT_BF16, block_rows=128)
        self.ctx.synchronize()
        x.free()

    def run(self, x, offsets, perm, top_k):
        """[rows][H] in the assignments' order."""
        ctx, rows = self.ctx, len(perm)
        dx, o, p = ctx.to_device(x), ctx.to_device(offsets), ctx.to_device(perm)
        xq, xs = ctx.empty((len(x), self.H), np.uint8), ctx.empty((len(x), ref.blocks(self.H)))
        q, qs = ctx.empty((rows, self.I), np.uint8), ctx.empty((rows, ref.blocks(self.I)))
        y = ctx.empty((rows, self.H))
        ctx.fp8_quantize(dx, len(x), self.H, xq, xs)
        g = lm.Fp8Groups(groups=self.E, rows=rows, offsets=o.ptr, source=p.ptr, divisor=top_k)
        ctx.fp8_grouped_swiglu(g, xq, xs, len(x), self.w, self.ws, self.I, self.H, q, qs)
        g = lm.Fp8Groups(groups=self.E, rows=rows, offsets=o.ptr, target=p.ptr)
        ctx.fp8_grouped_gemm(g, q, qs, rows, self.d, self.ds, self.H, self.I, y, rows)
        got = y.download()
        for b in (dx, o, p, xq, xs, q, qs, y):
            b.free()
        return got

    def alone(self, x):
        return self.run(x, np.array([0, len(x)], np.int32), np.arange(len(x), dtype=np.int32), 1)


@pytest.fixture(scope="module")
def lite(v2_layer):
    announce("fp8: a V2-Lite MoE layer and a dense one")
    ctx = lm.Context(D.moe_config(num_layers=2))
    dense = wl.dense_ffn(wl.MASTER_SEED, 0, D)
    ctx.upload_dense(0, *dense)
    ctx.finalize_layer(0)
    wl.upload_moe_layer(ctx, 1, v2_layer)
    for layer in (0, 1):
        ctx.fp8_layer(layer)
    m = v2_layer
    yield (ctx, Ffn(ctx, [dense[0]], [dense[1]], [dense[2]]), Ffn(ctx, m.gate, m.up, m.down),
           Ffn(ctx, [m.shared_gate], [m.shared_up], [m.shared_down]))
    ctx.close()


def near(got, want, gate_up_exact):
    """The FP8 matrix cores' sums of the down product are off by 4e-5 of their norm. SwiGLU's fp32 sums, maybe in another
    order, are off by 1e-7: that puts some 1e-6 of the activations' codes on the other side of a border, a step of
    2^-3.5 away, 1e-4 of an output's norm. On the FP8 matrix cores they are off by 4e-5, which puts 6e-4 of the codes
    there: 2e-3. Twice these for all rows. In one row the step may be its largest activation's, two fifths of the norm of
    all at most."""
    assert np.isfinite(got).all()
    d = np.linalg.norm(got - want, axis=1)
    norm = np.linalg.norm(want, axis=1)
    assert np.linalg.norm(d) <= 2 * (4e-5 + (1e-4 if gate_up_exact else 2e-3)) * np.linalg.norm(norm)
    assert (d <= 4e-2 * norm).all(), (d / norm).max()


def moe(ctx, layer, d, routed, shared, x, bias=None):
    """The layer's outputs, those of the operators for its routing, and the assignments of each expert."""
    T = len(x)
    dx, y, idx, w = ctx.to_device(x), ctx.empty((T, d.hidden)), ctx.empty((T, d.top_k), np.int32), ctx.empty((T, d.top_k))
    ctx.moe_forward(layer, dx, T, y, bias=bias, idx=idx, w=w, path=lm.PATH_FP8)
    got = y.download()
    ctx.moe_forward(layer, dx, T, y, bias=bias, idx=idx, w=w, path=lm.PATH_FP8)
    assert (y.download() == got).all()  # the same bits every time
    gi, gw = idx.download(), w.download().astype(np.float64)
    counts = np.bincount(gi.reshape(-1), minlength=d.experts)
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    perm = np.argsort(gi.reshape(-1), kind="stable").astype(np.int32)
    rows = routed.run(x, offsets, perm, d.top_k).reshape(T, d.top_k, -1)
    want = sum(gw[:, r, None] * rows[:, r] for r in range(d.top_k)) + shared.alone(x)
    return got, want, counts


# V2-Lite's calls: the single row's launch, few rows beside the shared experts', up to the last of these, the first with
# launches of their own, and prompts on the FP8 matrix cores
@pytest.mark.parametrize("skewed", [False, True])
@pytest.mark.parametrize("T", [1, 2, 8, 32, 100, 128, 129, 300, 512, 1000, 2048, 4096])
def test_moe_layer(lite, T, skewed):
    plan = lm.fp8_plan_layer(D.moe_config(num_layers=2), T)
    announce(f"fp8 V2-Lite MoE layer, {T} tokens{', skewed' if skewed else ''}: gate/up {plan.gate_up.kernel}, down "
             f"{plan.down.tile_rows} x {plan.down.tile_features}, beside {plan.beside}")
    assert plan.beside == (T <= 128)
    ctx, _, routed, shared = lite
    x, bias = wl.tokens(7, T, D.hidden), None
    if skewed:  # most assignments to eight experts, and experts without any
        b = np.zeros(D.experts, np.float32)
        b[3::8] = 2.5
        b[:3] = -1e4
        bias = ctx.to_device(b)
    got, want, counts = moe(ctx, 1, D, routed, shared, x, bias)
    if skewed:
        assert (counts[:3] == 0).all() and (T < 100 or counts.max() > 2 * T * D.top_k / D.experts)
    exact = plan.gate_up.fp32_sums and (plan.beside or plan.other_gate_up.fp32_sums)
    near(got, want, exact)
    y = ctx.empty(got.shape)
    if not skewed:
        ctx.moe_forward(1, ctx.to_device(x), T, y, path=lm.PATH_AUTO)
        assert np.linalg.norm(y.download() - got) <= 0.13 * np.linalg.norm(got)  # twice what rounding to e4m3 comes to


# few experts: the larger tiles with the shared experts' beside them
@pytest.mark.parametrize("experts,top_k,hidden,inter,n_shared,T,gate_up,down", [
    (20, 6, 5120, 1536, 2, 1, 0, 0), (16, 16, 1040, 144, 1, 128, 1, 1), (2, 2, 1040, 4112, 1, 128, 2, 0),
    (4, 4, 2064, 2064, 3, 100, 3, 1), (16, 16, 2064, 1408, 3, 128, 4, 2), (16, 16, 2048, 4112, 1, 100, 3, 3),
    (8, 8, 5120, 1040, 2, 117, 3, 4), (8, 3, 272, 2064, 2, 1, 0, -1)])
def test_beside(experts, top_k, hidden, inter, n_shared, T, gate_up, down):
    announce(f"fp8 layer of {experts} experts, {hidden} x {inter}, {T} tokens: gate/up {gate_up}, down {down}, beside")
    d = dataclasses.replace(D, hidden=hidden, inter=inter, experts=experts, top_k=top_k, n_shared=n_shared)
    plan = lm.fp8_plan_layer(d.moe_config(num_layers=1), T)
    assert (plan.beside, plan.gate_up.kernel, plan.down.kernel) == (1, gate_up, down)
    m = wl.moe_layer(17, 0, d)
    with lm.Context(d.moe_config(num_layers=1)) as ctx:
        wl.upload_moe_layer(ctx, 0, m)
        ctx.fp8_layer(0, only=True)
        routed, shared = Ffn(ctx, m.gate, m.up, m.down), Ffn(ctx, [m.shared_gate], [m.shared_up], [m.shared_down])
        got, want, _ = moe(ctx, 0, d, routed, shared, wl.tokens(7, T, hidden))
        near(got, want, bool(plan.gate_up.fp32_sums))


def test_every_launch_of_the_layers_ran():
    """What the sizes above reach, by the plan."""
    sizes = [1, 2, 8, 32, 100, 128, 129, 300, 512, 1000, 2048, 4096]
    plans = [lm.fp8_plan_layer(D.moe_config(num_layers=2), T) for T in sizes]
    beside = {(p.gate_up.kernel, p.down.kernel) for p in plans if p.beside}
    alone = {p.gate_up.kernel for p in plans if not p.beside} | {p.other_gate_up.kernel for p in plans if not p.beside}
    down = {p.down.kernel for p in plans if not p.beside} | {p.other_down.kernel for p in plans if not p.beside}
    assert beside == {(0, -1), (1, 0)} and alone >= {1, 3, 4} and down >= {0, 1, 2, 4}
    plans = [lm.fp8_plan_layer(D.moe_config(num_layers=2), T, dense=True) for T in (1, 32, 128, 512, 2048, 4096)]
    assert {p.other_gate_up.kernel for p in plans} >= {0, 3, 4}
    assert {p.other_down.kernel for p in plans} == {-1, 0, 1, 2, 3} and {p.other_down.shares > 1 for p in plans} == {False, True}


@pytest.mark.parametrize("T", [1, 32, 128, 512, 2048, 4096])
def test_dense_layer(lite, T):
    plan = lm.fp8_plan_layer(D.moe_config(num_layers=2), T, dense=True)
    announce(f"fp8 V2-Lite dense layer, {T} tokens: gate/up {plan.other_gate_up.kernel}, down {plan.other_down.tile_rows} x "
             f"{plan.other_down.tile_features} in {plan.other_down.shares}")
    ctx, dense, _, _ = lite
    x = wl.tokens(9, T, D.hidden)
    y = ctx.empty((T, D.hidden))
    ctx.dense_forward(0, ctx.to_device(x), T, y, path=lm.PATH_FP8)
    near(y.download(), dense.alone(x), bool(plan.other_gate_up.fp32_sums))


def test_stack_and_graph(lite):
    """Both layers by lm_stack_forward and a captured graph whose products share sums, other work between the replays."""
    ctx = lite[0]
    T = 32
    announce("fp8 V2-Lite stack and graph, 32 tokens")
    assert lm.fp8_plan_layer(D.moe_config(num_layers=2), T, dense=True).other_down.shares > 1
    for layer in (0, 1):
        ctx.upload_norm(layer, np.linspace(0.5, 1.5, D.hidden, dtype=np.float32))
    h0 = wl.tokens(10, T, D.hidden)
    h, other, y = ctx.to_device(h0), ctx.to_device(wl.tokens(11, T, D.hidden)), ctx.empty((T, D.hidden))
    want = []
    for _ in range(3):
        ctx.stack_forward(0, 1, h, T, path=lm.PATH_FP8)
        want.append(h.download())
    h.upload(h0)
    graph = ctx.stack_graph_create(0, 1, h, T, path=lm.PATH_FP8)
    try:
        for expected in want:
            ctx.stack_graph_launch(graph)
            ctx.dense_forward(0, other, T, y, path=lm.PATH_FP8)
            assert (h.download() == expected).all()
    finally:
        ctx.stack_graph_destroy(graph)
