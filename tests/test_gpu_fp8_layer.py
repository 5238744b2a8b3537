"""LM_PATH_FP8: the layers' FFNs from FP8 weights, against the FP8 operators run one after another, and what each state of
a layer's weights allows."""
import dataclasses

import numpy as np
import pytest

import fp8_ref as ref
import litemind_amd as lm
import oracle_lib as ol
from conftest import announce
from litemind_amd import workload as wl

pytestmark = pytest.mark.gpu

# widths that end inside a block of 128, and inside a group of 32 rows of the resident layout
SMALL = dataclasses.replace(wl.V2_LITE, hidden=272, inter=144, experts=12, top_k=3, n_shared=2, dense_inter=400, layers=2)
WIDE = dataclasses.replace(wl.V2_LITE, hidden=256, inter=128, experts=96, top_k=4, n_shared=1, dense_inter=1040, layers=2)
ALONE = dataclasses.replace(wl.V2_LITE, hidden=128, inter=272, experts=8, top_k=2, n_shared=0, dense_inter=16, layers=2)
DIMS = {"small": SMALL, "wide": WIDE, "no shared": ALONE}


class Model:
    """A dense layer 0 and a MoE layer 1, in FP8."""

    def __init__(self, dims, only=False):
        self.dims, self.moe, self.dense = dims, wl.moe_layer(31, 1, dims), wl.dense_ffn(31, 0, dims)
        self.ctx = lm.Context(dims.moe_config(num_layers=2))
        self.ctx.upload_dense(0, *self.dense)
        self.ctx.finalize_layer(0)
        wl.upload_moe_layer(self.ctx, 1, self.moe)
        for layer in (0, 1):
            self.ctx.upload_norm(layer, np.linspace(0.5, 1.5, dims.hidden, dtype=np.float32))
            self.ctx.fp8_layer(layer, only)

    def operators(self, gate_up, down, x, offsets=None, perm=None):
        """The outputs [rows, H] of the operators in turn; gate_up: pairs of matrices, down: matrices, one per group."""
        ctx, H, inter = self.ctx, x.shape[1], down[0].shape[1]
        if offsets is None:
            offsets, perm, k = np.array([0, len(x)], np.int32), np.arange(len(x), dtype=np.int32), 1
        else:
            k = self.dims.top_k
        rows = len(perm)
        xq, xs = (ctx.to_device(v) for v in ref.quantize(x))
        wide = [[ref.quantize(m, ref.BLOCK) for m in pair] for pair in gate_up]
        low = [ref.quantize(m, ref.BLOCK) for m in down]
        wq, ws = (ctx.to_device(np.stack([[m[i] for m in pair] for pair in wide])) for i in (0, 1))
        dq, ds = (ctx.to_device(np.stack([m[i] for m in low])) for i in (0, 1))
        o, s = ctx.to_device(offsets), ctx.to_device(perm)
        q, qs, y = ctx.empty((rows, inter), np.uint8), ctx.empty((rows, ref.blocks(inter))), ctx.empty((rows, H))
        g = lm.Fp8Groups(groups=len(down), rows=rows, offsets=o.ptr, source=s.ptr, divisor=k)
        ctx.fp8_grouped_swiglu(g, xq, xs, len(x), wq, ws, inter, H, q, qs)
        g = lm.Fp8Groups(groups=len(down), rows=rows, offsets=o.ptr, target=s.ptr)
        ctx.fp8_grouped_gemm(g, q, qs, rows, dq, ds, H, inter, y, rows)
        return y.download()

    def assignments(self, x, idx):
        """Outputs of each (token, rank) and of the shared experts, by the operators."""
        offsets = np.zeros(self.dims.experts + 1, np.int32)
        offsets[1:] = np.cumsum(np.bincount(idx.reshape(-1), minlength=self.dims.experts))
        perm = np.argsort(idx.reshape(-1), kind="stable").astype(np.int32)
        m = self.moe
        routed = self.operators(list(zip(m.gate, m.up)), m.down, x, offsets, perm)
        shared = None if m.shared_gate is None else self.operators([(m.shared_gate, m.shared_up)], [m.shared_down], x)
        return routed.reshape(len(x), self.dims.top_k, -1), shared


@pytest.fixture(scope="module", params=DIMS)
def model(request):
    announce(f"fp8 layers: {request.param}")
    m = Model(DIMS[request.param])
    yield m
    m.ctx.close()


def near(got, want, parts, exact):
    """Sums of the same fp32 numbers in another order: each of at most 20 additions and products is off by a step of
    what has been added up. Not `exact`: the layers' large tiles take the FP8 matrix cores' sums, off by 4e-5 of their
    norm, which puts 6e-4 of the activations' codes on the other side of a border, a step of 2^-3.5 away: 2e-3 of an
    output's norm."""
    assert np.isfinite(got).all()
    if exact:
        assert (np.abs(got - want) <= 20 * 2.0 ** -23 * parts + 2.0 ** -126).all()
    assert (np.linalg.norm(got - want, axis=-1) <= 1e-2 * np.linalg.norm(parts + np.zeros_like(want), axis=-1)).all()


TOKENS = [1, 2, 3, 17, 100, 128, 129, 300, 1500]


@pytest.mark.parametrize("T", TOKENS)
def test_moe_layer(model, T):
    announce(f"fp8 moe layer, {T} tokens")
    d, ctx = model.dims, model.ctx
    x = wl.tokens(7, T, d.hidden)
    idx, w, y = ctx.empty((T, d.top_k), np.int32), ctx.empty((T, d.top_k)), ctx.empty((T, d.hidden))
    dx = ctx.to_device(x)
    ctx.moe_forward(1, dx, T, y, idx=idx, w=w, path=lm.PATH_FP8)
    ctx.synchronize()
    gi, gw = idx.download(), w.download()
    oy, oi, ow, _ = ol.oracle_moe_layer(model.moe, x)
    assert (gi == oi).all() and (gw == ow).all()  # the router is the other paths'
    routed, shared = model.assignments(x, gi)
    terms = [gw[:, r, None].astype(np.float64) * routed[:, r] for r in range(d.top_k)]
    terms += [] if shared is None else [shared.astype(np.float64)]
    near(y.download(), sum(terms), sum(np.abs(t) for t in terms), T <= 17)
    # Rounding to e4m3 is off by 2.6e-2 of the norm (half a step of 2^-3 .. 2^-4, evenly spread): products of two such
    # operands by 3.7e-2, an activation by 5.2e-2 and its own rounding, an output by 6.4e-2. Twice that is far from
    # what a wrong weight or row gives.
    assert np.linalg.norm(y.download() - oy) <= 0.13 * np.linalg.norm(oy)


@pytest.mark.parametrize("T", TOKENS)
def test_grouped_swiglu(model, T):
    announce(f"fp8 lm_grouped_swiglu, {T} tokens")
    d, ctx = model.dims, model.ctx
    x = wl.tokens(8, T, d.hidden)
    rng = np.random.default_rng(T)
    idx = np.stack([rng.permutation(d.experts)[:d.top_k] for _ in range(T)]).astype(np.int32)
    idx[0] = idx[-1]
    out = ctx.empty((T * d.top_k + T, d.hidden))
    ctx.grouped_swiglu(1, ctx.to_device(x), T, ctx.to_device(idx), out, path=lm.PATH_FP8)
    routed, shared = model.assignments(x, idx)
    got = out.download()
    near(got[:T * d.top_k], routed.reshape(T * d.top_k, -1), np.abs(routed).reshape(T * d.top_k, -1), T <= 17)
    near(got[T * d.top_k:], np.zeros_like(got[T * d.top_k:]) if shared is None else shared, np.zeros_like(got[T * d.top_k:]) if shared is None else np.abs(shared),
         T <= 17)


@pytest.mark.parametrize("T", [1, 5, 40, 200, 2000])
def test_dense_layer(model, T):
    announce(f"fp8 dense layer, {T} tokens")
    d, ctx = model.dims, model.ctx
    x = wl.tokens(9, T, d.hidden)
    y = ctx.empty((T, d.hidden))
    ctx.dense_forward(0, ctx.to_device(x), T, y, path=lm.PATH_FP8)
    gate, up, down = model.dense
    want = model.operators([(gate, up)], [down], x)
    # The down product's sums may be in another order; 1040 terms of either sign add up to a thirtieth of their
    # magnitudes, the row's largest output to more than that.
    near(y.download(), want, 40 * np.abs(want).max(1, keepdims=True), T <= 17)


@pytest.mark.parametrize("T", [1, 3, 40])
def test_stack_and_graph(model, T):
    """Both layers through lm_stack_forward and a captured graph: the same bits, replay after replay, with other eager
    work between; and the layers' own calls chained by hand."""
    announce(f"fp8 stack and graph, {T} tokens")
    d, ctx = model.dims, model.ctx
    h0 = wl.tokens(10, T, d.hidden)
    h = ctx.to_device(h0)
    ctx.stack_forward(0, 1, h, T, path=lm.PATH_FP8)
    once = h.download()
    ctx.stack_forward(0, 1, h, T, path=lm.PATH_FP8)
    twice = h.download()
    norm = ctx.to_device(np.linspace(0.5, 1.5, d.hidden, dtype=np.float32))
    n, y = ctx.empty((T, d.hidden)), ctx.empty((T, d.hidden))
    want = h0.copy()
    for layer in (0, 1):
        dw = ctx.to_device(want)
        ctx.rms_norm(dw, norm, n, T, d.hidden, d.rms_norm_eps)
        if layer == 0:
            ctx.dense_forward(0, n, T, y, path=lm.PATH_FP8)
        else:
            ctx.moe_forward(1, n, T, y, path=lm.PATH_FP8)
        want = want + y.download()
    assert np.linalg.norm(once - want) <= 1e-2 * np.linalg.norm(want - h0) + 1e-6 * np.linalg.norm(want)
    h.upload(h0)
    graph = ctx.stack_graph_create(0, 1, h, T, path=lm.PATH_FP8)
    try:
        other = ctx.to_device(wl.tokens(11, 1, d.hidden))
        for expected in (once, twice):
            ctx.stack_graph_launch(graph)
            ctx.moe_forward(1, other, 1, ctx.empty((1, d.hidden)), path=lm.PATH_FP8)
            assert (h.download() == expected).all()
        with pytest.raises(lm.LmError) as e:  # the graph holds the workspace
            ctx.stack_forward(0, 1, ctx.to_device(wl.tokens(10, 2500, d.hidden)), 2500, path=lm.PATH_FP8)
        assert e.value.status == -1
        with pytest.raises(lm.LmError):
            ctx.fp8_layer(1, only=True)
    finally:
        ctx.stack_graph_destroy(graph)


def refused(status, call, *args, **kw):
    with pytest.raises(lm.LmError) as e:
        call(*args, **kw)
    assert e.value.status == status, str(e.value)


def test_weights_states():
    """Without FP8 weights, with FP8 weights beside the others, alone, after an upload, and uploaded anew."""
    announce("fp8 layers: states of the weights")
    d = SMALL
    x = wl.tokens(12, 4, d.hidden)
    with lm.Context(d.moe_config(num_layers=2)) as ctx:
        moe = wl.moe_layer(31, 1, d)
        refused(-4, ctx.fp8_layer, 1)
        wl.upload_moe_layer(ctx, 1, moe)
        dx, y = ctx.to_device(x), ctx.empty((4, d.hidden))
        refused(-4, ctx.moe_forward, 1, dx, 4, y, path=lm.PATH_FP8)
        before = ctx.resident_bytes()
        ctx.moe_forward(1, dx, 4, y)
        other = y.download()
        ctx.fp8_layer(1)
        beside = ctx.resident_bytes()
        ctx.moe_forward(1, dx, 4, y, path=lm.PATH_FP8)
        fp8 = y.download()
        ctx.moe_forward(1, dx, 4, y)
        assert (y.download() == other).all() and not (fp8 == other).all()
        refused(-1, ctx.moe_forward, 1, dx, 4, y, path=4)
        ctx.fp8_layer(1, only=True)
        alone = ctx.resident_bytes()
        weights = (d.experts + d.n_shared) * 3 * d.hidden * d.inter
        assert weights < beside - before < 1.3 * weights + 8 * 256 and alone < before / 3
        ctx.moe_forward(1, dx, 4, y, path=lm.PATH_FP8)
        assert (y.download() == fp8).all()
        for path in (lm.PATH_AUTO, lm.PATH_GEMV, lm.PATH_MFMA):
            refused(-4, ctx.moe_forward, 1, dx, 4, y, path=path)
        refused(-4, ctx.moe_forward_noalloc, 1, dx, 1, y)
        refused(-4, ctx.layer_fp16_inexact, 1)
        refused(-4, ctx.fp8_layer, 1)
        ctx.upload_expert(1, 0, moe.gate[0], moe.up[0], moe.down[0])  # the layer's weights begin anew
        refused(-4, ctx.moe_forward, 1, dx, 4, y, path=lm.PATH_FP8)
        refused(-4, ctx.finalize_layer, 1)
        wl.upload_moe_layer(ctx, 1, moe)
        refused(-4, ctx.moe_forward, 1, dx, 4, y, path=lm.PATH_FP8)
        ctx.moe_forward(1, dx, 4, y)
        assert (y.download() == other).all()
        ctx.fp8_layer(1)
        ctx.moe_forward(1, dx, 4, y, path=lm.PATH_FP8)
        assert (y.download() == fp8).all()
        ctx.upload_expert(1, 3, moe.gate[4], moe.up[4], moe.down[4])
        refused(-4, ctx.moe_forward, 1, dx, 4, y, path=lm.PATH_FP8)
        refused(-1, ctx.fp8_layer, 2)


def test_widths_of_8_are_refused():
    announce("fp8 layers: widths in multiples of 8")
    d = dataclasses.replace(SMALL, inter=136, n_shared=0)  # the hidden size is always one of 16
    with lm.Context(d.moe_config(num_layers=1)) as ctx:
        wl.upload_moe_layer(ctx, 0, wl.moe_layer(1, 0, d))
        refused(-1, ctx.fp8_layer, 0)


def test_decoder_loops():
    """lm_decoder_forward and lm_paged_decoder_forward with FP8 FFNs: tokens one after another and at once."""
    announce("fp8 layers: decoder loops")
    d = dataclasses.replace(SMALL, hidden=256, inter=160)
    md = dataclasses.replace(wl.V2_LITE_MLA, hidden=256, heads=4)
    T, page = 24, 16
    with lm.Context(d.moe_config(num_layers=2)) as ctx:
        ctx.attention_configure(wl.mla_config(md, context_length=64))
        ctx.upload_dense(0, *wl.dense_ffn(3, 0, d))
        ctx.finalize_layer(0)
        wl.upload_moe_layer(ctx, 1, wl.moe_layer(3, 1, d))
        ones = np.ones(d.hidden, np.float32)
        for layer in (0, 1):
            wl.upload_mla_layer(ctx, layer, wl.mla_layer(3, layer, md))
            ctx.upload_input_norm(layer, ones)
            ctx.upload_norm(layer, ones)
            ctx.fp8_layer(layer)
        h0 = wl.tokens(4, T, d.hidden)
        runs = {}
        for path in (lm.PATH_FP8, lm.PATH_AUTO):
            ctx.kv_cache_clear()
            h = ctx.to_device(h0)
            ctx.decoder_forward(0, 1, h, T, 0, path=path)
            runs[path] = h.download()
        change = np.linalg.norm(runs[lm.PATH_AUTO] - h0)
        off = np.linalg.norm(runs[lm.PATH_FP8] - runs[lm.PATH_AUTO])
        # the FFNs' outputs are off by 6.4e-2 of their norm, the change holds the attention's too
        assert 0 < off <= 0.13 * change
        ctx.paged_configure(8, page)
        step = lm.PagedStep(requests=1, tokens=T, pages=8, page_size=page, table_width=4, max_added=T)
        arrays = {"cached": np.zeros(1, np.int32), "added": np.array([T], np.int32), "table": np.zeros((1, 4), np.int32),
                  "ring": np.arange(8, dtype=np.int32), "queue_in": np.array([0, 8], np.int32),
                  "queue_out": np.zeros(2, np.int32), "lengths": np.zeros(1, np.int32), "starts": np.zeros(2, np.int32),
                  "positions": np.zeros(T, np.int32), "slots": np.zeros(T, np.int32), "info": np.zeros(4, np.int32)}
        held = {k: ctx.to_device(v) for k, v in arrays.items()}
        for k, b in held.items():
            setattr(step, k, b.ptr)
        ctx.page_plan(step)
        h = ctx.to_device(h0)
        ctx.paged_decoder_forward(0, 1, step, h, path=lm.PATH_FP8)
        assert np.linalg.norm(h.download() - runs[lm.PATH_FP8]) <= 0.13 * change


def test_sizes_past_32_bits_are_refused():
    announce("fp8 layers: sizes past 32 bits")
    d = ALONE
    T = 2 ** 32 // (d.top_k * d.inter)  # one token's activations are the widest rows
    with lm.Context(d.moe_config(num_layers=2)) as ctx:
        wl.upload_moe_layer(ctx, 1, wl.moe_layer(31, 1, d))
        ctx.fp8_layer(1)
        x, y = ctx.empty((T, d.hidden)), ctx.empty((T, d.hidden))
        refused(-1, ctx.moe_forward, 1, x, T, y, path=lm.PATH_FP8)
    d = dataclasses.replace(SMALL, hidden=16, dense_inter=2 ** 20 + 16)
    with lm.Context(d.moe_config(num_layers=1)) as ctx:
        ctx.upload_dense(0, *wl.dense_ffn(1, 0, d))
        ctx.finalize_layer(0)
        refused(-1, ctx.fp8_layer, 0)
