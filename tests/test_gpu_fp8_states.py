"""LM_PATH_FP8: what a layer's weights go through (freed, uploaded anew and of the other kind, beside live graphs)."""
import dataclasses

import numpy as np
import pytest

import fp8_ref as ref
import litemind_amd as lm
from conftest import announce
from litemind_amd import workload as wl
from test_gpu_serving_run import Hip

pytestmark = pytest.mark.gpu

SMALL = dataclasses.replace(wl.V2_LITE, hidden=256, inter=64, experts=160, top_k=6, n_shared=2, dense_inter=400, layers=1)
PATHS = (lm.PATH_AUTO, lm.PATH_GEMV, lm.PATH_MFMA, lm.PATH_FP8)
T = 40


def upload(ctx, kind, d, layer=0):
    if kind == "moe":
        wl.upload_moe_layer(ctx, layer, wl.moe_layer(31, 1, d))
    else:
        ctx.upload_dense(layer, *wl.dense_ffn(31, 0, d))
        ctx.finalize_layer(layer)


def outputs(ctx, kind, d, paths=PATHS, layer=0):
    x, y = ctx.to_device(wl.tokens(5, T, d.hidden)), ctx.empty((T, d.hidden))
    got = []
    for path in paths:
        (ctx.moe_forward if kind == "moe" else ctx.dense_forward)(layer, x, T, y, path=path)
        got.append(y.download())
    return got


@pytest.mark.parametrize("kinds", [("dense", "moe"), ("moe", "dense"), ("dense", "moe", "dense"), ("moe", "moe")], ids="-".join)
def test_another_kind_after_only(kinds):
    """A layer whose other weights were freed takes those of the other kind: the same bits as in a new context."""
    announce(f"fp8 layers: {' then '.join(kinds)} in one layer")
    with lm.Context(SMALL.moe_config(num_layers=1)) as ctx:
        for kind in kinds:
            upload(ctx, kind, SMALL)
            ctx.fp8_layer(0)
            got = outputs(ctx, kind, SMALL)
            with lm.Context(SMALL.moe_config(num_layers=1)) as fresh:
                upload(fresh, kind, SMALL)
                fresh.fp8_layer(0)
                want = outputs(fresh, kind, SMALL)
            for path, a, b in zip(PATHS, got, want):
                assert (a == b).all(), (kind, path)
            ctx.fp8_layer(0, only=True)
            assert (outputs(ctx, kind, SMALL, [lm.PATH_FP8])[0] == want[-1]).all()


def test_beside_a_graph_of_another_path():
    """A live graph of the MFMA path holds nothing of the FP8 path, whose calls grow their workspace beside it; a live
    graph of the FP8 path holds it."""
    announce("fp8 layers: calls beside a live graph of another path")
    d = dataclasses.replace(SMALL, experts=12)
    with lm.Context(d.moe_config(num_layers=1)) as ctx:
        upload(ctx, "moe", d)
        ctx.upload_norm(0, np.ones(d.hidden, np.float32))
        want = {}
        with lm.Context(d.moe_config(num_layers=1)) as fresh:
            upload(fresh, "moe", d)
            fresh.fp8_layer(0)
            for n in (3, 17, T):
                x, y = fresh.to_device(wl.tokens(5, n, d.hidden)), fresh.empty((n, d.hidden))
                fresh.moe_forward(0, x, n, y, path=lm.PATH_FP8)
                want[n] = y.download()
        h0 = wl.tokens(6, T, d.hidden)
        h = ctx.to_device(h0)
        ctx.stack_forward(0, 0, h, T, path=lm.PATH_MFMA)
        once = h.download()

        def fp8(n):
            x, y = ctx.to_device(wl.tokens(5, n, d.hidden)), ctx.empty((n, d.hidden))
            ctx.moe_forward(0, x, n, y, path=lm.PATH_FP8)
            assert (y.download() == want[n]).all(), n

        graph = ctx.stack_graph_create(0, 0, h, T, path=lm.PATH_MFMA)
        try:
            ctx.fp8_layer(0)  # the layer's first FP8 weights, and the path's first workspace
            for n in (3, 17, T):
                h.upload(h0)
                fp8(n)
                ctx.stack_graph_launch(graph)
                assert (h.download() == once).all(), n
        finally:
            ctx.stack_graph_destroy(graph)
        more = T + 24  # once the FP8 graph holds them, more tokens than T are refused
        h.upload(h0)
        graph = ctx.stack_graph_create(0, 0, h, T, path=lm.PATH_FP8)
        try:
            x, y = ctx.empty((more, d.hidden)).zero(), ctx.empty((more, d.hidden))
            with pytest.raises(lm.LmError) as e:
                ctx.moe_forward(0, x, more, y, path=lm.PATH_FP8)
            assert e.value.status == -1
            fp8(T)
        finally:
            ctx.stack_graph_destroy(graph)
        ctx.moe_forward(0, x, more, y, path=lm.PATH_FP8)
        ctx.synchronize()


def test_another_kind_under_a_graph():
    """A graph of a MoE layer's FP8 weights, and then a dense FFN in that layer whose FP8 weights take as many bytes."""
    announce("fp8 layers: another kind under a live graph")
    d = dataclasses.replace(SMALL, hidden=128, inter=128, experts=8, top_k=2, n_shared=0, dense_inter=1024)
    with lm.Context(d.moe_config(num_layers=1)) as ctx:
        upload(ctx, "moe", d)
        ctx.upload_norm(0, np.ones(d.hidden, np.float32))
        ctx.fp8_layer(0, only=True)
        as_moe = ctx.resident_bytes()
        h = ctx.to_device(wl.tokens(6, T, d.hidden))
        graph = ctx.stack_graph_create(0, 0, h, T, path=lm.PATH_FP8)
        try:
            upload(ctx, "dense", d)
            for call in (lambda: ctx.fp8_layer(0), lambda: ctx.stack_graph_launch(graph)):
                with pytest.raises(lm.LmError) as e:
                    call()
                assert e.value.status in (-1, -4)
        finally:
            ctx.stack_graph_destroy(graph)
        ctx.fp8_layer(0)
        got = outputs(ctx, "dense", d)
        with lm.Context(d.moe_config(num_layers=1)) as fresh:
            upload(fresh, "dense", d)
            fresh.fp8_layer(0)
            assert all((a == b).all() for a, b in zip(got, outputs(fresh, "dense", d)))
        ctx.fp8_layer(0, only=True)
        assert ctx.resident_bytes() == as_moe  # the sizes that this test is about


def test_layers_are_not_captured():
    """lm_fp8_layer under capture is refused and ends neither the capture nor the layer's FP8 weights."""
    announce("fp8 layers: lm_fp8_layer under capture")
    with lm.Context(SMALL.moe_config(num_layers=2)) as ctx:
        hip = Hip(ctx)
        for layer in (0, 1):
            upload(ctx, "dense", SMALL, layer)
        ctx.fp8_layer(0)
        want = outputs(ctx, "dense", SMALL)
        said = []
        x = np.random.default_rng(1).standard_normal((4, 128)).astype(np.float32)
        dx, q, s = ctx.to_device(x), ctx.empty((4, 128), np.uint8), ctx.empty((4, 1))

        def work():
            for layer in (0, 1):  # with FP8 weights, and without
                try:
                    ctx.fp8_layer(layer)
                except lm.LmError as e:
                    said.append(e.status)
            ctx.fp8_quantize(dx, 4, 128, q, s)

        graph = hip.capture(work)
        hip.replay(graph[1])
        ctx.synchronize()
        hip.free(*graph)
        assert said == [-1, -1]
        assert (q.download() == ref.quantize(x)[0]).all()
        assert all((a == b).all() for a, b in zip(outputs(ctx, "dense", SMALL), want))
        ctx.fp8_layer(1)
        assert all((a == b).all() for a, b in zip(outputs(ctx, "dense", SMALL, layer=1), want))
