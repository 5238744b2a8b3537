"""LM_PATH_FP8: what a layer's weights go through (freed, uploaded anew and of the other kind, beside live graphs)."""
import dataclasses

import numpy as np
import pytest

import litemind_amd as lm
from conftest import announce
from litemind_amd import workload as wl

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
