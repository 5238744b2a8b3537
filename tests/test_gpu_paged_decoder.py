"""lm_paged_forward and lm_paged_decoder_forward: the models' own latent widths, refused sizes, and what a
refused call leaves."""
import ctypes as C
import dataclasses

import numpy as np
import pytest

import litemind_amd as lm
from conftest import announce
from litemind_amd import workload as wl
from test_gpu_paged_layer import MEAN_REL, SMALL, Service, moe_dims, run_decoder
from test_gpu_paged_layer import test_forward_against_the_oracle as forward_against_the_oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("what", ["weight", "experts", "norm", "workspace"])
def test_a_layer_that_cannot_run_is_found_first(what):
    """A second layer with a weight outside fp16's range, without experts or norm, or a workspace that a captured graph
    holds: the call fails before the hidden state, its padded rows or a pool is touched."""
    announce(f"paged decoder: a second layer that cannot run: {what}")
    d = dataclasses.replace(SMALL, max_positions=64)
    dims = moe_dims(d.hidden)
    mla = [wl.mla_layer(80 + l, l, d) for l in range(2)]
    if what == "weight":
        mla[1].o_proj[3, 5] = wl.f32_to_bf16(np.array([1e6], np.float32))[0]
    pages, page, width = 6, 16, d.kv_lora_rank + d.qk_rope
    with lm.Context(dims.moe_config(num_layers=2)) as ctx:
        ctx.attention_configure(wl.mla_config(d))
        for l in range(2):
            wl.upload_mla_layer(ctx, l, mla[l])
            if what != "experts" or l == 0:
                wl.upload_moe_layer(ctx, l, wl.moe_layer(81, l, dims))
            if what != "norm" or l == 0:
                ctx.upload_norm(l, np.ones(d.hidden, np.float32))
            ctx.upload_input_norm(l, np.ones(d.hidden, np.float32))
        graph = None
        if what == "workspace":
            graph = ctx.stack_graph_create(0, 1, ctx.to_device(np.zeros((8, d.hidden), np.float32)), 8)
        s = Service(ctx, 2, pages, page, 3, 40, 30)
        starts = s.plan([30, 5])
        h = wl.tokens(82, 40, d.hidden)
        h[starts[-1]:] = 7.0
        dh = ctx.to_device(h)
        mark = np.full((2, pages * page, width), 0x3a55, np.uint16)
        for l in range(2):
            ctx._check(ctx.lib.lm_copy_h2d(ctx.handle, C.c_void_p(ctx.paged_pool(l)), mark[l].ctypes.data, mark[l].nbytes))

        def untouched():
            after = np.empty_like(mark)
            for l in range(2):
                ctx._check(ctx.lib.lm_copy_d2h(ctx.handle, after[l].ctypes.data, C.c_void_p(ctx.paged_pool(l)), after[l].nbytes))
            return np.array_equal(dh.download(), h) and np.array_equal(after, mark)

        with pytest.raises(lm.LmError):
            ctx.paged_decoder_forward(0, 1, s.step, dh)
        assert untouched()
        if what == "workspace":
            ctx.stack_graph_destroy(graph)
            ctx.paged_decoder_forward(0, 1, s.step, dh)
        else:
            ctx.paged_decoder_forward(0, 0, s.step, dh)  # the layer that can
        ctx.synchronize()
        y = dh.download()[:starts[-1]]
        assert np.isfinite(y).all() and (y != h[:starts[-1]]).any(axis=1).all()


@pytest.mark.parametrize("hidden,heads,tokens", [(32, 1, 2 ** 24), (64, 1, 2 ** 24), (32, 1, 2 ** 25), (32, 2, 2 ** 23 + 1),
                                                 (2048, 1, 2 ** 19)])
def test_more_tokens_than_a_launch_takes(hidden, heads, tokens):
    """Refused by its numbers, before an array is read or a kernel launched."""
    announce(f"paged layers: {tokens} tokens of {hidden} channels, {heads} heads")
    d = dataclasses.replace(SMALL, hidden=hidden, heads=heads, kv_lora_rank=32, qk_rope=8, max_positions=64)
    with lm.Context(moe_dims(hidden, 1).moe_config(num_layers=1)) as ctx:
        ctx.attention_configure(wl.mla_config(d))
        ctx.paged_configure(4, 16)
        step = lm.PagedStep(requests=1, tokens=tokens, pages=4, page_size=16, table_width=2, max_added=1)
        words = ctx.to_device(np.zeros(8, np.int32))
        for name in ("table", "lengths", "starts", "positions", "slots"):
            setattr(step, name, words.ptr)
        for call in (lambda: ctx.paged_forward(0, step, words, words), lambda: ctx.paged_decoder_forward(0, 0, step, words)):
            with pytest.raises(lm.LmError, match="too many tokens"):
                call()


@pytest.mark.parametrize("heads,page", [(128, 64), (20, 16)])
def test_forward_with_many_heads(heads, page):
    """DeepSeek-V2's 128 heads, and a number that no block of rows divides, against the oracle."""
    forward_against_the_oracle(dataclasses.replace(wl.V2_LITE_MLA, hidden=256, heads=heads), page)


@pytest.mark.parametrize("heads,path", [(16, lm.PATH_AUTO), (16, lm.PATH_MFMA), (128, lm.PATH_AUTO)])
def test_decoder_over_latents_of_512(heads, path):
    """The layer loop through the matrix-core attention, requests together and alone."""
    announce(f"paged decoder: rank 512, {heads} heads, path {path}")
    d = dataclasses.replace(wl.V2_LITE_MLA, hidden=256, heads=heads, max_positions=256)
    together, alone, states = run_decoder(d, path, 2, [37, 1, 64, 18], [1, 1, 3])
    for n, rows in enumerate(together):
        for r, y in enumerate(rows):
            want = alone[r][n]
            change = np.abs(want - states[n][r])
            rel = np.abs(y - want).sum() / change.sum()
            print(f"step {n} request {r}: mean_rel={rel:.3e} of the change")
            # two layers: their attention within its bar on both sides, and experts of 1e-3
            assert np.isfinite(y).all() and rel <= 2 * (2 * MEAN_REL + 1e-3)
