"""The model's layers over pages (lm_paged_forward, lm_paged_decoder_forward) against the oracle's Attention::forward
and the single-sequence decoder, and a run of planning, layers, head and sampling together.

Beside exact arithmetic the layer rounds to fp16 its input, the queries, the absorbed queries, the latents, the
softmax weights, the summed latents and the heads' outputs: along an output's path six relative roundings of 2^-11
(2.9e-3), and a score of size s moves its weight by 3 s 2^-11, of either sign from key to key.  That stays under the
MFMA path's bar on the mean, 5e-3; one element is held to 5e-2 on outputs of magnitude 1, as there."""
import ctypes as C
import dataclasses

import numpy as np
import pytest

import litemind_amd as lm
import oracle_lib as ol
import serving_ref as ref
from conftest import announce, layer_error
from litemind_amd import workload as wl

pytestmark = pytest.mark.gpu
MEAN_REL, MAX_ABS = 5e-3, 5e-2
SMALL = dataclasses.replace(wl.V2_LITE_MLA, hidden=256, heads=4, kv_lora_rank=64, qk_nope=32, qk_rope=16, v_head=32,
                            max_positions=256)


def moe_dims(hidden, layers=2):
    return wl.Dims(hidden=hidden, inter=128, experts=8, top_k=2, n_shared=1, dense_inter=256, layers=layers)


class Service:
    """Requests over a context's pages, planned on the GPU step by step."""

    def __init__(self, ctx, R, pages, page, width, tokens, max_added):
        self.ctx, self.R, self.tokens = ctx, R, tokens
        ctx.paged_configure(pages, page)
        self.cached = np.zeros(R, np.int32)
        order = np.random.default_rng(pages).permutation(pages).astype(np.int32)
        self.dev = {k: ctx.to_device(v) for k, v in {
            "cached": self.cached, "added": np.zeros(R, np.int32), "table": np.full((R, width), -1, np.int32),
            "ring": order, "queue_in": np.array([0, pages], np.int32), "lengths": np.zeros(R, np.int32),
            "starts": np.zeros(R + 1, np.int32), "positions": np.zeros(tokens, np.int32),
            "slots": np.zeros(tokens, np.int32), "info": np.zeros(4, np.int32)}.items()}
        self.step = lm.PagedStep(requests=R, tokens=tokens, pages=pages, page_size=page, table_width=width,
                                 max_added=max_added)
        for k, b in self.dev.items():
            setattr(self.step, k, b.ptr)
        self.step.queue_out = self.step.queue_in

    def put(self, name, value):
        self.ctx.synchronize()
        self.dev[name].upload(np.asarray(value, np.int32))

    def plan(self, added):
        self.put("cached", self.cached)
        self.put("added", added)
        self.ctx.page_plan(self.step)
        self.cached = self.dev["lengths"].download()
        assert self.dev["info"].download()[0] == lm.STEP_OK
        return self.dev["starts"].download()


def oracle_caches(d, R):
    return [ol.OracleKvCache(d, d.max_positions) for _ in range(R)]


@pytest.mark.parametrize("d,page", [(wl.V2_LITE_MLA, 64), (dataclasses.replace(wl.V2_LITE_MLA, q_lora_rank=1536), 16),
                                    (SMALL, 16), (dataclasses.replace(SMALL, q_lora_rank=96, yarn=False), 48)])
def test_forward_against_the_oracle(d, page):
    """Prompts of odd lengths, then chunks, single tokens and a request that rests, padded rows of NaN behind them."""
    d = dataclasses.replace(d, max_positions=256)
    announce(f"paged layer: hidden {d.hidden}, rank {d.kv_lora_rank}, q LoRA {d.q_lora_rank}, pages of {page}")
    L = wl.mla_layer(31, 0, d)
    with lm.Context(moe_dims(d.hidden).moe_config(num_layers=2)) as ctx:
        ctx.attention_configure(wl.mla_config(d))
        wl.upload_mla_layer(ctx, 1, L)
        steps = [[1, 17, 40, 64, 0], [1, 1, 0, 23, 5], [1, 1, 1, 1, 1], [0, 90, 1, -1, 2]]
        s = Service(ctx, 5, 40, page, 16, 130, 90)
        caches = oracle_caches(d, 5)
        seen = [0] * 5
        for n, added in enumerate(steps):
            starts = s.plan(added)
            x = wl.tokens(100 + n, s.tokens, d.hidden)
            x[starts[-1]:] = np.nan
            base = wl.tokens(200 + n, s.tokens, d.hidden)
            dx, dout, dsum = ctx.to_device(x), ctx.to_device(np.full_like(x, np.nan)), ctx.to_device(base)
            ctx.paged_forward(1, s.step, dx, dout)
            y = dout.download()
            ctx.paged_forward(1, s.step, dx, dsum, accumulate=True)  # the same latents into the same slots
            added_to = dsum.download()
            assert (y[starts[-1]:] == 0).all() and np.array_equal(added_to[starts[-1]:], base[starts[-1]:])
            for r in range(5):
                lo, hi = starts[r], starts[r + 1]
                if hi == lo:
                    continue
                want, k = ol.oracle_mla(L, x[lo:hi], seen[r], caches[r])
                assert k == hi - lo
                seen[r] += hi - lo
                mx, rel = layer_error(y[lo:hi], want)
                print(f"step {n} request {r}: {hi - lo} tokens max_abs={mx:.3e} mean_rel={rel:.3e}")
                assert mx <= MAX_ABS and rel <= MEAN_REL
                np.testing.assert_allclose(added_to[lo:hi], base[lo:hi] + y[lo:hi], rtol=0, atol=2.0 ** -20)


def test_pool_rows():
    """The slots hold the oracle's latents, rounded; every other row stays as it was, padded batch or not."""
    d = dataclasses.replace(SMALL, max_positions=64)
    announce("paged layer: what lies in the pool")
    L = wl.mla_layer(32, 0, d)
    width, pages, page = d.kv_lora_rank + d.qk_rope, 12, 16
    with lm.Context(moe_dims(d.hidden).moe_config(num_layers=2)) as ctx:
        ctx.attention_configure(wl.mla_config(d))
        for layer in (0, 1):
            wl.upload_mla_layer(ctx, layer, L)
        s = Service(ctx, 3, pages, page, 6, 70, 40)
        assert ctx.paged_pool(1) - ctx.paged_pool(0) == 2 * pages * page * width
        starts = s.plan([33, 1, 20])
        slots, positions = s.dev["slots"].download(), s.dev["positions"].download()
        x = wl.tokens(5, s.tokens, d.hidden)
        x[starts[-1]:] = 3e38
        before = np.full((pages * page, width), 0x3a55, np.uint16)
        ctx._check(ctx.lib.lm_copy_h2d(ctx.handle, C.c_void_p(ctx.paged_pool(1)), before.ctypes.data, before.nbytes))
        dx, dout = ctx.to_device(x), ctx.to_device(np.zeros_like(x))
        ctx.paged_forward(1, s.step, dx, dout)
        ctx.synchronize()
        pool, other = np.empty((2, pages * page, width), np.uint16)
        for layer, to in ((1, pool), (0, other)):
            ctx._check(ctx.lib.lm_copy_d2h(ctx.handle, to.ctypes.data, C.c_void_p(ctx.paged_pool(layer)), to.nbytes))
        assert (other == 0).all()
        n = int(starts[-1])
        rest = np.ones(pages * page, bool)
        rest[slots[:n]] = False
        assert (pool[rest] == 0x3a55).all()
        wide = (L.kv_a_proj.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
        lat = x[:n].astype(np.float64) @ wide.T
        # x rounds to fp16, relative 2^-11: no projected value moves by more than 2^-11 sum |w x|, to which 32-bit sums
        # add less than `hidden` 2^-24 of it
        unit = 2.0 ** -11 + d.hidden * 2.0 ** -24
        moved = unit * (np.abs(x[:n]).astype(np.float64) @ np.abs(wide).T)
        c, dc = lat[:, :d.kv_lora_rank], moved[:, :d.kv_lora_rank]
        root = np.sqrt((c * c).mean(1, keepdims=True) + d.rms_norm_eps)
        droot = np.sqrt((dc * dc).mean(1, keepdims=True))  # a norm moves by the change's norm at most
        gain = np.abs(L.kv_a_layernorm.astype(np.float64))
        dc = gain * (dc + np.abs(c) * droot / root) / (root - droot)
        c = c / root * L.kv_a_layernorm
        cos, sin = ol.oracle_rope_tables(d)
        e, o = lat[:, d.kv_lora_rank::2], lat[:, d.kv_lora_rank + 1::2]
        de, do = moved[:, d.kv_lora_rank::2], moved[:, d.kv_lora_rank + 1::2]
        co, si = cos[positions[:n]].astype(np.float64), sin[positions[:n]].astype(np.float64)
        want = np.concatenate([c, e * co - o * si, o * co + e * si], 1)
        bound = np.concatenate([dc, de * np.abs(co) + do * np.abs(si), do * np.abs(co) + de * np.abs(si)], 1)
        got = pool[slots[:n]].view(np.float16).astype(np.float64)
        # the row rounds to fp16 (2^-11 relative, 2^-25 under 2^-14), after 32-bit steps of a few units
        assert (np.abs(got - want) <= bound + (2.0 ** -11 + 2.0 ** -20) * (np.abs(want) + bound) + 2.0 ** -25).all()


def test_pages_past_four_gigabytes():
    """A layer's pool of 5 GB: latents stored to its last pages, and read there."""
    announce("paged layer: pages past 4 GiB")
    d = dataclasses.replace(SMALL, max_positions=64)
    L, pages, page = wl.mla_layer(33, 0, d), 8000, 4096
    with lm.Context(moe_dims(d.hidden).moe_config(num_layers=1)) as ctx:
        ctx.attention_configure(wl.mla_config(d))
        wl.upload_mla_layer(ctx, 0, L)
        s = Service(ctx, 2, pages, page, 1, 40, 30)
        s.put("ring", np.arange(pages)[::-1])
        caches, seen = oracle_caches(d, 2), [0, 0]
        for added in ([9, 30], [1, 1]):
            starts = s.plan(added)
            assert int(s.dev["slots"].download()[:starts[-1]].min()) * (d.kv_lora_rank + d.qk_rope) * 2 > 2 ** 32
            x = wl.tokens(7 + added[0], s.tokens, d.hidden)
            dout = ctx.to_device(np.zeros_like(x))
            ctx.paged_forward(0, s.step, ctx.to_device(x), dout)
            y = dout.download()
            for r in range(2):
                lo, hi = starts[r], starts[r + 1]
                want, _ = ol.oracle_mla(L, x[lo:hi], seen[r], caches[r])
                seen[r] += hi - lo
                mx, rel = layer_error(y[lo:hi], want)
                assert mx <= MAX_ABS and rel <= MEAN_REL


def run_decoder(d, path, layers, prompts, follow):
    """The same tokens through pages, all requests together, and alone through the single-sequence caches."""
    dims = moe_dims(d.hidden, layers)
    mla = [wl.mla_layer(40 + l, l, d) for l in range(layers)]
    moe = [wl.moe_layer(50, l, dims) for l in range(layers)]
    R = len(prompts)

    def build():
        ctx = lm.Context(dims.moe_config(num_layers=layers))
        ctx.attention_configure(wl.mla_config(d))
        for l in range(layers):
            wl.upload_mla_layer(ctx, l, mla[l])
            wl.upload_moe_layer(ctx, l, moe[l])
            ctx.upload_norm(l, np.full(d.hidden, 1.0, np.float32))
            ctx.upload_input_norm(l, np.full(d.hidden, 1.0 + 0.1 * l, np.float32))
        return ctx

    steps = [prompts] + [[f] * R for f in follow]
    states = [[wl.tokens(60 + 10 * n + r, k, d.hidden) for r, k in enumerate(added)] for n, added in enumerate(steps)]
    together, alone = [], []
    with build() as ctx:
        s = Service(ctx, R, 64, 16, 24, sum(prompts) + 3, max(prompts))
        for n, added in enumerate(steps):
            starts = s.plan(added)
            h = np.full((s.tokens, d.hidden), np.nan, np.float32)
            h[:starts[-1]] = np.concatenate(states[n])
            dh = ctx.to_device(h)
            ctx.paged_decoder_forward(0, layers - 1, s.step, dh, path)
            y = dh.download()
            together.append([y[starts[r]:starts[r + 1]] for r in range(R)])
    with build() as ctx:
        for r in range(R):
            ctx.kv_cache_clear()
            at, rows = 0, []
            for n, added in enumerate(steps):
                dh = ctx.to_device(states[n][r])
                ctx.decoder_forward(0, layers - 1, dh, added[r], at, path)
                rows.append(dh.download())
                at += added[r]
            alone.append(rows)
    return together, alone, states


@pytest.mark.parametrize("path", [lm.PATH_AUTO, lm.PATH_MFMA])
def test_decoder_together_as_alone(path):
    announce(f"paged decoder: path {path}")
    d = dataclasses.replace(SMALL, max_positions=256)
    together, alone, states = run_decoder(d, path, 2, [37, 1, 64, 18], [1, 1, 3])
    for n, rows in enumerate(together):
        for r, y in enumerate(rows):
            want = alone[r][n]
            change = np.abs(want - states[n][r])
            rel = np.abs(y - want).sum() / change.sum()
            print(f"step {n} request {r}: mean_rel={rel:.3e} of the change")
            # what two layers add: their attention each within its bar on both sides, and experts of 1e-3
            assert np.isfinite(y).all() and rel <= 2 * (2 * MEAN_REL + 1e-3)


def test_refusals():
    announce("paged layers: refused calls")
    d = dataclasses.replace(SMALL, max_positions=64)
    with lm.Context(moe_dims(d.hidden).moe_config(num_layers=2)) as ctx:
        step = lm.PagedStep(requests=1, tokens=1, pages=4, page_size=16, table_width=2, max_added=1)
        x, y = ctx.to_device(np.zeros((1, d.hidden), np.float32)), ctx.to_device(np.zeros((1, d.hidden), np.float32))

        def refused(f, *args, match):
            with pytest.raises(lm.LmError, match=match):
                f(*args)

        refused(ctx.paged_configure, 4, 16, match="not configured")
        ctx.attention_configure(wl.mla_config(d))
        refused(ctx.paged_pool, 0, match="not configured")
        refused(ctx.paged_forward, 0, step, x, y, match="pages are not configured")
        ctx.paged_configure(4, 16)
        refused(ctx.paged_configure, 4, 16, match="already")
        refused(ctx.paged_pool, 2, match="out of range")
        refused(ctx.paged_forward, 0, step, x, y, match="null or misaligned")
        s = np.zeros(8, np.int32)
        arrays = ctx.to_device(s)
        for name in ("table", "lengths", "starts", "positions", "slots"):
            setattr(step, name, arrays.ptr)
        refused(ctx.paged_forward, 2, step, x, y, match="out of range")
        refused(ctx.paged_forward, 0, step, None, y, match="null input")
        refused(ctx.paged_forward, 0, step, x, x, match="overlaps")
        refused(ctx.paged_forward, 0, step, x, y, match="no attention weights")
        refused(ctx.paged_decoder_forward, 0, 1, step, x, match="no attention weights or input norm")
        refused(ctx.paged_decoder_forward, 1, 0, step, x, match="first_layer > last_layer")
        refused(ctx.paged_decoder_forward, 0, 1, step, None, match="null hidden")
        step.pages = 5
        refused(ctx.paged_forward, 0, step, x, y, match="differ")
        step.pages, step.page_size = 4, 32
        refused(ctx.paged_forward, 0, step, x, y, match="differ")
        step.page_size, step.tokens = 16, 0
        ctx.paged_forward(0, step, x, y)  # nothing to do
    odd = dataclasses.replace(d, qk_nope=40)
    with lm.Context(moe_dims(d.hidden).moe_config(num_layers=1)) as ctx:
        ctx.attention_configure(wl.mla_config(odd))
        with pytest.raises(lm.LmError, match="multiples of 32"):
            ctx.paged_configure(4, 16)
