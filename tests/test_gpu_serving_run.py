"""The serving operators together, as a server runs them: a plan, the layers over pages, the head and sampled tokens,
step after step with requests that come and go; then captured and replayed, and on two contexts at once."""
import ctypes as C
import dataclasses

import numpy as np
import pytest

import litemind_amd as lm
import serving_ref as ref
from conftest import announce
from litemind_amd import workload as wl
from test_gpu_paged_attention import Batch
from test_gpu_paged_layer import MEAN_REL, SMALL, Service, moe_dims

pytestmark = pytest.mark.gpu


def settings(rows):
    return np.array([tuple(r) for r in rows], lm.SAMPLING)


class Model:
    def __init__(self, d, layers, vocab, seed=70):
        self.d, self.layers, self.vocab, self.dims = d, layers, vocab, moe_dims(d.hidden, layers)
        self.mla = [wl.mla_layer(seed + l, l, d) for l in range(layers)]
        self.moe = [wl.moe_layer(seed, l, self.dims) for l in range(layers)]
        rng = np.random.default_rng(seed)
        self.embed = rng.normal(size=(vocab, d.hidden)).astype(np.float32)
        self.head = wl.f32_to_bf16((rng.normal(size=(vocab, d.hidden)) * 0.15).astype(np.float32))

    def context(self):
        ctx = lm.Context(self.dims.moe_config(num_layers=self.layers))
        ctx.attention_configure(wl.mla_config(self.d))
        for l in range(self.layers):
            wl.upload_mla_layer(ctx, l, self.mla[l])
            wl.upload_moe_layer(ctx, l, self.moe[l])
            ctx.upload_norm(l, np.ones(self.d.hidden, np.float32))
            ctx.upload_input_norm(l, np.ones(self.d.hidden, np.float32))
        ctx.upload_head(np.ones(self.d.hidden, np.float32), self.head)
        return ctx


def test_requests_come_and_go():
    """Six steps of four rows whose requests end and begin anew.  Every token is the one that the definition takes from
    the logits at hand; every logit that of its request's tokens alone through the single-sequence caches, within the
    layers' tolerance; every page comes back."""
    announce("serving: plan, layers, head and samples over six steps")
    d = dataclasses.replace(SMALL, max_positions=256)
    m = Model(d, 2, 501)
    rng = np.random.default_rng(9)
    R, tokens, pages = 4, 48, 24
    prompts = {0: [list(rng.integers(0, 501, k)) for k in (21, 1, 9, 0)], 2: [None, None, None, list(rng.integers(0, 501, 30))],
               3: [None, list(rng.integers(0, 501, 17)), None, None]}
    ends = {2: [1], 5: [0]}
    sets = settings([(0.0, 0, 1.0, 0.0), (0.8, 20, 0.9, 0.0), (1.3, 0, 0.7, 0.02), (1.0, 0, 1.0, 0.0)])
    history, last, rows_seen = [[] for _ in range(R)], [None] * R, []
    with m.context() as ctx:
        s = Service(ctx, R, pages, 16, 8, tokens, 30)
        for step in range(6):
            fresh = prompts.get(step, [None] * R)
            added, feed = [], []
            for r in range(R):
                if r in ends.get(step, []):
                    added.append(-1)
                    history[r], last[r] = [], None
                    feed.append([])
                    continue
                now = fresh[r] if fresh[r] is not None else [last[r]] if last[r] is not None else []
                added.append(len(now))
                feed.append([int(t) for t in now])
                history[r] += feed[r]
            starts = s.plan(added)
            h = np.full((tokens, d.hidden), np.nan, np.float32)
            flat = [t for f in feed for t in f]
            h[:len(flat)] = m.embed[flat]
            dh, logits, token = ctx.to_device(h), ctx.empty((tokens, m.vocab)), ctx.to_device(np.full(tokens, -7, np.int32))
            u = rng.random(tokens).astype(np.float32)
            owner = np.zeros(tokens, int)
            for r in range(R):
                owner[starts[r]:starts[r + 1]] = r
            ctx.paged_decoder_forward(0, m.layers - 1, s.step, dh)
            ctx.head_forward(dh, tokens, logits=logits)
            ctx.sample(logits, tokens, m.vocab, ctx.to_device(sets[owner]), ctx.to_device(u), token)
            t, x = token.download(), logits.download()
            for r in range(R):
                if starts[r] == starts[r + 1]:
                    continue
                at = starts[r + 1] - 1
                want, _, near = ref.sample(x[at], *sets[r], u[at])
                assert near < 1e-9 or t[at] == want
                last[r] = int(t[at])
                rows_seen.append((list(history[r]), x[at]))
        s.plan([-1] * R)
        assert s.dev["queue_in"].download()[1] == pages
        assert sorted(s.dev["ring"].download()) == list(range(pages))
    with m.context() as ctx:
        for past, x in rows_seen:
            ctx.kv_cache_clear()
            dh, logits = ctx.to_device(m.embed[past]), ctx.empty((len(past), m.vocab))
            ctx.decoder_forward(0, m.layers - 1, dh, len(past), 0)
            ctx.head_forward(dh, len(past), logits=logits)
            want = logits.download()[-1]
            # logits of states whose change is within two layers' bars on both sides
            assert np.abs(x - want).sum() <= 2 * (2 * MEAN_REL + 1e-3) * np.abs(want).sum()


class Hip:
    """Capture and replay on a context's stream, through the HIP runtime that the library uses."""

    def __init__(self, ctx):
        self.ctx, self.rt, self.stream = ctx, C.CDLL("libamdhip64.so"), C.c_void_p(ctx.stream())

    def ok(self, status):
        assert status == 0, status

    def capture(self, work):
        graph, runnable = C.c_void_p(), C.c_void_p()
        self.ok(self.rt.hipStreamBeginCapture(self.stream, 2))  # relaxed
        try:
            work()
        finally:
            self.ok(self.rt.hipStreamEndCapture(self.stream, C.byref(graph)))
        if graph.value:
            self.ok(self.rt.hipGraphInstantiate(C.byref(runnable), graph, None, None, C.c_size_t(0)))
        return graph, runnable

    def replay(self, runnable):
        self.ok(self.rt.hipGraphLaunch(runnable, self.stream))

    def free(self, graph, runnable):
        self.ctx.synchronize()
        if runnable.value:
            self.ok(self.rt.hipGraphExecDestroy(runnable))
        if graph.value:
            self.ok(self.rt.hipGraphDestroy(graph))


@pytest.fixture(scope="module")
def ctx():
    c = lm.Context(wl.V2_LITE.moe_config(num_layers=1))
    yield c
    c.close()


@pytest.mark.parametrize("heads,added", [(16, [1, 1, 1]), (128, [1, 1, 1]), (16, [40, 1, 7])])
def test_captured_attention(ctx, heads, added):
    """Two captured calls over the same scratch, replayed in turn with eager calls of another shape between; lengths
    and tables are read at each replay, not at the capture."""
    announce(f"serving: attention captured and replayed, {heads} heads, {added}")
    first, second = (Batch([300, 40, n], added, heads, seed=n, page=32).upload(ctx) for n in (511, 64))
    other = Batch([700, 5], [1, 33], heads, seed=8).upload(ctx)
    first.check(first.run(ctx))
    second.upload(ctx)
    other.check(other.run(ctx))
    hip = Hip(ctx)
    graphs = [hip.capture(lambda b=b: b.call(ctx)) for b in (first, second)]
    try:
        for turn in range(4):
            for b in (first, second):
                b.dev["out"].upload(np.full((b.tokens + 1, heads, b.rank), 0x1234, np.uint16))
            if turn == 3:  # the second batch's first request shrinks: same queries, fewer keys
                second.cached = [100, 40, 64]
                second.lengths = np.array([c + a for c, a in zip(second.cached, added)], np.int32)
                second.rows[0] = second.rows[0][:second.lengths[0]]
                second.dev["lengths"].upload(second.lengths)
            hip.replay(graphs[0][1])
            hip.replay(graphs[1][1])
            other.call(ctx)
            first.check(first.dev["out"].download())
            second.check(second.dev["out"].download())
            other.check(other.dev["out"].download())
    finally:
        for g in graphs:
            hip.free(*g)


def test_captured_plan_and_samples(ctx):
    """A decode step's plan and its tokens in one graph: each replay takes the next step from the arrays that the one
    before left, as the eager steps of a second set do."""
    announce("serving: plan and samples captured and replayed")
    R, page, pages, width, vocab = 5, 16, 30, 6, 3001
    rng = np.random.default_rng(4)
    x = rng.normal(size=(R, vocab)).astype(np.float32) * 3
    sets = settings([(1.0, 0, 1.0, 0.0), (0.7, 20, 0.9, 0.0), (0.0, 0, 1.0, 0.0), (1.2, 0, 0.8, 0.01), (1.0, 400, 1.0, 0.0)])

    class Set:
        def __init__(self):
            self.dev = {k: ctx.to_device(v) for k, v in {
                "cached": np.array([0, 15, 16, 31, 60], np.int32), "added": np.ones(R, np.int32),
                "table": np.arange(R * width, dtype=np.int32).reshape(R, width) % 12,
                "ring": np.arange(pages, dtype=np.int32)[::-1].copy(), "queue_in": np.array([3, 18], np.int32),
                "starts": np.zeros(R + 1, np.int32), "positions": np.zeros(R, np.int32), "slots": np.zeros(R, np.int32),
                "info": np.zeros(4, np.int32)}.items()}
            self.step = lm.PagedStep(requests=R, tokens=R, pages=pages, page_size=page, table_width=width, max_added=1)
            for k, b in self.dev.items():
                setattr(self.step, k, b.ptr)
            self.step.queue_out, self.step.lengths = self.step.queue_in, self.step.cached  # the step's end is the next's start
            self.u, self.token = ctx.empty(R), ctx.to_device(np.zeros(R, np.int32))
            self.logits, self.sets = ctx.to_device(x), ctx.to_device(sets)

        def work(self):
            ctx.page_plan(self.step)
            ctx.sample(self.logits, R, vocab, self.sets, self.u, self.token)

        def state(self):
            ctx.synchronize()
            return {k: b.download() for k, b in [*self.dev.items(), ("token", self.token)]}

    eager, replayed = Set(), Set()
    eager.u.upload(np.zeros(R, np.float32))
    hip = Hip(ctx)
    graph, runnable = hip.capture(replayed.work)
    try:
        for turn in range(5):
            u = rng.random(R).astype(np.float32)
            for s in (eager, replayed):
                ctx.synchronize()
                s.u.upload(u)
            eager.work()
            hip.replay(runnable)
            a, b = eager.state(), replayed.state()
            for k in a:
                assert np.array_equal(a[k], b[k]), (turn, k)
            assert a["info"][0] == lm.STEP_OK
            assert list(a["cached"]) == [1 + turn, 16 + turn, 17 + turn, 32 + turn, 61 + turn]
            for r in range(R):
                want, _, near = ref.sample(x[r], *sets[r], u[r])
                assert near < 1e-9 or a["token"][r] == want
    finally:
        hip.free(graph, runnable)


def test_capture_refusals():
    """A context's first attention would allocate inside the capture, the layers always: both are refused and leave the
    capture usable."""
    announce("serving: refused captures")
    d = dataclasses.replace(SMALL, max_positions=64)
    with Model(d, 1, 64).context() as c:
        b = Batch([40, 3], [1, 1], 16, seed=1).upload(c)
        s = Service(c, 1, 4, 16, 2, 4, 4)
        s.plan([3])
        h = c.to_device(np.zeros((4, d.hidden), np.float32))
        out = c.to_device(np.zeros((4, d.hidden), np.float32))
        x, u, token = c.to_device(np.zeros((1, 64), np.float32)), c.to_device(np.zeros(1, np.float32)), c.empty(1, np.int32)
        sets = c.to_device(settings([(1.0, 0, 1.0, 0.0)]))
        hip = Hip(c)

        def work():
            with pytest.raises(lm.LmError, match="cannot be captured"):
                b.call(c)
            with pytest.raises(lm.LmError, match="cannot be captured"):
                c.paged_forward(0, s.step, h, out)
            with pytest.raises(lm.LmError, match="cannot be captured"):
                c.paged_decoder_forward(0, 0, s.step, h)
            c.sample(x, 1, 64, sets, u, token)

        graph, runnable = hip.capture(work)
        hip.replay(runnable)
        assert token.download()[0] == 0
        hip.free(graph, runnable)
        b.check(b.run(c))


def test_two_contexts_at_once(ctx):
    """Calls of two contexts in flight together, each with scratch of its own."""
    announce("serving: two contexts at once")
    with lm.Context(wl.V2_LITE.moe_config(num_layers=1)) as second:
        pairs = [(c, Batch([900, 40, 333, 2000 + n], [1, 50, 3, 1], 16, seed=n).upload(c))
                 for n, c in enumerate((ctx, second))]
        rng = np.random.default_rng(3)
        x = rng.normal(size=(40, 20011)).astype(np.float32) * 2
        u, sets = rng.random(40).astype(np.float32), settings([(1.0, 0, 0.9, 0.0)] * 40)
        draws = [(c, c.to_device(x), c.to_device(u), c.to_device(sets), c.empty(40, np.int32)) for c, _ in pairs]
        for _ in range(8):
            for (c, b), (_, dx, du, ds, token) in zip(pairs, draws):
                b.call(c)
                c.sample(dx, 40, 20011, ds, du, token)
        for (c, b), (_, _, _, _, token) in zip(pairs, draws):
            b.check(b.dev["out"].download())
            for r, t in enumerate(token.download()):
                want, _, near = ref.sample(x[r], *sets[r], u[r])
                assert near < 1e-9 or t == want
