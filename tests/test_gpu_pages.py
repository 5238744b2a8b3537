"""lm_page_plan on the GPU against the plain restatement: every array whole, and nothing else written."""
import random

import numpy as np
import pytest

import litemind_amd as lm
import serving_ref as ref
from conftest import announce
from litemind_amd import workload as wl

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = lm.Context(wl.V2_LITE.moe_config(num_layers=1))
    yield c
    c.close()


class Plan:
    """A step's arrays on the GPU with guard words behind each."""

    def __init__(self, ctx, cached, added, table, ring, queue, page, tokens, max_added, in_place=False):
        self.ctx, R = ctx, len(cached)
        self.host = {"cached": np.asarray(cached, np.int32), "added": np.asarray(added, np.int32),
                     "table": np.asarray(table, np.int32), "ring": np.asarray(ring, np.int32),
                     "queue_in": np.asarray(queue, np.int32), "queue_out": np.asarray(queue, np.int32),
                     "lengths": np.full(R, 77, np.int32), "starts": np.full(R + 1, 77, np.int32),
                     "positions": np.full(tokens, 77, np.int32), "slots": np.full(tokens, 77, np.int32),
                     "info": np.full(4, 77, np.int32)}
        self.dev = {k: ctx.to_device(np.concatenate([v.reshape(-1), np.full(9, 123, np.int32)]))
                    for k, v in self.host.items()}
        self.step = lm.PagedStep(requests=R, tokens=tokens, pages=len(ring), page_size=page,
                                 table_width=self.host["table"].shape[1], max_added=max_added)
        for k, b in self.dev.items():
            setattr(self.step, k, b.ptr)
        if in_place:
            self.step.queue_out = self.step.queue_in

    def read(self):
        out = {}
        for k, b in self.dev.items():
            whole = b.download()
            assert (whole[-9:] == 123).all(), k
            out[k] = whole[:-9].reshape(self.host[k].shape)
        out["queue"] = out["queue_in" if self.step.queue_out == self.step.queue_in else "queue_out"]
        return out


def service(seed, R, page, width, spare, most_added, over):
    """Requests in service, their pages scattered, a ring of free ones that wraps."""
    rng = random.Random(seed)
    cached = [rng.randint(0, page * (width - 1)) for _ in range(R)]
    added = [rng.choice([0, 1, 1, rng.randint(0, min(most_added, page * width - c))]) for c in cached]
    for r in rng.sample(range(R), over):
        added[r] = -rng.randint(1, 5)
    held = [ref.pages_of(c, page) for c in cached]
    need = sum(ref.pages_of(c + a, page) - h for c, a, h in zip(cached, added, held) if a > 0)
    pages = sum(held) + need + spare
    ids = list(range(pages))
    rng.shuffle(ids)
    table = np.full((R, width), -7, np.int32)
    for r, h in enumerate(held):
        table[r, :h] = [ids.pop() for _ in range(h)]
    ring, head = np.full(pages, -5, np.int32), rng.randrange(pages)
    for k, page_id in enumerate(ids):
        ring[(head + k) % pages] = page_id
    return cached, added, table, ring, [head, len(ids)], need


def check(plan, want):
    got = plan.read()
    for k in ref.STEP_ARRAYS:
        assert np.array_equal(got[k], want[k]), k
    for k in ("cached", "added"):
        assert np.array_equal(got[k], plan.host[k]), k


@pytest.mark.parametrize("R,page,width,spare,most,over", [
    (1, 16, 2, 0, 16, 0), (2, 16, 3, 1, 20, 1), (7, 48, 5, 2, 60, 2), (64, 64, 70, 11, 300, 5),
    (1023, 16, 9, 3, 30, 100), (1024, 32, 4, 0, 40, 0), (1025, 16, 9, 5, 50, 513), (3000, 16, 4, 7, 17, 1000)])
def test_plan(ctx, R, page, width, spare, most, over):
    announce(f"page plan of {R} requests, pages of {page}")
    cached, added, table, ring, queue, need = service(R + page, R, page, width, spare, most, over)
    tokens = sum(max(a, 0) for a in added)
    for pad in (0, 37):
        args = (cached, added, table, ring, queue, page, tokens + pad, most)
        plan = Plan(ctx, *args, in_place=pad > 0)
        ctx.page_plan(plan.step)
        want = ref.plan(*args)
        assert want["info"][0] == 0
        check(plan, want)
        if pad == 0:  # the same step planned again: the same
            ctx.page_plan(plan.step)
            check(plan, want)


def test_nothing_new(ctx):
    announce("page plan of a step without tokens")
    args = ([5, 0, 32], [0, 0, 0], np.arange(6).reshape(3, 2), np.arange(8), [3, 2], 16, 0, 0)
    plan = Plan(ctx, *args)
    ctx.page_plan(plan.step)
    check(plan, ref.plan(*args))


@pytest.mark.parametrize("what", ["length", "negative", "tokens", "added", "pages", "count", "long"])
def test_refused_steps_change_nothing(ctx, what):
    announce(f"page plan that cannot be served: {what}")
    cached, added, table, ring, queue, need = service(5, 40, 16, 6, 3, 40, 4)
    tokens, most, status = sum(max(a, 0) for a in added), 40, None
    if what == "length":
        cached[7], added[7], status = 95, 2, lm.STEP_LENGTH
    elif what == "negative":
        cached[39], status = -1, lm.STEP_LENGTH
    elif what == "long":  # in 64 bits: cached + added passes 2^31
        cached[3], added[3], status = 2 ** 31 - 1, 2 ** 31 - 1, lm.STEP_LENGTH
    elif what == "tokens":
        tokens, status = tokens - 1, lm.STEP_TOKENS
    elif what == "added":
        most, status = max(added) - 1, lm.STEP_TOKENS
    elif what == "pages":
        queue, status = [queue[0], need - 1], lm.STEP_PAGES
    elif what == "count":
        queue, status = [queue[0], -3], lm.STEP_PAGES
    args = (cached, added, table, ring, queue, 16, tokens, most)
    plan = Plan(ctx, *args)
    ctx.page_plan(plan.step)
    want = ref.plan(*args)
    assert want["info"][0] == status
    check(plan, want)


def test_page_ids_outside_the_pool(ctx):
    announce("page plan over a table and a ring with page ids outside the pool")
    table = np.array([[9, -1], [-2 ** 31, 0], [3, 0]], np.int32)
    ring = np.array([2 ** 31 - 1, 1, 2, 3, 4, 5, 6, 7, 8], np.int32)
    args = ([3, 15, 16], [2, 1, 2], table, ring, [0, 5], 16, 5, 2)
    plan = Plan(ctx, *args)
    ctx.page_plan(plan.step)
    want = ref.plan(*args)
    assert want["slots"].tolist() == [-1, -1, -1, -1, -1]
    check(plan, want)


def test_steps_in_turn(ctx):
    announce("page plans in turn: requests grow, end and begin again")
    rng, R, page, width, pages = random.Random(9), 30, 16, 12, 200
    cached, table = [0] * R, np.full((R, width), -1, np.int32)
    ring, queue = np.arange(pages, dtype=np.int32), [0, pages]
    plan = Plan(ctx, cached, [0] * R, table, ring, queue, page, 400, 40, in_place=True)
    for turn in range(12):
        added = [-1 if c > 100 and rng.random() < 0.5 else rng.choice([0, 1, rng.randint(0, 13)]) for c in cached]
        plan.dev["cached"].upload(np.array(cached, np.int32))
        plan.dev["added"].upload(np.array(added, np.int32))
        plan.host["cached"], plan.host["added"] = np.array(cached, np.int32), np.array(added, np.int32)
        ctx.page_plan(plan.step)
        want = ref.plan(cached, added, table, ring, queue, page, 400, 40)
        check(plan, want)
        assert want["info"][0] == 0
        cached, table, ring, queue = want["lengths"].tolist(), want["table"], want["ring"], want["queue"].tolist()
        live = [table[r, :ref.pages_of(c, page)].tolist() for r, c in enumerate(cached)]
        held = [x for row in live for x in row] + [ring[(queue[0] + k) % pages] for k in range(queue[1])]
        assert sorted(held) == list(range(pages))  # every page in one place


def test_rings_that_cannot_be(ctx):
    """A negative count, and requests that give back more pages than the pool has room for: refused, nothing changed."""
    announce("page plan: rings that cannot be")
    table, ring = np.arange(12, dtype=np.int32).reshape(3, 4) % 9, np.arange(9, dtype=np.int32)
    for cached, added, queue in (([1, 2, 3], [0, 0, 0], [0, -1]), ([64, 64, 64], [-1, -1, -1], [4, 0]),
                                 ([64, 64, 1], [-1, -1, 1], [4, 2]), ([1, 2, 3], [0, 0, 0], [0, 10])):
        plan = Plan(ctx, cached, added, table, ring, queue, 16, 4, 4)
        ctx.page_plan(plan.step)
        got = plan.read()
        assert got["info"].tolist() == [lm.STEP_RING, 0, 0, 0]
        assert got["queue_out"].tolist() == [queue[0], queue[1]] and got["starts"].tolist() == [0] * 4
        assert np.array_equal(got["table"], table) and np.array_equal(got["ring"], ring)
        assert got["lengths"].tolist() == cached and (got["slots"] == -1).all() and (got["positions"] == 0).all()
