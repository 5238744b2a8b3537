"""lm_page_plan and lm_paged_attention at the ends of the sizes and rings that they take."""
import ctypes as C

import numpy as np
import pytest

import litemind_amd as lm
import serving_ref as ref
from conftest import announce
from litemind_amd import workload as wl
from test_gpu_pages import Plan, check
from test_gpu_paged_attention import SCALE, Batch, decode, encode

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = lm.Context(wl.V2_LITE.moe_config(num_layers=1))
    yield c
    c.close()


def words(ctx, buffer, first, count):
    out = np.empty(count, np.int32)
    ctx._check(ctx.lib.lm_copy_d2h(ctx.handle, out.ctypes.data, C.c_void_p(buffer.ptr + 4 * first), out.nbytes))
    return out


def test_as_many_tokens_as_a_step_takes(ctx):
    """2^31 - 25 new tokens of two requests, a third without any between them, and five padded rows."""
    announce("page plan: 2^31 - 25 new tokens")
    page, pages = 16, 2 ** 27 - 1
    first = 16 * 62500000 + 7
    second = 16 * (pages - 62500001)
    new, tokens = first + second, first + second + 5
    assert new == 2 ** 31 - 25
    width = second // 16
    dev = {"cached": ctx.to_device(np.zeros(3, np.int32)), "added": ctx.to_device(np.array([first, 0, second], np.int32)),
           "table": ctx.empty((3, width), np.int32), "ring": ctx.to_device(np.arange(pages, dtype=np.int32)),
           "queue_in": ctx.to_device(np.array([0, pages], np.int32)), "queue_out": ctx.empty(2, np.int32),
           "lengths": ctx.empty(3, np.int32), "starts": ctx.empty(4, np.int32),
           "positions": ctx.empty(tokens + 64, np.int32), "slots": ctx.empty(tokens + 64, np.int32),
           "info": ctx.empty(4, np.int32)}
    step = lm.PagedStep(requests=3, tokens=tokens, pages=pages, page_size=page, table_width=width, max_added=second)
    for k, b in dev.items():
        setattr(step, k, b.ptr)
    for k in ("positions", "slots"):
        ctx._check(ctx.lib.lm_copy_h2d(ctx.handle, C.c_void_p(dev[k].ptr + 4 * (tokens - 100)),
                                       np.full(164, 123, np.int32).ctypes.data, 4 * 164))
    ctx.page_plan(step)
    assert dev["info"].download().tolist() == [lm.STEP_OK, new, pages, 0]
    assert dev["starts"].download().tolist() == [0, first, first, new]
    assert dev["lengths"].download().tolist() == [first, 0, second]
    assert dev["queue_out"].download().tolist() == [0, 0]
    count = 1 << 20
    for at in (0, first - count // 2, first, 2 ** 30 - 5000, 3 * 2 ** 29, new - 3 * count, new - count):
        t = np.arange(at, at + count, dtype=np.int64)
        position = np.where(t < first, t, t - first)
        slot = position + np.where(t < first, 0, 62500001 * 16)
        assert np.array_equal(words(ctx, dev["positions"], at, count), position), at
        assert np.array_equal(words(ctx, dev["slots"], at, count), slot), at
    assert words(ctx, dev["positions"], new, 5 + 64).tolist() == [0] * 5 + [123] * 64
    assert words(ctx, dev["slots"], new, 5 + 64).tolist() == [-1] * 5 + [123] * 64
    assert np.array_equal(words(ctx, dev["table"], 2 * width + width - 1000, 1000), np.arange(pages - 1000, pages))
    for b in dev.values():
        b.free()


@pytest.mark.parametrize("heads,added", [(1, 1), (8, 3)])
@pytest.mark.parametrize("dtype", [lm.DT_F16, lm.DT_BF16])
def test_attention_over_the_longest_row(ctx, heads, added, dtype):
    """2^31 - 16 keys: one page of zeros and ones named again and again, and another at the end.  Queries of zeros weigh
    all alike, so the outputs are counts of keys over their number: sums of whole numbers in 32 bits, 300 parts and 16
    tiles' roundings of 2^-24 at most where they pass 2^24, and the output's own."""
    announce(f"paged attention: {added} tokens at the end of 2^31 - 16 keys, {heads} heads, dtype {dtype}")
    page, columns, big = 16, 2 ** 27 - 1, 32768.0
    rows = np.zeros((2, page, 576))
    rows[0, :, 0], rows[0, ::2, 1], rows[1, :, 2] = 1.0, 1.0, big
    table = np.zeros((1, columns), np.int32)
    table[0, -1] = 1
    dev = {"table": ctx.to_device(table), "lengths": ctx.to_device(np.array([page * columns], np.int32)),
           "starts": ctx.to_device(np.array([0, added], np.int32)),
           "q": ctx.to_device(np.zeros((added, heads, 576), np.uint16)), "pool": ctx.to_device(encode(rows, dtype)),
           "out": ctx.to_device(np.full((added, heads, 512), 0x1234, np.uint16))}
    step = lm.PagedStep(requests=1, tokens=added, pages=2, page_size=page, table_width=columns, max_added=added)
    for k in ("table", "lengths", "starts"):
        setattr(step, k, dev[k].ptr)
    ctx.paged_attention(step, dev["q"], dev["pool"], heads, SCALE, dev["out"], dtype=dtype)
    got = decode(dev["out"].download(), dtype)
    for b in dev.values():
        b.free()
    unit = 2.0 ** -11 if dtype == lm.DT_F16 else 2.0 ** -8
    for i in range(added):
        last = page - added + i + 1
        n = page * (columns - 1) + last
        want = np.zeros(512)
        want[:3] = page * (columns - 1) / n, page // 2 * (columns - 1) / n, big * last / n
        assert (np.abs(got[i] - want) <= want * (unit + 316 * 2.0 ** -24)).all(), got[i, 0, :4]


@pytest.mark.parametrize("pages,count,taken,back", [(10, 4, 4, 10), (9, 4, 4, 8), (9, 4, 4, 6), (9, 4, 1, 6), (9, 11, 3, 0),
                                                    (9, 11, 11, 1), (9, 0, 0, 10), (1, 1, 1, 1)])
def test_rings_without_room(ctx, pages, count, taken, back):
    """Free and returned pages that need more places than the ring has, in steps that take pages too: refused, whatever
    is left after the step, and nothing changed."""
    announce(f"page plan: {count} free pages of {pages}, {taken} taken, {back} given back")
    assert count + back > pages and taken <= count
    width = max(taken, back, 1)
    table, ring = np.arange(2 * width, dtype=np.int32).reshape(2, width) % pages, np.arange(pages, dtype=np.int32)
    cached, added = [0, 16 * back], [16 * taken, -1]
    plan = Plan(ctx, cached, added, table, ring, [3, count], 16, 16 * taken + 2, 16 * taken)
    ctx.page_plan(plan.step)
    got = plan.read()
    assert got["info"].tolist() == [lm.STEP_RING, 0, 0, 0]
    assert got["queue_out"].tolist() == [3 % pages, count] and got["starts"].tolist() == [0] * 3
    assert np.array_equal(got["table"], table) and np.array_equal(got["ring"], ring)
    assert got["lengths"].tolist() == cached and (got["slots"] == -1).all() and (got["positions"] == 0).all()


@pytest.mark.parametrize("pages,count,taken,back", [(10, 4, 4, 6), (9, 4, 1, 5), (9, 9, 9, 0), (9, 0, 0, 9), (2, 1, 1, 1)])
def test_rings_just_full(ctx, pages, count, taken, back):
    """Free and returned pages that fill the ring: served, and the same when planned again."""
    announce(f"page plan: {count} free pages of {pages}, {taken} taken, {back} given back, the ring full")
    width = max(taken, back, 1)
    ids = np.random.default_rng(pages).permutation(pages).astype(np.int32)
    ring, table = np.full(pages, -5, np.int32), np.full((2, width), -7, np.int32)
    ring[(3 + np.arange(count)) % pages] = ids[:count]
    table[1, :back] = ids[count:count + back]
    args = ([0, 16 * back], [16 * taken, -1], table, ring, [3 % pages, count], 16, 16 * taken, 16 * taken)
    plan = Plan(ctx, *args)
    want = ref.plan(*args)
    assert want["info"].tolist() == [0, 16 * taken, taken, back]
    for _ in range(2):
        ctx.page_plan(plan.step)
        check(plan, want)


@pytest.mark.parametrize("rank,rope", [(512, 64), (64, 16)])
@pytest.mark.parametrize("starts", [[0, 2 ** 31 - 1, -2 ** 31, -2 ** 31], [-2 ** 31, 2 ** 31 - 1, -1, -2 ** 31],
                                    [-5, 3, -2 ** 31, -2 ** 31 + 2]])
def test_starts_that_run_backwards(ctx, starts, rank, rope):
    """Starts as far apart as 32 bits allow, in either direction: each is cut to the token rows, and a request that ends
    before it begins has none."""
    announce(f"paged attention: starts {starts}, rank {rank}")
    b = Batch([31, 40, 70], [3, 0, 0], 16, page=16, rank=rank, rope=rope, seed=19).upload(ctx)
    b.dev["starts"].upload(np.array(starts, np.int32))
    b.call(ctx)
    ctx.synchronize()
    b.check(b.dev["out"].download(), [0])


def test_as_many_requests_as_a_step_takes(ctx):
    """2^31 - 2 requests, the last with one token: its output is the one latent that it sees, to its bits."""
    announce("paged attention: 2^31 - 2 requests")
    requests, heads = 2 ** 31 - 2, 2
    dev = {"table": ctx.empty(requests, np.int32), "lengths": ctx.empty(requests, np.int32),
           "starts": ctx.empty(requests + 1, np.int32)}
    for b in dev.values():
        b.zero()
    for at in (dev["lengths"].ptr + 4 * (requests - 1), dev["starts"].ptr + 4 * requests):
        one = np.ones(1, np.int32)
        ctx._check(ctx.lib.lm_copy_h2d(ctx.handle, C.c_void_p(at), one.ctypes.data, 4))
    pool = encode(np.random.default_rng(23).normal(size=(1, 16, 576)), lm.DT_F16)
    dev |= {"q": ctx.to_device(np.zeros((1, heads, 576), np.uint16)), "pool": ctx.to_device(pool),
            "out": ctx.to_device(np.full((2, heads, 512), 0x1234, np.uint16))}
    step = lm.PagedStep(requests=requests, tokens=1, pages=1, page_size=16, table_width=1, max_added=1)
    for k in ("table", "lengths", "starts"):
        setattr(step, k, dev[k].ptr)
    ctx.paged_attention(step, dev["q"], dev["pool"], heads, SCALE, dev["out"])
    got = dev["out"].download()
    for b in dev.values():
        b.free()
    assert (got[0] == pool[0, 0, :512]).all() and (got[1] == 0x1234).all()
