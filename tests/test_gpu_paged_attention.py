"""lm_paged_attention on the GPU against the 64-bit restatement, within what its roundings allow element by element."""
import ctypes as C
import random

import numpy as np
import pytest

import litemind_amd as lm
import serving_ref as ref
from conftest import announce
from litemind_amd import workload as wl

pytestmark = pytest.mark.gpu
SCALE = 0.1147213867929261
UNIT = {lm.DT_F16: 2.0 ** -11, lm.DT_BF16: 2.0 ** -8}


@pytest.fixture(scope="module")
def ctx():
    c = lm.Context(wl.V2_LITE.moe_config(num_layers=1))
    yield c
    c.close()


def encode(x, dtype):
    """Rounded to the type, as 16-bit words."""
    x = np.ascontiguousarray(x, np.float32)
    if dtype == lm.DT_F16:
        return x.astype(np.float16).view(np.uint16)
    b = x.view(np.uint32).astype(np.uint64)
    b = np.where(np.isnan(x), 0x7fc00000, b + 0x7fff + ((b >> 16) & 1))
    return (b >> 16).astype(np.uint16)


def decode(w, dtype):
    if dtype == lm.DT_F16:
        return w.view(np.float16).astype(np.float64)
    return (w.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


class Batch:
    """Requests of given cached and new tokens over a pool whose other pages hold NaN."""

    def __init__(self, cached, added, heads, page=64, dtype=lm.DT_F16, rank=512, rope=64, seed=0, pad=0, spread=0.7,
                 scale=SCALE):
        rng = np.random.default_rng(seed)
        self.cached, self.added, self.heads, self.page, self.dtype = cached, added, heads, page, dtype
        self.rank, self.rope, self.scale, self.R = rank, rope, scale, len(cached)
        self.lengths = np.array([c + a for c, a in zip(cached, added)], np.int32)
        self.starts = np.concatenate([[0], np.cumsum(added)]).astype(np.int32)
        self.tokens = int(self.starts[-1]) + pad
        held = [ref.pages_of(n, page) for n in self.lengths]
        self.width, self.pages = max(held) + 1, sum(held) + 3
        order = rng.permutation(self.pages).astype(np.int32)
        self.table = np.full((self.R, self.width), -1, np.int32)
        at = 0
        for r, h in enumerate(held):
            self.table[r, :h] = order[at:at + h]
            at += h
        width = rank + rope
        self.pool = encode(np.full((self.pages, page, width), np.nan), dtype)
        self.rows = []
        for r, n in enumerate(self.lengths):
            words = encode(rng.normal(size=(n, width)), dtype)
            self.rows.append(words)
            for k in range(held[r]):
                part = words[k * page:(k + 1) * page]
                self.pool[self.table[r, k], :len(part)] = part
        self.q = encode(rng.normal(size=(self.tokens, heads, width)) * spread, dtype)

    def upload(self, ctx):
        self.dev = {"table": ctx.to_device(self.table), "lengths": ctx.to_device(self.lengths),
                    "starts": ctx.to_device(self.starts), "q": ctx.to_device(self.q), "pool": ctx.to_device(self.pool),
                    "out": ctx.to_device(np.full((self.tokens + 1, self.heads, self.rank), 0x1234, np.uint16))}
        self.step = lm.PagedStep(requests=self.R, tokens=self.tokens, pages=self.pages, page_size=self.page,
                                 table_width=self.width, max_added=max(self.added))
        for k in ("table", "lengths", "starts"):
            setattr(self.step, k, self.dev[k].ptr)
        return self

    def call(self, ctx):
        ctx.paged_attention(self.step, self.dev["q"], self.dev["pool"], self.heads, self.scale, self.dev["out"],
                            dtype=self.dtype, rank=self.rank, rope=self.rope)

    def run(self, ctx):
        self.upload(ctx)
        self.call(ctx)
        return self.dev["out"].download()

    def check(self, got, requests=None):
        used = int(self.starts[-1])
        assert (got[used:] == 0x1234).all()  # rows behind the last request's
        value = decode(got, self.dtype)
        for r in requests if requests is not None else range(self.R):
            b, e = self.starts[r], self.starts[r + 1]
            if b == e:
                continue
            want, bound = ref.attention(decode(self.q[b:e], self.dtype), decode(self.rows[r], self.dtype),
                                        self.cached[r], self.scale, self.rank, UNIT[self.dtype])
            off = np.abs(value[b:e] - want)
            assert np.isfinite(value[b:e]).all(), f"request {r}"
            assert (off <= bound).all(), f"request {r}: {np.max(off / bound):.3g} of the bound"


EDGES = [0, 1, 2, 14, 15, 16, 17, 30, 31, 32, 33, 62, 63, 64, 65, 95, 127, 128, 129, 255, 256, 257, 511, 513]


@pytest.mark.parametrize("dtype", [lm.DT_F16, lm.DT_BF16])
@pytest.mark.parametrize("heads", [1, 3, 8, 16, 17, 32, 40, 128, 130])
def test_one_token_at_every_edge(ctx, heads, dtype):
    announce(f"paged attention: one token each, {heads} heads, dtype {dtype}")
    b = Batch(EDGES, [1] * len(EDGES), heads, dtype=dtype, page=32, seed=heads, pad=2)
    b.check(b.run(ctx))


@pytest.mark.parametrize("page", [16, 48, 64, 128, 4096])
def test_pages(ctx, page):
    announce(f"paged attention: pages of {page}")
    b = Batch([0, 40, 333, 100, 1, 700], [1, 3, 1, 70, 2, 1], 16, page=page, seed=page)
    b.check(b.run(ctx))


@pytest.mark.parametrize("heads,added,cached", [
    (16, [1, 2, 3, 5, 7, 8, 9, 0, 33], [10, 31, 0, 64, 100, 5, 63, 200, 0]),
    (16, [129, 1, 64], [0, 500, 33]), (16, [300], [77]), (128, [1, 2, 17], [40, 0, 90]), (20, [40, 6, 7], [3, 66, 0]),
    (1, [140, 1, 16], [12, 300, 0]), (5, [51, 26, 1], [0, 17, 90]), (64, [3, 2, 1], [31, 32, 33]), (130, [2, 3], [5, 64])])
@pytest.mark.parametrize("dtype", [lm.DT_F16, lm.DT_BF16])
def test_chunks(ctx, heads, added, cached, dtype):
    announce(f"paged attention: chunks {added} after {cached}, {heads} heads, dtype {dtype}")
    b = Batch(cached, added, heads, dtype=dtype, page=16, seed=len(added) + heads, pad=3)
    b.check(b.run(ctx))


@pytest.mark.parametrize("rank,rope", [(8, 0), (16, 8), (32, 64), (64, 64), (256, 32), (504, 64), (512, 0), (512, 128),
                                       (1024, 256)])
def test_widths(ctx, rank, rope):
    announce(f"paged attention: rank {rank}, rope {rope}")
    b = Batch([0, 40, 129], [1, 3, 2], 4, page=16, rank=rank, rope=rope, seed=rank)
    b.check(b.run(ctx))


@pytest.mark.parametrize("spread,scale", [(30.0, SCALE), (0.0, SCALE), (0.7, 0.0), (0.7, -0.3), (2000.0, 1e-5)])
def test_scores(ctx, spread, scale):
    """Sharp, flat, zero-scaled and negatively scaled scores."""
    announce(f"paged attention: spread {spread}, scale {scale}")
    b = Batch([300, 64, 0, 1000], [1, 9, 40, 1], 16, seed=3, spread=spread, scale=scale)
    b.check(b.run(ctx))


def test_rising_scores(ctx):
    """Every later key scores higher than all before: the running maximum moves in every tile."""
    announce("paged attention: rising scores")
    b = Batch([600, 130], [1, 20], 16, seed=4)
    for r in range(2):
        words = decode(b.rows[r], b.dtype) * 0.05
        words[:, 0] = np.linspace(0.0, 60.0, len(words))
        b.rows[r] = encode(words, b.dtype)
        for k in range(ref.pages_of(len(words), b.page)):
            part = b.rows[r][k * b.page:(k + 1) * b.page]
            b.pool[b.table[r, k], :len(part)] = part
    q = decode(b.q, b.dtype) * 0.2
    q[..., 0] = 8.0
    b.q = encode(q, b.dtype)
    b.check(b.run(ctx))


@pytest.mark.parametrize("heads", [1, 16, 128])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_what_a_token_does_not_see(ctx, bad, heads):
    """NaN and infinities of a later token of the chunk reach that token and those after it, and none before."""
    announce(f"paged attention: {bad} in a later token, {heads} heads")
    b = Batch([20, 100, 3], [40, 12, 1], heads, page=16, seed=6)
    place = 20 + 25
    b.rows[0] = b.rows[0].copy()
    b.pool[b.table[0, place // 16], place % 16, ::3] = encode(np.full(192, bad), b.dtype)
    got = b.run(ctx)
    b.check(got, [1, 2])
    value = decode(got, b.dtype)
    want, bound = ref.attention(decode(b.q[:25], b.dtype), decode(b.rows[0], b.dtype), 20, b.scale, b.rank, UNIT[b.dtype])
    assert (np.abs(value[:25] - want) <= bound).all()
    assert np.isnan(value[25:40]).any(axis=2).all()


def test_infinite_scores_weigh_nothing(ctx):
    """A key whose score is -infinity (an infinite rotary channel) has no weight."""
    announce("paged attention: a key of score -infinity")
    b = Batch([70], [1], 16, page=16, seed=8)
    b.pool[b.table[0, 2], 5, 512] = encode(np.array([-np.inf]), b.dtype)[0]
    q = decode(b.q, b.dtype)
    q[..., 512] = np.abs(q[..., 512]) + 0.1
    b.q = encode(q, b.dtype)
    got = b.run(ctx)
    rows = decode(b.rows[0], b.dtype)
    want, bound = ref.attention(decode(b.q, b.dtype), np.delete(rows, 37, 0), 69, b.scale, b.rank, UNIT[b.dtype])
    assert (np.abs(decode(got, b.dtype)[:1] - want) <= bound).all()


def test_long_cache(ctx):
    announce("paged attention: 20000 keys, one and eleven tokens")
    b = Batch([20001, 8190], [1, 11], 16, page=128, seed=11)
    b.check(b.run(ctx))


def test_many_requests(ctx):
    announce("paged attention: 300 requests, some without tokens")
    rng = random.Random(3)
    cached = [rng.randint(0, 200) for _ in range(300)]
    b = Batch(cached, [rng.choice([0, 1, 1, 1]) for _ in cached], 16, page=16, seed=12, pad=5)
    b.check(b.run(ctx))
    cached = [rng.randint(0, 90) for _ in range(1500)]
    b = Batch(cached, [rng.choice([0, 1]) for _ in cached], 2, page=16, seed=13)
    b.check(b.run(ctx))


def test_no_tokens_at_all(ctx):
    announce("paged attention: requests without new tokens")
    b = Batch([5, 70], [0, 0], 16, pad=4, seed=1)
    got = b.run(ctx)
    assert (got == 0x1234).all()


def test_same_bits_again_and_between_others(ctx):
    """No atomics and no leftovers: the same call gives the same bits, whatever ran before."""
    announce("paged attention: repeated calls")
    one = Batch([3000, 500, 10], [1, 1, 1], 16, seed=14).upload(ctx)
    two = Batch([100, 900], [200, 33], 16, seed=15).upload(ctx)
    first = []
    for b in (one, two):
        b.call(ctx)
        first.append(b.dev["out"].download())
        b.check(first[-1])
    for _ in range(5):
        for b in (one, two):
            b.call(ctx)
        for b, f in zip((one, two), first):
            assert np.array_equal(b.dev["out"].download(), f)


def test_request_alone_and_in_a_batch(ctx):
    """A request's rows do not depend on its neighbours beyond the order of the sums."""
    announce("paged attention: a request alone and in a batch")
    b = Batch([1000, 77, 4000, 0], [1, 1, 1, 1], 16, seed=16)
    b.check(b.run(ctx))
    alone = Batch([1000], [1], 16, seed=16)
    alone.check(alone.run(ctx))


@pytest.mark.parametrize("page_id", [-1, 10 ** 6, 2 ** 31 - 1, -2 ** 31])
def test_page_ids_outside_the_pool(ctx, page_id):
    announce(f"paged attention: page id {page_id}")
    b = Batch([100, 70], [1, 1], 16, page=16, seed=17)
    b.table[0, 3] = page_id
    b.upload(ctx)
    b.call(ctx)
    with pytest.raises(lm.LmError) as e:
        ctx.synchronize()
    assert e.value.status == -5
    ctx.synchronize()  # reported once
    b.check(b.dev["out"].download(), [1])


def test_lengths_beyond_the_arrays(ctx):
    """Starts past the token rows and lengths past the table's row are cut to the arrays."""
    announce("paged attention: starts and lengths past their arrays")
    b = Batch([31, 30], [1, 2], 16, page=16, seed=18)
    b.upload(ctx)
    b.dev["starts"].upload(np.array([0, 1, 1000], np.int32))
    b.dev["lengths"].upload(np.array([32, 2 ** 31 - 1], np.int32))
    b.call(ctx)
    with pytest.raises(lm.LmError) as e:  # the last column of its row names no page
        ctx.synchronize()
    assert e.value.status == -5
    got = b.dev["out"].download()
    b.check(got, [0])


@pytest.mark.parametrize("requests,heads,rank,rope", [(70000, 1, 512, 64), (131072, 9, 8, 0)])
def test_very_many_requests(ctx, requests, heads, rank, rope):
    """Single tokens of requests that share one page: each row is the one latent that it sees, to its bits."""
    announce(f"paged attention: {requests} requests, {heads} heads, rank {rank}")
    rng = np.random.default_rng(20)
    width = rank + rope
    pool = encode(rng.normal(size=(1, 16, width)), lm.DT_F16)
    dev = {"table": ctx.to_device(np.zeros((requests, 1), np.int32)), "lengths": ctx.to_device(np.ones(requests, np.int32)),
           "starts": ctx.to_device(np.arange(requests + 1, dtype=np.int32)),
           "q": ctx.empty((requests, heads, width), np.uint16).zero(), "pool": ctx.to_device(pool),
           "out": ctx.empty((requests, heads, rank), np.uint16).zero()}
    step = lm.PagedStep(requests=requests, tokens=requests, pages=1, page_size=16, table_width=1, max_added=1)
    for k in ("table", "lengths", "starts"):
        setattr(step, k, dev[k].ptr)
    ctx.paged_attention(step, dev["q"], dev["pool"], heads, SCALE, dev["out"], rank=rank, rope=rope)
    out = dev["out"].download()
    for b in dev.values():
        b.free()
    assert (out == pool[0, 0, :rank]).all()


def put(ctx, ptr, host):
    host = np.ascontiguousarray(host)
    ctx._check(ctx.lib.lm_copy_h2d(ctx.handle, C.c_void_p(ptr), host.ctypes.data, host.nbytes))


def get(ctx, ptr, like):
    out = np.empty_like(like)
    ctx._check(ctx.lib.lm_copy_d2h(ctx.handle, out.ctypes.data, C.c_void_p(ptr), out.nbytes))
    return out


@pytest.mark.parametrize("rank,rope,added", [(512, 64, [1, 1, 1]), (512, 64, [1, 70, 3]), (64, 16, [1, 2, 1])])
def test_pages_past_four_gigabytes(ctx, rank, rope, added):
    announce(f"paged attention: pages past 4 GiB, rank {rank}, {added}")
    b = Batch([5000, 77, 300], added, 16, page=4096, rank=rank, rope=rope, seed=21)
    page_bytes = 2 * b.page * (rank + rope)
    base = (5 << 30) // page_bytes
    pool = ctx.empty((base + b.pages) * page_bytes // 2, np.uint16)
    b.table = np.where(b.table >= 0, b.table + base, -1).astype(np.int32)
    b.upload(ctx)
    put(ctx, pool.ptr + base * page_bytes, b.pool)
    b.step.pages = base + b.pages
    b.dev["pool"] = pool
    b.call(ctx)
    got = b.dev["out"].download()
    pool.free()
    b.check(got)


def test_rows_past_four_gigabytes(ctx):
    """Queries and outputs of 3.84 million rows: the last requests' rows are theirs."""
    announce("paged attention: query rows past 4 GiB")
    requests, heads, width = 30000, 128, 576
    rng = np.random.default_rng(22)
    pool, words = encode(rng.normal(size=(2, 16, width)), lm.DT_F16), heads * width
    table, lengths = np.zeros((requests, 1), np.int32), np.ones(requests, np.int32)
    table[-2:], lengths[-2:] = 1, 16
    dev = {"table": ctx.to_device(table), "lengths": ctx.to_device(lengths),
           "starts": ctx.to_device(np.arange(requests + 1, dtype=np.int32)),
           "q": ctx.empty((requests, heads, width), np.uint16).zero(), "pool": ctx.to_device(pool),
           "out": ctx.empty((requests, heads, 512), np.uint16).zero()}
    q = encode(rng.normal(size=(2, heads, width)) * 0.7, lm.DT_F16)
    put(ctx, dev["q"].ptr + 2 * (requests - 2) * words, q)
    step = lm.PagedStep(requests=requests, tokens=requests, pages=2, page_size=16, table_width=1, max_added=1)
    for k in ("table", "lengths", "starts"):
        setattr(step, k, dev[k].ptr)
    ctx.paged_attention(step, dev["q"], dev["pool"], heads, SCALE, dev["out"])
    tail = get(ctx, dev["out"].ptr + 2 * (requests - 40) * heads * 512, np.empty((40, heads, 512), np.uint16))
    for b in dev.values():
        b.free()
    assert (tail[:38] == pool[0, 0, :512]).all()
    for i in range(2):
        want, bound = ref.attention(decode(q[i:i + 1], lm.DT_F16), decode(pool[1], lm.DT_F16), 15, SCALE, 512, UNIT[lm.DT_F16])
        assert (np.abs(decode(tail[38 + i:39 + i], lm.DT_F16) - want) <= bound).all()
