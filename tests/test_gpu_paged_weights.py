"""The softmax weights of lm_paged_attention: what their 16 bits may cost, held to bounds that leave out what the
arithmetic does exactly.

Queries and keys lie on a grid on which their products add up exactly in 32 bits, so scores carry no rounding but those
of their scale and of the exponent's one step: 8 roundings of 2^-24 of the largest score, 2^-22 with the exponential.
Weights w_j round to 16 bits, relative `unit`, or in fp16 by half a step of 2^-24 where the row's largest is 2^5 at
least: 2^-30 of it.  Their total is that of the rounded ones, so a weight's error moves an output by its distance from
that output's value: sum_j |error_j| |c_j - out| / total.  Sums of 32 bits take one rounding a key tile, 300 for the
parts of a cut row and 64 within a tile.  The output rounds once, by half of its own step."""
import numpy as np
import pytest

import litemind_amd as lm
from conftest import announce
from litemind_amd import workload as wl
from test_gpu_paged_attention import SCALE, UNIT, Batch, decode, encode

pytestmark = pytest.mark.gpu
BITS = {lm.DT_F16: 10, lm.DT_BF16: 7}
RANK, WIDTH = 512, 576
DTYPES = [lm.DT_F16, lm.DT_BF16]


@pytest.fixture(scope="module")
def ctx():
    c = lm.Context(wl.V2_LITE.moe_config(num_layers=1))
    yield c
    c.close()


def half_step(v, dtype):
    """Half the distance between 16-bit numbers around |v|."""
    v = np.abs(v)
    low = -14 if dtype == lm.DT_F16 else -126
    return 2.0 ** (np.floor(np.log2(np.maximum(v, 2.0 ** low))) - BITS[dtype] - 1)


def lost(dtype):
    return 2.0 ** -30 if dtype == lm.DT_F16 else 0.0


def other(scores, keys):
    return 8 * 2.0 ** -24 * np.abs(scores).max() + 2.0 ** -22 + (-(-keys // 32) + 364) * 2.0 ** -24


def over_pages(pool, tables, lengths, starts, q, dtype, scale, pages):
    """A Batch over pages that its requests may share."""
    b = Batch.__new__(Batch)
    b.pool, b.table, b.lengths, b.starts, b.q = pool, tables, lengths, starts, q
    b.tokens, b.heads, b.rank, b.rope, b.dtype, b.scale = q.shape[0], q.shape[1], RANK, WIDTH - RANK, dtype, scale
    b.R, b.pages, b.page, b.width, b.added = len(lengths), pages, pool.shape[1], tables.shape[1], list(np.diff(starts))
    return b


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("requests,added", [(520, 1), (260, 9)])
@pytest.mark.parametrize("depth", [4.0, 14.3, 18.7, 22.3, 24.6, 28.6])
def test_a_first_key_above_a_long_tail(ctx, depth, requests, added, dtype):
    """The first of 65536 keys outweighs each of the others by 2^depth and has a latent of zeros, in blocks that one
    workgroup runs whole: what the others' weights lose shows in full."""
    announce(f"paged attention: a first key 2^{depth} above 65535 others, {requests} x {added} tokens, dtype {dtype}")
    keys, page, heads = 65536, 1024, 2
    scale = float(np.float32(depth * np.log(2.0) / 32.0))
    value = (np.arange(RANK) % 9 - 4) / 4.0
    rows = np.zeros((2, page, WIDTH))
    rows[:, :, :RANK] = value
    rows[0, 0, :RANK], rows[0, 0, RANK] = 0.0, 4.0
    table = np.ones((requests, keys // page), np.int32)
    table[:, 0] = 0
    q = np.zeros((requests * added, heads, WIDTH))
    q[..., RANK] = 8.0
    b = over_pages(encode(rows, dtype), table, np.full(requests, keys, np.int32),
                   np.arange(requests + 1, dtype=np.int32) * added, encode(q, dtype), dtype, scale, 2).upload(ctx)
    b.call(ctx)
    got = decode(b.dev["out"].download()[:-1], dtype).reshape(requests, added, heads, RANK)
    e = np.exp(-32.0 * scale)
    for i in range(added):
        tail = keys - added + i
        total = 1.0 + tail * e
        p = tail * e / total
        want = p * value
        bound = np.abs(value) * (tail * max(UNIT[dtype] * e, lost(dtype)) / total + 2 * other(np.array([32.0 * scale]), keys) * p)
        bound = bound + half_step(np.abs(want) + bound, dtype)
        off = np.abs(got[:, i] - want)
        assert (off <= bound).all(), f"token {i}: {got[0, i, 0, 0]:.6g}, not {want[0]:.6g}"


def grid(rng, shape, most):
    return rng.integers(-most, most + 1, shape) * 0.25


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,cached,added", [(16, [1, 33, 300, 1000, 64], [1, 1, 1, 1, 1]), (128, [500, 40], [1, 1]),
                                                (16, [700, 0, 31], [40, 70, 9])])
@pytest.mark.parametrize("most", [4, 24])
def test_rows_of_few_keys_that_count(ctx, heads, cached, added, dtype, most):
    """Scores so far apart that one or a few keys make up a row: their weights' rounding cancels against the total's."""
    announce(f"paged attention: peaked rows, {heads} heads, {added} after {cached}, queries up to {most / 4}, dtype {dtype}")
    rng = np.random.default_rng(heads + most + len(cached))
    b = Batch(cached, added, heads, dtype=dtype, page=32, seed=5)
    b.q = encode(grid(rng, b.q.shape, most), dtype)
    for r, n in enumerate(b.lengths):
        rows = grid(rng, (n, WIDTH), 4)
        rows[:, :RANK] += (rows[:, :RANK] == 0)  # (values next to each other for the keys that count)
        b.rows[r] = encode(rows, dtype)
        for k in range(-(-int(n) // b.page)):
            part = b.rows[r][k * b.page:(k + 1) * b.page]
            b.pool[b.table[r, k], :len(part)] = part
    got = decode(b.run(ctx), dtype)
    unit = UNIT[dtype]
    for r in range(b.R):
        rows = decode(b.rows[r], dtype)
        for t in range(b.starts[r], b.starts[r + 1]):
            seen = rows[:cached[r] + t - b.starts[r] + 1]
            s = (decode(b.q[t], dtype) @ seen.T) * np.float64(np.float32(SCALE))
            e = np.exp(s - s.max(1, keepdims=True))
            total = e.sum(1, keepdims=True)
            want = (e / total) @ seen[:, :RANK]
            error = np.maximum(unit * e, lost(dtype)) / total
            bound = np.empty_like(want)
            for h in range(heads):
                bound[h] = error[h] @ np.abs(seen[:, :RANK] - want[h])
            bound += 2 * other(s, len(seen)) * ((e / total) @ np.abs(seen[:, :RANK]))
            bound += half_step(np.abs(want) + bound, dtype)
            off = np.abs(got[t] - want)
            assert (off <= bound).all(), f"request {r}, row {t}: {np.max(off / bound):.3g} of the bound"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,cached,added", [(16, [20001, 131071], [1, 1]), (128, [20001], [2]), (16, [8190, 30000], [11, 40]),
                                                (3, [100000], [70]), (1, [50000, 77, 12345], [1, 1, 1])])
def test_every_key_counts_once(ctx, heads, cached, added, dtype):
    """Queries of zeros weigh all keys alike, and a channel of the latents counts the keys of every 256th tile or place: a
    tile left out or taken twice changes a count by 1 in 16 at least, a key by 1 in 512, more than the output's rounding
    but for bf16 past 60000 keys."""
    announce(f"paged attention: counted keys, {heads} heads, {added} after {cached}, dtype {dtype}")
    page, R = 64, len(cached)
    lengths = np.array([c + a for c, a in zip(cached, added)], np.int32)
    held = [-(-int(n) // page) for n in lengths]
    starts = np.concatenate([[0], np.cumsum(added)]).astype(np.int32)
    order = np.random.default_rng(7).permutation(sum(held)).astype(np.int32)
    table, at = np.full((R, max(held)), -1, np.int32), 0
    pool = np.zeros((sum(held), page, WIDTH), np.uint16)
    one = encode(np.ones(1), dtype)[0]
    for r, n in enumerate(lengths):
        table[r, :held[r]] = order[at:at + held[r]]
        at += held[r]
        j = np.arange(held[r] * page)
        rows = np.zeros((held[r] * page, WIDTH), np.uint16)
        rows[j, j // 32 % 256] = one
        rows[j, 256 + j % 256] = one
        pool[table[r, :held[r]]] = rows.reshape(held[r], page, WIDTH)
    q = np.zeros((int(starts[-1]), heads, WIDTH), np.uint16)
    b = over_pages(pool, table, lengths, starts, q, dtype, SCALE, len(pool)).upload(ctx)
    b.call(ctx)
    got = decode(b.dev["out"].download()[:-1], dtype)
    for r in range(R):
        for t in range(starts[r], starts[r + 1]):
            n = cached[r] + t - starts[r] + 1
            j = np.arange(n)
            want = np.concatenate([np.bincount(j // 32 % 256, minlength=256), np.bincount(j % 256, minlength=256)]) / n
            # equal weights of a power of two: sums are whole numbers, the quotient takes two roundings to 32 bits
            bound = want * 2.0 ** -22
            assert (np.abs(got[t] - want) <= bound + half_step(want + bound, dtype)).all(), f"request {r}, row {t}"


@pytest.mark.parametrize("rank,rope", [(512, 64), (64, 16)])
@pytest.mark.parametrize("size,scale", [(1e17, 0.0), (1e17, 1e-35), (1e17, -1e-35), (1e18, 5e-39), (1.0, 1e-45)])
def test_scales_of_any_size(ctx, size, scale, rank, rope):
    """Scores of large numbers and small scales: it is their product that counts, and a scale of 0 weighs all alike."""
    announce(f"paged attention: queries and keys of {size}, scale {scale}, rank {rank}")
    rng = np.random.default_rng(3)
    b = Batch([300, 0, 70], [1, 40, 3], 16, dtype=lm.DT_BF16, page=32, rank=rank, rope=rope, seed=4, scale=float(np.float32(scale)))
    b.q = encode(rng.normal(size=b.q.shape) * size, b.dtype)
    for r in range(b.R):
        b.rows[r] = encode(decode(b.rows[r], b.dtype) * size, b.dtype)
        for k in range(-(-int(b.lengths[r]) // b.page)):
            part = b.rows[r][k * b.page:(k + 1) * b.page]
            b.pool[b.table[r, k], :len(part)] = part
    b.check(b.run(ctx))


@pytest.mark.parametrize("heads,cached,added", [(16, [300, 40000], [1, 1]), (16, [100, 0], [40, 9])])
@pytest.mark.parametrize("power", [20, 44, 58])
def test_scores_of_any_size(ctx, power, heads, cached, added):
    """Scores up to 2^60, one step of which outweighs everything: a row is the mean of the keys of its largest score."""
    announce(f"paged attention: scores of 2^{power}, {heads} heads, {added} after {cached}")
    rng = np.random.default_rng(power)
    b = Batch(cached, added, heads, dtype=lm.DT_BF16, page=32, seed=6, scale=0.3)
    b.q = encode(grid(rng, b.q.shape, 12) * 2.0 ** (power // 2), b.dtype)
    for r, n in enumerate(b.lengths):
        rows = grid(rng, (n, WIDTH), 4)
        rows[:, RANK:] *= 2.0 ** (power - power // 2)  # (the rotary part alone is large, and alone counts)
        b.rows[r] = encode(rows, b.dtype)
        for k in range(-(-int(n) // b.page)):
            part = b.rows[r][k * b.page:(k + 1) * b.page]
            b.pool[b.table[r, k], :len(part)] = part
    q = decode(b.q, b.dtype)
    q[..., :RANK] = 0.0
    b.q = encode(q, b.dtype)
    got = decode(b.run(ctx), b.dtype)
    for r in range(b.R):
        rows = decode(b.rows[r], b.dtype)
        for t in range(b.starts[r], b.starts[r + 1]):
            seen = rows[:cached[r] + t - b.starts[r] + 1]
            s = q[t] @ seen.T
            first = (s == s.max(1, keepdims=True)).astype(np.float64)
            want = (first / first.sum(1, keepdims=True)) @ seen[:, :RANK]
            # equal weights: sums of a few values in 32 bits, and the quotient
            bound = 2.0 ** -20 * ((first / first.sum(1, keepdims=True)) @ np.abs(seen[:, :RANK]))
            off = np.abs(got[t] - want)
            assert (off <= bound + half_step(np.abs(want) + bound, b.dtype)).all(), f"request {r}, row {t}"


@pytest.mark.parametrize("heads", [16, 40])
@pytest.mark.parametrize("size", [1e3, 1e15, 1e17, 1e18])
def test_far_negative_scores_after_infinite_ones(ctx, size, heads):
    """Two tiles of scores of -infinity, then equal ones down to -2e36: those alone have weight."""
    announce(f"paged attention: 64 scores of -infinity, then -2 {size}^2, {heads} heads")
    rng = np.random.default_rng(9)
    b = Batch([140], [2], heads, dtype=lm.DT_BF16, page=16, seed=9, scale=1.0)
    rows = grid(rng, (142, WIDTH), 4)
    rows[:, RANK:] = 0.0
    rows[:64, RANK] = -np.inf
    rows[64:, RANK + 1] = -2.0 * size
    q = np.zeros(b.q.shape)
    q[..., RANK], q[..., RANK + 1] = 1.0, size
    b.q, b.rows[0] = encode(q, b.dtype), encode(rows, b.dtype)
    for k in range(9):
        part = b.rows[0][k * 16:(k + 1) * 16]
        b.pool[b.table[0, k], :len(part)] = part
    got = decode(b.run(ctx), b.dtype)[:2]
    for i in range(2):
        want = rows[64:141 + i, :RANK].mean(0)
        bound = 2.0 ** -20 * np.abs(rows[64:141 + i, :RANK]).mean(0)
        assert (np.abs(got[i] - want) <= bound + half_step(np.abs(want) + bound, b.dtype)).all()


@pytest.mark.parametrize("heads", [16, 40])
@pytest.mark.parametrize("cached,at", [(0, 0), (3, 1), (6, 6), (40, 35), (100, 99)])
def test_latents_near_the_end_of_the_range(ctx, cached, at, heads):
    """BF16 latents of up to 3e37, one of which outweighs the others by 2^9.5: sums of weights up to 1 stay in 32 bits."""
    announce(f"paged attention: latents of 3e37, {heads} heads, one token after {cached}")
    rng = np.random.default_rng(cached)
    b = Batch([cached], [1], heads, dtype=lm.DT_BF16, page=128, seed=10, scale=float(np.float32(9.5 * np.log(2.0))))
    rows = grid(rng, (cached + 1, WIDTH), 4)
    rows[:, :RANK] *= 3e37
    rows[:, RANK] = np.arange(cached + 1) == at
    q = np.zeros(b.q.shape)
    q[..., RANK] = 1.0
    b.q, b.rows[0] = encode(q, b.dtype), encode(rows, b.dtype)
    b.pool[b.table[0, 0], :cached + 1] = b.rows[0]
    b.check(b.run(ctx))
