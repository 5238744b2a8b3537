"""lm_sample on the GPU against the 64-bit restatement: the same tokens, and probabilities to single precision."""
import ctypes as C

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


def settings(rows):
    return np.array([tuple(r) for r in rows], lm.SAMPLING)


def run(ctx, logits, sets, u, stride=None):
    rows, vocab = logits.shape
    stride = stride or vocab
    wide = np.full((rows, stride), np.inf, np.float32)  # what lies between the rows is not read
    wide[:, :vocab] = logits
    token = ctx.to_device(np.full(rows + 1, -9, np.int32))
    chance = ctx.to_device(np.full(rows + 1, -9, np.float32))
    args = ctx.to_device(wide), rows, vocab, ctx.to_device(sets), ctx.to_device(np.asarray(u, np.float32)), token
    ctx.sample(*args, probability=chance, row_stride=stride)
    t, p = token.download(), chance.download()
    assert t[-1] == -9 and p[-1] == -9
    ctx.sample(*args, row_stride=stride)  # without probabilities
    assert np.array_equal(token.download(), t)
    return t[:-1], p[:-1]


def check(t, p, logits, sets, u):
    """Equal tokens wherever u and the cuts lie further from a border than 64-bit sums of the row can be off: n
    roundings of 2^-53 and the operator's units of 2^-46 (fewer bits for more than 2^17 tokens)."""
    doubtful = 0
    for i in range(len(t)):
        want, chance, near = ref.sample(logits[i], *sets[i], u[i])
        n = logits.shape[1]
        if near < n * 2.0 ** -50 + 2.0 ** -46 * n:
            doubtful += 1
            continue
        assert t[i] == want, f"row {i}: {t[i]}, not {want} ({sets[i]}, u {u[i]})"
        # the chosen e in units of 2^-46 (2^-39 at least), one rounding to 32 bits
        assert abs(p[i] - chance) <= 2.0 ** -24 * chance + 2.0 ** -38, f"row {i}"
    assert doubtful <= max(1, len(t) // 50)


def rows_of(rng, rows, vocab, grid=False, spread=2.2):
    x = rng.normal(size=(rows, vocab)).astype(np.float32) * np.float32(spread)
    for r in range(rows):
        at = rng.integers(0, vocab, 30)
        x[r, at] += np.abs(rng.normal(size=30)).astype(np.float32) * 4
    if grid:
        x = (x.view(np.uint32) & 0xffff0000).view(np.float32)
    return np.ascontiguousarray(x)


def any_settings(rng, rows):
    return settings([(rng.choice([0.0, 0.3, 0.7, 1.0, 1.7]), rng.choice([0, 1, 2, 20, 50, 400, 10 ** 6]),
                      rng.choice([1.0, 0.999, 0.95, 0.9, 0.5, 0.01]), rng.choice([0.0, 0.001, 0.02, 0.1, 0.9]))
                     for _ in range(rows)])


@pytest.mark.parametrize("vocab", [1, 2, 3, 63, 64, 65, 257, 1000, 1023, 1024, 1025, 4097, 32003, 102400, 131073, 200001])
@pytest.mark.parametrize("grid", [False, True])
def test_mixed_settings(ctx, vocab, grid):
    announce(f"sample: vocabulary {vocab}, grid {grid}")
    rng = np.random.default_rng(vocab)
    rows = 24 if vocab < 50000 else 8
    x, sets, u = rows_of(rng, rows, vocab, grid), any_settings(rng, rows), rng.random(rows).astype(np.float32)
    check(*run(ctx, x, sets, u), x, sets, u)


@pytest.mark.parametrize("kind", ["temperature", "top_k", "top_p", "min_p"])
def test_one_filter(ctx, kind):
    announce(f"sample: {kind} alone")
    rng = np.random.default_rng(5)
    rows, vocab = 40, 20011
    x, u = rows_of(rng, rows, vocab, True), rng.random(rows).astype(np.float32)
    base = (0.8, 0, 1.0, 0.0)
    sets = settings([(base[0], int(rng.integers(1, 3000)) if kind == "top_k" else 0,
                      rng.random() if kind == "top_p" else 1.0, rng.random() ** 4 if kind == "min_p" else 0.0)
                     for _ in range(rows)])
    check(*run(ctx, x, sets, u), x, sets, u)


@pytest.mark.parametrize("rows", [1, 2, 7, 100, 300, 1100])
def test_row_counts_and_strides(ctx, rows):
    announce(f"sample: {rows} rows, a stride past the vocabulary")
    rng = np.random.default_rng(rows)
    x, sets, u = rows_of(rng, rows, 523), any_settings(rng, rows), rng.random(rows).astype(np.float32)
    check(*run(ctx, x, sets, u, stride=531), x, sets, u)


@pytest.mark.parametrize("vocab", [5, 5000, 150000])
def test_ties(ctx, vocab):
    """All logits equal, and a few levels: cuts fall inside runs of equal logits, lowest index first."""
    announce(f"sample: ties, vocabulary {vocab}")
    rng = np.random.default_rng(2)
    flat = np.zeros((6, vocab), np.float32)
    few = rng.integers(0, 3, size=(6, vocab)).astype(np.float32)
    signed = np.where(rng.random((2, vocab)) < 0.5, np.float32(-0.0), np.float32(0.0))
    x = np.concatenate([flat, few, signed])
    sets = settings([(1.0, 0, 1.0, 0.0), (1.0, 3, 1.0, 0.0), (1.0, 0, 0.3, 0.0), (1.0, 4, 0.6, 0.0), (1.0, 0, 1.0, 0.9),
                     (1.0, vocab // 2 + 1, 0.7, 0.5)] * 2 + [(1.0, 2, 1.0, 0.0), (0.0, 0, 1.0, 0.0)])
    u = rng.random(len(x)).astype(np.float32)
    check(*run(ctx, x, sets, u), x, sets, u)


def test_borders_of_the_settings(ctx):
    announce("sample: settings at and past their borders")
    rng = np.random.default_rng(3)
    nan, inf = np.nan, np.inf
    sets = settings([(-1.0, 0, 1.0, 0.0), (nan, 0, 1.0, 0.0), (0.0, 5, 0.5, 0.5), (1.0, -3, 1.0, 0.0),
                     (1.0, 2 ** 31 - 1, 1.0, 0.0), (1.0, 0, 0.0, 0.0), (1.0, 0, -1.0, 0.0), (1.0, 0, nan, 0.0),
                     (1.0, 0, 2.0, 0.0), (1.0, 0, 1.0, nan), (1.0, 0, 1.0, -1.0), (1.0, 0, 1.0, 1.0),
                     (1.0, 0, 1.0, 1.5), (1.0, 0, 1e-30, 0.0), (1e-30, 0, 1.0, 0.0), (1e30, 0, 1.0, 0.0),
                     (inf, 0, 1.0, 0.0), (1.0, 1, 1e-9, 1.0)])
    x = rows_of(rng, len(sets), 3001)
    u = rng.random(len(sets)).astype(np.float32)
    check(*run(ctx, x, sets, u), x, sets, u)


def test_random_numbers_at_their_ends(ctx):
    announce("sample: random numbers at their ends")
    rng = np.random.default_rng(4)
    u = np.array([0.0, -0.0, 1.0 - 2.0 ** -24, 1.0, 5.0, -1.0, np.nan, 2.0 ** -149], np.float32)
    x = rows_of(rng, len(u), 777)
    sets = settings([(1.0, 0, 1.0, 0.0)] * len(u))
    t, _ = run(ctx, x, sets, u)
    first = np.zeros(len(u), int)
    last = np.full(len(u), 776)
    for i in (0, 1, 5, 6, 7):
        assert t[i] == first[i]
    for i in (3, 4):
        assert t[i] == last[i]


def test_masked_rows(ctx):
    """-infinity, NaN, +infinity, and rows that leave nothing."""
    announce("sample: masked rows")
    rng = np.random.default_rng(6)
    x = rows_of(rng, 9, 2000)
    x[0] = -np.inf
    x[1] = np.nan
    x[2, :] = -np.inf
    x[2, 1999] = -1e30
    x[3, ::2] = np.nan
    x[4, 7] = x[4, 1500] = np.inf
    x[5, :1990] = -np.inf
    x[6, :] = -np.finfo(np.float32).max
    x[7, 0] = np.nan
    x[8, 5:] = np.nan
    for sets in (settings([(1.0, 0, 1.0, 0.0)] * 9), settings([(0.7, 50, 0.9, 0.01)] * 9), settings([(0.0, 0, 1.0, 0.0)] * 9)):
        u = rng.random(9).astype(np.float32)
        t, p = run(ctx, x, sets, u)
        assert t[0] == -1 and t[1] == -1 and p[0] == 0 and p[1] == 0
        check(t, p, x, sets, u)


def test_as_often_as_their_probability(ctx):
    """Tokens come as often as the definition says: exactly, over an even grid of random numbers."""
    announce("sample: an even grid of random numbers")
    row = np.array([0.0, 1.0, 2.0, -1.0, 0.5], np.float32)
    rows = 4096
    u = (np.arange(rows) + 0.5).astype(np.float32) / rows
    t, _ = run(ctx, np.tile(row, (rows, 1)), settings([(1.3, 0, 1.0, 0.0)] * rows), u)
    e = np.exp(row.astype(np.float64) / np.float32(1.3))
    edges = np.cumsum(e) / e.sum()
    assert np.array_equal(t, np.searchsorted(edges, u.astype(np.float64), side="right"))


def test_greedy_is_the_heads_choice(ctx):
    announce("sample: greedy rows")
    rng = np.random.default_rng(7)
    x = rows_of(rng, 33, 5003, True)
    t, p = run(ctx, x, settings([(0.0, 0, 1.0, 0.0)] * 33), rng.random(33).astype(np.float32))
    assert np.array_equal(t, x.argmax(1)) and (p == 1).all()


@pytest.mark.parametrize("vocab", [1000, 6007, 20011])
def test_ranges(ctx, vocab):
    """Logits over the whole range of the type or in its smallest steps, far outliers on either side, masked and not,
    under temperatures as far apart: the stretches that the kernel divides a row into have nothing to hold on to."""
    announce(f"sample: ranges, vocabulary {vocab}")
    rng = np.random.default_rng(vocab)
    big, tiny = np.finfo(np.float32).max, np.float32(1e-45)

    def normal(k=1.0):
        return rng.normal(size=vocab).astype(np.float32) * np.float32(k)

    def masked(x):
        y = x.copy()
        y[rng.random(vocab) < 0.5] = -np.inf
        return y

    def put(x, v):
        y = x.copy()
        y[rng.integers(0, vocab)] = v
        return y

    rows = [(rng.uniform(-1, 1, vocab).astype(np.float32) * big, 1e38), (rng.uniform(-1, 1, vocab).astype(np.float32) * big, 1.0),
            (rng.integers(0, 90, vocab).astype(np.float32) * tiny, 1.0), (rng.integers(0, 90, vocab).astype(np.float32) * tiny, 2e-44),
            (put(normal(), big), 1.0), (put(normal(), -big), 1.0), (put(normal(), big), 1e38), (normal() + np.float32(1e6), 1.0),
            (normal(200.0), 0.01), (normal(), 40.0), (normal(), 1e-3), (masked(normal()), 0.9), (masked(normal(1e-3)), 1.0),
            (normal() - np.float32(2e38), 1e37), (masked(put(normal(), np.inf)), 1.0), (normal(), np.inf),
            (np.full(vocab, -big, np.float32), 1.0), (put(normal(), np.inf), 1e38)]
    for top_k, top_p, min_p in ((0, 1.0, 0.0), (50, 1.0, 0.0), (0, 0.9, 0.0), (3000, 0.8, 0.0), (0, 1.0, 0.3), (700, 0.6, 0.01)):
        x = np.ascontiguousarray([r[0] for r in rows])
        sets = settings([(r[1], top_k, top_p, min_p) for r in rows])
        u = rng.random(len(rows)).astype(np.float32)
        t, p = run(ctx, x, sets, u)
        for i in range(len(rows)):
            want, chance, near = ref.sample(x[i], *sets[i], u[i])
            if near < vocab * 2.0 ** -45:
                continue
            assert t[i] == want, f"row {i}: {t[i]}, not {want} ({sets[i]}, u {u[i]})"
            assert abs(p[i] - chance) <= 2.0 ** -24 * chance + 2.0 ** -38


def test_more_rows_than_a_launch_takes(ctx):
    announce("sample: two million rows")
    rows = 2 ** 21 + 3
    x = np.zeros((rows, 2), np.float32)
    x[1::2, 1] = 1.0
    token = ctx.to_device(np.full(rows + 1, -9, np.int32))
    sets = np.zeros(rows, lm.SAMPLING)
    ctx.sample(ctx.to_device(x), rows, 2, ctx.to_device(sets), ctx.to_device(np.zeros(rows, np.float32)), token)
    t = token.download()
    assert t[-1] == -9 and (t[:-1] == np.arange(rows) % 2).all()


def test_rows_far_apart(ctx):
    """Rows 4 GiB apart."""
    announce("sample: rows 4 GiB apart")
    rng = np.random.default_rng(11)
    rows, vocab, stride = 3, 5003, 2 ** 30 + 1
    x, sets, u = rows_of(rng, rows, vocab), any_settings(rng, rows), rng.random(rows).astype(np.float32)
    wide, token = ctx.empty((rows - 1) * stride + vocab), ctx.empty(rows, np.int32)
    for r in range(rows):
        ctx._check(ctx.lib.lm_copy_h2d(ctx.handle, C.c_void_p(wide.ptr + 4 * r * stride), x[r].ctypes.data, x[r].nbytes))
    ctx.sample(wide, rows, vocab, ctx.to_device(sets), ctx.to_device(u), token, row_stride=stride)
    t = token.download()
    wide.free()
    for r in range(rows):
        want, _, near = ref.sample(x[r], *sets[r], u[r])
        assert near < vocab * 2.0 ** -45 or t[r] == want
