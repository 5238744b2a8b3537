"""What the serving operators refuse, and the plain restatements that the GPU tests compare with (no GPU calls: every
argument is checked before the context)."""
import ctypes as C

import numpy as np
import pytest

import litemind_amd as lm
import serving_ref as ref

SOME = 0x10000  # an address that is never followed


def step(**kw):
    s = lm.PagedStep(requests=3, tokens=5, pages=8, page_size=16, table_width=4, max_added=5)
    for name in ("cached", "added", "table", "ring", "queue_in", "queue_out", "lengths", "starts", "positions", "slots",
                 "info"):
        setattr(s, name, SOME)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def refused(status):
    lib = lm.load_library()
    assert status == -1
    return lib.lm_last_error().decode()


SIZES = [dict(requests=0), dict(requests=2 ** 31), dict(tokens=-1), dict(tokens=2 ** 31), dict(pages=0),
         dict(pages=2 ** 31), dict(pages=2 ** 62), dict(pages=2 ** 27, page_size=16), dict(page_size=0),
         dict(page_size=8), dict(page_size=24), dict(page_size=8192), dict(page_size=-16), dict(table_width=0),
         dict(table_width=2 ** 27), dict(max_added=-1), dict(reserved=1)]


@pytest.mark.parametrize("bad", SIZES, ids=str)
def test_sizes(bad):
    lib = lm.load_library()
    assert "null context" not in refused(lib.lm_page_plan(None, C.byref(step(**bad))))
    assert "null context" not in refused(lib.lm_paged_attention(None, C.byref(step(**bad)), SOME, SOME, lm.DT_F16, 16,
                                                                512, 64, 0.1, SOME * 65536))


@pytest.mark.parametrize("name", ["cached", "added", "table", "ring", "queue_in", "queue_out", "lengths", "starts",
                                  "positions", "slots", "info"])
@pytest.mark.parametrize("value", [None, SOME + 2])
def test_plan_arrays(name, value):
    lib = lm.load_library()
    message = refused(lib.lm_page_plan(None, C.byref(step(**{name: value}))))
    assert "null context" not in message


def test_good_arguments_reach_the_context():
    lib = lm.load_library()
    assert "null context" in refused(lib.lm_page_plan(None, C.byref(step())))
    assert "null context" in refused(lib.lm_page_plan(None, C.byref(step(tokens=0, positions=None, slots=None))))
    assert "null context" in refused(lib.lm_paged_attention(None, C.byref(step()), SOME, SOME * 16, lm.DT_BF16, 16, 512,
                                                            64, 0.1, SOME * 65536))
    assert "null context" in refused(lib.lm_sample(None, SOME, 3, 100, 100, SOME, SOME, SOME, None))
    assert "null step" in refused(lib.lm_page_plan(None, None))


@pytest.mark.parametrize("bad", [
    dict(q=None), dict(pool=None), dict(out=None), dict(q=SOME + 8), dict(pool=SOME + 8), dict(out=SOME * 65536 + 8),
    dict(dtype=lm.DT_F32), dict(dtype=0), dict(heads=0), dict(heads=2 ** 30), dict(rank=0), dict(rank=12),
    dict(rank=1032), dict(rope=-8), dict(rope=4), dict(rope=264), dict(scale=float("nan")), dict(scale=float("inf")),
    dict(out=SOME), dict(out=SOME * 16),
    dict(step=dict(table=None)), dict(step=dict(lengths=None)), dict(step=dict(starts=SOME + 1)),
    dict(step=dict(tokens=2 ** 20, page_size=16, pages=1, table_width=2 ** 26), heads=1023)], ids=str)
def test_attention_arguments(bad):
    lib = lm.load_library()
    a = dict(q=SOME, pool=SOME * 16, dtype=lm.DT_F16, heads=16, rank=512, rope=64, scale=0.1, out=SOME * 65536)
    s = step(**bad.pop("step", {}))
    a.update(bad)
    message = refused(lib.lm_paged_attention(None, C.byref(s), a["q"], a["pool"], a["dtype"], a["heads"], a["rank"],
                                             a["rope"], a["scale"], a["out"]))
    assert "null context" not in message


@pytest.mark.parametrize("bad", [dict(logits=None), dict(logits=SOME + 1), dict(rows=-1), dict(rows=2 ** 31),
                                 dict(vocab=0), dict(vocab=2 ** 24 + 1, stride=2 ** 25), dict(stride=99),
                                 dict(settings=None), dict(uniform=None), dict(token=None), dict(probability=SOME + 2)],
                         ids=str)
def test_sample_arguments(bad):
    lib = lm.load_library()
    a = dict(logits=SOME, rows=3, vocab=100, stride=100, settings=SOME, uniform=SOME, token=SOME, probability=SOME)
    a.update(bad)
    message = refused(lib.lm_sample(None, *a.values()))
    assert "null context" not in message


# ---- the restatements themselves ----

def test_plan_takes_and_gives_back():
    table = np.array([[4, 5, -1], [6, -1, -1], [7, 8, -1]], np.int32)
    ring = np.array([2, 9, -1, -1, -1, -1, -1, 0, 1, 3], np.int32)
    out = ref.plan([17, 16, 32], [14, -1, 17], table, ring, [7, 5], 16, 33, 20)
    assert out["table"].tolist() == [[4, 5, -1], [6, -1, -1], [7, 8, 0]] or out["info"][0] == 1
    out = ref.plan([17, 16, 30], [14, -1, 17], table, ring, [7, 5], 16, 33, 20)
    assert out["info"].tolist() == [0, 31, 1, 1] and out["queue"].tolist() == [8, 5]
    assert out["table"][2].tolist() == [7, 8, 0] and out["ring"][2] == 6
    assert out["starts"].tolist() == [0, 14, 14, 31] and out["lengths"].tolist() == [31, 0, 47]
    assert out["slots"][:3].tolist() == [5 * 16 + 1, 5 * 16 + 2, 5 * 16 + 3] and out["slots"][-2:].tolist() == [-1, -1]
    assert out["slots"][14:18].tolist() == [8 * 16 + 14, 8 * 16 + 15, 0, 1]


@pytest.mark.parametrize("status,args", [(1, dict(cached=[49, 0])), (1, dict(cached=[-1, 0])), (2, dict(tokens=2)),
                                         (2, dict(max_added=1)), (3, dict(queue=[0, 0]))])
def test_plan_refuses(status, args):
    a = dict(cached=[16, 0], added=[2, 1], table=np.zeros((2, 3), np.int32), ring=np.arange(8, dtype=np.int32),
             queue=[0, 8], page=16, tokens=3, max_added=2)
    assert ref.plan(**a)["info"][0] == 0
    a.update(args)
    assert ref.plan(**a)["info"][0] == status


@pytest.mark.parametrize("setting,token", [((1.0, 0, 1.0, 0.0, 0.0), 0), ((1.0, 1, 1.0, 0.0, 0.99), 2),
                                           ((0.0, 0, 1.0, 0.0, 0.99), 2), ((1.0, 0, 0.0, 0.0, 0.99), 2),
                                           ((1.0, 2, 1.0, 0.0, 0.99), 4), ((1.0, 0, 1.0, 1.0, 0.99), 4),
                                           ((1.0, 0, 1.0, 0.9, 0.2), 2)])
def test_sample_rules(setting, token):
    x = np.array([0.0, np.nan, 3.0, -np.inf, 3.0, 1.0], np.float32)
    assert ref.sample(x, *setting)[0] == token


def test_attention_bound_is_tight_and_catches_a_dropped_key():
    rng = np.random.default_rng(1)
    q, rows = rng.normal(size=(2, 3, 24)) * 0.5, rng.normal(size=(40, 24))
    out, bound = ref.attention(q, rows, 38, 0.2, 16, 2.0 ** -11)
    assert bound.max() < 0.01
    less, _ = ref.attention(q, rows[1:], 37, 0.2, 16, 2.0 ** -11)
    assert (np.abs(less - out) > bound).mean() > 0.5


@pytest.mark.parametrize("pages,page_size", [(0, 64), (-1, 64), (2 ** 31, 64), (2 ** 25, 64), (4, 0), (4, 8), (4, 24), (4, 4112)])
def test_pool_arguments(pages, page_size):
    assert "null context" not in refused(lm.load_library().lm_paged_configure(None, pages, page_size))


def test_layers_need_a_context():
    lib, s, out = lm.load_library(), step(), C.c_void_p()
    assert "null output" in refused(lib.lm_paged_pool(None, 0, None))
    for f, *args in ((lib.lm_paged_configure, None, 4, 64), (lib.lm_paged_pool, None, 0, C.byref(out)),
                 (lib.lm_paged_forward, None, 0, C.byref(s), SOME, SOME * 16, 0),
                 (lib.lm_paged_decoder_forward, None, 0, 0, C.byref(s), SOME, 0)):
        assert "null context" in refused(f(*args))
    s.page_size = 17
    for f, *args in ((lib.lm_paged_forward, None, 0, C.byref(s), SOME, SOME * 16, 0),
                 (lib.lm_paged_decoder_forward, None, 0, 0, C.byref(s), SOME, 0), (lib.lm_paged_forward, None, 0, None, SOME, SOME * 16, 0)):
        assert "null context" not in refused(f(*args))
