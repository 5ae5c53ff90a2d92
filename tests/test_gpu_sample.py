"""Picks by temperature, top-k, top-p and min-p from given random numbers, equal to the definition in
64 bits: weights that are whole numbers of 2^-42 of the largest leave a row's running sums within V
2^-43 of the exact ones, so of the seeded rows here none has its random number that near a border."""
import numpy as np
import pytest

from paged import exact_pick, from_bits, to_type

pytestmark = pytest.mark.gpu


def pick(be, logits, u, temp=None, top_k=None, top_p=None, min_p=None, raw=False):
    logits = np.ascontiguousarray(logits, np.float32)
    S, V = logits.shape
    n32 = lambda a: be.upload(np.broadcast_to(np.asarray(a, np.float32), S).copy()) if a is not None else None
    t, p, m = n32(temp), n32(top_p), n32(min_p)
    k = be.upload(np.broadcast_to(np.asarray(top_k, np.int32), S).copy()) if top_k is not None else None
    ld, ud, td = be.upload(logits), be.upload(np.asarray(u, np.float32)), be.upload(np.full(S + 8, -5, np.int32))
    be.sample(ld, S, V, be.sample_params(t, k, p, m) if not raw else None, ud, td)
    got = be.d2h(td, (S + 8,), np.int32)
    for b in (t, p, m, k, ld, ud, td):
        if b:
            b.free()
    assert np.all(got[S:] == -5)
    return got[:S]


def want(logits, u, temp=1.0, top_k=0, top_p=1.0, min_p=0.0):
    S = len(logits)
    at = lambda a, i: np.broadcast_to(np.asarray(a), S)[i]
    return np.array([exact_pick(logits[i], u[i], at(temp, i), int(at(top_k, i)), at(top_p, i), at(min_p, i)) for i in range(S)])


def both(be, logits, u, **kw):
    assert np.array_equal(pick(be, logits, u, **kw), want(np.asarray(logits, np.float32), np.asarray(u, np.float32), **kw))


SETTINGS = [dict(), dict(temp=0.7), dict(temp=0.0), dict(temp=-1.0), dict(top_k=1), dict(top_k=2), dict(top_k=50), dict(top_k=1000),
            dict(top_p=0.9), dict(top_p=0.1), dict(top_p=0.999), dict(top_p=0.0), dict(min_p=0.05), dict(min_p=1.0), dict(min_p=0.5),
            dict(temp=1.4, top_k=40, top_p=0.95, min_p=0.02), dict(temp=0.3, top_k=500, top_p=0.5),
            dict(temp=2.5, top_p=0.8, min_p=1e-4), dict(temp=5.0, top_k=3000, top_p=0.99)]


@pytest.mark.parametrize("kw", SETTINGS, ids=str)
@pytest.mark.parametrize("V", [1, 2, 3, 63, 64, 65, 1000, 1023, 1024, 1025, 4096, 32000, 50257])
def test_settings_and_sizes(be, V, kw):
    rng = np.random.default_rng(V)
    S = 6
    logits = 3 * rng.standard_normal((S, V)).astype(np.float32)
    both(be, logits, rng.random(S, dtype=np.float32), **kw)


@pytest.mark.parametrize("V", [131072, 151937, 1 << 20])
def test_large_vocabularies(be, V):
    rng = np.random.default_rng(V)
    S = 3
    logits = 2.5 * rng.standard_normal((S, V)).astype(np.float32)
    for kw in (dict(), dict(top_k=40), dict(top_p=0.9), dict(temp=0.6, top_k=2000, top_p=0.97, min_p=0.01)):
        both(be, logits, rng.random(S, dtype=np.float32), **kw)


def test_each_row_its_own(be):
    rng = np.random.default_rng(1)
    S, V = 150, 5000
    logits = 3 * rng.standard_normal((S, V)).astype(np.float32)
    both(be, logits, rng.random(S, dtype=np.float32), temp=rng.choice([0.0, 0.2, 1.0, 1.7, np.nan], S),
         top_k=rng.choice([0, -3, 1, 7, 100, 4999, 5000, 10 ** 6], S), top_p=rng.choice([1.0, 2.0, np.nan, 0.9, 0.4, -1.0], S),
         min_p=rng.choice([0.0, -1.0, np.nan, 0.1, 0.003, 2.0], S))


def test_no_settings(be):
    rng = np.random.default_rng(2)
    logits = rng.standard_normal((4, 777)).astype(np.float32)
    u = rng.random(4, dtype=np.float32)
    assert np.array_equal(pick(be, logits, u, raw=True), want(logits, u))


@pytest.mark.parametrize("V", [5, 1024, 3001, 32000])
def test_equal_logits(be, V):
    """every logit alike, or of a few values: the lowest indices of a threshold's equals are kept"""
    rng = np.random.default_rng(V)
    S = 8
    u = np.concatenate([[0.0, np.float32(1 - 2.0 ** -24)], rng.random(S - 2, dtype=np.float32)]).astype(np.float32)
    for logits in (np.zeros((S, V)), np.full((S, V), -7.25), rng.integers(0, 3, (S, V)), -0.0 * rng.integers(0, 2, (S, V))):
        for kw in (dict(), dict(top_k=max(1, V // 3)), dict(top_p=0.371), dict(top_k=V - 1, top_p=0.5), dict(min_p=1.0), dict(temp=0.5, top_k=2)):
            both(be, logits.astype(np.float32), u, **kw)


def test_masked_and_special_logits(be):
    rng = np.random.default_rng(4)
    S, V = 12, 2000
    low, inf, nan = np.finfo(np.float32).min, np.inf, np.nan
    x = 2 * rng.standard_normal((S, V)).astype(np.float32)
    x[0, :] = -inf                                     # nothing left
    x[1, :] = -inf; x[1, 1234] = -3.0                  # one token left
    x[2, :] = low; x[2, 77] = 0.0                      # masked by the lowest value
    x[3, :] = low                                      # all of the lowest value
    x[4, rng.random(V) < 0.5] = -inf
    x[5, [10, 900]] = inf                              # two infinities share everything
    x[6, 500] = nan
    x[7, :] = nan
    x[8, 0] = nan
    x[9, ::2] = nan; x[9, 1::2] = -inf; x[9, 1501] = 1.0
    x[10, :] = 3e38; x[10, 5] = -3e38
    x[11, :] = 1e-45
    u = rng.random(S, dtype=np.float32)
    for kw in (dict(), dict(temp=0.7, top_k=50), dict(top_p=0.9), dict(min_p=0.1), dict(temp=0.0), dict(top_k=1, top_p=0.5, min_p=0.5),
               dict(temp=1e-30), dict(temp=1e30)):
        both(be, x, u, **kw)


def shapes_of_rows(rng, S, V):
    """rows of many kinds: smooth, rounded to 8 bits (many equal), flat but for a few, a beginning that is
    narrower or wider than the rest, masked by -inf or the lowest value"""
    x = np.empty((S, V), np.float32)
    for i, row in enumerate(x):
        row[:] = rng.choice([0.5, 2.5, 6.0]) * rng.standard_normal(V)
        kind = i % 8
        if kind == 1:
            row[:] = from_bits(to_type(row, "bf16")[0])
        elif kind == 2:
            row[:] = np.round(row)
        elif kind == 3:
            row[:] = 0.25
            row[rng.integers(0, V, 5)] += rng.standard_normal(5).astype(np.float32)
        elif kind == 4:
            row[:40000] = row.max() - 1e-3 * rng.random(row[:40000].size, dtype=np.float32)
        elif kind == 5:
            row[:40000] *= 3
        elif kind == 6:
            row[rng.random(V) < 0.9] = -np.inf
        elif kind == 7:
            row[rng.random(V) < 0.6] = np.finfo(np.float32).min
    return x


@pytest.mark.parametrize("top_k", [0, 30, 192, 193, 400, 600, 601, 1000, 1024, 1025, 3000])
@pytest.mark.parametrize("V", [260, 700, 1200, 5000, 40001, 70003])
def test_kinds_of_rows(be, V, top_k):
    rng = np.random.default_rng(V + top_k)
    S = 32
    x, u = shapes_of_rows(rng, S, V), rng.random(S, dtype=np.float32)
    for temp, top_p, min_p in ((1.0, 1.0, 0.0), (0.6, 0.93, 0.0), (1.7, 0.71, 0.03), (30.0, 0.52, 0.0)):
        both(be, x, u, temp=temp, top_k=top_k, top_p=top_p, min_p=min_p)


@pytest.mark.parametrize("temp", [1e-45, 1e-38, 1e-20, 1e-9, 1e-8, 1e-7, 3e-6, 1e36, 1e38, np.inf])
def test_extreme_temperatures(be, temp):
    """neighbours of the largest logit, a few units of the last place below it, at temperatures at which they weigh
    anything from nothing to nearly as much; differences beyond the largest float at temperatures of its size"""
    rng = np.random.default_rng(8)
    V, tops = 2000, (0.0, 5.0, -3.0, 100.0, 1e-30, 1e-40, 2e38, -2e38)
    x = np.zeros((len(tops), V), np.float32)
    for row, top in zip(x, tops):
        row[:] = np.float32(top) - np.float32(abs(top) * 0.5 + 1e-3) * (1 + rng.random(V, dtype=np.float32))
        at, f = rng.permutation(V)[:60], np.float32(top)
        for i, j in enumerate(at):
            row[j] = f
            if i % 3 == 2:
                f = np.nextafter(f, np.float32(-np.inf))
    x[6, ::2] = -3e38
    u = rng.random(len(x), dtype=np.float32)
    for kw in (dict(), dict(top_k=20), dict(top_k=700), dict(top_p=0.6), dict(min_p=0.3), dict(top_k=900, top_p=0.7, min_p=0.01)):
        both(be, x, u, temp=temp, **kw)


def test_ends_of_the_random_numbers(be):
    rng = np.random.default_rng(5)
    x = rng.standard_normal((6, 3000)).astype(np.float32)
    u = np.array([0.0, 2.0 ** -149, 1 - 2.0 ** -24, 2.0 ** -24, 0.5, 0.25], np.float32)
    both(be, x, u)
    both(be, x, u, top_k=17, top_p=0.8)
    # outside [0, 1): the first and the last kept token
    kept = want(x, np.array([0.0, 1 - 2.0 ** -24] * 3, np.float32), top_k=3)
    assert np.array_equal(pick(be, x, np.array([-1.0, 1.0, np.nan, 5.0, -np.inf, np.inf], np.float32), top_k=3), kept)


def test_frequencies(be):
    """picks over evenly spaced random numbers: each kept token as often as its weight says, to one"""
    rng = np.random.default_rng(6)
    V, S = 40, 4096
    row = rng.standard_normal(V).astype(np.float32)
    u = ((np.arange(S) + 0.5) / S).astype(np.float32)
    got = np.bincount(pick(be, np.tile(row, (S, 1)), u, temp=0.8, top_k=10), minlength=V)
    w = np.exp(row.astype(np.float64) / np.float32(0.8))
    w[np.argsort(-w)[10:]] = 0
    assert np.all(np.abs(got - S * w / w.sum()) <= 1.001)


def test_recorded(be):
    """a recording reads logits, settings and random numbers at each replay"""
    rng = np.random.default_rng(7)
    S, V = 3, 4001
    ld, ud, td, tp = be.upload(np.zeros((S, V), np.float32)), be.upload(np.zeros(S, np.float32)), be.upload(np.zeros(S, np.int32)), \
        be.upload(np.ones(S, np.float32))
    p = be.sample_params(None, None, tp)
    be.sample(ld, S, V, p, ud, td)
    be.graph_begin()
    be.sample(ld, S, V, p, ud, td)
    g = be.graph_end()
    for _ in range(4):
        x, u, t = rng.standard_normal((S, V)).astype(np.float32) * 3, rng.random(S, dtype=np.float32), rng.random(S, dtype=np.float32)
        be.h2d(ld, x); be.h2d(ud, u); be.h2d(tp, t)
        be.graph_launch(g)
        assert np.array_equal(be.d2h(td, (S,), np.int32), want(x, u, top_p=t))
    be.graph_destroy(g)
    for b in (ld, ud, td, tp):
        b.free()
