"""qw_sample (include/qw_attn.h) on the device against its definition in 64 bits."""
import numpy as np
import pytest

import qwental_amd as q

pytestmark = pytest.mark.gpu
ROW = np.dtype([("temperature", "<f4"), ("top_p", "<f4"), ("min_p", "<f4"), ("top_k", "<u4")])


def drawn(l, p, u):
    """(token, probability, how near u came to the border of another token or a filter to that of another set: a share of the whole, and the probability
    that lies between u and each token's own part, by token)."""
    l = l.astype(np.float64)
    t, top_p, min_p, k = float(p["temperature"]), float(p["top_p"]), float(p["min_p"]), int(p["top_k"])
    fine = ~np.isnan(l) & (l > -np.inf)
    if not fine.any():
        return 0xffffffff, 0.0, 1.0, None
    top = l[fine].max()
    if not t > 0:
        return int(np.argmax(np.where(fine, l, -np.inf))), 1.0, 1.0, None
    with np.errstate(invalid="ignore"):
        w = np.where(fine, np.exp((l - top) / t) if np.isfinite(top) else l == top, 0.0).astype(np.float64)
    order = np.lexsort((np.arange(len(l)), -np.where(fine, l, -np.inf)))
    order = order[fine[order]]
    near = 1.0
    if 0 < k < len(l):
        order = order[:k]
    if top_p < 1:
        c = np.cumsum(w[order])
        m = min(int(np.searchsorted(c, top_p * c[-1])), len(order) - 1)
        near = min(near, np.abs(c[:-1] / c[-1] - top_p).min() if len(c) > 1 else 1.0)
        order = order[:m + 1]
    if min_p > 0:
        near = min(near, np.abs(w[order] - min_p)[w[order] < 1].min(initial=1.0))
        order = order[w[order] >= min(min_p, 1.0)]
    order = np.sort(order)
    c = np.cumsum(w[order])
    i = int(np.searchsorted(c, u * c[-1], side="right"))
    near = min(near, np.abs(c[:-1] / c[-1] - u).min(initial=1.0))
    i = min(i, len(order) - 1)
    gap = np.full(len(l), near)  # tokens that a filter just took out are as far as the filter was near
    gap[order] = np.maximum(0, np.maximum((c - w[order]) / c[-1] - u, u - c / c[-1]))
    return int(order[i]), float(w[order[i]] / c[-1]), near, gap


def draw(gpu, logits, params, u, stride=0, probs=True):
    B, V = logits.shape
    x = logits
    if stride:
        x = np.full((B, stride), 99.0, np.float32)
        x[:, :V] = logits
    bufs = [gpu.buf_from(a, device_only=True) for a in (x, params, u, np.full(B, 77, np.uint32), np.full(B, 77.0, np.float32))]
    ws = gpu.buf(q.sample_ws_bytes(gpu, B, V), device_only=True)
    ws.fill(np.full(ws.size, 255, np.uint8))
    call = q.Sample(B, V, bufs[0], bufs[1], bufs[2], bufs[3], bufs[4] if probs else None, ws, stride=stride)
    got = []
    for _ in range(2):
        b = gpu.batch()
        call(b)
        b.end()
        got.append((bufs[3].read(4 * B, dtype=np.uint32), bufs[4].read(4 * B, dtype=np.float32)))
    assert np.array_equal(got[0][0], got[1][0]) and np.array_equal(got[0][1], got[1][1])
    for b in bufs + [ws]:
        b.free()
    return got[0]


def check(gpu, logits, params, u, **kw):
    """Tokens equal where no border is within 2^-20 of the draw. A weight is 2^43 times an exponential of 2^-22 relative error (one rounding of its argument's fraction, a step of the
    exponential), cut to whole numbers (V 2^-43 of the whole at most); a probability is the quotient of two such, rounded: 2^-21 + 2^-24, and V 2^-42. Where one is (of V tokens alike
    each has 1 / V: at 131072 a quarter of all draws), the token drawn has to be one that lies as near to u."""
    ids, probs = draw(gpu, logits, params, u, **kw)
    B, V = logits.shape
    for b in range(B):
        i, p, margin, gap = drawn(logits[b], params[b], float(u[b]))
        if margin < 2.0 ** -20:
            assert gap[ids[b]] < 2.0 ** -20, (b, params[b], u[b], ids[b], i)
            continue
        assert ids[b] == i, (b, params[b], u[b], ids[b], i)
        if kw.get("probs", True):
            assert abs(probs[b] - p) <= (2.0 ** -21 + 2.0 ** -24) * p + V * 2.0 ** -42
        else:
            assert probs[b] == 77
    return ids


SETTINGS = [(1.0, 1.0, 0.0, 0), (0.7, 0.95, 0.0, 40), (1.2, 0.9, 0.0, 0), (0.9, 1.0, 0.05, 0), (0.0, 0.5, 0.5, 3), (1.0, 0.3, 0.02, 1000), (1.5, 1.0, 0.0, 1), (0.05, 0.99, 0.0, 0),
            (1.0, 0.0, 0.0, 0), (1.0, 1.0, 1.0, 0), (3.0, 0.9999, 0.0, 100000), (1.0, 2.0, -1.0, 0)]


def model_like(rng, B, V, spread=2.5):
    x = rng.standard_normal((B, V)).astype(np.float32) * np.float32(spread)
    x += (rng.random((B, V)) < 30 / V) * (4 + 2 * rng.standard_normal((B, V))).astype(np.float32)
    return x.astype(np.float32)


@pytest.mark.parametrize("V", [1, 2, 63, 64, 1000, 4095, 4096, 4097, 32001, 131072, 1 << 20])
def test_settings(gpu, V):
    rng = np.random.default_rng(V)
    B = len(SETTINGS)
    check(gpu, model_like(rng, B, V), np.array(SETTINGS, ROW), rng.random(B, dtype=np.float32))


@pytest.mark.parametrize("seed", range(6))
def test_many_rows(gpu, seed):
    rng = np.random.default_rng(seed)
    B, V = 64, 5000 + 777 * seed
    p = np.zeros(B, ROW)
    p["temperature"], p["top_p"] = rng.uniform(0.1, 2, B), rng.choice([1.0, 0.95, 0.5, 0.1], B)
    p["min_p"], p["top_k"] = rng.choice([0, 0, 0.01, 0.3], B), rng.choice([0, 1, 5, 40, 500, V, V + 5], B)
    check(gpu, model_like(rng, B, V, 1 + seed), p, rng.random(B, dtype=np.float32), stride=V + 3)


def test_equal_logits_go_by_number(gpu):
    """All tokens alike, and long runs of them on a filter's border."""
    rng = np.random.default_rng(3)
    V = 9001
    x = np.zeros((8, V), np.float32)
    x[4:] = np.where(rng.random((4, V)) < 0.5, 1.0, -1.0)
    p = np.array([(1, 1, 0, 0), (1, 1, 0, 100), (1, 0.25, 0, 0), (1, 0.5, 0, 5000), (1, 1, 0, 3), (1, 0.6, 0, 0), (1, 1, 0, 8000), (1, 0.99, 0.2, 0)], ROW)
    ids = check(gpu, x, p, np.array([0.5, 0.995, 0.9999, 0.9999, 0.9, 0.9999, 0.9999, 0.0], np.float32))
    assert ids[1] == 99 and ids[2] < V // 4 + 1


@pytest.mark.parametrize("u", [0.0, 1 - 2.0 ** -24, 1.0, 2.0, -1.0, np.nan])
def test_ends_of_the_random_numbers(gpu, u):
    """The first token with any probability at 0, the last at the largest number below 1; anything outside [0, 1) counts as an end of it."""
    x = np.array([[-np.inf, 0.0, 1.0, 0.5, -np.inf]] * 2, np.float32)
    ids, _ = draw(gpu, x, np.array([(1, 1, 0, 0), (1, 1, 0, 2)], ROW), np.full(2, u, np.float32))
    assert list(ids) == ([1, 2] if not u > 0 else [3, 3])


def test_rows_that_hold_nothing_and_infinities(gpu):
    inf, nan = np.inf, np.nan
    x = np.array([[nan] * 5, [-inf] * 5, [nan, -inf, 2.0, nan, -inf], [inf, 1.0, inf, nan, 3.0], [-3e38, -3e38, -inf, 3e38, nan], [0.0, -0.0, -1e30, -0.0, 0.0], [-1e-45, 1e-45, 0, 0, 0], [-7.0] * 5], np.float32)
    for setting in SETTINGS:
        for u in (0.1, 0.6, 0.95):
            check(gpu, x, np.array([setting] * len(x), ROW), np.full(len(x), u, np.float32))


def test_extreme_settings(gpu):
    rng = np.random.default_rng(5)
    x = model_like(rng, 8, 3001)
    inf, nan = np.inf, np.nan
    p = np.array([(inf, 1, 0, 0), (1e-45, 1, 0, 0), (nan, 1, 0, 0), (-1, 1, 0, 0), (1, nan, nan, 0), (1, -1, 0, 0), (1e30, 0.5, 0, 0), (1, 1, inf, 0xffffffff)], ROW)
    check(gpu, x, p, rng.random(8, dtype=np.float32))


def test_without_probabilities(gpu):
    rng = np.random.default_rng(6)
    check(gpu, model_like(rng, 3, 777), np.array(SETTINGS[:3], ROW), rng.random(3, dtype=np.float32), probs=False)


@pytest.mark.parametrize("V,first,spread", [(20000, 100, 20000), (20000, 100, 100), (131072, 250, 131072), (8192, 64, 8192), (300, 30, 300), (131072, 40, 20000)])
def test_few_tokens_left(gpu, V, first, spread):
    """Some tens or hundreds of tokens far above all others, over the whole row or side by side (more in one stretch of it than are at hand), many of them equal; a filter's border among them."""
    rng = np.random.default_rng(V + first + spread)
    B = 24
    logits = rng.standard_normal((B, V)).astype(np.float32)
    for b in range(B):
        at = rng.permutation(spread)[:first]
        logits[b, at] = 9 + (rng.integers(0, 12, first) / 4 if b % 2 else rng.standard_normal(first))
    k = rng.integers(2, first, B)
    params = np.array([(0.8, *((0.9, 0.0), (1.0, 0.0), (0.95, 0.05), (1.0, 0.3))[b % 4], k[b] if b % 3 else 0) for b in range(B)], ROW)
    check(gpu, logits, params, rng.random(B).astype(np.float32))
