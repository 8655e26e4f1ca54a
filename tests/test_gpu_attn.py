"""The attention half of a decode step (include/qw_attn.h) on the device, against the operators' definitions in 64 bits."""
import numpy as np
import pytest

import qwental_amd as q
from attn_helpers import F16, Q8, Cache, Step, attention, scale_places, tolerance, turned

pytestmark = pytest.mark.gpu


def rows(rng, R, heads, D, spread=1.0):
    return (rng.standard_normal((R, heads, D)) * spread).astype(np.float16)


def filled(rng, kind, heads, D, page, step):
    """A cache whose slots hold random tokens, with a few large channels; all else is NaN (binary16 0xffff, codes -1 and scales NaN)."""
    c = Cache(kind, heads, D, page, step.pages, fill=0xffff)
    channel = 1 + 3 * (rng.random(D) < 0.06)
    for i, n in enumerate(step.len):
        for t in range(int(n)):
            c.put(step.table, i, t, (rng.standard_normal((heads, D)) * channel).astype(np.float16), rng.standard_normal((heads, D)).astype(np.float16))
    return c


class Device:
    """The buffers of a test, freed at its end."""

    def __init__(self, gpu):
        self.gpu, self.all = gpu, []

    def up(self, a):
        self.all.append(self.gpu.buf_from(a, device_only=True))
        return self.all[-1]

    def new(self, size):
        self.all.append(self.gpu.buf(size, device_only=True))
        return self.all[-1]

    def cache(self, c):
        return q.KvCache(self.up(c.raw), c.kind, c.heads, c.D, c.page, c.pages)

    def step(self, s):
        d = s.device(self.gpu)
        self.all += s.bufs
        return d

    def run(self, *calls):
        b = self.gpu.batch()
        for c in calls:
            c(b)
        b.end()


@pytest.fixture
def dev(gpu):
    d = Device(gpu)
    yield d
    for b in d.all:
        b.free()


SHAPES = [  # type, kv heads, query heads, dim, page, rows a slot, tokens a slot
    (F16, 1, 1, 64, 16, [1], [1]),
    (F16, 2, 16, 128, 64, [1], [700]),
    (Q8, 2, 16, 256, 64, [1], [333]),
    (F16, 4, 32, 128, 64, [1, 1, 1, 1], [1, 17, 64, 130]),
    (Q8, 4, 32, 128, 16, [1, 3, 5, 2], [31, 32, 33, 200]),
    (F16, 1, 5, 192, 32, [4, 1, 7], [4, 15, 90]),
    (Q8, 3, 3, 64, 32, [9, 20], [9, 77]),
    (F16, 2, 2, 256, 256, [33, 1], [40, 257]),
    (Q8, 1, 40, 192, 64, [2, 2], [2, 65]),
    (F16, 8, 64, 64, 16, [1, 0, 2], [16, 5, 48]),
    (F16, 256, 256, 64, 16, [1, 1], [20, 3]),      # the most heads there are
    (Q8, 1, 1024, 64, 32, [1, 2], [33, 70]),
    (F16, 1, 2, 64, 4096, [1, 2], [5000, 10]),     # pages larger than what they hold
]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("rot", ["halves", "adjacent", "part", "none"])
def test_rows_into_the_cache_and_back(gpu, dev, shape, rot):
    kind, H, Hq, D, page, n, length = shape
    rng = np.random.default_rng(D + page + len(n))
    s = Step(rng, n, length, page, rows=sum(n) + 3)  # three rows behind the last slot's
    c = Cache(kind, H, D, page, s.pages, rng=rng)
    R = s.rows
    qr, k, v = rows(rng, R, Hq, D), rows(rng, R, H, D, 2.0), rows(rng, R, H, D)
    dims = {"halves": D, "adjacent": D, "part": D // 2, "none": 0}[rot]
    pairs = [dims // 2] if rot == "adjacent" else [dims // 2 - 2 * (dims // 8), dims // 8, dims // 8]
    freq = 1e6 ** (-np.arange(dims // 2) / max(dims // 2, 1))
    pos = rng.integers(0, 200000, (R, len(pairs))).astype(np.int32)
    rope = q.Rope(dims, pairs, dev.up(freq), dev.up(pos), adjacent=rot == "adjacent") if dims else None
    kc, st = dev.cache(c), dev.step(s)
    back = rng.integers(0, 65536, (2, R, H, D), dtype=np.uint16)
    bufs = [dev.up(x) for x in (qr, np.zeros_like(qr), k, v, back[0], back[1])]
    bufs[1].fill(np.full(qr.size, 0x1234, np.uint16))
    dev.run(q.KvWrite(kc, st, Hq, bufs[0], bufs[1], bufs[2], bufs[3], rope), q.KvRead(kc, st, bufs[4], bufs[5]))
    qt, kt = (turned(x, pos, freq, pairs, rot == "adjacent") for x in (qr, k))
    want_q, want_k, want_v = np.full(qr.shape, 0x1234, np.uint16).view(np.float16), back[0].view(np.float16).copy(), back[1].view(np.float16).copy()
    for row, slot, token in s.rows_of():
        c.put(s.table, slot, token, kt[row], v[row])
        want_q[row] = qt[row]
        a, b = c.get(s.table, slot, [token])
        want_k[row], want_v[row] = a[0].astype(np.float16), b[0].astype(np.float16)
    same(bufs[1].read(dtype=np.float16).reshape(qr.shape), want_q, bool(dims))
    got = kc.keep.read().reshape(c.raw.shape)
    if dims and kind == F16:
        # turned keys: the 64-bit result may be rounded through 32 bits on its way (one step of binary16 where it lies beside a border)
        same(got.view(np.float16), c.raw.view(np.float16), True)
    elif not dims:
        assert np.array_equal(got, c.raw)  # every other byte of the cache as it was
    same(bufs[4].read(dtype=np.float16).reshape(k.shape), want_k, bool(dims), 2.0 ** -5 if kind == Q8 else 0)
    same(bufs[5].read(dtype=np.float16).reshape(v.shape), want_v, False)


def same(got, want, may_step, code=0):
    """Equal bits, but for at most one value in 500 that is a step of binary16 off (or, behind it, a code's: `code` of the largest key in sight)."""
    if not may_step:
        assert np.array_equal(got.view(np.uint16), want.view(np.uint16))
        return
    g, w = got.astype(np.float64), want.astype(np.float64)
    off = got.view(np.uint16) != want.view(np.uint16)
    assert off.mean() <= 1 / 500
    with np.errstate(invalid="ignore"):
        assert not (np.abs(g - w)[off] > 2.0 ** -10 * np.abs(w[off]) + code * np.abs(w[np.isfinite(w)]).max() + 2.0 ** -24).any()


def check(dev, gpu, rng, kind, H, Hq, D, page, s, window=0, scale=0.0, c=None, dead=()):
    c = c or filled(rng, kind, H, D, page, s)
    qr = rows(rng, s.rows, Hq, D)
    out = dev.up(np.full(qr.shape, 0x1234, np.uint16))
    ws = dev.new(q.attn_ws_bytes(gpu, D))
    ws.fill(np.full(ws.size // 4, 0xffffffff, np.uint32))  # the workspace need not be cleared
    call = q.Attn(dev.cache(c), dev.step(s), Hq, dev.up(qr), out, ws, scale=scale, window=window)
    dev.run(call)
    got = out.read(dtype=np.float16).reshape(qr.shape)
    want, tol = attention(c, s, qr, scale or 1 / np.sqrt(D), window, dead)
    none = np.isnan(want[:, 0, 0])
    assert (got[none].view(np.uint16) == 0x1234).all()
    with np.errstate(invalid="ignore"):
        bad = ~(np.abs(got[~none].astype(np.float64) - want[~none]) <= tol[~none])
    assert not bad.any(), "%d of %d values, first at %s: %s for %s" % (bad.sum(), bad.size, np.argwhere(bad)[0], got[~none][bad][0], want[~none][bad][0])
    dev.run(call)
    assert np.array_equal(out.read(dtype=np.uint16), got.view(np.uint16).ravel())  # the same bits again
    return got


@pytest.mark.parametrize("shape", SHAPES)
def test_attention(gpu, dev, shape):
    kind, H, Hq, D, page, n, length = shape
    rng = np.random.default_rng(sum(length) + D)
    check(dev, gpu, rng, kind, H, Hq, D, page, Step(rng, n, length, page, rows=sum(n) + 2))


@pytest.mark.parametrize("kind", [F16, Q8])
@pytest.mark.parametrize("window", [1, 15, 16, 33, 200])
def test_attention_in_a_window(gpu, dev, kind, window):
    rng = np.random.default_rng(window)
    check(dev, gpu, rng, kind, 2, 6, 128, 32, Step(rng, [1, 3, 12, 1], [1, 40, 190, 300], 32), window=window)


@pytest.mark.parametrize("kind", [F16, Q8])
@pytest.mark.parametrize("D", [64, 128, 192, 256])
def test_rows_without_tokens_and_short_slots(gpu, dev, kind, D):
    """Slots of zero and one tokens, slots with more rows than tokens: such rows see nothing and are zeros."""
    rng = np.random.default_rng(D)
    s = Step(rng, [1, 1, 4, 0, 2, 1], [0, 1, 2, 7, 16, 0], 16)
    got = check(dev, gpu, rng, kind, 2, 4, D, 16, s)
    assert not got[[0, 2, 3, 8]].any()


@pytest.mark.parametrize("kind,D,G,n,length", [(Q8, 128, 8, [1], [20000]), (F16, 64, 4, [1, 3], [9000, 100]), (Q8, 256, 8, [2], [6000]), (F16, 256, 1, [1, 1, 1], [4000, 1, 2500])])
def test_long_slots_are_cut_and_joined(gpu, dev, kind, D, G, n, length):
    rng = np.random.default_rng(D + G)
    check(dev, gpu, rng, kind, 2, 2 * G, D, 64, Step(rng, n, length, 64))


@pytest.mark.parametrize("kind", [F16, Q8])
@pytest.mark.parametrize("scale", [1e-3, 2.0])
def test_scales(gpu, dev, kind, scale):
    """Nearly equal weights, and one token that has all of it."""
    rng = np.random.default_rng(7)
    check(dev, gpu, rng, kind, 1, 8, 128, 64, Step(rng, [1, 2], [500, 77], 64), scale=scale)


@pytest.mark.parametrize("kind", [F16, Q8])
@pytest.mark.parametrize("what", [np.inf, -np.inf, np.nan, 65504.0])
def test_tokens_that_a_row_does_not_see_may_hold_anything(gpu, dev, kind, what):
    """The last draft's key and value are `what`: the rows before it are as they would be; with a window, so is a row that has left one behind."""
    rng = np.random.default_rng(11)
    s = Step(rng, [5, 3], [70, 33], 32)
    c = filled(rng, kind, 2, 64, 32, s)
    qr = rows(rng, s.rows, 4, 64)
    bad = np.full((2, 64), what, np.float16)
    c.put(s.table, 0, 69, bad, bad)
    c.put(s.table, 1, 32, bad, bad)
    c.put(s.table, 0, 3, bad, bad)  # (seen by nobody in a window of 60)
    out, ws = dev.new(qr.nbytes), dev.new(q.attn_ws_bytes(gpu, 64))
    dev.run(q.Attn(dev.cache(c), dev.step(s), 4, dev.up(qr), out, ws, window=60))
    got = out.read(dtype=np.float16).reshape(qr.shape)
    c.put(s.table, 0, 3, np.zeros((2, 64), np.float16), np.zeros((2, 64), np.float16))
    want, tol = attention(c, s, qr, 0.125, 60)
    for r in (0, 1, 2, 3, 5, 6):
        assert (np.abs(got[r] - want[r]) <= tol[r]).all()


@pytest.mark.parametrize("kind", [F16, Q8])
def test_pages_that_are_none(gpu, dev, kind):
    """A page number from `pages` on: its tokens are not attended to, not written, and read back as zeros."""
    rng = np.random.default_rng(13)
    s = Step(rng, [2, 1], [100, 64], 16)
    c = filled(rng, kind, 2, 128, 16, s)
    s.table[0, 2], s.table[0, 6], s.table[1, 0] = s.pages, 0xffffffff, 1 << 31
    check(dev, gpu, rng, kind, 2, 2, 128, 16, s, c=c, dead=(s.pages, 0xffffffff, 1 << 31))
    kc, st = dev.cache(c), dev.step(s)
    x = [dev.up(rows(rng, 3, 2, 128)) for _ in range(4)]
    back = [dev.up(np.full((3, 2, 128), 0x1234, np.uint16)) for _ in range(2)]
    dev.run(q.KvWrite(kc, st, 2, *x), q.KvRead(kc, st, *back))
    for b in back:
        got = b.read(dtype=np.uint16).reshape(3, 2, 128)
        assert not got[0].any() and not got[1].any() and got[2].any()


def test_steps_that_do_not_fit_touch_nothing(gpu, dev):
    """Rows that run backwards or beyond the step, lengths beyond the table: what lies in bounds is served, the rest is left alone."""
    rng = np.random.default_rng(17)
    s = Step(rng, [1, 1, 1], [20, 30, 25], 16)
    c = filled(rng, F16, 1, 64, 16, s)
    qr = rows(rng, 3, 1, 64)
    out, ws = dev.up(np.full(qr.shape, 0x1234, np.uint16)), dev.new(q.attn_ws_bytes(gpu, 64))
    st, kc, qb = dev.step(s), dev.cache(c), dev.up(qr)
    s.bufs[0].fill(np.array([0, 1, 700, 3], np.uint32))  # slot 1 ends at row 700, slot 2 begins there
    back = [dev.up(np.full((3, 1, 64), 0x1234, np.uint16)) for _ in range(2)]
    dev.run(q.Attn(kc, st, 1, qb, out, ws), q.KvWrite(kc, st, 1, qb, qb, dev.up(qr), dev.up(qr)), q.KvRead(kc, st, *back))
    got = out.read(dtype=np.uint16).reshape(3, 64)
    assert (got[0] != 0x1234).any() and (got[1:] == 0x1234).all()
    s.bufs[0].fill(np.array([0, 1, 2, 3], np.uint32))
    s.bufs[1].fill(np.array([20, 0xffffffff, 25], np.uint32))  # as many tokens as the table has room for: two pages
    dev.run(q.Attn(kc, st, 1, qb, out, ws))
    assert (out.read(dtype=np.uint16).reshape(3, 64) != 0x1234).any(1).all()


def test_strides_and_offsets(gpu, dev):
    """q, k and v as parts of one row of a fused projection, turned in place; the buffers' parts at odd multiples of 16 bytes."""
    rng = np.random.default_rng(19)
    H, Hq, D, page = 2, 6, 64, 16
    s = Step(rng, [2, 3], [30, 17], page, rows=6)
    c = Cache(Q8, H, D, page, s.pages, rng=rng)
    width = (Hq + 2 * H) * D + 24
    x = np.zeros((6, width), np.float16)
    x[:, :(Hq + 2 * H) * D] = rng.standard_normal((6, (Hq + 2 * H) * D))
    freq, pos = 1e4 ** (-np.arange(32) / 32), rng.integers(0, 5000, (6, 1)).astype(np.int32)
    lead = np.zeros(48, np.uint8)
    shifted = lambda a: (dev.up(np.concatenate([lead, np.ascontiguousarray(a).view(np.uint8).ravel()])), 48)  # noqa: E731
    at = shifted(x)
    part = lambda o: (at[0], 48 + 2 * o)  # noqa: E731
    s.device(gpu)
    dev.all += s.bufs
    step = q.KvStep(2, 6, s.max_pages, shifted(s.first.astype(np.uint32)), shifted(s.len.astype(np.uint32)), shifted(s.table))
    kc = q.KvCache(shifted(c.raw), Q8, H, D, page, s.pages)
    out = shifted(np.zeros((6, Hq * D + 8), np.float16))
    ws = (dev.new(q.attn_ws_bytes(gpu, D) + 16), 16)
    dev.run(q.KvWrite(kc, step, Hq, part(0), part(0), part(Hq * D), part((Hq + H) * D), q.Rope(64, [32], shifted(freq), shifted(pos)), strides=(width,) * 4),
            q.Attn(kc, step, Hq, part(0), out, ws, strides=(width, Hq * D + 8)))
    heads = lambda a, b: x[:, a * D:b * D].reshape(6, b - a, D)  # noqa: E731
    qt, kt, v = turned(heads(0, Hq), pos, freq, [32], False), turned(heads(Hq, Hq + H), pos, freq, [32], False), heads(Hq + H, Hq + 2 * H)
    got = at[0].read(offset=48, dtype=np.float16).reshape(6, width)
    same(got[:5, :Hq * D].reshape(5, Hq, D), qt[:5], True)
    assert np.array_equal(got[:, Hq * D:], x[:, Hq * D:]) and np.array_equal(got[5], x[5])
    c.raw = kc.keep[0].read(offset=48).reshape(c.raw.shape)
    for row, slot, token in s.rows_of():
        k1, v1 = c.get(s.table, slot, [token])
        assert np.abs(k1[0] - kt[row]).max() <= np.abs(kt[row]).max() / 127 * 0.51 and np.abs(v1[0] - v[row]).max() <= np.abs(v[row]).max() / 127 * 0.51
    # the tokens before the step's are random bytes: scales may be anything, so the slots' rows are compared where they are finite
    want, tol = attention(c, s, got[:, :Hq * D].reshape(6, Hq, D), 0.125)
    o = out[0].read(offset=48, dtype=np.float16).reshape(6, -1)
    fine = np.isfinite(want[:5]).all((1, 2)) & (np.abs(want[:5]).max((1, 2)) < 60000)
    assert (np.abs(o[:5, :Hq * D].reshape(5, Hq, D) - want[:5])[fine] <= tol[:5][fine]).all() and not o[:, Hq * D:].any() and not o[5].any()


@pytest.mark.parametrize("window", [(1 << 30) - 1, 1 << 30, (1 << 31) - 1])
def test_windows_larger_than_everything(gpu, dev, window):
    rng = np.random.default_rng(23)
    s = Step(rng, [5, 1, 40], [2, 70, 9], 16)  # rows before their slot's first token too
    c = filled(rng, Q8, 2, 64, 16, s)
    got = [check(dev, gpu, np.random.default_rng(1), Q8, 2, 8, 64, 16, s, window=w, c=c) for w in (window, 0)]
    assert np.array_equal(got[0].view(np.uint16), got[1].view(np.uint16))


@pytest.mark.parametrize("freq", [1e-300, 1e-42, 1e-20])
def test_angles_near_zero(gpu, dev, freq):
    """Products far below what 32 bits hold: zeros, of either sign."""
    rng = np.random.default_rng(29)
    s = Step(rng, [4], [4], 16)
    c = Cache(F16, 1, 64, 16, s.pages, rng=rng)
    x = rows(rng, 4, 1, 64)
    x[..., :32] = 0
    x[1, :, 32:] = -0.0
    pos = np.array([[1], [2], [-3], [4]], np.int32)
    out = dev.new(x.nbytes)
    xb = dev.up(x)
    dev.run(q.KvWrite(dev.cache(c), dev.step(s), 1, xb, out, xb, xb, q.Rope(64, [32], dev.up(np.full(32, freq)), dev.up(pos))))
    assert np.array_equal(out.read(dtype=np.float16).reshape(x.shape), turned(x, pos, np.full(32, freq), [32], False))


@pytest.mark.parametrize("rot", ["halves", "adjacent", "part", "none"])
@pytest.mark.parametrize("shape", [(F16, 2, 16, 64, 16, [600], [600]), (Q8, 4, 32, 128, 64, [1400], [3001]), (Q8, 1, 5, 256, 32, [1500, 1, 703], [1507, 1, 703]), (F16, 3, 3, 192, 16, [300, 900], [300, 1000])])
def test_many_rows_into_the_cache_and_back(gpu, dev, shape, rot):
    """Several heads a wave."""
    test_rows_into_the_cache_and_back(gpu, dev, shape, rot)


@pytest.mark.parametrize("kind", [F16, Q8])
@pytest.mark.parametrize("scale", [1.0, 1e5, 1e12, 1e30])
def test_scores_of_any_size(gpu, dev, kind, scale):
    """Whole numbers, so that scores are exact and their differences 2 at least: all weight lies on the largest, or on those that share it, whatever it is times the scale. (At scale 1 the others have
    e^-2 and less of it: as everywhere.) Results are off by their rounding, 2^-11, and what 4096 such sums lose, 2^-12 of the largest value."""
    rng = np.random.default_rng(37)
    s = Step(rng, [2, 1], [700, 90], 32)
    c = Cache(kind, 2, 64, 32, s.pages, fill=0xffff)
    for i, n in enumerate(s.len):
        for t in range(int(n)):
            c.put(s.table, i, t, (2 * rng.integers(-63, 64, (2, 64)) + 1).astype(np.float16), rng.standard_normal((2, 64)).astype(np.float16))
    if kind == Q8:  # scales of the keys: 1
        for values, w in ((False, 1.0),):
            at = scale_places(64, values)
            for b in range(2):
                c.raw[..., at + b] = np.frombuffer(np.float16(w).tobytes(), np.uint8)[b]
    qr = (2 * rng.integers(-3, 4, (3, 8, 64))).astype(np.float16)
    if scale == 1.0:
        qr = (qr / 4096).astype(np.float16)
    out, ws = dev.new(qr.nbytes), dev.new(q.attn_ws_bytes(gpu, 64))
    dev.run(q.Attn(dev.cache(c), dev.step(s), 8, dev.up(qr), out, ws, scale=scale))
    got = out.read(dtype=np.float16).reshape(qr.shape).astype(np.float64)
    for row, slot, token in s.rows_of():
        k, v = c.get(s.table, slot, range(token + 1))
        x = np.einsum("hgd,thd->hgt", qr[row].astype(np.float64).reshape(2, 4, 64), k)
        p = np.exp(np.maximum((x - x.max(-1, keepdims=True)) * scale, -1e4))
        want = np.einsum("hgt,thd->hgd", p / p.sum(-1, keepdims=True), v).reshape(8, 64)
        assert (np.abs(got[row] - want) <= 2.0 ** -11 * np.abs(want) + 2.0 ** -12 * np.abs(v).max()).all()


@pytest.mark.parametrize("kind", [F16, Q8])
def test_tokens_beyond_two_to_the_29(gpu, dev, kind):
    """The last tokens of slots of 2^29 and 2^30, of which two pages each are there: rows in, out, and attention in a window."""
    rng = np.random.default_rng(41)
    page, window = 65536, 150
    s = Step.__new__(Step)
    s.n, s.len, s.rows, s.pages, s.max_pages = np.array([2, 3]), np.array([(1 << 29) + 70, (1 << 30) - 1]), 5, 4, 1 << 14
    s.first, s.table = np.array([0, 2, 5]), np.full((2, 1 << 14), 0xffffffff, np.uint32)
    s.table[0, 8191:8193] = 2, 0
    s.table[1, 16382:] = 1, 3
    c = Cache(kind, 2, 64, page, 4, fill=0xffff)
    for i, n in enumerate(s.len):
        for t in range(int(n) - 300, int(n)):
            c.put(s.table, i, t, *rng.standard_normal((2, 2, 64)).astype(np.float16))
    k, v, qr = rows(rng, 5, 2, 64), rows(rng, 5, 2, 64), rows(rng, 5, 8, 64)
    kc, st, qb, back = dev.cache(c), dev.step(s), dev.up(qr), [dev.new(k.nbytes) for _ in range(2)]
    out, ws = dev.new(qr.nbytes), dev.new(q.attn_ws_bytes(gpu, 64))
    dev.run(q.KvWrite(kc, st, 0, None, None, dev.up(k), dev.up(v)), q.KvRead(kc, st, *back), q.Attn(kc, st, 8, qb, out, ws, window=window))
    for row, slot, token in s.rows_of():
        c.put(s.table, slot, token, k[row], v[row])
    assert np.array_equal(kc.keep.read(), c.raw.ravel())
    for row, slot, token in s.rows_of():
        for got, want in zip(back, c.get(s.table, slot, [token])):
            assert np.array_equal(got.read(dtype=np.float16).reshape(k.shape)[row], want[0].astype(np.float16))
    want, tol = attention(c, s, qr, 0.125, window)
    assert (np.abs(out.read(dtype=np.float16).reshape(qr.shape) - want) <= tol).all()


@pytest.mark.parametrize("kind", [F16, Q8])
@pytest.mark.parametrize("D,G", [(64, 4), (64, 10), (128, 4), (128, 10), (192, 8), (256, 8)])
def test_units_past_the_caches(gpu, dev, kind, D, G):
    """Pages enough for slots of any length that the kernels read past the caches."""
    rng = np.random.default_rng(D + G)
    page, H = 64, 1
    pages = (64 << 20) // (page // 16 * D * (64 if kind == F16 else 34)) + 1
    s = Step(rng, [1, 2], [700, 95], page, pages=pages)
    s.table = np.concatenate([s.table, np.full((2, pages), 0xffffffff, np.uint32)], 1)
    s.max_pages = s.table.shape[1]
    check(dev, gpu, rng, kind, H, H * G, D, page, s)


@pytest.mark.parametrize("window", [0, 40])
def test_the_most_rows(gpu, dev, window):
    """65536 rows of a slot, in, out and attended to; some of them checked."""
    rng = np.random.default_rng(43)
    R, page = 65536, 256
    s = Step(rng, [R], [R], page, spare=0)
    k, v, qr = rows(rng, R, 1, 64), rows(rng, R, 1, 64), rows(rng, R, 2, 64)
    kc = q.KvCache(dev.new(q.kv_bytes(gpu.L, F16, 1, 64, page, s.pages)), F16, 1, 64, page, s.pages)
    st, back, out, ws = dev.step(s), [dev.new(k.nbytes) for _ in range(2)], dev.new(qr.nbytes), dev.new(q.attn_ws_bytes(gpu, 64))
    qb = dev.up(qr)
    dev.run(q.KvWrite(kc, st, 2, qb, qb, dev.up(k), dev.up(v)), q.KvRead(kc, st, *back), q.Attn(kc, st, 2, qb, out, ws, window=window))
    assert np.array_equal(back[0].read(dtype=np.uint16), k.view(np.uint16).ravel()) and np.array_equal(back[1].read(dtype=np.uint16), v.view(np.uint16).ravel())
    got = out.read(dtype=np.float16).reshape(qr.shape).astype(np.float64)
    for row in [0, 1, 15, 16, 31, 32, R - 1] + rng.integers(0, R, 60).tolist():
        a = max(0, row + 1 - window) if window else 0
        kk, vv = (x[a:row + 1, 0].astype(np.float64) for x in (k, v))
        x = qr[row].astype(np.float64) @ kk.T / 8
        size = (np.abs(qr[row].astype(np.float64)) @ np.abs(kk).T / 8).max(1, keepdims=True)
        p = np.exp(x - x.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        want = p @ vv
        floor = len(kk) * p.max(1, keepdims=True) * 2.0 ** -39 * np.abs(vv).max()
        assert (np.abs(got[row] - want) <= tolerance(want, p @ np.abs(vv), size, len(kk), 64) + floor).all(), row
