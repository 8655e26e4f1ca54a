"""Pieces of the tests of include/qw_attn.h: caches and steps on the device, and what the operators are, in 64 bits."""
import numpy as np

import qwental_amd as q

F16, Q8 = 1, 8


def unit_bytes(kind, D):
    return D * (64 if kind == F16 else 34)


def places(kind, D, values):
    """[16, D]: where value v of token t lies, in bytes from the start of its unit (include/qw_attn.h)."""
    t, v = np.arange(16)[:, None], np.arange(D)[None, :]
    if kind == F16:
        return 32 * D + 2 * np.ravel_multi_index((v // 32, t // 4, v % 32, t % 4), (D // 32, 4, 32, 4)) if values else 2 * np.ravel_multi_index((v // 8, t, v % 8), (D // 8, 16, 8))
    if values:
        return 17 * D + np.ravel_multi_index((v // 64, t // 4, v % 32 // 2, v % 64 // 32, v % 2, t % 4), (D // 64, 4, 16, 2, 2, 4))
    return np.ravel_multi_index((v // 64, v % 32 // 8, t, v % 64 // 32, v % 8), (D // 64, 4, 16, 2, 8))


def scale_places(D, values):
    """[16, D / 32]: where a token's scales lie, in bytes."""
    t, b = np.arange(16)[:, None], np.arange(D // 32)[None, :]
    return (33 if values else 16) * D + 2 * np.ravel_multi_index((t // 4, b, t % 4), (4, D // 32, 4))


def quantised(x):
    """Codes and scales of x [..., D] binary16: 64-bit arithmetic, one rounding of the scale."""
    b = x.astype(np.float64).reshape(*x.shape[:-1], -1, 32)
    top = np.abs(b).max(-1)
    with np.errstate(invalid="ignore"):
        d = np.minimum(top / 127, 515.5).astype(np.float16)  # 127 * 516 is beyond binary16
        d = np.where(np.isfinite(top), d, np.float16(np.nan))
        c = np.where((d > 0)[..., None], np.rint(b / np.where(d > 0, d, 1).astype(np.float64)[..., None]), 0)
    return np.clip(c, -127, 127).astype(np.int8).reshape(x.shape), d


class Cache:
    """Pages of a cache as bytes on the host, [pages, heads, units, unit bytes], the same order as on the device."""

    def __init__(self, kind, heads, D, page, pages, rng=None, fill=None):
        self.kind, self.heads, self.D, self.page, self.pages = kind, heads, D, page, pages
        shape = (pages, heads, page // 16, unit_bytes(kind, D))
        self.raw = np.zeros(shape, np.uint8) if rng is None else rng.integers(0, 256, shape, dtype=np.uint8)
        if fill is not None:
            self.raw.view(np.uint16)[:] = fill

    def put(self, table, slot, token, k, v):
        """k, v [heads, D] binary16 as token `token` of the slot."""
        pg, u, t = table[slot, token // self.page], token % self.page // 16, token % 16
        for values, x in ((False, k), (True, v)):
            at = places(self.kind, self.D, values)[t]
            unit = self.raw[pg, :, u]
            if self.kind == F16:
                unit[:, at], unit[:, at + 1] = x.view(np.uint8)[:, 0::2], x.view(np.uint8)[:, 1::2]
                continue
            c, d = quantised(x)
            s = scale_places(self.D, values)[t]
            unit[:, at] = c.view(np.uint8)
            unit[:, s], unit[:, s + 1] = d.view(np.uint8)[:, 0::2], d.view(np.uint8)[:, 1::2]

    def get(self, table, slot, tokens):
        """K and V [tokens, heads, D] in 64 bits."""
        out = []
        tokens = np.asarray(tokens)
        unit = self.raw[table[slot, tokens // self.page], :, tokens % self.page // 16]  # [T, heads, bytes]
        for values in (False, True):
            at = places(self.kind, self.D, values)[tokens % 16][:, None]
            take = lambda a: np.take_along_axis(unit, np.broadcast_to(a, unit.shape[:2] + a.shape[2:]), 2)  # noqa: E731
            halves = lambda a: np.ascontiguousarray(np.stack([take(a), take(a + 1)], -1)).view(np.float16)[..., 0].astype(np.float64)  # noqa: E731
            if self.kind == F16:
                out.append(halves(at))
                continue
            d = halves(scale_places(self.D, values)[tokens % 16][:, None])
            with np.errstate(invalid="ignore"):
                out.append(take(at).view(np.int8).astype(np.float64) * np.repeat(d, 32, -1))
        return out


class Step:
    """Rows and tokens of some slots, with a page table in which any page may follow any other."""

    def __init__(self, rng, n, length, page, spare=2, rows=None, pages=None):
        self.n, self.len = np.asarray(n, np.int64), np.asarray(length, np.int64)
        self.first = np.concatenate([[0], np.cumsum(self.n)])
        self.rows = int(self.first[-1]) if rows is None else rows
        need = -(-self.len // page)
        self.max_pages = max(1, int(need.max()))
        self.pages = int(need.sum()) + spare if pages is None else pages
        order = rng.permutation(self.pages)
        self.table = np.full((len(n), self.max_pages), 0xffffffff, np.uint32)  # what no token needs is no page
        at = 0
        for i, m in enumerate(need):
            self.table[i, :m] = order[at:at + m]
            at += m

    def rows_of(self):
        """(row, slot, token) of every row that belongs to a slot."""
        return [(self.first[i] + j, i, int(self.len[i] - self.n[i] + j)) for i in range(len(self.n)) for j in range(int(self.n[i]))]

    def device(self, gpu):
        self.bufs = [gpu.buf_from(a.astype(np.uint32), device_only=True) for a in (self.first, self.len, self.table)]
        return q.KvStep(len(self.n), self.rows, self.max_pages, *self.bufs)


def turned(x, pos, freq, pairs, adjacent):
    """x [rows, heads, D] binary16 by positions [rows, axes]; 64 bits, one rounding."""
    half = len(freq)
    if not half:
        return x
    axis = np.repeat(np.arange(len(pairs)), pairs)
    angle = pos.astype(np.float64)[:, axis] * freq
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    y = x.copy()
    i = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if adjacent else (slice(0, half), slice(half, 2 * half))
    a, b = x[..., i[0]].astype(np.float64), x[..., i[1]].astype(np.float64)
    y[..., i[0]], y[..., i[1]] = (a * c - b * s).astype(np.float16), (b * c + a * s).astype(np.float16)
    return y


def attention(cache, step, query, scale, window=0, dead=()):
    """out [rows, q heads, D] in 64 bits, and how far a result may be off: see tolerance(). Rows of no slot: NaN. dead: page numbers that are none."""
    R, Hq, D = query.shape
    out, tol = np.full(query.shape, np.nan), np.zeros(query.shape)
    G = Hq // cache.heads
    for row, slot, token in step.rows_of():
        a = max(0, token + 1 - window) if window else 0
        seen = [t for t in range(a, token + 1) if step.table[slot, t // cache.page] not in dead]
        out[row] = 0
        if not seen:
            continue
        k, v = cache.get(step.table, slot, seen)
        qr = query[row].astype(np.float64).reshape(cache.heads, G, D)
        s = np.einsum("hgd,thd->hgt", qr, k) * scale
        size = (np.einsum("hgd,thd->hgt", np.abs(qr), np.abs(k)) * scale).max(-1, keepdims=True)
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        out[row] = np.einsum("hgt,thd->hgd", p, v).reshape(Hq, D)
        floor = len(seen) * p.max(-1, keepdims=True) * 2.0 ** -39 * np.abs(v).max()
        tol[row] = (tolerance(out[row], np.einsum("hgt,thd->hgd", p, np.abs(v)), size, len(seen), D) + floor).reshape(Hq, D)
    return out, tol


def tolerance(o, weight, size, T, D):
    """The result is rounded to binary16 once: half a step, 2^-11 of it, or 2^-25 where binary16 steps are 2^-24. A score is a sum of D products in binary32 (2^-24 a step, D steps at
    most, of at most `size` = scale * sum |q k|), times a scale rounded to 24 bits and log2(e) (two more steps), brought to its weight by a subtraction and an exponential
    (another two steps of the score's size, 2^-22 for the exponential): relative error e of a weight, which enters numerator and denominator. The weights of the second product
    are held in 21 bits, and the product of their last ten with a value's last seven, 2^-21 of the whole at most, is left out; its sums over T tokens run in tiles of 16, each lane's over T / 4 of them at most: T / 4 + 8 steps of 2^-24 of sum p |v|, as do those of the
    denominator. `weight` = sum p |v|. (The caller adds what the smallest weights lose: half of binary16's last step, 2^-25, where the largest weight is 2^14, each times a value.)"""
    e = (D + 6) * 2.0 ** -24 * size + 2.0 ** -22
    return 2.0 ** -11 * np.abs(o.reshape(weight.shape)) + 2.0 ** -25 + weight * (2 * e + 2.0 ** -20 + 2 * (T / 4 + 8) * 2.0 ** -24)
