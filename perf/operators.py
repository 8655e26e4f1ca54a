"""The attention half of a decode step and the token at its end: rows of keys and values written into a paged cache (with rotary
positions, and quantised where the cache is Q8_0), read back out of it, attended to, and a token drawn from the vocabulary's logits.

A case is a dict of plain values; "kind" says which operator it calls:
  attn    queries of a step's rows over the pages of their slots: slot i has some rows (one, or a few drafts) and len[i] tokens
  kv      the rows' queries and keys turned by their positions, keys and values written behind what the slots hold, and read back
  read    the last tokens of the slots out of the cache as binary16 rows (a prefix that is moved or kept)
  sample  one token a row under temperature, top-k, top-p and min-p, from given random numbers

A cache is bytes in the library's documented order (include/qw_attn.h): pages x heads x units of 16 tokens, a unit holding, for D values a head,
  F16 (type 1):  K [D/8][16][8], V [D/32][4][32][4] binary16 (tokens four at a time innermost)
  Q8_0 (type 8): K [D/64][4][16][2][8] int8, K scales [4][D/32][4] binary16, V [D/64][4][16][2][2][4] int8, V scales [4][D/32][4]
The head counts and sizes are those of the projections in perf/cases.py (rows of 4096 and 512 values: 32 and 4 heads of 128 values, or 16
and 2 of 256), a few generic ones beside them."""
import math

import numpy as np
import torch

own = False

F16, Q8 = 1, 8


def listed():
    a = {"q_heads": 32, "kv_heads": 4, "dim": 128, "page": 64, "window": 0}
    b = {"q_heads": 16, "kv_heads": 2, "dim": 256, "page": 64, "window": 0}
    rot = {"rot": 128, "axes": 3}
    return [
        # the first tokens of one conversation: the smallest call, where latency counts
        {"name": "attn_one_q8", "kind": "attn", "type": Q8, "slots": 1, "rows": 1, "len": 700, "even": True, **b},
        # sixteen conversations of up to 4096 tokens, one token each: the ordinary step
        {"name": "attn_chat_f16", "kind": "attn", "type": F16, "slots": 16, "rows": 16, "len": 4096, "even": False, **a},
        # twelve conversations, some with drafts beside their last token
        {"name": "attn_drafts_q8", "kind": "attn", "type": Q8, "slots": 12, "rows": 45, "len": 6001, "even": False, **a},
        # one conversation over a whole document: the long axis has to be split
        {"name": "attn_long_q8", "kind": "attn", "type": Q8, "slots": 1, "rows": 1, "len": 131072, "even": True, **b},
        # a full server: sixty-four conversations of 8192 tokens
        {"name": "attn_full_f16", "kind": "attn", "type": F16, "slots": 64, "rows": 64, "len": 8192, "even": True, **a},
        # one token of one conversation into the cache, text positions
        {"name": "kv_one_f16", "kind": "kv", "type": F16, "slots": 1, "rows": 1, "len": 700, "even": True, **b, "rot": 64, "axes": 1},
        # the drafts' step, positions in time, height and width
        {"name": "kv_drafts_q8", "kind": "kv", "type": Q8, "slots": 12, "rows": 45, "len": 6001, "even": False, **a, **rot},
        # a prefill segment of 4096 tokens with an image in it
        {"name": "kv_prefill_q8", "kind": "kv", "type": Q8, "slots": 1, "rows": 4096, "len": 12001, "even": True, **a, **rot},
        # a short answer taken out of the cache
        {"name": "read_short_f16", "kind": "read", "type": F16, "slots": 1, "rows": 333, "len": 1500, "even": True, **b},
        # prefixes of four conversations moved out
        {"name": "read_prefix_q8", "kind": "read", "type": Q8, "slots": 4, "rows": 16384, "len": 8192, "even": False, **a},
        # one conversation's next token, the usual settings
        {"name": "sample_one", "kind": "sample", "rows": 1, "vocab": 131072, "mix": False},
        # sixteen conversations, each with settings of its own
        {"name": "sample_16", "kind": "sample", "rows": 16, "vocab": 131072, "mix": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("attn", "attn", "attn", "kv", "kv", "read", "sample", "sample"))
    if kind == "sample":
        return {"kind": kind, "rows": rng.randint(1, 16), "vocab": _log(rng, 1000, 131072), "mix": rng.random() < 0.7}
    dim = rng.choice((64, 128, 128, 128, 192, 256))
    kv_heads = rng.choice((1, 2, 4, 8))
    case = {"kind": kind, "type": rng.choice((F16, Q8)), "dim": dim, "kv_heads": kv_heads, "q_heads": kv_heads * rng.choice((1, 2, 4, 5, 8)), "page": rng.choice((16, 32, 64, 64, 256)), "even": rng.random() < 0.3}
    slots = _log(rng, 1, 32)
    most = 64 * 8192 * 4 * 128 // (slots * kv_heads * dim)  # tokens a slot that the largest listed case has
    if kind == "attn":
        rows = slots if rng.random() < 0.5 else slots + rng.randint(1, 4 * slots)
        length = max(8, min(_log(rng, 30, 100000), most, 131072))
        return {**case, "slots": slots, "rows": rows, "len": length, "window": rng.choice((0, 0, 0, 512, 1000))}
    rows = max(slots, min(_log(rng, 1, 4000), 4096 * 4 * 128 // (kv_heads * dim)))
    length = min(rows + rng.randint(0, 8000), max(rows, most))
    return {**case, "slots": slots, "rows": rows, "len": length, "window": 0, "rot": rng.choice((dim, dim, dim // 2, 0)), "axes": rng.choice((1, 3))} if kind == "kv" else {**case, "slots": slots, "rows": rows, "len": length, "window": 0}


def _shape(case):
    """Rows and tokens of each slot: they follow from the case, so that work() knows them."""
    r = np.random.default_rng([case["slots"], case["rows"], case["len"], case["dim"]])
    S, R, L = case["slots"], case["rows"], case["len"]
    n = np.full(S, R // S) if case["even"] or R == S else 1 + np.bincount(r.integers(0, S, R - S), minlength=S)
    n[0] += R - n.sum()
    length = np.full(S, L) if case["even"] else r.integers(max(1, L // 4), L + 1, S)
    return n.astype(np.int64), np.maximum(length, n).astype(np.int64)


def _unit(case):
    return case["dim"] * (64 if case["type"] == F16 else 34)


class State:
    """What a serving loop keeps: the cache, its page table, the step's rows, the results' memory."""


def _pack_q8(x):
    """x [..., D] binary16 -> codes [..., D] int8 and scales [..., D/32] binary16: d = max |x| / 127 of 32 values in binary16, codes round(x / d)."""
    b = x.float().unflatten(-1, (-1, 32))
    d = (b.abs().amax(-1) / 127).half()
    c = torch.where(d[..., None] > 0, torch.round(b / d.float()[..., None]), torch.zeros((), device=x.device)).clamp(-127, 127)
    return c.to(torch.int8).flatten(-2), d


def _units(k, v, kind):
    """k, v [N, 16, D] binary16 -> units [N, bytes] in the cache's order."""
    N, _, D = k.shape
    raw = lambda t: t.contiguous().view(torch.uint8).reshape(N, -1)  # noqa: E731
    if kind == F16:
        return torch.cat([raw(k.view(N, 16, D // 8, 8).permute(0, 2, 1, 3)), raw(v.view(N, 4, 4, D // 32, 32).permute(0, 3, 1, 4, 2))], 1)
    (kc, kd), (vc, vd) = _pack_q8(k), _pack_q8(v)
    scales = lambda d: raw(d.view(N, 4, 4, D // 32).permute(0, 1, 3, 2))  # noqa: E731
    kc = kc.view(N, 16, D // 64, 2, 4, 8).permute(0, 2, 4, 1, 3, 5)
    vc = vc.view(N, 4, 4, D // 64, 2, 16, 2).permute(0, 3, 1, 5, 4, 6, 2)
    return torch.cat([raw(kc), scales(kd), raw(vc), scales(vd)], 1)


def prepare(case, seed):
    s = State()
    s.case = case
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rnd = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    if case["kind"] == "sample":
        B, V = case["rows"], case["vocab"]
        s.logits = rnd(B, V) * 2.5
        s.logits += (torch.rand(B, V, generator=gen, device="cuda") < 30 / V) * (4 + 2 * rnd(B, V))  # the few that the model has in mind
        r = np.random.default_rng(seed)
        p = np.zeros((B, 4), np.float32)  # temperature, top-p, min-p, top-k (its bits)
        for i in range(B):
            mix = r.integers(0, 5) if case["mix"] else 1
            t, tp, mp, tk = ((1.0, 1.0, 0.0, 0), (0.7, 0.95, 0.0, 40), (1.2, 0.9, 0.0, 0), (0.9, 1.0, 0.05, 0), (0.0, 1.0, 0.0, 0))[mix]
            p[i] = t, tp, mp, 0
            p.view(np.uint32)[i, 3] = tk
        s.params = torch.from_numpy(p).cuda()
        s.u = torch.from_numpy(r.random(B, dtype=np.float32)).cuda()
        s.ids = torch.zeros(B, dtype=torch.int32, device="cuda")
        s.probs = torch.zeros(B, dtype=torch.float32, device="cuda")
        return s
    n, length = _shape(case)
    S, R, H, D, page = case["slots"], case["rows"], case["kv_heads"], case["dim"], case["page"]
    need = -(-length // page)
    s.max_pages = int(need.max()) + 1
    s.pages = int(need.sum()) + 3
    order = np.random.default_rng(seed).permutation(s.pages)
    table, at = np.zeros((S, s.max_pages), np.int32), 0
    for i in range(S):  # any page may follow any other
        table[i, : need[i]] = order[at: at + need[i]]
        at += need[i]
    s.table = torch.from_numpy(table).cuda()
    s.first = torch.from_numpy(np.concatenate([[0], np.cumsum(n)]).astype(np.int32)).cuda()
    s.len = torch.from_numpy(length.astype(np.int32)).cuda()
    # keys as projections give them: a few channels larger than the others; what lies behind a slot's last token is some other conversation's
    channel = 1 + 3 * (torch.rand(D, generator=gen, device="cuda") < 0.06)
    s.cache = torch.empty(s.pages, H, page // 16, _unit(case), dtype=torch.uint8, device="cuda")
    flat, step = s.cache.view(-1, _unit(case)), (1 << 26) // (16 * D)
    for a in range(0, len(flat), step):
        m = min(step, len(flat) - a)
        flat[a: a + m] = _units((rnd(m, 16, D) * channel).half(), rnd(m, 16, D).half(), case["type"])
    if case["kind"] == "attn":
        s.most = int(n.max())
        s.q = rnd(R, case["q_heads"], D).half()
        s.out = torch.zeros_like(s.q)
    else:
        s.k_back, s.v_back = (torch.zeros(R, H, D, dtype=torch.float16, device="cuda") for _ in range(2))
    if case["kind"] == "kv":
        s.q, s.k, s.v = rnd(R, case["q_heads"], D).half(), (rnd(R, H, D) * channel).half(), rnd(R, H, D).half()
        s.q_out = torch.zeros_like(s.q)
        half = case["rot"] // 2
        s.freq = torch.from_numpy(1e6 ** (-np.arange(half) / max(half, 1))).cuda()
        s.pairs = _pairs(case)
        slot = np.repeat(np.arange(S), n)
        pos = length[slot] - n[slot] + np.arange(R) - np.concatenate([[0], np.cumsum(n)])[slot]
        if case["axes"] == 3:  # some rows are an image's: one time, a grid of heights and widths
            img = np.arange(R) % 100 < 60
            pos = np.stack([np.where(img, pos // 100 * 100, pos), np.where(img, pos // 100 * 100 + pos % 60 // 10, pos), np.where(img, pos // 100 * 100 + pos % 10, pos)], 1)
        s.pos = torch.from_numpy(np.ascontiguousarray(pos.reshape(R, -1)).astype(np.int32)).cuda()
    return s


def _pairs(case):
    """Pairs of values that turn by each axis."""
    half = case["rot"] // 2
    return [half] if case["axes"] == 1 else [half - 2 * (half * 3 // 8), half * 3 // 8, half * 3 // 8]


# ---------------------------------------------------------------- the plain forms
def _values(raw, kind, D):
    """Units [..., bytes] -> K and V [..., 16, D] in 32 bits."""
    lead = raw.shape[:-1]
    n = len(lead)
    at = lambda a, b, t: raw[..., a:b].contiguous().view(t)  # noqa: E731
    back = lambda x, dims: x.permute(*range(n), *(n + d for d in dims)).reshape(*lead, 16, D)  # noqa: E731
    if kind == F16:
        k, v = at(0, 32 * D, torch.float16).float(), at(32 * D, 64 * D, torch.float16).float()
        return back(k.view(*lead, D // 8, 16, 8), (1, 0, 2)), back(v.view(*lead, D // 32, 4, 32, 4), (1, 3, 0, 2))
    k, v = at(0, 16 * D, torch.int8).float(), at(17 * D, 33 * D, torch.int8).float()
    scales = lambda a: back(at(a, a + D, torch.float16).float().view(*lead, 4, D // 32, 4)[..., None].expand(*lead, 4, D // 32, 4, 32), (0, 2, 1, 3))  # noqa: E731
    return (back(k.view(*lead, D // 64, 4, 16, 2, 8), (2, 0, 3, 1, 4)) * scales(16 * D),
            back(v.view(*lead, D // 64, 4, 16, 2, 2, 4), (1, 5, 0, 3, 2, 4)) * scales(33 * D))


def _rows_of(s):
    """Slot and token of every row."""
    R = s.case["rows"]
    r = torch.arange(R, device="cuda")
    slot = torch.searchsorted(s.first[1:].long(), r, right=True)
    return r, slot, s.len.long()[slot] - s.first.long()[slot + 1] + r


def _attn(s):
    c = s.case
    S, R, H, D, page, G = c["slots"], c["rows"], c["kv_heads"], c["dim"], c["page"], c["q_heads"] // c["kv_heads"]
    r, slot, token = _rows_of(s)
    j = r - s.first.long()[slot]
    k, v = _values(s.cache[s.table.long()], c["type"], D)  # [S, pages, H, units, 16, D]
    flat = lambda x: x.permute(0, 2, 1, 3, 4, 5).reshape(S, H, -1, D)  # noqa: E731
    k, v = flat(k), flat(v)
    n = s.most
    q = torch.zeros(S, n, H, G, D, device="cuda")
    q[slot, j] = s.q.float().view(R, H, G, D)
    score = torch.matmul(q.permute(0, 2, 1, 3, 4).reshape(S, H, n * G, D), k.transpose(2, 3).contiguous()).view(S, H, n, G, -1) * (1 / math.sqrt(D))
    last = torch.full((S, n), -1, dtype=torch.long, device="cuda")
    last[slot, j] = token
    key = torch.arange(k.shape[2], device="cuda")
    seen = key <= last[..., None]
    if c["window"]:
        seen &= key > last[..., None] - c["window"]
    score = torch.where(seen[:, None, :, None], score, float("-inf"))
    e = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-1e30))
    o = torch.matmul(e.view(S, H, n * G, -1), v).view(S, H, n, G, D) / e.sum(-1, keepdim=True).clamp(min=1e-30)
    s.out.copy_(o.permute(0, 2, 1, 3, 4)[slot, j].reshape(R, H * G, D))
    return {"out": s.out}


def _turn(s, x):
    """Angles, and what becomes an 8-bit code, in 64 bits; one rounding to binary16."""
    half = s.case["rot"] // 2
    if not half:
        return x
    axis = torch.repeat_interleave(torch.arange(len(s.pairs), device="cuda"), torch.tensor(s.pairs, device="cuda"), output_size=half)
    angle = (s.pos.double()[:, axis] * s.freq)[:, None]
    cos, sin = torch.cos(angle), torch.sin(angle)
    a, b, rest = x[..., :half].double(), x[..., half: 2 * half].double(), x[..., 2 * half:]
    return torch.cat([(a * cos - b * sin).half(), (b * cos + a * sin).half(), rest], -1)


def _write(s):
    c = s.case
    D, page = c["dim"], c["page"]
    s.q_out.copy_(_turn(s, s.q))
    _, slot, token = _rows_of(s)
    where = s.table.long()[slot, token // page]
    unit, t = token % page // 16, token % 16
    k, v = _turn(s, s.k), s.v
    r = [x[:, None, None] for x in (where, unit, t)]
    h, d = torch.arange(c["kv_heads"], device="cuda")[None, :, None], torch.arange(D, device="cuda")
    if c["type"] == F16:
        u = s.cache.view(torch.float16)
        u[r[0], h, r[1], (d // 8 * 16 + r[2]) * 8 + d % 8] = k
        u[r[0], h, r[1], 16 * D + (d // 32 * 4 + r[2] // 4) * 128 + d % 32 * 4 + r[2] % 4] = v
        return
    (kc, kd), (vc, vd) = _pack_q8(k), _pack_q8(v)
    b, u, w = torch.arange(D // 32, device="cuda"), s.cache.view(torch.int8), s.cache.view(torch.float16)
    u[r[0], h, r[1], ((d // 64 * 4 + d % 32 // 8) * 16 + r[2]) * 16 + d % 64 // 32 * 8 + d % 8] = kc
    u[r[0], h, r[1], 17 * D + ((d // 64 * 4 + r[2] // 4) * 16 + d % 32 // 2) * 16 + d % 64 // 32 * 8 + d % 2 * 4 + r[2] % 4] = vc
    at = (r[2] // 4 * (D // 32) + b) * 4 + r[2] % 4
    w[r[0], h, r[1], 8 * D + at] = kd
    w[r[0], h, r[1], 33 * D // 2 + at] = vd


def _read(s):
    c = s.case
    _, slot, token = _rows_of(s)
    units = s.cache[s.table.long()[slot, token // c["page"]], :, token % c["page"] // 16]  # [R, H, bytes]
    k, v = _values(units, c["type"], c["dim"])
    t = (token % 16)[:, None, None, None].expand(-1, c["kv_heads"], 1, c["dim"])
    s.k_back.copy_(k.gather(2, t)[:, :, 0])
    s.v_back.copy_(v.gather(2, t)[:, :, 0])
    return {"k": s.k_back, "v": s.v_back}


def _sample(s):
    """In 64 bits: a token at the border of a filter or of the draw is decided as the definition does."""
    V = s.case["vocab"]
    p = s.params.double()
    temp, top_p, min_p = p[:, 0:1], p[:, 1:2], p[:, 2:3]
    k = s.params.view(torch.int32)[:, 3:4].long()
    l, order = torch.sort(s.logits.double(), dim=1, descending=True, stable=True)  # equal logits: the lower token first
    w = torch.exp((l - l[:, :1]) / torch.where(temp > 0, temp, 1))
    rank = torch.arange(V, device="cuda")
    kept = rank < torch.where(temp > 0, torch.where(k > 0, k, V), 1)
    w = w * kept
    before = torch.cumsum(w, 1) - w
    kept &= (before < top_p * w.sum(1, keepdim=True)) | (top_p >= 1)
    kept &= w >= min_p
    w = torch.zeros_like(w).scatter_(1, order, w * kept)
    cum = torch.cumsum(w, 1)
    i = (cum <= s.u.double()[:, None] * cum[:, -1:]).sum(1).clamp(max=V - 1)
    s.ids.copy_(i)
    s.probs.copy_(w.gather(1, i[:, None])[:, 0] / cum[:, -1])
    return {"ids": s.ids, "probs": s.probs}


def run(s):
    if own:
        return _own(s)
    kind = s.case["kind"]
    if kind == "attn":
        return _attn(s)
    if kind == "sample":
        return _sample(s)
    if kind == "read":
        return _read(s)
    _write(s)
    return {"q": s.q_out, **_read(s)}


# ---------------------------------------------------------------- the library's calls
_gpu, _ws = None, {}


def _workspace(size):
    """One a size for the whole program, whose calls follow one another on one stream."""
    if size not in _ws:
        _ws[size] = _gpu.buf(size, device_only=True)
    return _ws[size]


def _own(s):
    """As a program with its tensors in torch calls the library: views of them made once, then a recorder on the current stream a step."""
    global _gpu
    import qwental_amd as lib
    if _gpu is None:
        _gpu = lib.Gpu()
    if not hasattr(s, "calls"):
        s.calls = _calls(lib, s)
    b = _gpu.stream(torch.cuda.current_stream().cuda_stream)
    for c in s.calls:
        c(b)
    b.end()
    return s.result


def _calls(lib, s):
    c = s.case
    view = lambda t: _gpu.view(t.data_ptr(), t.numel() * t.element_size())  # noqa: E731
    if c["kind"] == "sample":
        s.result = {"ids": s.ids, "probs": s.probs}
        ws = _workspace(lib.sample_ws_bytes(_gpu, c["rows"], c["vocab"]))
        return [lib.Sample(c["rows"], c["vocab"], view(s.logits), view(s.params), view(s.u), view(s.ids), view(s.probs), ws)]
    cache = lib.KvCache(view(s.cache), c["type"], c["kv_heads"], c["dim"], c["page"], s.pages)
    step = lib.KvStep(c["slots"], c["rows"], s.max_pages, view(s.first), view(s.len), view(s.table))
    if c["kind"] == "attn":
        s.result = {"out": s.out}
        ws = _workspace(lib.attn_ws_bytes(_gpu, c["dim"]))
        return [lib.Attn(cache, step, c["q_heads"], view(s.q), view(s.out), ws, window=c["window"])]
    s.result = {"k": s.k_back, "v": s.v_back}
    read = lib.KvRead(cache, step, view(s.k_back), view(s.v_back))
    if c["kind"] == "read":
        return [read]
    s.result["q"] = s.q_out
    rope = lib.Rope(c["rot"], s.pairs, view(s.freq), view(s.pos)) if c["rot"] else None
    return [lib.KvWrite(cache, step, c["q_heads"], view(s.q), view(s.q_out), view(s.k), view(s.v), rope), read]


# ---------------------------------------------------------------- work
def work(case):
    if case["kind"] == "sample":
        B, V = case["rows"], case["vocab"]
        return {"bytes": B * V * 4, "flops": 4 * B * V}
    n, length = _shape(case)
    R, H, D, Hq = case["rows"], case["kv_heads"], case["dim"], case["q_heads"]
    token = H * D * (4 if case["type"] == F16 else 2.125)  # bytes of one token's keys and values
    if case["kind"] == "read":
        return {"bytes": R * (token + H * D * 4), "flops": R * H * D * 2}
    if case["kind"] == "kv":
        return {"bytes": R * (4 * Hq * D + 2 * token + 8 * H * D), "flops": R * (Hq + H) * D * 6}
    w = case["window"] or int(length.max())
    read = np.minimum(length, w + n - 1)  # tokens that any of a slot's rows sees
    seen = sum(int(np.minimum(a - m + 1 + np.arange(m), w).sum()) for m, a in zip(n, length))
    return {"bytes": float(read.sum() * token + R * Hq * D * 4), "flops": float(4 * seen * Hq * D)}


# ---------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "sample":
        return _exact_sample(s)
    n, length = _shape(case)
    first = np.concatenate([[0], np.cumsum(n)])
    H, D, page, kind = case["kv_heads"], case["dim"], case["page"], case["type"]
    raw, table = s.cache, s.table.cpu().numpy()

    def tokens(i, a, b):
        """Tokens a .. b of slot i: K and V [b - a, H, D] in 64 bits, each value fetched from its place."""
        t = np.arange(a, b)
        unit = torch.from_numpy(table[i, t // page].astype(np.int64)).cuda(), torch.from_numpy(t % page // 16).cuda()
        u = raw[unit[0], :, unit[1]]  # [T, H, bytes]
        t, d = torch.from_numpy(t % 16).cuda()[:, None], torch.arange(D, device="cuda")
        pick = lambda x, at: torch.gather(x, 2, at[:, None].expand(-1, H, -1)).double()  # noqa: E731
        if kind == F16:
            x = u.view(torch.float16)
            return pick(x, d // 8 * 128 + t * 8 + d % 8), pick(x, 16 * D + d // 32 * 512 + t // 4 * 128 + d % 32 * 4 + t % 4)
        x, y = u.view(torch.int8), u.view(torch.float16)
        at = t // 4 * (D // 8) + d // 32 * 4 + t % 4
        k = pick(x, d // 64 * 1024 + d % 32 // 8 * 256 + t * 16 + d // 32 % 2 * 8 + d % 8) * pick(y, 8 * D + at)
        v = pick(x, 17 * D + d // 64 * 1024 + t // 4 * 256 + d % 32 // 2 * 16 + d // 32 % 2 * 8 + d % 2 * 4 + t % 4) * pick(y, 33 * D // 2 + at)
        return k, v

    if case["kind"] == "attn":
        out = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
        for i in range(case["slots"]):
            k, v = tokens(i, 0, int(length[i]))
            for j in range(int(n[i])):
                end = int(length[i] - n[i] + j + 1)
                a = max(0, end - case["window"]) if case["window"] else 0
                q = s.q[first[i] + j].double().view(H, -1, D)
                p = torch.softmax(torch.matmul(q, k[a:end].permute(1, 2, 0)) / math.sqrt(D), -1)
                out[first[i] + j] = torch.matmul(p, v[a:end].permute(1, 0, 2)).reshape(-1, D)
        return {"out": out}
    if case["kind"] == "read":
        got = [tokens(i, int(length[i] - n[i]), int(length[i])) for i in range(case["slots"])]
        return {"k": torch.cat([g[0] for g in got]), "v": torch.cat([g[1] for g in got])}
    half = case["rot"] // 2
    pos = s.pos.cpu().numpy().astype(np.float64)
    axis = np.repeat(np.arange(len(s.pairs)), s.pairs)
    z = np.exp(1j * pos[:, axis] * s.freq.cpu().numpy())[:, None]

    def turned(x):
        x = x.cpu().numpy()
        if not half:
            return x.astype(np.float64)
        y = (x[..., :half] + 1j * x[..., half: 2 * half].astype(np.float64)) * z
        return np.concatenate([y.real.astype(np.float16), y.imag.astype(np.float16), x[..., 2 * half:]], -1).astype(np.float64)

    def held(x):
        if kind == F16:
            return x
        b = x.reshape(*x.shape[:-1], -1, 32)
        d = (np.abs(b).max(-1, keepdims=True) / 127).astype(np.float16).astype(np.float64)
        return (np.clip(np.rint(b / np.where(d > 0, d, 1)), -127, 127) * d).reshape(x.shape)

    return {"q": turned(s.q), "k": held(turned(s.k)), "v": held(s.v.cpu().numpy().astype(np.float64))}


def _exact_sample(s):
    p, k = s.params.cpu().numpy().astype(np.float64), s.params.cpu().numpy().view(np.uint32)[:, 3]
    u, logits = s.u.cpu().numpy().astype(np.float64), s.logits.cpu().numpy().astype(np.float64)
    ids, probs = [], []
    for b, l in enumerate(logits):
        t, top_p, min_p = p[b, :3]
        if t == 0:
            ids.append(int(np.argmax(l)))
            probs.append(1.0)
            continue
        w = np.exp((l - l.max()) / t)
        order = np.lexsort((np.arange(len(l)), -l))
        order = order[: k[b]] if k[b] else order
        if top_p < 1:
            c = np.cumsum(w[order])
            m = int(np.searchsorted(c, top_p * c[-1])) + 1
        else:
            m = len(order)
        chosen = np.sort([i for i in order[:m] if w[i] >= min_p])
        c = np.cumsum(w[chosen])
        i = int(np.searchsorted(c, u[b] * c[-1], side="right"))
        ids.append(int(chosen[i]))
        probs.append(float(w[chosen[i]] / c[-1]))
    return {"ids": np.array(ids, np.int32), "probs": np.array(probs, np.float64)}
