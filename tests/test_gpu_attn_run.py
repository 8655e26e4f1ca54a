"""The attention half of a decode step as programs use it (include/qw_attn.h): between the projections in one batch, on a stream of the caller's over
its own tensors, captured and replayed while the slots grow, over large caches and steps of many slots and rows."""
import numpy as np
import pytest
import torch

import qwental_amd as q
from attn_helpers import F16, Q8, Cache, Step, attention, turned, unit_bytes
from helpers import maxrel
from qwental_amd import synth
from test_gpu_attn import Device, check, filled, rows, same
from test_gpu_sample import ROW, drawn, model_like

pytestmark = pytest.mark.gpu


@pytest.fixture
def dev(gpu):
    d = Device(gpu)
    yield d
    for b in d.all:
        b.free()


# ---------------------------------------------------------------- steps of many slots and rows
@pytest.mark.parametrize("kind,H,G,D,n,length,window", [
    (Q8, 4, 1, 64, [1] * 256, [1 + i * 37 % 60 for i in range(253)] + [1500, 800, 1100], 0),  # the most slots there are, and more pairs than workgroups
    (F16, 8, 2, 64, [i % 3 for i in range(100)], [2 + i * 7 % 40 for i in range(100)], 0),      # slots without rows between them
    (F16, 2, 4, 128, [300, 5, 0, 77], [300, 700, 9, 100], 0),
    (Q8, 2, 4, 128, [300, 5, 0, 77], [300, 700, 9, 100], 50),
    (Q8, 8, 8, 64, [600, 400], [600, 450], 0),  # pairs of 1 to 19 tiles, more than workgroups
    (F16, 1, 3, 256, [65, 1], [2000, 2500], 0),
    (Q8, 1, 24, 256, [1, 2, 1], [2000, 2, 700], 0),  # two blocks of query heads in a row
])
def test_many_slots_and_rows(gpu, dev, kind, H, G, D, n, length, window):
    rng = np.random.default_rng(len(n) + D)
    check(dev, gpu, rng, kind, H, H * G, D, 16, Step(rng, n, length, 16), window=window)


@pytest.mark.parametrize("kind", [F16, Q8])
def test_slots_that_share_pages(gpu, dev, kind):
    """A prefix's pages in several slots' tables, and one page in two places of one table."""
    rng = np.random.default_rng(5)
    s = Step(rng, [1, 1, 2], [70, 70, 70], 32)
    s.table[1, :2] = s.table[0, :2]
    c = filled(rng, kind, 2, 64, 32, s)
    s.table[2, 1] = s.table[2, 0]
    check(dev, gpu, rng, kind, 2, 8, 64, 32, s, c=c)


# ---------------------------------------------------------------- offsets that pass 32 bits
@pytest.mark.parametrize("kind", [F16, Q8])
def test_a_cache_of_more_than_four_gigabytes(gpu, dev, kind):
    rng = np.random.default_rng(3)
    H, D, page = 8, 128, 256
    s = Step(rng, [1, 3], [500, 300], page, spare=0)
    page_bytes = H * page // 16 * unit_bytes(kind, D)
    pages = (5 << 30) // page_bytes + 1
    far = np.array([pages - 1, 3, pages - 2, pages // 2 + 1], np.uint32)[:s.pages]  # where the pages of the small cache lie in the large one
    c = Cache(kind, H, D, page, s.pages, rng=rng)
    k, v, qr = rows(rng, s.rows, H, D), rows(rng, s.rows, H, D), rows(rng, s.rows, 4 * H, D)
    for i, m in enumerate(s.len):
        for t in range(int(m)):
            c.put(s.table, i, t, *rng.standard_normal((2, H, D)).astype(np.float16))
    buf = dev.new(q.kv_bytes(gpu.L, kind, H, D, page, pages))
    assert buf.size > 5 << 30
    for p in range(s.pages):
        buf.fill(c.raw[p], offset=int(far[p]) * page_bytes)
    st = dev.step(s)
    s.bufs[2].fill(np.where(s.table < s.pages, far[np.minimum(s.table, s.pages - 1)], s.table).astype(np.uint32))
    kc = q.KvCache(buf, kind, H, D, page, pages)
    out, back, ws = dev.new(qr.nbytes), [dev.new(k.nbytes) for _ in range(2)], dev.new(q.attn_ws_bytes(gpu, D))
    qb = dev.up(qr)
    dev.run(q.KvWrite(kc, st, 4 * H, qb, qb, dev.up(k), dev.up(v)), q.KvRead(kc, st, *back), q.Attn(kc, st, 4 * H, qb, out, ws))
    for row, slot, token in s.rows_of():
        c.put(s.table, slot, token, k[row], v[row])
    for p in range(s.pages):
        assert np.array_equal(buf.read(page_bytes, offset=int(far[p]) * page_bytes), c.raw[p].ravel())
    for row, slot, token in s.rows_of():
        for got, want in zip(back, c.get(s.table, slot, [token])):
            assert np.array_equal(got.read(dtype=np.float16).reshape(k.shape)[row], want[0].astype(np.float16))
    want, tol = attention(c, s, qr, D ** -0.5)
    assert (np.abs(out.read(dtype=np.float16).reshape(qr.shape) - want) <= tol).all()


def test_logits_far_apart(gpu, dev):
    rng = np.random.default_rng(9)
    V, stride = 5000, (1 << 30) + 8
    logits = model_like(rng, 2, V)
    big = dev.new((stride + V) * 4)
    for i in range(2):
        big.fill(logits[i], offset=i * stride * 4)
    ids, ws = dev.new(8), dev.new(q.sample_ws_bytes(gpu, 2, V))
    p = np.array([(0.0, 1.0, 0.0, 0), (0.8, 0.9, 0.0, 50)], ROW)
    dev.run(q.Sample(2, V, big, dev.up(p), dev.up(np.array([0.5, 0.25], np.float32)), ids, None, ws, stride=stride))
    want = [drawn(logits[i], p[i], (0.5, 0.25)[i]) for i in range(2)]
    assert want[1][2] > 2.0 ** -20 and ids.read(dtype=np.uint32).tolist() == [w[0] for w in want]


# ---------------------------------------------------------------- a model's steps
@pytest.mark.parametrize("kind", [F16, Q8])
def test_steps_of_a_model(gpu, oracle, dev, kind):
    """Two layers' projections, cache, attention and output projection and the vocabulary's product with a token at its end, each step one batch: a prompt of eleven rows in two slots, then
    steps of a row a slot, the token drawn fed back. Every stage against its definition, from what the stage before it left."""
    rng = np.random.default_rng(kind)
    K, H, G, D, V, page, layers = 2048, 2, 8, 128, 3000, 32, 2
    Hq, Ns = H * G, [H * G * D, H * D, H * D]
    path = q.Path(gpu, K, 512, 16, 4, 16, device_scratch=True)
    embed = synth.activations(rng, V, K)
    W = [[synth.matrix(rng, f, n, K) for f, n in zip((14, 12, 1), Ns)] + [synth.matrix(rng, 14, K, Hq * D)] for _ in range(layers)]
    Wv = synth.matrix(rng, 14, V, K)
    wb = [[q.Tensor(dev.up(w), f) for w, f in zip(ws, (14, 12, 1, 14))] for ws in W]
    wv = q.Tensor(dev.up(Wv), 14)
    n, length = [8, 3], [8, 3]
    tokens = rng.integers(0, V, 11)
    s = Step(rng, [1, 1], [40, 33], page)  # pages for all that comes
    caches = [Cache(kind, H, D, page, s.pages, rng=rng) for _ in range(layers)]
    kcs = [dev.cache(c) for c in caches]
    bufs = {name: dev.new(size) for name, size in (("x", 16 * K * 2), ("q", 16 * Hq * D * 2), ("k", 16 * H * D * 2), ("v", 16 * H * D * 2), ("o", 16 * Hq * D * 2), ("h", 16 * K * 2), ("h2", 16 * K * 2), ("logits", 16 * V * 4), ("ids", 64), ("probs", 64))}
    pos, freq = dev.new(16 * 4), 10000.0 ** (-np.arange(D // 2) / (D // 2))
    fb, table, aws, sws = dev.up(freq), dev.up(s.table), dev.new(q.attn_ws_bytes(gpu, D)), dev.new(q.sample_ws_bytes(gpu, 16, V))
    first, lens, u, params = dev.new(12), dev.new(8), dev.new(64), dev.new(16 * 16)
    for step in range(4):
        R = sum(n)
        at = np.concatenate([length[i] - n[i] + np.arange(n[i]) for i in range(2)]).astype(np.int32)
        draws = rng.random(R).astype(np.float32)
        rules = np.array([(0.0 if i % 2 else 0.9, 0.95, 0.0, 40) for i in range(R)], ROW)
        for buf, a in ((bufs["x"], embed[tokens]), (pos, at), (first, np.cumsum([0] + n).astype(np.uint32)), (lens, np.array(length, np.uint32)), (u, draws), (params, rules)):
            buf.fill(a)
        st = q.KvStep(2, R, s.max_pages, first, lens, table)
        seen = []
        src = bufs["x"]
        for layer in range(layers):
            b = gpu.batch()
            dst = bufs["h" if layer == 0 else "h2"]
            path.qmv_ggm(b, wb[layer][:3], Ns, K, src, [bufs[c] for c in "qkv"], R, fout=False)
            b.end()
            raw = [bufs[c].read(R * w * 2, dtype=np.float16).reshape(R, -1, D) for c, w in zip("qkv", Ns)]
            b = gpu.batch()
            path.qmv_ggm(b, wb[layer][:3], Ns, K, src, [bufs[c] for c in "qkv"], R, fout=False)
            q.KvWrite(kcs[layer], st, Hq, bufs["q"], bufs["q"], bufs["k"], bufs["v"], q.Rope(D, [D // 2], fb, pos))(b)
            q.Attn(kcs[layer], st, Hq, bufs["q"], bufs["o"], aws)(b)
            path.qmv_gg(b, wb[layer][3], K, Hq * D, bufs["o"], dst, R, fout=False)
            if layer == layers - 1:
                path.qmv_gg(b, wv, V, K, dst, bufs["logits"], R)
                q.Sample(R, V, bufs["logits"], params, u, bufs["ids"], bufs["probs"], sws)(b)
            b.end()
            seen.append((raw, [bufs[c].read(R * w * 2, dtype=np.float16).reshape(R, -1, D) for c, w in (("q", Ns[0]), ("o", Ns[0]))], src.read(R * K * 2, dtype=np.float16).reshape(R, K), dst.read(R * K * 2, dtype=np.float16).reshape(R, K)))
            src = dst
        now = Step.__new__(Step)
        now.n, now.len, now.first, now.rows, now.table = np.array(n), np.array(length), np.cumsum([0] + n), R, s.table
        for layer, (raw, (qt, o), x, y) in enumerate(seen):
            c = caches[layer]
            for w, f, got in zip(W[layer], (14, 12, 1), raw):
                assert maxrel(got.reshape(R, -1).astype(np.float64), oracle.qmv(f, w, got.shape[1] * D, K, x, f64=True)) <= 2e-3
            same(qt, turned(raw[0], at[:, None], freq, [D // 2], False), True)
            kt = turned(raw[1], at[:, None], freq, [D // 2], False)
            for row, slot, token in now.rows_of():
                c.put(now.table, slot, token, kt[row], raw[2][row])
            have = kcs[layer].keep.read().reshape(c.raw.shape)
            assert (have != c.raw).mean() <= 1 / 500  # (keys a step of binary16 or a code off, as in same())
            c.raw = have
            want, tol = attention(c, now, qt, D ** -0.5)
            assert (np.abs(o.astype(np.float64) - want) <= tol).all()
            assert maxrel(y.astype(np.float64), oracle.qmv(14, W[layer][3], K, Hq * D, o.reshape(R, -1), f64=True)) <= 2e-3
        logits = bufs["logits"].read(R * V * 4, dtype=np.float32).reshape(R, V)
        ids = bufs["ids"].read(R * 4, dtype=np.uint32)
        for i in range(R):
            want, _, near, _ = drawn(logits[i], rules[i], float(draws[i]))
            assert near < 2.0 ** -20 or ids[i] == want
        tokens = ids[np.cumsum(n) - 1].astype(np.int64)
        n, length = [1, 1], [m + 1 for m in length]
    path.close()


@pytest.mark.parametrize("kind", [F16, Q8])
def test_buffers_with_a_host_side(gpu, dev, kind):
    """Everything but the cache and the workspaces in buffers that the host sees; written through their views, read there when the batch has ended."""
    rng = np.random.default_rng(70 + kind)
    H, G, D, page, V = 2, 4, 64, 32, 700
    s = Step(rng, [2, 1], [40, 7], page, rows=5)  # two rows of no slot
    c = filled(rng, kind, H, D, page, s)
    kc = dev.cache(c)
    keep = []

    def host(a):
        keep.append(gpu.buf(a.nbytes))
        keep[-1].fill(a)
        return keep[-1]

    first, lens, table = (host(a.astype(np.uint32)) for a in (s.first, s.len, s.table))
    st = q.KvStep(2, 5, s.max_pages, first, lens, table)
    shapes = [(5, H * G, D), (5, H, D), (5, H, D)]
    data = [rows(rng, *sh) for sh in shapes]
    qb, kb, vb = (host(a) for a in data)
    out, k2, v2, ids, probs = (host(np.full(n, 0x1234, np.uint16)) for n in (5 * H * G * D, 5 * H * D, 5 * H * D, 10, 10))
    logits, params, u = host(model_like(rng, 5, V)), host(np.array([(0.8, 0.9, 0.0, 30)] * 5, ROW)), host(rng.random(5).astype(np.float32))
    ws, sws = dev.new(q.attn_ws_bytes(gpu, D)), dev.new(q.sample_ws_bytes(gpu, 5, V))
    for step in range(3):
        b = gpu.batch()
        q.KvWrite(kc, st, 0, None, None, kb, vb)(b)
        q.KvRead(kc, st, k2, v2)(b)
        q.Attn(kc, st, H * G, qb, out, ws)(b)
        q.Sample(5, V, logits, params, u, ids, probs, sws)(b)
        b.end()
        for row, slot, token in s.rows_of():
            c.put(s.table, slot, token, data[1][row], data[2][row])
            for got, want in zip((k2, v2), c.get(s.table, slot, [token])):
                assert np.array_equal(got.view(np.float16).reshape(5, H, D)[row], want[0].astype(np.float16))
        want, tol = attention(c, s, data[0], D ** -0.5)
        got = out.view(np.float16).reshape(5, H * G, D)
        assert (np.abs(got[:3] - want[:3]) <= tol[:3]).all() and (out.view(np.uint16).reshape(5, -1)[3:] == 0x1234).all() and (k2.view(np.uint16).reshape(5, -1)[3:] == 0x1234).all()
        for i in range(5):
            token, p, near, _ = drawn(logits.view(np.float32).reshape(5, V)[i], params.view(ROW)[i], float(u.view(np.float32)[i]))
            assert near < 2.0 ** -20 or (ids.view(np.uint32)[i] == token and abs(probs.view(np.float32)[i] - p) < 1e-5)
        s.len = s.len + 1  # the next step, through the shadows
        lens.fill(s.len.astype(np.uint32))
        data = [rows(rng, *sh) for sh in shapes]
        for buf, a in zip((qb, kb, vb), data):
            buf.fill(a)
        logits.fill(model_like(rng, 5, V))
    for b in keep:
        b.free()


# ---------------------------------------------------------------- a stream and tensors of the caller's
class Torch:
    """A step of a captured or eager program: cache, rows, tokens, all torch's."""

    def __init__(self, gpu, rng, kind, n, length, room, H=2, G=4, D=128, page=32, V=2000):
        self.gpu, self.kind, self.H, self.G, self.D, self.page, self.V = gpu, kind, H, G, D, page, V
        self.s = Step(rng, n, room, page)
        self.s.len = np.array(length)
        self.c = Cache(kind, H, D, page, self.s.pages, fill=0xffff)
        for i, m in enumerate(length):
            for t in range(m):
                self.c.put(self.s.table, i, t, *rng.standard_normal((2, H, D)).astype(np.float16))
        up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        R = self.s.rows
        self.raw = up(self.c.raw)
        self.first, self.len, self.table = (up(a.astype(np.int32)) for a in (self.s.first, self.s.len, self.s.table.view(np.int32)))
        self.q, self.k, self.v = (torch.zeros(R, h, D, dtype=torch.float16, device="cuda") for h in (H * G, H, H))
        self.qt, self.out = torch.zeros_like(self.q), torch.zeros_like(self.q)
        self.pos, self.freq = torch.zeros(R, 1, dtype=torch.int32, device="cuda"), up(10000.0 ** (-np.arange(D // 2) / (D // 2)))
        self.logits, self.u = torch.zeros(R, V, device="cuda"), torch.zeros(R, device="cuda")
        self.params = up(np.array([(0.8, 0.9, 0.0, 60)] * R, ROW).view(np.uint8))
        self.ids, self.probs = torch.zeros(R, dtype=torch.int32, device="cuda"), torch.zeros(R, device="cuda")
        self.ws = torch.zeros(q.attn_ws_bytes(gpu, D), dtype=torch.uint8, device="cuda")
        self.sws = torch.zeros(q.sample_ws_bytes(gpu, R, V), dtype=torch.uint8, device="cuda")
        view = lambda t: gpu.view(t.data_ptr(), t.numel() * t.element_size())  # noqa: E731
        cache, step = q.KvCache(view(self.raw), kind, H, D, page, self.s.pages), q.KvStep(len(n), R, self.s.max_pages, view(self.first), view(self.len), view(self.table))
        self.calls = [q.KvWrite(cache, step, H * G, view(self.q), view(self.qt), view(self.k), view(self.v), q.Rope(D, [D // 2], view(self.freq), view(self.pos))),
                      q.Attn(cache, step, H * G, view(self.qt), view(self.out), view(self.ws)), q.Sample(R, V, view(self.logits), view(self.params), view(self.u), view(self.ids), view(self.probs), view(self.sws))]

    def feed(self, rng):
        """New rows: every slot a token longer."""
        self.s.len = self.s.len + 1
        self.len.copy_(torch.from_numpy(self.s.len.astype(np.int32)))
        for t in (self.q, self.k, self.v):
            t.copy_(torch.from_numpy(rng.standard_normal(t.shape).astype(np.float16)))
        at = np.zeros((self.s.rows, 1), np.int32)
        for row, slot, token in self.s.rows_of():
            at[row] = token
        self.at = at
        self.pos.copy_(torch.from_numpy(at))
        self.logits.copy_(torch.from_numpy(model_like(rng, *self.logits.shape)))
        self.u.copy_(torch.from_numpy(rng.random(self.s.rows).astype(np.float32)))
        for t in (self.qt, self.out, self.probs):
            t.fill_(float("nan"))
        self.ids.fill_(-7)

    def run(self, stream):
        with self.gpu.stream(stream) as b:
            for c in self.calls:
                c(b)

    def verify(self):
        freq, qh, kh = self.freq.cpu().numpy(), self.q.cpu().numpy(), self.k.cpu().numpy()
        qt = self.qt.cpu().numpy()
        same(qt, turned(qh, self.at, freq, [self.D // 2], False), True)
        kt, v = turned(kh, self.at, freq, [self.D // 2], False), self.v.cpu().numpy()
        for row, slot, token in self.s.rows_of():
            self.c.put(self.s.table, slot, token, kt[row], v[row])
        have = self.raw.cpu().numpy()
        assert (have != self.c.raw).mean() <= 1 / 500
        self.c.raw = have
        want, tol = attention(self.c, self.s, qt, self.D ** -0.5)
        assert (np.abs(self.out.cpu().numpy() - want) <= tol).all()
        logits, u, ids, params = self.logits.cpu().numpy(), self.u.cpu().numpy(), self.ids.cpu().numpy(), np.array([(0.8, 0.9, 0.0, 60)], ROW)[0]
        for i in range(self.s.rows):
            token, _, near, _ = drawn(logits[i], params, float(u[i]))
            assert near < 2.0 ** -20 or ids[i] == token


@pytest.mark.parametrize("kind", [F16, Q8])
def test_on_the_callers_stream(gpu, kind):
    rng = np.random.default_rng(40 + kind)
    t = Torch(gpu, rng, kind, [1, 2, 1], [5, 30, 70], [20, 50, 90])
    side = torch.cuda.Stream()
    for stream in (None, side, side, None):
        t.feed(rng)
        if stream is None:
            t.run(torch.cuda.current_stream().cuda_stream)
        else:
            side.wait_stream(torch.cuda.current_stream())
            t.run(side.cuda_stream)
            torch.cuda.current_stream().wait_stream(side)
        t.verify()


@pytest.mark.parametrize("kind", [F16, Q8])
def test_captured_and_replayed_while_the_slots_grow(gpu, kind):
    """Two graphs with workspaces of their own, replayed side by side; eager calls and other work between the replays. Pages and shares of the work change under them."""
    rng = np.random.default_rng(50 + kind)
    ts = [Torch(gpu, rng, kind, [1, 2, 1], [5, 30, 130], [60, 80, 300]), Torch(gpu, rng, kind, [1] * 5, [1, 2, 31, 32, 33], [20, 20, 90, 40, 200])]
    streams, graphs = [torch.cuda.Stream() for _ in ts], []
    for t in ts:
        t.feed(rng)
        t.run(torch.cuda.current_stream().cuda_stream)  # eagerly first
        t.verify()
    for t, stream in zip(ts, streams):
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            t.run(torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    for step in range(6):
        for t in ts:
            t.feed(rng)
        torch.cuda.synchronize()
        if step == 3:  # an eager step between
            for t in ts:
                t.run(torch.cuda.current_stream().cuda_stream)
        else:
            for g, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    g.replay()
        torch.cuda.synchronize()
        for t in ts:
            t.verify()
        (torch.randn(512, 512, device="cuda") @ torch.randn(512, 512, device="cuda")).sum().item()


def test_recorder_is_given_back(gpu, dev):
    rng = np.random.default_rng(8)
    t = Torch(gpu, rng, F16, [1], [3], [10])
    t.feed(rng)
    stream = torch.cuda.current_stream().cuda_stream
    b = gpu.stream(stream)
    with pytest.raises(RuntimeError, match="in use"):
        gpu.stream(stream)
    host = gpu.buf(t.q.numel() * 2)
    with pytest.raises(RuntimeError, match="host side"):
        q.Attn(q.KvCache(dev.up(t.c.raw), F16, 2, 128, 32, t.s.pages), dev.step(t.s), 8, host, dev.new(host.size), dev.new(q.attn_ws_bytes(gpu, 128)))(b)
    with pytest.raises(RuntimeError):
        b.end()
    host.free()
    with pytest.raises(ZeroDivisionError):
        with gpu.stream(stream) as b:
            t.calls[0](b)
            1 // 0
    gpu.stream(stream)  # (nobody holds it)
    t.run(stream)
    t.verify()
    with pytest.raises(RuntimeError, match="not memory"):
        gpu.view(np.zeros(64).ctypes.data, 64)
    with pytest.raises(RuntimeError, match="beyond"):
        gpu.view(t.ws.data_ptr(), 1 << 40)


def test_captured_at_a_devices_first_use():
    """Nothing has to be called before a capture; views outlive the device."""
    rng = np.random.default_rng(60)
    g = q.Gpu()
    t = Torch(g, rng, Q8, [1, 1], [40, 3], [60, 20], D=192, H=1, V=9000)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        t.run(torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        t.feed(rng)
        graph.replay()
        torch.cuda.synchronize()
        t.verify()
    late = g.stream(None)
    g.close()
    with pytest.raises(RuntimeError, match="closed"):
        late.end()
