"""The attention half of a decode step (include/qw_attn.h): a cache, a step's rows, and the calls over them. A call is an object made once, with
its buffers; applied to a batch (Gpu.batch or Gpu.stream) it records itself."""
import ctypes as C

from .gpu import QwBuf


class QwAt(C.Structure):
    _fields_ = [("buf", C.POINTER(QwBuf)), ("offset", C.c_size_t)]


class QwKv(C.Structure):
    _fields_ = [("at", QwAt)] + [(n, C.c_int) for n in ("type", "heads", "dim", "page", "pages")]


class QwKvStep(C.Structure):
    _fields_ = [(n, C.c_int) for n in ("slots", "rows", "max_pages")] + [(n, QwAt) for n in ("first", "len", "table")]


class QwKvRows(C.Structure):
    _fields_ = [("at", QwAt), ("stride", C.c_int)]


class QwRope(C.Structure):
    _fields_ = [("dims", C.c_int), ("axes", C.c_int), ("pairs", C.c_int * 3), ("adjacent", C.c_bool), ("freq", QwAt), ("pos", QwAt)]


def _at(x):
    """A buffer, or (buffer, byte offset)."""
    if x is None:
        return QwAt()
    buf, offset = x if isinstance(x, tuple) else (x, 0)
    return QwAt(C.pointer(buf.c), offset)


def kv_bytes(L, type, heads, dim, page, pages):
    return L.qw_kv_bytes(type, heads, dim, page, pages)


def attn_ws_bytes(gpu, dim):
    return gpu.L.qw_attn_ws_bytes(gpu.g, dim)


class KvCache:
    """A layer's keys and values in pages: buf holds qw_kv_bytes of device memory. type: 1 binary16, 8 Q8_0."""

    def __init__(self, buf, type, heads, dim, page, pages):
        self.keep, self.c = buf, QwKv(_at(buf), type, heads, dim, page, pages)


class KvStep:
    """The rows of a step: first [slots + 1], len [slots], table [slots][max_pages], all uint32 on the device."""

    def __init__(self, slots, rows, max_pages, first, len, table):
        self.keep, self.c = (first, len, table), QwKvStep(slots, rows, max_pages, _at(first), _at(len), _at(table))


class Rope:
    """dims values a head turn; pairs: how many pairs go by each axis (one axis or three); freq float64 [dims / 2], pos int32 [rows][axes]."""

    def __init__(self, dims, pairs, freq, pos, adjacent=False):
        self.keep = freq, pos
        self.c = QwRope(dims, len(pairs), (C.c_int * 3)(*pairs), adjacent, _at(freq), _at(pos))


class _Call:
    def __init__(self, name, keep, *args):
        self.name, self.keep = name, keep
        self.args = [C.byref(a) if isinstance(a, C.Structure) else a for a in args]
        self.f = None

    def __call__(self, batch):
        if self.f is None:
            self.f = getattr(batch.L, self.name)
        batch.keep.append(self)  # buffers of a call that nobody else holds last as long as the batch
        if not self.f(batch.b, *self.args):
            raise RuntimeError("%s failed: %s" % (self.name, batch.gpu.last_error()))


def _rows(x, stride=0):
    return QwKvRows(_at(x), stride)


class KvWrite(_Call):
    """Rows of q, k, v (binary16): q turned into q_out, k turned and v into the cache. strides: values from row to row of q, q_out, k, v (0: dense)."""

    def __init__(self, cache, step, q_heads, q, q_out, k, v, rope=None, strides=(0, 0, 0, 0)):
        super().__init__("qw_kv_write", (cache, step, q, q_out, k, v, rope), cache.c, step.c, rope.c if rope else None, q_heads, *(_rows(x, s) if x is not None else None for x, s in zip((q, q_out, k, v), strides)))


class KvRead(_Call):
    """The rows' keys and values (binary16) out of the cache. strides: values from row to row of k, v (0: dense)."""

    def __init__(self, cache, step, k, v, strides=(0, 0)):
        super().__init__("qw_kv_read", (cache, step, k, v), cache.c, step.c, _rows(k, strides[0]), _rows(v, strides[1]))


class Attn(_Call):
    """out = the attention of rows q over their slots' tokens (binary16 [rows][q_heads][dim]); scale 0: 1 / sqrt(dim); window 0: all tokens. ws: attn_ws_bytes of device memory, one call's at a time."""

    def __init__(self, cache, step, q_heads, q, out, ws, scale=0.0, window=0, strides=(0, 0)):
        super().__init__("qw_attn", (cache, step, q, out, ws), cache.c, step.c, q_heads, _rows(q, strides[0]), _rows(out, strides[1]), scale, window, _at(ws))


def sample_ws_bytes(gpu, rows, vocab):
    return gpu.L.qw_sample_ws_bytes(gpu.g, rows, vocab)


class Sample(_Call):
    """One token a row. params: [rows] of (temperature, top-p, min-p: float32, top-k: uint32); u float32 [rows]; ids uint32 [rows]; probs float32 [rows] or None."""

    def __init__(self, rows, vocab, logits, params, u, ids, probs, ws, stride=0):
        super().__init__("qw_sample", (logits, params, u, ids, probs, ws), rows, vocab, stride, *(_at(x) if x is not None else None for x in (logits, params, u, ids, probs, ws)))
