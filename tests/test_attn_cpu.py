"""The attention half of a decode step without a device: what its calls refuse, what they launch, its recorder and its views (include/qw_attn.h)."""
import os
import re
import subprocess

import numpy as np
import pytest

import hostrt
import qwental_amd as q
from attn_helpers import F16, Q8, Cache, Step, attention, places, quantised, scale_places, turned, unit_bytes
from qwental_amd import build
from qwental_amd.gpu import ATTN_SYMBOLS

HEAD = r"""
#include <math.h>
#include "qw_attn.c"
static int current_device = 0, launches;
static char seen[64][64];
static unsigned seen_gx[64];
static void on_launch(const char *fname, unsigned gx, unsigned bx, const void *args) {
    (void)bx, (void)args;
    if (!of_attn(fname)) return;
    seen_gx[launches % 64] = gx;
    snprintf(seen[launches++ % 64], 64, "%s", fname);
}
static char arena[1 << 20] __attribute__((aligned(4096))); // what the stand-in calls the memory of device 0
hipError_t hipGetDevice(int *d) { return *d = current_device, hipSuccess; }
hipError_t hipSetDevice(int d) { return current_device = d, hipSuccess; }
hipError_t hipStreamGetDevice(hipStream_t s, hipDevice_t *d) { return *d = (uintptr_t)s == 0x2000 ? 1 : 0, (uintptr_t)s == 0x3000 ? hipErrorInvalidHandle : hipSuccess; }
hipError_t hipPointerGetAttributes(hipPointerAttribute_t *a, const void *p) {
    memset(a, 0, sizeof *a);
    a->type = hipMemoryTypeDevice;
    if ((const char *)p < arena || (const char *)p >= arena + sizeof arena) return hipErrorInvalidValue;
    return hipSuccess;
}
hipError_t hipMemGetAddressRange(hipDeviceptr_t *base, size_t *size, hipDeviceptr_t p) { return (void)p, *base = arena, *size = sizeof arena, hipSuccess; }
static qw_gpu *with_recorder(void) {
    qw_gpu *g = device();
    g->na_batch = calloc(1, sizeof *g->na_batch);
    g->na_batch->capl = 64, g->na_batch->l = calloc(64, sizeof(qw_launch));
    g->na_batch->capuse = 1024, g->na_batch->use = calloc(1024, sizeof(qw_use));
    return g;
}
// Everything that a call takes, in one place: a test changes a field or two of what is right.
typedef struct {
    qw_kv c;
    qw_kv_step s;
    qw_rope rope;
    bool turn;
    int q_heads, window;
    float scale;
    qw_kv_rows q, q_out, k, v;
    qw_at ws;
    int rows, vocab, stride;
    qw_at logits, params, u, ids, probs, sws;
} all_of;
static qw_buf B[24];
static all_of right(qw_gpu *g) {
    static bool made;
    const size_t size[24] = {1 << 20, 64, 64, 1 << 12, 1 << 16, 1 << 16, 1 << 16, 1 << 16, 1 << 12, 1 << 12, qw_attn_ws_bytes(g, 128), 1 << 16, 1 << 12, 1 << 12, 1 << 12, 1 << 12, qw_sample_ws_bytes(g, 3, 1000)};
    for (int i = 0; i < 24 && !made; i++)
        if (size[i] && !qw_hip_buf_new_device(g, size[i], &B[i])) exit(3);
    made = true;
    return (all_of){.c = {{&B[0], 0}, 8, 2, 128, 32, 8}, .s = {3, 7, 4, {&B[1], 0}, {&B[2], 0}, {&B[3], 0}}, .rope = {64, 1, {32, 0, 0}, false, {&B[8], 0}, {&B[9], 0}}, .turn = true, .q_heads = 8,
                    .q = {{&B[4], 0}, 0}, .q_out = {{&B[5], 0}, 0}, .k = {{&B[6], 0}, 0}, .v = {{&B[7], 0}, 0}, .ws = {&B[10], 0}, .rows = 3, .vocab = 1000, .logits = {&B[11], 0}, .params = {&B[12], 0},
                    .u = {&B[13], 0}, .ids = {&B[14], 0}, .probs = {&B[15], 0}, .sws = {&B[16], 0}};
}
enum { WRITE, READ, ATTN, SAMPLE };
static bool call(qw_batch *b, int which, const all_of *a) {
    switch (which) {
    case WRITE: return qw_kv_write(b, &a->c, &a->s, a->turn ? &a->rope : NULL, a->q_heads, &a->q, &a->q_out, &a->k, &a->v);
    case READ: return qw_kv_read(b, &a->c, &a->s, &a->k, &a->v);
    case ATTN: return qw_attn(b, &a->c, &a->s, a->q_heads, &a->q, &a->q_out, a->scale, a->window, &a->ws);
    default: return qw_sample(b, a->rows, a->vocab, a->stride, &a->logits, &a->params, &a->u, &a->ids, a->probs.buf ? &a->probs : NULL, &a->sws);
    }
}
static const char *const call_names[] = {"write", "read", "attn", "sample"};
// Calls of the bits of `which` with *a: as many as are in `which` have to be refused (with a text that holds `say`) or taken, and nothing of a refused one is launched.
static int expect(qw_gpu *g, unsigned which, const all_of *a, const char *say, const char *what) {
    for (int i = 0; i < 4; i++) {
        if (!(which >> i & 1)) continue;
        const int before = launches;
        qw_batch *b = qw_batch_begin(g, false);
        const bool ok = call(b, i, a);
        if (ok != !say || (say && !strstr(qw_hip_last_error(g), say))) return printf("%s: %s: %s (%s)\n", what, call_names[i], ok ? "taken" : "refused", qw_hip_last_error(g)), 1;
        if ((qw_batch_end(b) < 0) != !ok || (launches > before) != ok) return printf("%s: %s: end\n", what, call_names[i]), 1;
    }
    return 0;
}
"""

REFUSALS = r"""
#define NO(which, say, ...) { all_of a = right(g); __VA_ARGS__; if (expect(g, which, &a, say, #__VA_ARGS__)) return 1; }
#define YES(which, ...) NO(which, NULL, __VA_ARGS__)
int main(void) {
    qw_gpu *g = device();
    const unsigned w = 1, r = 2, at = 4, sm = 8, kv = 7;
    YES(15, (void)a)
    // the cache
    NO(kv, "a cache of type", a.c.type = 0)
    NO(kv, "a cache of type", a.c.type = 2)
    NO(kv, "a cache of type", a.c.heads = 0)
    NO(kv, "a cache of type", a.c.heads = 257)
    NO(kv, "a cache of type", a.c.dim = 32)
    NO(kv, "a cache of type", a.c.dim = 96)
    NO(kv, "a cache of type", a.c.dim = 320)
    NO(kv, "a cache of type", a.c.dim = -64)
    NO(kv, "a cache of type", a.c.page = 8)
    NO(kv, "a cache of type", a.c.page = 48)
    NO(kv, "a cache of type", a.c.page = 1 << 17)
    NO(kv, "a cache of type", a.c.pages = 0)
    NO(kv, "needs", a.c.pages = 1 << 20)
    NO(kv, "needs", a.c.at.offset = (1 << 20) - 16)
    NO(kv, "aligned", a.c.at.offset = 8)
    NO(kv, "nothing bound", a.c.at.buf = NULL)
    // the step
    NO(kv, "slots", a.s.slots = 0)
    NO(kv, "slots", a.s.slots = 257)
    NO(kv, "slots", a.s.rows = 0)
    NO(kv, "slots", a.s.rows = 65537)
    NO(kv, "pages a slot", a.s.max_pages = 0)
    NO(kv, "pages a slot", a.s.max_pages = INT32_MAX)
    NO(kv, "needs", a.s.max_pages = 1 << 12)
    NO(kv, "needs", a.s.slots = 16)
    NO(kv, "needs", a.s.rows = 4096)
    NO(kv, "aligned", a.s.first.offset = 2)
    NO(kv, "aligned", a.s.len.offset = 2)
    NO(kv, "aligned", a.s.table.offset = 2)
    NO(kv, "nothing bound", a.s.len.buf = NULL)
    NO(kv, "beyond" + 6, a.s.table.offset = 1 << 13; a.s.max_pages = 1 << 13) // (past its buffer's end)
    // rows
    NO(w | r, "values from row to row", a.k.stride = 128)
    NO(w | r, "values from row to row", a.k.stride = 260)
    NO(w | r, "values from row to row", a.v.stride = -256)
    NO(w | at, "values from row to row", a.q.stride = 512)
    NO(w | at, "values from row to row", a.q_out.stride = 1020)
    NO(w | at, "aligned", a.q.at.offset = 8)
    NO(w | at, "aligned", a.q_out.at.offset = 2)
    NO(w | r, "aligned", a.k.at.offset = 4)
    NO(w | r, "nothing bound", a.v.at.buf = NULL)
    NO(w | at, "nothing bound", a.q.at.buf = NULL)
    NO(w | r, "needs", a.k.stride = 1 << 14)
    YES(w | r, a.k.stride = 264)
    YES(w, a.q_heads = 0; a.q.at.buf = NULL; a.q_out.at.buf = NULL)
    NO(w, "query heads", a.q_heads = -1)
    NO(w, "query heads", a.q_heads = 1025)
    NO(at, "query heads", a.q_heads = 0)
    NO(at, "query heads", a.q_heads = 7)
    NO(at, "query heads", a.q_heads = 1026)
    // positions
    YES(w, a.turn = false)
    YES(w, a.rope.dims = 0; a.rope.freq.buf = NULL; a.rope.pos.buf = NULL)
    NO(w, "turn", a.rope.dims = 63)
    NO(w, "turn", a.rope.dims = 130)
    NO(w, "turn", a.rope.dims = -2)
    NO(w, "axes", a.rope.axes = 2)
    NO(w, "axes", a.rope.axes = 0)
    YES(w, a.rope.axes = 3; a.rope.pairs[0] = 11; a.rope.pairs[1] = 11; a.rope.pairs[2] = 10)
    NO(w, "pairs of values", a.rope.axes = 3; a.rope.pairs[0] = 11; a.rope.pairs[1] = 11; a.rope.pairs[2] = 11)
    NO(w, "pairs of values", a.rope.axes = 3; a.rope.pairs[0] = 40; a.rope.pairs[1] = -8; a.rope.pairs[2] = 0)
    NO(w, "nothing bound", a.rope.pos.buf = NULL)
    NO(w, "nothing bound", a.rope.freq.buf = NULL)
    NO(w, "aligned", a.rope.freq.offset = 4)
    NO(w, "aligned", a.rope.pos.offset = 2)
    // attention
    NO(at, "window", a.window = -1)
    NO(at, "window", a.scale = -0.1f)
    NO(at, "window", a.scale = NAN)
    NO(at, "window", a.scale = INFINITY)
    NO(at, "nothing bound", a.ws.buf = NULL)
    NO(at, "needs", a.ws.offset = 16)
    NO(at, "needs", a.c.dim = 128; a.ws.offset = 32) // the workspace's end
    NO(at, "too many for one call", a.s.rows = 65536; a.c.page = 65536; a.c.pages = 1; a.s.max_pages = 1 << 14; a.q_heads = 1024; a.c.heads = 1; a.c.at.buf = &big; a.s.table.buf = &big)
    // tokens out of logits
    NO(sm, "rows of", a.rows = 0)
    NO(sm, "rows of", a.rows = 65537)
    NO(sm, "rows of", a.vocab = 0)
    NO(sm, "rows of", a.vocab = (1 << 20) + 1)
    NO(sm, "values from row to row", a.stride = 999)
    NO(sm, "values from row to row", a.stride = -1000)
    NO(sm, "needs", a.stride = 100000)
    NO(sm, "needs", a.vocab = 10000)
    NO(sm, "aligned", a.logits.offset = 2)
    NO(sm, "aligned", a.sws.offset = 8; a.rows = 1)
    NO(sm, "nothing bound", a.ids.buf = NULL)
    NO(sm, "nothing bound", a.u.buf = NULL)
    NO(sm, "nothing bound", a.params.buf = NULL)
    NO(sm, "nothing bound", a.sws.buf = NULL)
    YES(sm, a.probs.buf = NULL)
    // outputs over inputs
    YES(w, a.q_out = a.q)
    NO(w, "overlap", a.q_out = a.q; a.q_out.at.offset = 16)
    NO(w, "overlap", a.q_out = a.k)
    NO(w, "overlap", a.q_out = a.v)
    NO(w, "overlap", a.q_out.at.buf = &B[0])
    NO(w, "overlap", a.k.at.buf = &B[0])
    NO(w, "overlap", a.q_out.at = (qw_at){&B[9], 0}; a.s.rows = 1)
    NO(w, "overlap", a.s.first = a.c.at)
    NO(w, "overlap", a.s.table = (qw_at){&B[5], 64})
    YES(w, a.k.stride = a.v.stride = a.q.stride = 1600; a.k.at = (qw_at){&B[4], 2048}; a.v.at = (qw_at){&B[4], 2560}) // q, k and v of one product's rows
    YES(w, a.k.stride = a.v.stride = a.q.stride = 1600; a.k.at = (qw_at){&B[4], 2048}; a.v.at = (qw_at){&B[4], 2560}; a.q_out = a.q)
    NO(w, "overlap", a.k.stride = a.v.stride = a.q.stride = 1600; a.k.at = (qw_at){&B[4], 2032}; a.v.at = (qw_at){&B[4], 2560}; a.q_out = a.q)
    NO(r, "overlap", a.v = a.k)
    NO(r, "overlap", a.v.at.buf = &B[0])
    NO(r, "overlap", a.s.len = a.k.at)
    YES(r, a.v = a.k; a.k.stride = a.v.stride = 512; a.v.at.offset = 512)
    NO(at, "overlap", a.q_out = a.q)
    NO(at, "overlap", a.c.at.buf = &B[10])
    NO(at, "overlap", a.s.len = (qw_at){&B[5], 512})
    NO(at, "overlap", a.s.table = (qw_at){&B[10], 512})
    NO(sm, "overlap", a.ids = a.probs)
    NO(sm, "overlap", a.ids = a.logits)
    NO(sm, "overlap", a.u = a.ids)
    NO(sm, "overlap", a.params = (qw_at){&B[16], 64})
    NO(sm, "overlap", a.ids = (qw_at){&B[16], 64})
    // no batch, no cache, no step
    all_of a = right(g);
    for (int i = 0; i < 4; i++)
        if (call(NULL, i, &a)) return printf("no batch\n"), 1;
    qw_batch *b = qw_batch_begin(g, false);
    if (qw_kv_read(b, NULL, &a.s, &a.k, &a.v) || qw_attn(b, &a.c, NULL, 8, &a.q, &a.q_out, 0, 0, &a.ws) || qw_kv_write(b, NULL, NULL, NULL, 0, NULL, NULL, &a.k, &a.v)) return printf("no cache, no step\n"), 1;
    if (qw_attn(b, &a.c, &a.s, 8, NULL, &a.q_out, 0, 0, &a.ws) || !strstr(qw_hip_last_error(g), "nothing bound")) return printf("no queries\n"), 1;
    if (call(b, READ, &a)) return printf("a batch goes on after a failure\n"), 1;
    if (qw_batch_end(b) >= 0) return printf("a failed batch ends well\n"), 1;
    return 0;
}
"""

SIZES = r"""
int main(void) {
    if (qw_kv_bytes(1, 2, 128, 64, 10) != (size_t)10 * 2 * 4 * 128 * 64 || qw_kv_bytes(8, 2, 128, 64, 10) != (size_t)10 * 2 * 4 * 128 * 34 || qw_kv_bytes(8, 256, 256, 65536, 1 << 20) != ((size_t)1 << 40) * 256 * 34)
        return printf("bytes of a cache\n"), 1;
    if (qw_kv_bytes(2, 2, 128, 64, 10) || qw_kv_bytes(1, 2, 100, 64, 10) || qw_kv_bytes(1, 0, 128, 64, 10) || qw_kv_bytes(1, 1, 128, 0, 10) || qw_kv_bytes(1, 1, 128, -16, 10) || qw_kv_bytes(1, 1, 128, 16, -1)) return printf("no such cache\n"), 1;
    qw_gpu *g = device();
    if (qw_attn_ws_bytes(NULL, 128) || qw_attn_ws_bytes(g, 96) || qw_attn_ws_bytes(g, 0) || qw_attn_ws_bytes(g, 320) || qw_sample_ws_bytes(NULL, 1, 1) || qw_sample_ws_bytes(g, 0, 5) || qw_sample_ws_bytes(g, 1, (1 << 20) + 1))
        return printf("no such workspace\n"), 1;
    // the division by the query heads of a head: every divisor there is, at every multiple's two sides
    for (uint32_t d = 1; d <= QW_ATTN_MAX_Q_HEADS; d++) {
        const qwk_div m = div_of(d);
        for (uint64_t x = 0; x < (uint64_t)1 << 31; x = x < 100000 ? x + 1 : (x + x / 5000) / d * d + d * ((x & 1) ^ 1) - 1 + (x & 1) + 1) {
            const uint32_t y = m.mul ? (uint32_t)(x * m.mul >> 32) >> m.shift : (uint32_t)x;
            if (y != x / d) return printf("%llu / %u: %u\n", (unsigned long long)x, d, y), 1;
        }
        const uint32_t top = 0x7fffffff, y = m.mul ? (uint32_t)((uint64_t)top * m.mul >> 32) >> m.shift : top;
        if (y != top / d) return printf("the largest / %u: %u\n", d, y), 1;
    }
    return 0;
}
"""

LAUNCHES = r"""
static bool saw(const char *name, unsigned gx) { return !strcmp(seen[(launches - 1) % 64], name) && (!gx || seen_gx[(launches - 1) % 64] == gx); }
int main(void) {
    qw_gpu *g = device();
    all_of a = right(g);
    static qw_buf big;
    if (!qw_hip_buf_new_device(g, 1 << 24, &big)) return 3;
    a.q.at.buf = a.q_out.at.buf = a.k.at.buf = a.v.at.buf = &big;
    a.q_out.at.offset = 1 << 22, a.k.at.offset = 1 << 23, a.v.at.offset = 3 << 22;
    const struct { int type, dim, rows, q_heads; const char *attn, *join, *write; unsigned writes; } t[] = {
        {8, 128, 3, 8, "qwk_attn_f8_d128_q1", "qwk_attn_join_q1", "qwk_kv_write_f8_c1", 9}, {8, 128, 13, 8, "qwk_attn_f8_d128_q2", "qwk_attn_join_q2", "qwk_kv_write_f8_c1", 39}, {1, 64, 12, 8, "qwk_attn_f1_d64_q1", "qwk_attn_join_q1", "qwk_kv_write_f1_c1", 36},
        {1, 192, 1, 34, "qwk_attn_f1_d192_q1", "qwk_attn_join_q1", "qwk_kv_write_f1_c2", 10}, {1, 256, 1, 32, "qwk_attn_f1_d256_q1", "qwk_attn_join_q1", "qwk_kv_write_f1_c2", 9}, {8, 128, 1000, 8, "qwk_attn_f8_d128_q2", "qwk_attn_join_q2", "qwk_kv_write_f8_c1", 750}};
    for (size_t i = 0; i < sizeof t / sizeof *t; i++) {
        a.c.type = t[i].type, a.c.dim = t[i].dim, a.s.rows = t[i].rows, a.q_heads = t[i].q_heads, a.turn = false, a.c.pages = 2;
        a.ws.buf = &B[20];
        if (B[20].handle) qw_buf_free(&B[20]);
        if (!qw_hip_buf_new_device(g, qw_attn_ws_bytes(g, t[i].dim), &B[20])) return 3;
        qw_batch *b = qw_batch_begin(g, false);
        const int before = launches;
        if (!call(b, ATTN, &a) || qw_batch_end(b) < 0 || launches != before + 2 || !saw(t[i].join, 256)) return printf("%zu: %s, %s\n", i, seen[(launches - 1) % 64], g->err), 1;
        launches--;
        if (!saw(t[i].attn, 256)) return printf("%zu: %s\n", i, seen[(launches - 1) % 64]), 1;
        launches++;
        b = qw_batch_begin(g, false);
        if (!call(b, WRITE, &a) || qw_batch_end(b) < 0 || !saw(t[i].write, t[i].writes)) return printf("%zu: %s, %u: %s\n", i, seen[(launches - 1) % 64], seen_gx[(launches - 1) % 64], g->err), 1;
        b = qw_batch_begin(g, false);
        const unsigned units = (unsigned)t[i].rows / 16 + 2 * (t[i].rows < 3 ? (unsigned)t[i].rows : 3);
        if (!call(b, READ, &a) || qw_batch_end(b) < 0 || !saw(t[i].type == 1 ? "qwk_kv_read_f1" : "qwk_kv_read_f8", units)) return printf("%zu: %s, %u: %s\n", i, seen[(launches - 1) % 64], seen_gx[(launches - 1) % 64], g->err), 1;
    }
    // past the caches: one block a slot and 64 MB of pages that the slots may have
    static qw_buf pool, wide;
    if (!qw_hip_buf_new_device(g, (size_t)1 << 28, &pool) || !qw_hip_buf_new_device(g, qw_attn_ws_bytes(g, 128), &wide)) return 3;
    const struct { int rows, pages, max_pages; const char *attn; } past[] = {
        {3, 8192, 4096, "qwk_attn_f8_d128_q1_s"}, {12, 8192, 4096, "qwk_attn_f8_d128_q2_s"}, {13, 8192, 4096, "qwk_attn_f8_d128_q2"}, {3, 1024, 4096, "qwk_attn_f8_d128_q1"}, {3, 8192, 4, "qwk_attn_f8_d128_q1"}};
    for (size_t i = 0; i < sizeof past / sizeof *past; i++) {
        a = right(g);
        a.c.at.buf = &pool, a.c.heads = 1, a.ws.buf = &wide, a.s.table.buf = &big, a.s.rows = past[i].rows, a.c.pages = past[i].pages, a.s.max_pages = past[i].max_pages;
        qw_batch *b = qw_batch_begin(g, false);
        if (!call(b, ATTN, &a) || qw_batch_end(b) < 0 || strcmp(seen[(launches - 2) % 64], past[i].attn)) return printf("past %zu: %s, %s\n", i, seen[(launches - 2) % 64], g->err), 1;
    }
    a = right(g);
    qw_batch *b = qw_batch_begin(g, false);
    if (!call(b, SAMPLE, &a) || qw_batch_end(b) < 0 || !saw("qwk_sample", 3)) return printf("%s: %s\n", seen[(launches - 1) % 64], g->err), 1;
    // threads of a workgroup: no other number is recorded
    const struct { const char *fname; unsigned fits; } wg[] = {@names};
    static qw_kernel k = {.name = "test"};
    for (size_t i = 0; i < sizeof wg / sizeof *wg; i++)
        for (unsigned bx = 64; bx <= 1024; bx += 64) {
            b = qw_batch_begin(g, false);
            b->k = &k;
            const qwk_attn_args none = {0};
            if (add_launch(b, wg[i].fname, 1, bx, &none, sizeof none) != (bx == wg[i].fits)) return printf("%s with %u threads\n", wg[i].fname, bx), 1;
            batch_free(b);
        }
    return 0;
}
"""

RECORDER = r"""
int main(void) {
    qw_gpu *g = with_recorder();
    all_of a = right(g);
    qw_batch *b = qw_hip_stream_begin(g, (void *)0x1000);
    if (!b) return printf("%s\n", g->err), 1;
    if (qw_hip_stream_begin(g, NULL) || !strstr(qw_hip_last_error(g), "in use")) return printf("two at a time\n"), 1;
    for (int i = 0; i < 4; i++)
        if (!call(b, i, &a)) return printf("%s: %s\n", call_names[i], g->err), 1;
    if (launches || !qw_hip_stream_end(b) || launches != 6) return printf("%d launches\n", launches), 1;
    // a failure: nothing is launched, and the recorder is free again
    b = qw_hip_stream_begin(g, NULL);
    all_of bad = a;
    bad.c.dim = 100;
    if (!b || !call(b, READ, &a) || call(b, READ, &bad) || call(b, READ, &a) || qw_hip_stream_end(b) || launches != 6) return printf("failure\n"), 1;
    // buffers with a host side
    qw_buf host;
    if (!qw_buf_new(g, 1 << 16, &host)) return 3;
    b = qw_hip_stream_begin(g, NULL);
    bad = a, bad.k.at.buf = &host;
    if (!b || call(b, READ, &bad) || !strstr(qw_hip_last_error(g), "host side") || qw_hip_stream_end(b)) return printf("a buffer with a host side\n"), 1;
    if (expect(g, 1 << READ, &bad, NULL, "a buffer with a host side in a batch")) return 1;
    // as many launches as it holds
    const int before = launches;
    b = qw_hip_stream_begin(g, NULL);
    for (int i = 0; i < 64; i++)
        if (!call(b, READ, &a)) return printf("launch %d: %s\n", i, g->err), 1;
    if (call(b, READ, &a) || !strstr(qw_hip_last_error(g), "64 launches") || qw_hip_stream_end(b) || launches != before) return printf("65 launches\n"), 1;
    // not a batch: it is neither split nor ended as one, and takes no other functions
    b = qw_hip_stream_begin(g, NULL);
    qw_batch_flush(b), qw_batch_submit(b);
    if (!b || !call(b, READ, &a) || qw_batch_end(b) >= 0 || !strstr(qw_hip_last_error(g), "qw_hip_stream_end") || launches != before) return printf("ended as a batch\n"), 1;
    qw_path *op = qw_path_open(g, 1024, 256, 64, 4, 16, true);
    qw_buf ow;
    if (!qw_hip_buf_new_device(g, (size_t)64 * 1024 * 256 * 2, &ow)) return 3;
    b = qw_hip_stream_begin(g, NULL);
    const qw_tensor OW = {.buf = &ow, .type = 8};
    if (!b || (qw_path_qmv_gg(op, b, &OW, 64, 256, &B[4], 0, &B[5], 0, 1, true) && qw_hip_stream_end(b)) || !strstr(qw_hip_last_error(g), "qw_attn.h") || launches != before) return printf("another function: %s\n", g->err), 1;
    if (g->na_busy) (void)qw_hip_stream_end(b);
    // other devices' streams, and the current device put back
    if (qw_hip_stream_begin(g, (void *)0x2000) || qw_hip_stream_begin(g, (void *)0x3000) || qw_hip_stream_begin(NULL, NULL) || qw_hip_stream_end(NULL)) return printf("streams\n"), 1;
    current_device = 3;
    b = qw_hip_stream_begin(g, (void *)0x1000);
    if (!b || current_device != 0 || !call(b, READ, &a) || !qw_hip_stream_end(b) || current_device != 3) return printf("the current device\n"), 1;
    b = qw_hip_stream_begin(g, NULL);
    if (!b || qw_hip_stream_begin(g, NULL) || !qw_hip_stream_end(b) || current_device != 3) return printf("the current device, refused\n"), 1;
    current_device = 0;
    // views
    qw_buf view, other;
    if (!qw_hip_buf_view(g, arena + 4096, sizeof arena - 4096, &view) || view.ptr || view.size != sizeof arena - 4096) return printf("a view: %s\n", g->err), 1;
    if (qw_hip_buf_view(g, arena + 4096, sizeof arena - 4095, &other) || qw_hip_buf_view(g, arena, SIZE_MAX, &other) || qw_hip_buf_view(g, NULL, 16, &other) || qw_hip_buf_view(g, &view, 16, &other) || qw_hip_buf_view(NULL, arena, 16, &other) ||
        qw_hip_buf_view(g, arena, 16, NULL)) return printf("views of what is not there\n"), 1;
    all_of over = a;
    over.k.at = (qw_at){&view, 0}, over.v.at = (qw_at){&view, 1 << 16};
    if (expect(g, 1 << READ, &over, NULL, "a view in a batch")) return 1;
    b = qw_hip_stream_begin(g, NULL);
    if (!call(b, READ, &over) || !qw_hip_stream_end(b)) return printf("a view in a recorder: %s\n", g->err), 1;
    qw_path *p = qw_path_open(g, 1024, 256, 64, 4, 16, true);
    qw_buf w, lg, sel, out;
    if (!p || !qw_hip_buf_new_device(g, (size_t)64 * 1024 * 256 * 2, &w) || !qw_hip_buf_new_device(g, qw_path_logits_bytes(p, 16), &lg) || !qw_hip_buf_new_device(g, qw_path_sel_bytes(p, 16), &sel) || !qw_hip_buf_new_device(g, 16 * 2048, &out)) return 3;
    const qw_tensor W = {.buf = &w, .type = 8}, R = {.buf = &w, .type = 1};
    const qw_moe_layer M = {.router = R, .sh_gate_w = R, .gate = W, .up = W, .down = W, .sh_gate = W, .sh_up = W, .sh_down = W};
    b = qw_batch_begin(g, false);
    if ((qw_path_gg_moe(p, b, &M, 1, &view, &lg, &sel, &out) && qw_batch_end(b) >= 0) || !strstr(qw_hip_last_error(g), "view")) return printf("a view in another function: %s\n", g->err), 1;
    qw_buf_free(&view);
    memset(arena, 1, sizeof arena); // still there
    return 0;
}
"""


def run(tmp_path, source):
    (tmp_path / "qw_attn_gfx950.hsaco").write_bytes(b"\0")
    return hostrt.run(tmp_path, HEAD + source, "-I", os.path.join(build.CSRC, "kernels"), "-Wno-unused", "-lm")


def test_refusals(tmp_path):
    run(tmp_path, REFUSALS.replace("int main(void) {\n    qw_gpu *g = device();", "static qw_buf big;\nint main(void) {\n    qw_gpu *g = device();\n    if (!qw_hip_buf_new_device(g, (size_t)1 << 25, &big)) return 3;"))


def test_sizes(tmp_path):
    run(tmp_path, SIZES)


def test_launches_and_their_workgroups(tmp_path):
    if not os.path.exists(build.HIPCC):
        pytest.skip("no hipcc here")
    src = subprocess.run([build.HIPCC, "--offload-arch=gfx950", "-std=c++17", "--cuda-device-only", "-E", "-P", "-I", os.path.join(build.CSRC, "kernels"), os.path.join(build.CSRC, "kernels", "qw_attn.hip")],
                         stdout=subprocess.PIPE, text=True, check=True).stdout
    found = re.findall(r"amdgpu_flat_work_group_size\(1,\s*([0-9u* ]+)\)[^;{}]*?void\s+(qwk_\w+)\s*\(", src)
    assert len(found) == 24 + 2 + 4 + 2 + 2 == len(set(n for _, n in found))
    run(tmp_path, LAUNCHES.replace("@names", ", ".join('{"%s", %s}' % (n, t) for t, n in found)))


def test_recorder_on_a_stream_and_views(tmp_path):
    run(tmp_path, RECORDER)


def test_symbols():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(build.ROOT, "include", "qw_attn.h")).read(), flags=re.S)
    declared = set(re.findall(r"\b(qw_[a-z0-9_]+)\s*\(", text))
    assert declared == {n for n, _, _ in ATTN_SYMBOLS}
    L = q.load_lib()
    assert all(hasattr(L, n) for n in declared)


@pytest.mark.parametrize("kind", [F16, Q8])
@pytest.mark.parametrize("D", [64, 128, 192, 256])
def test_oracle_of_a_unit(kind, D):
    """Every byte of a unit is some value's or scale's, once."""
    size = 2 if kind == F16 else 1
    used = [places(kind, D, v).ravel() + i for v in (False, True) for i in range(size)]
    if kind == Q8:
        used += [scale_places(D, v).ravel() + i for v in (False, True) for i in range(2)]
    assert np.array_equal(np.sort(np.concatenate(used)), np.arange(unit_bytes(kind, D)))


def test_oracle_of_a_block():
    x = np.array([[0.0] * 32, [1.0] + [0.5] * 31, [65504.0] * 31 + [-65504.0], [np.inf] + [1.0] * 31, [2.0 ** -24] * 32], np.float16)
    c, d = quantised(x)
    assert (c[0] == 0).all() and d[0] == 0 and c[1, 0] == 127 and abs(float(d[1, 0]) * 127 - 1) < 2.0 ** -10
    assert float(d[2, 0]) == 515.5 and c[2, 0] == 127 and c[2, 31] == -127 and np.isnan(d[3, 0]) and (c[4] == 0).all()


def test_oracle_of_positions_and_attention():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((3, 2, 64)).astype(np.float16)
    pos, freq = np.array([[0], [3], [1000000]]), 10000.0 ** (-np.arange(16) / 16)
    for adjacent in (False, True):
        y = turned(x, pos, freq, [16], adjacent)
        assert np.array_equal(y[0], x[0]) and np.array_equal(y[..., 32:], x[..., 32:])
        i = (slice(0, 32, 2), slice(1, 32, 2)) if adjacent else (slice(0, 16), slice(16, 32))
        z = (x[..., i[0]] + 1j * x[..., i[1]].astype(np.float64)) * np.exp(1j * (pos * freq))[:, None]
        assert np.abs(y[..., i[0]] - z.real).max() < 2.0 ** -9 and np.abs(y[..., i[1]] - z.imag).max() < 2.0 ** -9
    s = Step(rng, [2, 1], [20, 5], 16)
    c = Cache(F16, 1, 64, 16, s.pages)
    k, v = (rng.standard_normal((2, 20, 1, 64)).astype(np.float16) for _ in range(2))
    for slot, n in ((0, 20), (1, 5)):
        for t in range(n):
            c.put(s.table, slot, t, k[slot, t], v[slot, t])
    qr = rng.standard_normal((3, 2, 64)).astype(np.float16)
    out, tol = attention(c, s, qr, 0.125)
    for row, slot, token in s.rows_of():
        p = np.exp(qr[row].astype(np.float64) @ k[slot, :token + 1, 0].astype(np.float64).T * 0.125)
        assert np.abs(out[row] - p @ v[slot, :token + 1, 0].astype(np.float64) / p.sum(1, keepdims=True)).max() < 1e-12 and (tol[row] > 0).all() and tol[row].max() < 0.01
