// Kernels of a decode step's attention half: rows of keys and values into a paged cache and out of it, and attention over it.
//
// The cache is made of units: 16 tokens of one head, in the order in which the matrix instructions take them (include/qw_attn.h).
#include <hip/hip_runtime.h>
#include "qw_attn_kargs.h"

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef uint32_t uint2_t __attribute__((ext_vector_type(2)));
typedef uint32_t uint4_t __attribute__((ext_vector_type(4)));

typedef unsigned long long u64;

enum { F16 = 1, Q8 = 8 };

// ---------------------------------------------------------------- attention
// S^T = K Q^T and O^T = V^T P^T: with the tokens as rows of the first product, a lane's results are scores of ONE query (lane & 15)
// for tokens 4 (lane >> 4) + i, which is what the second product takes from that lane. Nothing moves between lanes and nothing goes
// through LDS between the two; the cache's units are stored so that a lane's operands are 16 consecutive bytes of a wave's 1024.
//
// Work: a pair is (slot, head, block of 16 QT of the slot's rows x query heads of that head); its tiles of 32 tokens lie one behind another,
// pair after pair, and the workgroups of the grid take equal shares of that line, wherever pairs begin or end in it: a long slot is
// cut over many workgroups, short ones share one. All of it follows from first[] and len[] on the device, so a captured call goes on
// being right (and even) as the slots grow. A share that ends inside a pair leaves (maximum, sum, unnormalised result), which qwk_attn_join
// puts together in the order of the shares: the same bits every time.

struct Slot { int n, len, first; }; // rows, tokens, first row

// first, len and table are nobody's output: read as constants, with a uniform index through the scalar cache, whose loads do not wait for the streams'.
typedef const uint32_t __attribute__((address_space(4))) *const_words;
__device__ __forceinline__ const_words words(const uint32_t *p) { return (const_words)(uintptr_t)p; }

__device__ __forceinline__ Slot slot_of(const qwk_kv &c, uint32_t i) {
    uint32_t a = words(c.first)[i], b = words(c.first)[i + 1], l = words(c.len)[i];
    const uint32_t room = c.max_pages << c.page_log2; // (up to 2^30)
    Slot s;
    s.first = (int)a;
    s.n = (a <= b) & (b <= c.rows) ? (int)(b - a) : 0; // what is no row of the step is not touched
    s.len = (int)min(l, room);
    return s;
}
// The slot of a row, by a whole wave in one round trip; false: it belongs to none.
__device__ __forceinline__ bool slot_find(const qwk_kv &c, uint32_t row, uint32_t &i, Slot &s) {
    i = 0;
    for (uint32_t at = 0; at < c.slots; at += 64) {
        const uint32_t k = at + (threadIdx.x & 63);
        i += (uint32_t)__popcll(__ballot(k < c.slots && words(c.first)[k + 1] <= row));
    }
    if (i >= c.slots) return false;
    s = slot_of(c, i);
    return (int)row >= s.first && (int)row < s.first + s.n;
}
__device__ __forceinline__ int by(qwk_div d, int x) { return d.mul ? (int)(__umulhi((uint32_t)x, d.mul) >> d.shift) : x; } // x / d, 0 <= x < 2^31

struct Range { int t0, cnt; }; // a block's first tile, and how many (at least one: an empty one still gives its rows their zeros)
template <int QT> __device__ __forceinline__ Range block_range(const Slot &s, int b, const qwk_attn_args &a) {
    const int M = s.n * (int)a.group, j0 = by(a.by_group, b * 16 * QT), j1 = by(a.by_group, min((b + 1) * 16 * QT, M) - 1);
    const int hi = s.len - s.n + j1 + 1, lo = a.window ? max(0, s.len - s.n + j0 - (int)a.window + 1) : 0;
    Range r;
    r.t0 = hi > 0 ? lo / (int)QW_ATTN_TILE : 0;
    r.cnt = hi > 0 ? max(1, (hi + (int)QW_ATTN_TILE - 1) / (int)QW_ATTN_TILE - r.t0) : 1;
    return r;
}
template <int QT> __device__ __forceinline__ int blocks_of(const Slot &s, const qwk_attn_args &a) { return (s.n * (int)a.group + 16 * QT - 1) / (16 * QT); }

// Tiles of all slots, a lane a slot. Every wave makes it and writes it down for itself (all the same, where it is the same LDS): no barrier.
struct Plan { uint32_t each[QW_KV_SLOTS_MAX], end[QW_KV_SLOTS_MAX]; }; // tiles of one of the slot's heads; of all slots up to and with this one
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) { // sums over the lanes up to and with this one
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xf, 0xf, false); // row_shr:1, 2, 4, 8
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xf, 0xf, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xf, 0xf, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xf, 0xf, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xa, 0xf, false); // row_bcast:15, 31
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xc, 0xf, false);
    return x;
}
template <int QT> __device__ __forceinline__ uint32_t make_plan(Plan &p, const qwk_attn_args &a, uint32_t &pairs) { // returns the tiles of all
    const uint32_t lane = threadIdx.x & 63;
    uint32_t T = 0;
    pairs = 0;
#pragma unroll 1
    for (uint32_t k = 0; k < a.c.slots; k += 64) {
        const uint32_t i = k + lane;
        uint32_t each = 0;
        Slot s = slot_of(a.c, min(i, a.c.slots - 1));
        asm volatile("" : "+v"(s.n), "+v"(s.len)); // (all three loads at once, not the length's behind a branch on the others)
        const int nb = i < a.c.slots ? blocks_of<QT>(s, a) : 0;
#pragma unroll 1
        for (int b = 0; b < nb; b++) each += (uint32_t)block_range<QT>(s, b, a).cnt;
        const uint32_t end = T + wave_scan(each * a.c.heads);
        p.each[i] = each, p.end[i] = end;
        T = (uint32_t)__builtin_amdgcn_readlane((int)end, 63);
        pairs += (uint32_t)__builtin_amdgcn_readlane((int)wave_scan((uint32_t)nb), 63);
    }
    pairs *= a.c.heads;
    return T;
}
// Shares: workgroup w of g takes the next T / g tiles, the first T % g of them one more.
struct Shares {
    uint32_t g, base, more;
    // As many workgroups as there are four tiles for, one a wave, or pairs: behind its first pair's end a workgroup starts once more (3 us; a slot of one token and four heads: one
    // workgroup for all of them 15.9 us, four 6)
    __device__ __forceinline__ Shares(uint32_t T, uint32_t pairs, uint32_t grid) : g(min(grid, max((T + 3) / 4, pairs))), base(0), more(0) {
        if (g) base = T / g, more = T - base * g;
    }
    __device__ __forceinline__ uint32_t start(uint32_t w) const { return w * base + min(w, more); }
    __device__ __forceinline__ uint32_t owner(uint32_t x) const {
        const uint32_t big = more * (base + 1);
        return x < big ? x / (base + 1) : more + (x - big) / base;
    }
};

// Four codes -> binary16, exactly: 0x64 in front of a byte b is 1024 + b, and b is the code + 128.
__device__ __forceinline__ half4_t codes(uint32_t w) {
    w ^= 0x80808080u;
    const half2_t bias = {(_Float16)-1152.f, (_Float16)-1152.f};
    const half2_t lo = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) + bias;
    const half2_t hi = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) + bias;
    return half4_t{lo.x, lo.y, hi.x, hi.y};
}

template <int TYPE, int D> struct UnitData; // a lane's share of a unit: keys or values, and their scales
template <int D> struct UnitData<F16, D> {
    uint4_t x[D / 32];
    __device__ __forceinline__ void load(const uint8_t *u, bool values, uint32_t at, uint32_t) {
        const uint8_t *p = u + (values ? 32 * D : 0) + at;
#pragma unroll
        for (int c = 0; c < D / 32; c++) x[c] = *(const uint4_t *)(p + c * 1024);
    }
    // Of values: zeros in place of the lane's tokens that `keep` (two halves a word) has no bits for; which of the four tokens hold what is not finite (bits of 0x7c00 in each half)
    __device__ __forceinline__ void mask(uint2_t keep) {
#pragma unroll
        for (int c = 0; c < D / 32; c++) x[c] &= uint4_t{keep.x, keep.y, keep.x, keep.y};
    }
    __device__ __forceinline__ uint2_t odd() const {
        uint2_t o = {0, 0};
        const auto full = [](uint32_t w) { return ((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u; }; // (neither half carries into the other: its sign is masked)
#pragma unroll
        for (int c = 0; c < D / 32; c++) o |= uint2_t{full(x[c].x) | full(x[c].z), full(x[c].y) | full(x[c].w)};
        return o;
    }
    static __device__ __forceinline__ float value(const uint8_t *u, uint32_t t, uint32_t v) { return (float)*(const _Float16 *)(u + 32 * D + (v / 32 * 512 + t / 4 * 128 + v % 32 * 4 + t % 4) * 2); }
};
template <int D> struct UnitData<Q8, D> {
    uint4_t x[D / 64], s[D / 64];
    __device__ __forceinline__ void load(const uint8_t *u, bool values, uint32_t at, uint32_t scale_at) {
        const uint8_t *p = u + (values ? 17 * D : 0);
#pragma unroll
        for (int c = 0; c < D / 64; c++) x[c] = *(const uint4_t *)(p + c * 1024 + at);
#pragma unroll
        for (int c = 0; c < D / 64; c++) s[c] = *(const uint4_t *)(p + 16 * D + scale_at + c * 16);
    }
    __device__ __forceinline__ void mask(uint2_t keep) { // (codes are finite: it is the scales that are not)
#pragma unroll
        for (int c = 0; c < D / 64; c++) s[c] &= uint4_t{keep.x, keep.y, keep.x, keep.y};
    }
    __device__ __forceinline__ uint2_t odd() const {
        uint2_t o = {0, 0};
        const auto full = [](uint32_t w) { return ((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u; };
#pragma unroll
        for (int c = 0; c < D / 64; c++) o |= uint2_t{full(s[c].x) | full(s[c].z), full(s[c].y) | full(s[c].w)};
        return o;
    }
    static __device__ __forceinline__ float value(const uint8_t *u, uint32_t t, uint32_t v) {
        return (float)*(const int8_t *)(u + 17 * D + v / 64 * 1024 + t / 4 * 256 + v % 32 / 2 * 16 + v / 32 % 2 * 8 + v % 2 * 4 + t % 4) * (float)*(const _Float16 *)(u + 33 * D + (t / 4 * (D / 32) + v / 32) * 8 + t % 4 * 2);
    }
    __device__ __forceinline__ half4_t scales(int b) const { // of block b, tokens 4 (lane >> 4) + i
        return __builtin_bit_cast(half4_t, b & 1 ? uint2_t{s[b / 2].z, s[b / 2].w} : uint2_t{s[b / 2].x, s[b / 2].y});
    }
};

template <int TYPE, int D, int QT, int U> struct Attn {
    const qwk_attn_args &a;
    const uint32_t lane;
    half8_t q[QT][D / 32];
    float4_t acc[QT][D / 32][2]; // result: value 32 b + 8 (lane >> 4) + 2 i + c of query lane & 15
    float m[QT], l[QT];          // reference (log2) and this lane's part of the sum
    int hi[QT], lo[QT];          // tokens [lo, hi) that the lane's query sees
    UnitData<TYPE, D> K[U], V[U];

    __device__ __forceinline__ float4_t scores(int t, int i) {
        float4_t s = {0, 0, 0, 0};
        if constexpr (TYPE == F16) {
#pragma unroll
            for (int c = 0; c < D / 32; c++) s = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, K[i].x[c]), q[t][c], s, 0, 0, 0);
        } else {
#pragma unroll
            for (int c = 0; c < D / 32; c++) {
                const uint4_t x = K[i].x[c / 2];
                const half4_t k0 = codes(c & 1 ? x.z : x.x), k1 = codes(c & 1 ? x.w : x.y);
                const float4_t z = {0, 0, 0, 0};
                const float4_t d = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_shufflevector(k0, k1, 0, 1, 2, 3, 4, 5, 6, 7), q[t][c], z, 0, 0, 0);
                const half4_t f = K[i].scales(c);
#pragma unroll
                for (int j = 0; j < 4; j++) s[j] = __builtin_fmaf((float)f[j], d[j], s[j]);
            }
        }
        return s;
    }
    // Weights in two parts, binary16 each: together they hold 21 bits, so that the result is as exact as its own rounding. The largest weight is 2^TOP, not 1, so that the
    // small ones do not end at binary16's 2^-24: many tokens of 2^-25 of the largest's weight count for something together. (Q8_0: a weight is multiplied by a scale of up to 516.)
    static constexpr float TOP = TYPE == F16 ? 14.f : 6.f;
    __device__ __forceinline__ static void split(const float4_t &p, half4_t &h, half4_t &r) {
        const half2_t h0 = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_pkrtz(p[0], p[1])), h1 = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_pkrtz(p[2], p[3]));
        float d[4];
#pragma unroll
        for (int j = 0; j < 4; j++) d[j] = __builtin_fmaf((float)(j < 2 ? h0 : h1)[j & 1], -1.f, p[j]);
        const half2_t r0 = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_pkrtz(d[0], d[1])), r1 = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_pkrtz(d[2], d[3]));
        h = half4_t{h0.x, h0.y, h1.x, h1.y}, r = half4_t{r0.x, r0.y, r1.x, r1.y};
    }
    __device__ __forceinline__ half4_t values(int i, int b, int c) const {
        if constexpr (TYPE == F16) return __builtin_bit_cast(half4_t, c ? uint2_t{V[i].x[b].z, V[i].x[b].w} : uint2_t{V[i].x[b].x, V[i].x[b].y});
        else return codes(V[i].x[b / 2][(b & 1) * 2 + c]);
    }
    __device__ __forceinline__ bool hidden(int t, int key, uint32_t bad, int i) const { return key >= hi[t] || key < lo[t] || (bad >> i & 1); }
    // key0: first token of the step's first unit; bad: units without a page; edge: some query does not see all of the step's tokens
    __device__ __forceinline__ void softmax(int key0, uint32_t bad, bool edge, float4_t (&p)[QT][U]) {
        const float neg = -__builtin_inff();
        if (edge)
#pragma unroll
            for (int t = 0; t < QT; t++)
#pragma unroll
                for (int i = 0; i < U; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (hidden(t, key0 + i * 16 + (int)(lane >> 4) * 4 + j, bad, i)) p[t][i][j] = neg;
#pragma unroll
        for (int t = 0; t < QT; t++) {
            float top = neg;
#pragma unroll
            for (int i = 0; i < U; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) top = fmaxf(top, p[t][i][j]);
            top *= a.scale;
            if (__any(top > m[t])) { // (as a rule in a wave's first steps only)
                top = fmaxf(top, __shfl_xor(top, 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                const float now = fmaxf(m[t], top), f = m[t] == neg ? 0.f : __builtin_amdgcn_exp2f(m[t] - now);
                m[t] = now;
                l[t] *= f;
#pragma unroll
                for (int b = 0; b < D / 32; b++) acc[t][b][0] *= f, acc[t][b][1] *= f;
            }
            const float ref = m[t] == neg ? 0.f : TOP - m[t];
#pragma unroll
            for (int i = 0; i < U; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    p[t][i][j] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[t][i][j], a.scale, ref));
                    l[t] += p[t][i][j];
                }
        }
    }
    __device__ __forceinline__ void weigh(const float4_t (&p)[QT][U]) {
#pragma unroll
        for (int i = 0; i < U; i++) {
            half4_t h[QT], r[QT];
            if constexpr (TYPE == F16)
#pragma unroll
                for (int t = 0; t < QT; t++) split(p[t][i], h[t], r[t]);
#pragma unroll
            for (int b = 0; b < D / 32; b++) {
                const half4_t v0 = values(i, b, 0), v1 = values(i, b, 1);
                if constexpr (TYPE == Q8) {
                    const half4_t f = V[i].scales(b); // a token's scale belongs to its weight
#pragma unroll
                    for (int t = 0; t < QT; t++) {
                        float4_t w;
#pragma unroll
                        for (int k = 0; k < 4; k++) w[k] = p[t][i][k] * (float)f[k];
                        split(w, h[t], r[t]);
                    }
                }
#pragma unroll
                for (int t = 0; t < QT; t++) {
                    acc[t][b][0] = __builtin_amdgcn_mfma_f32_16x16x16f16(v0, h[t], acc[t][b][0], 0, 0, 0);
                    acc[t][b][1] = __builtin_amdgcn_mfma_f32_16x16x16f16(v1, h[t], acc[t][b][1], 0, 0, 0);
                    acc[t][b][0] = __builtin_amdgcn_mfma_f32_16x16x16f16(v0, r[t], acc[t][b][0], 0, 0, 0);
                    acc[t][b][1] = __builtin_amdgcn_mfma_f32_16x16x16f16(v1, r[t], acc[t][b][1], 0, 0, 0);
                }
            }
        }
    }
    // A token that some queries do not see may hold anything, infinities and NaN too, and 0 times those is not 0. So at the edges: values of tokens that no query of the
    // block sees become zeros; a token that some see and that holds what is not finite is taken out of the product too, and comes back by itself
    // (odd_tokens) for those that see it. Returns such tokens of unit i as bits.
    __device__ __forceinline__ uint32_t clean(int i, int key0, uint32_t bad, int all_lo, int all_hi) {
        const int key = key0 + i * 16 + (int)(lane >> 4) * 4;
        const auto unseen = [&](int k) { return key + k >= all_hi || key + k < all_lo || (bad >> i & 1); };
        V[i].mask(uint2_t{(unseen(0) ? 0u : 0xffffu) | (unseen(1) ? 0u : 0xffff0000u), (unseen(2) ? 0u : 0xffffu) | (unseen(3) ? 0u : 0xffff0000u)});
        const uint2_t o = V[i].odd();
        if (!__any((o.x | o.y) != 0)) return 0;
        uint32_t tokens = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const u64 at = __ballot((o[k / 2] >> (k & 1 ? 31 : 15) & 1) != 0);
#pragma unroll
            for (int g = 0; g < 4; g++) tokens |= (at >> g * 16 & 0xffff) ? 1u << (g * 4 + k) : 0;
        }
        const uint32_t mine = tokens >> (lane >> 4) * 4;
        V[i].mask(uint2_t{(mine & 1 ? 0u : 0xffffu) | (mine & 2 ? 0u : 0xffff0000u), (mine & 4 ? 0u : 0xffffu) | (mine & 8 ? 0u : 0xffff0000u)});
        return tokens;
    }
    __device__ __forceinline__ void odd_tokens(int i, uint32_t tokens, const uint8_t *u, int key0, uint32_t bad, const float4_t (&p)[QT][U]) {
#pragma unroll 1
        for (; tokens; tokens &= tokens - 1) {
            const int k = __builtin_ctz(tokens);
#pragma unroll
            for (int t = 0; t < QT; t++) {
                const float4_t x = p[t][i];
                const float w = __shfl(k & 2 ? (k & 1 ? x[3] : x[2]) : (k & 1 ? x[1] : x[0]), (int)(lane & 15) + (k >> 2) * 16);
                if (!hidden(t, key0 + i * 16 + k, bad, i))
#pragma unroll
                    for (int b = 0; b < D / 32; b++)
#pragma unroll
                        for (int j = 0; j < 8; j++) acc[t][b][j & 1][j >> 1] += w * UnitData<TYPE, D>::value(u, (uint32_t)k, (uint32_t)b * 32 + (lane >> 4) * 8 + (uint32_t)j);
            }
        }
    }
};

// What a workgroup leaves for the join, twice: of the pair that it went on with, and of the one that it began and did not end.
struct Part {
    uint32_t rows, row0, m0, head, w0, w1; // rows 0: none; the pair's block: first row of the slot, first row x query head, and the workgroups that share it
    uint32_t pad[2];
};
static_assert(sizeof(Part) == QW_ATTN_PART, "");

template <int TYPE, int D, int QT> __device__ __forceinline__ void attn_body(const qwk_attn_args &a) {
    constexpr int U = D <= 128 ? 2 : 1, W = QW_WG_ATTN / 64, LD = D + 4, STEPS = 2 / U; // U: units a wave has in hand; a tile is two
    __shared__ float4_t so[W][16][LD / 4];
    __shared__ float sm[W][16], sl[W][16];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const qwk_kv &c = a.c;
    const int group = (int)a.group, window = (int)a.window;
    Part *parts = (Part *)a.parts + blockIdx.x * 2;
    __shared__ Plan plan;
    uint32_t pairs;
    const uint32_t T = make_plan<QT>(plan, a, pairs);
    const Shares sh(T, pairs, a.grid);
    if (threadIdx.x < 2) parts[threadIdx.x].rows = 0;
    if (blockIdx.x >= sh.g) return;
    uint32_t x = sh.start(blockIdx.x);
    const uint32_t end = sh.start(blockIdx.x + 1);
    while (x < end) {
        uint32_t i = 0; // the slot that tile x belongs to
        for (uint32_t k = 0; k < c.slots; k += 64) i += (uint32_t)__popcll(__ballot(plan.end[k + lane] <= x));
        const Slot s = slot_of(c, i);
        const uint32_t each = (uint32_t)__builtin_amdgcn_readfirstlane((int)plan.each[i]), base = (uint32_t)__builtin_amdgcn_readfirstlane((int)plan.end[i]) - each * c.heads;
        const uint32_t head = (x - base) / each;
        int from = (int)(x - base - head * each), blk = 0;
        Range r = block_range<QT>(s, 0, a);
        while (from >= r.cnt) from -= r.cnt, r = block_range<QT>(s, ++blk, a);
        const int to = min(r.cnt, from + (int)(end - x));
        const int M = s.n * group, m0 = blk * 16 * QT;

        Attn<TYPE, D, QT, U> A{a, lane};
#pragma unroll
        for (int t = 0; t < QT; t++) {
            const int row = min(m0 + t * 16 + (int)(lane & 15), M - 1), j = by(a.by_group, row);
            A.hi[t] = s.len - s.n + j + 1;
            A.lo[t] = window ? max(0, A.hi[t] - window) : 0;
            A.m[t] = -__builtin_inff(), A.l[t] = 0;
            const uint16_t *q = a.q + (size_t)(s.first + j) * a.q_stride + ((size_t)head * group + (row - j * group)) * D + (lane >> 4) * 8;
#pragma unroll
            for (int k = 0; k < D / 32; k++) A.q[t][k] = *(const half8_t *)(q + k * 32);
#pragma unroll
            for (int b = 0; b < D / 32; b++) A.acc[t][b][0] = A.acc[t][b][1] = float4_t{0, 0, 0, 0};
        }
        // a step's units: where they lie, and which of them have no page
        const int pu = (int)c.page_log2 - 4; // log2 of a page's units
        const const_words table = words(c.table) + (size_t)i * c.max_pages;
        const size_t in_page = (size_t)head << pu;
        const uint8_t *u[U];
        uint32_t bad;
        const auto find = [&](int key0) {
            bad = 0;
#pragma unroll
            for (int k = 0; k < U; k++) {
                const uint32_t un = (uint32_t)(key0 >> 4) + k, at = un >> pu;
                uint32_t page = at < c.max_pages ? table[at] : 0xffffffffu;
                if (page >= c.pages) bad |= 1u << k, page = 0;
                u[k] = c.cache + page * c.page_bytes + (in_page + (un & ((1u << pu) - 1))) * c.unit;
            }
        };
        const int steps = max(0, (to - from - (int)wave + W - 1) / W) * STEPS;
        const auto key_of_step = [&](int n) { return (r.t0 + from + (int)wave + n / STEPS * W) * (int)QW_ATTN_TILE + n % STEPS * 16 * U; };
        // (The queries are asked for before the first step's units: behind them they would be waited for with everything, every step, as the loop's wait has to do for its first.)
        __builtin_amdgcn_sched_barrier(0);
        int key0 = key_of_step(0);
        const uint32_t at = lane * 16, scale_at = (lane >> 4) * (D / 4);
        find(key0);
#pragma unroll
        for (int k = 0; k < U; k++) A.K[k].load(u[k], false, steps ? at : 0, steps ? scale_at : 0);
#pragma unroll
        for (int k = 0; k < U; k++) A.V[k].load(u[k], true, steps ? at : 0, steps ? scale_at : 0);
        // what every query of the block sees: [see_lo, see_hi), and what any of them does: [all_lo, all_hi)
        const int see_hi = s.len - s.n + by(a.by_group, m0) + 1, all_hi = s.len - s.n + by(a.by_group, min(m0 + 16 * QT, M) - 1) + 1;
        const int see_lo = window ? max(0, all_hi - window) : 0, all_lo = window ? max(0, see_hi - window) : 0;
        for (int n = 0; n < steps; n++) {
            const int key = key0;
            const uint32_t none = bad;
            const uint8_t *now[U];
#pragma unroll
            for (int k = 0; k < U; k++) now[k] = u[k];
            const bool edge = none || key < see_lo || key + 16 * U > see_hi;
            // The next step's loads go out as registers come free: keys behind the scores, values behind the second product. There is one set a step, the last step's too
            // (16 bytes of its own units, which it does not use): the compiler then knows how many are in flight.
            const bool more = n + 1 < steps;
            key0 = more ? key_of_step(n + 1) : key;
            find(key0);
            const uint32_t nat = more ? at : 0, nscale = more ? scale_at : 0;
            float4_t p[QT][U];
#pragma unroll
            for (int k = 0; k < U; k++)
#pragma unroll
                for (int t = 0; t < QT; t++) p[t][k] = A.scores(t, k);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int k = 0; k < U; k++) A.K[k].load(u[k], false, nat, nscale);
            __builtin_amdgcn_sched_barrier(0);
            A.softmax(key, none, edge, p);
            uint32_t odd = 0;
            if (edge)
#pragma unroll
                for (int k = 0; k < U; k++) odd |= A.clean(k, key, none, all_lo, all_hi) << 16 * k;
            A.weigh(p);
            if (odd)
#pragma unroll
                for (int k = 0; k < U; k++) A.odd_tokens(k, odd >> 16 * k & 0xffff, now[k], key, none, p);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int k = 0; k < U; k++) A.V[k].load(u[k], true, nat, nscale);
        }
        // the waves' results together, in the waves' order
        const bool whole = from == 0 && to == r.cnt;
        const uint32_t which = from == 0, slot = blockIdx.x * 2 + which;
        if (!whole && threadIdx.x == 0) {
            const uint32_t x0 = x - (uint32_t)from;
            Part p = {(uint32_t)min(16 * QT, M - m0), (uint32_t)s.first, (uint32_t)m0, head, sh.owner(x0), sh.owner(x0 + (uint32_t)r.cnt - 1), {0, 0}};
            parts[which] = p;
        }
#pragma unroll
        for (int t = 0; t < QT; t++) {
            if (m0 + t * 16 >= M) break;
            float l = A.l[t];
            l += __shfl_xor(l, 16);
            l += __shfl_xor(l, 32);
            __syncthreads();
            if (lane < 16) sm[wave][lane] = A.m[t], sl[wave][lane] = l;
#pragma unroll
            for (int b = 0; b < D / 32; b++) {
                const float4_t u0 = A.acc[t][b][0], u1 = A.acc[t][b][1];
                float4_t *o = &so[wave][lane & 15][b * 8 + (lane >> 4) * 2];
                o[0] = float4_t{u0[0], u1[0], u0[1], u1[1]}, o[1] = float4_t{u0[2], u1[2], u0[3], u1[3]};
            }
            __syncthreads();
            const int row = threadIdx.x / 16, mr = m0 + t * 16 + row;
            if (mr < M) {
                float top = -__builtin_inff(), sum = 0, f[W];
                for (int w = 0; w < W; w++) top = fmaxf(top, sm[w][row]);
                for (int w = 0; w < W; w++) {
                    f[w] = sm[w][row] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(sm[w][row] - top);
                    sum += sl[w][row] * f[w];
                }
                const int j = by(a.by_group, mr);
                uint16_t *out = a.out + (size_t)(s.first + j) * a.out_stride + ((size_t)head * group + (mr - j * group)) * D;
                const size_t left = (size_t)slot * 16 * QT + t * 16 + row;
                if (!whole && threadIdx.x % 16 == 0) a.ml[left * 2] = top, a.ml[left * 2 + 1] = sum;
                const float inv = top == -__builtin_inff() ? 0.f : 1.f / sum; // a row that sees nothing: zeros
#pragma unroll
                for (int v = 0; v < D / 64; v++) {
                    const int at4 = v * 16 + (int)(threadIdx.x % 16);
                    float4_t o = {0, 0, 0, 0};
                    for (int w = 0; w < W; w++) o += so[w][row][at4] * f[w];
                    if (whole) {
                        half4_t h;
                        for (int k = 0; k < 4; k++) h[k] = (_Float16)(top == -__builtin_inff() ? 0.f : o[k] * inv);
                        *(half4_t *)(out + at4 * 4) = h;
                    } else *(float4_t *)(a.part + left * D + at4 * 4) = o;
                }
            }
        }
        __syncthreads();
        x += (uint32_t)(to - from);
    }
}

// Results of pairs that several workgroups share, put together by as many: of the pair's results, workgroup w takes its part, and its threads share
// what the others left of them. A pair of 256 shares (8 rows of 256 values, 131072 tokens) costs a thread two loads, as one of two shares does.
template <int QT> __device__ __forceinline__ void join_body(const qwk_attn_args &a) {
    __shared__ float4_t so[QW_WG_JOIN];
    __shared__ float sm[QW_WG_JOIN], sl[QW_WG_JOIN];
    const uint32_t D4 = a.c.dim / 4, t = threadIdx.x;
    const float neg = -__builtin_inff();
    const Part p = ((const Part *)a.parts)[blockIdx.x * 2 + blockIdx.y];
    if (!p.rows) return;
    const uint32_t np = p.w1 - p.w0 + 1, all = p.rows * D4, k = blockIdx.x - p.w0;
    const uint32_t o1 = (k + 1) * all / np;
    // one with what another left
    const auto add = [&](float &top, float &sum, float4_t &o, float mw, float lw, float4_t ow) {
        if (mw == neg) return;
        const float now = fmaxf(top, mw), f = top == neg ? 0.f : __builtin_amdgcn_exp2f(top - now), fw = __builtin_amdgcn_exp2f(mw - now);
        top = now, sum = sum * f + lw * fw, o = o * f + ow * fw;
    };
    for (uint32_t o0 = k * all / np; o0 < o1; o0 += QW_WG_JOIN) { // quads of results [o0, o1), at most as many as there are threads
        const uint32_t n = min(o1 - o0, QW_WG_JOIN), sub = t / n, mine = o0 + t - sub * n; // each by `lanes` threads
        uint32_t lanes = QW_WG_JOIN / n;
        const uint32_t row = mine / D4, at4 = mine - row * D4;
        float top = neg, sum = 0;
        float4_t o = {0, 0, 0, 0};
        if (sub < lanes)
            for (uint32_t w = p.w0 + sub; w <= p.w1; w += lanes) {
                const size_t at = ((size_t)w * 2 + (w == p.w0)) * 16 * QT + row;
                add(top, sum, o, a.ml[at * 2], a.ml[at * 2 + 1], *(const float4_t *)(a.part + at * a.c.dim + at4 * 4));
            }
        while (lanes > 1) {
            const uint32_t half = (lanes + 1) / 2;
            __syncthreads();
            if (sub >= half && sub < lanes) so[t] = o, sm[t] = top, sl[t] = sum;
            __syncthreads();
            if (sub + half < lanes) add(top, sum, o, sm[t + half * n], sl[t + half * n], so[t + half * n]);
            lanes = half;
        }
        if (t < n) {
            const int mr = (int)(p.m0 + row), j = by(a.by_group, mr);
            half4_t h;
            for (int v = 0; v < 4; v++) h[v] = (_Float16)(top == neg ? 0.f : o[v] / sum);
            *(half4_t *)(a.out + (size_t)(p.row0 + (uint32_t)j) * a.out_stride + ((size_t)p.head * a.group + (uint32_t)(mr - j * (int)a.group)) * a.c.dim + at4 * 4) = h;
        }
    }
}

#define QW_ATTN(TYPE, D, QT, PER) \
    extern "C" __global__ __launch_bounds__(QW_WG_ATTN, PER) void qwk_attn_f##TYPE##_d##D##_q##QT(qwk_attn_args a) { attn_body<TYPE, D, QT>(a); }
#define QW_ATTN_D(D, P1, P2) QW_ATTN(1, D, 1, P1) QW_ATTN(8, D, 1, P1) QW_ATTN(1, D, 2, P2) QW_ATTN(8, D, 2, P2)
QW_ATTN_D(64, 2, 2)
QW_ATTN_D(128, 2, 2)
QW_ATTN_D(192, 2, 1)
QW_ATTN_D(256, 2, 1)
#define QW_JOIN(QT) extern "C" __global__ __launch_bounds__(QW_WG_JOIN) void qwk_attn_join_q##QT(qwk_attn_args a) { join_body<QT>(a); }
QW_JOIN(1)
QW_JOIN(2)

// ---------------------------------------------------------------- rows into the cache and out of it
// The unit that holds token `token` of slot i; null: it has no page.
__device__ __forceinline__ uint8_t *unit_of(const qwk_kv &c, uint32_t i, int token, uint32_t head) {
    const uint64_t at = (uint64_t)i * c.max_pages + ((uint32_t)token >> c.page_log2);
    const uint32_t page = token < 0 ? 0xffffffffu : words(c.table)[at], pu = c.page_log2 - 4;
    return page < c.pages ? c.cache + page * c.page_bytes + (((size_t)head << pu) + ((uint32_t)token >> 4 & ((1u << pu) - 1))) * c.unit : nullptr;
}
// Where value v of token t (of its unit) lies: bytes into the unit.
template <int TYPE> __device__ __forceinline__ uint32_t place(uint32_t D, bool values, uint32_t t, uint32_t v) {
    if (TYPE == F16) return values ? 32 * D + (v / 32 * 512 + t / 4 * 128 + v % 32 * 4 + t % 4) * 2 : (v / 8 * 128 + t * 8 + v % 8) * 2;
    return values ? 17 * D + v / 64 * 1024 + t / 4 * 256 + v % 32 / 2 * 16 + v / 32 % 2 * 8 + v % 2 * 4 + t % 4 : v / 64 * 1024 + v % 32 / 8 * 256 + t * 16 + v / 32 % 2 * 8 + v % 8;
}
__device__ __forceinline__ uint32_t place_scale(uint32_t D, bool values, uint32_t t, uint32_t v) { return (values ? 33 : 16) * D + (t / 4 * (D / 32) + v / 32) * 8 + t % 4 * 2; }

__device__ __forceinline__ float half_of(uint16_t x) { return (float)__builtin_bit_cast(_Float16, x); }
__device__ __forceinline__ uint16_t half_bits(double x) { return __builtin_bit_cast(uint16_t, (_Float16)(float)x); }

// Values lane + 64 c of one head of one row: x, turned by the row's angles (cos, sin of value lane + 64 c) where they are below rot
__device__ __forceinline__ void put(const qwk_kv &c, int type, uint8_t *unit, bool values, uint32_t t, const uint16_t *x, uint32_t lane) {
    const uint32_t D = c.dim;
    for (uint32_t k = 0; k < D / 64; k++) {
        const uint32_t v = lane + 64 * k;
        if (type == F16) {
            *(uint16_t *)(unit + place<F16>(D, values, t, v)) = x[k];
            continue;
        }
        // d = max |x| / 127 of 32 values, in binary16; a code is round(x / d). Both operands of the division have 11 bits, so that its rounding to
        // 24 never crosses a border between two codes.
        const float f = half_of(x[k]);
        uint32_t b = x[k] & 0x7fff; // magnitudes order as their bits; NaN above infinity
        for (int o = 1; o < 32; o <<= 1) b = max(b, (uint32_t)__shfl_xor((int)b, o));
        const bool fine = b < 0x7c00;
        const _Float16 d = fine ? (_Float16)(half_of((uint16_t)b) / 127.f) : (_Float16)__builtin_nanf("");
        const float q = fine && (float)d > 0 ? fminf(fmaxf(rintf(f / (float)d), -127.f), 127.f) : 0.f;
        *(int8_t *)(unit + place<Q8>(D, values, t, v)) = (int8_t)q;
        if (lane % 32 == 0) *(_Float16 *)(unit + place_scale(D, values, t, v)) = d;
    }
}

// A wave a head of a row: queries, then keys, then values
__device__ __forceinline__ void kv_write_body(const qwk_kv_write_args &a, int type) {
    const qwk_kv &c = a.c;
    const uint32_t lane = threadIdx.x & 63, D = c.dim, row = blockIdx.x, h = __builtin_amdgcn_readfirstlane(blockIdx.y * (QW_WG_KV / 64) + (threadIdx.x >> 6));
    if (h >= a.q_heads + 2 * c.heads) return;
    const bool isq = h < a.q_heads, isv = h >= a.q_heads + c.heads;
    const uint32_t head = isq ? h : isv ? h - a.q_heads - c.heads : h - a.q_heads;
    uint32_t i;
    Slot s;
    if (!slot_find(c, row, i, s)) return;
    const int token = s.len - s.n + (int)row - s.first;
    uint8_t *unit = isq ? nullptr : unit_of(c, i, token, head);
    if (!isq && !unit) return;
    const uint16_t *src = isq ? a.q + (size_t)row * a.q_stride : isv ? a.v + (size_t)row * a.v_stride : a.k + (size_t)row * a.k_stride;
    src += (size_t)head * D;
    uint16_t x[4], y[4];
    const uint32_t half = a.rot / 2;
#pragma unroll
    for (uint32_t k = 0; k < 4; k++)
        if (k < D / 64) {
            const uint32_t v = lane + 64 * k;
            x[k] = src[v];
            y[k] = isv || v >= a.rot ? 0 : src[a.adjacent ? v ^ 1 : v < half ? v + half : v - half];
        }
#pragma unroll
    for (uint32_t k = 0; k < 4; k++)
        if (k < D / 64) {
            const uint32_t v = lane + 64 * k;
            if (isv || v >= a.rot) continue;
            const uint32_t p = a.adjacent ? v / 2 : v % half;
            const bool second = a.adjacent ? v & 1 : v >= half;
            const int32_t pos = a.pos[(size_t)row * a.axes + (a.axes == 1 || p < a.pairs0 ? 0 : p < a.pairs0 + a.pairs1 ? 1 : 2)];
            double sn, cs;
            sincos((double)pos * a.freq[p], &sn, &cs);
            x[k] = half_bits((double)half_of(x[k]) * cs + (second ? sn : -sn) * (double)half_of(y[k]));
        }
    if (isq) {
#pragma unroll
        for (uint32_t k = 0; k < 4; k++)
            if (k < D / 64) a.q_out[(size_t)row * a.qo_stride + (size_t)head * D + lane + 64 * k] = x[k];
    } else put(c, type, unit, isv, (uint32_t)token % 16, x, lane);
}
extern "C" __global__ __launch_bounds__(QW_WG_KV) void qwk_kv_write_f1(qwk_kv_write_args a) { kv_write_body(a, F16); }
extern "C" __global__ __launch_bounds__(QW_WG_KV) void qwk_kv_write_f8(qwk_kv_write_args a) { kv_write_body(a, Q8); }

// A wave a head of a row, keys and values
template <int TYPE> __device__ __forceinline__ void kv_read_body(const qwk_kv_read_args &a) {
    const qwk_kv &c = a.c;
    const uint32_t lane = threadIdx.x & 63, D = c.dim, row = blockIdx.x, head = __builtin_amdgcn_readfirstlane(blockIdx.y * (QW_WG_KV / 64) + (threadIdx.x >> 6));
    if (head >= c.heads) return;
    uint32_t i;
    Slot s;
    if (!slot_find(c, row, i, s)) return;
    const int token = s.len - s.n + (int)row - s.first;
    const uint8_t *unit = unit_of(c, i, token, head);
    const uint32_t t = (uint32_t)token % 16;
    for (uint32_t k = 0; k < 2 * (D / 64); k++) {
        const bool values = k >= D / 64;
        const uint32_t v = lane + 64 * (values ? k - D / 64 : k);
        uint16_t *dst = values ? a.v + (size_t)row * a.v_stride : a.k + (size_t)row * a.k_stride;
        if (!unit) { // (no page: nothing is held)
            dst[(size_t)head * D + v] = 0;
            continue;
        }
        const uint8_t *p = unit + place<TYPE>(D, values, t, v);
        dst[(size_t)head * D + v] = TYPE == F16 ? *(const uint16_t *)p
                                                : __builtin_bit_cast(uint16_t, (_Float16)((float)*(const int8_t *)p * (float)*(const _Float16 *)(unit + place_scale(D, values, t, v))));
    }
}
extern "C" __global__ __launch_bounds__(QW_WG_KV) void qwk_kv_read_f1(qwk_kv_read_args a) { kv_read_body<F16>(a); }
extern "C" __global__ __launch_bounds__(QW_WG_KV) void qwk_kv_read_f8(qwk_kv_read_args a) { kv_read_body<Q8>(a); }

#include "qw_sample.hip.h"
