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

__device__ __forceinline__ Slot slot_of(const qwk_kv &c, uint32_t i) {
    const uint32_t a = c.first[i], b = c.first[i + 1], l = c.len[i];
    const uint64_t room = (uint64_t)c.max_pages << c.page_log2;
    Slot s;
    s.first = (int)a;
    s.n = a <= b && b <= c.rows ? (int)(b - a) : 0; // what is no row of the step is not touched
    s.len = (int)(l < room ? l : room);
    return s;
}
// The slot of a row, by a whole wave in one round trip; false: it belongs to none.
__device__ __forceinline__ bool slot_find(const qwk_kv &c, uint32_t row, uint32_t &i, Slot &s) {
    i = 0;
    for (uint32_t at = 0; at < c.slots; at += 64) {
        const uint32_t k = at + (threadIdx.x & 63);
        i += (uint32_t)__popcll(__ballot(k < c.slots && c.first[k + 1] <= row));
    }
    if (i >= c.slots) return false;
    s = slot_of(c, i);
    return (int)row >= s.first && (int)row < s.first + s.n;
}
struct Range { int t0, cnt; }; // a block's first tile, and how many (at least one: an empty one still gives its rows their zeros)
template <int QT> __device__ __forceinline__ Range block_range(const Slot &s, int b, int group, int window) {
    const int M = s.n * group, j0 = b * 16 * QT / group, m1 = min((b + 1) * 16 * QT, M) - 1, j1 = m1 / group;
    const int hi = s.len - s.n + j1 + 1, lo = window ? max(0, s.len - s.n + j0 - window + 1) : 0;
    Range r;
    r.t0 = hi > 0 ? lo / (int)QW_ATTN_TILE : 0;
    r.cnt = hi > 0 ? max(1, (hi + (int)QW_ATTN_TILE - 1) / (int)QW_ATTN_TILE - r.t0) : 1;
    return r;
}
template <int QT> __device__ __forceinline__ int blocks_of(const Slot &s, int group) { return (s.n * group + 16 * QT - 1) / (16 * QT); }

struct Plan { // LDS
    uint64_t end[QW_KV_SLOTS_MAX]; // tiles of the slots up to and with this one
    uint64_t wave[4];
};
// Tiles of all slots, by the whole workgroup; returns the total.
template <int QT> __device__ uint64_t make_plan(Plan &p, const qwk_kv &c, int group, int window) {
    const uint32_t i = threadIdx.x, lane = i & 63;
    uint64_t t = 0;
    if (i < c.slots) {
        const Slot s = slot_of(c, i);
        const int nb = blocks_of<QT>(s, group);
        for (int b = 0; b < nb; b++) t += (uint64_t)block_range<QT>(s, b, group, window).cnt;
        t *= c.heads;
    }
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t o = __shfl_up(t, d);
        if (lane >= (uint32_t)d) t += o;
    }
    if (lane == 63) p.wave[i >> 6] = t;
    __syncthreads();
    for (uint32_t w = 0; w < (i >> 6); w++) t += p.wave[w];
    if (i < QW_KV_SLOTS_MAX) p.end[i] = t;
    __syncthreads();
    return p.end[QW_KV_SLOTS_MAX - 1];
}
// Shares: workgroup w of g takes the tiles [w T / g, (w + 1) T / g). No more workgroups than there are four tiles for (one a wave).
__device__ __forceinline__ uint64_t shares_of(uint64_t T, uint32_t grid) { return min((uint64_t)grid, (T + 3) / 4); }
__device__ __forceinline__ uint32_t owner_of(uint64_t x, uint64_t T, uint64_t g) { return (uint32_t)(((x + 1) * g - 1) / T); }

// Four codes -> binary16, exactly: 0x64 in front of a byte b is 1024 + b, and b is the code + 128.
__device__ __forceinline__ half4_t codes(uint32_t w) {
    w ^= 0x80808080u;
    const half2_t bias = {(_Float16)-1152.f, (_Float16)-1152.f};
    const half2_t lo = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) + bias;
    const half2_t hi = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) + bias;
    return half4_t{lo.x, lo.y, hi.x, hi.y};
}

template <int TYPE, int D> struct UnitData; // a lane's share of U units: keys or values, and their scales
template <int D> struct UnitData<F16, D> {
    uint4_t x[D / 32];
    __device__ __forceinline__ void load(const uint8_t *u, bool values, uint32_t lane) {
        const uint8_t *p = u + (values ? 32 * D : 0) + lane * 16;
#pragma unroll
        for (int c = 0; c < D / 32; c++) x[c] = *(const uint4_t *)(p + c * 1024);
    }
};
template <int D> struct UnitData<Q8, D> {
    uint4_t x[D / 64], s[D / 64];
    __device__ __forceinline__ void load(const uint8_t *u, bool values, uint32_t lane) {
        const uint8_t *p = u + (values ? 17 * D : 0);
#pragma unroll
        for (int c = 0; c < D / 64; c++) x[c] = *(const uint4_t *)(p + c * 1024 + lane * 16);
#pragma unroll
        for (int c = 0; c < D / 64; c++) s[c] = *(const uint4_t *)(p + 16 * D + (lane >> 4) * (D / 4) + c * 16);
    }
    __device__ __forceinline__ half4_t scales(int b) const { // of block b, tokens 4 (lane >> 4) + i
        return __builtin_bit_cast(half4_t, b & 1 ? uint2_t{s[b / 2].z, s[b / 2].w} : uint2_t{s[b / 2].x, s[b / 2].y});
    }
};

template <int TYPE, int D, int QT, int U> struct Attn {
    const qwk_attn_args &a;
    const uint32_t lane, wave;
    half8_t q[QT][D / 32];
    float4_t acc[QT][D / 32][2]; // result: value 32 b + 8 (lane >> 4) + 2 i + c of query lane & 15
    float m[QT], l[QT];          // reference (log2) and this lane's part of the sum
    int hi[QT], lo[QT], tok[QT]; // tokens [lo, hi) that the lane's query sees, and which of the slot's rows it is
    UnitData<TYPE, D> K[U], V[U];

    __device__ __forceinline__ void load(bool values, const uint8_t *const *u) {
#pragma unroll
        for (int i = 0; i < U; i++) (values ? V : K)[i].load(u[i], values, lane);
    }
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
    // Weights in two parts, binary16 each: together they hold 22 bits, so that the result is as exact as its own rounding. The largest weight is 2^TOP, not 1, so that the
    // small ones do not end at binary16's 2^-24: many tokens of 2^-25 of the largest's weight count for something together. (Q8_0: a weight is multiplied by a scale of up to 516.)
    static constexpr float TOP = TYPE == F16 ? 14.f : 6.f;
    __device__ __forceinline__ static void split(const float4_t &p, half4_t &h, half4_t &r) {
#pragma unroll
        for (int j = 0; j < 4; j++) h[j] = (_Float16)p[j], r[j] = (_Float16)(p[j] - (float)h[j]);
    }
    __device__ __forceinline__ half4_t values(int i, int b, int c) const {
        if constexpr (TYPE == F16) return __builtin_bit_cast(half4_t, c ? uint2_t{V[i].x[b].z, V[i].x[b].w} : uint2_t{V[i].x[b].x, V[i].x[b].y});
        else return codes(V[i].x[b / 2][(b & 1) * 2 + c]);
    }
    // key0: first token of the step's first unit; bad: units without a page; edge: some query does not see all of the step's tokens
    __device__ __forceinline__ void softmax(int key0, uint32_t bad, bool edge, float4_t (&p)[QT][U]) {
        const float neg = -__builtin_inff();
#pragma unroll
        for (int t = 0; t < QT; t++) {
#pragma unroll
            for (int i = 0; i < U; i++) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    p[t][i][j] *= a.scale;
                    if (edge) {
                        const int key = key0 + i * 16 + (int)(lane >> 4) * 4 + j;
                        if (key >= hi[t] || key < lo[t] || (bad >> i & 1)) p[t][i][j] = neg;
                    }
                }
            }
            float top = neg;
#pragma unroll
            for (int i = 0; i < U; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) top = fmaxf(top, p[t][i][j]);
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            if (__any(top > m[t])) {
                const float now = fmaxf(m[t], top), f = m[t] == neg ? 0.f : __builtin_amdgcn_exp2f(m[t] - now);
                m[t] = now;
                l[t] *= f;
#pragma unroll
                for (int b = 0; b < D / 32; b++) acc[t][b][0] *= f, acc[t][b][1] *= f;
            }
            const float ref = m[t] == neg ? 0.f : m[t] - TOP;
#pragma unroll
            for (int i = 0; i < U; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    p[t][i][j] = __builtin_amdgcn_exp2f(p[t][i][j] - ref);
                    l[t] += p[t][i][j];
                }
        }
    }
    __device__ __forceinline__ void weigh(int key0, uint32_t bad, bool edge, const float4_t (&p)[QT][U]) {
#pragma unroll
        for (int i = 0; i < U; i++) {
            const int key = key0 + i * 16 + (int)(lane >> 4) * 4;
            if constexpr (TYPE == F16) {
                half4_t h[QT], r[QT];
#pragma unroll
                for (int t = 0; t < QT; t++) split(p[t][i], h[t], r[t]);
                if (!edge) {
#pragma unroll
                    for (int b = 0; b < D / 32; b++)
#pragma unroll
                        for (int c = 0; c < 2; c++) {
                            const half4_t v = values(i, b, c);
#pragma unroll
                            for (int t = 0; t < QT; t++) {
                                acc[t][b][c] = __builtin_amdgcn_mfma_f32_16x16x16f16(v, h[t], acc[t][b][c], 0, 0, 0);
                                acc[t][b][c] = __builtin_amdgcn_mfma_f32_16x16x16f16(v, r[t], acc[t][b][c], 0, 0, 0);
                            }
                        }
                    continue;
                }
                // A token that some queries do not see may hold anything, infinities and NaN too, and 0 times those is not 0: the slot's rows
                // one after the other, each with the values that it sees and zeros in the others' place, its own columns kept
#pragma unroll
                for (int t = 0; t < QT; t++) {
                    const int j0 = __builtin_amdgcn_readfirstlane(tok[t]), j1 = __builtin_amdgcn_readlane(tok[t], 15);
                    for (int j = j0; j <= j1; j++) {
                        const int d = j - j0;
                        const int hj = __builtin_amdgcn_readfirstlane(hi[t]) + d, lj = a.window ? max(0, hj - (int)a.window) : 0;
                        const bool mine = tok[t] == j;
#pragma unroll
                        for (int b = 0; b < D / 32; b++)
#pragma unroll
                            for (int c = 0; c < 2; c++) {
                                half4_t v = values(i, b, c);
#pragma unroll
                                for (int k = 0; k < 4; k++)
                                    if (key + k >= hj || key + k < lj || (bad >> i & 1)) v[k] = (_Float16)0.f;
                                float4_t s = __builtin_amdgcn_mfma_f32_16x16x16f16(v, h[t], acc[t][b][c], 0, 0, 0);
                                s = __builtin_amdgcn_mfma_f32_16x16x16f16(v, r[t], s, 0, 0, 0);
                                if (mine) acc[t][b][c] = s;
                            }
                    }
                }
            } else {
#pragma unroll
                for (int b = 0; b < D / 32; b++) {
                    const half4_t f = V[i].scales(b);
                    const half4_t v0 = values(i, b, 0), v1 = values(i, b, 1);
#pragma unroll
                    for (int t = 0; t < QT; t++) {
                        float4_t w; // a token's scale belongs to its weight: codes are finite, so what is not seen is 0 whatever its scale
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            w[k] = p[t][i][k] * (float)f[k];
                            if (edge && (key + k >= hi[t] || key + k < lo[t] || (bad >> i & 1))) w[k] = 0.f;
                        }
                        half4_t h, r;
                        split(w, h, r);
                        acc[t][b][0] = __builtin_amdgcn_mfma_f32_16x16x16f16(v0, h, acc[t][b][0], 0, 0, 0);
                        acc[t][b][0] = __builtin_amdgcn_mfma_f32_16x16x16f16(v0, r, acc[t][b][0], 0, 0, 0);
                        acc[t][b][1] = __builtin_amdgcn_mfma_f32_16x16x16f16(v1, h, acc[t][b][1], 0, 0, 0);
                        acc[t][b][1] = __builtin_amdgcn_mfma_f32_16x16x16f16(v1, r, acc[t][b][1], 0, 0, 0);
                    }
                }
            }
        }
    }
};

template <int TYPE, int D, int QT> __device__ __forceinline__ void attn_body(const qwk_attn_args &a) {
    constexpr int U = D <= 128 ? 2 : 1, W = QW_WG_ATTN / 64, LD = D + 4; // U: units a wave has in hand; a tile is two
    __shared__ Plan plan;
    __shared__ float so[W][16][LD], sm[W][16], sl[W][16];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const qwk_kv &c = a.c;
    const int group = (int)a.group, window = (int)a.window;
    const uint64_t T = make_plan<QT>(plan, c, group, window), g = shares_of(T, a.grid);
    if (blockIdx.x >= g) return;
    uint64_t x = blockIdx.x * T / g;
    const uint64_t end = (blockIdx.x + 1) * T / g;
    while (x < end) {
        uint32_t i = 0; // the slot that tile x belongs to
        for (uint32_t step = QW_KV_SLOTS_MAX / 2; step; step >>= 1)
            if (plan.end[i + step - 1] <= x) i += step;
        const Slot s = slot_of(c, i);
        const uint64_t base = i ? plan.end[i - 1] : 0, per_head = (plan.end[i] - base) / c.heads;
        const uint32_t head = (uint32_t)((x - base) / per_head);
        uint64_t rest = x - base - head * per_head;
        int blk = 0;
        Range r = block_range<QT>(s, 0, group, window);
        while (rest >= (uint64_t)r.cnt) rest -= (uint64_t)r.cnt, r = block_range<QT>(s, ++blk, group, window);
        const int from = (int)rest, to = (int)min((uint64_t)r.cnt, rest + (end - x));
        const int M = s.n * group, m0 = blk * 16 * QT;

        Attn<TYPE, D, QT, U> A{a, lane, wave};
#pragma unroll
        for (int t = 0; t < QT; t++) {
            const int row = min(m0 + t * 16 + (int)(lane & 15), M - 1), j = row / group;
            A.tok[t] = j;
            A.hi[t] = s.len - s.n + j + 1;
            A.lo[t] = window ? max(0, A.hi[t] - window) : 0;
            A.m[t] = -__builtin_inff(), A.l[t] = 0;
            const uint16_t *q = a.q + (size_t)(s.first + j) * a.q_stride + ((size_t)head * group + (row - j * group)) * D + (lane >> 4) * 8;
#pragma unroll
            for (int k = 0; k < D / 32; k++) A.q[t][k] = *(const half8_t *)(q + k * 32);
#pragma unroll
            for (int b = 0; b < D / 32; b++) A.acc[t][b][0] = A.acc[t][b][1] = float4_t{0, 0, 0, 0};
        }
        // what every query of the block sees: [see_lo, see_hi); what some query sees ends at all_hi
        const int jl = m0 / group, jh = (min(m0 + 16 * QT, M) - 1) / group;
        const int see_hi = s.len - s.n + jl + 1, see_lo = window ? max(0, s.len - s.n + jh + 1 - window) : 0;
        const int pu = (int)c.page_log2 - 4; // log2 of a page's units
        const uint32_t *table = c.table + (size_t)i * c.max_pages;
        const size_t in_page = (size_t)head << pu;
        constexpr int STEPS = 2 / U; // of a tile
        for (int t = from + (int)wave; t < to; t += W)
            for (int h = 0; h < STEPS; h++) {
                const int key0 = (r.t0 + t) * (int)QW_ATTN_TILE + h * 16 * U;
                const uint8_t *u[U];
                uint32_t bad = 0;
#pragma unroll
                for (int k = 0; k < U; k++) {
                    const uint32_t un = (uint32_t)(key0 >> 4) + k, at = un >> pu;
                    uint32_t page = at < c.max_pages ? table[at] : 0xffffffffu;
                    if (page >= c.pages) bad |= 1u << k, page = 0;
                    u[k] = c.cache + page * c.page_bytes + (in_page + (un & ((1u << pu) - 1))) * c.unit;
                }
                A.load(false, u);
                A.load(true, u);
                const bool edge = bad || key0 < see_lo || key0 + 16 * U > see_hi;
                float4_t p[QT][U];
#pragma unroll
                for (int q = 0; q < QT; q++)
#pragma unroll
                    for (int k = 0; k < U; k++) p[q][k] = A.scores(q, k);
                A.softmax(key0, bad, edge, p);
                A.weigh(key0, bad, edge, p);
            }
        // the waves' results together, in the waves' order
        const bool whole = from == 0 && to == r.cnt;
        const size_t slot = (size_t)blockIdx.x * 2 + (from == 0);
#pragma unroll
        for (int t = 0; t < QT; t++) {
            float l = A.l[t];
            l += __shfl_xor(l, 16);
            l += __shfl_xor(l, 32);
            __syncthreads();
            if (lane < 16) sm[wave][lane] = A.m[t], sl[wave][lane] = l;
#pragma unroll
            for (int b = 0; b < D / 32; b++)
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    float *o = &so[wave][lane & 15][b * 32 + (lane >> 4) * 8 + 2 * k];
                    o[0] = A.acc[t][b][0][k], o[1] = A.acc[t][b][1][k];
                }
            __syncthreads();
            const int row = threadIdx.x / 16, mr = m0 + t * 16 + row, v0 = (int)(threadIdx.x % 16) * (D / 16);
            if (mr < M) {
                float top = -__builtin_inff(), sum = 0, f[W];
                for (int w = 0; w < W; w++) top = fmaxf(top, sm[w][row]);
                for (int w = 0; w < W; w++) {
                    f[w] = sm[w][row] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(sm[w][row] - top);
                    sum += sl[w][row] * f[w];
                }
                const int j = mr / group;
                uint16_t *out = a.out + (size_t)(s.first + j) * a.out_stride + ((size_t)head * group + (mr - j * group)) * D + v0;
                float *part = a.part + (slot * 16 * QT + t * 16 + row) * D + v0;
                if (!whole && v0 == 0) a.ml[(slot * 16 * QT + t * 16 + row) * 2] = top, a.ml[(slot * 16 * QT + t * 16 + row) * 2 + 1] = sum;
                const float inv = top == -__builtin_inff() ? 0.f : 1.f / sum; // a row that sees nothing: zeros
                for (int v = 0; v < D / 16; v++) {
                    float o = 0;
                    for (int w = 0; w < W; w++) o += so[w][row][v0 + v] * f[w];
                    if (whole) out[v] = __builtin_bit_cast(uint16_t, (_Float16)(top == -__builtin_inff() ? 0.f : o * inv));
                    else part[v] = o;
                }
            }
        }
        __syncthreads();
        x += (uint64_t)(to - from);
    }
}

// Results of pairs that several workgroups share, put together: a workgroup a row, query head and 64 values. Its sixteen groups of threads
// take the partial results in turn.
template <int QT> __device__ __forceinline__ void join_body(const qwk_attn_args &a) {
    __shared__ Plan plan;
    __shared__ float so[16][64], sm[16], sl[16];
    const qwk_kv &c = a.c;
    const int group = (int)a.group, window = (int)a.window, D = (int)c.dim;
    const uint64_t T = make_plan<QT>(plan, c, group, window), g = shares_of(T, a.grid);
    const uint32_t row = blockIdx.x, qh = blockIdx.z;
    uint32_t i;
    Slot s;
    if (!slot_find(c, row, i, s)) return;
    const uint32_t head = qh / a.group;
    const int mr = ((int)row - s.first) * group + (int)(qh % a.group), blk = mr / (16 * QT);
    const uint64_t base = i ? plan.end[i - 1] : 0, per_head = (plan.end[i] - base) / c.heads;
    uint64_t x = base + head * per_head;
    Range r = block_range<QT>(s, 0, group, window);
    for (int b = 0; b < blk; b++) x += (uint64_t)r.cnt, r = block_range<QT>(s, b + 1, group, window);
    const uint32_t w0 = owner_of(x, T, g), w1 = owner_of(x + (uint64_t)r.cnt - 1, T, g);
    if (w0 == w1) return; // written already
    const int sub = threadIdx.x / 16, v0 = (int)blockIdx.y * 64 + (int)(threadIdx.x % 16) * 4;
    const float neg = -__builtin_inff();
    float top = neg, sum = 0;
    float4_t o = {0, 0, 0, 0};
    for (uint32_t w = w0 + (uint32_t)sub; w <= w1; w += 16) {
        const size_t at = ((size_t)w * 2 + (w == w0)) * 16 * QT + (mr - blk * 16 * QT);
        const float mw = a.ml[at * 2], lw = a.ml[at * 2 + 1];
        const float4_t ow = *(const float4_t *)(a.part + at * D + v0);
        if (mw == neg) continue;
        const float now = fmaxf(top, mw), f = top == neg ? 0.f : __builtin_amdgcn_exp2f(top - now), fw = __builtin_amdgcn_exp2f(mw - now);
        top = now, sum = sum * f + lw * fw, o = o * f + ow * fw;
    }
    *(float4_t *)&so[sub][(threadIdx.x % 16) * 4] = o;
    if (threadIdx.x % 16 == 0) sm[sub] = top, sl[sub] = sum;
    __syncthreads();
    if (threadIdx.x >= 64) return;
    top = neg, sum = 0;
    for (int k = 0; k < 16; k++) top = fmaxf(top, sm[k]);
    float v = 0;
    for (int k = 0; k < 16; k++) {
        if (sm[k] == neg) continue;
        const float f = __builtin_amdgcn_exp2f(sm[k] - top);
        sum += sl[k] * f, v += so[k][threadIdx.x] * f;
    }
    a.out[(size_t)row * a.out_stride + (size_t)qh * D + blockIdx.y * 64 + threadIdx.x] = __builtin_bit_cast(uint16_t, (_Float16)(top == neg ? 0.f : v / sum));
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
    const uint32_t page = token < 0 ? 0xffffffffu : c.table[at], pu = c.page_log2 - 4;
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
