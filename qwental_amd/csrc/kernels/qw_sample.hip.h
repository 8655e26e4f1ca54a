// A token a row from logits, under temperature, top-k, top-p and min-p (include/qw_attn.h).
//
// The filters all keep the first few of the tokens in descending order (equal logits by their number), so that together they are one border: a
// logit, and of the tokens that have exactly that one the first few. It is found by selecting digits of the logits' bits, eight at a time, from
// histograms of counts (top-k) or weights (top-p); nothing is sorted. Weights are whole numbers, 2^43 times exp((l - max) / temperature): their sums do
// not depend on the order in which they are made, so neither does the token.
// Bits that order as the logits do; 0 for NaN, which is never drawn (nor is minus infinity: its weight is 0).
__device__ __forceinline__ uint32_t key_of(float l) {
    const uint32_t b = __builtin_bit_cast(uint32_t, l + 0.f); // (-0 is 0)
    return l != l ? 0 : b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __builtin_bit_cast(float, k >> 31 ? k & 0x7fffffffu : ~k); }
constexpr uint32_t KEY_LOWEST = 0x007fffffu; // minus infinity

struct Weigh { // of a row: weights of its tokens
    double top, c; // largest logit, log2(e) / temperature
    bool inf;      // the largest is infinity: such tokens share all of it
    __device__ __forceinline__ u64 operator()(float l) const {
        if (inf) return l == __builtin_inff() ? 1ull << 43 : 0;
        const double x = ((double)l - top) * c; // in 64 bits: a 24-bit product would cost a small weight its last digits
        if (!(x > -64.)) return 0;
        const float i = __builtin_rintf((float)x), f = __builtin_amdgcn_exp2f((float)(x - (double)i));
        return (u64)__builtin_ldexpf(f, (int)i + 43);
    }
};

constexpr uint32_t COPIES = 16; // of a histogram: lanes that meet in one bin take different banks
struct SampleShared {
    uint32_t count[256][COPIES];
    u64 weight[256][COPIES];
    u64 scan[2][256], tile[QW_SAMPLE_VOCAB / QW_SAMPLE_TILE], part[16];
    uint32_t pick, n;
    u64 before, total, w;
};

// One digit: of the tokens for which digit_of gives one (a number up to 255; others ~0), the largest digit d such that tokens of larger ones have less than
// `want` (of counts or weights) between them. Leaves d in pick, what the larger ones have in before, the digit's count in n, all digits' in total.
template <bool WEIGHTS, class F> __device__ void select_digit(SampleShared &s, const qwk_sample_args &a, const float *l, const Weigh &weigh, u64 want, float part, F digit_of) {
    const uint32_t t = threadIdx.x;
    for (uint32_t i = t; i < 256 * COPIES; i += QW_WG_SAMPLE) {
        (&s.count[0][0])[i] = 0;
        if (WEIGHTS) (&s.weight[0][0])[i] = 0;
    }
    __syncthreads();
    for (uint32_t i = t; i < a.vocab; i += QW_WG_SAMPLE) {
        const float x = l[i];
        const uint32_t d = digit_of(i, key_of(x));
        if (d > 255) continue;
        atomicAdd(&s.count[d][t % COPIES], 1u);
        if (WEIGHTS) atomicAdd(&s.weight[d][t % COPIES], weigh(x));
    }
    __syncthreads();
    uint32_t n = 0;
    u64 w = 0;
    if (t < 256) { // digits from the largest down
        for (uint32_t i = 0; i < COPIES; i++) n += s.count[255 - t][(i + t) % COPIES], w += WEIGHTS ? s.weight[255 - t][(i + t) % COPIES] : 0;
        if (!WEIGHTS) w = n;
        s.scan[0][t] = w;
    }
    __syncthreads();
    uint32_t from = 0;
    for (uint32_t d = 1; d < 256; d <<= 1, from ^= 1) {
        if (t < 256) s.scan[from ^ 1][t] = s.scan[from][t] + (t >= d ? s.scan[from][t - d] : 0);
        __syncthreads();
    }
    if (part > 0) { // want is a share of the whole
        const u64 all = s.scan[from][255] - want;
        want = (u64)ceil((double)part * (double)all);
        want = want < 1 ? 1 : want > all ? all : want;
    }
    if (t < 256 && s.scan[from][t] >= want && s.scan[from][t] - w < want) s.pick = 255 - t, s.n = n, s.before = s.scan[from][t] - w, s.total = want;
    __syncthreads();
}

__device__ __forceinline__ void sample_row(SampleShared &s, const qwk_sample_args &a, uint32_t row) {
    const float *l = a.logits + (size_t)row * a.stride;
    const qwk_sample_row p = a.p[row];
    const uint32_t t = threadIdx.x, lane = t & 63, wave = t >> 6;
    // the largest logit, and the first token that has it
    u64 best = 0;
    for (uint32_t i = t; i < a.vocab; i += QW_WG_SAMPLE) {
        const u64 k = (u64)key_of(l[i]) << 32 | ~i;
        best = k > best ? k : best;
    }
    for (int d = 32; d; d >>= 1) {
        const u64 o = __shfl_xor(best, d);
        best = o > best ? o : best;
    }
    if (lane == 0) s.part[wave] = best;
    __syncthreads();
    for (uint32_t i = 0; i < QW_WG_SAMPLE / 64; i++) best = s.part[i] > best ? s.part[i] : best;
    const uint32_t top = (uint32_t)(best >> 32), first = ~(uint32_t)best;
    if (top <= KEY_LOWEST || !(p.temperature > 0)) { // nothing to draw from, or no chance in it
        if (t == 0) a.ids[row] = top <= KEY_LOWEST ? 0xffffffffu : first;
        if (t == 0 && a.probs) a.probs[row] = top <= KEY_LOWEST ? 0.f : 1.f;
        return;
    }
    const Weigh weigh = {(double)of_key(top), 1.4426950408889634 / (double)p.temperature, of_key(top) == __builtin_inff()};
    uint32_t border = KEY_LOWEST + 1, equal = 0, keep = 0; // tokens above `border`, and the first `keep` of the `equal` ones that lie on it (equal 0: all of them)
    if (p.top_k && p.top_k < a.vocab) {
        uint32_t prefix = 0;
        u64 want = p.top_k;
        for (int shift = 24; shift >= 0; shift -= 8) {
            select_digit<false>(s, a, l, weigh, want, 0, [&](uint32_t, uint32_t k) { return shift == 24 || k >> (shift + 8) == prefix ? k >> shift & 255 : ~0u; });
            prefix = prefix << 8 | s.pick, want -= s.before;
            __syncthreads();
        }
        border = prefix, equal = s.n, keep = (uint32_t)want;
        if (border <= KEY_LOWEST) border = KEY_LOWEST + 1, equal = 0;
    }
    if (p.top_p < 1) {
        uint32_t prefix = 0;
        const u64 over = equal ? (u64)(equal - keep) * weigh(of_key(border)) : 0; // of those on the border, top-k has left some out
        u64 want = over;
        for (int shift = 24; shift >= 0; shift -= 8) {
            select_digit<true>(s, a, l, weigh, want, shift == 24 ? fmaxf(p.top_p, 1e-30f) : 0, [&](uint32_t, uint32_t k) { return k >= border && (shift == 24 || k >> (shift + 8) == prefix) ? k >> shift & 255 : ~0u; });
            prefix = prefix << 8 | s.pick, want = s.total - s.before;
            __syncthreads();
        }
        const u64 each = weigh(of_key(prefix)), need = each ? (want + each - 1) / each : s.n;
        const uint32_t most = equal && prefix == border ? keep : s.n;
        border = prefix, equal = s.n, keep = need < most ? (uint32_t)need : most;
    }
    uint32_t last = a.vocab; // of those on the border, the last one's number
    if (equal && keep < equal) {
        uint32_t prefix = 0;
        u64 want = keep;
        for (int shift = 16; shift >= 0; shift -= 8) { // numbers from the smallest up: complements from the largest down
            select_digit<false>(s, a, l, weigh, want, 0, [&](uint32_t i, uint32_t k) { return k == border && (shift == 16 || (~i & 0xffffff) >> (shift + 8) == prefix) ? (~i & 0xffffff) >> shift & 255 : ~0u; });
            prefix = prefix << 8 | s.pick, want -= s.before;
            __syncthreads();
        }
        last = ~prefix & 0xffffff;
    }
    const u64 least = p.min_p > 0 ? (u64)((double)fminf(p.min_p, 1.f) * 0x1p43) : 0;
    const auto weight = [&](uint32_t i) -> u64 {
        if (i >= a.vocab) return 0;
        const float x = l[i];
        const uint32_t k = key_of(x);
        if (k < border || (k == border && i > last)) return 0;
        const u64 w = weigh(x);
        return w < least ? 0 : w;
    };
    // sums of tiles, then the one that the draw falls into, token by token
    const uint32_t tiles = (a.vocab + QW_SAMPLE_TILE - 1) / QW_SAMPLE_TILE;
    for (uint32_t i = t; i < tiles; i += QW_WG_SAMPLE) s.tile[i] = 0;
    __syncthreads();
    for (uint32_t i = 0; i < tiles; i++) {
        u64 w = 0;
        for (uint32_t k = 0; k < QW_SAMPLE_TILE; k += QW_WG_SAMPLE) w += weight(i * QW_SAMPLE_TILE + k + t);
        for (int d = 32; d; d >>= 1) w += __shfl_xor(w, d);
        if (lane == 0) atomicAdd(&s.tile[i], w);
    }
    __syncthreads();
    u64 all = 0, below = 0;
    for (uint32_t i = 0; i < tiles; i++) all += s.tile[i];
    const double u = (double)a.u[row];
    const u64 at = u > 0 ? min((u64)(u * (double)all), all - 1) : 0; // the first token whose sum with those before it is larger
    uint32_t tile = 0;
    while (below + s.tile[tile] <= at) below += s.tile[tile++];
    u64 w[QW_SAMPLE_TILE / QW_WG_SAMPLE], sum = 0;
    const uint32_t base = tile * QW_SAMPLE_TILE + t * (QW_SAMPLE_TILE / QW_WG_SAMPLE);
    for (uint32_t k = 0; k < QW_SAMPLE_TILE / QW_WG_SAMPLE; k++) sum += w[k] = weight(base + k);
    u64 up = sum;
    for (uint32_t d = 1; d < 64; d <<= 1) {
        const u64 o = __shfl_up(up, d);
        if (lane >= d) up += o;
    }
    if (lane == 63) s.part[wave] = up;
    __syncthreads();
    for (uint32_t i = 0; i < wave; i++) up += s.part[i];
    u64 c = below + up - sum;
    if (c <= at && at < c + sum)
        for (uint32_t k = 0; k < QW_SAMPLE_TILE / QW_WG_SAMPLE; c += w[k++])
            if (c <= at && at < c + w[k]) {
                a.ids[row] = base + k;
                if (a.probs) a.probs[row] = (float)((double)w[k] / (double)all);
            }
}
extern "C" __global__ __launch_bounds__(QW_WG_SAMPLE) void qwk_sample(qwk_sample_args a) {
    __shared__ SampleShared s;
    sample_row(s, a, blockIdx.x);
}
