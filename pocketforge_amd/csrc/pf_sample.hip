// Tokens from rows of logits (pf_sample_rows of include/pf_gpu.h): temperature,
// top-k, top-p and min-p, from given random numbers.
//
// With the tokens in order of their logits (equal ones by number) each filter
// keeps a beginning of that order, so the kept set is a mass S = min(M_k, M_p,
// M_m): of the first k, of the first that reach p M_k, of those that weigh min_p.
// The token is the first whose cumulative weight exceeds u S.
//
// Two launches.  Workgroups of a slice of a row each read it once, into
// registers: its largest logit, its largest few tokens, those above a bound that
// the threads' own maxima give, and the sum of the others' weights.  What lies
// above the largest of these bounds, over all slices, is the beginning of the
// order: a thousand tokens or the top-k and some more.  A workgroup for each row
// finds the borders and the token among them, by a histogram and the order of the
// bins that the borders are in.  Where one lies further on, as in flat rows, it
// does the same over what is below the listed tokens, and where these do not fit
// or that has more equal logits than it can sort, over the whole row, digit by
// digit.  A row that one workgroup's registers hold takes one launch.
//
// Weights of listed tokens are whole numbers, exp((l - max) / T) in steps of 2^-43,
// so that sums are exact, whatever the order in which threads add to them: up to
// 2^20 tokens of up to 2^43 fit 64 bits, and what a step leaves of 2^20 sums is
// 2^-24 of the largest weight, what sums of fp32 would lose of the first few.
// The others', each below a thousandth of the row's or so, are fp32's: in fp64 they
// would be most of a slice's time.  A thread adds its own 16 or 32 of them, two by two
// within a chunk, and these sums are added as whole numbers.  Where o octaves lie
// between a weight and the largest, the logits' difference rounds and its product with
// the scale does, by 2^-24 o each; a weight is off by ln 2 times that and by exp2's
// 2^-23, a thread's sum by nine additions' 2^-24.  2^20 tokens that far down weigh
// r = 2^(20 - o) of the largest, so that all is off by r / (1 + r) (1.39 o + 11) 2^-24,
// which is 31.3 2^-24 at most (o = 16): less than 2^-19 of what stays.  (A slice's o
// is from its own largest, of 8192 tokens, a one-launch row has 2^15: 25 2^-24.)
#include "pf_attend.h"
#include "pf_context.h"

namespace pf {

constexpr int BINS = 1024;
constexpr float BIN_OCTAVES = 44.0f;   // of the weights, that the bins cover (the last one has the rest)
constexpr uint32_t LIST = 2048;        // tokens that are sorted at once
// top-k up to here needs no sums over the row.  Beyond it a row lists no more tokens,
// so its border takes the whole row (`Pick`), by one workgroup: one row of 130560 bf16
// logits 94 us, 14 with a top-k of 1000; 5 of 16384 fp32 ones 28 and 11.
constexpr uint32_t FEW_K = 1024;
constexpr double STEPS = 8796093022208.0;   // 2^43
constexpr double WHOLE = 6755399441055744.0;   // 2^52 + 2^51: what is added to it is whole, in its low bits

struct SampleArgs {
    const void* logits;
    const float *u, *temperature, *top_p, *min_p;   // of each row, or NULL
    const int32_t* top_k;
    float temperature1, top_p1, min_p1;
    uint32_t top_k1;
    uint32_t rows, vocab, stride, slices, room;   // room: listed tokens of a slice at most
    int32_t* tokens;
    float* probs;
    struct Slice* ws_slice;       // [rows][slices]
    uint64_t* ws_list;            // [rows][slices][room]
};

// What a slice's workgroup found: the largest logit and its first token, the bound
// from which on tokens are listed, their number (more than the room: not all of
// them are), and the weight of the others beside the largest logit's.
struct Slice {
    uint64_t rest;
    float max;
    int32_t first;
    float bound;
    uint32_t listed;
};

// A row in chunks of 16 bytes from the last multiple of 16 on; what lies before its
// first or behind its last token reads as -infinity.  (Masked tokens are those that
// do not compare above -infinity, so NaN too.)
template <int T>
struct Row {
    static constexpr int E = T == PF_TYPE_F32 ? 4 : 8;
    const uint8_t* at;            // first chunk
    int skip, n;                  // tokens of it before the row; tokens
    uint32_t chunks;
    __device__ __forceinline__ Row(const SampleArgs& a, uint32_t row) {
        const uint8_t* p = (const uint8_t*)a.logits + (size_t)row * a.stride * act_size<T>;
        skip = (int)((uintptr_t)p & 15) / act_size<T>;
        at = p - skip * act_size<T>;
        n = (int)a.vocab;
        chunks = (uint32_t)(skip + n + E - 1) / E;
    }
    // tokens E c - skip ..
    __device__ __forceinline__ u4v raw(uint32_t c) const {
        const int t0 = (int)(c * E) - skip;
        if (t0 >= 0 && t0 + E <= n) return *(const u4v*)(at + (size_t)c * 16);
        u4v w;
#pragma unroll
        for (int i = 0; i < E; i++) {
            const bool in = t0 + i >= 0 && t0 + i < n;
            if constexpr (T == PF_TYPE_F32) {
                w[i] = in ? ((const uint32_t*)at)[t0 + i + skip] : 0xFF800000u;
            } else {
                const uint32_t v = in ? ((const uint16_t*)at)[t0 + i + skip] : T == PF_TYPE_BF16 ? 0xFF80u : 0xFC00u;
                w[i / 2] = i % 2 ? w[i / 2] | v << 16 : v;
            }
        }
        return w;
    }
    static __device__ __forceinline__ float value(u4v w, int i) {
        if constexpr (T == PF_TYPE_F32) return __builtin_bit_cast(float, (uint32_t)w[i]);
        else if constexpr (T == PF_TYPE_BF16) return __builtin_bit_cast(float, i % 2 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
        else return (float)__builtin_bit_cast(_Float16, (uint16_t)(w[i / 2] >> (i % 2 * 16)));
    }
    __device__ __forceinline__ float one(int32_t token) const {
        if constexpr (T == PF_TYPE_F32) return ((const float*)at)[skip + token];
        else return to_float<T>(((const short*)at)[skip + token]);
    }
    // A workgroup of THREADS goes through the row, with many loads under way: f(chunks,
    // the first one's first token, a bit for each token that is in range); a thread's
    // chunks lie THREADS apart.
    template <int THREADS, class F>
    __device__ __forceinline__ void batches(F&& f) const {
        constexpr int U = 8;
        for (uint32_t c0 = threadIdx.x; c0 - threadIdx.x < chunks; c0 += U * THREADS) {
            u4v w[U];
            uint64_t in = 0;
#pragma unroll
            for (int u = 0; u < U; u++) {
                w[u] = (u4v)0u;
                if (c0 + u * THREADS < chunks) {
                    w[u] = raw(c0 + u * THREADS);
                    in |= ((1ull << E) - 1) << (u * E);
                }
            }
            f(w, (int32_t)(c0 * E) - skip, in);
        }
    }
    // f(value, token) of each
    template <int THREADS, class F>
    __device__ __forceinline__ void each(F&& f) const {
        batches<THREADS>([&](const auto& w, int32_t t0, uint64_t in) {
            constexpr int U = sizeof(w) / sizeof(u4v);
#pragma unroll
            for (int u = 0; u < U; u++)
                if (in >> (u * E) & 1)
#pragma unroll
                    for (int i = 0; i < E; i++) f(value(w[u], i), t0 + u * THREADS * E + i);
        });
    }
};

// A row's settings.
struct Setting {
    float max;
    int32_t first;                // the largest logit's token, -1: none
    bool greedy;
    uint32_t k;                   // 0: off
    double scale, p, least;       // log2(e) / T; p >= 1: off; min_p in steps, 0: off
    float to_bin, hi, lo;
    float far;                    // distance to the largest at which nothing weighs any more
    bool plain;
    bool few;                     // top-k alone decides how far to look: no sums over the row
    __device__ __forceinline__ void of(const SampleArgs& a, uint32_t row) {
        const float t = a.temperature ? a.temperature[row] : a.temperature1;
        const float pp = a.top_p ? a.top_p[row] : a.top_p1, m = a.min_p ? a.min_p[row] : a.min_p1;
        const int64_t kk = a.top_k ? (int64_t)a.top_k[row] : (int64_t)a.top_k1;
        greedy = !(t > 0.0f);
        k = kk > 0 && kk < (int64_t)a.vocab ? (uint32_t)kk : 0u;
        p = pp < 1.0f ? (double)pp : 1.0;
        least = m > 0.0f ? (double)fminf(m, 1.0f) * STEPS : 0.0;
        scale = 1.4426950408889634074 / (double)t;
        to_bin = fminf((float)(scale * (BINS / BIN_OCTAVES)), 3e38f);
        few = k && k <= FEW_K;
    }
    __device__ __forceinline__ int bin(float l) const {
        const float d = l == max ? 0.0f : max - l;
        return (int)fminf(d * to_bin, (float)(BINS - 1));      // (rounded alike for all: the order stays)
    }
    // (l - max) / T in octaves, as far as weights reach
    __device__ __forceinline__ double octaves(float l) const {
        return l == max ? 0.0 : fmax(((double)l - (double)max) * scale, -60.0);
    }
    // the same in fp32, where `plain`: off by 2^-23 of itself at most, to either side
    __device__ __forceinline__ void fp32() {
        hi = (float)scale;
        lo = (float)(scale - (double)hi);
        far = -1024.0f * __builtin_amdgcn_rcpf(hi);
        plain = max < INFINITY && hi > 1e-30f && hi < 1e30f;
    }
    // (1024 octaves and more, masked tokens among them, are 1024: beside a small
    // temperature's hi a larger distance's product with lo would be an infinity, of
    // either sign)
    __device__ __forceinline__ float distance32(float l) const { return fmaxf(l - max, far); }
    __device__ __forceinline__ float octaves32(float l) const {
        const float d = distance32(l);
        return fmaf(d, hi, d * lo);
    }
    // 2^43 2^x to the nearest whole number: 2^x = 2^n e^(f ln 2) with |f| <= 1/2, the
    // series up to z^11 (z^12 / 12! = 6e-15, 2^-47)
    static __device__ __forceinline__ uint64_t weight_of(double x) {
        const double t = x + WHOLE;
        const double z = (x - (t - WHOLE)) * 0.69314718055994530942;
        double y = 1.0 / 39916800.0;
        y = fma(y, z, 1.0 / 3628800.0);
        y = fma(y, z, 1.0 / 362880.0);
        y = fma(y, z, 1.0 / 40320.0);
        y = fma(y, z, 1.0 / 5040.0);
        y = fma(y, z, 1.0 / 720.0);
        y = fma(y, z, 1.0 / 120.0);
        y = fma(y, z, 1.0 / 24.0);
        y = fma(y, z, 1.0 / 6.0);
        y = fma(y, z, 0.5);
        y = fma(y, z, 1.0);
        y = fma(y, z, 1.0);
        // times 2^(n + 43), by its exponent; added to 2^52 a number is whole in the last place
        const uint64_t n = __builtin_bit_cast(uint64_t, t) + 43;
        const double w = __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, y) + (n << 52)) + 4503599627370496.0;
        return __builtin_bit_cast(uint64_t, w) - 0x4330000000000000ull;
    }
    __device__ __forceinline__ uint64_t weight(float l) const { return weight_of(octaves(l)); }
};

// Larger logits first: the value as an integer that falls with it.
__device__ __forceinline__ uint32_t falling(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);       // (-0 is 0)
    return u & 0x80000000u ? u : ~(u | 0x80000000u);
}
__device__ __forceinline__ float falling_value(uint32_t k) {
    return __builtin_bit_cast(float, k & 0x80000000u ? k : ~k & 0x7FFFFFFFu);
}

constexpr int32_t NO_TOKEN = 0x7FFFFFFF;

// Over a wave, by the adders' own lane shifts: rows of 16 lanes, then row to row.
// Lanes that a shift does not reach take `none`.
template <class F>
__device__ __forceinline__ uint32_t wave_fold(uint32_t v, uint32_t none, F&& f) {
    v = f(v, (uint32_t)__builtin_amdgcn_update_dpp((int)none, (int)v, 0x111, 0xf, 0xf, false));
    v = f(v, (uint32_t)__builtin_amdgcn_update_dpp((int)none, (int)v, 0x112, 0xf, 0xf, false));
    v = f(v, (uint32_t)__builtin_amdgcn_update_dpp((int)none, (int)v, 0x114, 0xf, 0xf, false));
    v = f(v, (uint32_t)__builtin_amdgcn_update_dpp((int)none, (int)v, 0x118, 0xf, 0xf, false));
    v = f(v, (uint32_t)__builtin_amdgcn_update_dpp((int)none, (int)v, 0x142, 0xa, 0xf, false));
    return f(v, (uint32_t)__builtin_amdgcn_update_dpp((int)none, (int)v, 0x143, 0xc, 0xf, false));
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {   // with its own
    return wave_fold(v, 0u, [](uint32_t a, uint32_t b) { return a + b; });
}
__device__ __forceinline__ uint32_t wave_least(uint32_t v) {
    v = wave_fold(v, ~0u, [](uint32_t a, uint32_t b) { return min(a, b); });
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ float wave_max(float v) {
    const uint32_t m = wave_fold(__builtin_bit_cast(uint32_t, v), 0xFF800000u, [](uint32_t a, uint32_t b) {
        return __builtin_bit_cast(uint32_t, fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)));
    });
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane((int)m, 63));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp64(uint64_t v) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL, ROWS, 0xf, false);
    return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ uint64_t wave_scan64(uint64_t v) {
    v += dpp64<0x111, 0xf>(v);
    v += dpp64<0x112, 0xf>(v);
    v += dpp64<0x114, 0xf>(v);
    v += dpp64<0x118, 0xf>(v);
    v += dpp64<0x142, 0xa>(v);
    return v + dpp64<0x143, 0xc>(v);
}
__device__ __forceinline__ uint64_t lane64(uint64_t v, int lane) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
}
__device__ __forceinline__ uint64_t wave_sum64(uint64_t v) { return lane64(wave_scan64(v), 63); }

// Two by two: the sum of eight rounds three times, not seven.
template <int N>
__device__ __forceinline__ float sum_pairs(float (&v)[N]) {
#pragma unroll
    for (int w = 1; w < N; w *= 2)
#pragma unroll
        for (int i = 0; i + w < N; i += 2 * w) v[i] += v[i + w];
    return v[0];
}

// A wave's c-th largest of its lanes' values, to 16 bits (the next lower such
// value), as an integer that rises with it; 0 where fewer than c are above -infinity.
__device__ __forceinline__ uint32_t nth_of_wave(float v, uint32_t c) {
    const uint32_t key = v == -INFINITY ? 0u : ~falling(v);
    uint32_t found = 0;
#pragma unroll
    for (int b = 31; b >= 16; b--) {
        const uint32_t to = found | 1u << b;
        if ((uint32_t)__popcll(__ballot(key >= to)) >= c) found = to;
    }
    return found;
}

// A slice: N chunks a thread.  The bound is the mean of the four waves' c-th
// largest lanes: of n listed tokens over 256 threads a thread has one with the
// probability 1 - e^(-n / 256), so c = 64 of that gives about n.  64 rows of 130560
// bf16 logits: 17 MB in 10 us; some ten instructions and an exponential a token are
// half of it, the launch and the loads' round trip most of the rest.
template <int T, int N>
__global__ __launch_bounds__(256) void k_sample_slice(SampleArgs a) {
    constexpr int E = Row<T>::E;
    __shared__ float s_max[4];
    __shared__ uint32_t s_bound[4], s_listed, s_first;
    __shared__ uint64_t s_mass[4];
    __shared__ float s_x[N * E][256];
    const uint32_t row = blockIdx.y, t = threadIdx.x, wave = t >> 6;
    if (t == 0) {
        s_listed = 0;
        s_first = NO_TOKEN;
    }
    const Row<T> r(a, row);
    // (chunks in turn: every slice has its share of each part of the vocabulary)
    float x[N][E], top = -INFINITY;
    const auto chunk = [&](int n) { return (blockIdx.x + a.slices * n) * 256 + t; };
    const auto token = [&](int n, int i) { return (int32_t)(chunk(n) * E) - r.skip + i; };
#pragma unroll
    for (int n = 0; n < N; n++) {
        u4v w = {};
        const bool in = chunk(n) < r.chunks;
        if (in) w = r.raw(chunk(n));
#pragma unroll
        for (int i = 0; i < E; i++) x[n][i] = in ? Row<T>::value(w, i) : -INFINITY;
    }
    Setting s;
    s.of(a, row);
#pragma unroll
    for (int n = 0; n < N; n++)
#pragma unroll
        for (int i = 0; i < E; i++) top = fmaxf(top, x[n][i]);
    // how many tokens are wanted of the row: top-k's and some more, or a thousand
    const float want = s.greedy ? 0.0f : fminf((s.few ? 1.5f * (float)s.k : 1024.0f) + 16.0f * (float)a.slices, 1700.0f);
    const uint32_t c = (uint32_t)(64.0f * (1.0f - __builtin_amdgcn_exp2f(want / (float)a.slices * (-1.4426950f / 256.0f)))) + 1;
    const uint32_t nth = nth_of_wave(top, min(c, 60u));
    const float wave_top = wave_max(top);
    if ((t & 63) == 0) {
        s_max[wave] = wave_top;
        s_bound[wave] = nth;
    }
    __syncthreads();
    s.max = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
    if (s.max > -INFINITY && wave_top == s.max) {
        uint32_t first = NO_TOKEN;
#pragma unroll
        for (int n = N - 1; n >= 0; n--)
#pragma unroll
            for (int i = E - 1; i >= 0; i--)
                if (x[n][i] == s.max) first = (uint32_t)token(n, i);
        first = wave_least(first);
        if ((t & 63) == 0) atomicMin(&s_first, first);
    }
    float bound = -INFINITY;
    uint64_t mass = 0;
    if (!s.greedy && s.max > -INFINITY) {
        uint64_t sum = 0;
        uint32_t some = 0;
#pragma unroll
        for (int w = 0; w < 4; w++) {
            sum += s_bound[w];
            some += s_bound[w] != 0;
        }
        if (some) bound = falling_value(~(uint32_t)(sum / some));
        // a bit for each of the thread's tokens that are listed; the values to LDS, where
        // a number picks one
        const float above = fmaxf(bound, -3.4028234663852886e38f);
        uint32_t hits = 0;
        // (the others' weights in fp32)
        s.fp32();
        float rest = 0.0f;
#pragma unroll
        for (int n = 0; n < N; n++) {
            float w[E];
#pragma unroll
            for (int i = 0; i < E; i++) {
                const bool hit = x[n][i] >= above;
                hits |= (hit ? 1u : 0u) << (n * E + i);
                s_x[n * E + i][t] = x[n][i];
                if (!s.few) w[i] = __builtin_amdgcn_exp2f(hit ? -INFINITY : s.octaves32(x[n][i]));
            }
            if (!s.few) rest += sum_pairs(w);
        }
        const uint32_t upto = wave_scan((uint32_t)__popc(hits));
        uint32_t at = 0;
        if ((t & 63) == 63) at = atomicAdd(&s_listed, upto);
        if (!s.few) {
            mass = (uint64_t)((double)rest * STEPS);
            if (!s.plain) {
                mass = 0;
                for (uint32_t b = ~hits & (~0u >> (32 - N * E)); b; b &= b - 1) mass += s.weight(s_x[__builtin_ctz(b)][t]);
            }
            mass = wave_sum64(mass);
        }
        at = (uint32_t)__builtin_amdgcn_readlane((int)at, 63) + upto - (uint32_t)__popc(hits);
        uint64_t* list = a.ws_list + ((size_t)row * a.slices + blockIdx.x) * a.room;
        for (; hits; hits &= hits - 1, at++) {
            const int b = __builtin_ctz(hits);
            if (at < a.room) list[at] = (uint64_t)falling(s_x[b][t]) << 32 | (uint32_t)token(b / E, b % E);
        }
    }
    if ((t & 63) == 0) s_mass[wave] = mass;
    __syncthreads();
    if (t == 0)
        a.ws_slice[(size_t)row * a.slices + blockIdx.x] =
            Slice{s_mass[0] + s_mass[1] + s_mass[2] + s_mass[3], s.max, (int32_t)s_first, bound, s_listed};
}

// ------------------------------------------------------ one row, 1024 threads

constexpr int PICK = 1024;
static_assert(PICK == BINS, "a thread a bin");

// A place in the order: the cumulative weight up to and with it, its own, and its token.
struct Found {
    uint64_t upto, weight;
    int32_t token;
};

constexpr int TAIL_BINS = 256, TAIL_COPIES = 32;
constexpr float TAIL_OCTAVES = 32.0f;  // of weights below the listed tokens', that these bins cover
struct PickLds {
    uint32_t count[BINS];         // tokens of a bin; then before it
    uint64_t mass[BINS];          // weight of a bin; then before it
    uint64_t list[LIST];          // falling(logit) << 32 | token; or a digit's histogram
    uint64_t upto[LIST];          // cumulative weights of the sorted list
    uint64_t wide[TAIL_BINS * TAIL_COPIES];
    uint64_t part[PICK / 64], found[4];
    uint32_t part32[PICK / 64], n, bin, turn[2];
};

// Sum over the threads before this one; the sum of all in *total.
__device__ __forceinline__ uint64_t scan64(PickLds& m, uint64_t v, uint64_t* total) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint64_t s = wave_scan64(v);
    __syncthreads();
    if (lane == 63) m.part[wave] = s;
    __syncthreads();
    const uint64_t p = lane < PICK / 64 ? m.part[lane] : 0, q = wave_scan64(p);
    *total = lane64(q, PICK / 64 - 1);
    return lane64(q - p, (int)__builtin_amdgcn_readfirstlane(wave)) + s - v;
}

// m.list's first n entries in rising order, as many threads as half of them.
__device__ __forceinline__ void sort_list(PickLds& m, uint32_t n) {
    uint32_t size = 2;
    while (size < n) size <<= 1;
    for (uint32_t i = n + threadIdx.x; i < size; i += PICK) m.list[i] = ~0ull;
    __syncthreads();
    for (uint32_t k = 2; k <= size; k <<= 1)
        for (uint32_t j = k >> 1; j; j >>= 1) {
            for (uint32_t t = threadIdx.x; t < size / 2; t += PICK) {
                const uint32_t i = 2 * t - (t & (j - 1)), o = i | j;
                const uint64_t x = m.list[i], y = m.list[o];
                if ((x > y) == ((i & k) == 0)) {
                    m.list[i] = y;
                    m.list[o] = x;
                }
            }
            __syncthreads();
        }
}

// A whole row.
template <int T>
struct Pick {
    static constexpr int E = Row<T>::E;
    const Row<T> r;
    const Setting& s;
    PickLds& m;
    uint32_t valid;               // tokens that are not masked
    uint64_t all, least;          // their weight; of those that weigh min_p
    uint32_t from, sorted = 0;    // the bin whose tokens the sorted list has, and how many these are

    template <class F>
    __device__ __forceinline__ void each(F&& f) const {
        r.template each<PICK>([&](float x, int32_t token) {
            if (x > -INFINITY) f(x, token);
        });
    }

    // the histogram, then what lies before each bin
    __device__ __forceinline__ Pick(const SampleArgs& a, const Setting& s, PickLds& m, uint32_t row) : r(a, row), s(s), m(m) {
        const uint32_t t = threadIdx.x;
        least = 0;
        __syncthreads();
        m.count[t] = 0;
        m.mass[t] = 0;
        __syncthreads();
        each([&](float x, int32_t) {
            const int b = s.bin(x);
            const uint64_t w = s.weight(x);
            atomicAdd(&m.count[b], 1u);
            if (w) atomicAdd((unsigned long long*)&m.mass[b], (unsigned long long)w);
            if ((double)w >= s.least) least += w;
        });
        if (s.least > 0.0) scan64(m, least, &least);
        __syncthreads();
        uint64_t total;
        const uint64_t n = scan64(m, m.count[t], &total);
        valid = (uint32_t)total;
        const uint64_t w = scan64(m, m.mass[t], &all);
        m.count[t] = (uint32_t)n;
        m.mass[t] = w;
        __syncthreads();
    }
    __device__ __forceinline__ uint32_t count_after(uint32_t b) const { return b + 1 < BINS ? m.count[b + 1] : valid; }
    __device__ __forceinline__ uint64_t mass_after(uint32_t b) const { return b + 1 < BINS ? m.mass[b + 1] : all; }

    // the tokens of a bin (at most LIST), sorted, with the cumulative weights
    __device__ __forceinline__ void gather(uint32_t bin) {
        __syncthreads();
        if (threadIdx.x == 0) m.n = 0;
        __syncthreads();
        each([&](float x, int32_t token) {
            if ((uint32_t)s.bin(x) != bin) return;
            m.list[atomicAdd(&m.n, 1u)] = (uint64_t)falling(x) << 32 | (uint32_t)token;
        });
        __syncthreads();
        sorted = m.n;
        from = bin;
        sort_list(m, sorted);
        const uint32_t t = threadIdx.x;
        uint64_t w[2], total;
#pragma unroll
        for (int i = 0; i < 2; i++) w[i] = 2 * t + i < sorted ? s.weight(falling_value((uint32_t)(m.list[2 * t + i] >> 32))) : 0;
        const uint64_t at = m.mass[bin] + scan64(m, w[0] + w[1], &total);
        m.upto[2 * t] = at + w[0];
        m.upto[2 * t + 1] = at + w[0] + w[1];
        __syncthreads();
    }

    // A place in a bin of more tokens than the list holds: three digits of the
    // falling value, each a histogram of the row, then the number among equals.
    // `counted`: w counts tokens, not weight.
    __device__ Found search(uint32_t b, uint64_t w, bool counted, bool want_token) {
        uint64_t* hist = m.list;                  // [2048]
        sorted = 0;
        uint32_t prefix = 0, known = 0;           // digits found, and their mask
        uint64_t left = w - (counted ? (uint64_t)m.count[b] : m.mass[b]), mass_before = m.mass[b];
        const uint32_t t = threadIdx.x;
        for (int digit = 0; digit < 3; digit++) {
            const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0;
            const uint32_t size = digit == 2 ? 1024 : 2048;
            __syncthreads();
            hist[2 * t] = hist[2 * t + 1] = 0;
            m.upto[2 * t] = m.upto[2 * t + 1] = 0;
            __syncthreads();
            each([&](float x, int32_t) {
                const uint32_t k = falling(x);
                if ((uint32_t)s.bin(x) != b || (k & known) != prefix) return;
                const uint64_t wt = s.weight(x);
                const uint32_t at = (k >> shift) & (size - 1);
                atomicAdd((unsigned long long*)&hist[at], (unsigned long long)(counted ? 1 : wt));
                if (counted) atomicAdd((unsigned long long*)&m.upto[at], (unsigned long long)wt);
            });
            __syncthreads();
            uint64_t total, n0 = hist[2 * t], n1 = hist[2 * t + 1];
            const uint64_t w0 = m.upto[2 * t], w1 = m.upto[2 * t + 1];
            const uint64_t at = scan64(m, n0 + n1, &total), wat = counted ? scan64(m, w0 + w1, &total) : at;
            if (at < left && left <= at + n0) {
                m.found[0] = 2 * t;
                m.found[1] = at;
                m.found[2] = wat;
            } else if (at + n0 < left && left <= at + n0 + n1) {
                m.found[0] = 2 * t + 1;
                m.found[1] = at + n0;
                m.found[2] = counted ? wat + w0 : at + n0;
            }
            __syncthreads();
            prefix |= (uint32_t)m.found[0] << shift;
            known |= (size - 1) << shift;
            left -= m.found[1];
            mass_before += m.found[2];
        }
        Found f;
        f.weight = s.weight(falling_value(prefix));
        const uint64_t nth = counted ? left - 1 : (left - 1) / (f.weight ? f.weight : 1);   // among equals, from 0
        f.upto = mass_before + (nth + 1) * f.weight;
        f.token = -1;
        uint64_t seen = 0;
        for (uint32_t c0 = 0; want_token && c0 < r.chunks; c0 += PICK) {       // (as many rounds for every thread)
            float x[E];
            uint64_t n = 0, total;
            const bool in = c0 + t < r.chunks;
            if (in) {
                const u4v w4 = r.raw(c0 + t);
#pragma unroll
                for (int i = 0; i < E; i++) x[i] = Row<T>::value(w4, i);
#pragma unroll
                for (int i = 0; i < E; i++) n += x[i] > -INFINITY && falling(x[i]) == prefix;
            }
            uint64_t at = seen + scan64(m, n, &total);
            if (in && at <= nth && nth < at + n)
#pragma unroll
                for (int i = 0; i < E; i++)
                    if (x[i] > -INFINITY && falling(x[i]) == prefix && at++ == nth) m.found[3] = (uint64_t)((int64_t)((c0 + t) * E) - r.skip + i);
            seen += total;
            __syncthreads();
            if (nth < seen) {
                f.token = (int32_t)m.found[3];
                break;
            }
        }
        __syncthreads();
        return f;
    }
    // The first place whose cumulative weight reaches w (from 1, to `all`), or the w-th (`counted`, from 1 to `valid`).
    __device__ __forceinline__ Found place(uint64_t w, bool counted, bool want_token) {
        const uint32_t t = threadIdx.x;
        __syncthreads();
        if (counted ? m.count[t] < w && w <= count_after(t) : m.mass[t] < w && w <= mass_after(t)) m.bin = t;
        __syncthreads();
        const uint32_t b = m.bin;
        if (count_after(b) - m.count[b] > LIST) return search(b, w, counted, want_token);
        if (!sorted || b != from) gather(b);
        const uint64_t before = m.mass[b];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint32_t at = 2 * t + i;
            const uint64_t last = at ? m.upto[at - 1] : before;
            if (at < sorted && (counted ? at + 1 == w - m.count[b] : last < w && w <= m.upto[at])) {
                m.found[0] = m.upto[at];
                m.found[1] = m.upto[at] - last;
                m.found[2] = (uint32_t)m.list[at];
            }
        }
        __syncthreads();
        return {m.found[0], m.found[1], (int32_t)m.found[2]};
    }
};

constexpr uint32_t AT_ONCE = 256;      // tokens of one bin that are put in order by comparing each with each

// Of k entries of m.list, weights in m.upto: the one at which the weight behind
// `before` reaches v, or the number behind `tokens` (every wave for itself).
__device__ __forceinline__ bool in_order(const PickLds& m, uint32_t k, uint64_t before, uint32_t tokens, uint64_t v, bool counted,
                                         Found& f) {
    const uint32_t lane = threadIdx.x & 63;
    bool found = false;
    for (uint32_t i0 = 0; i0 < k; i0 += 64) {
        const uint32_t i = i0 + lane;
        const uint64_t e = i < k ? m.list[i] : 0, own = i < k ? m.upto[i] : 0;
        uint64_t upto = before;
        uint32_t nth = tokens;
        for (uint32_t j = 0; j < k; j++) {
            const bool le = m.list[j] <= e;
            upto += le ? m.upto[j] : 0;
            nth += le;
        }
        const uint64_t who = __ballot(i < k && (counted ? nth == v : upto - own < v && v <= upto));
        if (who) {
            const int l = (int)__builtin_ctzll(who);
            f = Found{lane64(upto, l), lane64(own, l), (int32_t)__builtin_amdgcn_readlane((int)(uint32_t)e, l)};
            found = true;
        }
    }
    return found;
}

// The listed tokens of a row: eight waves have them in registers, the others take
// part where all are needed (64 rows of 130560 logits: 19.0 us, 19.7 with four waves
// or with all sixteen).
constexpr uint32_t FAST = 512;
struct Listed {
    static constexpr int N = LIST / FAST, B = BINS / FAST;
    Setting& s;
    PickLds& m;
    float x[N];                   // -infinity: none
    int32_t token[N];
    uint64_t w[N];
    uint32_t bin[N];
    uint32_t turns = 0;           // calls of place, by which m.turn is taken in turn
    uint64_t mass[B + 1];         // before each of the thread's bins, and behind the last
    uint32_t count[B + 1];
    uint32_t n;                   // tokens
    uint64_t all;                 // their weight
    float bound;                  // what is not listed is below it
    uint64_t row_mass;            // of what is below it, where top-k does not end the row

    __device__ __forceinline__ Listed(Setting& s, PickLds& m) : s(s), m(m) {}

    // The row's largest logit, where the listed tokens end, and these tokens.  False: more than fit, or not all.
    __device__ __forceinline__ bool load(const SampleArgs& a, uint32_t row) {
        const uint32_t t = threadIdx.x, lane = t & 63;
        const Slice* slices = a.ws_slice + (size_t)row * a.slices;
        const uint64_t* list = a.ws_list + (size_t)row * a.slices * a.room;
        m.count[t] = 0;
        m.mass[t] = 0;
        if (t == 0) m.n = 0;
        // (a wave 256 tokens of a slice, asked for before its bound is known)
        constexpr uint32_t W = PICK / 64;
        const uint32_t first = __builtin_amdgcn_readfirstlane(t >> 6), parts = (a.room + 255) / 256;
        uint64_t e[4];
        if (first < a.slices * parts)
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) e[j] = lane + 64 * j < a.room ? list[first * min(a.room, 256u) + lane + 64 * j] : 0;
        float top = -INFINITY;
        uint32_t none = NO_TOKEN, most = 0;
        bound = -INFINITY;
        for (uint32_t i = lane; i < a.slices; i += 64) {
            const Slice q = slices[i];
            bound = fmaxf(bound, q.bound);
            most = max(most, q.listed);
            if (q.max > top || (q.max == top && (uint32_t)q.first < none)) {
                top = q.max;
                none = (uint32_t)q.first;
            }
        }
        s.max = wave_max(top);
        bound = wave_max(bound);
        none = wave_least(top == s.max ? none : (uint32_t)NO_TOKEN);
        s.first = none == NO_TOKEN ? -1 : (int32_t)none;
        if (s.greedy || s.first < 0) return true;
        if (__any(most > a.room)) return false;
        // the slices' weights beside the row's largest logit
        row_mass = 0;
        for (uint32_t i = lane; i < a.slices && !s.few; i += 64) {
            const Slice q = slices[i];
            if (q.max == s.max) row_mass += q.rest;
            else if (q.rest) row_mass += (uint64_t)rint((double)q.rest * ((double)s.weight(q.max) / STEPS));
        }
        row_mass = wave_sum64(row_mass);
        uint64_t below = 0;                       // of listed tokens that others may come before
        __syncthreads();
        for (uint32_t i = first; i < a.slices * parts; i += W) {
            const uint32_t from = (i & (parts - 1)) * 256, some = slices[i >> __builtin_ctz(parts)].listed, listed = some - min(from, some);
            uint32_t keep = 0, on = 0;
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) {
                if (i != first) e[j] = lane + 64 * j < listed ? list[i * min(a.room, 256u) + lane + 64 * j] : 0;
                const float x = falling_value((uint32_t)(e[j] >> 32));
                if (lane + 64 * j < listed) {
                    if (x >= bound) on |= 1u << j;
                    else if (!s.few) below += s.weight(x);
                }
                keep += (uint32_t)__popcll(__ballot(on >> j & 1));
            }
            uint32_t at = 0;
            if (lane == 0) at = atomicAdd(&m.n, keep);
            at = (uint32_t)__builtin_amdgcn_readfirstlane((int)at);
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) {
                const uint64_t who = __ballot(on >> j & 1);
                const uint32_t to = at + (uint32_t)__popcll(who & ((1ull << lane) - 1));
                if ((on >> j & 1) && to < LIST) m.list[to] = e[j];
                at += (uint32_t)__popcll(who);
            }
        }
        if (!s.few) {
            below = wave_sum64(below);
            if (lane == 0) m.part[first] = below;
        }
        __syncthreads();
        n = m.n;
        if (!s.few) row_mass += wave_sum64(lane < W ? m.part[lane] : 0);
        return n <= LIST;
    }

    // the histogram, then what lies before each bin
    __device__ __forceinline__ void count_all(bool counts) {
        const uint32_t t = threadIdx.x;
        if (t < FAST)
#pragma unroll
            for (int i = 0; i < N; i++) {
                x[i] = -INFINITY;
                w[i] = 0;
                bin[i] = ~0u;
                if (i * FAST >= n) continue;
                const uint64_t e = t + i * FAST < n ? m.list[t + i * FAST] : 0xFF800000ull << 32;
                x[i] = falling_value((uint32_t)(e >> 32));
                token[i] = (int32_t)(uint32_t)e;
                w[i] = s.weight(x[i]);
                if (x[i] == -INFINITY) continue;
                bin[i] = (uint32_t)s.bin(x[i]);
                if (counts) atomicAdd(&m.count[bin[i]], 1u);
                atomicAdd((unsigned long long*)&m.mass[bin[i]], (unsigned long long)w[i]);
            }
        __syncthreads();
        uint64_t sum = 0;
        uint32_t cnt = 0;
        if (t < FAST) {
            for (int i = 0; i < B; i++) {
                mass[i] = sum;
                count[i] = cnt;
                sum += m.mass[B * t + i];
                cnt += m.count[B * t + i];
            }
            mass[B] = sum;
            count[B] = cnt;
            sum = wave_scan64(sum);
            cnt = wave_scan(cnt);
            if ((t & 63) == 63) {
                m.part[t >> 6] = sum;
                m.part32[t >> 6] = cnt;
            }
        }
        __syncthreads();
        all = 0;
        uint64_t before = 0;
        uint32_t cbefore = 0;
#pragma unroll
        for (int i = 0; i < (int)FAST / 64; i++) {
            if (i < (int)(t >> 6)) {
                before += m.part[i];
                cbefore += m.part32[i];
            }
            all += m.part[i];
        }
        if (t < FAST) {
            before += sum - mass[B];
            cbefore += cnt - count[B];
#pragma unroll
            for (int i = 0; i <= B; i++) {
                mass[i] += before;
                count[i] += cbefore;
            }
        }
    }
    // of those that weigh min_p
    __device__ __forceinline__ uint64_t weighing() {
        const uint32_t t = threadIdx.x;
        uint64_t v = 0;
        if (t < FAST)
#pragma unroll
            for (int i = 0; i < N; i++) v += (double)w[i] >= s.least ? w[i] : 0;
        __syncthreads();
        if (t < FAST) {
            v = wave_sum64(v);
            if ((t & 63) == 0) m.part[t >> 6] = v;
        }
        __syncthreads();
        v = 0;
#pragma unroll
        for (int i = 0; i < (int)FAST / 64; i++) v += m.part[i];
        return v;
    }
    // The place whose cumulative weight reaches v, or the v-th (`counted`).  False: too
    // many tokens in its bin.  (What one call's slower waves still read, the next call
    // leaves alone until all have come to its first barrier.)
    __device__ __forceinline__ bool place(uint64_t v, bool counted, Found& f) {
        const uint32_t t = threadIdx.x;
        uint32_t* number = &m.turn[turns++ & 1];
        if (t < FAST)
#pragma unroll
            for (int i = 0; i < B; i++)
                if (counted ? count[i] < v && v <= count[i + 1] : mass[i] < v && v <= mass[i + 1]) {
                    m.bin = B * t + i;
                    m.found[0] = mass[i];
                    m.found[1] = count[i];
                    *number = 0;
                }
        __syncthreads();
        const uint32_t b = m.bin;
        const uint64_t before = m.found[0];
        const uint32_t tokens = (uint32_t)m.found[1];
        if (t < FAST)
#pragma unroll
            for (int i = 0; i < N; i++)
                if (i * FAST < n && bin[i] == b) {
                    const uint32_t at = atomicAdd(number, 1u);
                    m.list[at] = (uint64_t)falling(x[i]) << 32 | (uint32_t)token[i];
                    m.upto[at] = w[i];
                }
        __syncthreads();
        const uint32_t k = *number;
        if (k > AT_ONCE) return false;
        in_order(m, k, before, tokens, v, counted, f);
        return true;
    }
};

// What a row has below its listed tokens, in weights beside `bound`'s, to the nearest
// of steps of 2^-42 of it (of 2^20 tokens far below it no more than 2^-23 is lost, and
// the bound's own token stays; steps of 2^-30, all that 32 bits hold, would lose
// 2^-15 of a row with 16 listed tokens): a border or a token in flat rows.  One compute unit goes through the row:
// once for a histogram by value, kept 32 times so that a pair of lanes has one in
// LDS banks of its own, and once for the tokens of the bin; these again by a finer
// histogram, so that only a few have to be put in order, or all are equal.  Bound by
// that one compute unit: 27 us for each border or token in a row of 130560 bf16 logits
// (drawn from a normal distribution, one row: 14 us without a tail, 53 at temperature
// 1, 72 with top-p; the whole row instead, `Pick`, takes 133 and 160).
template <int T>
struct Tail {
    static constexpr uint32_t MOST = 8192;   // tokens of a bin
    static_assert(offsetof(PickLds, upto) == offsetof(PickLds, list) + sizeof(PickLds::list) && MOST * 4 <= 2 * sizeof(PickLds::list), "list and upto");
    const Row<T> r;
    const Setting& s;
    PickLds& m;
    const float bound;
    float per_bin;                // values to bins
    double unit, by;              // weights to steps; steps of 2^43 to these
    uint64_t all, least = 0;      // of all; of those that weigh min_p

    // (the exponent's product in two pieces: 16-bit logits have few values, whose
    // roundings would add up)
    __device__ __forceinline__ uint64_t weight(float x) const {
        const float d = s.distance32(x), o = d * s.hi, more = fmaf(d, s.lo, fmaf(d, s.hi, -o));
        const float w = __builtin_amdgcn_exp2f(o);
        // (below 2^52, and added to it whole in the last place)
        const double y = fma((double)fmaf(w, more * 0.693147181f, w), unit, 4503599627370496.0);
        return __builtin_bit_cast(uint64_t, y) - 0x4330000000000000ull;
    }
    // 0 .. TAIL_BINS - 1 (and what is left behind the point, up to the last); never falls as x falls
    __device__ __forceinline__ float place_of(float x) const { return __builtin_amdgcn_fmed3f((bound - x) * per_bin, 0.0f, TAIL_BINS - 0.001f); }
    __device__ __forceinline__ uint32_t bin(float x) const { return (uint32_t)place_of(x); }

    __device__ __forceinline__ Tail(const SampleArgs& a, const Setting& s, PickLds& m, uint32_t row, float bound)
        : r(a, row), s(s), m(m), bound(bound) {
        const uint32_t t = threadIdx.x;
        const float o = floorf(s.octaves32(bound));
        unit = exp2(42.0 - (double)o);
        by = exp2(-1.0 - (double)o);
        per_bin = s.hi * (TAIL_BINS / TAIL_OCTAVES);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TAIL_BINS * TAIL_COPIES / PICK; i++) m.wide[t + i * PICK] = 0;
        __syncthreads();
        // (min_p's weight, where it lies below the bound's)
        const bool lightest = s.least > 0.0 && s.least * by < 8796093022208.0;
        const uint64_t some = lightest ? (uint64_t)(s.least * by) : 0;
        uint64_t* own = m.wide + t % TAIL_COPIES;
        // (no branch: a masked token weighs nothing, nor does a listed one here)
        const auto add = [&](float x) {
            const uint64_t w = x < bound ? weight(x) : 0;
            atomicAdd((unsigned long long*)&own[bin(x) * TAIL_COPIES], (unsigned long long)w);
            return w;
        };
        if (!lightest) r.template each<PICK>([&](float x, int32_t) { add(x); });
        else
            r.template each<PICK>([&](float x, int32_t) {
                const uint64_t w = add(x);
                least += w >= some ? w : 0;
            });
        __syncthreads();
        uint64_t w = 0;
        if (t < TAIL_BINS)
            for (int i = 0; i < TAIL_COPIES; i++) w += m.wide[t * TAIL_COPIES + (t + i) % TAIL_COPIES];
        const uint64_t before = scan64(m, w, &all);
        m.mass[t] = before;
        if (s.least > 0.0) scan64(m, least, &least);
        __syncthreads();
    }
    // The place whose cumulative weight reaches v (from 1, to `all`): f.upto in these
    // weights, f.weight of 2^43.  False: more tokens in its bin than are kept.
    __device__ __forceinline__ bool place(uint64_t v, Found& f) {
        const uint32_t t = threadIdx.x, lane = t & 63;
        __syncthreads();
        if (t < TAIL_BINS && m.mass[t] < v && v <= m.mass[t + 1]) m.bin = t;      // (behind the last: all)
        if (t == 0) m.n = 0;
        m.wide[t] = 0;
        __syncthreads();
        const uint32_t b = m.bin;
        uint64_t before = m.mass[b];
        // the largest values of the bin and of the next one, digit by digit (the bins never fall as values fall)
        uint32_t key = 0;
        for (uint32_t bit = 1u << 31; bit; bit >>= 1) {
            const float x = falling_value(~(key | bit));
            if (x <= bound && bin(x) >= b + (lane & 1)) key |= bit;
        }
        const float top = falling_value(~(uint32_t)__builtin_amdgcn_readlane((int)key, 0));
        const float under = b + 1 < TAIL_BINS ? falling_value(~(uint32_t)__builtin_amdgcn_readlane((int)key, 1)) : -INFINITY;
        uint32_t* tokens = (uint32_t*)m.list;
        r.template batches<PICK>([&](const auto& w, int32_t t0, uint64_t in) {
            typedef std::remove_reference_t<decltype(w)> W;
            constexpr int U = sizeof(W) / sizeof(u4v), E = Row<T>::E;
            uint64_t hits = 0;
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int i = 0; i < E; i++) {
                    const float x = Row<T>::value(w[u], i);
                    hits |= (x <= top && x > under && x < bound ? 1ull : 0ull) << (u * E + i);
                }
            hits &= in;
            const uint32_t n = (uint32_t)__popcll(hits), upto = wave_scan(n);
            uint32_t at = 0;
            if (lane == 63 && upto) at = atomicAdd(&m.n, upto);
            at = (uint32_t)__builtin_amdgcn_readlane((int)at, 63) + upto - n;
            for (; hits; hits &= hits - 1, at++) {
                const int h = __builtin_ctzll(hits);
                if (at < MOST) tokens[at] = (uint32_t)(t0 + h / E * (int)(PICK * E) + h % E);
            }
        });
        __syncthreads();
        const uint32_t n = m.n;
        if (n > MOST) return false;
        // finer: each thread some of them
        float x[MOST / PICK];
        int32_t token[MOST / PICK];
        uint32_t fine[MOST / PICK];
#pragma unroll
        for (int i = 0; i < (int)(MOST / PICK); i++) {
            const uint32_t at = t + i * PICK;
            fine[i] = ~0u;
            if (at >= n) continue;
            token[i] = (int32_t)tokens[at];
            x[i] = r.one(token[i]);
        }
#pragma unroll
        for (int i = 0; i < (int)(MOST / PICK); i++) {
            if (t + i * PICK >= n) continue;
            const uint64_t w = weight(x[i]);
            fine[i] = min((uint32_t)((place_of(x[i]) - (float)b) * (float)BINS), (uint32_t)BINS - 1);
            if (w) atomicAdd((unsigned long long*)&m.wide[fine[i]], (unsigned long long)w);
        }
        __syncthreads();
        uint64_t total;
        const uint64_t own = m.wide[t];
        uint64_t at = before + scan64(m, own, &total);
        if (at < v && v <= at + own) {
            m.bin = t;
            m.found[0] = at;
        }
        if (t == 0) m.n = 0;
        __syncthreads();
        before = m.found[0];
#pragma unroll
        for (int i = 0; i < (int)(MOST / PICK); i++)
            if (fine[i] == m.bin) {
                const uint32_t to = atomicAdd(&m.n, 1u);
                if (to >= LIST) continue;
                m.list[to] = (uint64_t)falling(x[i]) << 32 | (uint32_t)token[i];
                m.upto[to] = weight(x[i]);
            }
        __syncthreads();
        const uint32_t k = m.n;
        if (k > LIST) return false;
        // more than a few are mostly all of one value, in the order of their numbers
        bool same = k > 32;
        if (same) {
            const uint64_t e = m.list[0];
            for (uint32_t i = t; i < k; i += PICK) same &= m.list[i] >> 32 == e >> 32;
            same = __syncthreads_and(same);
        }
        if (!same) {
            if (k > AT_ONCE || !in_order(m, k, before, 0, v, false, f)) return false;
        } else {
            const uint64_t each = m.upto[0];
            uint32_t nth = (uint32_t)((v - before - 1) / each);
            f.upto = before + (nth + 1) * each;
            int32_t found = 0;
#pragma unroll
            for (int shift = 10; shift >= 0; shift -= 10) {
                __syncthreads();
                m.wide[t] = 0;
                __syncthreads();
                for (uint32_t i = t; i < k; i += PICK) {
                    const uint32_t number = (uint32_t)m.list[i];
                    if (shift || number >> 10 == (uint32_t)found) atomicAdd((unsigned long long*)&m.wide[number >> shift & 1023], 1ull);
                }
                __syncthreads();
                const uint64_t c = m.wide[t], to = scan64(m, c, &total);
                if (to <= nth && nth < to + c) {
                    m.found[0] = t;
                    m.found[1] = to;
                }
                __syncthreads();
                nth -= (uint32_t)m.found[1];
                found = found << 10 | (int32_t)m.found[0];
            }
            f.token = found;
        }
        f.weight = s.weight(r.one(f.token));
        __syncthreads();
        return true;
    }
};

// The row's token, of what was listed where that is enough, of
// the rest of the row where a border or the token lies there, of the whole row
// where listed tokens do not fit or top-k goes beyond them.
template <int T>
__device__ __forceinline__ void pick_token(const SampleArgs& a, PickLds& m, uint32_t row, Setting& s, Listed& p, bool done, float uu) {
    const uint32_t t = threadIdx.x;
    Found f{};
    uint64_t kept = 0;
    const double u = uu > 0.0f ? (double)uu : 0.0;
    const auto reach = [&](uint64_t mass) { return (uint64_t)fmax(1.0, ceil(s.p * (double)mass)); };
    const auto drawn = [&](uint64_t mass) { return min((uint64_t)(u * (double)mass), mass - 1) + 1; };
    if (s.greedy || s.first < 0) {
        if (t == 0) {
            a.tokens[row] = s.first;
            if (a.probs) a.probs[row] = s.first < 0 ? 0.0f : 1.0f;
        }
        return;
    }
    if (done) {
        p.count_all(s.k != 0);
        s.fp32();
        const bool whole = p.bound == -INFINITY;
        const uint32_t k = whole && s.k >= p.n ? 0 : s.k;
        uint64_t rest = whole ? 0 : p.row_mass;
        done = k <= p.n && (k || !s.few || whole);
        if (done && k) {
            done = p.place(k, true, f);
            kept = f.upto;
            rest = 0;
        } else {
            kept = p.all + rest;
        }
        // borders among the listed tokens
        bool p_below = s.p < 1.0, m_below = s.least > 0.0 && !whole && !((double)s.weight(p.bound) < s.least);
        if (done && p_below) {
            const uint64_t w = reach(kept);
            p_below = w > p.all;
            if (!p_below) {
                done = p.place(w, false, f);
                kept = min(kept, f.upto);
                rest = 0;
            }
        }
        if (done && s.least > 0.0 && !m_below) {
            kept = min(kept, p.weighing());
            rest = 0;
        }
        // (borders further on matter if none was found)
        if (done && (rest == 0 || !(p_below || m_below))) {
            const uint64_t w = drawn(kept);
            if (w <= p.all) {
                done = p.place(w, false, f);
                rest = 0;
            }
        }
        if (done && rest) {
            done = s.plain;
            if (done) {
                Tail<T> q(a, s, m, row, p.bound);
                // weights of 2^43 to those beside the bound's and back
                const double by = q.by;
                const auto to = [&](uint64_t v) { return min(max((uint64_t)ceil((double)(v - p.all) * by), (uint64_t)1), q.all); };
                const auto back = [&](uint64_t v) { return p.all + (uint64_t)rint((double)v / by); };
                done = q.all > 0;
                kept = back(q.all);
                if (done && p_below) {
                    // (to either side: these weights' sum is not the slices' to the last bit)
                    const uint64_t w = reach(kept);
                    if (w > p.all) {
                        done = q.place(to(w), f);
                        kept = min(kept, back(f.upto));
                    } else {
                        done = p.place(w, false, f);
                        kept = min(kept, f.upto);
                    }
                }
                if (done && m_below) kept = min(kept, back(q.least));
                if (done) {
                    const uint64_t w = drawn(kept);
                    done = w > p.all ? q.place(to(w), f) : p.place(w, false, f);
                }
            }
        }
    }
    if (!done) {
        Pick<T> q(a, s, m, row);
        const uint32_t k = s.k < q.valid ? s.k : 0;
        kept = k ? q.place(k, true, false).upto : q.all;
        if (s.p < 1.0) kept = min(kept, q.place(reach(kept), false, false).upto);
        if (s.least > 0.0) kept = min(kept, q.least);
        f = q.place(drawn(kept), false, true);
    }
    if (t == 0) {
        a.tokens[row] = f.token;
        if (a.probs) a.probs[row] = (float)((double)f.weight / (double)kept);
    }
}

template <int T>
__global__ __launch_bounds__(PICK) void k_sample_pick(SampleArgs a) {
    __shared__ PickLds m;
    Setting s;
    s.of(a, blockIdx.x);
    const float u = a.u[blockIdx.x];
    Listed p(s, m);
    const bool done = p.load(a, blockIdx.x);
    pick_token<T>(a, m, blockIdx.x, s, p, done, u);
}

// A row of up to 32 tokens a thread, listed and picked by one workgroup, in one launch
// (5 rows of 16384 fp32 logits, top-p: 10.3 us, 13.5 in two; 5 of 32000 bf16: 12.2 and
// 13.3; 300 of 27000 fp32: 24.8 and 34).  Bound by one compute unit's instructions for
// each token, then by a few barriers and LDS round trips a border, 1 us each.  Its 16
// waves leave a thread 128 registers, and 2 to 9 of a thread's values spill (12 to 40
// bytes a lane; of k_sample_pick's 2 to 4).
template <int T, int TOKENS>
__global__ __launch_bounds__(PICK) void k_sample_row(SampleArgs a) {
    constexpr int E = Row<T>::E, N = TOKENS / E;
    constexpr uint32_t W = PICK / 64;
    __shared__ PickLds m;
    __shared__ float s_max[W];
    __shared__ uint32_t s_bound[W], s_first;
    const uint32_t row = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6;
    m.count[t] = 0;
    m.mass[t] = 0;
    if (t == 0) {
        m.n = 0;
        s_first = NO_TOKEN;
    }
    const Row<T> r(a, row);
    float x[N][E], top = -INFINITY;
#pragma unroll
    for (int n = 0; n < N; n++) {
        const bool in = t + n * PICK < r.chunks;
        u4v w = {};
        if (in) w = r.raw(t + n * PICK);
#pragma unroll
        for (int i = 0; i < E; i++) x[n][i] = in ? Row<T>::value(w, i) : -INFINITY;
    }
    Setting s;
    s.of(a, row);
    const float u = a.u[row];
#pragma unroll
    for (int n = 0; n < N; n++)
#pragma unroll
        for (int i = 0; i < E; i++) top = fmaxf(top, x[n][i]);
    // (as in k_sample_slice, of the threads that have tokens; of fewer than c lanes all are listed)
    const float want = s.few ? fminf(1.5f * (float)s.k + 16.0f, 1700.0f) : 1040.0f;
    const float each = want / (float)min((r.chunks + 63) & ~63u, (uint32_t)PICK);
    const uint32_t nth = nth_of_wave(top, (uint32_t)(64.0f * (1.0f - __builtin_amdgcn_exp2f(each * -1.4426950f))) + 1);
    const float wave_top = wave_max(top);
    if (lane == 0) {
        s_max[wave] = wave_top;
        s_bound[wave] = nth;
    }
    __syncthreads();
    s.max = wave_max(lane < W ? s_max[lane] : -INFINITY);
    if (s.max > -INFINITY && wave_top == s.max) {
        uint32_t first = NO_TOKEN;
#pragma unroll
        for (int n = N - 1; n >= 0; n--)
#pragma unroll
            for (int i = E - 1; i >= 0; i--)
                if (x[n][i] == s.max) first = (uint32_t)((int32_t)((t + n * PICK) * E) - r.skip + i);
        first = wave_least(first);
        if (lane == 0) atomicMin(&s_first, first);
    }
    Listed p(s, m);
    p.bound = -INFINITY;
    p.n = 0;
    uint64_t rest = 0;
    if (!s.greedy && s.max > -INFINITY) {
        const uint64_t sum = wave_sum64(lane < W ? s_bound[lane] : 0);
        const uint32_t some = (uint32_t)__popcll(__ballot(lane < W && s_bound[lane] != 0));
        if (some) p.bound = falling_value(~(uint32_t)(sum / some));
        const float above = fmaxf(p.bound, -3.4028234663852886e38f);
        s.fp32();
        // (as there: a bit for each listed token, the values to LDS)
        static_assert(sizeof(m.wide) >= 4 * 16 * PICK, "16 tokens of each thread");
        float* values = (float*)m.wide + t;
        uint32_t hits = 0;
        float others = 0.0f;
#pragma unroll
        for (int n = 0; n < N; n++) {
            float w[E];
#pragma unroll
            for (int i = 0; i < E; i++) {
                const bool hit = x[n][i] >= above;
                hits |= (hit ? 1u : 0u) << (n * E + i);
                if (!s.few) w[i] = __builtin_amdgcn_exp2f(hit ? -INFINITY : s.octaves32(x[n][i]));
            }
            if (!s.few) others += sum_pairs(w);
        }
        if (!s.few) {
            rest = (uint64_t)((double)others * STEPS);
            if (!s.plain) {
                rest = 0;
#pragma unroll
                for (int n = 0; n < N; n++)
#pragma unroll 1
                    for (int i = 0; i < E; i++) rest += hits >> (n * E + i) & 1 ? 0 : s.weight(x[n][i]);
            }
            rest = wave_sum64(rest);
        }
        const uint32_t upto = wave_scan((uint32_t)__popc(hits));
        uint32_t at = 0;
        if (lane == 63) at = atomicAdd(&m.n, upto);
        at = (uint32_t)__builtin_amdgcn_readlane((int)at, 63) + upto - (uint32_t)__popc(hits);
#pragma unroll
        for (int n0 = 0; n0 < N; n0 += 16 / E) {
#pragma unroll
            for (int j = 0; j < 16; j++) values[j * PICK] = x[n0 + j / E][j % E];
            for (uint32_t some = hits >> (n0 * E) & 0xFFFFu; some; some &= some - 1, at++) {
                const int b = __builtin_ctz(some);
                if (at < LIST)
                    m.list[at] = (uint64_t)falling(values[b * PICK]) << 32 |
                                 (uint32_t)((int32_t)((t + (n0 + b / E) * PICK) * E) - r.skip + b % E);
            }
        }
    }
    if (lane == 0) m.part[wave] = rest;
    __syncthreads();
    s.first = s_first == NO_TOKEN ? -1 : (int32_t)s_first;
    p.n = m.n;
    p.row_mass = wave_sum64(lane < W ? m.part[lane] : 0);
    __syncthreads();
    pick_token<T>(a, m, row, s, p, p.n <= LIST, u);
}

}  // namespace pf

using namespace pf;

// ================================================================== host

constexpr uint32_t SAMPLE_VOCAB = 1u << 20;
constexpr size_t SAMPLE_SCRATCH = 64u << 20;

template <int T>
static void sample_type(hipStream_t st, uint32_t tokens, const SampleArgs& a) {
    constexpr int E = Row<T>::E;
    const dim3 grid(a.slices, a.rows);
    if (tokens == 16) hipLaunchKernelGGL((k_sample_slice<T, 16 / E>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_sample_slice<T, 32 / E>), grid, dim3(256), 0, st, a);
    hipLaunchKernelGGL((k_sample_pick<T>), dim3(a.rows), dim3(PICK), 0, st, a);
}

template <int T>
static void sample_row(hipStream_t st, uint32_t tokens, const SampleArgs& a) {
    if (tokens == 16) hipLaunchKernelGGL((k_sample_row<T, 16>), dim3(a.rows), dim3(PICK), 0, st, a);
    else hipLaunchKernelGGL((k_sample_row<T, 32>), dim3(a.rows), dim3(PICK), 0, st, a);
}

extern "C" pf_status pf_sample_rows(pf_ctx* c, const pf_sample_desc* d, const void* logits, const float* u, uint32_t rows,
                                    int32_t* tokens, float* probs) {
    if (!c || !d) return PF_ERR_ARG;
    if (d->type != PF_TYPE_F32 && d->type != PF_TYPE_F16 && d->type != PF_TYPE_BF16)
        return fail(c, PF_ERR_ARG, "sample: logits are PF_TYPE_F32, F16 or BF16");
    if (!d->n_vocab || d->n_vocab > SAMPLE_VOCAB) return fail(c, PF_ERR_UNSUPPORTED, "sample: n_vocab is 1 to 2^20");
    const uint32_t stride = d->stride ? d->stride : d->n_vocab;
    if (stride < d->n_vocab) return fail(c, PF_ERR_ARG, "sample: stride is n_vocab or more");
    if (!rows) return PF_OK;
    if (rows > 65535) return fail(c, PF_ERR_UNSUPPORTED, "sample: over 65535 rows at once");
    if (!logits || !u || !tokens) return fail(c, PF_ERR_ARG, "sample: a buffer is NULL");
    const size_t es = d->type == PF_TYPE_F32 ? 4 : 2, n = (size_t)rows * 4;
    if ((uintptr_t)logits % es) return fail(c, PF_ERR_ARG, "sample: logits start on a multiple of their size");
    const size_t bytes = ((size_t)(rows - 1) * stride + d->n_vocab) * es;
    const void* given[] = {u, d->temperature_dev, d->top_k_dev, d->top_p_dev, d->min_p_dev};
    for (const void* g : given)
        if ((uintptr_t)g & 3) return fail(c, PF_ERR_ARG, "sample: settings start on 4 bytes");
    const void* out[] = {tokens, probs};
    for (const void* o : out) {
        if (!o) continue;
        if ((uintptr_t)o & 3) return fail(c, PF_ERR_ARG, "sample: outputs start on 4 bytes");
        bool meets = overlaps(o, n, logits, bytes) || (o == probs && overlaps(o, n, tokens, n));
        for (const void* g : given) meets |= g && overlaps(o, n, g, n);
        if (meets) return fail(c, PF_ERR_ARG, "sample: an output overlaps another buffer");
    }
    DeviceScope on(c);
    SampleArgs a{};
    a.logits = logits; a.u = u; a.temperature = d->temperature_dev; a.top_k = d->top_k_dev; a.top_p = d->top_p_dev; a.min_p = d->min_p_dev;
    a.temperature1 = d->temperature; a.top_k1 = d->top_k; a.top_p1 = d->top_p; a.min_p1 = d->min_p;
    a.rows = rows; a.vocab = d->n_vocab; a.stride = stride; a.tokens = tokens; a.probs = probs;
    const uint32_t chunk = 16 / (uint32_t)es, off = aligned16(logits) && stride % chunk == 0 ? 0 : chunk - 1;
    const uint32_t chunks = (off + d->n_vocab + chunk - 1) / chunk;
    if (chunks * chunk <= 32 * PICK) {
        const uint32_t tokens = chunks * chunk <= 16 * PICK ? 16 : 32;
        if (d->type == PF_TYPE_F32) sample_row<PF_TYPE_F32>(c->stream, tokens, a);
        else if (d->type == PF_TYPE_F16) sample_row<PF_TYPE_F16>(c->stream, tokens, a);
        else sample_row<PF_TYPE_BF16>(c->stream, tokens, a);
        PF_LAUNCHED(c);
        return PF_OK;
    }
    // tokens of a thread of the slices' workgroups: 32, or 16 where a row has up to 8
    // slices of 32 (one row of 40000 fp32 logits: 13.2 us, 15.4 with 32; 64 of them 15.5
    // and 16.8, 512 41.0 and 43.5; 128 of 65536 bf16 ones 19.3 and 18.8, 512 46.4 and 46.2).
    // More slices cost the row's workgroup, that takes their lists together, more than
    // they save (one row of 250000 bf16 logits: 15.4 us, 16.8 with 16, 21 with 8).  How
    // many rows there are does not matter here, so that a row's sums, and its token, are
    // the same among any others.
    const auto cut = [&](uint32_t tokens) { return (chunks + 256 * (tokens / chunk) - 1) / (256 * (tokens / chunk)); };
    const uint32_t per = cut(32) <= 8 ? 16 : 32;
    a.slices = cut(per);
    a.room = a.slices <= 8 ? 512 : a.slices <= 16 ? 256 : 128;   // (1700 tokens in all, unevenly)
    // as many rows at a time as keep their lists in SAMPLE_SCRATCH
    const size_t row_bytes = a.slices * (sizeof(Slice) + (size_t)a.room * 8);
    const uint32_t most = (uint32_t)std::min<size_t>(rows, std::max<size_t>(1, SAMPLE_SCRATCH / row_bytes));
    void* ws = nullptr;
    if (pf_status st = ctx_scratch(c, most * row_bytes, &ws)) return st;
    a.ws_list = (uint64_t*)ws;
    a.ws_slice = (Slice*)(a.ws_list + (size_t)most * a.slices * a.room);
    for (uint32_t at = 0; at < rows; at += most) {
        SampleArgs b = a;
        b.rows = std::min(most, rows - at);
        b.logits = (const uint8_t*)logits + (size_t)at * stride * es;
        b.u += at;
        b.tokens += at;
        if (probs) b.probs += at;
        if (b.temperature) b.temperature += at;
        if (b.top_k) b.top_k += at;
        if (b.top_p) b.top_p += at;
        if (b.min_p) b.min_p += at;
        if (d->type == PF_TYPE_F32) sample_type<PF_TYPE_F32>(c->stream, per, b);
        else if (d->type == PF_TYPE_F16) sample_type<PF_TYPE_F16>(c->stream, per, b);
        else sample_type<PF_TYPE_BF16>(c->stream, per, b);
    }
    PF_LAUNCHED(c);
    return PF_OK;
}
