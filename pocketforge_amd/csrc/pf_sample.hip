// Tokens from rows of logits (pf_sample_rows of include/pf_gpu.h): temperature,
// top-k, top-p and min-p, from given random numbers.
//
// With the tokens in order of their logits (equal ones by number) each filter
// keeps a beginning of that order, so the kept set is a mass S = min(M_k, M_p,
// M_m): of the first k, of the first that reach p M_k, of those that weigh min_p.
// The token is the first whose cumulative weight exceeds u S.  Nothing has to be
// sorted but what lies next to those three borders and the token: a histogram
// over the distance from the largest logit finds their bins, and only these bins'
// tokens are sorted, or all up to the last where they are few.
//
// Weights are whole numbers, exp((l - max) / T) in steps of 2^-43, so that every
// sum is exact, whatever the order in which threads add to it: up to 2^20 tokens
// of up to 2^43 fit 64 bits, and what a step leaves of 2^20 sums is 2^-24 of the
// largest weight, what sums of fp32 would lose of the first few.
#include "pf_attend.h"
#include "pf_context.h"

namespace pf {

constexpr int BINS = 1024;
constexpr float BIN_OCTAVES = 44.0f;   // of the weights, that the bins cover (the last one has the rest)
constexpr uint32_t LIST = 2048;        // tokens that are sorted at once
constexpr uint32_t FEW_K = 1024;       // top-k up to here needs no sums over the row
constexpr double STEPS = 8796093022208.0;   // 2^43
constexpr uint64_t ONE = 1ull << 43;

struct SampleArgs {
    const void* logits;
    const float *u, *temperature, *top_p, *min_p;   // of each row, or NULL
    const int32_t* top_k;
    float temperature1, top_p1, min_p1;
    uint32_t top_k1;
    uint32_t rows, vocab, stride, slices, per;      // per: chunks of a slice
    int32_t* tokens;
    float* probs;
    float2* ws_max;               // [rows][slices]: value, token
    uint64_t* ws_mass;            // [rows][slices][BINS]
    uint32_t* ws_count;           // [rows][slices][BINS]
    uint64_t* ws_least;           // [rows][slices]: mass of those that weigh min_p
};

// A row in chunks of 16 bytes from the last multiple of 16 on; what lies before its
// first or behind its last token reads as -infinity, and so does a NaN.
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
    __device__ __forceinline__ void load(uint32_t c, float (&x)[E]) const {
        const int t0 = (int)(c * E) - skip;
        if (t0 >= 0 && t0 + E <= n) {
            if constexpr (T == PF_TYPE_F32) load4<T>(at + (size_t)c * 16, x);
            else load8<T>(at + (size_t)c * 16, x);
        } else {
#pragma unroll
            for (int i = 0; i < E; i++) {
                x[i] = -INFINITY;
                if (t0 + i >= 0 && t0 + i < n) {
                    if constexpr (T == PF_TYPE_F32) x[i] = ((const float*)at)[t0 + i + skip];
                    else x[i] = to_float<T>(((const short*)at)[t0 + i + skip]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < E; i++) x[i] = x[i] == x[i] ? x[i] : -INFINITY;
    }
};

// A row's settings.
struct Setting {
    float max;
    int32_t first;                // the largest logit's token, -1: none
    bool greedy;
    uint32_t k;                   // 0: off
    double scale, p, least;       // log2(e) / T; p >= 1: off; min_p in steps, 0: off
    float to_bin;
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
    // 2^43 e^((l - max) / T) to the nearest whole number: 2^x = 2^n e^(f ln 2) with
    // |f| <= 1/2, the series up to z^11 (z^12 / 12! = 6e-15, 2^-47)
    __device__ __forceinline__ uint64_t weight(float l) const {
        const double x = ((double)l - (double)max) * scale;
        if (l == max) return ONE;
        if (!(x > -44.5)) return 0;
        const double n = rint(x), z = (x - n) * 0.69314718055994530942;
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
        // (added to 2^52, a number is whole in the last place)
        const double w = __builtin_ldexp(y, (int)n + 43) + 4503599627370496.0;
        return __builtin_bit_cast(uint64_t, w) - 0x4330000000000000ull;
    }
};

// Larger logits first: the value as an integer that falls with it.
__device__ __forceinline__ uint32_t falling(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);       // (-0 is 0)
    return u & 0x80000000u ? u : ~(u | 0x80000000u);
}
__device__ __forceinline__ float falling_value(uint32_t k) {
    return __builtin_bit_cast(float, k & 0x80000000u ? k : ~k & 0x7FFFFFFFu);
}

struct Best {
    float v;
    int32_t i;
};
__device__ __forceinline__ Best better(Best a, Best b) { return b.v > a.v || (b.v == a.v && b.i < a.i) ? b : a; }
__device__ __forceinline__ Best wave_best(Best b) {
#pragma unroll
    for (int o = 32; o; o >>= 1) b = better(b, Best{__shfl_xor(b.v, o), __shfl_xor(b.i, o)});
    return b;
}
constexpr int32_t NO_TOKEN = 0x7FFFFFFF;

// The largest logit of a slice and its first token.
template <int T>
__global__ __launch_bounds__(256) void k_sample_max(SampleArgs a) {
    __shared__ Best s_best[4];
    const Row<T> r(a, blockIdx.y);
    const uint32_t c0 = blockIdx.x * a.per, c1 = min(c0 + a.per, r.chunks);
    Best b{-INFINITY, NO_TOKEN};
#pragma unroll 4
    for (uint32_t c = c0 + threadIdx.x; c < c1; c += 256) {
        float x[Row<T>::E];
        r.load(c, x);
#pragma unroll
        for (int i = 0; i < Row<T>::E; i++)
            if (x[i] > b.v) b = Best{x[i], (int32_t)(c * Row<T>::E) - r.skip + i};
    }
    b = wave_best(b);
    if ((threadIdx.x & 63) == 0) s_best[threadIdx.x >> 6] = b;
    __syncthreads();
    if (threadIdx.x == 0) {
        b = better(better(s_best[0], s_best[1]), better(s_best[2], s_best[3]));
        a.ws_max[(size_t)blockIdx.y * a.slices + blockIdx.x] = float2{b.v, __builtin_bit_cast(float, b.i)};
    }
}

// The row's largest logit, of its slices'.
__device__ __forceinline__ void row_max(const SampleArgs& a, uint32_t row, Setting& s) {
    Best b{-INFINITY, NO_TOKEN};
    const uint32_t lane = threadIdx.x & 63;
    if (lane < a.slices) {
        const float2 m = a.ws_max[(size_t)row * a.slices + lane];
        b = Best{m.x, __builtin_bit_cast(int32_t, m.y)};
    }
    b = wave_best(b);
    s.max = b.v;
    s.first = b.i == NO_TOKEN ? -1 : b.i;
}

// The tokens of a chunk into the bins.
template <int E>
__device__ __forceinline__ void count_chunk(const Setting& s, const float (&x)[E], bool sums, uint32_t* count, uint64_t* mass,
                                            uint64_t& least) {
#pragma unroll
    for (int i = 0; i < E; i++) {
        if (x[i] == -INFINITY) continue;
        const int b = s.bin(x[i]);
        atomicAdd(&count[b], 1u);
        if (sums) {
            const uint64_t w = s.weight(x[i]);
            if (w) atomicAdd((unsigned long long*)&mass[b], (unsigned long long)w);
            if ((double)w >= s.least) least += w;
        }
    }
}

__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, int o) {
    return (uint64_t)(uint32_t)__shfl_up((int)(uint32_t)v, o) | (uint64_t)(uint32_t)__shfl_up((int)(v >> 32), o) << 32;
}
__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int o) {
    return (uint64_t)(uint32_t)__shfl_xor((int)(uint32_t)v, o) | (uint64_t)(uint32_t)__shfl_xor((int)(v >> 32), o) << 32;
}
__device__ __forceinline__ uint64_t wave_sum64(uint64_t v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += shfl_xor64(v, o);
    return v;
}

// A slice's histogram.
template <int T>
__global__ __launch_bounds__(256) void k_sample_count(SampleArgs a) {
    __shared__ uint32_t s_count[BINS];
    __shared__ uint64_t s_mass[BINS], s_least[4];
    const uint32_t row = blockIdx.y;
    Setting s;
    s.of(a, row);
    row_max(a, row, s);
    if (s.greedy || s.first < 0) return;
    const bool sums = !s.few;
    for (int i = threadIdx.x; i < BINS; i += 256) s_count[i] = 0, s_mass[i] = 0;
    __syncthreads();
    const Row<T> r(a, row);
    const uint32_t c0 = blockIdx.x * a.per, c1 = min(c0 + a.per, r.chunks);
    uint64_t least = 0;
#pragma unroll 2
    for (uint32_t c = c0 + threadIdx.x; c < c1; c += 256) {
        float x[Row<T>::E];
        r.load(c, x);
        count_chunk(s, x, sums, s_count, s_mass, least);
    }
    least = wave_sum64(least);
    if ((threadIdx.x & 63) == 0) s_least[threadIdx.x >> 6] = least;
    __syncthreads();
    const size_t at = (size_t)row * a.slices + blockIdx.x;
    for (int i = threadIdx.x; i < BINS; i += 256) {
        a.ws_count[at * BINS + i] = s_count[i];
        if (sums) a.ws_mass[at * BINS + i] = s_mass[i];
    }
    if (threadIdx.x == 0) a.ws_least[at] = s_least[0] + s_least[1] + s_least[2] + s_least[3];
}

// ------------------------------------------------------ one row, 1024 threads

constexpr int PICK = 1024;
static_assert(PICK == BINS, "a thread a bin");

// A place in the order: the cumulative weight up to and with it, its own, and its token.
struct Found {
    uint64_t upto, weight;
    int32_t token;
};

struct PickLds {
    uint32_t count[BINS];         // then: tokens before a bin
    uint64_t mass[BINS];          // then: weight before a bin
    uint64_t list[LIST];          // falling(logit) << 32 | token; or a digit's histogram
    uint64_t upto[LIST];          // cumulative weights of the sorted list
    uint64_t part[PICK / 64];
    uint64_t found[4];
    uint32_t n;
    Best best[PICK / 64];
};

// Sum over the threads before this one; the sum of all in *total.
__device__ __forceinline__ uint64_t scan64(PickLds& m, uint64_t v, uint64_t* total) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint64_t s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t x = shfl_up64(s, o);
        if (lane >= (uint32_t)o) s += x;
    }
    __syncthreads();
    if (lane == 63) m.part[wave] = s;
    __syncthreads();
    uint64_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < PICK / 64; w++) {
        const uint64_t x = m.part[w];
        if (w < (int)wave) before += x;
        all += x;
    }
    *total = all;
    return before + s - v;
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

template <int T>
struct Pick {
    static constexpr int E = Row<T>::E;
    const SampleArgs& a;
    const Row<T> r;
    Setting s;
    PickLds& m;
    uint32_t row, valid;          // tokens that are not masked
    uint64_t all, least;          // their weight; of those that weigh min_p
    uint32_t from = 0, upto = 0;  // bins whose tokens the sorted list has, and how many these are
    uint32_t listed = 0;

    __device__ __forceinline__ Pick(const SampleArgs& args, PickLds& lds, uint32_t row) : a(args), r(args, row), m(lds), row(row) {}

    template <class F>
    __device__ __forceinline__ void each_chunk(F&& f) const {
#pragma unroll 2
        for (uint32_t c = threadIdx.x; c < r.chunks; c += PICK) {
            float x[E];
            r.load(c, x);
            f(x, (int32_t)(c * E) - r.skip);
        }
    }

    __device__ __forceinline__ void largest() {
        Best b{-INFINITY, NO_TOKEN};
        each_chunk([&](const float (&x)[E], int32_t t0) {
#pragma unroll
            for (int i = 0; i < E; i++)
                if (x[i] > b.v) b = Best{x[i], t0 + i};
        });
        b = wave_best(b);
        if ((threadIdx.x & 63) == 0) m.best[threadIdx.x >> 6] = b;
        __syncthreads();
        b = m.best[0];
#pragma unroll
        for (int w = 1; w < PICK / 64; w++) b = better(b, m.best[w]);
        s.max = b.v;
        s.first = b.i == NO_TOKEN ? -1 : b.i;
    }

    // the histogram, of the slices' or of the row; then what lies before each bin
    __device__ __forceinline__ void count(bool slices, bool sums) {
        const uint32_t t = threadIdx.x;
        least = 0;
        uint32_t n = 0;
        uint64_t w = 0;
        if (slices) {
            for (uint32_t i = 0; i < a.slices; i++) {
                const size_t at = (size_t)row * a.slices + i;
                n += a.ws_count[at * BINS + t];
                if (sums) {
                    w += a.ws_mass[at * BINS + t];
                    least += a.ws_least[at];
                }
            }
        } else {
            __syncthreads();
            m.count[t] = 0;
            m.mass[t] = 0;
            __syncthreads();
            each_chunk([&](const float (&x)[E], int32_t) { count_chunk(s, x, sums, m.count, m.mass, least); });
            scan64(m, least, &least);
            n = m.count[t];
            w = m.mass[t];
        }
        uint64_t total;
        const uint64_t before = scan64(m, n, &total);
        valid = (uint32_t)total;
        m.count[t] = (uint32_t)before;
        all = 0;
        if (sums) m.mass[t] = scan64(m, w, &all);
        __syncthreads();
    }
    __device__ __forceinline__ uint32_t count_after(uint32_t b) const { return b + 1 < BINS ? m.count[b + 1] : valid; }
    __device__ __forceinline__ uint64_t mass_after(uint32_t b) const { return b + 1 < BINS ? m.mass[b + 1] : all; }
    // the bin with the n-th token (from 1), with the weight `t` (from 1)
    __device__ __forceinline__ uint32_t bin_of_count(uint32_t n) {
        const uint32_t t = threadIdx.x;
        if (m.count[t] < n && n <= count_after(t)) m.n = t;
        __syncthreads();
        const uint32_t b = m.n;
        __syncthreads();
        return b;
    }
    __device__ __forceinline__ uint32_t bin_of_mass(uint64_t w) {
        const uint32_t t = threadIdx.x;
        if (m.mass[t] < w && w <= mass_after(t)) m.n = t;
        __syncthreads();
        const uint32_t b = m.n;
        __syncthreads();
        return b;
    }

    // the tokens of bins b0 .. b1 (at most LIST), sorted, with their cumulative weights behind `before`
    __device__ __forceinline__ void gather(uint32_t b0, uint32_t b1, uint64_t before) {
        __syncthreads();
        if (threadIdx.x == 0) m.n = 0;
        __syncthreads();
        each_chunk([&](const float (&x)[E], int32_t t0) {
#pragma unroll
            for (int i = 0; i < E; i++) {
                if (x[i] == -INFINITY) continue;
                const uint32_t b = (uint32_t)s.bin(x[i]);
                if (b >= b0 && b <= b1) {
                    const uint32_t at = atomicAdd(&m.n, 1u);
                    if (at < LIST) m.list[at] = (uint64_t)falling(x[i]) << 32 | (uint32_t)(t0 + i);
                }
            }
        });
        __syncthreads();
        listed = min(m.n, LIST);
        from = b0;
        upto = b1;
        sort_list(m, listed);
        const uint32_t t = threadIdx.x;
        uint64_t w[2], total;
#pragma unroll
        for (int i = 0; i < 2; i++) w[i] = 2 * t + i < listed ? s.weight(falling_value((uint32_t)(m.list[2 * t + i] >> 32))) : 0;
        const uint64_t at = before + scan64(m, w[0] + w[1], &total);
        m.upto[2 * t] = at + w[0];
        m.upto[2 * t + 1] = at + w[0] + w[1];
        __syncthreads();
    }
    // the first place of the list whose cumulative weight reaches w
    __device__ __forceinline__ Found find(uint64_t w, uint64_t before) {
        const uint32_t t = threadIdx.x;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint32_t at = 2 * t + i;
            const uint64_t last = at ? m.upto[at - 1] : before;
            if (at < listed && last < w && w <= m.upto[at]) {
                m.found[0] = m.upto[at];
                m.found[1] = m.upto[at] - last;
                m.found[2] = (uint32_t)m.list[at];
            }
        }
        __syncthreads();
        const Found f{m.found[0], m.found[1], (int32_t)m.found[2]};
        __syncthreads();
        return f;
    }

    // The same in a bin of more tokens than the list holds: three digits of the
    // falling value, each a histogram of the row, then the number among equals.
    // `counted`: w counts tokens, not weight.
    __device__ Found search(uint32_t b, uint64_t w, uint64_t before, uint64_t tokens_before, bool counted, bool want_token) {
        uint64_t* hist = m.list;                  // [2048]
        listed = 0;
        uint32_t prefix = 0, known = 0;           // digits found, and their mask
        uint64_t left = w - (counted ? tokens_before : before), mass_before = before;
        const uint32_t t = threadIdx.x;
        for (int digit = 0; digit < 3; digit++) {
            const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0;
            const uint32_t size = digit == 2 ? 1024 : 2048;
            __syncthreads();
            hist[2 * t] = hist[2 * t + 1] = 0;
            m.upto[2 * t] = m.upto[2 * t + 1] = 0;
            __syncthreads();
            each_chunk([&](const float (&x)[E], int32_t) {
#pragma unroll
                for (int i = 0; i < E; i++) {
                    if (x[i] == -INFINITY || (uint32_t)s.bin(x[i]) != b) continue;
                    const uint32_t k = falling(x[i]);
                    if ((k & known) != prefix) continue;
                    const uint64_t wt = s.weight(x[i]);
                    const uint32_t at = (k >> shift) & (size - 1);
                    atomicAdd((unsigned long long*)&hist[at], (unsigned long long)(counted ? 1 : wt));
                    if (counted) atomicAdd((unsigned long long*)&m.upto[at], (unsigned long long)wt);
                }
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
                r.load(c0 + t, x);
#pragma unroll
                for (int i = 0; i < E; i++) n += x[i] != -INFINITY && falling(x[i]) == prefix;
            }
            uint64_t at = seen + scan64(m, n, &total);
            if (in && at <= nth && nth < at + n)
#pragma unroll
                for (int i = 0; i < E; i++)
                    if (x[i] != -INFINITY && falling(x[i]) == prefix && at++ == nth) m.found[3] = (uint64_t)((int64_t)((c0 + t) * E) - r.skip + i);
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

    // the first place whose cumulative weight reaches w, or the w-th (`counted`)
    __device__ __forceinline__ Found place(uint64_t w, bool counted, bool want_token) {
        const uint32_t b = counted ? bin_of_count((uint32_t)w) : bin_of_mass(w);
        const uint64_t before = m.mass[b];
        const uint32_t tokens = m.count[b];
        if (count_after(b) - tokens > LIST) return search(b, w, before, tokens, counted, want_token);
        if (!listed || b < from || b > upto) gather(b, b, before);
        if (counted) {
            Found f{m.upto[(uint32_t)w - 1 - m.count[from]], 0, -1};
            __syncthreads();
            return f;
        }
        return find(w, m.mass[from]);
    }
};

// The row's token.  SLICES: the largest logits and histograms of its slices are in
// the workspace.
template <int T>
__global__ __launch_bounds__(PICK) void k_sample_pick(SampleArgs a) {
    __shared__ PickLds m;
    const uint32_t row = blockIdx.x, t = threadIdx.x;
    Pick<T> p(a, m, row);
    Setting& s = p.s;
    s.of(a, row);
    const bool slices = a.slices > 0;
    if (slices) row_max(a, row, s);
    else p.largest();
    if (s.greedy || s.first < 0) {
        if (t == 0) {
            a.tokens[row] = s.first;
            if (a.probs) a.probs[row] = s.first < 0 ? 0.0f : 1.0f;
        }
        return;
    }
    bool sums = !s.few;
    p.count(slices, sums);
    const uint32_t k = s.k < p.valid ? s.k : 0;
    const double u = a.u[row] > 0.0f ? (double)a.u[row] : 0.0;
    const auto reach = [&](uint64_t mass) { return (uint64_t)fmax(1.0, ceil(s.p * (double)mass)); };
    const auto drawn = [&](uint64_t mass) { return min((uint64_t)(u * (double)mass), mass - 1) + 1; };
    // the bins that the kept set can reach: up to the k-th token; without top-k up to
    // top-p's border or min_p's (two bins more than where the weight falls below it),
    // whichever comes first
    uint32_t end = BINS - 1;
    bool by_p = s.p < 1.0;
    if (k) {
        end = p.bin_of_count(k);
    } else if (sums) {
        if (by_p) end = p.bin_of_mass(reach(p.all));
        if (s.least > 0.0) {
            const float d = -__builtin_amdgcn_logf((float)(s.least / STEPS)) * (BINS / BIN_OCTAVES) + 2.0f;
            const uint32_t b = (uint32_t)fminf(d, (float)(BINS - 1));
            by_p &= end <= b;
            end = min(end, b);
        }
    }
    Found f;
    uint64_t kept;
    if (p.count_after(end) <= LIST) {
        p.gather(0, end, 0);
        const uint32_t n = p.listed;
        kept = sums ? p.all : m.upto[n - 1];
        if (k) kept = m.upto[k - 1];
        uint64_t mine = kept;
        if (by_p) mine = min(mine, p.find(reach(kept), 0).upto);
        if (s.least > 0.0) {
            // the weights fall: the last that weighs min_p
            __syncthreads();
            if (t == 0) m.found[3] = 0;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint32_t at = 2 * t + i;
                const auto weighs = [&](uint32_t j) { return (double)(m.upto[j] - (j ? m.upto[j - 1] : 0)) >= s.least; };
                if (at < n && weighs(at) && (at + 1 == n || !weighs(at + 1))) m.found[3] = m.upto[at];
            }
            __syncthreads();
            mine = min(mine, m.found[3]);
        }
        kept = mine;
        __syncthreads();
        f = p.find(drawn(kept), 0);
    } else {
        if (!sums) p.count(false, sums = true);
        kept = k ? p.place(k, true, false).upto : p.all;
        if (s.p < 1.0) kept = min(kept, p.place(reach(kept), false, false).upto);
        if (s.least > 0.0) kept = min(kept, p.least);
        f = p.place(drawn(kept), false, true);
    }
    if (t == 0) {
        a.tokens[row] = f.token;
        if (a.probs) a.probs[row] = (float)((double)f.weight / (double)kept);
    }
}

}  // namespace pf

using namespace pf;

// ================================================================== host

constexpr uint32_t SAMPLE_VOCAB = 1u << 20;
constexpr uint32_t MOST_SLICES = 16;

template <int T>
static void sample_type(hipStream_t st, const SampleArgs& a) {
    if (a.slices) {
        hipLaunchKernelGGL((k_sample_max<T>), dim3(a.slices, a.rows), dim3(256), 0, st, a);
        hipLaunchKernelGGL((k_sample_count<T>), dim3(a.slices, a.rows), dim3(256), 0, st, a);
    }
    hipLaunchKernelGGL((k_sample_pick<T>), dim3(a.rows), dim3(PICK), 0, st, a);
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
    if (d->n_vocab > 16384 && rows < 512) {
        const uint32_t chunks = (uint32_t)(d->n_vocab * es + 15 + 15) / 16;      // (the first and the last not whole)
        a.slices = std::min(MOST_SLICES, (1024 + rows - 1) / rows);
        a.per = (chunks + a.slices - 1) / a.slices;
        const size_t parts = (size_t)rows * a.slices;
        void* ws = nullptr;
        if (pf_status st = ctx_scratch(c, parts * (BINS * 12 + 16), &ws)) return st;
        a.ws_mass = (uint64_t*)ws;
        a.ws_least = a.ws_mass + parts * BINS;
        a.ws_max = (float2*)(a.ws_least + parts);
        a.ws_count = (uint32_t*)(a.ws_max + parts);
    }
    if (d->type == PF_TYPE_F32) sample_type<PF_TYPE_F32>(c->stream, a);
    else if (d->type == PF_TYPE_F16) sample_type<PF_TYPE_F16>(c->stream, a);
    else sample_type<PF_TYPE_BF16>(c->stream, a);
    PF_LAUNCHED(c);
    return PF_OK;
}
