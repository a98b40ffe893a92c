// Rotary positions (pf_rotary_* and pf_pages_store_rotary of include/pf_gpu.h):
// rows of heads turned by their positions, alone or while a pass's keys and
// values go into their pages.
//
// Pair (a, b) of a head at position p becomes (a c - b s, a s + b c), c and s the
// cosine and sine of p f.  The table holds each pair's frequency in turns, f /
// (2 pi), as the sum of two doubles: p times it loses nothing that matters, its
// fraction is exact, and the rest is a polynomial on an eighth of a turn.
#include <cmath>

#include "pf_paged.h"

struct pf_rotary {
    pf_ctx* ctx = nullptr;
    pf_rotary_desc desc{};
    double* table = nullptr;          // device [turn / 2][2]: high and low part
    uint32_t turn = 0;
};

namespace pf {

constexpr uint32_t ROTARY_MOST = 64;   // pairs

struct RotaryArgs {
    const double* table;
    double magnitude;
    uint32_t turn, dim;
};

// Cosine and sine of p times a pair's frequency, times the magnitude.  f is at
// most an eighth of a turn to either side of a quarter's multiple; the polynomials
// are the Taylor series of sine and cosine up to pi / 4, cut where the next term
// is below half a step of the type (x^17 / 17! = 5e-17, x^18 / 18! = 2e-18; for
// fp32 x^11 / 11! = 2e-9, x^12 / 12! = 1e-10).
template <class F>
__device__ __forceinline__ void turn_of(const double* table, uint32_t pair, double p, double magnitude, F& c, F& s) {
    const double hi = table[2 * pair], lo = table[2 * pair + 1];
    const double t = p * hi;
    double r = (t - rint(t)) + fma(p, lo, fma(p, hi, -t));
    const double q = rint(4.0 * r);
    r = fma(q, -0.25, r) * 6.283185307179586476925;
    F cs, sn;
    if constexpr (sizeof(F) == 8) {
        const double z = r * r;
        sn = -1.0 / 1307674368000.0;
        sn = fma(sn, z, 1.0 / 6227020800.0);
        sn = fma(sn, z, -1.0 / 39916800.0);
        sn = fma(sn, z, 1.0 / 362880.0);
        sn = fma(sn, z, -1.0 / 5040.0);
        sn = fma(sn, z, 1.0 / 120.0);
        sn = fma(sn, z, -1.0 / 6.0);
        sn = fma(sn * z, r, r);
        cs = 1.0 / 20922789888000.0;
        cs = fma(cs, z, -1.0 / 87178291200.0);
        cs = fma(cs, z, 1.0 / 479001600.0);
        cs = fma(cs, z, -1.0 / 3628800.0);
        cs = fma(cs, z, 1.0 / 40320.0);
        cs = fma(cs, z, -1.0 / 720.0);
        cs = fma(cs, z, 1.0 / 24.0);
        cs = fma(cs, z, -0.5);
        cs = fma(cs, z, 1.0);
    } else {
        const float x = (float)r, z = x * x;
        sn = 1.0f / 362880.0f;
        sn = fmaf(sn, z, -1.0f / 5040.0f);
        sn = fmaf(sn, z, 1.0f / 120.0f);
        sn = fmaf(sn, z, -1.0f / 6.0f);
        sn = fmaf(sn * z, x, x);
        cs = -1.0f / 3628800.0f;
        cs = fmaf(cs, z, 1.0f / 40320.0f);
        cs = fmaf(cs, z, -1.0f / 720.0f);
        cs = fmaf(cs, z, 1.0f / 24.0f);
        cs = fmaf(cs, z, -0.5f);
        cs = fmaf(cs, z, 1.0f);
    }
    // quarters of a turn: (c, s) -> (-s, c) -> (-c, -s) -> (s, -c)
    const int quarter = (int)q & 3;
    const F m = (F)magnitude, a = quarter & 1 ? sn : cs, b = quarter & 1 ? cs : sn;
    c = (quarter == 1 || quarter == 2 ? -a : a) * m;
    s = (quarter >= 2 ? -b : b) * m;
}

// A lane's part of a turn: dims d .. d + 7 of a head.  Pairs 2i, 2i + 1 lie in the
// lane; of pairs i, i + turn / 2 the lane holds one half and reads the other from
// where the row came from (turn is a multiple of 8, so four dims are in one half).
// A wave has a pair for each lane at most, and forms each pair's angle once: its
// lanes then read theirs from LDS (24 prompts of up to 700 rows into 4-bit pages:
// 31 us with every lane forming its own, 24 so).
template <int T, bool INTER, class F>
struct Turn {
    static constexpr int N = INTER ? 4 : 8;
    typedef F cs __attribute__((ext_vector_type(2)));
    F c[N], s[N];
    // lds: [64], of the wave
    __device__ __forceinline__ Turn(const RotaryArgs& a, uint32_t d, int32_t position, cs* lds) {
        const uint32_t lane = threadIdx.x & 63, half = a.turn / 2;
        F cosine = 1, sine = 0;
        if (lane < half) turn_of<F>(a.table, lane, position, a.magnitude, cosine, sine);
        lds[lane] = cs{cosine, sine};
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int e = 0; e < N / 4; e++) {
            const uint32_t g = INTER ? d : d + 4 * e;
            const bool first = INTER || g < half;
            const uint32_t pair = g < a.turn ? (INTER ? g / 2 : first ? g : g - half) : 0;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const cs v = lds[pair + i];
                c[4 * e + i] = v.x;
                s[4 * e + i] = !INTER && first ? -v.y : v.y;
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
    // x: the values at `head` + d
    __device__ __forceinline__ void operator()(const RotaryArgs& a, const uint8_t* head, uint32_t d, float (&x)[8]) const {
        if (INTER) {
            if (d >= a.turn) return;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const F u = x[2 * i], w = x[2 * i + 1];
                x[2 * i] = (float)fma(u, c[i], -(w * s[i]));
                x[2 * i + 1] = (float)fma(u, s[i], w * c[i]);
            }
        } else {
            const uint32_t half = a.turn / 2;
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const uint32_t g = d + 4 * e;
                if (g >= a.turn) return;
                float p[4];
                load4<T>(head + (size_t)(g < half ? g + half : g - half) * act_size<T>, p);
#pragma unroll
                for (int i = 0; i < 4; i++) x[4 * e + i] = (float)fma((F)x[4 * e + i], c[4 * e + i], (F)p[i] * s[4 * e + i]);
            }
        }
    }
};

// Past the caches: a prompt's rows would evict what the next calls read.  24 prompts of
// up to 700 rows turned and stored into 4-bit pages, 1 / 2 / 3 / 4 batches in turn:
// 20 / 20 / 20 / 29 us, 21 / 21 / 30 / 31 with plain stores; the pages read back as well 27.6 /
// 27.6 / 33 / 39, 28 / 34 / 40 / 40.6; 8192 rows of 16 heads of 128, four in turn, 11.4 and 13.7.
// A kernel that reads the turned rows at once pays a part of it back: prompt attention
// after the store 71 / 71 / 78 / 82, 70 / 70 / 79 / 81; the 8192 rows turned again 25 and 23.
// A decode step's few rows take the same either way (64 turned, stored and attended
// over contexts of 300: 12.3 us).
template <int T>
__device__ __forceinline__ void store8(void* p, const float (&x)[8]) {
    if constexpr (T == PF_TYPE_F32) {
        f4v lo = {x[0], x[1], x[2], x[3]}, hi = {x[4], x[5], x[6], x[7]};
        __builtin_nontemporal_store(lo, (f4v*)p);
        __builtin_nontemporal_store(hi, (f4v*)p + 1);
    } else {
        __builtin_nontemporal_store(pack8<T == PF_TYPE_BF16>(x), (s8v*)p);
    }
}

// Heads h0, h0 + 4, .. before h1 of a row, four at a time (16 lanes, 8 dims each),
// the next four's rows under way.
template <int T, bool INTER>
__device__ __forceinline__ void turn_heads(const RotaryArgs& r, const uint8_t* in, uint8_t* out, uint32_t h0, uint32_t h1,
                                           int32_t position, void* lds) {
    typedef Turn<T, INTER, float> turn_t;
    const uint32_t lane = threadIdx.x & 63, d = (lane & 15) * 8;
    const auto at = [&](uint32_t h) { return (size_t)h * r.dim * act_size<T>; };
    uint32_t h = h0 + (lane >> 4);
    float next[8] = {};
    if (d < r.dim && h < h1) load8<T>(in + at(h) + d * act_size<T>, next);
    const turn_t turn(r, d, position, (typename turn_t::cs*)lds);
    if (d >= r.dim) return;
    for (; h < h1; h += 4) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = next[i];
        if (h + 4 < h1) load8<T>(in + at(h + 4) + d * act_size<T>, next);
        turn(r, in + at(h), d, x);
        store8<T>(out + at(h) + d * act_size<T>, x);
    }
}

struct ApplyArgs {
    RotaryArgs r;
    const void* x;
    void* out;
    const int32_t* positions;
    uint32_t rows, heads, per, xstride, ostride;   // per: heads of a wave
};

// Rows turned where they lie, or into other rows.  Bound by its bytes: 8192 bf16 rows
// of 16 heads of 128: 67 MB in 10.7 us, 6.3 TB/s (part of them from the last cache).
template <int T, bool INTER>
__global__ __launch_bounds__(256) void k_rotary(ApplyArgs a) {
    __shared__ __align__(16) float s_turn[4][128];
    const uint32_t parts = (a.heads + a.per - 1) / a.per;
    const uint64_t unit = (uint64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t row = (uint32_t)(unit / parts), h0 = (uint32_t)(unit % parts) * a.per;
    if (row >= a.rows) return;
    turn_heads<T, INTER>(a.r, (const uint8_t*)a.x + (size_t)row * a.xstride * act_size<T>,
                         (uint8_t*)a.out + (size_t)row * a.ostride * act_size<T>, h0, min(h0 + a.per, a.heads), a.positions[row],
                         s_turn[threadIdx.x >> 6]);
}

struct TurnedArgs {
    RotaryArgs r;
    const PageSeq* seqs;
    const int32_t* table;
    const void *q, *k, *v;
    void *out, *pk, *pv, *ks, *vs;
    uint32_t n_seq, rows, uniform, per_seq, shift, kv_heads, heads, per;
    uint32_t qstride, kstride, vstride, ostride;
};

// A pass's rows: waves of a row's queries, `per` heads each, and of four of its kv
// heads, whose keys are turned on their way into the pages.  Codes of 8 or 4 bits
// come of products in 64 bits, rounded to fp32: what rounding in fp32 products
// moves over a code's border would be a whole step.  Bound by its bytes: 24 prompts
// of up to 700 bf16 rows of 16 heads of 128, 4 kv heads into 4-bit pages: 114 MB in 23
// us, 4.9 TB/s; 64 rows 3.5 us, a launch's latency.
template <int T, int CT, bool INTER>
__global__ __launch_bounds__(256) void k_pages_turned(TurnedArgs a) {
    __shared__ __align__(16) double s_turn[4][128];
    const uint32_t kv4 = (a.kv_heads + 3) / 4, parts = kv4 + (a.heads + a.per - 1) / a.per;
    const uint64_t unit = (uint64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t row = (uint32_t)(unit / parts), part = (uint32_t)(unit % parts);
    if (row >= a.rows) return;
    const uint32_t s = a.uniform ? row / a.uniform : seq_of_row(a.seqs, a.n_seq, row);
    const PageSeq q = a.seqs[s];
    const uint32_t pos = q.len - q.rows + (row - q.q0);
    if (part >= kv4) {
        const uint32_t h0 = (part - kv4) * a.per;
        turn_heads<T, INTER>(a.r, (const uint8_t*)a.q + (size_t)row * a.qstride * act_size<T>,
                             (uint8_t*)a.out + (size_t)row * a.ostride * act_size<T>, h0, min(h0 + a.per, a.heads), (int32_t)pos,
                             s_turn[threadIdx.x >> 6]);
        return;
    }
    const uint32_t lane = threadIdx.x & 63, d = (lane & 15) * 8, head = part * 4 + (lane >> 4);
    const uint32_t page = (uint32_t)a.table[(size_t)q.slot * a.per_seq + (pos >> a.shift)];
    const bool live = head < a.kv_heads, on = live && d < a.r.dim;
    const size_t place = (((size_t)page * a.kv_heads + head) << a.shift) + (pos & ((1u << a.shift) - 1));
    const uint8_t* kh = (const uint8_t*)a.k + ((size_t)row * a.kstride + (size_t)head * a.r.dim) * act_size<T>;
    const uint8_t* vh = (const uint8_t*)a.v + ((size_t)row * a.vstride + (size_t)head * a.r.dim) * act_size<T>;
    float x[8] = {}, y[8] = {};
    if (on) {
        load8<T>(kh + d * act_size<T>, x);
        load8<T>(vh + d * act_size<T>, y);
    }
    typedef std::conditional_t<CT == PF_TYPE_I8 || CT == PF_TYPE_FP4, double, float> F;
    typedef Turn<T, INTER, F> turn_t;
    const turn_t turn(a.r, d, (int32_t)pos, (typename turn_t::cs*)s_turn[threadIdx.x >> 6]);
    if (on) turn(a.r, kh, d, x);
    page_put8<CT>(x, live, a.pk, a.ks, place, d, a.r.dim);
    page_put8<CT>(y, live, a.pv, a.vs, place, d, a.r.dim);
}

}  // namespace pf

using namespace pf;

// ================================================================== host

extern "C" void pf_rotary_destroy(pf_rotary* r) {
    if (!r) return;
    DeviceScope on(r->ctx);
    (void)hipStreamSynchronize(r->ctx->stream);
    dfree(r->ctx, r->table, ROTARY_MOST * 16);
    delete r;
}

extern "C" pf_status pf_rotary_create(pf_ctx* c, const pf_rotary_desc* d, pf_rotary** out) {
    if (!c || !d || !out) return PF_ERR_ARG;
    *out = nullptr;
    if (!d->head_dim || d->head_dim % 16 || d->head_dim > 128)
        return fail(c, PF_ERR_UNSUPPORTED, "rotary: head_dim is a multiple of 16 up to 128");
    if (d->turn % 8 || d->turn > d->head_dim) return fail(c, PF_ERR_ARG, "rotary: turn is a multiple of 8 up to head_dim");
    const float base = d->base == 0.0f ? 5e6f : d->base, factor = d->factor == 0.0f ? 1.0f : d->factor;
    const float magnitude = d->magnitude == 0.0f ? 1.0f : d->magnitude;
    if (!(base > 1.0f) || !std::isfinite(base)) return fail(c, PF_ERR_ARG, "rotary: base is above 1");
    if (!(factor > 0.0f) || !std::isfinite(factor)) return fail(c, PF_ERR_ARG, "rotary: factor is positive");
    if (!(magnitude > 0.0f) || !std::isfinite(magnitude)) return fail(c, PF_ERR_ARG, "rotary: magnitude is positive");
    const bool ramp = d->low != 0.0f || d->high != 0.0f;
    if (ramp && !(d->low >= 0.0f && d->high > d->low && std::isfinite(d->high)))
        return fail(c, PF_ERR_ARG, "rotary: low and high are 0, or low below high");
    if (ramp && !d->original) return fail(c, PF_ERR_ARG, "rotary: original is the rows of the original context");
    DeviceScope on(c);
    pf_rotary* r = new (std::nothrow) pf_rotary();
    if (!r) return fail(c, PF_ERR_CAPACITY, "out of host memory");
    r->ctx = c;
    r->desc = *d;
    r->desc.magnitude = magnitude;
    r->turn = d->turn ? d->turn : d->head_dim;
    double table[2 * ROTARY_MOST] = {};
    const long double two_pi = 6.283185307179586476925286766559L;
    for (uint32_t i = 0; i < r->turn / 2; i++) {
        long double f = powl((long double)base, -2.0L * i / r->turn) / two_pi;
        long double keep = 0.0L;
        if (ramp) {
            keep = (f * d->original - (long double)d->low) / ((long double)d->high - (long double)d->low);
            keep = std::min(std::max(keep, 0.0L), 1.0L);
        }
        f *= keep + (1.0L - keep) / (long double)factor;
        table[2 * i] = (double)f;
        table[2 * i + 1] = (double)(f - (long double)table[2 * i]);
    }
    pf_status s = dalloc(c, (void**)&r->table, ROTARY_MOST * 16);
    if (!s && hipMemcpy(r->table, table, sizeof(table), hipMemcpyHostToDevice) != hipSuccess)
        s = fail(c, PF_ERR_HIP, "rotary: the table's copy failed");
    if (s) {
        const std::string msg = c->err;
        pf_rotary_destroy(r);
        return fail(c, s, msg);
    }
    *out = r;
    return PF_OK;
}

static RotaryArgs rotary_args(const pf_rotary* r) { return {r->table, (double)r->desc.magnitude, r->turn, r->desc.head_dim}; }

// Heads of a wave: all of a row's, as few waves as fill the card (8 on each of its
// 1024 SIMDs), since a wave forms its angles once (8192 bf16 rows of 16 heads of 128:
// 11.3 us, 14.1 with four heads a wave); fewer of them otherwise, which a wave
// has one after another (64 rows of 128 heads: 5.8 us, 11.7 with all in a wave).
static uint32_t heads_of_wave(uint32_t rows, uint32_t heads) {
    uint32_t per = (heads + 3) / 4 * 4;
    while (per > 4 && (uint64_t)rows * ((heads + per - 1) / per) < 8192) per = (per / 2 + 3) / 4 * 4;
    return per;
}

static pf_status row_stride(pf_ctx* c, uint32_t* stride, uint32_t heads, uint32_t dim, int32_t type) {
    const uint64_t least = (uint64_t)heads * dim, w = *stride ? *stride : least;
    if (w < least || w > 0xFFFFFFFFu || w % (type == PF_TYPE_F32 ? 4 : 8))
        return fail(c, PF_ERR_ARG, "rotary: strides hold every head and are multiples of 16 bytes");
    *stride = (uint32_t)w;
    return PF_OK;
}

static pf_status heads_check(pf_ctx* c, int32_t type, uint32_t heads) {
    if (type != PF_TYPE_F32 && type != PF_TYPE_F16 && type != PF_TYPE_BF16)
        return fail(c, PF_ERR_ARG, "rotary: rows are PF_TYPE_F32, F16 or BF16");
    if (!heads || heads > 65535) return fail(c, PF_ERR_ARG, "rotary: 1 to 65535 heads");
    return PF_OK;
}

// A launch's workgroups: a grid dimension holds fewer than 2^32 threads.
constexpr uint64_t ROTARY_BLOCKS = 1u << 23;

template <int T>
static void apply_type(hipStream_t st, bool inter, uint32_t blocks, const ApplyArgs& a) {
    if (inter) hipLaunchKernelGGL((k_rotary<T, true>), dim3(blocks), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_rotary<T, false>), dim3(blocks), dim3(256), 0, st, a);
}

extern "C" pf_status pf_rotary_apply(const pf_rotary* r, int32_t type, uint32_t heads, const void* x, void* out,
                                     const int32_t* positions, uint32_t rows, uint32_t xs, uint32_t os) {
    if (!r) return PF_ERR_ARG;
    pf_ctx* c = r->ctx;
    const uint32_t dim = r->desc.head_dim;
    if (pf_status st = heads_check(c, type, heads)) return st;
    for (uint32_t* s : {&xs, &os})
        if (pf_status st = row_stride(c, s, heads, dim, type)) return st;
    if (!rows) return PF_OK;
    if (!x || !out || !positions) return fail(c, PF_ERR_ARG, "rotary: a buffer is NULL");
    if (!aligned16(x) || !aligned16(out)) return fail(c, PF_ERR_ARG, "rotary: buffers start on 16 bytes");
    if ((uintptr_t)positions & 3) return fail(c, PF_ERR_ARG, "rotary: positions start on 4 bytes");
    const size_t es = type == PF_TYPE_F32 ? 4 : 2, w = (size_t)heads * dim * es;
    if (!(out == x && xs == os) && rows_overlap(out, os * es, x, xs * es, w, w, rows))
        return fail(c, PF_ERR_ARG, "rotary: out overlaps x");
    if (overlaps(out, (rows - 1) * (size_t)os * es + w, positions, (size_t)rows * 4))
        return fail(c, PF_ERR_ARG, "rotary: out overlaps the positions");
    ApplyArgs a{rotary_args(r), x, out, positions, rows, heads, heads_of_wave(rows, heads), xs, os};
    const uint64_t blocks = ((uint64_t)rows * ((heads + a.per - 1) / a.per) + 3) / 4;
    if (blocks > ROTARY_BLOCKS) return fail(c, PF_ERR_UNSUPPORTED, "rotary: too many rows at once");
    DeviceScope on(c);
    const bool inter = r->desc.interleaved != 0;
    if (type == PF_TYPE_F32) apply_type<PF_TYPE_F32>(c->stream, inter, (uint32_t)blocks, a);
    else if (type == PF_TYPE_F16) apply_type<PF_TYPE_F16>(c->stream, inter, (uint32_t)blocks, a);
    else apply_type<PF_TYPE_BF16>(c->stream, inter, (uint32_t)blocks, a);
    PF_LAUNCHED(c);
    return PF_OK;
}

template <int T, int CT>
static void turned_inter(hipStream_t st, bool inter, uint32_t blocks, const TurnedArgs& a) {
    if (inter) hipLaunchKernelGGL((k_pages_turned<T, CT, true>), dim3(blocks), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_pages_turned<T, CT, false>), dim3(blocks), dim3(256), 0, st, a);
}
template <int CT>
static void turned_type(hipStream_t st, int32_t type, bool inter, uint32_t blocks, const TurnedArgs& a) {
    if (type == PF_TYPE_F32) turned_inter<PF_TYPE_F32, CT>(st, inter, blocks, a);
    else if (type == PF_TYPE_F16) turned_inter<PF_TYPE_F16, CT>(st, inter, blocks, a);
    else turned_inter<PF_TYPE_BF16, CT>(st, inter, blocks, a);
}

extern "C" pf_status pf_pages_store_rotary(pf_pages* p, uint32_t layer, const pf_rotary* r, int32_t type, uint32_t heads,
                                           const void* q, const void* k, const void* v, void* out, uint32_t qs, uint32_t ks,
                                           uint32_t vs, uint32_t os) {
    if (!p || !r) return PF_ERR_ARG;
    pf_ctx* c = p->ctx;
    const pf_pages_config& g = p->cfg;
    const uint32_t dim = g.head_dim;
    if (r->ctx != c || r->desc.head_dim != dim) return fail(c, PF_ERR_ARG, "pages: the rotary handle is of the cache's context and head_dim");
    if (layer >= g.n_layers) return fail(c, PF_ERR_ARG, "pages: layer out of range");
    if (pf_status st = heads_check(c, type, heads)) return st;
    for (uint32_t* s : {&qs, &os})
        if (pf_status st = row_stride(c, s, heads, dim, type)) return st;
    for (uint32_t* s : {&ks, &vs})
        if (pf_status st = row_stride(c, s, g.n_kv_heads, dim, type)) return st;
    if (!p->open) return fail(c, PF_ERR_STATE, "pages: no open pass (pf_pages_append begins one)");
    const uint32_t rows = p->pass_rows;
    if (!rows) return PF_OK;
    if (!q || !k || !v || !out) return fail(c, PF_ERR_ARG, "pages: a buffer is NULL");
    for (const void* b : {q, k, v, (const void*)out})
        if (!aligned16(b)) return fail(c, PF_ERR_ARG, "pages: buffers start on 16 bytes");
    const size_t es = type == PF_TYPE_F32 ? 4 : 2, w = (size_t)heads * dim * es, wk = (size_t)g.n_kv_heads * dim * es;
    if ((!(out == q && qs == os) && rows_overlap(out, os * es, q, qs * es, w, w, rows)) ||
        rows_overlap(out, os * es, k, ks * es, w, wk, rows) || rows_overlap(out, os * es, v, vs * es, w, wk, rows))
        return fail(c, PF_ERR_ARG, "pages: q_out overlaps the rows");
    TurnedArgs a{};
    a.r = rotary_args(r);
    a.seqs = p->seqs; a.table = p->table; a.q = q; a.k = k; a.v = v; a.out = out;
    a.pk = (uint8_t*)p->k + layer * p->plane; a.pv = (uint8_t*)p->v + layer * p->plane;
    a.ks = (uint8_t*)p->ks + layer * p->scales; a.vs = (uint8_t*)p->vs + layer * p->scales;
    a.n_seq = (uint32_t)p->pass.size(); a.rows = rows; a.uniform = p->uniform; a.per_seq = p->per_seq;
    a.shift = p->shift; a.kv_heads = g.n_kv_heads; a.heads = heads; a.per = heads_of_wave(rows, heads);
    a.qstride = qs; a.kstride = ks; a.vstride = vs; a.ostride = os;
    const uint64_t blocks = ((uint64_t)rows * ((g.n_kv_heads + 3) / 4 + (heads + a.per - 1) / a.per) + 3) / 4;
    if (blocks > ROTARY_BLOCKS) return fail(c, PF_ERR_UNSUPPORTED, "pages: too many rows in one pass; cut it");
    DeviceScope on(c);
    const bool inter = r->desc.interleaved != 0;
    if (g.type == PF_TYPE_FP4) turned_type<PF_TYPE_FP4>(c->stream, type, inter, (uint32_t)blocks, a);
    else if (g.type == PF_TYPE_I8) turned_type<PF_TYPE_I8>(c->stream, type, inter, (uint32_t)blocks, a);
    else if (g.type == PF_TYPE_F16) turned_type<PF_TYPE_F16>(c->stream, type, inter, (uint32_t)blocks, a);
    else turned_type<PF_TYPE_BF16>(c->stream, type, inter, (uint32_t)blocks, a);
    PF_LAUNCHED(c);
    return PF_OK;
}
