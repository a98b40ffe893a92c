// The paged cache's host object and the arguments of its kernels (pf_pages.hip:
// bookkeeping, stores and moves; pf_paged.hip: attention).
#pragma once
#include <vector>

#include "pf_attend.h"
#include "pf_context.h"

namespace pf {

// A sequence of the open pass: its rows are q0 .. q0 + rows - 1 of the packed
// rows and the last `rows` of the `len` that the sequence holds.
struct PageSeq {
    uint32_t slot, q0, rows, len;
};

// One workgroup's share of a sequence's keys: tiles t0 .. t1 - 1 of PG_KEYS of
// the keys that its rows see.  Part `part` of `parts`; its results go to rows
// ws0 + part * rows .. of the partial results, or, where parts == 1, to the
// output.
struct PageItem {
    uint32_t slot, q0, rows, len, t0, t1, ws0, parts, part;
};
constexpr uint32_t PG_KEYS = 32;
constexpr uint32_t PG_MOST_PARTS = 1024;   // of one sequence
constexpr uint32_t PG_MOST_ITEMS = 1024;   // of a pass, or two for each sequence

// How the pass's keys are cut, kept for the layers that follow.
struct PageSplit {
    uint32_t window = 0, sink = 0, heads = 0;
    int32_t type = -1;
    uint32_t n_items = 0, ws_rows = 0, most_rows = 0;
    uint32_t longest = 0;         // keys of the longest sequence
    uint32_t waves = 4;
    bool split = false;
};

// Keys that a sequence's pass sees, in tiles: the sink tiles before the first
// tile of the window, then the window's to the end.
struct PageTiles {
    int first, sinks, count;
};
__host__ __device__ __forceinline__ PageTiles page_tiles(uint32_t rows, uint32_t len, uint32_t window, uint32_t sink) {
    PageTiles t;
    const int p0 = (int)(len - rows);
    const int lo = window && p0 >= (int)window ? p0 - (int)window + 1 : 0;
    t.first = lo / (int)PG_KEYS;
    const int s = (int)((sink + PG_KEYS - 1) / PG_KEYS);
    t.sinks = s < t.first ? s : t.first;
    t.count = (int)((len + PG_KEYS - 1) / PG_KEYS) - t.first + t.sinks;
    return t;
}

struct PagedArgs {
    const PageItem* items;
    const int32_t* table;
    uint32_t table_stride;
    const void *k, *v;            // this layer's planes
    const void *ks, *vs;          // int8: fp32 scales; 4 bits: exponent bytes
    const void* q;
    void* out;
    uint32_t qs, os, n_heads, kv_heads, group, dim, page_shift;
    int32_t causal, window, sink;
    float scale_log2;
    float above, down;            // as in pf_prompt.hip
    float* ws_o;                  // [ws_rows][n_heads][dim]
    float* ws_ml;                 // [ws_rows][n_heads][2]
};

// The sequence of a packed row: the last one whose first row is not past it
// (sequences without rows share their first row with the next one's, and come
// before it).  A wave looks at 64 of them at a time.
__device__ __forceinline__ uint32_t seq_of_row(const PageSeq* seqs, uint32_t n, uint32_t row) {
    uint32_t lo = 0, count = n;
    while (count > 64) {
        const uint32_t step = (count + 63) / 64, i = (threadIdx.x & 63) * step;
        const uint64_t b = __ballot(i < count && seqs[lo + i].q0 <= row);
        const uint32_t k = 63 - (uint32_t)__builtin_clzll(b);
        lo += k * step;
        count = min(step, count - k * step);
    }
    const uint32_t i = threadIdx.x & 63;
    const uint64_t b = __ballot(i < count && seqs[lo + i].q0 <= row);
    return lo + 63 - (uint32_t)__builtin_clzll(b);
}

// Eight values of a row of one head (dims d .. d + 7, one of 16 lanes that hold
// it; zeros past the last dim) into the row's place in a layer's plane.  Lanes of
// a head that is not there (`live` false) take part.  int8:
// KVCache::quantize_row's arithmetic (code = round(x * (127 / max|x|)), scale =
// max|x| / 127).
template <int CT>
__device__ __forceinline__ void page_put8(const float (&x)[8], bool live, void* plane, void* scales, size_t place, uint32_t d,
                                          uint32_t dim) {
    const bool on = live && d < dim;
    if constexpr (CT == PF_TYPE_I8 || CT == PF_TYPE_FP4) {
        float amax = 0.0f;
        bool odd = false;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            amax = fmaxf(amax, fabsf(x[i]));
            odd |= !(fabsf(x[i]) < INFINITY);
        }
        uint32_t bad = odd;
        // (4 lanes hold a block of 32)
#pragma unroll
        for (int b = 1; b < (CT == PF_TYPE_FP4 ? 4 : 16); b <<= 1) {
            amax = fmaxf(amax, __shfl_xor(amax, b));
            bad |= (uint32_t)__shfl_xor((int)bad, b);
        }
        if constexpr (CT == PF_TYPE_FP4) {
            const uint32_t blocks = fp4_blocks(dim), e = fp4_exponent(amax);
            if (!live || d >= blocks * FP4_BLOCK) return;
            *(uint32_t*)((uint8_t*)plane + place * blocks * 16 + d / 2) = bad ? 0u : fp4_pack(x, fp4_scale(e));
            if (d % FP4_BLOCK == 0) ((uint8_t*)scales)[place * blocks + d / FP4_BLOCK] = (uint8_t)(bad ? 255u : e);
        } else {
            // (rows below 2^-121 have an infinite 127 / max|x|: the largest float keeps their codes finite)
            const float inv = amax == 0.0f ? 1.0f : fminf(127.0f / amax, 3.4028234663852886e38f);
            uint32_t c[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int code = bad ? 0 : (int)__builtin_roundf(x[i] * inv);
                c[i / 4] |= (uint32_t)(uint8_t)(int8_t)code << (8 * (i % 4));
            }
            if (on) {
                u2v r = {c[0], c[1]};
                *(u2v*)((uint8_t*)plane + place * dim + d) = r;
                if (d == 0) ((float*)scales)[place] = bad ? NAN : amax == 0.0f ? 1.0f : amax / 127.0f;
            }
        }
    } else if (on) {
        *(s8v*)((uint8_t*)plane + (place * dim + d) * 2) = pack8<CT == PF_TYPE_BF16>(x);
    }
}

}  // namespace pf

struct PageStaging;

struct pf_pages {
    pf_ctx* ctx = nullptr;
    pf_pages_config cfg{};
    uint32_t shift = 0, per_seq = 0;               // log2(page_size), table entries of a sequence
    uint32_t row_bytes = 0, scale_bytes = 0;       // of a row of one head, of its scales (0: none)
    size_t plane = 0, scales = 0;                  // bytes of a layer's rows, of their scales
    size_t bytes = 0;
    void *k = nullptr, *v = nullptr;
    void *ks = nullptr, *vs = nullptr;
    int32_t* table = nullptr;                      // device [max_seqs][per_seq]
    pf::PageSeq* seqs = nullptr;                   // device: the open pass
    pf::PageItem* items = nullptr;                 // device
    size_t items_cap = 0;
    uint32_t* pairs = nullptr;                     // device: page copies under way
    PageStaging* staging = nullptr;

    std::vector<uint32_t> refs, len;               // per page, per sequence
    std::vector<std::vector<uint32_t>> pages;      // per sequence
    std::vector<uint32_t> heap;                    // free pages, lowest first
    std::vector<uint32_t> dirty;                   // table entries that the device has not heard of
    std::vector<uint32_t> mark;                    // per sequence: last call that named it
    uint32_t stamp = 0;

    bool open = false;
    std::vector<pf::PageSeq> pass;
    uint32_t pass_rows = 0, uniform = 0;           // rows in all; rows of each sequence, 0 if they differ
    pf::PageSplit cut;
};

// (pf_pages.hip) copies words to device memory in stream order.
pf_status pages_upload(pf_pages* p, void* dst_dev, const void* src, size_t bytes);
