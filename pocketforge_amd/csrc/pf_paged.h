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
    const float *ks, *vs;
    const void* q;
    void* out;
    uint32_t qs, os, n_heads, kv_heads, group, dim, page_shift;
    int32_t causal, window, sink;
    float scale_log2;
    float above, down;            // as in pf_prompt.hip
    float* ws_o;                  // [ws_rows][n_heads][dim]
    float* ws_ml;                 // [ws_rows][n_heads][2]
};

}  // namespace pf

struct PageStaging;

struct pf_pages {
    pf_ctx* ctx = nullptr;
    pf_pages_config cfg{};
    uint32_t shift = 0, per_seq = 0;               // log2(page_size), table entries of a sequence
    size_t plane = 0, esize = 0, scales = 0;       // bytes of a plane, of a value; scales of a plane
    size_t bytes = 0;
    void *k = nullptr, *v = nullptr;
    float *ks = nullptr, *vs = nullptr;
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
