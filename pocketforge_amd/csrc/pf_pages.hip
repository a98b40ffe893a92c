// The paged cache (pf_pages_* of include/pf_gpu.h but for its attention):
// page bookkeeping on the host, mirrored to the device in stream order, and the
// kernels that store, read back and copy rows.
//
// The host decides everything: a call checks its arguments, changes the
// tables, and sends the device what changed through a ring of pinned
// buffers, so that a page number that a kernel reads always names a page of
// the pool.  Rows are row-major in a page ([kv head][row][dim]), K and V
// alike: a page's rows of one head are one piece of memory for the attention's
// loads, a new row is two lines, and a copy is a plain copy.
#include "pf_paged.h"

#include <cstring>
#include <functional>

using namespace pf;

namespace pf {

// Takes a message to its places: `words` words to dst, then `pairs` (index,
// value) pairs into the page table.  One workgroup.  Small messages come as the
// kernel's arguments (nothing to keep until it has run: fork and grow 18 us,
// 44 by way of a copy from pinned memory), others lie in pinned host memory.
__device__ __forceinline__ void pages_apply(const uint32_t* msg, uint32_t words, uint32_t* dst, uint32_t pairs,
                                            int32_t* table) {
    for (uint32_t i = threadIdx.x; i < words; i += blockDim.x) dst[i] = msg[i];
    for (uint32_t i = threadIdx.x; i < pairs; i += blockDim.x) table[msg[words + 2 * i]] = (int32_t)msg[words + 2 * i + 1];
}
__global__ __launch_bounds__(1024) void k_pages_apply(const uint32_t* msg, uint32_t words, uint32_t* dst, uint32_t pairs,
                                                     int32_t* table) {
    pages_apply(msg, words, dst, pairs, table);
}
constexpr uint32_t SMALL_WORDS = 640;
struct SmallMessage {
    uint32_t* dst;
    int32_t* table;
    uint32_t words, pairs;
    uint32_t msg[SMALL_WORDS];
};

struct StoreArgs {
    const PageSeq* seqs;
    const int32_t* table;
    const void *k, *v;
    void *pk, *pv, *ks, *vs;
    uint32_t n_seq, rows, uniform, per_seq, shift, kv_heads, dim, kstride, vstride;
};

// New rows into their pages.  16 lanes hold a row of one head, 8 values each; a
// wave has 4 heads of a token, K and V in turn.  Bound by
// its bytes where there are many: 4717 fp32 rows of 16 heads of 128 to int8, 97
// MB in 19 us, 5.1 TB/s, to 4 bits 88 MB in 16 us, 5.5 TB/s; a decode step's 64
// bf16 rows 3 us, a launch's latency.
template <int T, int CT>
__global__ __launch_bounds__(256) void k_pages_store(StoreArgs a) {
    const uint32_t lane = threadIdx.x & 63, quarter = lane >> 4, d = (lane & 15) * 8;
    const uint32_t heads4 = (a.kv_heads + 3) / 4;
    const uint64_t unit = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);   // (row, 4 heads)
    const uint32_t row = (uint32_t)(unit / heads4), head = (uint32_t)(unit % heads4) * 4 + quarter;
    if (row >= a.rows) return;                   // (whole waves)
    const uint32_t s = a.uniform ? row / a.uniform : seq_of_row(a.seqs, a.n_seq, row);
    const PageSeq q = a.seqs[s];
    const uint32_t pos = q.len - q.rows + (row - q.q0);
    const uint32_t page = (uint32_t)a.table[(size_t)q.slot * a.per_seq + (pos >> a.shift)];
    const bool live = head < a.kv_heads, on = live && d < a.dim;
    const size_t place = (((size_t)page * a.kv_heads + head) << a.shift) + (pos & ((1u << a.shift) - 1));
#pragma unroll
    for (int w = 0; w < 2; w++) {
        const void* src = w ? a.v : a.k;
        const uint32_t stride = w ? a.vstride : a.kstride;
        float x[8] = {};
        if (on) load8<T>((const uint8_t*)src + ((size_t)row * stride + (size_t)head * a.dim + d) * act_size<T>, x);
        page_put8<CT>(x, live, w ? a.pv : a.pk, w ? a.vs : a.ks, place, d, a.dim);
    }
}

constexpr int GATHER_SEQS = 64;
struct GatherArgs {
    const int32_t* table;
    const void *pk, *pv, *ks, *vs;
    void *k, *v;
    uint32_t n_seq, rows, per_seq, shift, kv_heads, dim, kstride, vstride, row0;
    uint32_t first[GATHER_SEQS], slot[GATHER_SEQS];   // first packed row, sequence
};

// Pages back into packed rows; lanes as in k_pages_store.  4867 rows of 16 heads
// of 128, int8 to fp32: 100 MB in 19 us, 5.3 TB/s; 4 bits: 90 MB in 19, 4.8.
template <int T, int CT>
__global__ __launch_bounds__(256) void k_pages_gather(GatherArgs a) {
    const uint32_t lane = threadIdx.x & 63, quarter = lane >> 4, d = (lane & 15) * 8;
    const uint32_t heads4 = (a.kv_heads + 3) / 4;
    const uint64_t unit = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const uint32_t row = (uint32_t)(unit / heads4), head = (uint32_t)(unit % heads4) * 4 + quarter;
    if (row >= a.rows) return;
    const uint64_t b = __ballot(lane < a.n_seq && a.first[lane] <= row);
    const uint32_t s = 63 - (uint32_t)__builtin_clzll(b), pos = row - a.first[s];
    if (head >= a.kv_heads || d >= a.dim) return;
    const uint32_t page = (uint32_t)a.table[(size_t)a.slot[s] * a.per_seq + (pos >> a.shift)];
    const size_t place = (((size_t)page * a.kv_heads + head) << a.shift) + (pos & ((1u << a.shift) - 1));
#pragma unroll
    for (int w = 0; w < 2; w++) {
        const uint8_t* src = (const uint8_t*)(w ? a.pv : a.pk);
        float x[8];
        if constexpr (CT == PF_TYPE_I8) {
            const u2v c = *(const u2v*)(src + place * a.dim + d);
            const float sc = ((const float*)(w ? a.vs : a.ks))[place];
            codes8(c[0], c[1], x);
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] *= sc;
        } else if constexpr (CT == PF_TYPE_FP4) {
            const uint32_t blocks = fp4_blocks(a.dim);
            const uint32_t c = *(const uint32_t*)(src + place * blocks * 16 + d / 2);
            fp4_floats(c, fp4_scale(((const uint8_t*)(w ? a.vs : a.ks))[place * blocks + d / FP4_BLOCK]), x);
        } else {
            load8<CT>(src + (place * a.dim + d) * 2, x);
        }
        uint8_t* dst = (uint8_t*)(w ? a.v : a.k) +
                       ((size_t)(a.row0 + row) * (w ? a.vstride : a.kstride) + (size_t)head * a.dim + d) * act_size<T>;
        if constexpr (T == PF_TYPE_F32) {
            f4v lo = {x[0], x[1], x[2], x[3]}, hi = {x[4], x[5], x[6], x[7]};
            ((f4v*)dst)[0] = lo;
            ((f4v*)dst)[1] = hi;
        } else {
            *(s8v*)dst = pack8<T == PF_TYPE_BF16>(x);
        }
    }
}

// Copies pages: (from, to, rows) of every layer and head, K and V and their
// scales.  One workgroup takes one (copy, layer) and a share of its heads.
// Outputs pass the caches: 12 sequences of 24 pages, 24 layers, write 905 MB in
// 176 us, 5.1 TB/s (their one source stays in the caches), 227 us otherwise.
struct MoveArgs {
    uint8_t *k, *v, *ks, *vs;
    uint32_t kv_heads, page_size, row_bytes, scale_bytes;
    size_t plane, scales;         // bytes of one layer's
};
__device__ __forceinline__ void move_page(const MoveArgs& a, uint32_t src, uint32_t dst, uint32_t rows, uint32_t layer,
                                          uint32_t h0, uint32_t dh) {
    const size_t head_bytes = (size_t)a.page_size * a.row_bytes, page = head_bytes * a.kv_heads;
    const uint32_t n16 = rows * a.row_bytes / 16;             // of one head
    for (uint32_t h = h0; h < a.kv_heads; h += dh) {
        const size_t at = layer * a.plane + h * head_bytes;
#pragma unroll
        for (int w = 0; w < 2; w++) {
            uint8_t* p = (w ? a.v : a.k) + at;
            const u4v* s = (const u4v*)(p + src * page);
            u4v* d = (u4v*)(p + dst * page);
            uint32_t i = threadIdx.x;
            for (; i + 768 < n16; i += 1024) {                // four loads under way
                const u4v x0 = s[i], x1 = s[i + 256], x2 = s[i + 512], x3 = s[i + 768];
                __builtin_nontemporal_store(x0, d + i);
                __builtin_nontemporal_store(x1, d + i + 256);
                __builtin_nontemporal_store(x2, d + i + 512);
                __builtin_nontemporal_store(x3, d + i + 768);
            }
            for (; i < n16; i += 256) d[i] = s[i];
            if (a.ks) {
                // whole words (a head's scales in a page are words, whatever the rows' are)
                const size_t head_scales = (size_t)a.page_size * a.scale_bytes, per = head_scales * a.kv_heads;
                uint8_t* sc = (w ? a.vs : a.ks) + layer * a.scales + h * head_scales;
                const uint32_t* s = (const uint32_t*)(sc + src * per);
                uint32_t* d = (uint32_t*)(sc + dst * per);
                for (uint32_t r = threadIdx.x; r < (rows * a.scale_bytes + 3) / 4; r += 256) d[r] = s[r];
            }
        }
    }
}
__global__ __launch_bounds__(256) void k_pages_move(MoveArgs a, const uint32_t* pairs) {
    const uint32_t* pr = pairs + 3 * blockIdx.x;
    move_page(a, pr[0], pr[1], pr[2], blockIdx.y, blockIdx.z, gridDim.z);
}

// A small message and a few copies in one launch; neither reads what the other
// writes.  2 us for a message, 5 with 8 copies of 40 rows of 12 layers; latency.
constexpr uint32_t FEW_MOVES = 64;
struct FewMoves {
    uint32_t list[3 * FEW_MOVES];
};
__global__ __launch_bounds__(256) void k_pages_change(SmallMessage m, MoveArgs a, FewMoves few) {
    if (blockIdx.x == 0) {
        if (blockIdx.y == 0 && blockIdx.z == 0) pages_apply(m.msg, m.words, m.dst, m.pairs, m.table);
        return;
    }
    const uint32_t* pr = few.list + 3 * (blockIdx.x - 1);
    move_page(a, pr[0], pr[1], pr[2], blockIdx.y, blockIdx.z, gridDim.z);
}

}  // namespace pf

// =============================================================== staging

// Messages to the device: a ring of pinned buffers, each free again once the
// kernel that reads it is done.
constexpr size_t STAGE_BYTES = 32 << 10;
constexpr int STAGE_SLOTS = 32;
struct PageStaging {
    uint32_t* mem = nullptr;
    hipEvent_t done[STAGE_SLOTS] = {};
    bool used[STAGE_SLOTS] = {};
    int at = 0;
};

static pf_status stage_slot(pf_pages* p, uint32_t** out) {
    PageStaging* s = p->staging;
    if (s->used[s->at]) PF_HIP(p->ctx, hipEventSynchronize(s->done[s->at]));
    *out = s->mem + (size_t)s->at * (STAGE_BYTES / 4);
    return PF_OK;
}

static pf_status stage_send(pf_pages* p, const uint32_t* msg, uint32_t words, void* dst, uint32_t pairs) {
    PageStaging* s = p->staging;
    hipStream_t st = p->ctx->stream;
    hipLaunchKernelGGL(k_pages_apply, dim3(1), dim3(1024), 0, st, msg, words, (uint32_t*)dst, pairs, p->table);
    PF_LAUNCHED(p->ctx);
    PF_HIP(p->ctx, hipEventRecord(s->done[s->at], st));
    s->used[s->at] = true;
    s->at = (s->at + 1) % STAGE_SLOTS;
    return PF_OK;
}

static MoveArgs move_args(const pf_pages* p) {
    const pf_pages_config& g = p->cfg;
    MoveArgs a{};
    a.k = (uint8_t*)p->k; a.v = (uint8_t*)p->v; a.ks = (uint8_t*)p->ks; a.vs = (uint8_t*)p->vs;
    a.kv_heads = g.n_kv_heads; a.page_size = g.page_size; a.row_bytes = p->row_bytes; a.scale_bytes = p->scale_bytes;
    a.plane = p->plane; a.scales = p->scales;
    return a;
}

// Words to device memory, table entries (by index; the values are the host's)
// behind them, and page copies (from, to, rows) if they fit: *moved says so.
static pf_status stage_all(pf_pages* p, void* dst, const void* src, size_t bytes, const std::vector<uint32_t>& changed,
                           const std::vector<uint32_t>& moves, bool* moved) {
    *moved = moves.empty();
    const size_t n = changed.size();
    const auto value = [&](uint32_t at, uint32_t* v) {
        const std::vector<uint32_t>& t = p->pages[at / p->per_seq];
        if (at % p->per_seq >= t.size()) return false;       // dropped since
        *v = t[at % p->per_seq];
        return true;
    };
    const uint32_t few = moves.size() / 3 <= FEW_MOVES ? (uint32_t)(moves.size() / 3) : 0;
    if (!bytes && !n && !few) return PF_OK;
    if (bytes / 4 + 2 * n <= SMALL_WORDS) {
        SmallMessage m;
        m.dst = (uint32_t*)dst; m.table = p->table; m.words = (uint32_t)(bytes / 4); m.pairs = 0;
        if (bytes) std::memcpy(m.msg, src, bytes);
        for (uint32_t at : changed) {
            uint32_t* w = m.msg + m.words + 2 * m.pairs;
            if (!value(at, w + 1)) continue;
            w[0] = at;
            m.pairs++;
        }
        FewMoves f;
        if (few) std::memcpy(f.list, moves.data(), (size_t)few * 12);
        const dim3 grid = few ? dim3(1 + few, p->cfg.n_layers, p->cfg.n_kv_heads) : dim3(1);
        hipLaunchKernelGGL(k_pages_change, grid, dim3(256), 0, p->ctx->stream, m, move_args(p), f);
        PF_LAUNCHED(p->ctx);
        *moved |= few != 0;
        return PF_OK;
    }
    size_t at = 0, c = 0;
    while (at < bytes || c < n) {
        uint32_t* m = nullptr;
        if (pf_status st = stage_slot(p, &m)) return st;
        const size_t take = std::min(bytes - at, STAGE_BYTES);
        if (take) std::memcpy(m, (const uint8_t*)src + at, take);
        const uint32_t words = (uint32_t)(take / 4), room = (uint32_t)(STAGE_BYTES / 4 - words) / 2;
        uint32_t pairs = 0;
        if (at + take == bytes)
            for (; c < n && pairs < room; c++) {
                uint32_t* w = m + words + 2 * pairs;
                if (!value(changed[c], w + 1)) continue;
                w[0] = changed[c];
                pairs++;
            }
        if (pf_status st = stage_send(p, m, words, dst ? (uint8_t*)dst + at : nullptr, pairs)) return st;
        at += take;
    }
    return PF_OK;
}

pf_status pages_upload(pf_pages* p, void* dst_dev, const void* src, size_t bytes) {
    bool moved;
    return stage_all(p, dst_dev, src, bytes, {}, {}, &moved);
}

// Table entries that have changed since the device last heard.
static pf_status tables_to_device(pf_pages* p) {
    bool moved;
    if (pf_status st = stage_all(p, nullptr, nullptr, 0, p->dirty, {}, &moved)) return st;
    p->dirty.clear();
    return PF_OK;
}

// ============================================================ page copies

// Copies of (from, to, rows); no page is both.
constexpr size_t MOVE_MOST = STAGE_BYTES / 12;
static pf_status move_pages(pf_pages* p, const std::vector<uint32_t>& moves) {
    for (size_t at = 0; at < moves.size() / 3; at += MOVE_MOST) {
        const uint32_t n = (uint32_t)std::min(MOVE_MOST, moves.size() / 3 - at);
        if (pf_status st = pages_upload(p, p->pairs, moves.data() + 3 * at, (size_t)n * 12)) return st;
        hipLaunchKernelGGL(k_pages_move, dim3(n, p->cfg.n_layers, p->cfg.n_kv_heads), dim3(256), 0, p->ctx->stream,
                           move_args(p), p->pairs);
        PF_LAUNCHED(p->ctx);
    }
    return PF_OK;
}

// ============================================================ bookkeeping

static uint32_t take_page(pf_pages* p) {
    std::pop_heap(p->heap.begin(), p->heap.end(), std::greater<uint32_t>());
    const uint32_t page = p->heap.back();
    p->heap.pop_back();
    p->refs[page] = 1;
    return page;
}
static void drop_page(pf_pages* p, uint32_t page) {
    if (--p->refs[page]) return;
    p->heap.push_back(page);
    std::push_heap(p->heap.begin(), p->heap.end(), std::greater<uint32_t>());
}
static uint32_t pages_for(const pf_pages* p, uint32_t rows) { return (rows + p->cfg.page_size - 1) >> p->shift; }
static void cut_pages(pf_pages* p, uint32_t seq, uint32_t rows) {
    std::vector<uint32_t>& t = p->pages[seq];
    const uint32_t keep = pages_for(p, rows);
    while (t.size() > keep) {
        drop_page(p, t.back());
        t.pop_back();
    }
    p->len[seq] = rows;
}
static void more_pages(pf_pages* p, uint32_t seq, size_t n) {
    std::vector<uint32_t>& t = p->pages[seq];
    if (t.capacity() < n) t.reserve(std::max(n, 2 * t.capacity()));
}
// The device's tables learn of changes with the next pass, or the next call that
// reads them, or when there are many.  (Room for `n` more before anything
// changes.)
constexpr size_t DIRTY_MOST = 1 << 16;
static pf_status more_changes(pf_pages* p, size_t n) {
    if (p->dirty.size() > DIRTY_MOST)
        if (pf_status st = tables_to_device(p)) return st;
    if (p->dirty.capacity() - p->dirty.size() < n) p->dirty.reserve(std::max(p->dirty.size() + n, 2 * p->dirty.capacity()));
    return PF_OK;
}
static void change(pf_pages* p, uint32_t seq, uint32_t at) { p->dirty.push_back(seq * p->per_seq + at); }

// In range and named once.
static pf_status distinct(pf_pages* p, const uint32_t* seqs, uint32_t n) {
    if (n && !seqs) return fail(p->ctx, PF_ERR_ARG, "pages: a list is NULL");
    if (++p->stamp == 0) {
        std::fill(p->mark.begin(), p->mark.end(), 0u);
        p->stamp = 1;
    }
    for (uint32_t i = 0; i < n; i++) {
        if (seqs[i] >= p->cfg.max_seqs) return fail(p->ctx, PF_ERR_ARG, "pages: sequence out of range");
        if (p->mark[seqs[i]] == p->stamp) return fail(p->ctx, PF_ERR_ARG, "pages: a sequence is named twice");
        p->mark[seqs[i]] = p->stamp;
    }
    return PF_OK;
}
static pf_status all_empty(pf_pages* p, const uint32_t* seqs, uint32_t n) {
    if (pf_status st = distinct(p, seqs, n)) return st;
    for (uint32_t i = 0; i < n; i++)
        if (p->len[seqs[i]]) return fail(p->ctx, PF_ERR_STATE, "pages: a sequence to fill is not empty");
    return PF_OK;
}
static void end_pass(pf_pages* p) { p->open = false; }

static bool cache_type(int32_t t) {
    return t == PF_TYPE_F16 || t == PF_TYPE_BF16 || t == PF_TYPE_I8 || t == PF_TYPE_FP4;
}

static pf_status pages_alloc(pf_pages* p) {
    pf_ctx* c = p->ctx;
    const pf_pages_config& g = p->cfg;
    p->refs.assign(g.n_pages, 0);
    p->len.assign(g.max_seqs, 0);
    p->mark.assign(g.max_seqs, 0);
    p->pages.resize(g.max_seqs);
    p->pass.reserve(g.max_seqs);
    p->heap.resize(g.n_pages);
    for (uint32_t i = 0; i < g.n_pages; i++) p->heap[i] = i;   // ascending: a heap
    p->staging = new PageStaging();
    const size_t pool = p->plane * g.n_layers, sc = p->scales * g.n_layers;
    pf_status s = dalloc(c, &p->k, pool);
    if (!s) s = dalloc(c, &p->v, pool);
    if (!s && sc) s = dalloc(c, &p->ks, sc);
    if (!s && sc) s = dalloc(c, &p->vs, sc);
    if (!s) s = dalloc_t(c, &p->table, (size_t)g.max_seqs * p->per_seq);
    if (!s) s = dalloc_t(c, &p->seqs, g.max_seqs);
    if (!s) s = dalloc_t(c, &p->items, p->items_cap);
    if (!s) s = dalloc_t(c, &p->pairs, 3 * MOVE_MOST);
    if (s) return s;
    p->bytes = 2 * pool + 2 * sc + (size_t)g.max_seqs * p->per_seq * 4;
    PF_HIP(c, hipHostMalloc((void**)&p->staging->mem, STAGE_BYTES * STAGE_SLOTS, hipHostMallocDefault));
    for (hipEvent_t& e : p->staging->done) PF_HIP(c, hipEventCreateWithFlags(&e, hipEventDisableTiming));
    return PF_OK;
}

extern "C" void pf_pages_destroy(pf_pages* p) {
    if (!p) return;
    pf_ctx* c = p->ctx;
    DeviceScope on(c);
    (void)hipStreamSynchronize(c->stream);
    const pf_pages_config& g = p->cfg;
    const size_t pool = p->plane * g.n_layers, sc = p->scales * g.n_layers;
    dfree(c, p->k, pool);
    dfree(c, p->v, pool);
    dfree(c, p->ks, sc);
    dfree(c, p->vs, sc);
    dfree(c, p->table, (size_t)g.max_seqs * p->per_seq * 4);
    dfree(c, p->seqs, g.max_seqs * sizeof(PageSeq));
    dfree(c, p->items, p->items_cap * sizeof(PageItem));
    dfree(c, p->pairs, 3 * MOVE_MOST * 4);
    if (p->staging) {
        for (hipEvent_t e : p->staging->done)
            if (e) (void)hipEventDestroy(e);
        if (p->staging->mem) (void)hipHostFree(p->staging->mem);
        delete p->staging;
    }
    delete p;
}

extern "C" pf_status pf_pages_create(pf_ctx* c, const pf_pages_config* g, pf_pages** out) {
    if (!c || !g || !out) return PF_ERR_ARG;
    *out = nullptr;
    if (!cache_type(g->type)) return fail(c, PF_ERR_ARG, "pages: type is PF_TYPE_F16, BF16, I8 or FP4");
    if (!g->n_layers || !g->n_kv_heads || !g->n_pages || !g->max_seqs || !g->max_context)
        return fail(c, PF_ERR_ARG, "pages: a size is 0");
    if (g->n_layers > 65535 || g->n_kv_heads > 65535) return fail(c, PF_ERR_UNSUPPORTED, "pages: over 65535 layers or heads");
    if (!g->head_dim || g->head_dim % 16 || g->head_dim > 128)
        return fail(c, PF_ERR_UNSUPPORTED, "pages: head_dim is a multiple of 16 up to 128");
    if (g->page_size < 16 || g->page_size > 256 || (g->page_size & (g->page_size - 1)))
        return fail(c, PF_ERR_UNSUPPORTED, "pages: page_size is 16, 32, 64, 128 or 256");
    if (g->max_context > SEQ_ROWS || g->n_pages > 0x7FFFFFFFu)
        return fail(c, PF_ERR_UNSUPPORTED, "pages: max_context up to 2^30, n_pages below 2^31");
    const uint32_t per_seq = (g->max_context + g->page_size - 1) / g->page_size;
    if ((uint64_t)per_seq * g->max_seqs > 0xFFFFFFFFull)
        return fail(c, PF_ERR_UNSUPPORTED, "pages: max_seqs times the pages of max_context is 2^32 at most");
    const bool fp4 = g->type == PF_TYPE_FP4, i8 = g->type == PF_TYPE_I8;
    const uint32_t row_bytes = fp4 ? 16 * fp4_blocks(g->head_dim) : g->head_dim * (i8 ? 1 : 2);
    const size_t rows = (size_t)g->n_pages * g->n_kv_heads * g->page_size;
    const size_t plane = rows * row_bytes;                       // (below 2^63 within the limits above)
    if (plane > (SIZE_MAX >> 2) / g->n_layers) return fail(c, PF_ERR_UNSUPPORTED, "pages: a pool of over 2^62 bytes");
    DeviceScope on(c);
    pf_pages* p = new (std::nothrow) pf_pages();
    if (!p) return fail(c, PF_ERR_CAPACITY, "out of host memory");
    p->ctx = c;
    p->cfg = *g;
    p->shift = (uint32_t)__builtin_ctz(g->page_size);
    p->per_seq = per_seq;
    p->row_bytes = row_bytes;
    p->scale_bytes = fp4 ? fp4_blocks(g->head_dim) : i8 ? 4 : 0;
    p->scales = rows * p->scale_bytes;
    p->plane = plane;
    p->items_cap = (size_t)2 * g->max_seqs + PG_MOST_ITEMS;
    if (pf_status s = no_throw(c, [&] { return pages_alloc(p); })) {
        const std::string msg = c->err;
        pf_pages_destroy(p);
        return fail(c, s, msg);
    }
    *out = p;
    return PF_OK;
}

extern "C" size_t pf_pages_memory_usage(const pf_pages* p) { return p ? p->bytes : 0; }
extern "C" uint32_t pf_pages_free_count(const pf_pages* p) { return p ? (uint32_t)p->heap.size() : 0; }
extern "C" uint32_t pf_pages_length(const pf_pages* p, uint32_t seq) {
    return p && seq < p->cfg.max_seqs ? p->len[seq] : 0;
}

extern "C" pf_status pf_pages_tables(const pf_pages* p, const uint32_t* seqs, uint32_t n, int64_t* pages, uint32_t cap,
                                     int64_t* lengths) {
    if (!p || (n && !seqs)) return PF_ERR_ARG;
    for (uint32_t i = 0; i < n; i++) {
        if (seqs[i] >= p->cfg.max_seqs) return fail(p->ctx, PF_ERR_ARG, "pages: sequence out of range");
        if (pages && p->pages[seqs[i]].size() > cap) return fail(p->ctx, PF_ERR_CAPACITY, "pages: a sequence has more pages");
    }
    for (uint32_t i = 0; i < n; i++) {
        const std::vector<uint32_t>& t = p->pages[seqs[i]];
        if (pages)
            for (uint32_t j = 0; j < cap; j++) pages[(size_t)i * cap + j] = j < t.size() ? (int64_t)t[j] : -1;
        if (lengths) lengths[i] = p->len[seqs[i]];
    }
    return PF_OK;
}

extern "C" pf_status pf_pages_planes(const pf_pages* p, void** k, void** v, float** ks, float** vs) {
    if (!p || !k || !v || !ks || !vs) return PF_ERR_ARG;
    *k = p->k; *v = p->v; *ks = (float*)p->ks; *vs = (float*)p->vs;
    return PF_OK;
}

// ================================================================== passes

static pf_status pages_append(pf_pages* p, const uint32_t* seqs, const uint32_t* rows, uint32_t n) {
    pf_ctx* c = p->ctx;
    if (n && !rows) return fail(c, PF_ERR_ARG, "pages: a list is NULL");
    if (pf_status st = distinct(p, seqs, n)) return st;
    // pages needed: a shared last page is copied by all of its sequences that
    // grow, but for the last one where no other keeps it
    uint64_t need = 0, total = 0;
    for (uint32_t i = 0; i < n; i++) {
        if (rows[i] > p->cfg.max_context - p->len[seqs[i]])
            return fail(c, PF_ERR_CAPACITY, "pages: a sequence would exceed max_context");
        total += rows[i];
    }
    std::vector<uint32_t> leaving;
    leaving.reserve(n);
    for (uint32_t i = 0; i < n; i++) {
        const uint32_t have = p->len[seqs[i]];
        if (!rows[i]) continue;
        need += pages_for(p, have + rows[i]) - p->pages[seqs[i]].size();
        if (have & (p->cfg.page_size - 1)) {
            const uint32_t last = p->pages[seqs[i]].back();
            if (p->refs[last] > 1) {
                p->refs[last]--;
                leaving.push_back(last);
                need++;
            }
        }
    }
    for (uint32_t page : leaving) p->refs[page]++;
    const size_t copies = leaving.size();
    if (need > p->heap.size()) return fail(c, PF_ERR_CAPACITY, "pages: too few free pages");
    if (total > 0x7FFFFFFFu) return fail(c, PF_ERR_UNSUPPORTED, "pages: over 2^31 rows in one pass");

    DeviceScope on(c);
    // (all host memory that the changes need first)
    std::vector<uint32_t> moves;
    if (pf_status st = more_changes(p, need)) return st;
    moves.reserve(3 * copies);
    for (uint32_t i = 0; i < n; i++) more_pages(p, seqs[i], pages_for(p, p->len[seqs[i]] + rows[i]));
    p->pass.clear();
    uint32_t q0 = 0, uniform = n ? rows[0] : 0;
    for (uint32_t i = 0; i < n; i++) {
        const uint32_t s = seqs[i], have = p->len[s];
        std::vector<uint32_t>& t = p->pages[s];
        const uint32_t used = have & (p->cfg.page_size - 1);
        if (rows[i] && used && p->refs[t.back()] > 1) {
            const uint32_t old = t.back();
            t.back() = take_page(p);
            p->refs[old]--;
            moves.insert(moves.end(), {old, t.back(), used});
            change(p, s, (uint32_t)t.size() - 1);
        }
        while (t.size() < pages_for(p, have + rows[i])) {
            t.push_back(take_page(p));
            change(p, s, (uint32_t)t.size() - 1);
        }
        p->len[s] = have + rows[i];
        p->pass.push_back({s, q0, rows[i], p->len[s]});
        q0 += rows[i];
        if (rows[i] != uniform) uniform = 0;
    }
    p->pass_rows = q0;
    p->uniform = uniform;
    p->cut = PageSplit();
    p->open = false;
    bool moved;
    if (pf_status st = stage_all(p, p->seqs, p->pass.data(), p->pass.size() * sizeof(PageSeq), p->dirty, moves, &moved)) return st;
    p->dirty.clear();
    if (!moved)
        if (pf_status st = move_pages(p, moves)) return st;
    p->open = true;
    return PF_OK;
}
extern "C" pf_status pf_pages_append(pf_pages* p, const uint32_t* seqs, const uint32_t* rows, uint32_t n) {
    if (!p) return PF_ERR_ARG;
    return no_throw(p->ctx, [&] { return pages_append(p, seqs, rows, n); });
}

static pf_status rows_check(pf_pages* p, uint32_t layer, int32_t type, const void* k, const void* v, uint32_t* kst,
                            uint32_t* vst) {
    pf_ctx* c = p->ctx;
    if (layer >= p->cfg.n_layers) return fail(c, PF_ERR_ARG, "pages: layer out of range");
    if (type != PF_TYPE_F32 && type != PF_TYPE_F16 && type != PF_TYPE_BF16)
        return fail(c, PF_ERR_ARG, "pages: rows are PF_TYPE_F32, F16 or BF16");
    const uint64_t least = (uint64_t)p->cfg.n_kv_heads * p->cfg.head_dim;
    const uint32_t per16 = type == PF_TYPE_F32 ? 4 : 8;
    for (uint32_t* s : {kst, vst}) {
        const uint64_t w = *s ? *s : least;
        if (w < least || w > 0xFFFFFFFFu || w % per16)
            return fail(c, PF_ERR_ARG, "pages: strides hold every head and are multiples of 16 bytes");
        *s = (uint32_t)w;
    }
    if (!aligned16(k) || !aligned16(v)) return fail(c, PF_ERR_ARG, "pages: buffers start on 16 bytes");
    return PF_OK;
}

// One launch's workgroups: a grid dimension holds fewer than 2^32 threads.
constexpr uint64_t STORE_BLOCKS = 1u << 23;
template <int CT>
static void store_type(hipStream_t st, int32_t type, uint32_t blocks, const StoreArgs& a) {
    if (type == PF_TYPE_F32) hipLaunchKernelGGL((k_pages_store<PF_TYPE_F32, CT>), dim3(blocks), dim3(256), 0, st, a);
    else if (type == PF_TYPE_F16) hipLaunchKernelGGL((k_pages_store<PF_TYPE_F16, CT>), dim3(blocks), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_pages_store<PF_TYPE_BF16, CT>), dim3(blocks), dim3(256), 0, st, a);
}
template <int CT>
static void gather_type(hipStream_t st, int32_t type, uint32_t blocks, const GatherArgs& a) {
    if (type == PF_TYPE_F32) hipLaunchKernelGGL((k_pages_gather<PF_TYPE_F32, CT>), dim3(blocks), dim3(256), 0, st, a);
    else if (type == PF_TYPE_F16) hipLaunchKernelGGL((k_pages_gather<PF_TYPE_F16, CT>), dim3(blocks), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_pages_gather<PF_TYPE_BF16, CT>), dim3(blocks), dim3(256), 0, st, a);
}

extern "C" pf_status pf_pages_store(pf_pages* p, uint32_t layer, int32_t type, const void* k, const void* v,
                                    uint32_t kst, uint32_t vst) {
    if (!p) return PF_ERR_ARG;
    pf_ctx* c = p->ctx;
    if (pf_status st = rows_check(p, layer, type, k, v, &kst, &vst)) return st;
    if (!p->open) return fail(c, PF_ERR_STATE, "pages: no open pass (pf_pages_append begins one)");
    if (!p->pass_rows) return PF_OK;
    if (!k || !v) return fail(c, PF_ERR_ARG, "pages: a buffer is NULL");
    const uint64_t waves = (uint64_t)p->pass_rows * ((p->cfg.n_kv_heads + 3) / 4);
    if ((waves + 3) / 4 > STORE_BLOCKS) return fail(c, PF_ERR_UNSUPPORTED, "pages: too many rows in one pass; cut it");
    DeviceScope on(c);
    StoreArgs a{};
    a.seqs = p->seqs; a.table = p->table; a.k = k; a.v = v;
    a.pk = (uint8_t*)p->k + layer * p->plane; a.pv = (uint8_t*)p->v + layer * p->plane;
    a.ks = (uint8_t*)p->ks + layer * p->scales; a.vs = (uint8_t*)p->vs + layer * p->scales;
    a.n_seq = (uint32_t)p->pass.size(); a.rows = p->pass_rows; a.uniform = p->uniform; a.per_seq = p->per_seq;
    a.shift = p->shift; a.kv_heads = p->cfg.n_kv_heads; a.dim = p->cfg.head_dim; a.kstride = kst; a.vstride = vst;
    const uint32_t blocks = (uint32_t)((waves + 3) / 4);
    if (p->cfg.type == PF_TYPE_FP4) store_type<PF_TYPE_FP4>(c->stream, type, blocks, a);
    else if (p->cfg.type == PF_TYPE_I8) store_type<PF_TYPE_I8>(c->stream, type, blocks, a);
    else if (p->cfg.type == PF_TYPE_F16) store_type<PF_TYPE_F16>(c->stream, type, blocks, a);
    else store_type<PF_TYPE_BF16>(c->stream, type, blocks, a);
    PF_LAUNCHED(c);
    return PF_OK;
}

extern "C" pf_status pf_pages_gather(pf_pages* p, uint32_t layer, const uint32_t* seqs, uint32_t n, int32_t type, void* k,
                                     void* v, uint32_t kst, uint32_t vst) {
    if (!p) return PF_ERR_ARG;
    pf_ctx* c = p->ctx;
    if (pf_status st = rows_check(p, layer, type, k, v, &kst, &vst)) return st;
    if (n && !seqs) return fail(c, PF_ERR_ARG, "pages: a list is NULL");
    uint64_t total = 0;
    for (uint32_t i = 0; i < n; i++) {
        if (seqs[i] >= p->cfg.max_seqs) return fail(c, PF_ERR_ARG, "pages: sequence out of range");
        total += p->len[seqs[i]];
    }
    if (!total) return PF_OK;
    if (!k || !v) return fail(c, PF_ERR_ARG, "pages: a buffer is NULL");
    const uint32_t heads4 = (p->cfg.n_kv_heads + 3) / 4;
    if ((total * heads4 + 3) / 4 > STORE_BLOCKS || total > 0x7FFFFFFFu)
        return fail(c, PF_ERR_UNSUPPORTED, "pages: too many rows at once");
    const size_t es = type == PF_TYPE_F32 ? 4 : 2, w = (size_t)p->cfg.n_kv_heads * p->cfg.head_dim;
    if (overlaps(k, ((total - 1) * kst + w) * es, v, ((total - 1) * vst + w) * es)) {
        // rows of both may alternate in one buffer
        const size_t a = (uintptr_t)k, b = (uintptr_t)v, off = (b > a ? b - a : a - b) % (kst * es);
        if (kst != vst || off < w * es || off > (kst - w) * es) return fail(c, PF_ERR_ARG, "pages: k and v overlap");
    }
    DeviceScope on(c);
    if (pf_status st = no_throw(c, [&] { return tables_to_device(p); })) return st;
    GatherArgs a{};
    a.table = p->table; a.k = k; a.v = v;
    a.pk = (const uint8_t*)p->k + layer * p->plane; a.pv = (const uint8_t*)p->v + layer * p->plane;
    a.ks = (const uint8_t*)p->ks + layer * p->scales; a.vs = (const uint8_t*)p->vs + layer * p->scales;
    a.per_seq = p->per_seq; a.shift = p->shift; a.kv_heads = p->cfg.n_kv_heads; a.dim = p->cfg.head_dim;
    a.kstride = kst; a.vstride = vst;
    uint32_t row0 = 0;
    for (uint32_t i = 0; i < n;) {
        a.n_seq = a.rows = 0;
        a.row0 = row0;
        for (; i < n && a.n_seq < GATHER_SEQS; i++) {
            if (!p->len[seqs[i]]) continue;
            a.first[a.n_seq] = a.rows;
            a.slot[a.n_seq++] = seqs[i];
            a.rows += p->len[seqs[i]];
        }
        if (!a.rows) break;
        row0 += a.rows;
        const uint32_t blocks = (uint32_t)(((uint64_t)a.rows * heads4 + 3) / 4);
        if (p->cfg.type == PF_TYPE_FP4) gather_type<PF_TYPE_FP4>(c->stream, type, blocks, a);
        else if (p->cfg.type == PF_TYPE_I8) gather_type<PF_TYPE_I8>(c->stream, type, blocks, a);
        else if (p->cfg.type == PF_TYPE_F16) gather_type<PF_TYPE_F16>(c->stream, type, blocks, a);
        else gather_type<PF_TYPE_BF16>(c->stream, type, blocks, a);
        PF_LAUNCHED(c);
    }
    return PF_OK;
}

// ============================================== fork, copy, free, compact

static pf_status pages_fork(pf_pages* p, uint32_t src, const uint32_t* dst, uint32_t n) {
    if (src >= p->cfg.max_seqs) return fail(p->ctx, PF_ERR_ARG, "pages: sequence out of range");
    if (pf_status st = all_empty(p, dst, n)) return st;
    DeviceScope on(p->ctx);
    if (pf_status st = more_changes(p, (size_t)n * p->pages[src].size())) return st;
    for (uint32_t i = 0; i < n; i++) more_pages(p, dst[i], p->pages[src].size());
    end_pass(p);
    for (uint32_t i = 0; i < n; i++) {
        p->pages[dst[i]] = p->pages[src];
        p->len[dst[i]] = p->len[src];
        for (uint32_t j = 0; j < p->pages[src].size(); j++) {
            p->refs[p->pages[src][j]]++;
            change(p, dst[i], j);
        }
    }
    return PF_OK;
}
extern "C" pf_status pf_pages_fork(pf_pages* p, uint32_t src, const uint32_t* dst, uint32_t n) {
    if (!p) return PF_ERR_ARG;
    return no_throw(p->ctx, [&] { return pages_fork(p, src, dst, n); });
}

static pf_status pages_copy(pf_pages* p, const uint32_t* src, const uint32_t* dst, uint32_t n) {
    if (n && !src) return fail(p->ctx, PF_ERR_ARG, "pages: a list is NULL");
    if (pf_status st = all_empty(p, dst, n)) return st;
    uint64_t need = 0;
    for (uint32_t i = 0; i < n; i++) {
        if (src[i] >= p->cfg.max_seqs) return fail(p->ctx, PF_ERR_ARG, "pages: sequence out of range");
        if (p->mark[src[i]] != p->stamp) need += p->pages[src[i]].size();
    }
    if (need > p->heap.size()) return fail(p->ctx, PF_ERR_CAPACITY, "pages: too few free pages");
    DeviceScope on(p->ctx);
    std::vector<uint32_t> moves;
    if (pf_status st = more_changes(p, need)) return st;
    moves.reserve(3 * need);
    for (uint32_t i = 0; i < n; i++) more_pages(p, dst[i], p->pages[src[i]].size());
    end_pass(p);
    for (uint32_t i = 0; i < n; i++) {
        if (p->mark[src[i]] == p->stamp) continue;           // one of the empty ones
        const std::vector<uint32_t>& from = p->pages[src[i]];
        for (uint32_t j = 0; j < from.size(); j++) {
            const uint32_t page = take_page(p);
            p->pages[dst[i]].push_back(page);
            moves.insert(moves.end(), {from[j], page, p->cfg.page_size});
            change(p, dst[i], j);
        }
        p->len[dst[i]] = p->len[src[i]];
    }
    return move_pages(p, moves);
}
extern "C" pf_status pf_pages_copy(pf_pages* p, const uint32_t* src, const uint32_t* dst, uint32_t n) {
    if (!p) return PF_ERR_ARG;
    return no_throw(p->ctx, [&] { return pages_copy(p, src, dst, n); });
}

static pf_status pages_truncate(pf_pages* p, const uint32_t* seqs, const uint32_t* lengths, uint32_t n) {
    if (n && !lengths) return fail(p->ctx, PF_ERR_ARG, "pages: a list is NULL");
    if (pf_status st = distinct(p, seqs, n)) return st;
    for (uint32_t i = 0; i < n; i++)
        if (lengths[i] > p->len[seqs[i]]) return fail(p->ctx, PF_ERR_ARG, "pages: a sequence is shorter than that");
    end_pass(p);
    for (uint32_t i = 0; i < n; i++) cut_pages(p, seqs[i], lengths[i]);
    return PF_OK;
}
extern "C" pf_status pf_pages_truncate(pf_pages* p, const uint32_t* seqs, const uint32_t* lengths, uint32_t n) {
    if (!p) return PF_ERR_ARG;
    return no_throw(p->ctx, [&] { return pages_truncate(p, seqs, lengths, n); });
}

static pf_status pages_free(pf_pages* p, const uint32_t* seqs, uint32_t n) {
    if (pf_status st = distinct(p, seqs, n)) return st;
    end_pass(p);
    for (uint32_t i = 0; i < n; i++) cut_pages(p, seqs[i], 0);
    return PF_OK;
}
extern "C" pf_status pf_pages_free(pf_pages* p, const uint32_t* seqs, uint32_t n) {
    if (!p) return PF_ERR_ARG;
    return no_throw(p->ctx, [&] { return pages_free(p, seqs, n); });
}

static pf_status pages_compact(pf_pages* p, uint32_t* moved) {
    if (moved) *moved = 0;
    const uint32_t used = p->cfg.n_pages - (uint32_t)p->heap.size();
    // old and new number of the pages that move, then the tables that name them
    std::vector<uint32_t> moves, to(p->cfg.n_pages - used);
    uint32_t hole = 0;
    for (uint32_t page = used; page < p->cfg.n_pages; page++) {
        if (!p->refs[page]) continue;
        while (p->refs[hole]) hole++;
        moves.insert(moves.end(), {page, hole, p->cfg.page_size});
        to[page - used] = hole++;
    }
    size_t named = 0;
    for (const std::vector<uint32_t>& t : p->pages)
        for (uint32_t page : t) named += page >= used;
    DeviceScope on(p->ctx);
    if (pf_status st = more_changes(p, named)) return st;
    end_pass(p);
    if (moves.empty()) return PF_OK;
    for (uint32_t s = 0; s < p->cfg.max_seqs; s++)
        for (uint32_t j = 0; j < p->pages[s].size(); j++)
            if (p->pages[s][j] >= used) {
                p->pages[s][j] = to[p->pages[s][j] - used];
                change(p, s, j);
            }
    for (size_t i = 0; i < moves.size(); i += 3) std::swap(p->refs[moves[i]], p->refs[moves[i + 1]]);
    for (uint32_t i = 0; i < p->heap.size(); i++) p->heap[i] = used + i;
    if (moved) *moved = (uint32_t)(moves.size() / 3);
    return move_pages(p, moves);
}
extern "C" pf_status pf_pages_compact(pf_pages* p, uint32_t* moved) {
    if (!p) return PF_ERR_ARG;
    return no_throw(p->ctx, [&] { return pages_compact(p, moved); });
}
