// The library's context and what every translation unit of the host runtime
// shares: error text, HIP checks, counted device memory, the context's scratch.
#pragma once
#include <hip/hip_runtime.h>

#include <algorithm>
#include <new>
#include <string>

#include "../../include/pf_gpu.h"

struct pf_ctx {
    int device = 0;
    hipStream_t stream = nullptr;
    std::string err;
    size_t bytes = 0;
    // growable scratch for the kernel-level entry points
    void* scratch = nullptr;
    size_t scratch_bytes = 0;
};

[[maybe_unused]] static pf_status fail(const pf_ctx* c, pf_status s, const std::string& msg) {
    if (c) const_cast<pf_ctx*>(c)->err = msg;
    return s;
}

#define PF_HIP(ctx, call)                                                                        \
    do {                                                                                         \
        hipError_t e_ = (call);                                                                  \
        if (e_ != hipSuccess)                                                                    \
            return fail(ctx, PF_ERR_HIP, std::string(#call) + " failed: " + hipGetErrorString(e_)); \
    } while (0)

#define PF_LAUNCHED(ctx) PF_HIP(ctx, hipGetLastError())

[[maybe_unused]] static pf_status dalloc(pf_ctx* c, void** p, size_t bytes) {
    *p = nullptr;
    if (bytes == 0) bytes = 256;
    hipError_t e = hipMalloc(p, bytes);
    if (e != hipSuccess) {
        (void)hipGetLastError();   // (else the next launch's check would report it)
        return fail(c, PF_ERR_HIP, "hipMalloc(" + std::to_string(bytes) + ") failed: " + hipGetErrorString(e));
    }
    c->bytes += bytes;
    return PF_OK;
}

[[maybe_unused]] static void dfree(pf_ctx* c, void* p, size_t bytes) {
    if (!p) return;
    (void)hipFree(p);
    if (bytes == 0) bytes = 256;
    c->bytes -= std::min(c->bytes, bytes);
}

template <class T>
[[maybe_unused]] static pf_status dalloc_t(pf_ctx* c, T** p, size_t n) {
    return dalloc(c, reinterpret_cast<void**>(p), n * sizeof(T));
}

[[maybe_unused]] static pf_status ctx_scratch(pf_ctx* c, size_t bytes, void** out) {
    if (bytes > c->scratch_bytes) {
        if (c->scratch) {
            PF_HIP(c, hipStreamSynchronize(c->stream));
            dfree(c, c->scratch, c->scratch_bytes);
            c->scratch = nullptr;
            c->scratch_bytes = 0;
        }
        pf_status s = dalloc(c, &c->scratch, bytes);
        if (s) return s;
        c->scratch_bytes = bytes;
    }
    *out = c->scratch;
    return PF_OK;
}

// Runs the body of an entry point: no C++ exception leaves it.
template <class F>
static pf_status no_throw(const pf_ctx* c, F&& body) {
    try {
        return body();
    } catch (const std::bad_alloc&) {
        return fail(c, PF_ERR_CAPACITY, "out of host memory");
    } catch (const std::exception& e) {
        return fail(c, PF_ERR_HIP, e.what());
    }
}

// Makes the context's device current for a call, and the caller's again after it.
struct DeviceScope {
    int before = -1;
    explicit DeviceScope(const pf_ctx* c) {
        int d = -1;
        if (hipGetDevice(&d) == hipSuccess && d != c->device && hipSetDevice(c->device) == hipSuccess) before = d;
    }
    ~DeviceScope() {
        if (before >= 0) (void)hipSetDevice(before);
    }
    DeviceScope(const DeviceScope&) = delete;
    DeviceScope& operator=(const DeviceScope&) = delete;
};

[[maybe_unused]] static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

[[maybe_unused]] static bool overlaps(const void* a, size_t na, const void* b, size_t nb) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return x < y + nb && y < x + na;
}

// Whether rows of `width` bytes, `n` of them `sa` and `sb` bytes apart, share memory
// (columns of one buffer's rows do not).
[[maybe_unused]] static bool rows_overlap(const void* a, size_t sa, const void* b, size_t sb, size_t wa, size_t wb, size_t n) {
    if (!n || !overlaps(a, (n - 1) * sa + wa, b, (n - 1) * sb + wb)) return false;
    if (sa != sb || n == 1) return true;
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    const size_t off = x < y ? (y - x) % sa : (sa - (x - y) % sa) % sa;   // of b's columns behind a's
    return off < wa || off + wb > sa;
}

// A pf_attn_desc's checked values (pf_prompt.hip).
constexpr uint32_t SEQ_ROWS = 1u << 30;   // of one sequence
struct AttnShape {
    uint32_t qs, ks, vs, os;   // row strides in elements
    uint32_t window, sink;
    float scale_log2;          // scores to base 2
};
pf_status attn_desc_check(pf_ctx* c, const pf_attn_desc* d, AttnShape* s);

// Which kernels a call takes, for tests that cover each of them (host only; not
// part of the library's interface).  Prompts: query rows of a workgroup, parts of
// the keys.  Pages (a pass of `rows` new rows of sequences of `lens`): waves of a
// workgroup, key tiles of a share and of the longest sequence; `_of` pages of a
// type, and also how many workgroups of 4 waves share a compute unit.
extern "C" pf_status pf_test_prompt_plan(const pf_attn_desc* d, const uint32_t* q_lens, const uint32_t* k_lens,
                                         uint32_t n_seq, uint32_t* rows, uint32_t* parts);
extern "C" pf_status pf_test_pages_plan_of(const pf_attn_desc* d, int32_t cache, const uint32_t* rows, const uint32_t* lens,
                                           uint32_t n, uint32_t* waves, uint32_t* chunk, uint32_t* longest, uint32_t* held);
extern "C" pf_status pf_test_pages_plan(const pf_attn_desc* d, const uint32_t* rows, const uint32_t* lens, uint32_t n,
                                        uint32_t* waves, uint32_t* chunk, uint32_t* longest);
