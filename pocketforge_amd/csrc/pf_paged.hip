// Attention of a pass's rows over their sequences' pages (pf_pages_attention of
// include/pf_gpu.h): one new token per sequence, a verify pass's few, or more.
//
// The mathematics is that of pf_prompt.hip.  A workgroup takes one kv head and
// a share of one sequence's keys; where there are few sequences the keys are
// shared among many workgroups, whose partial results (running maximum m, sum
// l, unnormalised output o) are joined:
//   M = max_p m_p,  out = sum_p 2^(m_p - M) o_p / sum_p 2^(m_p - M) l_p.
#include "pf_paged.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

using namespace pf;

namespace pf {

// Waves of a SIMD (workgroups of a compute unit) that the registers allow: the
// next tile's rows wait in registers, and fp32 rows take three operands each.
__host__ __device__ constexpr int paged_waves(int act, int ct, int dp, int nt) {
    const bool wide = act == PF_TYPE_F32;
    if (ct == PF_TYPE_FP4 && dp == 128 && nt == 1) return 3;
    return dp == 64 ? (nt == 1 ? (wide ? 3 : 4) : 2) : nt == 1 ? 2 : wide ? 1 : 2;
}

// A workgroup: W waves (4 or 8), each on 32-key tiles of its own.
// A lane's matrix operands of K are 16 bytes of a row as the page holds them,
// straight from memory; V's rows go through LDS, which transposes them.  The
// rows of all query heads of the kv head are the columns of the score tile
// S^T = K Q^T, 16 at a time (NT tiles); exp(S)^T is the operand of O^T = V^T P^T
// without moving a value between lanes.
//
// Each key and value row is read once, and with many sequences these bytes bound
// it: 64 contexts of 2000 to 8000 bf16 keys, 16 heads of 128 over 4, one row:
// 657 MB in 122 us, 5.4 TB/s (a large copy: 5.1).  Contexts of 60000 and 32000
// fp16 keys, 16 heads over 2, in 241 shares: 94 MB in 18 us and the join's 6.
// 16 verify passes of five fp32 rows over 500 to 2100 int8 keys, 16 heads of
// 128: 94 MB in 24 us; one round of workgroups with up to 9 tiles a wave, each a memory
// round trip, the codes' way to bf16 and three products per piece of the rows.
// One context of 700 keys: 5.8 us and the join's 3.5, both latency.
//
// 4-bit rows are a quarter of the bytes for the same products, after conversions of
// two codes an instruction: 64 contexts of 4100 to 16000 keys, 16 heads of 128 over
// 4: 349 MB in 73 us, 4.8 TB/s, vector units issuing 53% of the time, matrix units busy
// 26%; the 16 verify passes: 50 MB in 19 us, nine tiles a wave one after another.
template <int ACT, int CT, int DP, int NT, bool EXACT, int W>
__global__ __launch_bounds__(64 * W, paged_waves(ACT, CT, DP, NT)) void k_paged_attn(PagedArgs a) {
    // Weights over int8 rows take the rows' scales, whose range fp16 does not
    // have, so their products with the codes are in bf16 for fp16 rows too.  4-bit
    // values are bf16 (with their scales: fp16 has not their range either), and
    // fp16 query rows two bf16 pieces beside them, which hold all of a value.
    constexpr bool I8 = CT == PF_TYPE_I8, F4 = CT == PF_TYPE_FP4, BF = F4 || op_bf<ACT>, VB = I8 || BF;
    constexpr int NP = F4 && ACT == PF_TYPE_F16 ? 2 : op_pieces<ACT>, PP = weight_pieces<ACT>, C = DP / 32, DT = DP / 16;
    constexpr int STR = DP + 16;                 // LDS row stride in values
    constexpr int CB = F4 && DP == 64 ? 8 : 16;  // bytes of a chunk: 4 bits, a quarter of a row
    constexpr int VCH = F4 ? 4 : I8 ? DP / 16 : DP / 8;   // chunks of a V row
    constexpr int VL = 32 * VCH / 64;            // V loads of a lane
    constexpr int KL = F4 ? 1 : I8 ? DP / 64 : C;         // K loads of a lane per 16 keys
    typedef std::conditional_t<CB == 8, u2v, u4v> chunk;
    __shared__ __align__(16) short sv[W][32][STR];
    __shared__ float s_ml[W][16][2];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, col = lane & 15, g = lane >> 4;

    const PageItem it = a.items[blockIdx.x];
    const uint32_t head0 = blockIdx.y * a.group;
    const int R = (int)(it.rows * a.group), rt0 = (int)blockIdx.z * 16 * NT;
    if (rt0 >= R) return;
    const int len = (int)it.len, p0 = len - (int)it.rows;
    const PageTiles pt = page_tiles(it.rows, it.len, (uint32_t)a.window, (uint32_t)a.sink);
    const int lo0 = a.window ? max(0, p0 - a.window + 1) : 0;
    const int lo1 = a.window ? max(0, len - a.window) : 0;
    const auto pos_of = [&](int t) { return (t < pt.sinks ? t : t - pt.sinks + pt.first) * 32; };

    // The share's tiles in this wave's order: first those that all rows see whole,
    // wa .. wb - 1, then the others; the waves take them in turn.
    const int t0 = (int)it.t0, t1 = (int)it.t1;
    const int wa = min(max(pt.sinks + (lo1 + 31) / 32 - pt.first, max(t0, pt.sinks)), t1);
    const int wb = min(max(pt.sinks + (a.causal ? p0 + 1 : len) / 32 - pt.first, wa), t1);
    const int n_whole = (wb - wa + W - 1 - wave) / W, n_tiles = n_whole + (t1 - t0 - (wb - wa) + wave) / W;
    const auto tile_of = [&](int n) {
        if (n < n_whole) return wa + wave + W * n;
        const int e = t0 + W - 1 - wave + W * (n - n_whole);      // (the waves in the other order)
        return e < wa ? e : e + wb - wa;
    };

    // Page numbers of this wave's next 32 tiles, two for each: lane 2 n + s has
    // the one of tile n's keys 16 s ..
    const int32_t* table = a.table + (size_t)it.slot * a.table_stride;
    const int last_page = (len - 1) >> a.page_shift, in_page = (1 << a.page_shift) - 1;
    int pages = 0;
    auto look_up = [&](int n) {
        const int at = tile_of(min(n + (lane >> 1), n_tiles - 1));
        pages = table[min((pos_of(at) + 16 * (lane & 1)) >> a.page_shift, last_page)];
    };
    if (n_tiles) look_up(0);

    s8v qf[NT][NP][C];
    int hi[NT], lo[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int r = min(rt0 + n * 16 + col, R - 1), j = r / (int)a.group, h = r - j * (int)a.group;
        hi[n] = a.causal ? p0 + j : len - 1;
        lo[n] = a.window ? p0 + j - a.window + 1 : 0;
        const uint8_t* qp = (const uint8_t*)a.q +
                            ((size_t)(it.q0 + (uint32_t)j) * a.qs + (size_t)(head0 + (uint32_t)h) * a.dim) * act_size<ACT>;
#pragma unroll
        for (int c = 0; c < C; c++) {
            // the dims of K's operand: int8 rows give a lane 16 codes at a time, 4 bits a quarter of a row
            const int d = F4 ? g * (DP / 4) + c * 8 : I8 ? (c >> 1) * 64 + g * 16 + (c & 1) * 8 : c * 32 + g * 8;
            float x[8] = {};
            if (EXACT || d < (int)a.dim) load8<ACT>(qp + (size_t)d * act_size<ACT>, x);
            s8v t[NP];
            pieces<BF, NP>(x, t);
#pragma unroll
            for (int n2 = 0; n2 < NP; n2++) qf[n][n2][c] = t[n2];
        }
    }

    const float above = ACT == PF_TYPE_F32 ? 0.0f : VB ? a.above : FP16_ABOVE;
    f4v o[NT][DT];
    float m[NT], l[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        m[n] = -INFINITY;
        l[n] = 0.0f;
#pragma unroll
        for (int t = 0; t < DT; t++) o[n][t] = (f4v)0.0f;
    }

    const uint32_t blocks = fp4_blocks(EXACT ? DP : a.dim);
    const uint32_t row_bytes = F4 ? blocks * 16 : (EXACT ? DP : a.dim) * (I8 ? 1 : 2);
    const uint32_t k_off = (uint32_t)col * row_bytes + (uint32_t)g * CB;
    const uint32_t v_row = (uint32_t)lane / VCH, v_off = v_row * row_bytes + (uint32_t)lane % VCH * CB;
    constexpr int VR = 64 / VCH;                 // V rows of one load of the wave
    const uint32_t k_block = (uint32_t)g * CB / 16, v_block = (uint32_t)lane % VCH * CB / 16;

    chunk kr[2][KL], vr[VL];
    f4v ksc[2], vsc[2];                          // int8
    uint32_t kex[2], vex[VL];                    // 4 bits: exponents
    auto load = [&](int n) {                     // this wave's n-th tile
        const int pos0 = pos_of(tile_of(n));
#pragma unroll
        for (int s = 0; s < 2; s++) {
            const uint32_t pg = (uint32_t)__builtin_amdgcn_readlane(pages, 2 * (n & 31) + s);
            const size_t row0 = (((size_t)pg * a.kv_heads + blockIdx.y) << a.page_shift) + (size_t)((pos0 + 16 * s) & in_page);
            const uint8_t *kp = (const uint8_t*)a.k + row0 * row_bytes, *vp = (const uint8_t*)a.v + row0 * row_bytes;
#pragma unroll
            for (int c = 0; c < KL; c++)
                kr[s][c] = (EXACT || c * 64 + g * CB < (int)row_bytes) ? *(const chunk*)(kp + k_off + c * 64) : (chunk)0u;
#pragma unroll
            for (int i = 0; i < VL / 2; i++)
                vr[s * (VL / 2) + i] = (EXACT || lane % VCH * CB < (int)row_bytes) ? *(const chunk*)(vp + v_off + i * VR * row_bytes) : (chunk)0u;
            if constexpr (I8) {
                ksc[s] = *(const f4v*)((const uint8_t*)((const float*)a.ks + row0) + 16 * g);
                vsc[s] = *(const f4v*)((const uint8_t*)((const float*)a.vs + row0) + 16 * g);
            }
            if constexpr (F4) {
                kex[s] = EXACT || k_block < blocks ? ((const uint8_t*)a.ks)[(row0 + (uint32_t)col) * blocks + k_block] : 0u;
                vex[s] = EXACT || v_block < blocks ? ((const uint8_t*)a.vs)[(row0 + v_row) * blocks + v_block] : 0u;
            }
        }
    };

    // this wave's n-th tile, already in registers; the next one's loads are under
    // way while its weights are formed.  MASKED: some rows do not see all of it
    auto body = [&](auto masked, int n_tile) {
        const int pos0 = pos_of(tile_of(n_tile));
        constexpr bool MASKED = decltype(masked)::value;
        short* sw = &sv[wave][0][0];
        auto place = [&](int i) { return sw + (i * VR + v_row) * STR + (lane % VCH) * (F4 ? 2 * CB : I8 ? 16 : 8); };
        f4v kscale[2], vscale[2];
        s8v kf[2][C];
#pragma unroll
        for (int s = 0; s < 2; s++) {
            if constexpr (I8) {
                kscale[s] = ksc[s];
                vscale[s] = vsc[s];
#pragma unroll
                for (int c = 0; c < C; c++) {
                    float x[8];
                    codes8(kr[s][c >> 1][(c & 1) * 2], kr[s][c >> 1][(c & 1) * 2 + 1], x);
                    kf[s][c] = pack8<BF>(x);
                }
            } else if constexpr (F4) {
#pragma unroll
                for (int c = 0; c < C; c++) kf[s][c] = fp4_bf16(kr[s][0][c], fp4_scale(kex[s]));
            } else {
#pragma unroll
                for (int c = 0; c < C; c++) kf[s][c] = __builtin_bit_cast(s8v, kr[s][c]);
            }
        }
        f4v sc[NT][2];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int s = 0; s < 2; s++) {
                sc[n][s] = (f4v)0.0f;
#pragma unroll
                for (int c = 0; c < C; c++)
#pragma unroll
                    for (int x = 0; x < NP; x++) sc[n][s] = mfma16<BF>(kf[s][c], qf[n][x][c], sc[n][s]);
            }
        // V's rows to LDS; rows that nobody sees (past the end, between sinks and window) as zeros
        const uint32_t any = !MASKED ? 0u : (uint32_t)(first_bits(len - pos0) & (~first_bits(lo0 - pos0) | first_bits(a.sink - pos0)));
        float z = 0.0f;
#pragma unroll
        for (int i = 0; i < VL; i++) {
            chunk w = vr[i];
            const uint32_t on = MASKED ? (uint32_t)-(int)((any >> (i * VR + v_row)) & 1u) : ~0u;
            if constexpr (MASKED) w &= on;
            if constexpr (I8) {
                float x[8];
                codes8(w[0], w[1], x);
                *(s8v*)place(i) = pack8<VB>(x);
                codes8(w[2], w[3], x);
                *(s8v*)(place(i) + 8) = pack8<VB>(x);
            } else if constexpr (F4) {
                const uint32_t e = MASKED ? vex[i] & on : vex[i];
                if (e == 255) z = NAN;
#pragma unroll
                for (int c = 0; c < CB / 4; c++) *(s8v*)(place(i) + 8 * c) = fp4_bf16(w[c], fp4_scale(e));
            } else {
                z = sum8<BF>(__builtin_bit_cast(s8v, w), z, 0.0f);
                *(u4v*)place(i) = w;
            }
        }
        if (n_tile + 1 < n_tiles) {
            if (((n_tile + 1) & 31) == 0) look_up(n_tile + 1);
            load(n_tile + 1);
        }
        s8v pf[NT][PP];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            uint32_t part = ~0u;                 // one bit per key, from 4 g on
            if constexpr (MASKED)
                part = (uint32_t)(first_bits(hi[n] + 1 - pos0) & (~first_bits(lo[n] - pos0) | first_bits(a.sink - pos0))) >> (4 * g);
            float x[8], top = -INFINITY;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                x[e] = sc[n][e / 4][e % 4] * (I8 ? kscale[e / 4][e % 4] * a.scale_log2 : a.scale_log2);
                if constexpr (MASKED) x[e] = bits_or(x[e], -INFINITY, __builtin_amdgcn_sbfe((int)part, 16 * (e / 4) + e % 4, 1));
                top = fmaxf(top, x[e]);
            }
            if (__any(top > m[n] + (m_slack<VB> - above))) {
                const float to = fmaxf(m[n], max16(top) + above);
                const float f = to == -INFINITY ? 1.0f : exp2_fast(m[n] - to);
                m[n] = to;
                l[n] *= f;
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int i = 0; i < 4; i++) o[n][d][i] *= f;
            }
            const float ms = m[n] == -INFINITY ? 0.0f : m[n];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                x[e] = exp2_fast(x[e] - ms);
                if constexpr (ACT == PF_TYPE_F32) x[e] *= a.down;
                l[n] += x[e];
                if constexpr (I8) {
                    x[e] *= vscale[e / 4][e % 4];
                    if constexpr (MASKED) x[e] = bits_or(x[e], 0.0f, __builtin_amdgcn_sbfe((int)part, 16 * (e / 4) + e % 4, 1));
                }
            }
            pieces<VB, PP>(x, pf[n]);
        }
        __builtin_amdgcn_wave_barrier();
        if constexpr (!I8) {
            if (__any(z != z)) {
                // infinities and NaN reach the rows that see them, whatever their weight,
                // and the products find zeros in their places (a weight's second piece is
                // zero or negative as often as not, which would make a NaN of an infinity;
                // looking every tile through takes 0.3 us of 24 where two contexts are cut)
                for (int r = 0; r < 32; r++)
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        if (MASKED && (pos0 + r >= len || !key_visible(pos0 + r, hi[n], lo[n], a.sink))) continue;
#pragma unroll
                        for (int d = 0; d < DT; d++)
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                const short w = sw[r * STR + d * 16 + 4 * g + i];
                                if (not_finite<BF>(w)) o[n][d][i] += to_float<BF ? PF_TYPE_BF16 : PF_TYPE_F16>(w);
                            }
                    }
                __builtin_amdgcn_wave_barrier();
                for (int i = 0; i < VL; i++)
                    for (int c = 0; c < (F4 ? CB / 4 : 1); c++)
                        *(s8v*)(place(i) + 8 * c) = finite_or_zero<BF>(*(const s8v*)(place(i) + 8 * c));
                __builtin_amdgcn_wave_barrier();
            }
        }
        auto v_operand = [&](int d) {
            const short* vp = sw + (4 * g + (lane & 15) / 4) * STR + d * 16 + (lane & 3) * 4;
            const s4v x0 = lds_read_tr(vp), x1 = lds_read_tr(vp + 16 * STR);
            return __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7);
        };
        s8v vf[DT];
#pragma unroll
        for (int d = 0; d < DT; d++) vf[d] = v_operand(d);
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int x = 0; x < PP; x++) o[n][d] = mfma16<VB>(vf[d], pf[n][x], o[n][d]);
        __builtin_amdgcn_wave_barrier();
    };

    if (n_tiles) load(0);
    int n_tile = 0;
    for (; n_tile < n_whole; n_tile++) body(std::false_type{}, n_tile);
    for (; n_tile < n_tiles; n_tile++) body(std::true_type{}, n_tile);

    // the waves' results meet in LDS, 16 rows at a time
    constexpr int OS = DP + 4;                   // (16 rows' chunks of 16 bytes in different banks)
    float* so = (float*)&sv[0][0][0];            // [W][16][OS]
    static_assert(W * 16 * OS * 4 <= (int)sizeof(sv), "the waves' results fit V's tiles");
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const float lw = sum16(l[n]);
        __syncthreads();
#pragma unroll
        for (int d = 0; d < DT; d++) *(f4v*)&so[(wave * 16 + col) * OS + d * 16 + 4 * g] = o[n][d];
        if (g == 0) {
            s_ml[wave][col][0] = m[n];
            s_ml[wave][col][1] = lw;
        }
        __syncthreads();
        constexpr int PER = DP / (4 * W);        // dims of a thread
        const int r = tid / (4 * W), d0 = tid % (4 * W) * PER, row = rt0 + n * 16 + r;
        float M = -INFINITY, L = 0.0f, acc[PER] = {};
#pragma unroll
        for (int w = 0; w < W; w++) M = fmaxf(M, s_ml[w][r][0]);
        const float ms = M == -INFINITY ? 0.0f : M;
#pragma unroll
        for (int w = 0; w < W; w++) {
            const float f = exp2_fast(s_ml[w][r][0] - ms);
            L += f * s_ml[w][r][1];
#pragma unroll
            for (int i = 0; i < PER; i++) acc[i] += f * so[(w * 16 + r) * OS + d0 + i];
        }
        if (row >= R || (!EXACT && d0 >= (int)a.dim)) continue;   // (pairs of threads together)
        const int j = row / (int)a.group, h = (int)head0 + row - j * (int)a.group;
        if (it.parts == 1) {
            const float inv = 1.0f / L;
            uint8_t* op = (uint8_t*)a.out + ((size_t)(it.q0 + (uint32_t)j) * a.os + (size_t)h * a.dim + d0) * act_size<ACT>;
#pragma unroll
            for (int i = 0; i < PER; i += 4) {
                float x[4];
                if constexpr (PER >= 4) {
#pragma unroll
                    for (int e = 0; e < 4; e++) x[e] = acc[i + e] * inv;
                    if (EXACT || d0 + i < (int)a.dim) store4<ACT>(op + i * act_size<ACT>, x);
                } else {
                    // two dims a thread (8 waves, 64 dims): pairs of threads meet
                    static_assert(PER == 2 || PER >= 4, "two dims a thread at least");
                    const float y0 = acc[0] * inv, y1 = acc[1] * inv;
                    x[0] = y0; x[1] = y1;
                    x[2] = __shfl_down(y0, 1); x[3] = __shfl_down(y1, 1);
                    if ((tid & 1) == 0 && (EXACT || d0 < (int)a.dim)) store4<ACT>(op, x);
                }
            }
        } else {
            const size_t w = (size_t)(it.ws0 + it.part * it.rows + (uint32_t)j) * a.n_heads + (uint32_t)h;
#pragma unroll
            for (int i = 0; i < PER; i++)
                if (EXACT || d0 + i < (int)a.dim) a.ws_o[w * a.dim + d0 + i] = acc[i];
            if (d0 == 0) {
                a.ws_ml[2 * w] = M;
                a.ws_ml[2 * w + 1] = L;
            }
        }
    }
}

// Joins the parts of the sequences that were cut: one workgroup per (sequence's
// first item, head), its rows one after another.  8 groups of 32 threads take
// every eighth part, 4 dims a thread; then the groups meet in LDS, in order.
// Latency: 3.5 us for one sequence of 6 parts, 6.4 for two of 241.  (The last
// workgroup to end joining inside the attention, with a fence of the whole
// device, took more: 64 contexts 158 us instead of 128.)
template <int ACT>
__global__ __launch_bounds__(256) void k_paged_join(PagedArgs a) {
    const PageItem it = a.items[blockIdx.x];
    if (it.part != 0 || it.parts == 1) return;
    __shared__ float s_f[PG_MOST_PARTS], s_red[2][4];
    __shared__ __align__(16) float s_o[8][128];
    const uint32_t h = blockIdx.y, tid = threadIdx.x, grp = tid >> 5, d = (tid & 31) * 4, wave = tid >> 6;
    for (uint32_t j = blockIdx.z; j < it.rows; j += gridDim.z) {
        const size_t w0 = (size_t)(it.ws0 + j) * a.n_heads + h, step = (size_t)it.rows * a.n_heads;
        float M = -INFINITY, L = 0.0f;
        for (uint32_t p = tid; p < it.parts; p += 256) M = fmaxf(M, a.ws_ml[2 * (w0 + p * step)]);
#pragma unroll
        for (int b = 1; b < 64; b <<= 1) M = fmaxf(M, __shfl_xor(M, b));
        if ((tid & 63) == 0) s_red[0][wave] = M;
        __syncthreads();
        M = fmaxf(fmaxf(s_red[0][0], s_red[0][1]), fmaxf(s_red[0][2], s_red[0][3]));
        const float ms = M == -INFINITY ? 0.0f : M;
        for (uint32_t p = tid; p < it.parts; p += 256) {
            const float f = exp2_fast(a.ws_ml[2 * (w0 + p * step)] - ms);
            L += f * a.ws_ml[2 * (w0 + p * step) + 1];
            s_f[p] = f;
        }
#pragma unroll
        for (int b = 1; b < 64; b <<= 1) L += __shfl_xor(L, b);
        if ((tid & 63) == 0) s_red[1][wave] = L;
        __syncthreads();
        L = (s_red[1][0] + s_red[1][1]) + (s_red[1][2] + s_red[1][3]);
        f4v acc = (f4v)0.0f;
        if (d < a.dim) {
#pragma unroll 4
            for (uint32_t p = grp; p < it.parts; p += 8) {
                const f4v x = *(const f4v*)(a.ws_o + (w0 + p * step) * a.dim + d);
                const float f = s_f[p];
#pragma unroll
                for (int i = 0; i < 4; i++) acc[i] += f * x[i];
            }
        }
        *(f4v*)&s_o[grp][d] = acc;
        __syncthreads();
        if (tid < 32 && d < a.dim) {
            float y[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float t = 0.0f;
#pragma unroll
                for (int g = 0; g < 8; g++) t += s_o[g][d + i];
                y[i] = t / L;
            }
            store4<ACT>((uint8_t*)a.out + ((size_t)(it.q0 + j) * a.os + (size_t)h * a.dim + d) * act_size<ACT>, y);
        }
        __syncthreads();
    }
}

}  // namespace pf

// ================================================================== host

template <int ACT, int CT, int DP, int NT, bool EXACT>
static void paged_one(hipStream_t st, const PageSplit& u, uint32_t z, const PagedArgs& a) {
    const dim3 grid(u.n_items, a.kv_heads, z);
    if constexpr (paged_waves(ACT, CT, DP, NT) > 1)
        if (u.waves == 8) {
            hipLaunchKernelGGL((k_paged_attn<ACT, CT, DP, NT, EXACT, 8>), grid, dim3(512), 0, st, a);
            return;
        }
    hipLaunchKernelGGL((k_paged_attn<ACT, CT, DP, NT, EXACT, 4>), grid, dim3(256), 0, st, a);
}

template <int ACT, int CT, int DP, bool EXACT>
static void paged_rows(hipStream_t st, const PageSplit& u, const PagedArgs& a) {
    const uint32_t R = u.most_rows * a.group;
    // one tile of 16 rows, or two: the keys are read once for both (64 contexts of
    // up to 4000 bf16 keys, 20 rows a kv head: 65 us, 104 as two single tiles)
    if (R <= 16) paged_one<ACT, CT, DP, 1, EXACT>(st, u, 1, a);
    else paged_one<ACT, CT, DP, 2, EXACT>(st, u, (R + 31) / 32, a);
}

template <int ACT, int CT>
static void paged_dim(hipStream_t st, const PageSplit& u, const PagedArgs& a) {
    if (a.dim == 128) paged_rows<ACT, CT, 128, true>(st, u, a);
    else if (a.dim == 64) paged_rows<ACT, CT, 64, true>(st, u, a);
    else if (a.dim < 64) paged_rows<ACT, CT, 64, false>(st, u, a);
    else paged_rows<ACT, CT, 128, false>(st, u, a);
}

// Cuts the pass's keys into shares of at most `chunk` tiles, by what they would
// take, in half tiles' times: the rounds of workgroups (`per` for each share),
// each as long as its longest wave's run of tiles and a tile's time more (two
// with 8 waves, whose results meet in LDS: one bf16 row over 700 keys, 16 heads,
// 10.5 us uncut with 8, 9.3 cut with 4), and where a sequence is cut the second
// kernel, PG_JOIN and one for each PG_JOIN_ROWS rows and heads (48 contexts of
// up to 3000 bf16 keys, 32 heads of 64, five rows: 39 us cut, 31 uncut).  Looked
// at: no cut, and the smallest shares that one round of workgroups holds, or two
// for each sequence (a long one beside short ones), but of a tile for each wave;
// with workgroups of 4 waves, and of 8 (half as many shares, to join as well: 16
// verify passes of five fp32 rows over up to 2100 int8 keys of 16 heads, 23 us
// uncut with 8, 27 cut with 4).  Contexts of 60000 and 32000 fp16 keys take 23
// us cut, 510 uncut.
//
// Tiles of 4-bit rows take a third of the time, so joining counts twice as much
// (PG_JOIN4; one context of 700, 16 heads: 9.5 us cut, 7.5 uncut), and a third
// workgroup on each compute unit, which the registers allow, keeps more bytes
// under way where a wave has many of them (PG_LONG or more; 64 contexts of up to
// 16000: 72 us with three, 78.5 with two; two of 120000 and 64000, 6 a wave: 21 and 19).
constexpr uint32_t PG_CUS = 256, PG_JOIN = 5, PG_JOIN4 = 10, PG_JOIN_ROWS = 512, PG_LONG = 24;
struct PageShares {
    uint32_t chunk = 1, waves = 4;
    uint64_t cost = ~0ull;
};
static uint64_t page_shares_of(const std::vector<uint32_t>& tiles, uint32_t chunk) {
    uint64_t n = 0;
    for (uint32_t t : tiles) n += (t + chunk - 1) / chunk;
    return n;
}
static void page_shares(const std::vector<uint32_t>& tiles, uint32_t longest, uint64_t per, uint64_t round, uint32_t waves,
                        uint64_t join, PageShares* best) {
    const auto take = [&](uint32_t chunk) {
        const uint64_t rounds = (page_shares_of(tiles, chunk) * per + round - 1) / round;
        const uint64_t cost = 2 * rounds * ((chunk + waves - 1) / waves + waves / 4) + (chunk < longest ? join : 0);
        if (cost < best->cost) *best = {chunk, waves, cost};
    };
    const uint32_t least = std::max<uint32_t>(waves, (longest + PG_MOST_PARTS - 1) / PG_MOST_PARTS);
    take(std::max(longest, 1u));
    for (const uint64_t budget : {round / per, (uint64_t)2 * tiles.size()}) {
        uint32_t chunk = least, high = std::max(least, longest);
        while (chunk < high) {
            const uint32_t mid = chunk + (high - chunk) / 2;
            if (page_shares_of(tiles, mid) <= budget) high = mid;
            else chunk = mid + 1;
        }
        if (chunk < longest) take(chunk);
    }
}
// What a pass's attention takes: its sequences' tiles (of those with rows), and
// how they are cut.
struct PagePlan {
    std::vector<uint32_t> tiles;
    uint32_t most = 0, longest = 0, keys = 0;   // rows, tiles and keys of a sequence at most
    uint32_t held = 0;                          // workgroups of 4 waves on a compute unit
    PageShares shares;
};
static PagePlan paged_plan(const std::vector<PageSeq>& pass, const pf_attn_desc* d, int32_t ct, const AttnShape& s) {
    PagePlan n;
    n.tiles.reserve(pass.size());
    uint64_t rows = 0;
    for (const PageSeq& q : pass) {
        if (!q.rows) continue;
        n.tiles.push_back((uint32_t)page_tiles(q.rows, q.len, s.window, s.sink).count);
        n.longest = std::max(n.longest, n.tiles.back());
        n.most = std::max(n.most, q.rows);
        n.keys = std::max(n.keys, q.len);
        rows += q.rows;
    }
    const uint64_t R = (uint64_t)n.most * (d->n_heads / d->n_kv_heads), per = (uint64_t)d->n_kv_heads * (R <= 16 ? 1 : (R + 31) / 32);
    uint32_t& held = n.held = (uint32_t)paged_waves(d->type, ct, d->head_dim <= 64 ? 64 : 128, R <= 16 ? 1 : 2);
    const bool fp4 = ct == PF_TYPE_FP4;
    if (fp4 && held == 3) {
        uint64_t all = 0;
        for (uint32_t t : n.tiles) all += t;
        if (all * per < PG_LONG * 4 * 2 * PG_CUS) held = 2;
    }
    const uint64_t join = (fp4 ? PG_JOIN4 : PG_JOIN) + rows * d->n_heads / PG_JOIN_ROWS;
    page_shares(n.tiles, n.longest, per, (uint64_t)PG_CUS * held, 4, join, &n.shares);
    if (held > 1) page_shares(n.tiles, n.longest, per, (uint64_t)PG_CUS * (held / 2), 8, join, &n.shares);
    return n;
}
extern "C" pf_status pf_test_pages_plan_of(const pf_attn_desc* d, int32_t cache, const uint32_t* rows, const uint32_t* lens,
                                           uint32_t n, uint32_t* waves, uint32_t* chunk, uint32_t* longest, uint32_t* held) {
    AttnShape s;
    if (pf_status st = attn_desc_check(nullptr, d, &s)) return st;
    return no_throw(nullptr, [&] {
        std::vector<PageSeq> pass;
        for (uint32_t i = 0; i < n; i++) pass.push_back({i, 0, rows[i], lens[i]});
        const PagePlan plan = paged_plan(pass, d, cache, s);
        *waves = plan.shares.waves;
        *chunk = plan.shares.chunk;
        *longest = plan.longest;
        *held = plan.held;
        return (pf_status)PF_OK;
    });
}
extern "C" pf_status pf_test_pages_plan(const pf_attn_desc* d, const uint32_t* rows, const uint32_t* lens, uint32_t n,
                                        uint32_t* waves, uint32_t* chunk, uint32_t* longest) {
    uint32_t held;
    return d ? pf_test_pages_plan_of(d, d->type, rows, lens, n, waves, chunk, longest, &held) : PF_ERR_ARG;
}
static pf_status paged_cut(pf_pages* p, const pf_attn_desc* d, const AttnShape& s) {
    PageSplit& u = p->cut;
    if (u.type == d->type && u.window == s.window && u.sink == s.sink && u.heads == d->n_heads) return PF_OK;
    const PagePlan plan = paged_plan(p->pass, d, p->cfg.type, s);
    if ((uint64_t)plan.most * (d->n_heads / d->n_kv_heads) > 32 * 65535u)
        return fail(p->ctx, PF_ERR_UNSUPPORTED, "pages: too many rows in one pass; cut it");
    const uint32_t chunk = plan.shares.chunk;
    PageSplit n;
    n.waves = plan.shares.waves;
    std::vector<PageItem> items;
    items.reserve(page_shares_of(plan.tiles, chunk));
    uint64_t ws = 0;
    uint32_t i = 0;
    for (const PageSeq& q : p->pass) {
        if (!q.rows) continue;
        const uint32_t t = plan.tiles[i++], parts = (t + chunk - 1) / chunk;
        for (uint32_t k = 0; k < parts; k++)
            items.push_back({q.slot, q.q0, q.rows, q.len, (uint32_t)((uint64_t)t * k / parts),
                             (uint32_t)((uint64_t)t * (k + 1) / parts), (uint32_t)ws, parts, k});
        if (parts == 1) continue;
        ws += (uint64_t)parts * q.rows;
        n.split = true;
    }
    if (ws * d->n_heads > 0x7FFFFFFFu) return fail(p->ctx, PF_ERR_UNSUPPORTED, "pages: too many rows in one pass; cut it");
    if (items.size() > p->items_cap) return fail(p->ctx, PF_ERR_STATE, "pages: work list exceeded");
    if (pf_status st = pages_upload(p, p->items, items.data(), items.size() * sizeof(PageItem))) return st;
    n.window = s.window; n.sink = s.sink; n.heads = d->n_heads; n.type = d->type;
    n.n_items = (uint32_t)items.size(); n.ws_rows = (uint32_t)ws; n.most_rows = plan.most; n.longest = plan.keys;
    u = n;
    return PF_OK;
}

extern "C" pf_status pf_pages_attention(pf_pages* p, const pf_attn_desc* d, uint32_t layer, const void* q, void* out) {
    if (!p || !d) return PF_ERR_ARG;
    pf_ctx* c = p->ctx;
    AttnShape s;
    if (pf_status st = attn_desc_check(c, d, &s)) return st;
    if (layer >= p->cfg.n_layers) return fail(c, PF_ERR_ARG, "pages: layer out of range");
    if (d->n_kv_heads != p->cfg.n_kv_heads || d->head_dim != p->cfg.head_dim)
        return fail(c, PF_ERR_ARG, "pages: n_kv_heads and head_dim are the cache's");
    const int32_t ct = p->cfg.type;
    if (ct != PF_TYPE_I8 && ct != PF_TYPE_FP4 && ct != d->type && !(ct == PF_TYPE_BF16 && d->type == PF_TYPE_F32))
        return fail(c, PF_ERR_UNSUPPORTED, "pages: rows of this type over a cache of that type");
    if (!p->open) return fail(c, PF_ERR_STATE, "pages: no open pass (pf_pages_append begins one)");
    if (!p->pass_rows) return PF_OK;
    if (!q || !out) return fail(c, PF_ERR_ARG, "pages: a buffer is NULL");
    if (!aligned16(q) || !aligned16(out)) return fail(c, PF_ERR_ARG, "pages: buffers start on 16 bytes");
    const size_t es = d->type == PF_TYPE_F32 ? 4 : 2, qw = (size_t)d->n_heads * d->head_dim;
    if (overlaps(out, ((size_t)(p->pass_rows - 1) * s.os + qw) * es, q, ((size_t)(p->pass_rows - 1) * s.qs + qw) * es))
        return fail(c, PF_ERR_ARG, "pages: out overlaps q");
    DeviceScope on(c);
    if (pf_status st = no_throw(c, [&] { return paged_cut(p, d, s); })) return st;
    const PageSplit& u = p->cut;
    PagedArgs a{};
    if (u.split) {
        const size_t rows = (size_t)u.ws_rows * d->n_heads;
        void* ws = nullptr;
        if (pf_status st = ctx_scratch(c, rows * (d->head_dim + 2) * 4, &ws)) return st;
        a.ws_o = (float*)ws;
        a.ws_ml = a.ws_o + rows * d->head_dim;
    }
    a.items = p->items; a.table = p->table; a.table_stride = p->per_seq;
    a.k = (const uint8_t*)p->k + layer * p->plane; a.v = (const uint8_t*)p->v + layer * p->plane;
    a.ks = (const uint8_t*)p->ks + layer * p->scales; a.vs = (const uint8_t*)p->vs + layer * p->scales;
    a.q = q; a.out = out; a.qs = s.qs; a.os = s.os;
    a.n_heads = d->n_heads; a.kv_heads = d->n_kv_heads; a.group = d->n_heads / d->n_kv_heads; a.dim = d->head_dim;
    a.page_shift = p->shift;
    a.causal = d->causal != 0; a.window = (int32_t)s.window; a.sink = (int32_t)s.sink;
    a.scale_log2 = s.scale_log2;
    a.above = (float)keys_shift(u.longest);
    a.down = std::ldexp(1.0f, -keys_shift(u.longest));
    hipStream_t st = c->stream;
#define PF_PAGED(A, T) paged_dim<A, T>(st, u, a)
    if (ct == PF_TYPE_I8) {
        if (d->type == PF_TYPE_F32) PF_PAGED(PF_TYPE_F32, PF_TYPE_I8);
        else if (d->type == PF_TYPE_F16) PF_PAGED(PF_TYPE_F16, PF_TYPE_I8);
        else PF_PAGED(PF_TYPE_BF16, PF_TYPE_I8);
    } else if (ct == PF_TYPE_FP4) {
        if (d->type == PF_TYPE_F32) PF_PAGED(PF_TYPE_F32, PF_TYPE_FP4);
        else if (d->type == PF_TYPE_F16) PF_PAGED(PF_TYPE_F16, PF_TYPE_FP4);
        else PF_PAGED(PF_TYPE_BF16, PF_TYPE_FP4);
    } else if (ct == PF_TYPE_F16) PF_PAGED(PF_TYPE_F16, PF_TYPE_F16);
    else if (d->type == PF_TYPE_F32) PF_PAGED(PF_TYPE_F32, PF_TYPE_BF16);
    else PF_PAGED(PF_TYPE_BF16, PF_TYPE_BF16);
#undef PF_PAGED
    PF_LAUNCHED(c);
    if (u.split) {
        const dim3 grid(u.n_items, d->n_heads, std::min(u.most_rows, 64u));
        if (d->type == PF_TYPE_F32) hipLaunchKernelGGL(k_paged_join<PF_TYPE_F32>, grid, dim3(256), 0, st, a);
        else if (d->type == PF_TYPE_F16) hipLaunchKernelGGL(k_paged_join<PF_TYPE_F16>, grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL(k_paged_join<PF_TYPE_BF16>, grid, dim3(256), 0, st, a);
        PF_LAUNCHED(c);
    }
    return PF_OK;
}
