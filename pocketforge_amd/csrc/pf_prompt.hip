// Attention over whole prompts: packed sequences, grouped heads, causal and
// windowed masks (pf_prompt_attention of include/pf_gpu.h).
//
// A query row i of a sequence sees keys j with j <= p (causal) and, with a
// window, j > p - window or j < sink, where p is its position:
//   out_i = sum_j exp(s_ij - m_i) v_j / sum_j exp(s_ij - m_i),
//   s_ij = scale * q_i . k_j,   m_i = max_j s_ij.
// One pass over the keys: the running maximum m and sum l of a row are
// corrected when m moves, so nothing of size rows x keys is stored.
#include "pf_attend.h"
#include "pf_context.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

using namespace pf;

namespace pf {

constexpr int PR_SEQS = 64;       // sequences of one launch
constexpr int PR_KEYS = 64;       // keys of a tile
constexpr uint32_t PR_HEADS = 4;  // kv heads that an XCD takes together
constexpr uint32_t PR_CUS = 256;  // compute units
constexpr uint64_t PR_MOST_UNITS = (1u << 24) - 64;   // workgroups of a launch

struct PromptSeq {
    uint32_t q0, nq, k0, nk;      // first rows and lengths
};
struct PromptArgs {
    const void *q, *k, *v;
    void* out;
    uint32_t n_seq, n_heads, group, dim;
    uint32_t qs, ks, vs, os;      // row strides in elements
    int32_t causal, window, sink;
    float scale_log2;
    float above, down;            // how far m is held above the scores (bf16 rows), what weights are held to (fp32)
    uint32_t tiles;               // query tiles of all sequences
    uint32_t parts, rows;         // parts that the keys are cut in (grid y), rows of a part's results
    float* ws_o;                  // parts > 1: [parts][rows][n_heads][dim]
    float* ws_ml;                 // [parts][rows][n_heads][2]
    uint32_t tile0[PR_SEQS];      // first query tile of each sequence
    PromptSeq seq[PR_SEQS];
};

// The workgroups of a launch.  Workgroup u runs on XCD u mod 8, each with an L2
// of its own, so the query heads and tiles that read one kv head's rows go to
// one XCD (8 kv heads or a multiple), or to the 8 / kv_heads XCDs of theirs
// (1, 2 or 4); within it the query heads of a tile come one after another, and
// tiles from the last: a causal sequence's last tiles see the most keys, and
// the short ones fill the end.  An XCD takes a tile of up to PR_HEADS kv heads
// before the next tile (6000 bf16 rows, 32 heads of 128: 300 us; 309 with two,
// 306 with eight, 320 with one head after the other).
struct PromptUnit {
    uint32_t head, tile;
    bool none;
};
__host__ __device__ __forceinline__ uint32_t prompt_units(uint32_t tiles, uint32_t kv, uint32_t group) {
    const uint32_t per = tiles * group;
    return kv < 8 && 8 % kv == 0 ? 8 * ((per + 8 / kv - 1) / (8 / kv)) : kv * per;
}
__device__ __forceinline__ PromptUnit prompt_unit(uint32_t u, uint32_t tiles, uint32_t kv, uint32_t group) {
    const uint32_t per = tiles * group, x = u % 8, i = u / 8;
    uint32_t h, j;
    if (kv % 8 == 0) {
        const uint32_t of = i / (PR_HEADS * per) * PR_HEADS, n = min(PR_HEADS, kv / 8 - of), r = i - of * per;
        h = x + 8 * (of + r / group % n);
        j = r / (group * n) * group + r % group;
    } else if (8 % kv == 0) {
        h = x % kv;
        j = i * (8 / kv) + x / kv;
    } else {
        h = u % (kv * group) / group;
        j = u / (kv * group) * group + u % (kv * group) % group;
    }
    return {h * group + j % group, tiles - 1 - j / group, j >= per};
}

// A workgroup: 4 waves of one head, each with 32 query rows; SPLIT 2: two and
// two waves share 32 rows, and each takes half of every key tile.  Scores are
// formed as S^T = K Q^T, so that a lane holds 16 keys of one row: its maximum
// and sum need one exchange between two lanes, and exp(S)^T is already the
// operand of O^T = V^T P^T, whose other operand comes from V's rows in LDS
// through transposing reads.

// What a workgroup knows of its tile of 128 / SPLIT query rows.
template <int SPLIT>
struct PromptTile {
    static constexpr int ROWS = 128 / SPLIT;
    uint32_t q0, k0, head;
    int nq, nk, r0, off;          // lengths, first row, position of row 0
    int p0, p1;                   // positions of the first and the last row
    int first, sinks, wa, wb, whole;
    int at, tiles, n_whole;       // this part's: first key tile in that order, tiles, whole ones (they are first)

    // The key tiles that some row sees, in the order they are taken: those that
    // all rows see whole (wa .. wb - 1), then the sinks' and the rest from `first`.
    __device__ __forceinline__ int key_tile(int it) const {
        it += at;
        if (it < whole) return wa + it;
        it -= whole;
        if (it < sinks) return it;
        it += first - sinks;
        return it < wa ? it : it + whole;
    }
    // this wave's rows see something of the keys from key0 on
    __device__ __forceinline__ bool some(const PromptArgs& a, int key0, int wave) const {
        const int w0 = p0 + wave % (4 / SPLIT) * 32, w1 = min(w0 + 31, p1);
        return !((a.causal && key0 > w1) | (a.window && key0 + PR_KEYS <= w0 - a.window + 1 && key0 >= a.sink));
    }
};
template <int SPLIT>
__device__ __forceinline__ bool prompt_tile(const PromptArgs& a, PromptTile<SPLIT>* t) {
    const PromptUnit unit = prompt_unit(blockIdx.x, a.tiles, a.n_heads / a.group, a.group);
    if (unit.none) return false;
    const int lane = threadIdx.x & 63;
    const uint64_t before = __ballot(lane < (int)a.n_seq && a.tile0[lane] <= unit.tile);
    const int seq = 63 - __builtin_clzll(before);
    t->head = unit.head;
    t->q0 = a.seq[seq].q0; t->k0 = a.seq[seq].k0;
    t->nq = (int)a.seq[seq].nq; t->nk = (int)a.seq[seq].nk;
    t->off = t->nk - t->nq;
    t->r0 = (int)(unit.tile - a.tile0[seq]) * t->ROWS;
    t->p0 = t->off + t->r0;
    t->p1 = t->off + min(t->r0 + t->ROWS, t->nq) - 1;
    const int end = min(t->nk, a.causal ? t->p1 + 1 : t->nk), last = end <= 0 ? 0 : (end + PR_KEYS - 1) / PR_KEYS;
    t->first = (a.window ? max(0, t->p0 - a.window + 1) : 0) / PR_KEYS;
    t->sinks = min(min((a.sink + PR_KEYS - 1) / PR_KEYS, t->first), last);
    const int tiles = max(0, last - t->first) + t->sinks;
    t->wa = a.window ? max(t->first, (max(0, t->p1 - a.window + 1) + PR_KEYS - 1) / PR_KEYS) : 0;
    t->wb = max(t->wa, min(t->nk, a.causal ? max(0, t->p0 + 1) : t->nk) / PR_KEYS);
    t->whole = tiles ? t->wb - t->wa : 0;
    t->at = 0;
    t->tiles = tiles;
    if (SPLIT == 2) {
        t->at = (int)((uint32_t)tiles * blockIdx.y / a.parts);
        t->tiles = (int)((uint32_t)tiles * (blockIdx.y + 1) / a.parts) - t->at;
    }
    t->n_whole = min(max(0, t->whole - t->at), t->tiles);
    return true;
}

// The scores of keys key0 .. that a row does not see become -infinity; one bit
// per key, lanes of the upper half four keys on.
template <int G>
__device__ __forceinline__ void mask_scores(f16v (&s)[G], const PromptArgs& a, int nk, int hi, int lo, int key0, int half) {
    const uint64_t see = first_bits(min(hi, nk - 1) + 1 - key0) & (~first_bits(lo - key0) | first_bits(a.sink - key0));
    const uint32_t part[2] = {(uint32_t)see >> (4 * half), (uint32_t)(see >> 32) >> (4 * half)};
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
        for (int i = 0; i < 16; i++)
            s[g][i] = bits_or(s[g][i], -INFINITY, __builtin_amdgcn_sbfe((int)part[g], 8 * (i / 4) + i % 4, 1));
}

// The running maximum over a tile's scores (scaled to base 2), with the sum and
// the output corrected where it moves; the value to subtract.
template <bool BF, int DT, int G>
__device__ __forceinline__ float new_maximum(const f16v (&s)[G], float scale, float above, float& m, float& l, f16v (&o)[DT]) {
    float top = s[0][0];
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
        for (int i = 0; i < 16; i++) top = fmaxf(top, s[g][i]);
    top *= scale;
    if (__any(top > m + (m_slack<BF> - above))) {
        const float to = fmaxf(m, max32(top) + above);
        const float f = m == -INFINITY ? 1.0f : exp2_fast(m - to);   // (nothing yet, or infinities that stay)
        m = to;
        l *= f;
#pragma unroll
        for (int t = 0; t < DT; t++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[t][i] *= f;
    }
    return m == -INFINITY ? 0.0f : m;
}

// SPLIT 2: the waves of the upper key halves hand their results to the others
// through LDS: DT / 2 pieces of 8 KB in x0 and in x1, 2 KB in x2.
template <int DT>
__device__ __forceinline__ void join_halves(int wave, float& m, float& l, f16v (&o)[DT], void* x0, void* x1, void* x2) {
    const int lane = threadIdx.x & 63, at = (wave & 1) * 256 + lane;
    f4v* ml = (f4v*)x2 + (wave & 1) * 64 + lane;
    l = sum32(l);
    __syncthreads();
    if (wave >= 2) {
#pragma unroll
        for (int n = 0; n < DT; n++) {
            f4v* p = (f4v*)(n < DT / 2 ? x0 : x1) + n % (DT / 2) * 512 + at;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const f4v x = {o[n][4 * i], o[n][4 * i + 1], o[n][4 * i + 2], o[n][4 * i + 3]};
                p[i * 64] = x;
            }
        }
        const f4v x = {m, l, 0.0f, 0.0f};
        *ml = x;
    }
    __syncthreads();
    if (wave >= 2) return;
    const f4v x = *ml;
    const float to = fmaxf(m, x[0]), ms = to == -INFINITY ? 0.0f : to, f1 = exp2_fast(x[0] - ms);
    const float f0 = m == -INFINITY ? 1.0f : exp2_fast(m - ms);      // (as in new_maximum)
    m = to;
    l = l * f0 + x[1] * f1;
#pragma unroll
    for (int n = 0; n < DT; n++) {
        const f4v* p = (const f4v*)(n < DT / 2 ? x0 : x1) + n % (DT / 2) * 512 + at;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const f4v y = p[i * 64];
#pragma unroll
            for (int j = 0; j < 4; j++) o[n][4 * i + j] = o[n][4 * i + j] * f0 + y[j] * f1;
        }
    }
}

// What a row's output is multiplied by.  A row that sees no key is zero; one
// whose scores are all -infinity is 0 / 0.
template <int ROWS>
__device__ __forceinline__ float row_factor(const PromptArgs& a, const PromptTile<ROWS>& t, int my, float l, bool* none) {
    *none = !(a.causal ? t.off + my >= 0 : t.nk > 0);
    return *none ? 0.0f : 1.0f / l;
}

// SPLIT 2: a part's results, where the keys are cut.
template <bool EXACT, int DT>
__device__ __forceinline__ void store_part(const PromptArgs& a, const PromptTile<2>& t, int my, int half, float m, float l,
                                           const f16v (&o)[DT]) {
    if (my >= t.nq) return;
    bool none;
    row_factor(a, t, my, l, &none);
    const size_t w = ((size_t)blockIdx.y * a.rows + t.q0 + (uint32_t)my) * a.n_heads + t.head;
    float* op = a.ws_o + w * a.dim;
#pragma unroll
    for (int n = 0; n < DT; n++)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int d = n * 32 + 8 * (i / 4) + 4 * half;
            if (!EXACT && d >= (int)a.dim) continue;
            const f4v x = {o[n][i], o[n][i + 1], o[n][i + 2], o[n][i + 3]};
            *(f4v*)(op + d) = none ? (f4v)0.0f : x;
        }
    if (half == 0) {                             // (a row that sees no key: zeros of weight 1)
        a.ws_ml[2 * w] = none ? 0.0f : m;
        a.ws_ml[2 * w + 1] = none ? 1.0f : l;
    }
}

// Joins the parts (up to 32): 32 threads take a row of a head, 4 dims each.
// Bound by a launch's latency and the parts' bytes.
constexpr uint32_t PR_MOST_PARTS = 32;
template <int ACT>
__global__ __launch_bounds__(256) void k_prompt_join(PromptArgs a) {
    const uint32_t lane = threadIdx.x & 31, unit = blockIdx.x * 8 + (threadIdx.x >> 5), d = lane * 4;
    const size_t step = (size_t)a.rows * a.n_heads;
    if (unit >= step) return;
    float m = -INFINITY, l = 0.0f;
    if (lane < a.parts) {
        m = a.ws_ml[2 * (unit + lane * step)];
        l = a.ws_ml[2 * (unit + lane * step) + 1];
    }
    float top = m;
#pragma unroll
    for (int b = 1; b < 32; b <<= 1) top = fmaxf(top, __shfl_xor(top, b));
    const float f = exp2_fast(m - (top == -INFINITY ? 0.0f : top));
    l *= f;
#pragma unroll
    for (int b = 1; b < 32; b <<= 1) l += __shfl_xor(l, b);
    f4v acc = (f4v)0.0f;
    const float* op = a.ws_o + (size_t)unit * a.dim + d;
#pragma unroll 4
    for (uint32_t p = 0; p < a.parts; p++) {
        const float fp = __shfl(f, (int)p, 32);
        if (d < a.dim) {
            const f4v x = *(const f4v*)(op + p * step * a.dim);
#pragma unroll
            for (int i = 0; i < 4; i++) acc[i] += fp * x[i];
        }
    }
    if (d >= a.dim) return;
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; i++) y[i] = acc[i] / l;
    const uint32_t row = unit / a.n_heads, h = unit % a.n_heads;
    store4<ACT>((uint8_t*)a.out + ((size_t)row * a.os + (size_t)h * a.dim + d) * act_size<ACT>, y);
}

// fp32 rows, three bf16 pieces each: six matrix instructions where 16-bit rows
// take one, which bound it (a bf16 instruction does 16 times the fp32 one's
// work).  A tile's rows wait in registers while the tile before is worked on,
// and are cut into pieces on their way to LDS.  3 prompts of up to 1100 rows
// after 333 cached, 12 heads of 64, window 1024: 62 us, or 96 TFLOP/s of fp32
// products (a large one by the library reaches 137); 516 workgroups of 64 rows
// are one round, whose longest ends last.
template <int DP, bool EXACT, int SPLIT>
__global__ __launch_bounds__(256, DP == 64 ? 2 : 1) void k_prompt_attn32(PromptArgs a) {
    constexpr int ACT = PF_TYPE_F32, NP = 3;
    constexpr int KS = DP + 8, VS = DP + 32;     // LDS row strides without bank conflicts for either kind of read
    constexpr int C = DP / 16, DT = DP / 32, CH = DP / 8, LOADS = PR_KEYS * CH / 256;
    constexpr int G = 2 / SPLIT;                 // 32-key halves of a tile that a wave takes
    __shared__ __align__(16) short sk[NP][PR_KEYS][KS];
    __shared__ __align__(16) short sv[NP][PR_KEYS][VS];
    __shared__ int s_odd;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, row = lane & 31, half = lane >> 5;
    PromptTile<SPLIT> T;
    if (!prompt_tile(a, &T)) return;
    const int nk = T.nk, my = T.r0 + wave % (4 / SPLIT) * 32 + row, p = T.off + my;
    const int part = SPLIT == 2 ? wave / 2 * 32 : 0;   // first key of a tile that this wave takes
    const int hi = a.causal ? p : nk - 1, lo = a.window ? max(0, p - a.window + 1) : 0;

    s8v qf[NP][C];                               // Q^T: 16 dims of a row per matrix instruction
    {
        const uint32_t qr = T.q0 + (uint32_t)min(my, T.nq - 1);
        const float* qp = (const float*)a.q + (size_t)qr * a.qs + (size_t)T.head * a.dim + half * 8;
#pragma unroll
        for (int c = 0; c < C; c++) {
            float x[8] = {};
            if (EXACT || c * 16 + half * 8 < (int)a.dim) load8<ACT>(qp + c * 16, x);
            s8v t[NP];
            split3(x, t);
#pragma unroll
            for (int n = 0; n < NP; n++) qf[n][c] = t[n];
        }
    }

    const size_t kv_head = (size_t)(T.head / a.group) * a.dim;
    const float* kg = (const float*)a.k + (size_t)T.k0 * a.ks + kv_head;
    const float* vg = (const float*)a.v + (size_t)T.k0 * a.vs + kv_head;
    float xk[LOADS][8], xv[LOADS][8];
    auto load = [&](int it) {
        const int key0 = T.key_tile(it) * PR_KEYS;
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            const int e = i * 256 + tid, d = e % CH * 8;
            const uint32_t kr = (uint32_t)min(key0 + e / CH, nk - 1);   // (rows past the end: masked)
            const bool on = EXACT || d < (int)a.dim;
            const size_t at = on ? d : 0;
            load8<ACT>(kg + (size_t)kr * a.ks + at, xk[i]);
            load8<ACT>(vg + (size_t)kr * a.vs + at, xv[i]);
            if (!EXACT && !on)
#pragma unroll
                for (int j = 0; j < 8; j++) xk[i][j] = xv[i][j] = 0.0f;
        }
    };

    f16v o[DT];
#pragma unroll
    for (int t = 0; t < DT; t++) o[t] = (f16v)0.0f;
    float m = -INFINITY, l = 0.0f;

    auto body = [&](auto masked, int it) {
        constexpr bool MASKED = decltype(masked)::value;
        const int key0 = T.key_tile(it) * PR_KEYS;
        __syncthreads();                         // nobody reads the tile before
        float z = 0.0f;
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            const int e = i * 256 + tid, r = e / CH, d = e % CH * 8;
            s8v tk[NP], tv[NP];
            split3(xk[i], tk);
            split3(xv[i], tv);
#pragma unroll
            for (int n = 0; n < NP; n++) {
                *(s8v*)&sk[n][r][d] = tk[n];
                *(s8v*)&sv[n][r][d] = tv[n];
            }
            if constexpr (MASKED)
#pragma unroll
                for (int j = 0; j < 8; j++) z = __builtin_fmaf(xv[i][j], 0.0f, z);
        }
        if (MASKED && z != z) s_odd = it;
        __syncthreads();
        if (it + 1 < T.tiles) load(it + 1);
        if constexpr (MASKED) {
            // values that are not finite reach the rows that see them, whatever
            // their weight, and the products find zeros in their places
            if (s_odd == it) {
                for (int r = 0; r < PR_KEYS; r++) {
                    const int key = key0 + r;
                    if (key >= nk || !key_visible(key, hi, lo, a.sink) || (SPLIT == 2 && wave >= 2)) continue;
#pragma unroll
                    for (int t = 0; t < DT; t++)
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            const int d = t * 32 + 8 * (i / 4) + 4 * half + i % 4;
                            if (not_finite<true>(sv[0][r][d])) o[t][i] += to_float<PF_TYPE_BF16>(sv[0][r][d]);
                        }
                }
                __syncthreads();
                for (int i = 0; i < LOADS; i++) {
                    const int e = i * 256 + tid, r = e / CH, d = e % CH * 8;
                    const s8v x = *(const s8v*)&sv[0][r][d];
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        if (not_finite<true>(x[j])) sv[0][r][d + j] = sv[1][r][d + j] = sv[2][r][d + j] = 0;
                }
                __syncthreads();
            }
            if (!T.some(a, key0, wave)) return;
        }
        f16v s[G];
#pragma unroll
        for (int g = 0; g < G; g++) s[g] = (f16v)0.0f;
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int g = 0; g < G; g++) {
                s8v kf[NP];
#pragma unroll
                for (int n = 0; n < NP; n++) kf[n] = *(const s8v*)&sk[n][part + g * 32 + row][c * 16 + half * 8];
#pragma unroll
                for (int x = 0; x < NP; x++)
#pragma unroll
                    for (int y = 0; x + y < NP; y++) s[g] = mfma32<true>(kf[x], qf[y][c], s[g]);
            }
        if constexpr (MASKED) mask_scores(s, a, nk, hi, lo, key0 + part, half);
        const float ms = new_maximum<true>(s, a.scale_log2, 0.0f, m, l, o);
#pragma unroll
        for (int gh = 0; gh < 2 * G; gh++) {     // 16 keys: a lane's 8 are 4 half .. + 3 and 8 + 4 half .. + 3
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[i] = exp2_fast(__builtin_fmaf(s[gh / 2][8 * (gh & 1) + i], a.scale_log2, -ms)) * a.down;
                l += x[i];
            }
            s8v pf[NP];
            split3(x, pf);
            const int r = part + gh * 16 + 4 * half + (lane & 15) / 4;
#pragma unroll
            for (int t = 0; t < DT; t++) {
                const int d = t * 32 + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
                s8v vf[NP];
#pragma unroll
                for (int n = 0; n < NP; n++) {
                    const s4v x0 = lds_read_tr(&sv[n][r][d]), x1 = lds_read_tr(&sv[n][r + 8][d]);
                    vf[n] = __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7);
                }
#pragma unroll
                for (int u = 0; u < NP; u++)
#pragma unroll
                    for (int y = 0; u + y < NP; y++) o[t] = mfma32<true>(vf[u], pf[y], o[t]);
            }
        }
    };
    if (tid == 0) s_odd = -1;
    if (T.tiles) load(0);
    int it = 0;
    for (; it < T.n_whole; it++) body(std::false_type{}, it);
    for (; it < T.tiles; it++) body(std::true_type{}, it);
    if constexpr (SPLIT == 2) {
        uint8_t* x = (uint8_t*)&sv[0][0][0];
        static_assert(DT * 8192 + 2048 <= sizeof(sv), "the halves' exchange fits V's tile");
        join_halves(wave, m, l, o, x, x + DT / 2 * 8192, x + DT * 8192);
        if (wave >= 2) return;
        if (a.parts > 1) return store_part<EXACT>(a, T, my, half, m, l, o);
    } else {
        l = sum32(l);
    }
    if (my >= T.nq) return;
    bool none;
    const float f = row_factor(a, T, my, l, &none);
    float* op = (float*)a.out + (size_t)(T.q0 + (uint32_t)my) * a.os + (size_t)T.head * a.dim;
#pragma unroll
    for (int n = 0; n < DT; n++)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int d = n * 32 + 8 * (i / 4) + 4 * half;
            if (!EXACT && d >= (int)a.dim) continue;
            float x[4];
#pragma unroll
            for (int j = 0; j < 4; j++) x[j] = none ? 0.0f : o[n][i + j] * f;
            store4<ACT>(op + d, x);
        }
}

// fp16 and bf16 rows: K and V tiles go from memory straight to LDS, two tiles
// deep, while the tile before is worked on; a wave whose rows see nothing of a
// tile leaves it out, and only tiles that some of its rows see in part are
// masked.
//
// LDS rows are not padded (a wave's load writes 1 KiB in a row), so their
// 16-byte chunks are permuted: K's so that the 16 rows that one read cycle
// takes chunk c of lie in 16 different places, V's so that the four rows of a
// transposing read lie in different quarters of the banks: no counted conflicts
// beyond 1% of the LDS cycles.
//
// 8192 causal bf16 rows, 16 heads of 128: 288 us, 950 TFLOP/s of the 1210 that a
// large bf16 product by the library reaches.  What bounds it: the matrix and the
// exp instructions at the clock that they leave (1.95-2.05 GHz; matrix unit busy
// 50% of the cycles that a compute unit has work): without loads, LDS reads and
// barriers 238.  24 packed prompts of 175 to 700 rows, 16 heads of 128 over 4:
// 54 us, three rounds of workgroups with 3 to 11 key tiles each, so the way in
// (lengths, then Q and the first tile) and out counts as much as the tiles.
// Two workgroups of 4 waves a compute unit: three spill, one of 8 waves in
// lockstep takes 282 and 75, and the next tile's scores before this tile's
// weights spill.
template <int DP>
__device__ __forceinline__ int k_place(int r, int c) {
    return DP == 128 ? c ^ (r & 15) : c ^ ((r >> 1) & 7);
}
template <int DP>
__device__ __forceinline__ int v_place(int r, int c) {
    return DP == 128 ? c ^ ((r & 3) << 2) : c ^ (((r >> 1) & 1) << 2);
}

typedef __attribute__((address_space(1))) const void gvoid;
typedef __attribute__((address_space(3))) void lvoid;

template <int ACT, int DP, bool EXACT, int SPLIT>
__global__ __launch_bounds__(256, 2) void k_prompt_attn16(PromptArgs a) {
    constexpr bool BF = op_bf<ACT>;
    constexpr int C = DP / 16, DT = DP / 32;
    constexpr int CH = DP / 8, RPL = 64 / CH;    // chunks of a row, rows of one load of a wave
    constexpr int LOADS = PR_KEYS / 4 / RPL;     // loads of a wave per tile, K or V
    constexpr int G = 2 / SPLIT;                 // 32-key halves of a tile that a wave takes
    // (buffers of their own: the compiler lets reads of one pass loads into the other)
    __shared__ __align__(16) short sk0[PR_KEYS * DP], sk1[PR_KEYS * DP], sv0[PR_KEYS * DP], sv1[PR_KEYS * DP];
    __shared__ int s_odd;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, row = lane & 31, half = lane >> 5;

    PromptTile<SPLIT> T;
    if (!prompt_tile(a, &T)) return;
    const int nk = T.nk, my = T.r0 + wave % (4 / SPLIT) * 32 + row, p = T.off + my;
    const int part = SPLIT == 2 ? wave / 2 * 32 : 0;   // first key of a tile that this wave takes
    const int hi = a.causal ? p : nk - 1, lo = a.window ? max(0, p - a.window + 1) : 0;

    s8v qf[C];
    {
        const uint32_t qr = T.q0 + (uint32_t)min(my, T.nq - 1);
        const short* qp = (const short*)a.q + (size_t)qr * a.qs + (size_t)T.head * a.dim + half * 8;
#pragma unroll
        for (int c = 0; c < C; c++) {
            qf[c] = (s8v)(short)0;
            if (EXACT || c * 16 + half * 8 < (int)a.dim) qf[c] = *(const s8v*)(qp + c * 16);
        }
    }

    const size_t kv_head = (size_t)(T.head / a.group) * a.dim;
    const short* kg = (const short*)a.k + (size_t)T.k0 * a.ks + kv_head;
    const short* vg = (const short*)a.v + (size_t)T.k0 * a.vs + kv_head;
    // a lane's place in a tile's rows as 32-bit offsets from the tile's first row
    const int lr = lane / CH, lc = lane % CH;
    const bool near = (uint64_t)max(a.ks, a.vs) * (PR_KEYS * 2) <= 0xFFFFFFFFull;
    uint32_t ko[LOADS], vo[LOADS];
    auto chunks = [&](int r, int* ck, int* cv) {
        *ck = k_place<DP>(r, lc);
        *cv = v_place<DP>(r, lc);
        if (!EXACT) {                            // (past head_dim: unused)
            *ck = min(*ck, (int)a.dim / 8 - 1);
            *cv = min(*cv, (int)a.dim / 8 - 1);
        }
    };
#pragma unroll
    for (int i = 0; i < LOADS; i++) {
        const int r = (wave * LOADS + i) * RPL + lr;
        int ck, cv;
        chunks(r, &ck, &cv);
        ko[i] = (uint32_t)r * a.ks * 2 + (uint32_t)ck * 16;
        vo[i] = (uint32_t)r * a.vs * 2 + (uint32_t)cv * 16;
    }
    auto load = [&](auto buf, int it) {
        constexpr bool B = decltype(buf)::value;
        const int key0 = T.key_tile(it) * PR_KEYS;
        const uint8_t* kt = (const uint8_t*)(kg + (size_t)(uint32_t)key0 * a.ks);
        const uint8_t* vt = (const uint8_t*)(vg + (size_t)(uint32_t)key0 * a.vs);
        short *sk = B ? sk1 : sk0, *sv = B ? sv1 : sv0;
        if (near && key0 + PR_KEYS <= nk) {
#pragma unroll
            for (int i = 0; i < LOADS; i++) {
                const int at = (wave * LOADS + i) * 64 * 8;
                __builtin_amdgcn_global_load_lds((gvoid*)(kt + ko[i]), (lvoid*)&sk[at], 16, 0, 0);
                __builtin_amdgcn_global_load_lds((gvoid*)(vt + vo[i]), (lvoid*)&sv[at], 16, 0, 0);
            }
            return;
        }
        const int left = nk - 1 - key0;          // (rows past the end: the last one, masked)
        for (int i = 0; i < LOADS; i++) {
            const int r = (wave * LOADS + i) * RPL + lr, at = (wave * LOADS + i) * 64 * 8;
            int ck, cv;
            chunks(r, &ck, &cv);
            const size_t kr = (size_t)(uint32_t)min(r, left);
            __builtin_amdgcn_global_load_lds((gvoid*)(kt + kr * a.ks * 2 + ck * 16), (lvoid*)&sk[at], 16, 0, 0);
            __builtin_amdgcn_global_load_lds((gvoid*)(vt + kr * a.vs * 2 + cv * 16), (lvoid*)&sv[at], 16, 0, 0);
        }
    };

    f16v o[DT];
#pragma unroll
    for (int t = 0; t < DT; t++) o[t] = (f16v)0.0f;
    float m = -INFINITY, l = 0.0f;

    // one tile; MASKED: some rows do not see all of it
    auto body = [&](auto masked, auto buf, int key0) {
        constexpr bool MASKED = decltype(masked)::value, B = decltype(buf)::value;
        const short* sk = B ? sk1 : sk0;
        const short* sv = B ? sv1 : sv0;
        f16v s[G];
#pragma unroll
        for (int g = 0; g < G; g++) s[g] = (f16v)0.0f;
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int g = 0; g < G; g++) {
                if (!EXACT && c * 16 >= (int)a.dim) break;   // (no dims: zeros would meet another chunk's infinities)
                const s8v kf = *(const s8v*)&sk[(part + g * 32 + row) * DP + k_place<DP>(row, c * 2 + half) * 8];
                s[g] = mfma32<BF>(kf, qf[c], s[g]);
            }
        if constexpr (MASKED) mask_scores(s, a, nk, hi, lo, key0 + part, half);
        const float ms = new_maximum<BF>(s, a.scale_log2, BF ? a.above : FP16_ABOVE, m, l, o);
        s8v pf[2 * G];
        float l1 = 0.0f;
#pragma unroll
        for (int g = 0; g < G; g++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                float x[8];
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] = exp2_fast(__builtin_fmaf(s[g][8 * h + i], a.scale_log2, -ms));
                pf[g * 2 + h] = pack8<BF>(x);
                if (h) l = sum8<BF>(pf[g * 2 + h], l);
                else l1 = sum8<BF>(pf[g * 2 + h], l1);
            }
        l += l1;
        // V^T of 16 keys (a lane's 8 are 4 half .. + 3 and 8 + 4 half .. + 3) and 32 dims
        auto v_operand = [&](int gh, int t) {
            const int r = part + gh * 16 + 4 * half + (lane & 15) / 4;
            const int c = t * 4 + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
            const short* vp = &sv[r * DP + v_place<DP>(r, c) * 8 + (lane & 1) * 4];
            const s4v x0 = lds_read_tr(vp), x1 = lds_read_tr(vp + 8 * DP);
            return __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7);
        };
        s8v vf[2][DT];
#pragma unroll
        for (int t = 0; t < DT; t++) vf[0][t] = v_operand(0, t);
#pragma unroll
        for (int gh = 0; gh < 2 * G; gh++) {
            if (gh + 1 < 2 * G)
#pragma unroll
                for (int t = 0; t < DT; t++) vf[(gh + 1) & 1][t] = v_operand(gh + 1, t);
#pragma unroll
            for (int t = 0; t < DT; t++) o[t] = mfma32<BF>(vf[gh & 1][t], pf[gh], o[t]);
        }
    };
    // A tile that some rows see in part: weights of zero must not meet
    // infinities, so V's values are looked through first (any of them times zero
    // is a NaN).  Those that are not finite reach the rows that see them,
    // whatever their weight, and the products find zeros in their places.
    auto clean = [&](auto buf, int it, int key0) {
        constexpr bool B = decltype(buf)::value;
        short* sv = B ? sv1 : sv0;
        float z = 0.0f;
#pragma unroll
        for (int i = 0; i < LOADS; i++) z = sum8<BF>(*(const s8v*)&sv[((wave * LOADS + i) * 64 + lane) * 8], z, 0.0f);
        if (z != z) s_odd = it;
        __syncthreads();
        if (s_odd != it) return;
        for (int r = 0; r < PR_KEYS; r++) {
            const int key = key0 + r;
            if (key >= nk || !key_visible(key, hi, lo, a.sink) || (SPLIT == 2 && wave >= 2)) continue;
#pragma unroll
            for (int t = 0; t < DT; t++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int d = t * 32 + 8 * (i / 4) + 4 * half + i % 4;
                    const short w = sv[r * DP + v_place<DP>(r, d / 8) * 8 + d % 8];
                    if (not_finite<BF>(w)) o[t][i] += to_float<ACT>(w);
                }
        }
        __syncthreads();
        for (int i = 0; i < LOADS; i++) {
            s8v* x = (s8v*)&sv[((wave * LOADS + i) * 64 + lane) * 8];
            *x = finite_or_zero<BF>(*x);
        }
        __syncthreads();
    };
    // before a tile: it is whole in LDS, and nobody reads the one before it
    auto turn = [&] {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    };
    constexpr std::false_type no{};
    constexpr std::true_type yes{};

    if (tid == 0) s_odd = -1;
    if (T.tiles) load(no, 0);
    int it = 0;
    for (; it + 1 < T.n_whole; it += 2) {
        turn();
        load(yes, it + 1);
        body(no, no, 0);
        turn();
        if (it + 2 < T.tiles) load(no, it + 2);
        body(no, yes, 0);
    }
    for (; it < T.tiles; it += 2) {                // (at most one whole tile among these)
        int key0 = T.key_tile(it) * PR_KEYS;
        turn();
        if (it + 1 < T.tiles) load(yes, it + 1);
        clean(no, it, key0);
        if (T.some(a, key0, wave)) body(yes, no, key0);
        if (it + 1 >= T.tiles) break;
        key0 = T.key_tile(it + 1) * PR_KEYS;
        turn();
        if (it + 2 < T.tiles) load(no, it + 2);
        clean(yes, it + 1, key0);
        if (T.some(a, key0, wave)) body(yes, yes, key0);
    }

    if constexpr (SPLIT == 2) {
        static_assert(DT / 2 * 8192 <= sizeof(sk0) && 2048 <= sizeof(sv1), "the halves' exchange fits the tiles");
        join_halves(wave, m, l, o, sk0, sk1, sv1);
        if (wave >= 2) return;
        if (a.parts > 1) return store_part<EXACT>(a, T, my, half, m, l, o);
    } else {
        l = sum32(l);
        __syncthreads();                         // nobody reads V any more
    }
    // rows go out whole, 16 bytes a lane, by way of LDS (8 bytes of 32 rows at a
    // time take 6 us more of 57 for 24 packed prompts)
    bool none;
    const float f = row_factor(a, T, my, l, &none);
    short* st = (wave < 2 ? sv0 : sv1) + (wave & 1) * 32 * DP;
#pragma unroll
    for (int n = 0; n < DT; n++)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            float x[4];
#pragma unroll
            for (int j = 0; j < 4; j++) x[j] = none ? 0.0f : o[n][i + j] * f;
            store4<ACT>(st + row * DP + k_place<DP>(row, n * 4 + i / 4) * 8 + 4 * half, x);
        }
    __builtin_amdgcn_wave_barrier();
    short* op = (short*)a.out + (size_t)T.head * a.dim + lc * 8;
#pragma unroll
    for (int i = 0; i < 32 / RPL; i++) {
        const int r = i * RPL + lr, at = my - row + r;
        if (at < T.nq && (EXACT || lc * 8 < (int)a.dim))
            *(s8v*)(op + (size_t)(T.q0 + (uint32_t)at) * a.os) = *(const s8v*)&st[r * DP + k_place<DP>(r, lc) * 8];
    }
}

}  // namespace pf

// ================================================================== host

pf_status attn_desc_check(pf_ctx* c, const pf_attn_desc* d, AttnShape* s) {
    if (d->type != PF_TYPE_F32 && d->type != PF_TYPE_F16 && d->type != PF_TYPE_BF16)
        return fail(c, PF_ERR_ARG, "attention: type is PF_TYPE_F32, F16 or BF16");
    if (!d->n_heads || !d->n_kv_heads || d->n_heads % d->n_kv_heads || d->n_heads > 65535)
        return fail(c, PF_ERR_ARG, "attention: n_heads is a multiple of n_kv_heads");
    if (!d->head_dim || d->head_dim % 16 || d->head_dim > 128)
        return fail(c, PF_ERR_UNSUPPORTED, "attention: head_dim is a multiple of 16 up to 128");
    if (!std::isfinite(d->scale) || d->scale < 0.0f) return fail(c, PF_ERR_ARG, "attention: scale is 0 or positive");
    s->window = std::min(d->window, SEQ_ROWS);
    s->sink = std::min(d->sink, SEQ_ROWS);
    const uint64_t q = (uint64_t)d->n_heads * d->head_dim, k = (uint64_t)d->n_kv_heads * d->head_dim;
    const uint32_t per16 = d->type == PF_TYPE_F32 ? 4 : 8;
    const uint32_t given[4] = {d->q_stride, d->k_stride, d->v_stride, d->o_stride};
    uint32_t* out[4] = {&s->qs, &s->ks, &s->vs, &s->os};
    for (int i = 0; i < 4; i++) {
        const uint64_t least = i == 1 || i == 2 ? k : q, st = given[i] ? given[i] : least;
        if (st < least || st > 0xFFFFFFFFu || st % per16)
            return fail(c, PF_ERR_ARG, "attention: strides hold every head and are multiples of 16 bytes");
        *out[i] = (uint32_t)st;
    }
    s->scale_log2 = (d->scale == 0.0f ? 1.0f / std::sqrt((float)d->head_dim) : d->scale) * LOG2E;
    if (!std::isfinite(s->scale_log2)) return fail(c, PF_ERR_ARG, "attention: scale is below 2^127");
    return PF_OK;
}

template <int ACT, int DP, bool EXACT, int SPLIT>
static void prompt_one(hipStream_t st, const PromptArgs& a) {
    const uint32_t units = prompt_units(a.tiles, a.n_heads / a.group, a.group);
    if constexpr (ACT == PF_TYPE_F32)
        hipLaunchKernelGGL((k_prompt_attn32<DP, EXACT, SPLIT>), dim3(units, a.parts), dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((k_prompt_attn16<ACT, DP, EXACT, SPLIT>), dim3(units, a.parts), dim3(256), 0, st, a);
}

template <int ACT, int DP, bool EXACT>
static void prompt_rows(hipStream_t st, uint32_t rows, const PromptArgs& a) {
    if (rows == 128) prompt_one<ACT, DP, EXACT, 1>(st, a);
    else prompt_one<ACT, DP, EXACT, 2>(st, a);
}

template <int ACT>
static void prompt_dim(hipStream_t st, uint32_t rows, const PromptArgs& a) {
    if (a.dim == 128) prompt_rows<ACT, 128, true>(st, rows, a);
    else if (a.dim == 64) prompt_rows<ACT, 64, true>(st, rows, a);
    else if (a.dim < 64) prompt_rows<ACT, 64, false>(st, rows, a);
    else prompt_rows<ACT, 128, false>(st, rows, a);
}

// The parts that the keys are cut in, where 64-row workgroups are few and some
// see many key tiles: as many as fill the compute units with at least four
// tiles each (two of fp32 rows), where the longest workgroup's tiles are fewer
// then, with the join: six tiles' time (two) and what its rows add.  64 bf16
// rows after 2000 cached, 16 heads of 128 over 4: 34 us whole, 18.5 cut; 8000
// rows of one head of 64: 70 and 32; 1000 of 16 heads: 20.4, and 27.9 cut in
// two; 1000 fp32 rows of 12 heads of 64: 18.5 and 16.3.
static uint32_t prompt_parts(const pf_attn_desc* d, const AttnShape& s, const uint32_t* q_lens, const uint32_t* k_lens,
                             uint32_t n_seq, uint32_t full) {
    uint64_t units = 0, keys = 0;
    for (uint32_t i = 0; i < n_seq; i++) {
        if (!q_lens[i]) continue;
        units += (uint64_t)((q_lens[i] + 63) / 64) * d->n_heads;
        uint64_t seen = k_lens[i];
        if (s.window) seen = std::min<uint64_t>(seen, (uint64_t)s.window + std::min(q_lens[i], 64u) + s.sink);
        keys = std::max(keys, seen);
    }
    const uint64_t tiles = (keys + PR_KEYS - 1) / PR_KEYS;
    const bool wide = d->type == PF_TYPE_F32;
    const uint64_t parts = std::min<uint64_t>({full / units, tiles / (wide ? 2 : 4), PR_MOST_PARTS});
    if (parts < 2 || (tiles + parts - 1) / parts + (wide ? 2 : 6) + parts * units / 128 >= tiles) return 1;
    return (uint32_t)parts;
}

// 128 query rows a workgroup, or 64 where those would not fill the compute
// units (two workgroups each; one of fp32 rows of over 64 dims).  One prompt of
// 1000 bf16 rows, 16 heads of 128: 21 us instead of 27; 16 prompts of up to 300:
// 23.0 instead of 20.2, where 128 rows make 528 workgroups
struct PromptPlan {
    uint32_t rows, parts;
};
static PromptPlan prompt_plan(const pf_attn_desc* d, const AttnShape& s, const uint32_t* q_lens, const uint32_t* k_lens,
                              uint32_t n_seq) {
    uint64_t units = 0;
    for (uint32_t i = 0; i < n_seq; i++) units += (uint64_t)((q_lens[i] + 127) / 128) * d->n_heads;
    const uint32_t full = PR_CUS * (d->type == PF_TYPE_F32 && d->head_dim > 64 ? 1 : 2);
    if (units >= full) return {128, 1};
    return {64, prompt_parts(d, s, q_lens, k_lens, n_seq, full)};
}
extern "C" pf_status pf_test_prompt_plan(const pf_attn_desc* d, const uint32_t* q_lens, const uint32_t* k_lens,
                                         uint32_t n_seq, uint32_t* rows, uint32_t* parts) {
    AttnShape s;
    if (pf_status st = attn_desc_check(nullptr, d, &s)) return st;
    const PromptPlan plan = prompt_plan(d, s, q_lens, k_lens, n_seq);
    *rows = plan.rows;
    *parts = plan.parts;
    return PF_OK;
}

extern "C" pf_status pf_prompt_attention(pf_ctx* c, const pf_attn_desc* d, const void* q, const void* k, const void* v,
                                         void* out, const uint32_t* q_lens, const uint32_t* k_lens, uint32_t n_seq) {
    if (!c || !d || (n_seq && !q_lens)) return PF_ERR_ARG;
    AttnShape s;
    if (pf_status st = attn_desc_check(c, d, &s)) return st;
    if (!k_lens) k_lens = q_lens;
    uint64_t nq = 0, nk = 0;
    uint32_t longest = 0;
    for (uint32_t i = 0; i < n_seq; i++) {
        if (q_lens[i] > SEQ_ROWS || k_lens[i] > SEQ_ROWS) return fail(c, PF_ERR_UNSUPPORTED, "attention: a sequence of over 2^30 rows");
        nq += q_lens[i];
        nk += k_lens[i];
        longest = std::max(longest, k_lens[i]);
    }
    if (!nq) return PF_OK;
    // (a grid has fewer than 2^32 threads)
    if ((nq / 64 + n_seq) * d->n_heads > PR_MOST_UNITS) return fail(c, PF_ERR_UNSUPPORTED, "attention: too many rows at once");
    if (nq > 0x7FFFFFFFu || nk > 0x7FFFFFFFu) return fail(c, PF_ERR_UNSUPPORTED, "attention: over 2^31 rows in all");
    if (!q || !out || (nk && (!k || !v))) return fail(c, PF_ERR_ARG, "attention: a buffer is NULL");
    if (!aligned16(q) || !aligned16(out) || !aligned16(k) || !aligned16(v))
        return fail(c, PF_ERR_ARG, "attention: buffers start on 16 bytes");
    const size_t es = d->type == PF_TYPE_F32 ? 4 : 2;
    const size_t qw = (size_t)d->n_heads * d->head_dim, kw = (size_t)d->n_kv_heads * d->head_dim;
    const size_t ob = ((nq - 1) * s.os + qw) * es;
    if (overlaps(out, ob, q, ((nq - 1) * s.qs + qw) * es) ||
        (nk && (overlaps(out, ob, k, ((nk - 1) * s.ks + kw) * es) || overlaps(out, ob, v, ((nk - 1) * s.vs + kw) * es))))
        return fail(c, PF_ERR_ARG, "attention: out overlaps an input");
    DeviceScope on(c);
    PromptArgs a{};
    a.q = q; a.k = k; a.v = v; a.out = out;
    a.n_heads = d->n_heads; a.group = d->n_heads / d->n_kv_heads; a.dim = d->head_dim;
    a.qs = s.qs; a.ks = s.ks; a.vs = s.vs; a.os = s.os;
    a.causal = d->causal != 0; a.window = (int32_t)s.window; a.sink = (int32_t)s.sink;
    a.scale_log2 = s.scale_log2;
    a.above = (float)keys_shift(longest);
    a.down = std::ldexp(1.0f, -keys_shift(longest));
    a.rows = (uint32_t)nq;
    const PromptPlan plan = prompt_plan(d, s, q_lens, k_lens, n_seq);
    const uint32_t rows = plan.rows;
    a.parts = plan.parts;
    if (a.parts > 1) {
        const size_t n = (size_t)a.parts * a.rows * a.n_heads;
        void* ws = nullptr;
        if (pf_status st = ctx_scratch(c, n * (a.dim + 2) * 4, &ws)) return st;
        a.ws_o = (float*)ws;
        a.ws_ml = a.ws_o + n * a.dim;
    }
    uint32_t qa = 0, ka = 0;
    for (uint32_t b = 0; b < n_seq;) {
        a.n_seq = 0;
        for (; b < n_seq && a.n_seq < PR_SEQS; b++) {
            if (q_lens[b]) a.seq[a.n_seq++] = {qa, q_lens[b], ka, k_lens[b]};
            qa += q_lens[b];
            ka += k_lens[b];
        }
        // Tiles are taken from the last: the sequences with the most keys go first, so
        // that short ones fill the end (10 prompts of up to 1000 fp32 rows, 12 heads of
        // 64: 79 us in the order given, 66 so).  All sequences' last tiles first, then
        // the ones before, balances more (62) but parts the tiles that share keys in
        // L2 (64 prompts of up to 2000 bf16 rows, 16 heads of 128: 660 -> 710)
        std::sort(a.seq, a.seq + a.n_seq, [](const PromptSeq& x, const PromptSeq& y) { return x.nk < y.nk; });
        uint32_t tiles = 0;
        for (uint32_t i = 0; i < a.n_seq; i++) {
            a.tile0[i] = tiles;
            tiles += (a.seq[i].nq + rows - 1) / rows;
        }
        if (!tiles) continue;
        a.tiles = tiles;
        switch (d->type) {
            case PF_TYPE_F32: prompt_dim<PF_TYPE_F32>(c->stream, rows, a); break;
            case PF_TYPE_F16: prompt_dim<PF_TYPE_F16>(c->stream, rows, a); break;
            default: prompt_dim<PF_TYPE_BF16>(c->stream, rows, a); break;
        }
        PF_LAUNCHED(c);
    }
    if (a.parts > 1) {
        const dim3 grid((uint32_t)((nq * a.n_heads + 7) / 8));
        if (d->type == PF_TYPE_F32) hipLaunchKernelGGL(k_prompt_join<PF_TYPE_F32>, grid, dim3(256), 0, c->stream, a);
        else if (d->type == PF_TYPE_F16) hipLaunchKernelGGL(k_prompt_join<PF_TYPE_F16>, grid, dim3(256), 0, c->stream, a);
        else hipLaunchKernelGGL(k_prompt_join<PF_TYPE_BF16>, grid, dim3(256), 0, c->stream, a);
        PF_LAUNCHED(c);
    }
    return PF_OK;
}
