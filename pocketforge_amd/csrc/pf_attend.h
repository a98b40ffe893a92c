// Shared by the attention kernels over prompts (pf_prompt.hip) and over paged
// caches (pf_paged.hip): 16-bit operands of the gfx950 matrix core, fp32 rows
// as three bf16 pieces, and conversions.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/pf_gpu.h"

namespace pf {

typedef short s4v __attribute__((ext_vector_type(4)));
typedef short s8v __attribute__((ext_vector_type(8)));
typedef float f4v __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef uint32_t u4v __attribute__((ext_vector_type(4)));
typedef uint32_t u2v __attribute__((ext_vector_type(2)));
typedef __bf16 b8v __attribute__((ext_vector_type(8)));
typedef __bf16 b4v __attribute__((ext_vector_type(4)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef _Float16 h4v __attribute__((ext_vector_type(4)));

constexpr float LOG2E = 1.4426950408889634f;

// Operands are fp16 for fp16 rows, bf16 otherwise.  fp32 rows become three
// bf16 pieces (split3), the second at most 2^-8 and the third 2^-16 of the
// value: a product of two such values is the six piece products that are not
// below 2^-16 of it, and what is left out is below 2^-23 of it, with either
// sign.  Over rows that bf16 holds exactly (a bf16 or int8 cache) the three
// products are the whole product.
template <int ACT> constexpr bool op_bf = ACT != PF_TYPE_F16;
template <int ACT> constexpr int op_pieces = ACT == PF_TYPE_F32 ? 3 : 1;
// Weights over a cache are two pieces of 16-bit rows' type: the matrix core is
// idle there, and a weight rounded once would add as much error as the result's
// own rounding.
template <int ACT> constexpr int weight_pieces = ACT == PF_TYPE_F32 ? 3 : 2;
template <int ACT> constexpr int act_size = ACT == PF_TYPE_F32 ? 4 : 2;

template <bool BF>
__device__ __forceinline__ f4v mfma16(s8v a, s8v b, f4v c) {
    if constexpr (BF)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8v, a), __builtin_bit_cast(b8v, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8v, a), __builtin_bit_cast(h8v, b), c, 0, 0, 0);
}
template <bool BF>
__device__ __forceinline__ f16v mfma32(s8v a, s8v b, f16v c) {
    if constexpr (BF)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8v, a), __builtin_bit_cast(b8v, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8v, a), __builtin_bit_cast(h8v, b), c, 0, 0, 0);
}

// Eight floats as 16-bit values, rounded to nearest even.
template <bool BF>
__device__ __forceinline__ s8v pack8(const float (&x)[8]) {
    if constexpr (BF) {
        b8v r;
#pragma unroll
        for (int i = 0; i < 8; i++) r[i] = (__bf16)x[i];
        return __builtin_bit_cast(s8v, r);
    } else {
        h8v r;
#pragma unroll
        for (int i = 0; i < 8; i++) r[i] = (_Float16)x[i];
        return __builtin_bit_cast(s8v, r);
    }
}

template <int T>
__device__ __forceinline__ float to_float(short bits) {
    if constexpr (T == PF_TYPE_F16) return (float)__builtin_bit_cast(_Float16, bits);
    else return __builtin_bit_cast(float, (uint32_t)(uint16_t)bits << 16);
}

// x = hi + mid + lo exactly, each piece the bf16 nearest to what is left (8
// significant bits each, the remainders signed; below 2^-126 the last bits are
// lost).  An infinity leaves a NaN.
__device__ __forceinline__ void split3(const float (&x)[8], s8v (&out)[3]) {
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; i++) r[i] = x[i];
#pragma unroll
    for (int n = 0; n < 3; n++) {
        out[n] = pack8<true>(r);
        if (n < 2)
#pragma unroll
            for (int i = 0; i < 8; i++) r[i] -= __builtin_bit_cast(float, (uint32_t)(uint16_t)out[n][i] << 16);
    }
}

// Eight floats as NP operand pieces.
template <bool BF, int NP>
__device__ __forceinline__ void pieces(const float (&x)[8], s8v (&out)[NP]) {
    if constexpr (NP == 3) {
        split3(x, out);
    } else {
        out[0] = pack8<BF>(x);
        if constexpr (NP == 2) {
            float r[8];
#pragma unroll
            for (int i = 0; i < 8; i++) r[i] = x[i] - to_float<BF ? PF_TYPE_BF16 : PF_TYPE_F16>(out[0][i]);
            out[1] = pack8<BF>(r);
        }
    }
}

// Eight int8 codes (two words) as floats.
__device__ __forceinline__ void codes8(uint32_t w0, uint32_t w1, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        x[i] = (float)(int32_t)(int8_t)(w0 >> (8 * i));
        x[4 + i] = (float)(int32_t)(int8_t)(w1 >> (8 * i));
    }
}

// Eight values of a row of type T at p (16-byte aligned).
template <int T>
__device__ __forceinline__ void load8(const void* p, float (&x)[8]) {
    if constexpr (T == PF_TYPE_F32) {
        const f4v a = ((const f4v*)p)[0], b = ((const f4v*)p)[1];
#pragma unroll
        for (int i = 0; i < 4; i++) { x[i] = a[i]; x[4 + i] = b[i]; }
    } else {
        const s8v a = *(const s8v*)p;
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = to_float<T>(a[i]);
    }
}

// Four values to a row of type T.
template <int T>
__device__ __forceinline__ void store4(void* p, const float (&x)[4]) {
    if constexpr (T == PF_TYPE_F32) {
        f4v r = {x[0], x[1], x[2], x[3]};
        *(f4v*)p = r;
    } else if constexpr (T == PF_TYPE_BF16) {
        b4v r;
#pragma unroll
        for (int i = 0; i < 4; i++) r[i] = (__bf16)x[i];
        *(b4v*)p = r;
    } else {
        h4v r;
#pragma unroll
        for (int i = 0; i < 4; i++) r[i] = (_Float16)x[i];
        *(h4v*)p = r;
    }
}

// Whether a 16-bit value is an infinity or a NaN.
template <bool BF>
__device__ __forceinline__ bool not_finite(short v) {
    const uint16_t mask = BF ? 0x7F80u : 0x7C00u;
    return ((uint16_t)v & mask) == mask;
}
template <bool BF>
__device__ __forceinline__ s8v finite_or_zero(s8v v) {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = not_finite<BF>(v[i]) ? (short)0 : v[i];
    return v;
}

// l plus f times the eight values of an operand.  With f = 1 a row's sum of
// weights as the products take them, so that they sum to one whatever they were
// rounded to; with f = 0 a NaN if one of the values is not finite.
template <bool BF>
__device__ __forceinline__ float sum8(s8v v, float l, float f = 1.0f) {
    const u4v w = __builtin_bit_cast(u4v, v);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t two = w[i];
        if constexpr (BF) {
            typedef __bf16 b2v __attribute__((ext_vector_type(2)));
            const b2v one = {(__bf16)f, (__bf16)f};
            l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2v, two), one, l, false);
        } else {
            typedef _Float16 h2v __attribute__((ext_vector_type(2)));
            const h2v one = {(_Float16)f, (_Float16)f};
            l = __builtin_amdgcn_fdot2(__builtin_bit_cast(h2v, two), one, l, false);
        }
    }
    return l;
}

// Transposing LDS read: the 16 lanes of a group give the addresses of the 16
// four-value chunks of a 4 x 16 tile, row by row; lane i gets column i.
__device__ __forceinline__ s4v lds_read_tr(const short* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4v*)p);
}

// The sum and the maximum over the lanes that differ in bit 4 and bit 5 (16 x
// 16 tiles) or bit 5 (32 x 32 tiles) of their number; all of them get it.
__device__ __forceinline__ float max32(float x) { return fmaxf(x, __shfl_xor(x, 32)); }
__device__ __forceinline__ float sum32(float x) { return x + __shfl_xor(x, 32); }
__device__ __forceinline__ float max16(float x) { x = fmaxf(x, __shfl_xor(x, 16)); return fmaxf(x, __shfl_xor(x, 32)); }
__device__ __forceinline__ float sum16(float x) { x += __shfl_xor(x, 16); return x + __shfl_xor(x, 32); }

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Softmax runs in base 2 (scores times log2 e).  The running maximum m moves only
// when a score exceeds it by more than m_slack, so that most tiles need no
// reduction over lanes and no rescaling of the output.  Outputs are summed as
// they come and divided by the sum of the weights at the end, so the weights are
// held at a distance from one that keeps those sums in fp32's range:
//  * fp32 rows: weights 2^(s - m), which reach 2^m_slack, times 2^-K with K =
//    keys_shift of the call's longest sequence.  2^K is over 2^m_slack times the
//    keys, so values up to the type's largest do not overflow; what is lost below
//    is less than 2^-126+K for each key.
//  * bf16 operands of 16-bit rows: m is held K above the scores' own maximum,
//    which is the same without the product, but rounds s - m to 2^-19.
//  * fp16 operands cannot overflow, but their smallest step is 2^-24: m is held so
//    far below that the weights reach 2^15.  What rounding takes of one is then
//    below 2^-36 of the largest weight (2^-25 of it if they were held against 1,
//    and a thousand keys that weigh that little beside a sink key would vanish).
//    8192 fp16 rows, 16 heads of 128: 295 us with a slack of 4, 296 with 8
//    (2^-32), 299 with 2 (2^-38).
template <bool BF> constexpr float m_slack = BF ? 8.0f : 4.0f;
constexpr float FP16_ABOVE = m_slack<false> - 15.0f;
inline int keys_shift(uint32_t keys) { return (int)m_slack<true> + 1 + (keys ? 32 - __builtin_clz(keys) : 0); }

// Visibility of a key at position `pos` for a query whose last visible
// position is hi: the last `window` of the causal range start at lo.
__device__ __host__ __forceinline__ bool key_visible(int pos, int hi, int lo, int sink) {
    return (pos <= hi) & ((pos >= lo) | (pos < sink));
}

// x where `on` is all ones, y where it is 0.
__device__ __forceinline__ float bits_or(float x, float y, int on) {
    return __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, x) & (uint32_t)on) |
                                         (__builtin_bit_cast(uint32_t, y) & ~(uint32_t)on));
}

// A word with its first n bits set (none for n <= 0, all from 64 on).
__device__ __forceinline__ uint64_t first_bits(int n) {
    return n <= 0 ? 0 : ~0ull >> (64 - min(n, 64));
}

}  // namespace pf
