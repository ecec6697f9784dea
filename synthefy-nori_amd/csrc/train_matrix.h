// The matrix instructions as the training kernels use them, alike for float16, bfloat16 and float32: products of 32 x 32
// results over 16 steps of a contraction, operands out of LDS tiles whose rows lie as in memory.
//
// v_mfma_f32_32x32x16 takes row (left) or column (right) lane % 32 and steps 8 (lane / 32) .. + 7 of either operand and
// leaves column lane % 32, rows 8 (i / 4) + 4 (lane / 32) + i % 4 in register i. In float32 the same operands go through eight
// v_mfma_f32_32x32x2, a step of either half-wave each.
#pragma once

#include "nori_common.h"

namespace nori {
namespace train {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// An operand of 16 steps of a contraction: 8 elements a lane.  kRows: rows of an attention tile that
// passes; kPad: elements between the rows of a tile in LDS. kBias: the power of two on probabilities in their 16-bit form.
template <int DT> struct El;
template <> struct El<NORI_F16> {
    using T = uint16_t;
    using Frag = f16x8;
    static constexpr int kRows = 64, kPad = 8;
    // p is below 2^-14, where float16 loses bits, for most keys of a long context: times 2^15 it keeps them to 2^-29,
    // and beside a running maximum, which p may pass by 2^kSlack, times 2^kTop to 2^-22
    static constexpr float kBias = 15.f, kTop = 8.f, kSlack = 7.f;
    static constexpr bool kScaled = true;
};
template <> struct El<NORI_BF16> {
    using T = uint16_t;
    using Frag = bf16x8;
    static constexpr int kRows = 64, kPad = 8;
    static constexpr float kBias = 0.f, kTop = 0.f, kSlack = 8.f;
    static constexpr bool kScaled = false;
};
template <> struct El<NORI_F32> {
    using T = float;
    struct Frag { float v[8]; };
    static constexpr int kRows = 32, kPad = 4;
    static constexpr float kBias = 0.f, kTop = 0.f, kSlack = 8.f;
    static constexpr bool kScaled = false;
};

// Element j of an operand.
__device__ __forceinline__ float& at(El<NORI_F32>::Frag& f, int j) { return f.v[j]; }
template <class V>
struct Element {
    V& f;
    int j;
    __device__ __forceinline__ operator float() const { return (float)f[j]; }
    __device__ __forceinline__ void operator=(float v) { f[j] = (__typeof__(f[0] + f[0]))v; }
};
__device__ __forceinline__ Element<f16x8> at(f16x8& f, int j) { return {f, j}; }
__device__ __forceinline__ Element<bf16x8> at(bf16x8& f, int j) { return {f, j}; }

__device__ __forceinline__ f32x16 mma(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma(const El<NORI_F32>::Frag& a, const El<NORI_F32>::Frag& b, f32x16 c) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[i], b.v[i], c, 0, 0, 0);
    return c;
}

// Value of lane l ^ 32.
__device__ __forceinline__ float other_half(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), true, false);
    return __uint_as_float((__lane_id() < 32) ? r[1] : r[0]);
}

// Left operand transposed: column `col` + lane % 32 of a tile of rows LS elements apart, its rows first + 4 h .. + 3 and
// first + 8 + 4 h .. + 3 in half-wave h, the order in which a product leaves its rows. ds_read_b64_tr_b16 gives lane i of 16
// element i % 4 of the 8 bytes that lanes i / 4 + 4 j point at, j = 0 .. 3: lanes 4 j .. 4 j + 3 point along row j.
template <int DT, int LS>
__device__ __forceinline__ typename El<DT>::Frag transposed(const typename El<DT>::T* tile, int first, int col, int lane) {
    if constexpr (DT == NORI_F32) {
        typename El<DT>::Frag f;
        const float* p = tile + (first + 4 * (lane >> 5)) * LS + col + (lane & 31);
#pragma unroll
        for (int j = 0; j < 8; ++j) f.v[j] = p[((j & 3) + 8 * (j >> 2)) * LS];
        return f;
    } else {
        const uint16_t* p = tile + (first + 4 * (lane >> 5) + ((lane & 15) >> 2)) * LS + col + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 8 * LS));
        typedef short s16x8 __attribute__((ext_vector_type(8)));
        const s16x8 both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        return __builtin_bit_cast(typename El<DT>::Frag, both);
    }
}

// Right operand of the contraction over a result's rows: registers 8 t .. 8 t + 7, rounded to the type (to nearest even).
template <int DT>
__device__ __forceinline__ typename El<DT>::Frag rounded(const float (&x)[16], int t) {
    typename El<DT>::Frag f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if constexpr (DT == NORI_F32) f.v[j] = x[8 * t + j];
        else if constexpr (DT == NORI_F16) f[j] = (_Float16)x[8 * t + j];
        else f[j] = (__bf16)x[8 * t + j];
    }
    return f;
}

}  // namespace train
}  // namespace nori
