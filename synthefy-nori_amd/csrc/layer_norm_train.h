// What the forward and the backward kernels of the trainable LayerNorm share.
//
// Rows in registers. A group of G lanes owns a row and holds it as NV vectors of V elements a lane: vector
// i of lane l is at column (i * G + l) * V. G is 16 (rows up to 128), 64 or 256 (a workgroup), V is 4
// where rows, strides and pointers keep vectors whole and 1 elsewhere. Rows too wide for that are looped over.
#pragma once

#include <algorithm>

#include "nori_common.h"

namespace nori_ln {

using namespace nori;

constexpr int kThreads = 256;

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

template <int DT, int V>
__device__ __forceinline__ void load(const void* p, int64_t i, float (&v)[V]) {
    if constexpr (V == 1) {
        v[0] = load_elem<DT>(p, i);
    } else if constexpr (DT == NORI_F32) {
        const f32x4 c = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(p) + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = c[k];
    } else {
        const u32x2 c = *reinterpret_cast<const u32x2*>(reinterpret_cast<const uint16_t*>(p) + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint16_t h = (uint16_t)(c[k >> 1] >> (16 * (k & 1)));
            v[k] = DT == NORI_F16 ? f16_to_f32(h) : bf16_to_f32(h);
        }
    }
}

template <int DT, int V>
__device__ __forceinline__ void store(void* p, int64_t i, const float (&v)[V]) {
    if constexpr (V == 1) {
        store_elem<DT>(p, i, v[0]);
    } else if constexpr (DT == NORI_F32) {
        *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(p) + i) = f32x4{v[0], v[1], v[2], v[3]};
    } else {
        u32x2 c;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const uint32_t lo = DT == NORI_F16 ? f32_to_f16(v[2 * k]) : f32_to_bf16(v[2 * k]);
            const uint32_t hi = DT == NORI_F16 ? f32_to_f16(v[2 * k + 1]) : f32_to_bf16(v[2 * k + 1]);
            c[k] = lo | (hi << 16);
        }
        *reinterpret_cast<u32x2*>(reinterpret_cast<uint16_t*>(p) + i) = c;
    }
}

// affine parameters, of a type known at run time; `none` where there are none
__device__ __forceinline__ float param(const void* p, int dt, int64_t i, float none) {
    if (!p) return none;
    if (dt == NORI_F32) return reinterpret_cast<const float*>(p)[i];
    const uint16_t v = reinterpret_cast<const uint16_t*>(p)[i];
    return dt == NORI_F16 ? f16_to_f32(v) : bf16_to_f32(v);
}

template <int V>
__device__ __forceinline__ void params(const void* p, int dt, int64_t i, float none, float (&v)[V]) {
    if (V == 4 && p && (uintptr_t)p % (dt == NORI_F32 ? 16 : 8) == 0) {
        if (dt == NORI_F32) load<NORI_F32, V>(p, i, v);
        else if (dt == NORI_F16) load<NORI_F16, V>(p, i, v);
        else load<NORI_BF16, V>(p, i, v);
        return;
    }
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = param(p, dt, i + k, none);
}

// The sums of a and b over the group's lanes, in every one of them. A workgroup's partial sums pass through
// `slots` (16 floats), whose halves take turns: one barrier a call.
template <int G>
__device__ __forceinline__ void group_sums(float& a, float& b, float* slots, int& turn) {
#pragma unroll
    for (int off = (G < 64 ? G : 64) / 2; off > 0; off >>= 1) {
        a += __shfl_xor(a, off, 64);
        b += __shfl_xor(b, off, 64);
    }
    if constexpr (G > 64) {
        float* s = slots + 8 * turn;
        turn ^= 1;
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) s[2 * wave] = a, s[2 * wave + 1] = b;
        __syncthreads();
        a = (s[0] + s[2]) + (s[4] + s[6]);
        b = (s[1] + s[3]) + (s[5] + s[7]);
    }
}

// the kernel for rows of `cols`: calls go(V, G, NV) with integral constants, or loop() past what registers hold
template <class Go, class Loop>
void choose(int cols, bool vectors, Go go, Loop loop) {
#define NORI_LN_TRY(V, G, NV) \
    if (cols <= (V) * (G) * (NV)) return go(std::integral_constant<int, V>{}, std::integral_constant<int, G>{}, std::integral_constant<int, NV>{})
    if (vectors) {
        NORI_LN_TRY(4, 16, 1);
        NORI_LN_TRY(4, 16, 2);
        NORI_LN_TRY(4, 64, 1);
        NORI_LN_TRY(4, 64, 2);
        NORI_LN_TRY(4, 64, 3);
        NORI_LN_TRY(4, 64, 4);
        NORI_LN_TRY(4, 64, 6);
        NORI_LN_TRY(4, 64, 8);
        NORI_LN_TRY(4, 256, 4);
        NORI_LN_TRY(4, 256, 8);
    } else {
        NORI_LN_TRY(1, 16, 4);
        NORI_LN_TRY(1, 64, 4);
        NORI_LN_TRY(1, 64, 8);
        NORI_LN_TRY(1, 64, 16);
        NORI_LN_TRY(1, 256, 8);
        NORI_LN_TRY(1, 256, 16);
    }
#undef NORI_LN_TRY
    loop();
}

inline bool is_float(int dt) { return dt == NORI_F32 || dt == NORI_F16 || dt == NORI_BF16; }

// whether rows of `cols` at `stride` from p are whole vectors of 4
inline bool whole4(const void* p, int dt, int cols, int64_t stride) {
    return cols % 4 == 0 && stride % 4 == 0 && (uintptr_t)p % (4 * dtype_size(dt)) == 0;
}

inline int check(const char* what, int64_t rows, int32_t cols, int x_dtype, int y_dtype, int64_t xs, int64_t ys) {
    if (!is_float(x_dtype) || !is_float(y_dtype))
        return fail(NORI_ERR_UNSUPPORTED, "%s: unsupported dtypes %s and %s", what, dtype_name(x_dtype), dtype_name(y_dtype));
    if (rows < 0 || cols <= 0) return fail(NORI_ERR_INVALID, "%s: bad shape (%lld rows of %d)", what, (long long)rows, cols);
    if (xs < 0 || ys < 0) return fail(NORI_ERR_INVALID, "%s: negative row strides", what);
    return NORI_OK;
}

}  // namespace nori_ln
