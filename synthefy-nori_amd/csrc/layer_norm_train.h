// What the forward and the backward kernels of the trainable LayerNorm share.
//
// Rows in registers. A group of G lanes owns a row and holds it as NV vectors of V elements a lane: vector
// i of lane l is at column (i * G + l) * V. V is 16 bytes of x, read and written at any alignment (global memory
// takes vectors at any byte); where a row is no whole number of vectors (RAGGED) its last one is moved back to
// end with the row, and the elements that it shares with the one before are left out of the sums (stored twice,
// the same value). G is 4, 8 or 16 (rows up to 128), 64 or 256 (a workgroup). Rows shorter than a vector are held an
// element a lane, rows too wide for registers are looped over.
#pragma once

#include <algorithm>
#include <type_traits>

#include "nori_common.h"

namespace nori_ln {

using namespace nori;

constexpr int kThreads = 256;

template <int DT>
using elem = std::conditional_t<DT == NORI_F32, uint32_t, uint16_t>;

// V elements as they lie in memory
template <int DT, int V>
struct Raw {
    elem<DT> e[V];
};

template <int DT, int V>
__device__ __forceinline__ Raw<DT, V> fetch(const void* p, int64_t i) {
    Raw<DT, V> r;
    __builtin_memcpy(&r, reinterpret_cast<const elem<DT>*>(p) + i, sizeof r);
    return r;
}

template <int DT, int V>
__device__ __forceinline__ void widen(const Raw<DT, V>& r, float (&v)[V]) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
        if constexpr (DT == NORI_F32) v[k] = __uint_as_float(r.e[k]);
        else v[k] = DT == NORI_F16 ? f16_to_f32(r.e[k]) : bf16_to_f32(r.e[k]);
    }
}

template <int DT, int V>
__device__ __forceinline__ void store(void* p, int64_t i, const float (&v)[V]) {
    Raw<DT, V> r;
#pragma unroll
    for (int k = 0; k < V; ++k) {
        if constexpr (DT == NORI_F32) r.e[k] = __float_as_uint(v[k]);
        else r.e[k] = DT == NORI_F16 ? f32_to_f16(v[k]) : f32_to_bf16(v[k]);
    }
    __builtin_memcpy(reinterpret_cast<elem<DT>*>(p) + i, &r, sizeof r);
}

// vector i of a lane: its column, and how many of its elements the vector before it holds too
template <int V, int G, bool RAGGED>
__device__ __forceinline__ int column(int i, int lane, int cols, int& shared) {
    const int c = (i * G + lane) * V;
    shared = 0;
    if (RAGGED && c < cols && c + V > cols) {
        shared = c + V - cols;
        return cols - V;
    }
    return c;
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
    if (!p) {
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = none;
    } else if (dt == NORI_F32) {
        widen<NORI_F32, V>(fetch<NORI_F32, V>(p, i), v);
    } else if (dt == NORI_F16) {
        widen<NORI_F16, V>(fetch<NORI_F16, V>(p, i), v);
    } else {
        widen<NORI_BF16, V>(fetch<NORI_BF16, V>(p, i), v);
    }
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

// The kernel for rows of `cols`: calls go(V, G, NV, RAGGED) with integral constants, or loop() past what registers
// hold. A row goes to the fewest lanes that hold it in 32 values each, a workgroup to the ones that a wavefront
// does not.
template <int DT, class Go, class Loop>
void choose(int cols, Go go, Loop loop) {
    constexpr int VW = DT == NORI_F32 ? 4 : 8;
#define NORI_LN_CALL(V, G, NV, R) \
    go(std::integral_constant<int, V>{}, std::integral_constant<int, G>{}, std::integral_constant<int, NV>{}, \
       std::integral_constant<bool, R>{})
#define NORI_LN_TRY(G, NV) \
    if (cols <= VW * (G) * (NV)) return cols % VW ? NORI_LN_CALL(VW, G, NV, true) : NORI_LN_CALL(VW, G, NV, false)
    if (cols < VW) return NORI_LN_CALL(1, 8, 1, false);
    NORI_LN_TRY(4, 1);
    NORI_LN_TRY(8, 1);
    if constexpr (VW == 8) {
        NORI_LN_TRY(16, 1);
        NORI_LN_TRY(64, 1);
        NORI_LN_TRY(64, 2);
        NORI_LN_TRY(64, 3);
        NORI_LN_TRY(64, 4);
        NORI_LN_TRY(256, 2);
        NORI_LN_TRY(256, 4);
    } else {
        NORI_LN_TRY(16, 1);
        NORI_LN_TRY(16, 2);
        NORI_LN_TRY(64, 1);
        NORI_LN_TRY(64, 2);
        NORI_LN_TRY(64, 3);
        NORI_LN_TRY(64, 4);
        NORI_LN_TRY(64, 6);
        NORI_LN_TRY(64, 8);
        NORI_LN_TRY(256, 4);
        NORI_LN_TRY(256, 8);
    }
#undef NORI_LN_TRY
#undef NORI_LN_CALL
    loop();
}

inline bool is_float(int dt) { return dt == NORI_F32 || dt == NORI_F16 || dt == NORI_BF16; }

inline int check(const char* what, int64_t rows, int32_t cols, int x_dtype, int y_dtype, int64_t xs, int64_t ys) {
    if (!is_float(x_dtype) || !is_float(y_dtype))
        return fail(NORI_ERR_UNSUPPORTED, "%s: unsupported dtypes %s and %s", what, dtype_name(x_dtype), dtype_name(y_dtype));
    if (rows < 0 || cols <= 0) return fail(NORI_ERR_INVALID, "%s: bad shape (%lld rows of %d)", what, (long long)rows, cols);
    if (cols > NORI_LAYER_NORM_MAX)
        return fail(NORI_ERR_UNSUPPORTED, "%s: rows of %d columns (up to %d)", what, cols, NORI_LAYER_NORM_MAX);
    if (xs < 0 || ys < 0) return fail(NORI_ERR_INVALID, "%s: negative row strides", what);
    return NORI_OK;
}

}  // namespace nori_ln
