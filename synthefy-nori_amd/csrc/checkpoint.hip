// Activations kept in 8 bits for the backward pass: rows quantised in groups of 128 columns, and the SwiGLU gate with its
// gradient over gate and up kept so. One pass each, HBM-bound: 16 lanes hold a group, 8 elements each, in registers
// between the largest magnitude (DPP) and the codes.
//
// The code of x is the whole number nearest to x / s, ties to even, exactly: k = rint(x * (1 / s)) may be one off beside a
// half, and the remainder x - k s, which one fma gives without error there, says so. (Both terms are multiples of half
// the last place of s, and their difference is not above s: it has 24 bits.)
#include <math.h>

#include "layer_norm_train.h"

namespace {

using namespace nori;
using nori_ln::fetch;
using nori_ln::store;
using nori_ln::widen;

constexpr int kThreads = 256;
constexpr int kGroup = NORI_CHECKPOINT_GROUP, kLanes = 16, kEach = kGroup / kLanes;
constexpr int kItems = kThreads / kLanes;  // groups a workgroup

// 8 elements from column c of a row of cols, zeros past its end.
template <int DT>
__device__ __forceinline__ void load8(const void* p, int64_t row, int c, int cols, float (&v)[kEach]) {
    if (c + kEach <= cols) {
        widen<DT, kEach>(fetch<DT, kEach>(p, row + c), v);
    } else {
#pragma unroll
        for (int i = 0; i < kEach; ++i) v[i] = c + i < cols ? load_elem<DT>(p, row + c + i) : 0.f;
    }
}

template <int DT>
__device__ __forceinline__ void store8(void* p, int64_t row, int c, int cols, const float (&v)[kEach]) {
    if (c + kEach <= cols) {
        store<DT, kEach>(p, row + c, v);
    } else {
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (c + i < cols) store_elem<DT>(p, row + c + i, v[i]);
    }
}

// The largest of a value over 16 lanes (whole numbers: float magnitudes, NaN on top).
__device__ __forceinline__ uint32_t max16(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, false));  // row_ror:8
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xf, 0xf, false));
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xf, 0xf, false));
}

// The group's scale and this lane's codes.
__device__ __forceinline__ float quantize8(const float (&v)[kEach], uint64_t& codes) {
    uint32_t key = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) key = max(key, __float_as_uint(v[i]) & 0x7fffffffu);
    key = max16(key);
    const float s = key < 0x7f800000u ? __uint_as_float(key) / 127.0f : NAN;  // an infinity or NaN: NaN throughout
    const bool normal = s >= 0x1p-126f;
    const float y = normal ? 1.0f / s : 0.0f;
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        float k = rintf(v[i] * y);
        if (normal) {
            const float rest = fmaf(-k, s, v[i]), twice = 2.0f * fabsf(rest);
            if (twice > s || (twice == s && ((int)k & 1))) k += copysignf(1.0f, rest);
        } else if (s > 0.0f) {
            k = rintf(v[i] / s);  // a scale of few bits: quotients up to 190
        }
        k = fminf(fmaxf(k, -127.0f), 127.0f);
        w[i >> 2] |= ((uint32_t)(int)k & 0xffu) << (8 * (i & 3));
    }
    codes = (uint64_t)w[1] << 32 | w[0];
    return s;
}

__device__ __forceinline__ void restore8(const uint64_t codes, float s, float (&v)[kEach]) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) v[i] = (float)(int8_t)(codes >> (8 * i)) * s;
}

// Where a thread works: group `group` of row `row`, its 8 columns from `col`.
struct Item { int64_t row; int group, col; bool there; };
__device__ __forceinline__ Item item_of(int64_t rows, int groups) {
    const int64_t i = (int64_t)blockIdx.x * kItems + threadIdx.x / kLanes;
    Item it;
    it.row = i / groups;
    it.group = (int)(i - it.row * groups);
    it.col = it.group * kGroup + (threadIdx.x % kLanes) * kEach;
    it.there = it.row < rows;
    return it;
}

__host__ __device__ inline int code_stride(int cols) { return (cols + 15) / 16 * 16; }
inline int group_count(int cols) { return (cols + kGroup - 1) / kGroup; }

template <int DT>
__global__ __launch_bounds__(kThreads) void quantize_kernel(const void* x, int64_t rows, int cols, int64_t stride, int groups,
                                                            uint8_t* codes, float* scales) {
    const Item it = item_of(rows, groups);
    if (!it.there) return;  // (16 lanes alike)
    float v[kEach];
    load8<DT>(x, it.row * stride, it.col, cols, v);
    uint64_t w;
    const float s = quantize8(v, w);
    const int to = code_stride(cols);
    if (it.col < to) *reinterpret_cast<uint64_t*>(codes + it.row * to + it.col) = w;
    if (threadIdx.x % kLanes == 0) scales[it.row * groups + it.group] = s;
}

template <int DT, bool KEEP>
__global__ __launch_bounds__(kThreads) void silu_mul_forward_kernel(const void* gu, int64_t rows, int hidden, int64_t stride, int groups,
                                                                    void* y, uint8_t* codes, float* scales) {
    const Item it = item_of(rows, groups);
    if (!it.there) return;
    float g[kEach], u[kEach], o[kEach];
    load8<DT>(gu, it.row * stride, it.col, hidden, g);
    load8<DT>(gu, it.row * stride + hidden, it.col, hidden, u);
#pragma unroll
    for (int i = 0; i < kEach; ++i) o[i] = g[i] / (1.0f + expf(-g[i])) * u[i];
    store8<DT>(y, it.row * hidden, it.col, hidden, o);
    if constexpr (KEEP) {
        const int to = code_stride(hidden);
        uint64_t w[2];
        const float s[2] = {quantize8(g, w[0]), quantize8(u, w[1])};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int64_t at = j * rows + it.row;
            if (it.col < to) *reinterpret_cast<uint64_t*>(codes + at * to + it.col) = w[j];
            if (threadIdx.x % kLanes == 0) scales[at * groups + it.group] = s[j];
        }
    }
}

template <int DT>
__global__ __launch_bounds__(kThreads) void silu_mul_backward_kernel(const uint8_t* codes, const float* scales, int64_t rows, int hidden,
                                                                     int groups, const void* dy, int64_t stride, void* dgu) {
    const Item it = item_of(rows, groups);
    if (!it.there || it.col >= hidden) return;
    const int to = code_stride(hidden);
    float g[kEach], u[kEach], d[kEach];
    restore8(*reinterpret_cast<const uint64_t*>(codes + it.row * to + it.col), scales[it.row * groups + it.group], g);
    restore8(*reinterpret_cast<const uint64_t*>(codes + (rows + it.row) * to + it.col), scales[(rows + it.row) * groups + it.group], u);
    load8<DT>(dy, it.row * stride, it.col, hidden, d);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const float sig = 1.0f / (1.0f + expf(-g[i]));
        const float du = d[i] * g[i] * sig;
        g[i] = d[i] * u[i] * (sig * (1.0f + g[i] * (1.0f - sig)));
        u[i] = du;
    }
    store8<DT>(dgu, it.row * 2 * hidden, it.col, hidden, g);
    store8<DT>(dgu, it.row * 2 * hidden + hidden, it.col, hidden, u);
}

constexpr int kMostCols = 1 << 24;

int check(const char* what, int dtype, int64_t rows, int32_t cols, int64_t stride, int64_t width) {
    if (rows < 0 || cols < 1) return fail(NORI_ERR_INVALID, "%s: bad shape (%lld rows of %d)", what, (long long)rows, cols);
    if (dtype != NORI_F32 && dtype != NORI_F16 && dtype != NORI_BF16)
        return fail(NORI_ERR_UNSUPPORTED, "%s: unsupported dtype %s", what, dtype_name(dtype));
    if (cols > kMostCols || rows > (1LL << 40) / cols) return fail(NORI_ERR_UNSUPPORTED, "%s: too many elements", what);
    if (stride < 0 || (rows > 1 && stride != 0 && stride < width))
        return fail(NORI_ERR_INVALID, "%s: a row stride of %lld below rows of %lld", what, (long long)stride, (long long)width);
    if (!one_launch((rows * group_count(cols) + kItems - 1) / kItems, kThreads)) return fail(NORI_ERR_UNSUPPORTED, "%s: too many rows", what);
    return NORI_OK;
}

dim3 grid_of(int64_t rows, int groups) { return dim3((unsigned)((rows * groups + kItems - 1) / kItems)); }

}  // namespace

extern "C" int nori_checkpoint_quantize(const void* x, int dtype, int64_t rows, int32_t cols, int64_t x_row_stride, void* codes,
                                        float* scales, void* stream_v) {
    clear_error();
    if (int rc = check("checkpoint_quantize", dtype, rows, cols, x_row_stride, cols)) return rc;
    if (rows == 0) return NORI_OK;
    if (!x || !codes || !scales || (uintptr_t)codes % 16) return fail(NORI_ERR_INVALID, "checkpoint_quantize: null or unaligned pointer");
    const int groups = group_count(cols);
    NORI_DISPATCH_FLOAT(dtype, DT, {
        hipLaunchKernelGGL((quantize_kernel<DT>), grid_of(rows, groups), dim3(kThreads), 0, (hipStream_t)stream_v, x, rows, cols,
                           x_row_stride, groups, (uint8_t*)codes, scales);
    });
    return launch_status("checkpoint_quantize");
}

extern "C" int nori_checkpoint_silu_mul(const void* gu, int dtype, int64_t rows, int32_t hidden, int64_t gu_row_stride, void* y,
                                        void* codes, float* scales, void* stream_v) {
    clear_error();
    if (int rc = check("checkpoint_silu_mul", dtype, rows, hidden, gu_row_stride, 2LL * hidden)) return rc;
    if (rows == 0) return NORI_OK;
    if (!gu || !y || !codes != !scales || (uintptr_t)codes % 16) return fail(NORI_ERR_INVALID, "checkpoint_silu_mul: null or unaligned pointer");
    const int groups = group_count(hidden);
    NORI_DISPATCH_FLOAT(dtype, DT, {
        if (codes)
            hipLaunchKernelGGL((silu_mul_forward_kernel<DT, true>), grid_of(rows, groups), dim3(kThreads), 0, (hipStream_t)stream_v, gu,
                               rows, hidden, gu_row_stride, groups, y, (uint8_t*)codes, scales);
        else
            hipLaunchKernelGGL((silu_mul_forward_kernel<DT, false>), grid_of(rows, groups), dim3(kThreads), 0, (hipStream_t)stream_v, gu,
                               rows, hidden, gu_row_stride, groups, y, nullptr, nullptr);
    });
    return launch_status("checkpoint_silu_mul");
}

extern "C" int nori_checkpoint_silu_mul_backward(const void* codes, const float* scales, int dtype, int64_t rows, int32_t hidden,
                                                 const void* dy, int64_t dy_row_stride, void* dgu, void* stream_v) {
    clear_error();
    if (int rc = check("checkpoint_silu_mul_backward", dtype, rows, hidden, dy_row_stride, hidden)) return rc;
    if (rows == 0) return NORI_OK;
    if (!codes || !scales || !dy || !dgu || (uintptr_t)codes % 16)
        return fail(NORI_ERR_INVALID, "checkpoint_silu_mul_backward: null or unaligned pointer");
    const int groups = group_count(hidden);
    NORI_DISPATCH_FLOAT(dtype, DT, {
        hipLaunchKernelGGL((silu_mul_backward_kernel<DT>), grid_of(rows, groups), dim3(kThreads), 0, (hipStream_t)stream_v,
                           (const uint8_t*)codes, scales, rows, hidden, groups, dy, dy_row_stride, dgu);
    });
    return launch_status("checkpoint_silu_mul_backward");
}
