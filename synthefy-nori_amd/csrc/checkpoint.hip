// Activations kept in 8 bits for the backward pass: rows quantised in groups of 128 columns, and the SwiGLU gate with its
// gradient over gate and up kept so. One pass each, HBM-bound: 16 lanes hold a group, 8 elements each, in registers
// between the largest magnitude (DPP) and the codes. 131,072 x 560 bf16 quantised: 44-47 us (4.9 TB/s); gate of 938, bf16: 186 us
// with its codes, 177 for its gradient (5.3 and 5.6 TB/s).
//
// The code of x is the whole number nearest to x / s, ties to even, exactly: k, the nearest to x (1 / s), may be one off beside a
// half, and the remainder x - k s, which one fma gives without error there, says so. (Both terms are multiples of 2^-149 or half
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

template <int DT>
using Raw8 = nori_ln::Raw<DT, kEach>;

// 8 elements from column c of a row of cols as they lie in memory, zeros past its end: at most three accesses there.
template <int DT>
__device__ __forceinline__ Raw8<DT> load8(const void* p, int64_t row, int c, int cols) {
    if (c + kEach <= cols) return fetch<DT, kEach>(p, row + c);
    Raw8<DT> r = {};
    const int n = cols - c;
    if (n <= 0) return r;
    if (n & 4) {
        const auto x = fetch<DT, 4>(p, row + c);
#pragma unroll
        for (int i = 0; i < 4; ++i) r.e[i] = x.e[i];
    }
    if (n & 2) {
        const auto x = fetch<DT, 2>(p, row + c + (n & 4));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            r.e[i] = n & 4 ? +r.e[i] : +x.e[i];
            if (n & 4) r.e[4 + i] = x.e[i];
        }
    }
    if (n & 1) {
        const auto x = fetch<DT, 1>(p, row + c + (n & 6)).e[0];
#pragma unroll
        for (int i = 0; i < 8; i += 2)
            if ((n & 6) == i) r.e[i] = x;
    }
    return r;
}

template <int DT>
__device__ __forceinline__ void store8(void* p, int64_t row, int c, int cols, const float (&v)[kEach]) {
    const int n = cols - c;
    if (n <= 0) return;
    if (n >= kEach) return store<DT, kEach>(p, row + c, v);
    // (taken out before the choices: a choice between places would put v into memory)
    const float v0 = v[0], v1 = v[1], v2 = v[2], v3 = v[3], v4 = v[4], v5 = v[5], v6 = v[6];
    if (n & 4) store<DT, 4>(p, row + c, {v0, v1, v2, v3});
    const float pair[2] = {n & 4 ? v4 : v0, n & 4 ? v5 : v1};
    if (n & 2) store<DT, 2>(p, row + c + (n & 4), pair);
    const float low = n & 2 ? v2 : v0, high = n & 2 ? v6 : v4;
    if (n & 1) store_elem<DT>(p, row + c + (n & 6), n & 4 ? high : low);
}

// The largest magnitude of 8 elements as a whole number, NaN on top: of their own bits, two at a time in the 16-bit types.
template <int DT>
__device__ __forceinline__ uint32_t magnitude(const Raw8<DT>& r) {
    if constexpr (DT == NORI_F32) {
        uint32_t key = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) key = max(key, r.e[i] & 0x7fffffffu);
        return key;
    } else {
        typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
        u16x2 w[4];
        __builtin_memcpy(w, r.e, sizeof w);
        u16x2 key = {0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) key = __builtin_elementwise_max(key, w[i] & (uint16_t)0x7fff);
        return max((uint32_t)key[0], (uint32_t)key[1]);
    }
}

// The largest of a value over 16 lanes.
__device__ __forceinline__ uint32_t max16(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, false));  // row_ror:8
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xf, 0xf, false));
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xf, 0xf, false));
}

// The group's scale and this lane's codes of elements r, v widened. A scale that is a normal number: k in one fma with a number
// whose last place is 1, the code in its low byte (quotients stay below 127.5: no code passes 127); of few bits: by division. Looked at again
// only where a lane of the wavefront has a remainder of half a scale.
template <int DT>
__device__ __forceinline__ float quantize8(const Raw8<DT>& r, const float (&v)[kEach], uint64_t& codes) {
    constexpr float kOnes = 12582912.0f;  // 3 * 2^22
    const uint32_t key = max16(magnitude<DT>(r));
    const float amax = DT == NORI_F32 ? __uint_as_float(key) : (DT == NORI_F16 ? f16_to_f32((uint16_t)key) : bf16_to_f32((uint16_t)key));
    const float s = amax <= 3.402823466e38f ? amax * (1.0f / 127.0f) : NAN;  // an infinity or NaN: NaN throughout
    const bool normal = s >= 0x1p-126f;
    const float y = normal ? 1.0f / s : 0.0f;
    float k[kEach], rest[kEach], most = 0.f;
#pragma unroll
    for (int i = 0; i < kEach; ++i) k[i] = fmaf(v[i], y, kOnes);
    if (__any(s > 0.0f && !normal)) {  // a scale of few bits: quotients up to 190
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (s > 0.0f && !normal) k[i] = fminf(fmaxf(rintf(v[i] / s), -127.0f), 127.0f) + kOnes;
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        rest[i] = fmaf(kOnes - k[i], s, v[i]);
        most = fmaxf(most, fabsf(rest[i]));
    }
    // twice a remainder against s: half of s may be no number. (bfloat16's halves are not rare: amax / 2 is one)
    if (__any(s > 0.0f && 2.0f * most >= s)) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const float far = 2.0f * fabsf(rest[i]);
            const bool up = s > 0.0f && (far > s || (far == s && (__float_as_uint(k[i]) & 1u)));
            const float next = fminf(fmaxf(k[i] + copysignf(1.0f, rest[i]), kOnes - 127.0f), kOnes + 127.0f);
            k[i] = up ? next : k[i];
        }
    }
    uint32_t w[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(k[4 * j + 1]), __float_as_uint(k[4 * j]), 0x0c0c0400u);
        const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(k[4 * j + 3]), __float_as_uint(k[4 * j + 2]), 0x04000c0cu);
        w[j] = lo | hi;
    }
    codes = (uint64_t)w[1] << 32 | w[0];
    return s;
}

// What codes stand for, rounded once.
__device__ __forceinline__ void restore8(const uint64_t codes, float s, float (&v)[kEach]) {
    const uint32_t w[2] = {(uint32_t)codes, (uint32_t)(codes >> 32)};
#pragma unroll
    for (int i = 0; i < kEach; ++i) v[i] = (float)(int8_t)(w[i >> 2] >> (8 * (i & 3))) * s;
}

// 1 / (1 + exp(-g)), to about 2^-22 of itself and |g| 2^-24.
__device__ __forceinline__ float sigmoid(float g) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -1.4426950408889634f));
}

// Where a thread works: group `group` of row `row`, its 8 columns from `col`. (A launch has fewer than 2^28 groups.)
struct Item { int64_t row; int group, col; bool there; };
__device__ __forceinline__ Item item_of(int64_t rows, int groups) {
    const uint32_t i = blockIdx.x * kItems + threadIdx.x / kLanes, row = i / (uint32_t)groups;
    Item it;
    it.row = row;
    it.group = (int)(i - row * (uint32_t)groups);
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
    const auto r = load8<DT>(x, it.row * stride, it.col, cols);
    float v[kEach];
    widen<DT, kEach>(r, v);
    uint64_t w;
    const float s = quantize8<DT>(r, v, w);
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
    const auto rg = load8<DT>(gu, it.row * stride, it.col, hidden);
    const auto ru = load8<DT>(gu, it.row * stride + hidden, it.col, hidden);
    widen<DT, kEach>(rg, g);
    widen<DT, kEach>(ru, u);
#pragma unroll
    for (int i = 0; i < kEach; ++i) o[i] = g[i] * sigmoid(g[i]) * u[i];
    store8<DT>(y, it.row * hidden, it.col, hidden, o);
    if constexpr (KEEP) {
        const int to = code_stride(hidden);
        uint64_t w[2];
        const float s[2] = {quantize8<DT>(rg, g, w[0]), quantize8<DT>(ru, u, w[1])};
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
    widen<DT, kEach>(load8<DT>(dy, it.row * stride, it.col, hidden), d);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const float sig = sigmoid(g[i]);
        const float du = d[i] * g[i] * sig;
        g[i] = d[i] * u[i] * (sig * (1.0f + g[i] * (1.0f - sig)));
        u[i] = du;
    }
    store8<DT>(dgu, it.row * 2 * hidden, it.col, hidden, g);
    store8<DT>(dgu, it.row * 2 * hidden + hidden, it.col, hidden, u);
}

constexpr int kMostCols = 1 << 24;

int check(const char* what, int dtype, int64_t rows, int32_t cols, int64_t stride) {
    if (rows < 0 || cols < 1) return fail(NORI_ERR_INVALID, "%s: bad shape (%lld rows of %d)", what, (long long)rows, cols);
    if (dtype != NORI_F32 && dtype != NORI_F16 && dtype != NORI_BF16)
        return fail(NORI_ERR_UNSUPPORTED, "%s: unsupported dtype %s", what, dtype_name(dtype));
    if (cols > kMostCols || rows > (1LL << 40) / cols) return fail(NORI_ERR_UNSUPPORTED, "%s: too many elements", what);
    if (stride < 0) return fail(NORI_ERR_INVALID, "%s: a row stride of %lld", what, (long long)stride);
    if (!one_launch((rows * group_count(cols) + kItems - 1) / kItems, kThreads)) return fail(NORI_ERR_UNSUPPORTED, "%s: too many rows", what);
    return NORI_OK;
}

dim3 grid_of(int64_t rows, int groups) { return dim3((unsigned)((rows * groups + kItems - 1) / kItems)); }

}  // namespace

extern "C" int nori_checkpoint_quantize(const void* x, int dtype, int64_t rows, int32_t cols, int64_t x_row_stride, void* codes,
                                        float* scales, void* stream_v) {
    clear_error();
    if (int rc = check("checkpoint_quantize", dtype, rows, cols, x_row_stride)) return rc;
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
    if (int rc = check("checkpoint_silu_mul", dtype, rows, hidden, gu_row_stride)) return rc;
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
    if (int rc = check("checkpoint_silu_mul_backward", dtype, rows, hidden, dy_row_stride)) return rc;
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
