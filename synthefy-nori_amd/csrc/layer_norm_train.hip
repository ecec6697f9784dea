// LayerNorm with its backward pass for gfx950:
//     y = xh * w + b,  xh = (x - mean) * rstd,  rstd = 1 / sqrt(var + eps)   (biased variance)
//     dx = rstd * (g - mean(g) - xh * mean(g * xh)),  g = dy * w
//     dw = sum over rows of dy * xh,  db = sum over rows of dy
// Statistics, sums and the affine are fp32; each output is rounded once, to its own type.
//
// HBM-bound: a forward row is read and written once, a backward row (x, dy) read and dx written.
#include <algorithm>

#include "nori_common.h"

namespace {

using namespace nori;

constexpr int kThreads = 256;

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

// an affine parameter of a type known at run time
__device__ __forceinline__ float param(const void* p, int dt, int64_t i, float none) {
    if (!p) return none;
    if (dt == NORI_F32) return reinterpret_cast<const float*>(p)[i];
    const uint16_t v = reinterpret_cast<const uint16_t*>(p)[i];
    return dt == NORI_F16 ? f16_to_f32(v) : bf16_to_f32(v);
}

__device__ __forceinline__ void store_param(void* p, int dt, int64_t i, float v) {
    if (dt == NORI_F32) reinterpret_cast<float*>(p)[i] = v;
    else reinterpret_cast<uint16_t*>(p)[i] = dt == NORI_F16 ? f32_to_f16(v) : f32_to_bf16(v);
}

struct Forward {
    const void* x;
    int64_t rows, xs;
    int cols;
    const void *w, *b;
    int wdt, bdt;
    float eps;
    void* y;
    float *mean, *rstd;  // null: not kept
};

// a wavefront a row
template <int XDT, int YDT>
__global__ void __launch_bounds__(kThreads) forward_kernel(const Forward a) {
    const int64_t row = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (row >= a.rows) return;
    const int64_t at = row * a.xs, to = row * a.cols;
    const float inv_n = 1.0f / (float)a.cols;
    float s = 0.f;
    for (int c = lane; c < a.cols; c += 64) s += load_elem<XDT>(a.x, at + c);
    const float mean = wave_sum(s) * inv_n;
    s = 0.f;
    for (int c = lane; c < a.cols; c += 64) {
        const float d = load_elem<XDT>(a.x, at + c) - mean;
        s += d * d;
    }
    const float rstd = 1.0f / sqrtf(wave_sum(s) * inv_n + a.eps);
    for (int c = lane; c < a.cols; c += 64) {
        const float xh = (load_elem<XDT>(a.x, at + c) - mean) * rstd;
        store_elem<YDT>(a.y, to + c, xh * param(a.w, a.wdt, c, 1.f) + param(a.b, a.bdt, c, 0.f));
    }
    if (lane == 0 && a.mean) {
        a.mean[row] = mean;
        a.rstd[row] = rstd;
    }
}

struct Backward {
    const void *x, *dy;
    int64_t rows, xs, dys;
    int cols;
    const void* w;
    int wdt, bdt;
    const float *mean, *rstd;
    void *dx, *dw, *db;
    float* partial;  // [parts][2][cols]
    int parts;
};

template <int XDT, int YDT>
__global__ void __launch_bounds__(kThreads) backward_rows_kernel(const Backward a) {
    const int64_t row = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (row >= a.rows) return;
    const float mean = a.mean[row], rstd = a.rstd[row], inv_n = 1.0f / (float)a.cols;
    float s1 = 0.f, s2 = 0.f;
    for (int c = lane; c < a.cols; c += 64) {
        const float g = load_elem<YDT>(a.dy, row * a.dys + c) * param(a.w, a.wdt, c, 1.f);
        s1 += g;
        s2 += g * ((load_elem<XDT>(a.x, row * a.xs + c) - mean) * rstd);
    }
    s1 = wave_sum(s1) * inv_n;
    s2 = wave_sum(s2) * inv_n;
    for (int c = lane; c < a.cols; c += 64) {
        const float g = load_elem<YDT>(a.dy, row * a.dys + c) * param(a.w, a.wdt, c, 1.f);
        const float xh = (load_elem<XDT>(a.x, row * a.xs + c) - mean) * rstd;
        store_elem<XDT>(a.dx, row * a.cols + c, rstd * (g - s1 - xh * s2));
    }
}

// a thread a column over one part of the rows
template <int XDT, int YDT>
__global__ void __launch_bounds__(kThreads) backward_columns_kernel(const Backward a) {
    const int c = blockIdx.x * kThreads + threadIdx.x;
    if (c >= a.cols) return;
    float w = 0.f, b = 0.f;
    for (int64_t row = blockIdx.y; row < a.rows; row += a.parts) {
        const float dy = load_elem<YDT>(a.dy, row * a.dys + c);
        w += dy * ((load_elem<XDT>(a.x, row * a.xs + c) - a.mean[row]) * a.rstd[row]);
        b += dy;
    }
    a.partial[((int64_t)blockIdx.y * 2) * a.cols + c] = w;
    a.partial[((int64_t)blockIdx.y * 2 + 1) * a.cols + c] = b;
}

// the parts' sums in their order: the same bits on every call
__global__ void __launch_bounds__(kThreads) join_kernel(const Backward a) {
    const int c = blockIdx.x * kThreads + threadIdx.x;
    if (c >= a.cols) return;
    float w = 0.f, b = 0.f;
    for (int p = 0; p < a.parts; ++p) {
        w += a.partial[((int64_t)p * 2) * a.cols + c];
        b += a.partial[((int64_t)p * 2 + 1) * a.cols + c];
    }
    if (a.dw) store_param(a.dw, a.wdt, c, w);
    if (a.db) store_param(a.db, a.bdt, c, b);
}

int parts_of(int64_t rows) { return (int)std::min<int64_t>(std::max<int64_t>(rows / 64, 1), 512); }

bool is_float(int dt) { return dt == NORI_F32 || dt == NORI_F16 || dt == NORI_BF16; }

int check(const char* what, int64_t rows, int32_t cols, int x_dtype, int y_dtype, int64_t xs, int64_t ys) {
    if (!is_float(x_dtype) || !is_float(y_dtype))
        return fail(NORI_ERR_UNSUPPORTED, "%s: unsupported dtypes %s and %s", what, dtype_name(x_dtype), dtype_name(y_dtype));
    if (rows < 0 || cols <= 0) return fail(NORI_ERR_INVALID, "%s: bad shape (%lld rows of %d)", what, (long long)rows, cols);
    if (xs < 0 || ys < 0) return fail(NORI_ERR_INVALID, "%s: negative row strides", what);
    if (rows > (int64_t)1 << 32) return fail(NORI_ERR_UNSUPPORTED, "%s: too many rows", what);
    return NORI_OK;
}

}  // namespace

extern "C" int nori_layer_norm_train_forward(const void* x, int x_dtype, int64_t rows, int32_t cols, int64_t x_row_stride,
                                             const void* weight, int w_dtype, const void* bias, int b_dtype, float eps,
                                             void* y, int y_dtype, float* mean, float* rstd, void* stream_v) {
    clear_error();
    if (int rc = check("layer_norm_train_forward", rows, cols, x_dtype, y_dtype, x_row_stride, 0)) return rc;
    if ((weight && !is_float(w_dtype)) || (bias && !is_float(b_dtype)))
        return fail(NORI_ERR_UNSUPPORTED, "layer_norm_train_forward: unsupported weight or bias dtype");
    if (!(eps >= 0.0f)) return fail(NORI_ERR_INVALID, "layer_norm_train_forward: eps must be a non-negative number");
    if (rows == 0) return NORI_OK;
    if (!x || !y || !mean != !rstd) return fail(NORI_ERR_INVALID, "layer_norm_train_forward: null pointer");
    const Forward a{x, rows, x_row_stride, cols, weight, bias, w_dtype, b_dtype, eps, y, mean, rstd};
    const unsigned grid = (unsigned)((rows + 3) / 4);
    NORI_DISPATCH_FLOAT(x_dtype, XDT, {
        NORI_DISPATCH_FLOAT(y_dtype, YDT, {
            hipLaunchKernelGGL((forward_kernel<XDT, YDT>), dim3(grid), dim3(kThreads), 0, (hipStream_t)stream_v, a);
        });
    });
    return launch_status("layer_norm_train_forward");
}

extern "C" int64_t nori_layer_norm_train_workspace_bytes(int64_t rows, int32_t cols) {
    return rows <= 0 || cols <= 0 ? 0 : (int64_t)parts_of(rows) * 2 * cols * 4;
}

extern "C" int nori_layer_norm_train_backward(const void* x, int x_dtype, int64_t rows, int32_t cols, int64_t x_row_stride,
                                              const void* dy, int dy_dtype, int64_t dy_row_stride, const void* weight,
                                              int w_dtype, int b_dtype, const float* mean, const float* rstd, void* dx,
                                              void* dw, void* db, void* workspace, int64_t workspace_bytes,
                                              void* stream_v) {
    clear_error();
    if (int rc = check("layer_norm_train_backward", rows, cols, x_dtype, dy_dtype, x_row_stride, dy_row_stride)) return rc;
    if (((weight || dw) && !is_float(w_dtype)) || (db && !is_float(b_dtype)))
        return fail(NORI_ERR_UNSUPPORTED, "layer_norm_train_backward: unsupported weight or bias dtype");
    if (rows == 0) return NORI_OK;
    if (!x || !dy || !mean || !rstd) return fail(NORI_ERR_INVALID, "layer_norm_train_backward: null pointer");
    const bool columns = dw || db;
    if (columns && (!workspace || workspace_bytes < nori_layer_norm_train_workspace_bytes(rows, cols)))
        return fail(NORI_ERR_INVALID, "layer_norm_train_backward: workspace of %lld bytes, %lld needed",
                    (long long)workspace_bytes, (long long)nori_layer_norm_train_workspace_bytes(rows, cols));
    const Backward a{x,    dy, rows, x_row_stride, dy_row_stride, cols, weight, w_dtype, b_dtype, mean, rstd, dx, dw, db,
                     reinterpret_cast<float*>(workspace), parts_of(rows)};
    hipStream_t stream = (hipStream_t)stream_v;
    const unsigned grid = (unsigned)((rows + 3) / 4), chunks = (unsigned)((cols + kThreads - 1) / kThreads);
    NORI_DISPATCH_FLOAT(x_dtype, XDT, {
        NORI_DISPATCH_FLOAT(dy_dtype, YDT, {
            if (dx)
                hipLaunchKernelGGL((backward_rows_kernel<XDT, YDT>), dim3(grid), dim3(kThreads), 0, stream, a);
            if (columns)
                hipLaunchKernelGGL((backward_columns_kernel<XDT, YDT>), dim3(chunks, a.parts), dim3(kThreads), 0, stream, a);
        });
    });
    if (columns) hipLaunchKernelGGL(join_kernel, dim3(chunks), dim3(kThreads), 0, stream, a);
    return launch_status("layer_norm_train_backward");
}
