// LayerNorm that can be trained, forward pass, for gfx950:
//     y = xh * w + b,  xh = (x - mean) * rstd,  rstd = 1 / sqrt(var + eps)   (biased variance)
// mean and rstd kept in fp32 for the backward pass (layer_norm_train_backward.hip). Statistics and affine are
// fp32, y is rounded once. The variance is summed from the centred row, held in registers: a mean far from
// zero costs no digits.
//
// HBM-bound: each row is read and written once, c (e_x + e_y) bytes. Groups walk the rows in a grid-stride
// loop, so that the affine parameters are read once a group and not once a row.
#include "layer_norm_train.h"

namespace {

using namespace nori_ln;

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

template <int XDT, int YDT, int V, int G, int NV, bool RAGGED>
__global__ void __launch_bounds__(kThreads) forward_kernel(const Forward a) {
    __shared__ float slots[16];
    int turn = 0;
    const int lane = threadIdx.x % G;
    const float inv_n = 1.0f / (float)a.cols;
    float w[NV][V], b[NV][V];
    int at[NV], shared[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        at[i] = column<V, G, RAGGED>(i, lane, a.cols, shared[i]);
        if (at[i] < a.cols) {
            params<V>(a.w, a.wdt, at[i], 1.f, w[i]);
            params<V>(a.b, a.bdt, at[i], 0.f, b[i]);
        }
    }
    const int64_t per = kThreads / G, step = (int64_t)gridDim.x * per;
    Raw<XDT, V> next[NV];
    auto ask = [&](int64_t row) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            next[i] = {};
            if (row < a.rows && at[i] < a.cols) next[i] = fetch<XDT, V>(a.x, row * a.xs + at[i]);
        }
    };
    ask((int64_t)blockIdx.x * per + threadIdx.x / G);
    // every group of a wavefront, every wavefront of a workgroup, goes round as often: the sums stay uniform
    for (int64_t row0 = (int64_t)blockIdx.x * per; row0 < a.rows; row0 += step) {
        const int64_t row = row0 + threadIdx.x / G;
        float v[NV][V];
        float s = 0.f, none = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) widen<XDT, V>(next[i], v[i]);
        ask(row + step);  // the next row's loads run under this row's sums
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int k = 0; k < V; ++k) s += !RAGGED || k >= shared[i] ? v[i][k] : 0.f;
        group_sums<G>(s, none, slots, turn);
        const float mean = s * inv_n;
        s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                v[i][k] -= mean;
                s += at[i] < a.cols && (!RAGGED || k >= shared[i]) ? v[i][k] * v[i][k] : 0.f;
            }
        group_sums<G>(s, none, slots, turn);
        const float rstd = rsqrtf(s * inv_n + a.eps);
        if (row >= a.rows) continue;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (at[i] >= a.cols) continue;
#pragma unroll
            for (int k = 0; k < V; ++k) v[i][k] = v[i][k] * rstd * w[i][k] + b[i][k];
            store<YDT, V>(a.y, row * a.cols + at[i], v[i]);
        }
        if (lane == 0 && a.mean) {
            a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
    }
}

// rows wider than registers hold, a workgroup each: read three times, the second and third from the L2
template <int XDT, int YDT>
__global__ void __launch_bounds__(kThreads) forward_loop_kernel(const Forward a) {
    __shared__ float slots[16];
    int turn = 0;
    const float inv_n = 1.0f / (float)a.cols;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const int64_t at = row * a.xs, to = row * a.cols;
        float s = 0.f, none = 0.f;
        for (int c = threadIdx.x; c < a.cols; c += kThreads) s += load_elem<XDT>(a.x, at + c);
        group_sums<256>(s, none, slots, turn);
        const float mean = s * inv_n;
        s = 0.f;
        for (int c = threadIdx.x; c < a.cols; c += kThreads) {
            const float d = load_elem<XDT>(a.x, at + c) - mean;
            s += d * d;
        }
        group_sums<256>(s, none, slots, turn);
        const float rstd = rsqrtf(s * inv_n + a.eps);
        for (int c = threadIdx.x; c < a.cols; c += kThreads) {
            const float xh = (load_elem<XDT>(a.x, at + c) - mean) * rstd;
            store_elem<YDT>(a.y, to + c, xh * param(a.w, a.wdt, c, 1.f) + param(a.b, a.bdt, c, 0.f));
        }
        if (threadIdx.x == 0 && a.mean) {
            a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
    }
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
    hipStream_t stream = (hipStream_t)stream_v;
    const int64_t most = (int64_t)device_cus() * 16;
    NORI_DISPATCH_FLOAT(x_dtype, XDT, {
        NORI_DISPATCH_FLOAT(y_dtype, YDT, {
            choose<XDT>(
                cols,
                [&](auto V_, auto G_, auto NV_, auto R_) {
                    constexpr int V = decltype(V_)::value, G = decltype(G_)::value, NV = decltype(NV_)::value;
                    constexpr bool R = decltype(R_)::value;
                    const int64_t need = (rows + kThreads / G - 1) / (kThreads / G);
                    hipLaunchKernelGGL((forward_kernel<XDT, YDT, V, G, NV, R>), dim3((unsigned)std::min(need, most)),
                                       dim3(kThreads), 0, stream, a);
                },
                [&] {
                    hipLaunchKernelGGL((forward_loop_kernel<XDT, YDT>), dim3((unsigned)std::min(rows, most)), dim3(kThreads), 0,
                                       stream, a);
                });
        });
    });
    return launch_status("layer_norm_train_forward");
}
