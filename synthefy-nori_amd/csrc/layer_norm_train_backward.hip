// LayerNorm that can be trained, backward pass, for gfx950:
//     dx = rstd * (g - mean(g) - xh * mean(g * xh)),  g = dy * w,  xh = (x - mean) * rstd
//     dw = sum over rows of dy * xh,  db = sum over rows of dy
// One pass over x and dy makes dx and the column sums of its rows; sums are fp32, results rounded once.
//
// HBM-bound: x and dy are read and dx written once, c (2 e_x + e_y) bytes a row. A group holds its columns'
// sums in registers over all of its rows; a workgroup adds its groups' in LDS and writes one partial row, and
// a second launch adds the partial rows, in their order, so the same inputs give the same bits.
#include "layer_norm_train.h"

namespace {

using namespace nori_ln;

struct Backward {
    const void *x, *dy;
    int64_t rows, xs, dys;
    int cols;
    const void* w;
    int wdt, bdt;
    const float *mean, *rstd;
    void *dx, *dw, *db;
    float* partial;  // [parts][2][cols], parts the workgroups of the first launch; null: no column sums
    int parts;
};

__device__ __forceinline__ void store_param(void* p, int dt, int64_t i, float v) {
    if (dt == NORI_F32) reinterpret_cast<float*>(p)[i] = v;
    else reinterpret_cast<uint16_t*>(p)[i] = dt == NORI_F16 ? f32_to_f16(v) : f32_to_bf16(v);
}

template <int XDT, int YDT, int V, int G, int NV, bool RAGGED>
__global__ void __launch_bounds__(kThreads) backward_kernel(const Backward a) {
    __shared__ float slots[16];
    int turn = 0;
    const int lane = threadIdx.x % G;
    const float inv_n = 1.0f / (float)a.cols;
    float w[NV][V], dw[NV][V], db[NV][V];
    int at[NV], shared[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        at[i] = column<V, G, RAGGED>(i, lane, a.cols, shared[i]);
#pragma unroll
        for (int k = 0; k < V; ++k) w[i][k] = dw[i][k] = db[i][k] = 0.f;
        if (at[i] < a.cols) params<V>(a.w, a.wdt, at[i], 1.f, w[i]);
    }
    const int64_t per = kThreads / G, step = (int64_t)gridDim.x * per;
    Raw<XDT, V> next_x[NV];
    Raw<YDT, V> next_dy[NV];
    float next_mean, next_rstd;
    auto ask = [&](int64_t row) {
        next_mean = next_rstd = 0.f;
        if (row < a.rows) next_mean = a.mean[row], next_rstd = a.rstd[row];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            next_x[i] = {};
            next_dy[i] = {};
            if (row < a.rows && at[i] < a.cols) {
                next_x[i] = fetch<XDT, V>(a.x, row * a.xs + at[i]);
                next_dy[i] = fetch<YDT, V>(a.dy, row * a.dys + at[i]);
            }
        }
    };
    ask((int64_t)blockIdx.x * per + threadIdx.x / G);
    for (int64_t row0 = (int64_t)blockIdx.x * per; row0 < a.rows; row0 += step) {
        const int64_t row = row0 + threadIdx.x / G;
        float x[NV][V], dy[NV][V];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            widen<XDT, V>(next_x[i], x[i]);
            widen<YDT, V>(next_dy[i], dy[i]);
        }
        const float mean = next_mean, rstd = next_rstd;
        ask(row + step);  // the next row's loads run under this row's sums
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                x[i][k] = (x[i][k] - mean) * rstd;  // xh; past the row's end dy and w are zero
                const float d = !RAGGED || k >= shared[i] ? dy[i][k] : 0.f;
                const float g = d * w[i][k];
                s1 += g;
                s2 += g * x[i][k];
                dw[i][k] += d * x[i][k];
                db[i][k] += d;
            }
        if (!a.dx) continue;
        group_sums<G>(s1, s2, slots, turn);
        s1 *= inv_n;
        s2 *= inv_n;
        if (row >= a.rows) continue;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (at[i] >= a.cols) continue;
            float d[V];
#pragma unroll
            for (int k = 0; k < V; ++k) d[k] = rstd * (dy[i][k] * w[i][k] - s1 - x[i][k] * s2);
            store<XDT, V>(a.dx, row * a.cols + at[i], d);
        }
    }
    if (!a.partial) return;
    float* out = a.partial + (int64_t)blockIdx.x * 2 * a.cols;
    if constexpr (G < kThreads) {
        // The groups' sums: a wavefront's by shuffles, the wavefronts' one after another. A moved vector's shared elements, zero in its sums, are another
        // lane's of the same instruction: they are left to it.
        constexpr int kWide = V * G * NV;
        __shared__ float sums[2][kWide];
#pragma unroll
        for (int off = G; off < 64; off <<= 1)
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    dw[i][k] += __shfl_xor(dw[i][k], off, 64);
                    db[i][k] += __shfl_xor(db[i][k], off, 64);
                }
        for (int g = 0; g < kThreads / 64; ++g) {
            if (threadIdx.x / 64 == g && threadIdx.x % 64 < G) {
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        if (RAGGED && k < shared[i]) continue;
                        const int c = at[i] + k;
                        sums[0][c] = g == 0 ? dw[i][k] : sums[0][c] + dw[i][k];
                        sums[1][c] = g == 0 ? db[i][k] : sums[1][c] + db[i][k];
                    }
            }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < a.cols; c += kThreads) {
            out[c] = sums[0][c];
            out[a.cols + c] = sums[1][c];
        }
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const int c = at[i] + k;
                if (c < a.cols && (!RAGGED || k >= shared[i])) {
                    out[c] = dw[i][k];
                    out[a.cols + c] = db[i][k];
                }
            }
    }
}

// rows wider than registers hold: dx a workgroup a row, read twice
template <int XDT, int YDT>
__global__ void __launch_bounds__(kThreads) backward_rows_kernel(const Backward a) {
    __shared__ float slots[16];
    int turn = 0;
    const float inv_n = 1.0f / (float)a.cols;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const float mean = a.mean[row], rstd = a.rstd[row];
        float s1 = 0.f, s2 = 0.f;
        for (int c = threadIdx.x; c < a.cols; c += kThreads) {
            const float g = load_elem<YDT>(a.dy, row * a.dys + c) * param(a.w, a.wdt, c, 1.f);
            s1 += g;
            s2 += g * ((load_elem<XDT>(a.x, row * a.xs + c) - mean) * rstd);
        }
        group_sums<256>(s1, s2, slots, turn);
        s1 *= inv_n;
        s2 *= inv_n;
        for (int c = threadIdx.x; c < a.cols; c += kThreads) {
            const float g = load_elem<YDT>(a.dy, row * a.dys + c) * param(a.w, a.wdt, c, 1.f);
            const float xh = (load_elem<XDT>(a.x, row * a.xs + c) - mean) * rstd;
            store_elem<XDT>(a.dx, row * a.cols + c, rstd * (g - s1 - xh * s2));
        }
    }
}

// and the column sums a thread a column over one part of the rows
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
    float* out = a.partial + (int64_t)blockIdx.y * 2 * a.cols;
    out[c] = w;
    out[a.cols + c] = b;
}

// Adds the partial rows: 32 columns a workgroup, 32 threads a column that take every 32nd row and are joined in
// LDS. blockIdx.y 0 makes dw, 1 db.
constexpr int kJoin = 32;

__global__ void __launch_bounds__(kJoin * kJoin) join_kernel(const Backward a) {
    __shared__ float sums[kJoin][kJoin + 1];
    const int first = threadIdx.x / kJoin, lane = threadIdx.x % kJoin;
    for (int c0 = blockIdx.x * kJoin; c0 < a.cols; c0 += gridDim.x * kJoin) {
        const int c = c0 + lane;
        float s = 0.f;
        if (c < a.cols) {
            const float* p = a.partial + (int64_t)blockIdx.y * a.cols + c;
#pragma unroll 8
            for (int i = first; i < a.parts; i += kJoin) s += p[(int64_t)i * 2 * a.cols];
        }
        sums[first][lane] = s;
        __syncthreads();
        if (first == 0 && c < a.cols) {
            s = 0.f;
#pragma unroll
            for (int i = 0; i < kJoin; ++i) s += sums[i][lane];
            if (blockIdx.y == 0 && a.dw) store_param(a.dw, a.wdt, c, s);
            if (blockIdx.y == 1 && a.db) store_param(a.db, a.bdt, c, s);
        }
        __syncthreads();
    }
}

// Workgroups of the first launch: four rows each while there are few, then as many as a compute unit holds, by the
// registers of a row: `held` values a lane. Fewer idle, more wait their turn, and each costs 8 c bytes of sums,
// twice (262144 x 1680 bf16: 577 us with one a unit, 525 with two, 552 with three; 1048576 x 128 fp16: 282, 170
// and 152; 4096 x 8192 fp16, whose rows take all registers: 56, 68 and 81).
int64_t parts_of(int64_t rows, int held, bool workgroup_a_row) {
    const int per = held <= 8 ? 3 : workgroup_a_row && held > 16 ? 1 : 2;
    return std::min<int64_t>((rows + 3) / 4, (int64_t)device_cus() * per);
}

}  // namespace

extern "C" int64_t nori_layer_norm_train_workspace_bytes(int64_t rows, int32_t cols) {
    return rows <= 0 || cols <= 0 ? 0 : parts_of(rows, 1, false) * 2 * cols * 4;  // the most there can be
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
    if (rows == 0 || (!dx && !dw && !db)) return NORI_OK;
    if (!x || !dy || !mean || !rstd) return fail(NORI_ERR_INVALID, "layer_norm_train_backward: null pointer");
    const bool columns = dw || db;
    if (columns && (!workspace || (uintptr_t)workspace % 4 || workspace_bytes < nori_layer_norm_train_workspace_bytes(rows, cols)))
        return fail(NORI_ERR_INVALID, "layer_norm_train_backward: workspace of %lld bytes, %lld needed",
                    (long long)workspace_bytes, (long long)nori_layer_norm_train_workspace_bytes(rows, cols));
    Backward a{x,    dy, rows, x_row_stride, dy_row_stride, cols, weight, w_dtype, b_dtype, mean, rstd, dx, dw, db,
               columns ? reinterpret_cast<float*>(workspace) : nullptr, (int)parts_of(rows, 1, false)};
    hipStream_t stream = (hipStream_t)stream_v;
    NORI_DISPATCH_FLOAT(x_dtype, XDT, {
        NORI_DISPATCH_FLOAT(dy_dtype, YDT, {
            choose<XDT>(
                cols,
                [&](auto V_, auto G_, auto NV_, auto R_) {
                    constexpr int V = decltype(V_)::value, G = decltype(G_)::value, NV = decltype(NV_)::value;
                    constexpr bool R = decltype(R_)::value;
                    a.parts = (int)std::min<int64_t>((rows + kThreads / G - 1) / (kThreads / G), parts_of(rows, V * NV, G == 256));
                    hipLaunchKernelGGL((backward_kernel<XDT, YDT, V, G, NV, R>), dim3((unsigned)a.parts), dim3(kThreads), 0,
                                       stream, a);
                },
                [&] {
                    if (dx)
                        hipLaunchKernelGGL((backward_rows_kernel<XDT, YDT>),
                                           dim3((unsigned)std::min<int64_t>(rows, (int64_t)device_cus() * 8)), dim3(kThreads), 0,
                                           stream, a);
                    if (columns)
                        hipLaunchKernelGGL((backward_columns_kernel<XDT, YDT>),
                                           dim3((unsigned)((cols + kThreads - 1) / kThreads), (unsigned)a.parts), dim3(kThreads),
                                           0, stream, a);
                });
        });
    });
    if (columns)
        // at most 2^31 threads (one_launch): past 2^26 columns a workgroup goes round
        hipLaunchKernelGGL(join_kernel, dim3((unsigned)std::min((cols + kJoin - 1) / kJoin, 1 << 21), 2), dim3(kJoin * kJoin), 0,
                           stream, a);
    return launch_status("layer_norm_train_backward");
}
