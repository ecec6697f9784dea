// Low-rank updates of a projection's output, each row with the adapter of its table (or none), gfx950:
//     out[i] = y[i] + (s_a x[i] A_a^T) B_a^T,   a the adapter of row i,  A_a [r, k],  B_a [n, r]
// and its gradients: dx[i] = (s_a dy[i] B_a) A_a -- the same two products with the factors' roles
// swapped -- and, with h = s_a x A_a^T and g = s_a dy B_a kept from them in fp32,
//     dA_a = sum over a's rows of g[i]^T x[i],   dB_a = sum over a's rows of dy[i]^T h[i].
//
// Rows are taken by adapter: order[] lists the rows of group 0, then of group 1, ..., a group being
// every row of the batch with one adapter id (-1: the rows without one), starts[] where each begins.
#include <algorithm>

#include "nori_common.h"

namespace {

using namespace nori;

constexpr int kThreads = 256;

struct Update {
    const void *x, *y, *a, *b;
    int64_t xs, ys, os;
    int k, n, rank, adapters;
    int64_t a_rank, a_k, b_n, b_rank;  // element strides of the factors within an adapter
    const float* scales;
    const int32_t *order, *starts, *ids;
    int64_t rows;
    int groups;
    void* out;
    float* h;  // [rows][rank], rows as in x
};

// the group of position p
__device__ __forceinline__ int group_of(const int32_t* starts, int groups, int64_t p) {
    int lo = 0, hi = groups - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (starts[mid] <= p) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// h: a wavefront a row
template <int DT>
__global__ void __launch_bounds__(kThreads) shrink_kernel(const Update u) {
    const int64_t p = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (p >= u.rows) return;
    const int id = u.ids[group_of(u.starts, u.groups, p)];
    if (id < 0 || id >= u.adapters) return;
    const int64_t row = u.order[p], base = (int64_t)id * u.rank * u.k;
    const float s = u.scales ? u.scales[id] : 1.0f;
    for (int j = 0; j < u.rank; ++j) {
        float v = 0.f;
        for (int c = lane; c < u.k; c += 64)
            v += load_elem<DT>(u.x, row * u.xs + c) * load_elem<DT>(u.a, base + j * u.a_rank + c * u.a_k);
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
        if (lane == 0) u.h[row * u.rank + j] = v * s;
    }
}

// out: a thread a column, a row a workgroup
template <int DT>
__global__ void __launch_bounds__(kThreads) expand_kernel(const Update u) {
    const int64_t p = blockIdx.x;
    const int c = blockIdx.y * kThreads + threadIdx.x;
    if (c >= u.n) return;
    const int id = u.ids[group_of(u.starts, u.groups, p)];
    const int64_t row = u.order[p];
    float v = u.y ? load_elem<DT>(u.y, row * u.ys + c) : 0.f;
    if (id >= 0 && id < u.adapters) {
        const int64_t base = (int64_t)id * u.n * u.rank + c * u.b_n;
        float d = 0.f;
        for (int j = 0; j < u.rank; ++j) d += u.h[row * u.rank + j] * load_elem<DT>(u.b, base + j * u.b_rank);
        v += d;
    }
    store_elem<DT>(u.out, row * u.os + c, v);
}

struct Grad {
    const void* t;  // [rows][cols]
    const float* h; // [rows][rank]
    int64_t ts;
    int cols, rank, adapters;
    const int32_t *order, *starts, *ids;
    int groups;
    void* out;  // [adapters][...]
    int64_t o_col, o_rank;
};

// a workgroup per (group, 256 columns, rank)
template <int DT>
__global__ void __launch_bounds__(kThreads) grad_kernel(const Grad g) {
    const int c = blockIdx.y * kThreads + threadIdx.x, j = blockIdx.z;
    const int id = g.ids[blockIdx.x];
    if (c >= g.cols || id < 0 || id >= g.adapters) return;
    float v = 0.f;
    for (int p = g.starts[blockIdx.x]; p < g.starts[blockIdx.x + 1]; ++p) {
        const int64_t row = g.order[p];
        v += load_elem<DT>(g.t, row * g.ts + c) * g.h[row * g.rank + j];
    }
    store_elem<DT>(g.out, (int64_t)id * g.cols * g.rank + c * g.o_col + j * g.o_rank, v);
}

bool is_float(int dt) { return dt == NORI_F32 || dt == NORI_F16 || dt == NORI_BF16; }

int check(const char* what, int dtype, int64_t rows, int32_t groups, int32_t k, int32_t n, int32_t rank, int32_t adapters) {
    if (!is_float(dtype)) return fail(NORI_ERR_UNSUPPORTED, "%s: unsupported dtype %s", what, dtype_name(dtype));
    if (rows < 0 || groups < 0 || k <= 0 || n <= 0 || adapters <= 0)
        return fail(NORI_ERR_INVALID, "%s: bad shape (%lld rows, %d -> %d, %d adapters)", what, (long long)rows, k, n, adapters);
    if (rank <= 0 || rank > NORI_LOW_RANK_MAX)
        return fail(rank <= 0 ? NORI_ERR_INVALID : NORI_ERR_UNSUPPORTED, "%s: rank %d (1 to %d)", what, rank, NORI_LOW_RANK_MAX);
    if (rows > 0x7fffffff) return fail(NORI_ERR_UNSUPPORTED, "%s: too many rows", what);
    return NORI_OK;
}

}  // namespace

extern "C" int nori_low_rank_update(const void* x, int dtype, int64_t rows, int32_t k, int64_t x_row_stride, const void* y,
                                    int64_t y_row_stride, const void* a, const void* b, int32_t transposed,
                                    const float* scales, int32_t adapters, int32_t rank, int32_t n, const int32_t* order,
                                    const int32_t* starts, const int32_t* ids, int32_t groups, void* out,
                                    int64_t out_row_stride, float* h, void* stream_v) {
    clear_error();
    if (int rc = check("low_rank_update", dtype, rows, groups, k, n, rank, adapters)) return rc;
    if (rows == 0) return NORI_OK;
    if (!x || !a || !b || !order || !starts || !ids || !out || !h || groups <= 0)
        return fail(NORI_ERR_INVALID, "low_rank_update: null pointer");
    Update u{x, y, a, b, x_row_stride, y_row_stride, out_row_stride, k, n, rank, adapters, k, 1, rank, 1,
             scales, order, starts, ids, rows, groups, out, h};
    if (transposed) u.a_rank = 1, u.a_k = rank, u.b_n = 1, u.b_rank = n;
    hipStream_t stream = (hipStream_t)stream_v;
    NORI_DISPATCH_FLOAT(dtype, DT, {
        hipLaunchKernelGGL((shrink_kernel<DT>), dim3((unsigned)((rows + 3) / 4)), dim3(kThreads), 0, stream, u);
        hipLaunchKernelGGL((expand_kernel<DT>), dim3((unsigned)rows, (unsigned)((n + kThreads - 1) / kThreads)), dim3(kThreads),
                           0, stream, u);
    });
    return launch_status("low_rank_update");
}

extern "C" int nori_low_rank_weight_grad(const void* t, int dtype, int64_t rows, int32_t cols, int64_t t_row_stride,
                                         const float* h, int32_t rank, int32_t adapters, const int32_t* order,
                                         const int32_t* starts, const int32_t* ids, int32_t groups, int32_t transposed,
                                         void* out, void* stream_v) {
    clear_error();
    if (int rc = check("low_rank_weight_grad", dtype, rows, groups, cols, 1, rank, adapters)) return rc;
    if (rows == 0) return NORI_OK;
    if (!t || !h || !order || !starts || !ids || !out || groups <= 0)
        return fail(NORI_ERR_INVALID, "low_rank_weight_grad: null pointer");
    Grad g{t, h, t_row_stride, cols, rank, adapters, order, starts, ids, groups, out, rank, 1};
    if (transposed) g.o_col = 1, g.o_rank = cols;
    NORI_DISPATCH_FLOAT(dtype, DT, {
        hipLaunchKernelGGL((grad_kernel<DT>), dim3(groups, (unsigned)((cols + kThreads - 1) / kThreads), rank), dim3(kThreads), 0,
                           (hipStream_t)stream_v, g);
    });
    return launch_status("low_rank_weight_grad");
}
