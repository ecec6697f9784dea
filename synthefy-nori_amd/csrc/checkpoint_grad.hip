// The gradients of a projection's weight and bias over rows kept in 8 bits: dw = dy^T x with x what the codes stand for, db = the
// column sums of dy. A workgroup owns 128 x 128 of dw over a part of the rows; dy and x pass through LDS as they lie, both
// operands are transposed reads, the codes are widened on their way in. A k tile is one group: a scale a row.
#include <algorithm>

#include "layer_norm_train.h"
#include "train_matrix.h"

namespace {

using namespace nori;
using namespace nori::train;
using nori_ln::fetch;
using nori_ln::widen;

constexpr int kThreads = 256;
constexpr int kTile = 128;  // columns of dy and of x a workgroup; the latter a group of the codes
static_assert(kTile == NORI_CHECKPOINT_GROUP, "a k tile has one scale a row");
constexpr int kRows = 32;   // rows a step
constexpr int64_t kLeast = 256;  // rows of a part

struct Args {
    const void* dy; int64_t rows, dy_stride; int n, k;
    const int8_t* codes; const float* scales;
    int code_stride, groups;
    int64_t per_split; int splits, n_tiles, k_tiles;
    void *dw, *db; int dw_dtype, db_dtype;
    float *part_w, *part_b;  // sums of parts where splits > 1
};

// Eight elements of a row in the tile's type.
template <int DT> struct Eight { typename El<DT>::T e[8]; };

template <int DT>
__device__ __forceinline__ void put(void* p, int dtype, int64_t i, float v) {
    if (dtype == NORI_F32) reinterpret_cast<float*>(p)[i] = v;
    else store_elem<DT == NORI_F32 ? NORI_F16 : DT>(p, i, v);
}

template <int DT>
__global__ __launch_bounds__(kThreads) void grad_kernel(const Args a) {
    using E = El<DT>;
    using T = typename E::T;
    constexpr int LS = kTile + E::kPad;
    constexpr int kEights = kRows * kTile / 8 / kThreads;  // of dy and of x, a thread
    __shared__ __attribute__((aligned(16))) T ys[kRows * LS];
    __shared__ __attribute__((aligned(16))) T xs[kRows * LS];
    __shared__ float sums[kThreads / (kTile / 8)][kTile];
    int i = blockIdx.x;
    const int kt = i % a.k_tiles;
    i /= a.k_tiles;
    const int nt = i % a.n_tiles, split = i / a.n_tiles;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wn = 64 * (wave & 1), wk = 64 * (wave >> 1);
    const int64_t begin = split * a.per_split, end = min(a.rows, begin + a.per_split);
    const bool own_db = a.db && kt == 0;
    // this thread's eight columns of either tile are the same in every row it takes
    const int col = 8 * (threadIdx.x % (kTile / 8)), first_row = threadIdx.x / (kTile / 8);
    constexpr int kStep = kThreads / (kTile / 8);
    const int yc = nt * kTile + col, xc = kt * kTile + col;

    Eight<DT> ye[kEights];
    uint64_t xe[kEights];
    float xsc[kEights];
    const auto load = [&](int64_t from) {
#pragma unroll
        for (int j = 0; j < kEights; ++j) {
            const int64_t r = from + first_row + j * kStep;
            ye[j] = {};
            xe[j] = 0;
            xsc[j] = 0.f;
            if (r >= end) continue;
            const T* p = reinterpret_cast<const T*>(a.dy) + r * a.dy_stride;
            if (yc + 8 <= a.n) {
                __builtin_memcpy(&ye[j], p + yc, sizeof ye[j]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (yc + e < a.n) ye[j].e[e] = p[yc + e];
            }
            if (a.dw && xc < a.code_stride) {
                xe[j] = *reinterpret_cast<const uint64_t*>(a.codes + r * a.code_stride + xc);
                xsc[j] = a.scales[r * a.groups + kt];
            }
        }
    };
    float colsum[8] = {};
    f32x16 acc[2][2] = {};
    load(begin);
    for (int64_t from = begin; from < end; from += kRows) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kEights; ++j) {
            const int at = (first_row + j * kStep) * LS + col;
            *reinterpret_cast<Eight<DT>*>(&ys[at]) = ye[j];
            if (own_db) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if constexpr (DT == NORI_F32) colsum[e] += ye[j].e[e];
                    else colsum[e] += DT == NORI_F16 ? f16_to_f32(ye[j].e[e]) : bf16_to_f32(ye[j].e[e]);
                }
            }
            Eight<DT> x;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float v = (float)(int8_t)(xe[j] >> (8 * e)) * xsc[j];
                if constexpr (DT == NORI_F32) x.e[e] = v;
                else x.e[e] = DT == NORI_F16 ? f32_to_f16(v) : f32_to_bf16(v);
            }
            *reinterpret_cast<Eight<DT>*>(&xs[at]) = x;
        }
        __syncthreads();
        if (from + kRows < end) load(from + kRows);
        if (!a.dw) continue;
#pragma unroll
        for (int t = 0; t < kRows / 16; ++t) {
            typename E::Frag y[2], x[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                y[j] = transposed<DT, LS>(ys, 16 * t, wn + 32 * j, lane);
                x[j] = transposed<DT, LS>(xs, 16 * t, wk + 32 * j, lane);
            }
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int l = 0; l < 2; ++l) acc[j][l] = mma(y[j], x[l], acc[j][l]);
        }
    }
    if (own_db) {
#pragma unroll
        for (int e = 0; e < 8; ++e) sums[first_row][col + e] = colsum[e];
        __syncthreads();
        const int c = threadIdx.x;
        if (c < kTile && nt * kTile + c < a.n) {
            float s = 0.f;
            for (int j = 0; j < kStep; ++j) s += sums[j][c];
            if (a.splits > 1) a.part_b[(int64_t)split * a.n + nt * kTile + c] = s;
            else put<DT>(a.db, a.db_dtype, nt * kTile + c, s);
        }
    }
    if (!a.dw) return;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int l = 0; l < 2; ++l)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int row = nt * kTile + wn + 32 * j + 8 * (e / 4) + 4 * (lane >> 5) + e % 4;
                const int c = kt * kTile + wk + 32 * l + (lane & 31);
                if (row >= a.n || c >= a.k) continue;
                const int64_t at = (int64_t)row * a.k + c;
                if (a.splits > 1) a.part_w[(int64_t)split * a.n * a.k + at] = acc[j][l][e];
                else put<DT>(a.dw, a.dw_dtype, at, acc[j][l][e]);
            }
}

template <int DT>
__global__ __launch_bounds__(kThreads) void join_kernel(const Args a) {
    const int64_t nk = a.dw ? (int64_t)a.n * a.k : 0, all = nk + (a.db ? a.n : 0);
    for (int64_t i = blockIdx.x * (int64_t)kThreads + threadIdx.x; i < all; i += (int64_t)gridDim.x * kThreads) {
        const bool w = i < nk;
        const float* p = w ? a.part_w + i : a.part_b + (i - nk);
        const int64_t step = w ? nk : a.n;
        float s = 0.f;
        for (int j = 0; j < a.splits; ++j) s += p[j * step];
        if (w) put<DT>(a.dw, a.dw_dtype, i, s);
        else put<DT>(a.db, a.db_dtype, i - nk, s);
    }
}

constexpr int kMost = 1 << 20;  // columns

Args plan(int dtype, int64_t rows, int32_t n, int32_t k) {
    Args a{};
    a.rows = rows;
    a.n = n;
    a.k = k;
    a.code_stride = (k + 15) / 16 * 16;
    a.groups = (k + kTile - 1) / kTile;
    a.n_tiles = (n + kTile - 1) / kTile;
    a.k_tiles = a.groups;
    const int64_t tiles = (int64_t)a.n_tiles * a.k_tiles, want = 2 * device_cus();
    int64_t splits = std::min<int64_t>((want + tiles - 1) / tiles, rows / kLeast);
    splits = std::max<int64_t>(1, std::min<int64_t>(splits, 256));
    a.per_split = std::max<int64_t>(kRows, ((rows + splits - 1) / splits + kRows - 1) / kRows * kRows);
    a.splits = (int)std::max<int64_t>(1, (rows + a.per_split - 1) / a.per_split);
    return a;
}

int64_t part_w_bytes(const Args& a) { return ((int64_t)a.splits * a.n * a.k * 4 + 15) / 16 * 16; }

}  // namespace

extern "C" int64_t nori_checkpoint_grad_workspace_bytes(int dtype, int64_t rows, int32_t n, int32_t k) {
    if (rows < 0 || n < 1 || k < 1) return 0;
    const Args a = plan(dtype, rows, n, k);
    return a.splits > 1 ? part_w_bytes(a) + (int64_t)a.splits * n * 4 : 0;
}

extern "C" int nori_checkpoint_grad(const void* dy, int dtype, int64_t rows, int32_t n, int64_t dy_row_stride, const void* codes,
                                    const float* scales, int32_t k, void* dw, int dw_dtype, void* db, int db_dtype, void* workspace,
                                    int64_t workspace_bytes, void* stream_v) {
    clear_error();
    if (dtype != NORI_F32 && dtype != NORI_F16 && dtype != NORI_BF16)
        return fail(NORI_ERR_UNSUPPORTED, "checkpoint_grad: unsupported dtype %s", dtype_name(dtype));
    if (rows < 0 || n < 1 || k < 1) return fail(NORI_ERR_INVALID, "checkpoint_grad: bad shape (%lld rows, %d x %d)", (long long)rows, n, k);
    if (n > kMost || k > kMost || rows > (1LL << 40) / std::max(n, k)) return fail(NORI_ERR_UNSUPPORTED, "checkpoint_grad: too many elements");
    if ((dw && dw_dtype != dtype && dw_dtype != NORI_F32) || (db && db_dtype != dtype && db_dtype != NORI_F32))
        return fail(NORI_ERR_UNSUPPORTED, "checkpoint_grad: gradients are of the rows' dtype or float32");
    if (dy_row_stride < 0 || (rows > 1 && dy_row_stride != 0 && dy_row_stride < n))
        return fail(NORI_ERR_INVALID, "checkpoint_grad: a row stride of %lld below rows of %d", (long long)dy_row_stride, n);
    if (!dw && !db) return NORI_OK;
    if (rows > 0 && (!dy || (dw && (!codes || !scales || (uintptr_t)codes % 16))))
        return fail(NORI_ERR_INVALID, "checkpoint_grad: null or unaligned pointer");
    Args a = plan(dtype, rows, n, k);
    a.dy = dy;
    a.dy_stride = dy_row_stride;
    a.codes = (const int8_t*)codes;
    a.scales = scales;
    a.dw = dw;
    a.db = db;
    a.dw_dtype = dw_dtype;
    a.db_dtype = db_dtype;
    if (!dw) a.k_tiles = 1;
    const int64_t blocks = (int64_t)a.n_tiles * a.k_tiles * a.splits;
    if (!one_launch(blocks, kThreads)) return fail(NORI_ERR_UNSUPPORTED, "checkpoint_grad: more workgroups than one launch has");
    if (a.splits > 1) {
        const int64_t need = nori_checkpoint_grad_workspace_bytes(dtype, rows, n, k);
        if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16)
            return fail(NORI_ERR_INVALID, "checkpoint_grad: a 16-byte aligned workspace of %lld bytes is needed", (long long)need);
        a.part_w = (float*)workspace;
        a.part_b = (float*)((char*)workspace + part_w_bytes(a));
    }
    hipStream_t stream = (hipStream_t)stream_v;
    NORI_DISPATCH_FLOAT(dtype, DT, {
        hipLaunchKernelGGL((grad_kernel<DT>), dim3((unsigned)blocks), dim3(kThreads), 0, stream, a);
        if (a.splits > 1) {
            const int64_t items = (dw ? (int64_t)n * k : 0) + (db ? n : 0);
            hipLaunchKernelGGL((join_kernel<DT>), dim3((unsigned)std::min<int64_t>((items + kThreads - 1) / kThreads, 16 * device_cus())),
                               dim3(kThreads), 0, stream, a);
        }
    });
    return launch_status("checkpoint_grad");
}
