// The gradients of a projection's weight and bias over rows kept in 8 bits: dw = dy^T x with x what the codes stand for, db = the
// column sums of dy. A workgroup owns 256 or 128 x 128 of dw over a part of the rows; dy and x pass through LDS as they lie, both
// operands are transposed reads, the codes are widened on their way in. A k tile is one group: a scale a row.
//
// Bound by the matrix instructions and what stands between them (reads of both operands, codes to values): 131,072 rows 560 -> 2,240
// bf16, 437 us (753 TFLOP/s; a library product of these sizes with both operands as it wants them: 331-488). 256 columns of dy a
// workgroup halve the reads of x's tile a product; where n fills no pair of 128s, or dy takes two pieces or 4 bytes, it is 128.
#include <algorithm>

#include "train_matrix.h"

namespace {

using namespace nori;
using namespace nori::train;

constexpr int kThreads = 256;
constexpr int kGroup = NORI_CHECKPOINT_GROUP;  // columns of x a workgroup: one scale a row
constexpr int64_t kLeast = 256;                // rows of a part

struct Args {
    const void* dy; int64_t rows, dy_stride; int n, k;
    const int8_t* codes; const float* scales;
    int code_stride, groups;
    int64_t per_split; int splits, tile_n, n_tiles, k_tiles;
    void *dw, *db; int dw_dtype, db_dtype;
    float *part_w, *part_b;  // sums of parts where splits > 1; those of db are of the rows' steps that a k tile takes
};

// Eight elements of a row in the tile's type.
template <int DT> struct Eight { typename El<DT>::T e[8]; };

template <int DT>
__device__ __forceinline__ void put(void* p, int dtype, int64_t i, float v) {
    if (dtype == NORI_F32) reinterpret_cast<float*>(p)[i] = v;
    else store_elem<DT == NORI_F32 ? NORI_F16 : DT>(p, i, v);
}

// The values of 8 codes.
template <int DT>
__device__ __forceinline__ Eight<DT> values(uint32_t lo, uint32_t hi, float s) {
    const uint32_t w[2] = {lo, hi};
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)(int8_t)(w[i >> 2] >> (8 * (i & 3))) * s;
    if constexpr (DT == NORI_F32) {
        return __builtin_bit_cast(Eight<DT>, v);
    } else {
        typename El<DT>::Frag f;
#pragma unroll
        for (int i = 0; i < 8; ++i) at(f, i) = v[i];
        return __builtin_bit_cast(Eight<DT>, f);
    }
}

// dy s in two float16 pieces, to 2^-22 of itself, beside codes that are whole numbers: what an fp32 gradient of 16-bit rows takes. x
// rounded to the rows' type would leave 2^-12 (float16) or 2^-9 of every term, above what the gradient's type can tell.
template <int DT>
__device__ __forceinline__ float wide(const Eight<DT>& y, int e) {
    if constexpr (DT == NORI_F32) return y.e[e];
    else return DT == NORI_F16 ? f16_to_f32(y.e[e]) : bf16_to_f32(y.e[e]);
}
template <int DT>
__device__ __forceinline__ void pieces(const Eight<DT>& y, float s, float power, Eight<NORI_F16>& hi, Eight<NORI_F16>& lo) {
    f16x8 h, l;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float v = wide<DT>(y, e) * s * power;
        // one value for both pieces: a product folded into one of its roundings to float16, and not into the other, rounds otherwise
        asm("" : "+v"(v));
        h[e] = (_Float16)v;
        const float w = (float)h[e];
        l[e] = (_Float16)(fabsf(w) == INFINITY ? 0.f : v - w);
    }
    hi = __builtin_bit_cast(Eight<NORI_F16>, h);
    lo = __builtin_bit_cast(Eight<NORI_F16>, l);
}

// TN columns of dy by 128 of x a workgroup, half of each a wavefront. FINE: dw in fp32 of 16-bit rows, two products a pair.
template <int DT, int TN, bool FINE>
__global__ __launch_bounds__(kThreads, 2) void grad_kernel(const Args a) {
    constexpr int MT = FINE ? NORI_F16 : DT;  // the products' type
    using E = El<MT>;
    using T = typename El<DT>::T;
    constexpr int kRows = DT == NORI_F32 ? 32 : 64;  // rows a step
    // transposed reads take 64 bytes of four rows at once: rows 16 banks apart (mod 64) meet no other's
    constexpr int kPad = DT == NORI_F32 ? El<DT>::kPad : 32, YS = TN + kPad, XS = kGroup + kPad;
    constexpr int MY = TN / 64, MX = 2;              // products of 32 columns a wavefront
    constexpr int kPerRow = TN / 8, kYStep = kThreads / kPerRow, NY = kRows / kYStep;
    constexpr int kXStep = kThreads / (kGroup / 16), NX = kRows / kXStep;
    __shared__ __attribute__((aligned(16))) T ys[kRows * YS];
    __shared__ __attribute__((aligned(16))) T xs[kRows * XS];
    __shared__ __attribute__((aligned(16))) T ls[FINE ? kRows * YS : 8];  // dy's low pieces
    const int64_t i = blockIdx.x, eights = gridDim.x & ~7u;  // neighbours, which read the same rows, on one XCD
    const int64_t work = i < eights ? (i & 7) * (eights >> 3) + (i >> 3) : i;
    const int kt = (int)(work % a.k_tiles), nt = (int)(work / a.k_tiles % a.n_tiles), split = (int)(work / a.k_tiles / a.n_tiles);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wn = TN / 2 * (wave & 1), wk = kGroup / 2 * (wave >> 1);
    const int64_t begin = split * a.per_split, end = min(a.rows, begin + a.per_split);
    // a thread's eight columns of dy and sixteen of x are the same in every row it takes
    const int ycol = 8 * (threadIdx.x % kPerRow), yrow = threadIdx.x / kPerRow, yc = nt * TN + ycol;
    const int xcol = 16 * (threadIdx.x % (kGroup / 16)), xrow = threadIdx.x / (kGroup / 16), xc = kt * kGroup + xcol;
    // lanes past the last column read the first ones: their sums are not used
    const int yat = yc < a.n ? yc : 0, xat = xc < a.code_stride ? xc : 0;
    const uint32_t yoff = ((uint32_t)yrow * (uint32_t)a.dy_stride + yat) * sizeof(T), xoff = xrow * a.code_stride + xat;

    Eight<DT> ye[NY];
    uint4 xe[NX];
    float xsc[FINE ? 1 : NX], ysc[FINE ? NY : 1];
    // A step whose rows are all there, and not the last, whose eight columns past the row's end reach into the next row
    const auto whole = [&](int64_t from) { return from + kRows <= end && from + kRows < a.rows && a.dy_stride >= 8; };
    const auto load = [&](int64_t from) {
        const char* py = reinterpret_cast<const char*>(a.dy) + from * a.dy_stride * (int64_t)sizeof(T);
        const int8_t* px = a.codes + from * a.code_stride;
        const float* ps = a.scales + from * a.groups + kt;
#pragma unroll
        for (int j = 0; j < NY; ++j) __builtin_memcpy(&ye[j], py + j * kYStep * a.dy_stride * (int64_t)sizeof(T) + yoff, sizeof ye[j]);
        if (!a.dw) return;
#pragma unroll
        for (int j = 0; j < NX; ++j) {
            xe[j] = *reinterpret_cast<const uint4*>(px + j * kXStep * a.code_stride + xoff);
            if constexpr (!FINE) xsc[j] = ps[j * kXStep * a.groups + xrow * a.groups];
        }
        if constexpr (FINE) {
#pragma unroll
            for (int j = 0; j < NY; ++j) ysc[j] = ps[j * kYStep * a.groups + yrow * a.groups];
        }
    };
    // of a row at the end of the rows or of the columns
    const auto partial = [&](int64_t r) {
        Eight<DT> y = {};
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (r < end && yc + e < a.n) y.e[e] = reinterpret_cast<const T*>(a.dy)[r * a.dy_stride + yc + e];
        return y;
    };
    const auto put_y = [&](int j, const Eight<DT>& y, float s, float power) {
        const int at = (yrow + j * kYStep) * YS + ycol;
        if constexpr (FINE) pieces<DT>(y, s, power, *reinterpret_cast<Eight<NORI_F16>*>(&ys[at]), *reinterpret_cast<Eight<NORI_F16>*>(&ls[at]));
        else *reinterpret_cast<Eight<DT>*>(&ys[at]) = y;
    };
    const auto put_x = [&](int j, uint4 x, float s) {
        Eight<MT>* to = reinterpret_cast<Eight<MT>*>(&xs[(xrow + j * kXStep) * XS + xcol]);
        to[0] = values<MT>(x.x, x.y, s);
        to[1] = values<MT>(x.z, x.w, s);
    };
    float colsum[8] = {};
    const auto add = [&](const Eight<DT>& y) {
#pragma unroll
        for (int e = 0; e < 8; ++e) colsum[e] += wide<DT>(y, e);
    };
    f32x16 acc[MY][MX] = {};
    // FINE: a power of two on dy s, which float16 has no range for. It brings the first step's largest to 2^8 and falls where a later
    // one would pass 2^15; the sums are brought along.
    __shared__ float tops[kThreads / 64];
    float power = 0.f, top = 0.f;
    const int live = min(8, a.n - yat);  // past the row's end anything may lie
    const auto look = [&](const Eight<DT>& y, float s) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float v = fabsf(wide<DT>(y, e)) * s;
            top = fmaxf(top, e < live && v < INFINITY ? v : 0.f);
        }
    };
    const auto share = [&] {
        for (int i = 32; i > 0; i /= 2) top = fmaxf(top, __shfl_xor(top, i));
        if (lane == 0) tops[wave] = top;
    };
    const auto agree = [&] {
        top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
        if (power == 0.f ? top > 0.f : top * power > 32768.f) {
            int e = 8 + 127 - (int)(__float_as_uint(top) >> 23);
            e = e > 120 ? 120 : (e < -120 ? -120 : e);
            const float next = __uint_as_float((uint32_t)(e + 127) << 23), by = power == 0.f ? 1.f : next / power;
#pragma unroll
            for (int i = 0; i < 16 * MY * MX; ++i) acc[i / 16 / MX][i / 16 % MX][i % 16] *= by;
            power = next;
        }
        top = 0.f;
    };
    int turn = a.db ? (a.splits > 1 ? kt : (kt == 0 ? 0 : -1)) : -1;  // steps until this k tile's next one of db
    if (whole(begin)) load(begin);
    for (int64_t from = begin; from < end; from += kRows) {
        if constexpr (FINE) {
            if (whole(from)) {
#pragma unroll
                for (int j = 0; j < NY; ++j) look(ye[j], ysc[j]);
            } else if (a.dw) {
#pragma unroll 1
                for (int j = 0; j < NY; ++j) {
                    const int64_t r = from + yrow + j * kYStep;
                    look(partial(r), r < end ? a.scales[r * a.groups + kt] : 0.f);
                }
            }
            share();
        }
        __syncthreads();
        if constexpr (FINE) agree();
        const float factor = power == 0.f ? 1.f : power;  // (nothing but zeros so far, or infinities, which stay)
        if (whole(from)) {
#pragma unroll
            for (int j = 0; j < NY; ++j) put_y(j, ye[j], FINE ? ysc[FINE ? j : 0] : 1.f, factor);
#pragma unroll
            for (int j = 0; j < NX; ++j) put_x(j, xe[j], FINE ? 1.f : xsc[FINE ? 0 : j]);
            if (turn == 0) {
#pragma unroll
                for (int j = 0; j < NY; ++j) add(ye[j]);
            }
        } else {
#pragma unroll 1
            for (int j = 0; j < NY; ++j) {
                const int64_t r = from + yrow + j * kYStep;
                const Eight<DT> y = partial(r);
                put_y(j, y, FINE && a.dw && r < end ? a.scales[r * a.groups + kt] : 1.f, factor);
                if (turn == 0) add(y);
            }
#pragma unroll 1
            for (int j = 0; a.dw && j < NX; ++j) {
                const int64_t r = from + xrow + j * kXStep;
                uint4 x = {};
                float sc = 0.f;
                if (r < end) {
                    x = *reinterpret_cast<const uint4*>(a.codes + r * a.code_stride + xat);
                    sc = FINE ? 1.f : a.scales[r * a.groups + kt];
                }
                put_x(j, x, sc);
            }
        }
        if (turn == 0) turn = a.splits > 1 ? a.k_tiles : 1;
        if (turn > 0) --turn;
        __syncthreads();
        if (from + kRows < end && whole(from + kRows)) load(from + kRows);
        if (!a.dw) continue;
#pragma unroll 2
        for (int t = 0; t < kRows / 16; ++t) {
            typename E::Frag y[MY], x[MX];
#pragma unroll
            for (int j = 0; j < MX; ++j) x[j] = transposed<MT, XS>(xs, 16 * t, wk + 32 * j, lane);
#pragma unroll
            for (int j = 0; j < MY; ++j) y[j] = transposed<MT, YS>(ys, 16 * t, wn + 32 * j, lane);
#pragma unroll
            for (int j = 0; j < MY; ++j)
#pragma unroll
                for (int l = 0; l < MX; ++l) acc[j][l] = mma(y[j], x[l], acc[j][l]);
            if constexpr (FINE) {
#pragma unroll
                for (int j = 0; j < MY; ++j) y[j] = transposed<MT, YS>(ls, 16 * t, wn + 32 * j, lane);
#pragma unroll
                for (int j = 0; j < MY; ++j)
#pragma unroll
                    for (int l = 0; l < MX; ++l) acc[j][l] = mma(y[j], x[l], acc[j][l]);
            }
        }
    }
    if (a.db && (a.splits > 1 || kt == 0)) {
        float* sums = reinterpret_cast<float*>(ys);  // [kYStep][TN]
        static_assert(kYStep * TN * 4 <= (int)sizeof(ys), "the column sums fit the tile");
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 8; ++e) sums[yrow * TN + ycol + e] = colsum[e];
        __syncthreads();
        const int c = threadIdx.x;
        if (c < TN && nt * TN + c < a.n) {
            float s = 0.f;
            for (int j = 0; j < kYStep; ++j) s += sums[j * TN + c];
            if (a.splits > 1) a.part_b[((int64_t)split * a.k_tiles + kt) * a.n + nt * TN + c] = s;
            else put<DT>(a.db, a.db_dtype, nt * TN + c, s);
        }
    }
    if (!a.dw) return;
    const float by = FINE && power != 0.f ? 1.f / power : 1.f;
#pragma unroll
    for (int j = 0; j < MY; ++j)
#pragma unroll
        for (int l = 0; l < MX; ++l)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int row = nt * TN + wn + 32 * j + 8 * (e / 4) + 4 * (lane >> 5) + e % 4;
                const int c = kt * kGroup + wk + 32 * l + (lane & 31);
                if (row >= a.n || c >= a.k) continue;
                const int64_t at = (int64_t)row * a.k + c;
                if (a.splits > 1) a.part_w[(int64_t)split * a.n * a.k + at] = acc[j][l][e] * by;
                else put<DT>(a.dw, a.dw_dtype, at, acc[j][l][e] * by);
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
        const int parts = w ? a.splits : a.splits * a.k_tiles;
#pragma unroll 8
        for (int j = 0; j < parts; ++j) s += p[j * step];
        if (w) put<DT>(a.dw, a.dw_dtype, i, s);
        else put<DT>(a.db, a.db_dtype, i - nk, s);
    }
}

constexpr int kMost = 1 << 20;  // columns

// fine: dw in fp32 of 16-bit rows
Args plan(int dtype, bool fine, int64_t rows, int32_t n, int32_t k) {
    Args a{};
    a.rows = rows;
    a.n = n;
    a.k = k;
    a.code_stride = (k + 15) / 16 * 16;
    a.groups = (k + kGroup - 1) / kGroup;
    a.tile_n = dtype == NORI_F32 || fine || (n + 127) / 128 % 2 ? 128 : 256;
    a.n_tiles = (n + a.tile_n - 1) / a.tile_n;
    a.k_tiles = a.groups;
    // one round of the workgroups that the compute units hold
    const int64_t tiles = (int64_t)a.n_tiles * a.k_tiles, hold = 2 * device_cus();
    const int64_t splits = std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(hold / tiles, rows / kLeast), 256));
    a.per_split = std::max<int64_t>(64, ((rows + splits - 1) / splits + 63) / 64 * 64);
    a.splits = (int)std::max<int64_t>(1, (rows + a.per_split - 1) / a.per_split);
    return a;
}

int64_t part_w_bytes(const Args& a) { return ((int64_t)a.splits * a.n * a.k * 4 + 15) / 16 * 16; }

}  // namespace

extern "C" int64_t nori_checkpoint_grad_workspace_bytes(int dtype, int dw_dtype, int64_t rows, int32_t n, int32_t k) {
    if (rows < 0 || n < 1 || k < 1) return 0;
    const Args a = plan(dtype, dw_dtype != dtype, rows, n, k);
    return a.splits > 1 ? part_w_bytes(a) + (int64_t)a.splits * a.k_tiles * n * 4 : 0;
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
    if (dy_row_stride < 0) return fail(NORI_ERR_INVALID, "checkpoint_grad: a row stride of %lld", (long long)dy_row_stride);
    if (dy_row_stride > (1 << 24)) return fail(NORI_ERR_UNSUPPORTED, "checkpoint_grad: a row stride of %lld; up to 2^24 is taken", (long long)dy_row_stride);
    if (!dw && !db) return NORI_OK;
    if (rows > 0 && (!dy || (dw && (!codes || !scales || (uintptr_t)codes % 16))))
        return fail(NORI_ERR_INVALID, "checkpoint_grad: null or unaligned pointer");
    const bool fine = dw && dw_dtype != dtype;
    Args a = plan(dtype, fine, rows, n, k);
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
        const int64_t need = nori_checkpoint_grad_workspace_bytes(dtype, dw ? dw_dtype : dtype, rows, n, k);
        if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16)
            return fail(NORI_ERR_INVALID, "checkpoint_grad: a 16-byte aligned workspace of %lld bytes is needed", (long long)need);
        a.part_w = (float*)workspace;
        a.part_b = (float*)((char*)workspace + part_w_bytes(a));
    }
    hipStream_t stream = (hipStream_t)stream_v;
    NORI_DISPATCH_FLOAT(dtype, DT, {
        const dim3 grid((unsigned)blocks), threads(kThreads);
        if constexpr (DT == NORI_F32) {
            hipLaunchKernelGGL((grad_kernel<DT, 128, false>), grid, threads, 0, stream, a);
        } else {
            if (fine) hipLaunchKernelGGL((grad_kernel<DT, 128, true>), grid, threads, 0, stream, a);
            else if (a.tile_n == 256) hipLaunchKernelGGL((grad_kernel<DT, 256, false>), grid, threads, 0, stream, a);
            else hipLaunchKernelGGL((grad_kernel<DT, 128, false>), grid, threads, 0, stream, a);
        }
        if (a.splits > 1) {
            const int64_t items = (dw ? (int64_t)n * k : 0) + (db ? n : 0);
            hipLaunchKernelGGL((join_kernel<DT>), dim3((unsigned)std::min<int64_t>((items + kThreads - 1) / kThreads, 16 * device_cus())),
                               dim3(kThreads), 0, stream, a);
        }
    });
    return launch_status("checkpoint_grad");
}
