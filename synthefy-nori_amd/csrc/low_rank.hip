// Low-rank updates of a projection's output, each row with the adapter of its table (or none), gfx950:
//     out[i] = y[i] + (s_a x[i] A_a^T) B_a^T,   a the adapter of row i,  A_a [r, k],  B_a [n, r]
// and its gradients: dx[i] = (s_a dy[i] B_a) A_a -- the same two products with the factors' roles
// swapped -- and, with h = s_a x A_a^T and g = s_a dy B_a kept from them in fp32,
//     dA_a = sum over a's rows of g[i]^T x[i],   dB_a = sum over a's rows of dy[i]^T h[i].
//
// Rows are taken by adapter: order[] lists the rows of group 0, then of group 1, ..., a group being
// every row of the batch with one adapter id (-1: the rows without one), starts[] where each begins.
//
// HBM-bound at the ranks this is used with: e (k + 2 n) bytes against 2 r (k + n) FLOP a row. A workgroup
// therefore takes a tile of one group's rows through both products, h staying in LDS; x, the factors and y come
// straight to the registers that the matrix instructions read, h is the only thing exchanged between lanes.
#include <algorithm>
#include <type_traits>

#include "nori_common.h"

namespace {

using namespace nori;

constexpr int kThreads = 256, kWaves = kThreads / 64;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));

// What a lane holds of a matrix instruction's operand: W consecutive elements along the sum. Lane l has row
// l % 16 and elements (l / 16) * W ...; a result has column l % 16 and rows (l / 16) * 4 ....
template <int DT>
struct Mma {
    static constexpr int W = 8;
    typedef uint16_t elem;
    typedef u16x8 frag;
    static __device__ __forceinline__ f32x4 mul(frag a, frag b, f32x4 c) {
        if constexpr (DT == NORI_F16)
            return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
        else
            return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <>
struct Mma<NORI_F32> {
    static constexpr int W = 4;
    typedef float elem;
    typedef f32x4 frag;
    static __device__ __forceinline__ f32x4 mul(frag a, frag b, f32x4 c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
};

template <int DT>
__device__ __forceinline__ float widen(typename Mma<DT>::elem v) {
    if constexpr (DT == NORI_F32) return v;
    else return DT == NORI_F16 ? f16_to_f32(v) : bf16_to_f32(v);
}

template <int DT>
__device__ __forceinline__ typename Mma<DT>::elem narrow(float v) {
    if constexpr (DT == NORI_F32) return v;
    else return DT == NORI_F16 ? f32_to_f16(v) : f32_to_bf16(v);
}

// W elements at p, at any alignment; of fewer than W (`there`), zeros behind them
template <int DT>
__device__ __forceinline__ typename Mma<DT>::frag fetch(const typename Mma<DT>::elem* p) {
    typename Mma<DT>::frag f;
    __builtin_memcpy(&f, p, sizeof f);
    return f;
}

template <int DT>
__device__ __forceinline__ typename Mma<DT>::frag fetch(const typename Mma<DT>::elem* p, int there) {
    if (there >= Mma<DT>::W) return fetch<DT>(p);
    typename Mma<DT>::frag f = {};
#pragma unroll
    for (int i = 0; i < Mma<DT>::W; ++i)
        if (i < there) f[i] = p[i];
    return f;
}

// The group that a tile of `size` rows belongs to and the tile's number in it. Group g has the tiles from
// starts[g] / size + g on: enough for all of its rows, whatever the lengths, so no tile list is made. 64 groups
// are looked at a time, one a lane.
__device__ __forceinline__ int group_of_tile(const int32_t* starts, int groups, int size, int tile, int& number) {
    const int lane = threadIdx.x & 63;
    int g = 0;
    for (int base = 0; base < groups; base += 64) {
        const int i = base + lane;
        const bool before = i < groups && starts[i] / size + i <= tile;
        const int count = __popcll(__ballot(before));
        g = count ? base + count - 1 : g;
        if (count < 64) break;
    }
    number = tile - (starts[g] / size + g);
    return g;
}

struct Update {
    const void *x, *y, *a, *b;
    int64_t xs, ys, os;
    int k, n, rank, adapters;
    const float* scales;
    const int32_t *order, *starts, *ids;
    int groups;
    int columns;  // of out, a workgroup's
    void* out;
    float* h;  // [rows][rank], rows as in x; null: not kept
};

// RP: the rank rounded up to 16, 32, 64 or 128. TM rows a tile. With 64 rows each wavefront sums its own 16 rows
// of h over all of k; with 16 rows the wavefronts share the rows and split k (few rows: the latency of k counts).
// Both products put the factor's rows where results run along the lane's registers: h comes as 4 ranks a lane, out
// as W consecutive columns of a row.
// h enters the second product in two pieces of the inputs' type, high and low, which keep 22 bits of a row's
// largest element in fp16 (after a power of two that brings the row near 1, so that nothing leaves fp16's range)
// and 16 in bf16; in fp32 it stays as it is. The result, rounded once, holds at most 11 and 8 bits.
template <int DT, int RP, int TM>
__global__ void __launch_bounds__(kThreads) update_kernel(const Update u) {
    using M = Mma<DT>;
    using E = typename M::elem;
    using F = typename M::frag;
    constexpr int W = M::W, KS = 4 * W, RT = RP / 16, TILES = TM / 16;
    constexpr bool F32 = DT == NORI_F32;
    constexpr int PIECES = F32 ? 1 : 2;
    constexpr int PITCH = RP + W;  // of a row of h in LDS, in elements
    __shared__ __align__(16) E hs[PIECES][TM][PITCH];
    __shared__ float factor[TM];
    __shared__ f32x4 part[TM == 16 ? kWaves : 1][TM == 16 ? RT : 1][64];

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, g = lane >> 4;
    int number;
    const int group = group_of_tile(u.starts, u.groups, TM, blockIdx.x, number);
    const int end = u.starts[group + 1];
    const int64_t first64 = (int64_t)u.starts[group] + (int64_t)number * TM;
    if (first64 >= end) return;
    const int first = (int)first64;
    const int id = u.ids[group];
    const bool active = id >= 0 && id < u.adapters;

    if (active) {
        // ---- h = s x A^T
        const int mine = TM == 16 ? 0 : 16 * wave;
        const int64_t row = u.order[min(first + mine + m, end - 1)];
        const E* x = reinterpret_cast<const E*>(u.x) + row * u.xs + W * g;
        const E* a = reinterpret_cast<const E*>(u.a) + (int64_t)id * u.rank * u.k + W * g;
        f32x4 acc[RT];
        const E* at[RT];
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
            at[t] = a + (int64_t)min(16 * t + m, u.rank - 1) * u.k;  // ranks past the last are dropped below
        }
        const int whole = u.k / KS;
        constexpr int kStep = TM == 16 ? kWaves : 1;
#pragma unroll 4
        for (int s = TM == 16 ? wave : 0; s < whole; s += kStep) {
            const F xf = fetch<DT>(x + s * KS);
#pragma unroll
            for (int t = 0; t < RT; ++t) acc[t] = M::mul(fetch<DT>(at[t] + s * KS), xf, acc[t]);
        }
        if (u.k % KS && (TM != 16 || wave == whole % kWaves)) {
            const int there = u.k - whole * KS - W * g;
            const F xf = fetch<DT>(x + whole * KS, there);
#pragma unroll
            for (int t = 0; t < RT; ++t) acc[t] = M::mul(fetch<DT>(at[t] + whole * KS, there), xf, acc[t]);
        }
        if constexpr (TM == 16) {
#pragma unroll
            for (int t = 0; t < RT; ++t) part[wave][t][lane] = acc[t];
            __syncthreads();
#pragma unroll
            for (int t = 0; t < RT; ++t)
                acc[t] = (part[0][t][lane] + part[1][t][lane]) + (part[2][t][lane] + part[3][t][lane]);
        }
        const float s = u.scales ? u.scales[id] : 1.0f;
        float largest = 0.f;
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                acc[t][j] = 16 * t + 4 * g + j < u.rank ? acc[t][j] * s : 0.f;
                const float v = fabsf(acc[t][j]);
                largest = v < __builtin_inff() ? fmaxf(largest, v) : largest;
            }
        if (TM != 16 || wave == 0) {
            if (u.h && blockIdx.y == 0 && first + mine + m < end) {
                float* h = u.h + row * u.rank;
#pragma unroll
                for (int t = 0; t < RT; ++t)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (16 * t + 4 * g + j < u.rank) h[16 * t + 4 * g + j] = acc[t][j];
            }
            float up = 1.0f, down = 1.0f;
            if constexpr (DT == NORI_F16) {
                largest = fmaxf(largest, __shfl_xor(largest, 16, 64));
                largest = fmaxf(largest, __shfl_xor(largest, 32, 64));
                // 2^e, the largest element's binade, and 2^-e; e within what both are normal for
                const int e = min(max((int)(__float_as_uint(largest) >> 23) - 127, -120), 120);
                up = __uint_as_float((uint32_t)(127 + e) << 23);
                down = __uint_as_float((uint32_t)(127 - e) << 23);
            }
            if (g == 0) factor[mine + m] = up;
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float v = acc[t][j] * down;
                    const E high = narrow<DT>(v);
                    hs[0][mine + m][16 * t + 4 * g + j] = high;
                    if constexpr (!F32) {
                        const float rest = v - widen<DT>(high);
                        hs[1][mine + m][16 * t + 4 * g + j] = fabsf(v) < __builtin_inff() ? narrow<DT>(rest) : E(0);
                    }
                }
        }
        __syncthreads();
    } else if (u.y == u.out) {
        return;  // the rows stay as they are
    }

    // ---- out = y + h B^T
    constexpr int PER = W / 4;        // tiles of 16 columns that make a lane's W consecutive ones
    constexpr int NT = 4, NV = NT / PER;  // tiles and vectors a step
    constexpr int KC = F32 ? RP / 16 : (RP + 31) / 32;  // operands along the rank
    int64_t yrow[TILES], orow[TILES];
#pragma unroll
    for (int r = 0; r < TILES; ++r) {
        const int64_t row = u.order[min(first + 16 * r + m, end - 1)];
        yrow[r] = row * u.ys;
        orow[r] = row * u.os;
    }
    const E* b = reinterpret_cast<const E*>(u.b) + (int64_t)(active ? id : 0) * u.n * u.rank;
    const int64_t behind = (int64_t)(u.adapters - (active ? id : 0)) * u.n * u.rank;  // elements from b to the bank's end
    const int stop = min(u.n, ((int)blockIdx.y + 1) * u.columns);
    for (int n0 = blockIdx.y * u.columns + 64 * wave; n0 < stop; n0 += 64 * kWaves) {
        F yv[TILES][NV];
#pragma unroll
        for (int r = 0; r < TILES; ++r)
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int c = n0 + 16 * PER * v + W * g;
                yv[r][v] = F{};
                if (u.y) yv[r][v] = fetch<DT>(reinterpret_cast<const E*>(u.y) + yrow[r] + c, u.n - c);
            }
        f32x4 acc[TILES][NT];
#pragma unroll
        for (int r = 0; r < TILES; ++r)
#pragma unroll
            for (int t = 0; t < NT; ++t) acc[r][t] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (active) {
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                // a rank of 16 fills half an operand: its other half takes the low pieces
                const int rank0 = (!F32 && RP == 16 ? W * (g & 1) : 4 * W * c + W * g);
                F bf[NT];
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const int n = min(n0 + 16 * PER * (t / PER) + W * (m >> 2) + 4 * (t % PER) + (m & 3), u.n - 1);
                    const int64_t i = (int64_t)n * u.rank + rank0;
                    bf[t] = F{};
                    if (rank0 < u.rank) {
                        if (i + W <= behind) bf[t] = fetch<DT>(b + i);  // past its rank's end: dropped next
                        else bf[t] = fetch<DT>(b + i, u.rank - rank0);
#pragma unroll
                        for (int e = 0; e < W; ++e)
                            if (rank0 + e >= u.rank) bf[t][e] = 0;
                    }
                }
#pragma unroll
                for (int p = 0; p < (!F32 && RP == 16 ? 1 : PIECES); ++p)
#pragma unroll
                    for (int r = 0; r < TILES; ++r) {
                        const int piece = !F32 && RP == 16 ? g >> 1 : p;
                        const F hf = *reinterpret_cast<const F*>(&hs[piece][16 * r + m][rank0]);
#pragma unroll
                        for (int t = 0; t < NT; ++t) acc[r][t] = M::mul(bf[t], hf, acc[r][t]);
                    }
            }
        }
#pragma unroll
        for (int r = 0; r < TILES; ++r) {
            if (first + 16 * r + m >= end) continue;
            const float f = active ? factor[16 * r + m] : 0.f;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int c = n0 + 16 * PER * v + W * g;
                if (c >= stop) continue;
                F o;
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    // rows without an adapter keep y's bits
                    o[e] = active ? narrow<DT>(widen<DT>(yv[r][v][e]) + f * acc[r][v * PER + e / 4][e % 4]) : yv[r][v][e];
                }
                E* to = reinterpret_cast<E*>(u.out) + orow[r] + c;
                if (c + W <= u.n) {
                    __builtin_memcpy(to, &o, sizeof o);
                } else {
#pragma unroll
                    for (int e = 0; e < W; ++e)
                        if (c + e < u.n) to[e] = o[e];
                }
            }
        }
    }
}

// [adapter][rows][cols] -> [adapter][cols][rows] of the groups' adapters, 32 x 32 elements a workgroup
template <typename E>
__global__ void __launch_bounds__(kThreads) transpose_kernel(const E* from, E* to, int rows, int cols, const int32_t* ids,
                                                             int adapters) {
    __shared__ E tile[32][33];
    const int id = ids[blockIdx.z];
    if (id < 0 || id >= adapters) return;
    const int64_t base = (int64_t)id * rows * cols;
    const int c = threadIdx.x % 32, r = threadIdx.x / 32, row0 = blockIdx.y * 32, col0 = blockIdx.x * 32;
#pragma unroll
    for (int i = r; i < 32; i += 8)
        if (row0 + i < rows && col0 + c < cols) tile[i][c] = from[base + (int64_t)(row0 + i) * cols + col0 + c];
    __syncthreads();
#pragma unroll
    for (int i = r; i < 32; i += 8)
        if (col0 + i < cols && row0 + c < rows) to[base + (int64_t)(col0 + i) * rows + row0 + c] = tile[c][i];
}

struct Grad {
    const void* t;   // [rows][cols]
    const float* h;  // [rows][rank]
    int64_t ts;
    int cols, rank, adapters;
    const int32_t *order, *starts, *ids;
    int groups;
    void* out;  // [adapters][cols][rank], transposed: [adapters][rank][cols]
    int64_t o_col, o_rank;
    int part;        // rows of one; a multiple of 128
    float* partial;  // [parts of the groups with more than one][cols][rank]
};

// Where the partial sums of a group with several parts begin: 2 starts / part is enough for the ones before it,
// since a length above `part` has at most twice length / part, less one, rounded up.
__device__ __forceinline__ int64_t partial_of(const Grad& q, int group) { return 2 * (int64_t)q.starts[group] / q.part; }

__device__ __forceinline__ void store_grad(const Grad& q, int dt, int id, int c, int j, float v) {
    const int64_t i = (int64_t)id * q.cols * q.rank + c * q.o_col + j * q.o_rank;
    if (dt == NORI_F32) reinterpret_cast<float*>(q.out)[i] = v;
    else reinterpret_cast<uint16_t*>(q.out)[i] = dt == NORI_F16 ? f32_to_f16(v) : f32_to_bf16(v);
}

// t^T h over one part of a group's rows: 128 (fp32: 64) columns by up to 64 ranks a workgroup, whose wavefronts
// take every fourth step of rows and add their sums in LDS, in order.
// The sum runs over rows, which t has apart. 16-bit: a lane reads 16 bytes of each of 8 rows and turns the 8 x 8
// block in registers, so that it holds 8 rows of one column for each of 8 instructions; column t of a lane's
// block belongs to instruction t. fp32: an instruction takes 4 rows, no turning. h, in fp32, enters in two pieces
// of the 16-bit type as in the update; a power of two per wavefront that follows the largest element so far keeps
// fp16's pieces in range (sums so far are brought to a new one).
template <int DT, int RT>
__global__ void __launch_bounds__(kThreads) grad_kernel(const Grad q) {
    using M = Mma<DT>;
    using E = typename M::elem;
    using F = typename M::frag;
    constexpr bool F32 = DT == NORI_F32;
    constexpr int W = M::W, CT = W;            // a lane's columns, an instruction each
    constexpr int STEP = F32 ? 4 : 32;         // rows of a step
    constexpr int U = F32 ? 4 : 1;             // steps whose loads go together
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, g = lane >> 4;
    int number;
    const int group = group_of_tile(q.starts, q.groups, q.part, blockIdx.x, number);
    const int begin = q.starts[group], last = q.starts[group + 1];
    const int64_t first64 = (int64_t)begin + (int64_t)number * q.part;
    const int id = q.ids[group];
    if (first64 >= last || id < 0 || id >= q.adapters) return;
    const int first = (int)first64, end = min(last, first + q.part);
    const int c0 = blockIdx.y * 16 * W + W * m, j0 = blockIdx.z * 16 * RT;
    const E* t = reinterpret_cast<const E*>(q.t) + c0;
    const int there = q.cols - c0;

    f32x4 acc[RT][CT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int i = 0; i < CT; ++i) acc[r][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float up = 1.0f, down = 1.0f;
    float reach = 0.f;  // elements below it fit the present power of two
    constexpr int EACH = F32 ? 1 : 8;  // rows a lane holds of a step
    for (int p0 = first + wave * STEP * U; p0 < end; p0 += STEP * U * kWaves) {
        F raw[U][EACH];
        float h[U][EACH][RT];
#pragma unroll
        for (int s = 0; s < U; ++s)
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                const int p = p0 + STEP * s + EACH * g + i;
                const int64_t row = q.order[min(p, end - 1)];
                raw[s][i] = F{};
                if (p < end) raw[s][i] = fetch<DT>(t + row * q.ts, there);
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    const int j = j0 + 16 * r + m;
                    h[s][i][r] = p < end && j < q.rank ? q.h[row * q.rank + j] : 0.f;
                }
            }
        if constexpr (F32) {
#pragma unroll
            for (int s = 0; s < U; ++s)
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int i = 0; i < CT; ++i)
                        acc[r][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(raw[s][0][i], h[s][0][r], acc[r][i], 0, 0, 0);
        } else {
            if constexpr (DT == NORI_F16) {
                float largest = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int r = 0; r < RT; ++r) {
                        const float v = fabsf(h[0][i][r]);
                        largest = v < __builtin_inff() ? fmaxf(largest, v) : largest;
                    }
#pragma unroll
                for (int off = 32; off > 0; off >>= 1) largest = fmaxf(largest, __shfl_xor(largest, off, 64));
                if (largest > reach) {  // the same in every lane
                    const int e = min(max((int)(__float_as_uint(largest) >> 23) - 127 - 8, -110), 110);
                    const float to = __uint_as_float((uint32_t)(127 - e) << 23);
                    const float change = reach > 0.f ? to * up : 0.f;  // no sums yet: they are zero
#pragma unroll
                    for (int r = 0; r < RT; ++r)
#pragma unroll
                        for (int i = 0; i < CT; ++i) acc[r][i] = reach > 0.f ? acc[r][i] * change : acc[r][i];
                    up = __uint_as_float((uint32_t)(127 + e) << 23);
                    down = to;
                    reach = up * 512.0f;  // scaled: below 2^9, the pieces of the smallest that counts above 2^-24
                }
            }
            F high[RT], low[RT];
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float v = h[0][i][r] * down;
                    high[r][i] = narrow<DT>(v);
                    low[r][i] = fabsf(v) < __builtin_inff() ? narrow<DT>(v - widen<DT>(high[r][i])) : E(0);
                }
#pragma unroll
            for (int i = 0; i < CT; ++i) {
                F col;
#pragma unroll
                for (int e = 0; e < 8; ++e) col[e] = raw[0][e][i];
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    acc[r][i] = M::mul(col, high[r], acc[r][i]);
                    acc[r][i] = M::mul(col, low[r], acc[r][i]);
                }
            }
        }
    }
    // the wavefronts' sums, a rank tile at a time. acc[r][i][j] of lane (m, g): column W (4 g + j) + i, rank 16 r + m
    __shared__ f32x4 sums[kWaves][CT][64];
    const bool whole = last - begin <= q.part;
    float* part = whole ? nullptr : q.partial + (partial_of(q, group) + number) * q.cols * q.rank;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < CT; ++i) sums[wave][i][lane] = acc[r][i] * up;
        __syncthreads();
        for (int i = wave; i < CT; i += kWaves) {
            const f32x4 v = (sums[0][i][lane] + sums[1][i][lane]) + (sums[2][i][lane] + sums[3][i][lane]);
            const int j = j0 + 16 * r + m;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int c = blockIdx.y * 16 * W + W * (4 * g + e) + i;
                if (c >= q.cols || j >= q.rank) continue;
                if (whole) store_grad(q, DT, id, c, j, v[e]);
                else part[(int64_t)c * q.rank + j] = v[e];
            }
        }
    }
}

// the parts of the groups that have several, in their order
__global__ void __launch_bounds__(kThreads) grad_join_kernel(const Grad q, int dt) {
    const int group = blockIdx.y, id = q.ids[group];
    const int length = q.starts[group + 1] - q.starts[group];
    const int64_t size = (int64_t)q.cols * q.rank, i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (length <= q.part || id < 0 || id >= q.adapters || i >= size) return;
    const float* part = q.partial + partial_of(q, group) * size + i;
    const int parts = (length + q.part - 1) / q.part;
    float v = 0.f;
#pragma unroll 8
    for (int p = 0; p < parts; ++p) v += part[p * size];
    store_grad(q, dt, id, (int)(i / q.rank), (int)(i % q.rank), v);
}

// Rows of a part: about four workgroups a compute unit, and no part so short that its sums cost as much as its rows
// (8 rank bytes a column, twice, against 2 to 4 a row).
int part_of(int64_t rows, int cols, int rank, int dtype) {
    const int wide = dtype == NORI_F32 ? 64 : 128;
    const int64_t chunks = (int64_t)((cols + wide - 1) / wide) * ((rank + 63) / 64);
    const int64_t want = rows * chunks / (4 * (int64_t)device_cus());
    return (int)std::min<int64_t>(std::max<int64_t>((want + 127) / 128 * 128, 256), 8192);
}

bool is_float(int dt) { return dt == NORI_F32 || dt == NORI_F16 || dt == NORI_BF16; }

int check(const char* what, int dtype, int64_t rows, int32_t groups, int32_t k, int32_t n, int32_t rank, int32_t adapters) {
    if (!is_float(dtype)) return fail(NORI_ERR_UNSUPPORTED, "%s: unsupported dtype %s", what, dtype_name(dtype));
    if (rows < 0 || groups < 0 || k <= 0 || n <= 0 || adapters <= 0)
        return fail(NORI_ERR_INVALID, "%s: bad shape (%lld rows, %d -> %d, %d adapters)", what, (long long)rows, k, n, adapters);
    if (rank <= 0 || rank > NORI_LOW_RANK_MAX)
        return fail(rank <= 0 ? NORI_ERR_INVALID : NORI_ERR_UNSUPPORTED, "%s: rank %d (1 to %d)", what, rank, NORI_LOW_RANK_MAX);
    if (rows > (int64_t)1 << 29) return fail(NORI_ERR_UNSUPPORTED, "%s: too many rows", what);
    if (groups > 65535) return fail(NORI_ERR_UNSUPPORTED, "%s: %d adapters in one call (65535 at most)", what, groups);
    return NORI_OK;
}

}  // namespace

extern "C" int64_t nori_low_rank_workspace_bytes(int dtype, int32_t k, int32_t n, int32_t rank, int32_t adapters) {
    return (int64_t)adapters * rank * ((int64_t)k + n) * dtype_size(dtype);
}

extern "C" int nori_low_rank_update(const void* x, int dtype, int64_t rows, int32_t k, int64_t x_row_stride, const void* y,
                                    int64_t y_row_stride, const void* a, const void* b, int32_t transposed,
                                    const float* scales, int32_t adapters, int32_t rank, int32_t n, const int32_t* order,
                                    const int32_t* starts, const int32_t* ids, int32_t groups, void* out,
                                    int64_t out_row_stride, float* h, void* workspace, int64_t workspace_bytes,
                                    void* stream_v) {
    clear_error();
    if (int rc = check("low_rank_update", dtype, rows, groups, k, n, rank, adapters)) return rc;
    if (rows == 0) return NORI_OK;
    if (!x || !a || !b || !order || !starts || !ids || !out || groups <= 0)
        return fail(NORI_ERR_INVALID, "low_rank_update: null pointer");
    if (out_row_stride < n && rows > 1) return fail(NORI_ERR_INVALID, "low_rank_update: rows of out overlap");
    if (out == y && out_row_stride != y_row_stride && rows > 1)
        return fail(NORI_ERR_INVALID, "low_rank_update: out is y, at another row stride");
    if (transposed && (!workspace || workspace_bytes < nori_low_rank_workspace_bytes(dtype, k, n, rank, adapters)))
        return fail(NORI_ERR_INVALID, "low_rank_update: workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
                    (long long)nori_low_rank_workspace_bytes(dtype, k, n, rank, adapters));
    Update u{x, y, a, b, x_row_stride, y_row_stride, out_row_stride, k, n, rank, adapters, scales, order, starts, ids, groups,
             0, out, h};
    hipStream_t stream = (hipStream_t)stream_v;
    if (transposed) {
        // the factors as the products read them: rows along their sums
        auto turn = [&](auto e) {
            using E = decltype(e);
            E* at = reinterpret_cast<E*>(workspace);
            E* bt = at + (int64_t)adapters * rank * k;
            hipLaunchKernelGGL((transpose_kernel<E>), dim3((rank + 31) / 32, (k + 31) / 32, groups), dim3(kThreads), 0, stream,
                               reinterpret_cast<const E*>(a), at, k, rank, ids, adapters);
            hipLaunchKernelGGL((transpose_kernel<E>), dim3((n + 31) / 32, (rank + 31) / 32, groups), dim3(kThreads), 0, stream,
                               reinterpret_cast<const E*>(b), bt, rank, n, ids, adapters);
            u.a = at;
            u.b = bt;
        };
        if (dtype == NORI_F32) turn(float{});
        else turn(uint16_t{});
    }
    const int cus = device_cus();
    auto go = [&](auto DT_, auto RP_, auto TM_) {
        constexpr int DT = decltype(DT_)::value, RP = decltype(RP_)::value, TM = decltype(TM_)::value;
        const int64_t tiles = rows / TM + groups;
        // out's columns are shared among workgroups, each with an h of its own, while there are few tiles
        const int most = (n + 64 * kWaves - 1) / (64 * kWaves);
        const int split = (int)std::min<int64_t>(most, std::max<int64_t>(1, 2 * cus / tiles));
        const int steps = (most + split - 1) / split;
        u.columns = steps * 64 * kWaves;
        // tiles in multiples of 8: a tile's workgroups stay on one XCD, whose L2 holds its x
        const unsigned gx = (unsigned)((tiles + 7) / 8 * 8), gy = (unsigned)((most + steps - 1) / steps);
        hipLaunchKernelGGL((update_kernel<DT, RP, TM>), dim3(gx, gy), dim3(kThreads), 0, stream, u);
    };
    auto by_tile = [&](auto DT_, auto RP_) {
        if (rows <= 16 * (int64_t)groups) go(DT_, RP_, std::integral_constant<int, 16>{});
        else go(DT_, RP_, std::integral_constant<int, 64>{});
    };
    NORI_DISPATCH_FLOAT(dtype, DT, {
        constexpr std::integral_constant<int, DT> DT_{};
        if (rank <= 16) by_tile(DT_, std::integral_constant<int, 16>{});
        else if (rank <= 32) by_tile(DT_, std::integral_constant<int, 32>{});
        else if (rank <= 64) by_tile(DT_, std::integral_constant<int, 64>{});
        else by_tile(DT_, std::integral_constant<int, 128>{});
    });
    return launch_status("low_rank_update");
}

extern "C" int64_t nori_low_rank_weight_grad_workspace_bytes(int dtype, int64_t rows, int32_t cols, int32_t rank,
                                                             int64_t longest) {
    if (rows <= 0 || cols <= 0 || rank <= 0) return 0;
    const int part = part_of(rows, cols, rank, dtype);
    return longest <= part ? 0 : (2 * rows / part + 1) * cols * rank * 4;
}

extern "C" int nori_low_rank_weight_grad(const void* t, int dtype, int64_t rows, int32_t cols, int64_t t_row_stride,
                                         const float* h, int32_t rank, int32_t adapters, const int32_t* order,
                                         const int32_t* starts, const int32_t* ids, int32_t groups, int64_t longest,
                                         int32_t transposed, void* out, void* workspace, int64_t workspace_bytes,
                                         void* stream_v) {
    clear_error();
    if (int rc = check("low_rank_weight_grad", dtype, rows, groups, cols, 1, rank, adapters)) return rc;
    if (rows == 0) return NORI_OK;
    if (!t || !h || !order || !starts || !ids || !out || groups <= 0)
        return fail(NORI_ERR_INVALID, "low_rank_weight_grad: null pointer");
    if (longest < 1 || longest > rows)
        return fail(NORI_ERR_INVALID, "low_rank_weight_grad: a longest group of %lld rows of %lld", (long long)longest, (long long)rows);
    const int64_t need = nori_low_rank_weight_grad_workspace_bytes(dtype, rows, cols, rank, longest);
    if (need && (!workspace || (uintptr_t)workspace % 4 || workspace_bytes < need))
        return fail(NORI_ERR_INVALID, "low_rank_weight_grad: workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
                    (long long)need);
    Grad q{t, h, t_row_stride, cols, rank, adapters, order, starts, ids, groups, out, rank, 1, part_of(rows, cols, rank, dtype),
           reinterpret_cast<float*>(workspace)};
    if (transposed) q.o_col = 1, q.o_rank = cols;
    hipStream_t stream = (hipStream_t)stream_v;
    const int64_t parts = rows / q.part + groups;
    auto go = [&](auto DT_, auto RT_) {
        constexpr int DT = decltype(DT_)::value, RT = decltype(RT_)::value, WIDE = 16 * Mma<DT>::W;
        hipLaunchKernelGGL((grad_kernel<DT, RT>),
                           dim3((unsigned)parts, (unsigned)((cols + WIDE - 1) / WIDE), (unsigned)((rank + 16 * RT - 1) / (16 * RT))),
                           dim3(kThreads), 0, stream, q);
    };
    NORI_DISPATCH_FLOAT(dtype, DT, {
        constexpr std::integral_constant<int, DT> DT_{};
        if (rank <= 16) go(DT_, std::integral_constant<int, 1>{});
        else if (rank <= 32) go(DT_, std::integral_constant<int, 2>{});
        else go(DT_, std::integral_constant<int, 4>{});
    });
    if (need) {
        const int64_t size = (int64_t)cols * rank;
        hipLaunchKernelGGL(grad_join_kernel, dim3((unsigned)((size + kThreads - 1) / kThreads), groups), dim3(kThreads), 0, stream,
                           q, dtype);
    }
    return launch_status("low_rank_weight_grad");
}
