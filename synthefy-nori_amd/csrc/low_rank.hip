// Low-rank updates of a projection's output, each row with the adapter of its table (or none), gfx950:
//     out[i] = y[i] + (s_a x[i] A_a^T) B_a^T,   a the adapter of row i,  A_a [r, k],  B_a [n, r]
// and its gradients: dx[i] = (s_a dy[i] B_a) A_a -- the same two products with the factors' roles
// swapped -- and, with h = s_a x A_a^T and g = s_a dy B_a kept from them in fp32,
//     dA_a = sum over a's rows of g[i]^T x[i],   dB_a = sum over a's rows of dy[i]^T h[i].
//
// Rows are taken by adapter: order[] lists the rows of group 0, then of group 1, ..., a group being
// every row of the batch with one adapter id (-1: the rows without one), starts[] where each begins.
//
// HBM-bound at the ranks this is used with: e (k + 2 n) bytes against 2 r (k + n) FLOP a row. A tile of one
// group's rows therefore goes through both products in one kernel, h staying in LDS.
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

// v as two numbers of a 16-bit type, high and low: v cut to the type's bits, and what that leaves, rounded (2^-22 of v in
// fp16, 2^-16 in bf16). Both have v's sign, and low is zero only where v is: times an infinity each gives the infinity that v
// gives. The low that stands for zero is fp16's smallest number, and bf16's smallest normal one where that is 2^-16 of v or less.
template <int DT>
__device__ __forceinline__ void split(float v, uint16_t& high, uint16_t& low) {
    if constexpr (DT == NORI_F16) high = __builtin_bit_cast(uint16_t, __builtin_amdgcn_cvt_pkrtz(v, 0.f)[0]);
    else high = (uint16_t)(__float_as_uint(v) >> 16);
    low = fabsf(v) < __builtin_inff() ? narrow<DT>(v - widen<DT>(high)) : high;
    const uint16_t least = DT == NORI_F16 || fabsf(v) < 0x1p-110f ? 0x0001 : 0x0080;
    if (v != 0.f && (low & 0x7fff) < least) low = (uint16_t)(least | (__float_as_uint(v) >> 16 & 0x8000));
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

// What this wavefront wrote to LDS is what its lanes read after this: LDS serves a wavefront in order, the compiler
// has to keep it.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
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
    void *pa, *pb;  // the groups' factors as operands (Packed), or null: read where they lie
};

// The factors in the order that the matrix instructions take them: an operand's 64 lanes side by side, ranks and ends
// padded with zeros. The factor of the first product: [step along k][rank tile], KB elements of k (128 bytes of a row of
// x) rounded up; of the second: [tile of 16 columns][operand along the rank], 64 columns rounded up. Read from where
// they lie, an operand's lanes are 16 rows apart, which takes the address units four times as long.
template <int DT, int RP>
struct Packed {
    using M = Mma<DT>;
    static constexpr int W = M::W, KS = 4 * W, KB = 8 * W, RT = RP / 16;
    static constexpr bool F32 = DT == NORI_F32;
    static constexpr bool HALF = !F32 && RP == 16;  // a rank of 16 fills half an operand: its other half takes the low pieces
    static constexpr int KC = F32 ? RP / 16 : (RP + 31) / 32;
    static constexpr int PER = W / 4;  // tiles of 16 columns that make a lane's W consecutive ones

    __host__ __device__ static int batches(int k) { return (k + KB - 1) / KB; }
    __host__ __device__ static int tiles(int n) { return (n + 63) / 64 * 4; }
    static constexpr int LANES = HALF ? 32 : 64;  // of an operand of the second product
    // vectors of one adapter
    __host__ __device__ static int64_t first(int k) { return (int64_t)batches(k) * 2 * RT * 64; }
    __host__ __device__ static int64_t second(int n) { return (int64_t)tiles(n) * KC * LANES; }
    // of tile t, the column of a lane's row m: its result then is W columns side by side, in lanes of one m 16 PER apart
    __device__ static int column(int t, int m) { return 16 * PER * (t / PER) + W * (m >> 2) + 4 * (t % PER) + (m & 3); }
    __device__ static int rank_of(int c, int g) { return HALF ? W * (g & 1) : KS * c + W * g; }
};

// a lane's W elements of an operand a thread
template <int DT, int RP>
__global__ void __launch_bounds__(kThreads) pack_kernel(const Update u, int transposed) {
    using P = Packed<DT, RP>;
    using E = typename Mma<DT>::elem;
    const int group = blockIdx.y, id = u.ids[group];
    if (id < 0 || id >= u.adapters) return;
    const int64_t first = P::first(u.k), i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    const int lane = (int)(i % 64), m = lane & 15, g = lane >> 4;  // (first is a multiple of 64)
    using F = typename Mma<DT>::frag;
    // elements i0 ... of a row of `count` at a stride, zeros behind its end; every load before the first use
    auto gather = [](const E* p, int i0, int count, int64_t stride) {
        if (stride == 1 && i0 + P::W <= count) return fetch<DT>(p + i0);
        E v[P::W];
#pragma unroll
        for (int e = 0; e < P::W; ++e) v[e] = p[min(i0 + e, count - 1) * stride];
        F f;
#pragma unroll
        for (int e = 0; e < P::W; ++e) f[e] = i0 + e < count ? v[e] : E(0);
        return f;
    };
    F f = {};
    if (i < first) {
        const int op = (int)(i / 64), j = 16 * (op % P::RT) + m, k0 = op / P::RT * P::KS + P::W * g;
        const E* a = reinterpret_cast<const E*>(u.a) + (int64_t)id * u.rank * u.k;
        if (j < u.rank) f = gather(a + (transposed ? (int64_t)j : (int64_t)j * u.k), k0, u.k, transposed ? u.rank : 1);
        reinterpret_cast<typename Mma<DT>::frag*>(u.pa)[group * first + i] = f;
        return;
    }
    const int64_t second = P::second(u.n), at = i - first;
    if (at >= second) return;
    const int op = (int)(at / P::LANES), n = P::column(op / P::KC, m), rank0 = P::rank_of(op % P::KC, g);
    const E* b = reinterpret_cast<const E*>(u.b) + (int64_t)id * u.n * u.rank;
    if (n < u.n) f = gather(b + (transposed ? (int64_t)n : (int64_t)n * u.rank), rank0, u.rank, transposed ? u.n : 1);
    reinterpret_cast<typename Mma<DT>::frag*>(u.pb)[group * second + at] = f;
}

// A lane's ranks of h, rank 16 t + 4 g + j of row m in acc[t][j], times s: kept in fp32 (`keep`, null: not), and put
// into LDS as the second product takes them, in two pieces of the inputs' type, high and low, which keep an element to
// 2^-22 of itself in fp16 and to 2^-16 in bf16; in fp32 h stays as it is. The result, rounded once, is kept to 2^-11 and
// 2^-8. fp16's are taken after a power of two that brings the row's largest element to 2^14, the top of its range: what
// is lost below its subnormal numbers is 2^-38 of that element, and a second product sums 2^15 2^16 128 at most.
template <int DT, int RT, int ROWS, int PITCH, int PIECES>
__device__ __forceinline__ void put_h(f32x4 (&acc)[RT], float s, int rank, float* keep, int g, int row,
                                      typename Mma<DT>::elem (&hs)[PIECES][ROWS][PITCH], float (&factor)[ROWS]) {
    float largest = 0.f;
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool in = 16 * t + 4 * g + j < rank;
            acc[t][j] = in ? acc[t][j] * s : 0.f;
            if (in && keep) keep[16 * t + 4 * g + j] = acc[t][j];
            const float v = fabsf(acc[t][j]);
            largest = v < __builtin_inff() ? fmaxf(largest, v) : largest;
        }
    float up = 1.0f, down = 1.0f;
    if constexpr (DT == NORI_F16) {
        largest = fmaxf(largest, __shfl_xor(largest, 16, 64));
        largest = fmaxf(largest, __shfl_xor(largest, 32, 64));
        // e: the largest element's binade less 14; within what 2^e and 2^-e are normal for
        const int e = min(max((int)(__float_as_uint(largest) >> 23) - 127, -112), 127) - 14;
        up = __uint_as_float((uint32_t)(127 + e) << 23);
        down = __uint_as_float((uint32_t)(127 - e) << 23);
    }
    if (g == 0) factor[row] = up;
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float v = acc[t][j] * down;
            if constexpr (PIECES == 2) split<DT>(v, hs[0][row][16 * t + 4 * g + j], hs[1][row][16 * t + 4 * g + j]);
            else hs[0][row][16 * t + 4 * g + j] = v;
        }
}

// A workgroup's LDS in update_kernel, sizes in elements.
template <int DT, int RP, int R>
struct UpdateLds {
    using P = Packed<DT, RP>;
    using E = typename Mma<DT>::elem;
    static constexpr int PIECES = P::F32 ? 1 : 2, PITCH = RP + P::W;  // of a row of h
    static constexpr int CB = P::KB;                                  // columns of a window: 128 bytes
    static constexpr int RING = 2 * CB, OUT = RING + P::W + 4;        // a row of the result: two blocks, the first W columns again
    static constexpr int XROW = P::KB + P::W;                         // a row of x
    union Stage {
        E x[2][16 * R][XROW];
        float out[16 * R][OUT];
    };
    alignas(16) Stage stage[kWaves];
    alignas(16) E hs[kWaves][PIECES][16 * R][PITCH];
    float factor[kWaves][16 * R];
    // workgroups that a compute unit's registers hold, where that is more than one or two, and whether more are better where
    // fewer would end as soon
    static constexpr int HELD = RP > 32 ? 0 : P::F32 ? 4 : 3;
    static constexpr bool MORE = P::F32 || RP == 16;
};

// Many rows. A wavefront takes 16 R rows of one group through both products by itself; the four of a workgroup share
// the factors' cache lines only. R is 1, or 2 for ranks above 32, where reading the factors costs more than the
// registers and the LDS of twice the rows (65536 rows 1408 -> 1408 rank 64 fp16: 165 us with 1, 147 with 2; 560 -> 1680
// rank 16: 132 and 173), unless that leaves too many compute units idle (short_round).
// x, y and out pass through the wavefront's LDS between the order they lie in memory (8 lanes a run of 128 bytes) and
// the operands' (a lane a row), and the packed factors are read as operands: every access takes the address units as few
// cycles as its bytes do.
// y and out go in windows of 128 bytes that begin where a line of out does, each row at columns of its own: the
// result's last two blocks of columns stay in LDS. Windows at the same columns of every row leave lines half written
// where rows are not whole lines (65536 rows of 1680 fp16, y to out alone: 136 us against 95, of 999: 65 against 45).
// RP: the rank rounded up to 16, 32, 64 or 128.
template <int DT, int RP, int R>
__global__ void __launch_bounds__(kThreads, RP <= 32 ? 3 : 1) update_kernel(const Update u) {
    using M = Mma<DT>;
    using P = Packed<DT, RP>;
    using E = typename M::elem;
    using F = typename M::frag;
    using L = UpdateLds<DT, RP, R>;
    constexpr int W = M::W, RT = P::RT, KB = P::KB, KC = P::KC, PER = P::PER;
    constexpr int PIECES = L::PIECES, PITCH = L::PITCH, CB = L::CB, NT = CB / 16, RING = L::RING, OUT = L::OUT, XROW = L::XROW;
    constexpr int AHEAD = !P::F32 && RP == 16 ? 3 : 2;  // batches of x, windows of y asked for in advance
    __shared__ L lds;

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, g = lane >> 4;
    int number;
    const int group = group_of_tile(u.starts, u.groups, 64 * R, blockIdx.x, number);
    const int end = u.starts[group + 1];
    const int64_t first64 = (int64_t)u.starts[group] + ((int64_t)number * 64 + 16 * wave) * R;
    if (first64 >= end) return;
    const int first = (int)first64;
    const int id = u.ids[group];
    const bool active = id >= 0 && id < u.adapters;
    if (!active && u.y == u.out) return;  // the rows stay as they are

    // this lane's 2 R rows in memory's order, its elements of a run, and where the rows' windows begin
    const int r0 = lane >> 3, lc = W * (lane & 7);
    const E* yrow[2 * R];
    E* orow[2 * R];
    int begin[2 * R];
    int shift = 0, any = 0;
#pragma unroll
    for (int i = 0; i < 2 * R; ++i) {
        const int64_t row = u.order[min(first + 8 * i + r0, end - 1)];
        orow[i] = reinterpret_cast<E*>(u.out) + row * u.os;
        yrow[i] = reinterpret_cast<const E*>(u.y) + row * u.ys;
        const int past = (int)((uintptr_t)orow[i] / sizeof(E) % CB);
        begin[i] = lc - past;
        shift = max(shift, past);
        any |= begin[i];
    }
    const int blocks = (u.n + CB - 1) / CB;
    const int windows = u.out ? blocks + (__ballot(shift > blocks * CB - u.n) ? 1 : 0) : 0;  // null: h alone is asked for
    const bool vectors = !__ballot((any & 3) != 0) && u.n % 4 == 0;  // of the result in LDS
    // A lane's W columns of a window. Where a row ends, or begins, inside them it takes the row's last, or first, W
    // instead and writes those it shares with its neighbour again, the same values: both have read their y before either
    // writes, also where out is y, since a window's y is asked for before the window before it is written.
    auto column = [&](int k, int i) { return min(max(k * CB + begin[i], 0), u.n - W); };
    auto inside = [&](int k, int i) { return k * CB + begin[i] > -W && k * CB + begin[i] < u.n; };
    const int vector_windows = u.n >= W ? windows : 0;  // shorter rows are taken an element at a time
    const F* pb = reinterpret_cast<const F*>(u.pb) + group * P::second(u.n) + lane % P::LANES;
    F y[AHEAD][2 * R], bf[AHEAD][KC * NT];
    // Loads come back in the order they were asked for: a window's operands are asked for beside its y, or waiting for
    // them would be waiting for every later y too. The first windows' wait for h: beside A's they would take the registers
    // of a third wavefront (40000 rows 1408 -> 1408 rank 32 fp16: 101 us so, 93 with three, 108 with them held).
    auto ask_operands = [&](int k, F (&b)[KC * NT]) {
        if (!active || k >= blocks) return;
#pragma unroll
        for (int q = 0; q < KC * NT; ++q) b[q] = pb[(int64_t)(k * NT * KC + q) * P::LANES];
    };
    auto ask = [&](int k, F (&f)[2 * R]) {
        if (!u.y) return;
#pragma unroll
        for (int i = 0; i < 2 * R; ++i) {
            if (inside(k, i)) f[i] = fetch<DT>(yrow[i] + column(k, i));
        }
    };
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
#pragma unroll
        for (int i = 0; i < 2 * R; ++i) y[j][i] = F{};
        if (j < vector_windows) ask(j, y[j]);
    }

    constexpr int HF = P::HALF ? 1 : KC * PIECES;
    F hf[R][HF];
    float f[R];
#pragma unroll
    for (int r = 0; r < R; ++r) f[r] = 0.f;
    if (active) {
        // ---- h = s x A^T
        const F* pa = reinterpret_cast<const F*>(u.pa) + group * P::first(u.k) + lane;
        const int batches = P::batches(u.k);
        const bool odd = u.k % W != 0;
        const E* x[2 * R];
#pragma unroll
        for (int i = 0; i < 2 * R; ++i)
            x[i] = reinterpret_cast<const E*>(u.x) + (int64_t)u.order[min(first + 8 * i + r0, end - 1)] * u.xs + lc;
        F xf[AHEAD][2 * R], af[AHEAD][2 * RT];
        auto askx = [&](int i, F (&f)[2 * R], F (&a)[2 * RT]) {
#pragma unroll
            for (int q = 0; q < 2 * RT; ++q) a[q] = pa[(int64_t)(i * 2 * RT + q) * 64];
#pragma unroll
            for (int q = 0; q < 2 * R; ++q) {
                f[q] = F{};
                if (i * KB + lc + W <= u.k) f[q] = fetch<DT>(x[q] + i * KB);
            }
        };
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
            if (j < batches) askx(j, xf[j], af[j]);
        f32x4 acc[R][RT];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int t = 0; t < RT; ++t) acc[r][t] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int i0 = 0; i0 < batches; i0 += AHEAD) {
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                const int i = i0 + j;
                if (i >= batches) break;
                E(&xs)[16 * R][XROW] = lds.stage[wave].x[j & 1];
#pragma unroll
                for (int q = 0; q < 2 * R; ++q) *reinterpret_cast<F*>(&xs[8 * q + r0][lc]) = xf[j][q];
                if (odd && i == batches - 1) {  // the elements behind the last whole vector
                    const int c = (u.k / W * W + g) % KB, k = u.k / W * W + g;
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const E* from = reinterpret_cast<const E*>(u.x) + (int64_t)u.order[min(first + 16 * r + m, end - 1)] * u.xs;
                        if (k < u.k) xs[16 * r + m][c] = from[k];
                        if (k + 4 < u.k) xs[16 * r + m][c + 4] = from[k + 4];
                    }
                }
                wave_sync();
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const F v = *reinterpret_cast<const F*>(&xs[16 * r + m][q * 4 * W + W * g]);
#pragma unroll
                        for (int t = 0; t < RT; ++t) acc[r][t] = M::mul(af[j][q * RT + t], v, acc[r][t]);
                    }
                if (i + AHEAD < batches) askx(i + AHEAD, xf[j], af[j]);
                wave_sync();
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int p = first + 16 * r + m;
            float* keep = u.h && p < end ? u.h + (int64_t)u.order[min(p, end - 1)] * u.rank : nullptr;
            put_h<DT, RT, 16 * R, PITCH, PIECES>(acc[r], u.scales ? u.scales[id] : 1.0f, u.rank, keep, g, 16 * r + m,
                                                 lds.hs[wave], lds.factor[wave]);
        }
        wave_sync();
#pragma unroll
        for (int r = 0; r < R; ++r) {
            f[r] = lds.factor[wave][16 * r + m];
#pragma unroll
            for (int q = 0; q < HF; ++q)
                hf[r][q] = *reinterpret_cast<const F*>(&lds.hs[wave][P::HALF ? g >> 1 : q % PIECES][16 * r + m][P::rank_of(q / PIECES, g)]);
        }
    }

    // ---- out = y + h B^T
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
        if (j < vector_windows) ask_operands(j, bf[j]);
    float(&os)[16 * R][OUT] = lds.stage[wave].out;
    // block k of the result, into its half of the ring
    auto product = [&](int k, const F (&b)[KC * NT]) {
        const int half = k % 2 * CB;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            f32x4 acc[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < KC; ++c)
#pragma unroll
                for (int q = 0; q < (P::HALF ? 1 : PIECES); ++q)
#pragma unroll
                    for (int t = 0; t < NT; ++t) acc[t] = M::mul(b[t * KC + c], hf[r][P::HALF ? 0 : c * PIECES + q], acc[t]);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const int c = 16 * PER * (t / PER) + W * g + 4 * (t % PER);
                const f32x4 v = acc[t] * f[r];
                *reinterpret_cast<f32x4*>(&os[16 * r + m][half + c]) = v;
                if (t < PER && g == 0 && half == 0) *reinterpret_cast<f32x4*>(&os[16 * r + m][RING + c]) = v;
            }
        }
    };
    for (int k0 = 0; k0 < vector_windows; k0 += AHEAD) {
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            const int k = k0 + j;
            if (k >= vector_windows) break;
            if (active && k < blocks) product(k, bf[j]);
            wave_sync();
            F o[2 * R];
#pragma unroll
            for (int i = 0; i < 2 * R; ++i) o[i] = y[j][i];  // rows without an adapter keep y's bits
            if (k + AHEAD < vector_windows) {
                ask_operands(k + AHEAD, bf[j]);
                ask(k + AHEAD, y[j]);
            }
#pragma unroll
            for (int i = 0; i < 2 * R; ++i) {
                const int c = column(k, i);
                if (active) {
                    const float* from = &os[8 * i + r0][c & (RING - 1)];
                    float d[W];
                    if (vectors) {
#pragma unroll
                        for (int e = 0; e < W; e += 4)
                            *reinterpret_cast<f32x4*>(&d[e]) = *reinterpret_cast<const f32x4*>(from + e);
                    } else {
#pragma unroll
                        for (int e = 0; e < W; ++e) d[e] = from[e];
                    }
#pragma unroll
                    for (int e = 0; e < W; ++e) o[i][e] = narrow<DT>(widen<DT>(o[i][e]) + d[e]);
                }
                if (first + 8 * i + r0 < end && inside(k, i)) __builtin_memcpy(orow[i] + c, &o[i], sizeof(F));
            }
            wave_sync();
        }
    }
    if (u.n >= W) return;
    // one block of fewer than W columns: 4 lanes a row, each every fourth element
    if (windows && active) {
        F b[KC * NT];
#pragma unroll
        for (int q = 0; q < KC * NT; ++q) b[q] = pb[(int64_t)q * P::LANES];
        product(0, b);
    }
    wave_sync();
#pragma unroll 1
    for (int r = 0; r < R; ++r) {
        const int64_t row = u.order[min(first + 16 * r + m, end - 1)];
        const E* from = reinterpret_cast<const E*>(u.y) + row * u.ys;
        E* to = reinterpret_cast<E*>(u.out) + row * u.os;
        for (int c = g; c < u.n; c += 4) {
            if (!windows || first + 16 * r + m >= end) continue;
            E o = u.y ? from[c] : E(0);
            if (active) o = narrow<DT>(widen<DT>(o) + os[16 * r + m][c]);
            to[c] = o;
        }
    }
}

// Few rows, where what counts is how long one tile takes: the wavefronts of a workgroup share a tile of 16 rows, split
// k among them, and take 32 columns each at a time. The factors are read where they lie (u.pa null) or packed.
template <int DT, int RP>
__global__ void __launch_bounds__(kThreads) update_few_kernel(const Update u) {
    using M = Mma<DT>;
    using P = Packed<DT, RP>;
    using E = typename M::elem;
    using F = typename M::frag;
    constexpr int W = M::W, KS = P::KS, RT = P::RT, KC = P::KC, PER = P::PER;
    constexpr int PIECES = P::F32 ? 1 : 2, PITCH = RP + W;
    constexpr int NT = 2, CB = 16 * NT, NV = NT / PER;
    __shared__ __align__(16) E hs[PIECES][16][PITCH];
    __shared__ float factor[16];
    __shared__ f32x4 part[kWaves][RT][64];

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, g = lane >> 4;
    int number;
    const int group = group_of_tile(u.starts, u.groups, 16, blockIdx.x, number);
    const int end = u.starts[group + 1];
    const int64_t first64 = (int64_t)u.starts[group] + (int64_t)number * 16;
    if (first64 >= end) return;
    const int first = (int)first64;
    const int id = u.ids[group];
    const bool active = id >= 0 && id < u.adapters;
    if (!active && u.y == u.out) return;  // the rows stay as they are

    const int stop = u.out ? min(u.n, ((int)blockIdx.y + 1) * u.columns) : 0;  // null: h alone is asked for
    const int64_t row = u.order[min(first + m, end - 1)];
    F y[NV];
    auto ask = [&](int n0) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = n0 + 16 * PER * v + W * g;
            y[v] = F{};
            if (u.y && n0 < stop) y[v] = fetch<DT>(reinterpret_cast<const E*>(u.y) + row * u.ys + c, u.n - c);
        }
    };
    int n0 = blockIdx.y * u.columns + CB * wave;
    ask(n0);

    if (active) {
        // ---- h = s x A^T
        const E* x = reinterpret_cast<const E*>(u.x) + row * u.xs + W * g;
        const E* a = reinterpret_cast<const E*>(u.a) + (int64_t)id * u.rank * u.k + W * g;
        const F* pa = reinterpret_cast<const F*>(u.pa) + group * P::first(u.k) + lane;
        f32x4 acc[RT];
#pragma unroll
        for (int t = 0; t < RT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        constexpr int AHEAD = RT <= 2 ? 4 : RT == 4 ? 2 : 1;  // steps whose loads go together
        auto steps = [&](int s, auto many, auto whole) {
            constexpr int N = decltype(many)::value;
            F xf[N], af[N][RT];
#pragma unroll
            for (int p = 0; p < N; ++p) {
                const int k0 = (s + p * kWaves) * KS;
                const int there = decltype(whole)::value ? W : u.k - k0 - W * g;
                xf[p] = fetch<DT>(x + k0, there);
#pragma unroll
                for (int t = 0; t < RT; ++t)  // ranks past the last are dropped by put_h
                    af[p][t] = u.pa ? pa[(int64_t)((s + p * kWaves) * RT + t) * 64]
                                    : fetch<DT>(a + (int64_t)min(16 * t + m, u.rank - 1) * u.k + k0, there);
            }
#pragma unroll
            for (int p = 0; p < N; ++p)
#pragma unroll
                for (int t = 0; t < RT; ++t) acc[t] = M::mul(af[p][t], xf[p], acc[t]);
        };
        int s = wave;
        for (; (s + (AHEAD - 1) * kWaves + 1) * KS <= u.k; s += AHEAD * kWaves)
            steps(s, std::integral_constant<int, AHEAD>{}, std::true_type{});
        for (; s * KS < u.k; s += kWaves) steps(s, std::integral_constant<int, 1>{}, std::false_type{});
#pragma unroll
        for (int t = 0; t < RT; ++t) part[wave][t][lane] = acc[t];
        __syncthreads();
        if (wave == 0) {
#pragma unroll
            for (int t = 0; t < RT; ++t)
                acc[t] = (part[0][t][lane] + part[1][t][lane]) + (part[2][t][lane] + part[3][t][lane]);
            float* keep = u.h && blockIdx.y == 0 && first + m < end ? u.h + row * u.rank : nullptr;
            put_h<DT, RT, 16, PITCH, PIECES>(acc, u.scales ? u.scales[id] : 1.0f, u.rank, keep, g, m, hs, factor);
        }
        __syncthreads();
    }

    // ---- out = y + h B^T
    const E* b = reinterpret_cast<const E*>(u.b) + (int64_t)(active ? id : 0) * u.n * u.rank;
    const int64_t behind = (int64_t)(u.adapters - (active ? id : 0)) * u.n * u.rank;  // elements from b to the bank's end
    const F* pb = reinterpret_cast<const F*>(u.pb) + group * P::second(u.n) + lane % P::LANES;
    const float f = active ? factor[m] : 0.f;
    for (; n0 < stop; n0 += CB * kWaves) {
        f32x4 acc[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (active) {
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                const int rank0 = P::rank_of(c, g);
                F bf[NT];
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    if (u.pb) {
                        bf[t] = pb[(int64_t)((n0 / 16 + t) * KC + c) * P::LANES];
                        continue;
                    }
                    const int64_t i = (int64_t)min(n0 + P::column(t, m), u.n - 1) * u.rank + rank0;
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
                for (int p = 0; p < (P::HALF ? 1 : PIECES); ++p) {
                    const F hf = *reinterpret_cast<const F*>(&hs[P::HALF ? g >> 1 : p][m][rank0]);
#pragma unroll
                    for (int t = 0; t < NT; ++t) acc[t] = M::mul(bf[t], hf, acc[t]);
                }
            }
        }
        F o[NV];
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            o[v] = y[v];  // rows without an adapter keep y's bits
            if (active) {
#pragma unroll
                for (int e = 0; e < W; ++e) o[v][e] = narrow<DT>(widen<DT>(o[v][e]) + f * acc[v * PER + e / 4][e % 4]);
            }
        }
        ask(n0 + CB * kWaves);
        if (first + m >= end) continue;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = n0 + 16 * PER * v + W * g;
            E* to = reinterpret_cast<E*>(u.out) + row * u.os + c;
            if (c + W <= u.n) {
                __builtin_memcpy(to, &o[v], sizeof(F));
            } else {
#pragma unroll
                for (int e = 0; e < W; ++e)
                    if (c + e < u.n) to[e] = o[v][e];
            }
        }
    }
}

// Tiles of 16 ranks a workgroup of the gradients' kernel sums, and workgroups of it that a compute unit holds.
constexpr int grad_tiles(int rank) { return rank <= 16 ? 1 : rank <= 32 ? 2 : 4; }
constexpr int grad_held(int tiles) { return tiles == 1 ? 3 : tiles == 2 ? 2 : 1; }

// One of the two sums t^T h over each group's rows.
struct Task {
    const void* t;   // [rows][cols]
    const float* h;  // [rows][rank]
    void* ops;       // h as operands (pack_rows_kernel)
    int* exps;       // and the power of two of each step of them
    int64_t ts;
    int cols;
    int chunks;  // of its columns, a workgroup's each
    void* out;   // [adapters][...]
    int64_t o_col, o_rank;
    float* partial;  // [parts of the groups with more than one][cols][rank]
};

struct Grads {
    Task task[2];
    int rank, adapters;
    const int32_t *order, *starts, *ids;
    int groups;
    int part;  // rows of one; a multiple of 128
    int dt;    // of what is written: the inputs' type or fp32
};

// Where the partial sums of a group with several parts begin: 2 starts / part is enough for the ones before it,
// since a length above `part` has at most twice length / part, less one, rounded up.
__device__ __forceinline__ int64_t partial_of(const Grads& q, int group) { return 2 * (int64_t)q.starts[group] / q.part; }

__device__ __forceinline__ void store_grad(const Task& k, int rank, int dt, int id, int c, int j, float v) {
    const int64_t i = (int64_t)id * k.cols * rank + c * k.o_col + j * k.o_rank;
    if (dt == NORI_F32) reinterpret_cast<float*>(k.out)[i] = v;
    else reinterpret_cast<uint16_t*>(k.out)[i] = dt == NORI_F16 ? f32_to_f16(v) : f32_to_bf16(v);
}

// h in the order that grad_kernel's instructions take it, 32 rows of a group a step: [step][tile of 16 ranks][lane],
// a lane's 8 rows 8 g ... 8 g + 7 of rank 16 tile + m, zeros past the group's end. 16-bit: two pieces of the type, high
// and low, as in the update, fp16's after a power of two that brings the step's largest element to 2^14 (exps[step]; no
// piece then leaves fp16's range, the smallest bit kept is 2^-38 of the largest). fp32: as they are. Every chunk of
// columns reads them, so they are made once (split in the sums themselves: 60 % of a wavefront's instructions).
constexpr int kStep = 32;  // rows

// steps of group g: from starts[g] / 32 + g
__device__ __forceinline__ int64_t step_of(const int32_t* starts, int group, int in_group) {
    return (int64_t)starts[group] / kStep + group + in_group;
}

template <int DT>
__global__ void __launch_bounds__(kThreads) pack_rows_kernel(const Grads q) {
    using E = typename Mma<DT>::elem;
    const Task& k = q.task[blockIdx.y];
    const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    const int slot = blockIdx.x * kWaves + (threadIdx.x >> 6);
    int number;
    const int group = group_of_tile(q.starts, q.groups, kStep, slot, number);
    const int end = q.starts[group + 1], id = q.ids[group];
    const int64_t first = (int64_t)q.starts[group] + (int64_t)number * kStep;
    if (first >= end || id < 0 || id >= q.adapters) return;
    const int tiles = (q.rank + 15) / 16;
    const float* row[8];
    bool in[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int p = (int)first + 8 * g + i;
        in[i] = p < end;
        row[i] = k.h + (int64_t)q.order[min(p, end - 1)] * q.rank;
    }
    auto load = [&](int t, float (&v)[8]) {
        const int j = 16 * t + m;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = row[i][min(j, q.rank - 1)];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = in[i] && j < q.rank ? v[i] : 0.f;
    };
    float down = 1.0f;
    if constexpr (DT == NORI_F16) {
        float largest = 0.f;
        for (int t = 0; t < tiles; ++t) {
            float v[8];
            load(t, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) largest = fabsf(v[i]) < __builtin_inff() ? fmaxf(largest, fabsf(v[i])) : largest;
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) largest = fmaxf(largest, __shfl_xor(largest, off, 64));
        const int e = min(max((int)(__float_as_uint(largest) >> 23) - 127 - 14, -113), 113);
        down = __uint_as_float((uint32_t)(127 - e) << 23);
        if (lane == 0) k.exps[slot] = e;
    }
    for (int t = 0; t < tiles; ++t) {
        float v[8];
        load(t, v);
        const int64_t at = ((int64_t)slot * tiles + t) * 64 + lane;
        if constexpr (DT == NORI_F32) {
            f32x4* to = reinterpret_cast<f32x4*>(k.ops) + 2 * at;
            to[0] = f32x4{v[0], v[1], v[2], v[3]};
            to[1] = f32x4{v[4], v[5], v[6], v[7]};
        } else {
            u16x8 high, low;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                E h, l;
                split<DT>(v[i] * down, h, l);
                high[i] = h;
                low[i] = l;
            }
            u16x8* to = reinterpret_cast<u16x8*>(k.ops) + 2 * at;
            to[0] = high;
            to[1] = low;
        }
    }
}

// t^T h over one part of a group's rows: 128 (fp32: 64) columns by up to 64 ranks a workgroup, whose wavefronts
// take every fourth step of rows and add their sums in LDS, in order. HBM-bound: t is read once for every 64
// ranks, h once a chunk of columns, from the L2; the next step's rows are on their way while one is summed.
// The sum runs over rows, which t has apart. 16-bit: a lane reads 16 bytes of each of 8 rows and turns the 8 x 8
// block in registers, so that it holds 8 rows of one column for each of 8 instructions; column i of a lane's
// block belongs to instruction i. fp32: instruction i takes row 8 g + i of the lane groups g, no turning. fp16's sums
// are kept at the largest power of two of the steps so far: a larger one rescales them, a smaller one its own sums.
// Where a row ends inside a lane's columns, the lane takes the last ones instead and writes them again, the same
// values. SHORT: rows of fewer columns than a lane takes.
template <int DT, int RT, bool SHORT>
__global__ void __launch_bounds__(kThreads, grad_held(RT)) grad_kernel(const Grads q) {
    using M = Mma<DT>;
    using E = typename M::elem;
    using F = typename M::frag;
    constexpr bool F32 = DT == NORI_F32;
    constexpr int W = M::W, CT = W;  // a lane's columns, an instruction each
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, g = lane >> 4;
    int number;
    const int group = group_of_tile(q.starts, q.groups, q.part, blockIdx.x, number);
    const int begin = q.starts[group], last = q.starts[group + 1];
    const int64_t first64 = (int64_t)begin + (int64_t)number * q.part;
    const int id = q.ids[group];
    if (first64 >= last || id < 0 || id >= q.adapters) return;
    const int first = (int)first64, end = min(last, first + q.part);
    const bool second = (int)blockIdx.y >= q.task[0].chunks;
    const Task& k = q.task[second];
    const int chunk = blockIdx.y - (second ? q.task[0].chunks : 0), t0 = blockIdx.z * RT, tiles = (q.rank + 15) / 16;
    auto column = [&](int of) { return SHORT ? 0 : min(chunk * 16 * W + W * of, k.cols - W); };
    const E* t = reinterpret_cast<const E*>(k.t) + column(m);
    const int64_t step0 = step_of(q.starts, group, number * (q.part / kStep));

    int row[8];
    F raw[8];
    F ops[RT][2];
    int exp_asked = 0;
    auto ask_rows = [&](int s) {
        const int p = first + s * kStep + 8 * g;
#pragma unroll
        for (int i = 0; i < 8; ++i) row[i] = q.order[min(p + i, end - 1)];
    };
    auto ask = [&](int s) {
        const int p = first + s * kStep + 8 * g;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            raw[i] = F{};
            if (p + i < end) {
                if constexpr (SHORT) raw[i] = fetch<DT>(t + row[i] * k.ts, k.cols);
                else raw[i] = fetch<DT>(t + row[i] * k.ts);
            }
        }
#pragma unroll
        for (int r = 0; r < RT; ++r) {  // tiles past the last sum what is never written
            const F* from = reinterpret_cast<const F*>(k.ops) + (((step0 + s) * tiles + min(t0 + r, tiles - 1)) * 64 + lane) * 2;
            ops[r][0] = from[0];
            ops[r][1] = from[1];
        }
        if constexpr (DT == NORI_F16) exp_asked = k.exps[step0 + s];
    };

    f32x4 acc[RT][CT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int i = 0; i < CT; ++i) acc[r][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    int scale = -1000;  // the sums' power of two; none yet
    const int steps = (end - first + kStep - 1) / kStep;
    if (wave < steps) {
        ask_rows(wave);
        ask(wave);
        if (wave + kWaves < steps) ask_rows(wave + kWaves);
    }
    for (int s = wave; s < steps; s += kWaves) {
        F now[8], hn[RT][2];
#pragma unroll
        for (int i = 0; i < 8; ++i) now[i] = raw[i];
#pragma unroll
        for (int r = 0; r < RT; ++r) hn[r][0] = ops[r][0], hn[r][1] = ops[r][1];
        const int e = exp_asked;
        if (s + kWaves < steps) ask(s + kWaves);
        if (s + 2 * kWaves < steps) ask_rows(s + 2 * kWaves);
        if constexpr (F32) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int c = 0; c < CT; ++c)
                        acc[r][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(now[i][c], hn[r][i / 4][i % 4], acc[r][c], 0, 0, 0);
        } else {
            float step = 1.0f;  // of this step's sums
            if constexpr (DT == NORI_F16) {
                // (the same in every lane; 2^-126 stands for less, beside a 2^-38 that the pieces leave out)
                if (e > scale) {
                    if (scale > -1000) {
                        const float change = __uint_as_float((uint32_t)max(127 + scale - e, 1) << 23);
#pragma unroll
                        for (int r = 0; r < RT; ++r)
#pragma unroll
                            for (int c = 0; c < CT; ++c) acc[r][c] = acc[r][c] * change;
                    }
                    scale = e;
                }
                step = __uint_as_float((uint32_t)max(127 + e - scale, 1) << 23);
            }
            auto sum = [&](auto apart) {
#pragma unroll
                for (int c = 0; c < CT; ++c) {
                    F col;
#pragma unroll
                    for (int i = 0; i < 8; ++i) col[i] = now[i][c];
#pragma unroll
                    for (int r = 0; r < RT; ++r) {
                        if constexpr (decltype(apart)::value) {
                            const f32x4 d = M::mul(col, hn[r][1], M::mul(col, hn[r][0], f32x4{0.f, 0.f, 0.f, 0.f}));
                            acc[r][c] = acc[r][c] + d * step;
                        } else {
                            acc[r][c] = M::mul(col, hn[r][0], acc[r][c]);
                            acc[r][c] = M::mul(col, hn[r][1], acc[r][c]);
                        }
                    }
                }
            };
            if (DT == NORI_F16 && step != 1.0f) sum(std::true_type{});
            else sum(std::false_type{});
        }
    }
    // the wavefronts' sums, a rank tile at a time. acc[r][c][j] of lane (m, g): column c of operand row 4 g + j, rank 16 r + m
    __shared__ f32x4 sums[kWaves][CT][64];
    const float up = DT == NORI_F16 && scale > -1000 ? __uint_as_float((uint32_t)(127 + scale) << 23) : 1.0f;
    const bool whole = last - begin <= q.part;
    float* part = whole ? nullptr : k.partial + (partial_of(q, group) + number) * k.cols * q.rank;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        __syncthreads();
#pragma unroll
        for (int c = 0; c < CT; ++c) sums[wave][c][lane] = acc[r][c] * up;
        __syncthreads();
        for (int i = wave; i < CT; i += kWaves) {
            const f32x4 v = (sums[0][i][lane] + sums[1][i][lane]) + (sums[2][i][lane] + sums[3][i][lane]);
            const int j = 16 * (t0 + r) + m;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int c = column(4 * g + e) + i;
                if (j >= q.rank || (SHORT && (c >= k.cols || 4 * g + e > 0))) continue;
                if (whole) store_grad(k, q.rank, q.dt, id, c, j, v[e]);
                else part[(int64_t)c * q.rank + j] = v[e];
            }
        }
    }
}

// the parts of the groups that have several, in their order; blocks0: workgroups of the first task
__global__ void __launch_bounds__(kThreads) grad_join_kernel(const Grads q, int blocks0) {
    const bool second = (int)blockIdx.x >= blocks0;
    const Task& k = q.task[second];
    const int group = blockIdx.y, id = q.ids[group];
    const int length = q.starts[group + 1] - q.starts[group];
    const int64_t size = (int64_t)k.cols * q.rank;
    const int64_t i = (int64_t)(blockIdx.x - (second ? blocks0 : 0)) * kThreads + threadIdx.x;
    if (length <= q.part || id < 0 || id >= q.adapters || i >= size) return;
    const float* part = k.partial + partial_of(q, group) * size + i;
    const int parts = (length + q.part - 1) / q.part;
    float v = 0.f;
#pragma unroll 8
    for (int p = 0; p < parts; ++p) v += part[p * size];
    store_grad(k, q.rank, q.dt, id, (int)(i / q.rank), (int)(i % q.rank), v);
}

int chunks_of(int cols, int dtype) { return (cols + (dtype == NORI_F32 ? 63 : 127)) / (dtype == NORI_F32 ? 64 : 128); }

// Rows of a part: the longest group is cut into the number of parts that costs a compute unit the fewest rows. A
// workgroup costs its rows, 64 for its start, and for its sums, written and joined, 64 a tile of ranks (128 columns of
// 16 ranks, twice, against 256 bytes a row); where all of a unit's workgroups run at once, their starts and ends fall
// together and cost a quarter more. (65536 rows of 32 adapters, 1680 columns, rank 16 fp16: 70 us in 448 workgroups
// of 2048 rows, 57 in 896 of 1024; 64 adapters, 1408 columns: 54 in 704 of 1024, 44 in 1408 of 512; 65536 rows of one
// adapter, 1408 columns, rank 64, where a unit holds one workgroup: 85 in 253 of 2816, 113 in 473 of 1536.)
int part_of(int64_t rows, int64_t longest, int groups, int chunks, int rank) {
    const int tiles = grad_tiles(rank), held = grad_held(tiles), cus = device_cus();
    const int64_t slices = (int64_t)chunks * ((rank + 16 * tiles - 1) / (16 * tiles)), mean = (rows + groups - 1) / groups;
    int64_t best = 0, least = 0;
    for (int64_t p = 1; p <= 64; ++p) {
        const int64_t part = std::max<int64_t>((longest + p - 1) / p + 127, 256) / 128 * 128;
        const int64_t each = (groups * ((mean + part - 1) / part) * slices + cus - 1) / cus;  // workgroups of a unit
        const int64_t cost = each * (part + 64 * (tiles + 1)) * (held > 1 && each <= held ? 5 : 4);
        if (!best || cost < least) best = part, least = cost;
        if (part == 256) break;
    }
    return (int)best;
}

// h or g as operands, in bytes
int64_t operand_bytes(int64_t rows, int groups, int rank) { return (rows / kStep + groups) * ((rank + 15) / 16) * 64 * 32; }

// partial sums of one task, in bytes
int64_t partial_bytes(int64_t rows, int part, int cols, int rank) { return (2 * rows / part + 1) * cols * rank * 4; }

bool is_float(int dt) { return dt == NORI_F32 || dt == NORI_F16 || dt == NORI_BF16; }

int check(const char* what, int dtype, int64_t rows, int32_t groups, int32_t k, int32_t n, int32_t rank, int32_t adapters) {
    if (!is_float(dtype)) return fail(NORI_ERR_UNSUPPORTED, "%s: unsupported dtype %s", what, dtype_name(dtype));
    if (rows < 0 || groups < 0 || k <= 0 || n <= 0 || adapters <= 0)
        return fail(NORI_ERR_INVALID, "%s: bad shape (%lld rows, %d -> %d, %d adapters)", what, (long long)rows, k, n, adapters);
    if (rank <= 0 || rank > NORI_LOW_RANK_MAX)
        return fail(rank <= 0 ? NORI_ERR_INVALID : NORI_ERR_UNSUPPORTED, "%s: rank %d (1 to %d)", what, rank, NORI_LOW_RANK_MAX);
    if (k > NORI_LOW_RANK_COLUMNS || n > NORI_LOW_RANK_COLUMNS)  // offsets in one adapter's factors, and the grids, stay in range
        return fail(NORI_ERR_UNSUPPORTED, "%s: %d -> %d columns (up to %d)", what, k, n, NORI_LOW_RANK_COLUMNS);
    if (rows > (int64_t)1 << 29) return fail(NORI_ERR_UNSUPPORTED, "%s: too many rows", what);
    if (groups > 65535) return fail(NORI_ERR_UNSUPPORTED, "%s: %d adapters in one call (65535 at most)", what, groups);
    return NORI_OK;
}

}  // namespace

// Whether there are few tiles of 16 rows a compute unit, or tiles of 64 are mostly empty. Packing the factors costs a launch, and
// 64 rows an adapter read lower ranks' as fast where they lie (512 tables x 64 rows 256 -> 384 rank 16: 34 us packed, 25
// not; 65536 rows of 32 adapters 560 -> 1680: 119 and 160). The time of a tile is the latency of its passes over k and n,
// which few rows' kernel shares among its wavefronts; the more ranks, the sooner reading the factors costs it more. Out,
// then dx, in us, packed against not: 1408 -> 1408 rank 32 fp16 17000 rows 41 + 37 and 45 + 33, 24000 42 + 39 and
// 62 + 40; rank 64 bf16 8000 44 + 42 and 41 + 32, 14000 44 + 42 and 58 + 38; 560 -> 1680 rank 128 fp16 4000 54 + 43
// and 40 + 32, 11000 54 + 44 and 111 + 55.
static bool few_rows(int64_t rows, int32_t groups, int32_t rank) {
    const int held = rank <= 32 ? 5 : rank <= 64 ? 3 : 2;
    return rows / 16 + groups < held * device_cus() || rows <= (rank <= 32 ? 64 : 16) * (int64_t)groups;
}

// Whether tiles of 128 rows, of which a compute unit holds one, leave too many units idle: while tiles of 64 rows fit the
// units, two each to rank 64 and one above, and, to rank 64, where the last of few rounds is less than half full.
// Out, then dx, in us, tiles of 64 rows against 128: 1408 -> 1408 rank 64, 20000 rows 53 + 50 and 59 + 56, 40000 133 + 83
// and 133 + 103, but 64000 159 + 133 and 144 + 126; 560 -> 1680 rank 128, 14000 54 + 45 and 75 + 58, but 20000
// 92 + 74 and 75 + 58.
static bool short_round(int64_t rows, int ranks) {
    const int cus = device_cus();
    if (ranks > 64) return rows / 64 <= cus;
    return rows / 64 <= 2 * cus || (rows / 128 < 3 * cus && (rows / 128 + cus - 1) % cus < cus / 2);
}

// LDS that a workgroup of update_kernel asks for beside its own, so that a compute unit takes `c` of them at a time and not
// all `held`: the c whose rounds, c as long each, end first. In us, out with h, then dx with g: 16-bit types hold 3; 40000
// rows 1408 -> 1408 rank 32 fp16, one round or two: 88 + 76 with 3 and 98 + 81 with 2; 65536, two rounds each: 144 + 112 and
// 125 + 108. Where rounds tie (`more`): 75000 rows 352 -> 999 rank 16 fp16: 82 + 69 with 3, 89 + 71 with 2; 560 -> 1680 rank
// 32 fp32, which holds 4: 65536 rows 253 + 191 with 4, 277 + 182 with 2, and 98304 rows 354 + 264 with 3, 385 + 261
// with 2; but rank 32 bf16, 89324 rows of 48 tables 1408 -> 999, a sixth of them not adapted: 150 + 134 and 147 + 133.
static unsigned unused_lds(int64_t tiles, int held, bool more, int own) {
    const int64_t cus = device_cus();
    int64_t least = 0;
    int take = 0;
    for (int c = 2; c <= held; ++c) {
        const int64_t rounds = (tiles + c * cus - 1) / (c * cus);
        if (!take || rounds * c < least + more) least = rounds * c, take = c;
        if (rounds == 1) break;  // no unit then takes more than its share (8 x 4096 352 -> 1408 rank 32: 47 us with 3, 42 with 2)
    }
    const int whole = take == held ? 0 : take == 2 ? 60 * 1024 : 52 * 1024;  // of 160 KB
    return (unsigned)std::max(0, whole - own);
}

template <class Go>
static int by_rank(int32_t rank, Go go) {
    if (rank <= 16) return go(std::integral_constant<int, 16>{});
    if (rank <= 32) return go(std::integral_constant<int, 32>{});
    if (rank <= 64) return go(std::integral_constant<int, 64>{});
    return go(std::integral_constant<int, 128>{});
}

// of the packed factors; 0 where they are read as they lie
static int64_t packed_bytes(int dtype, int64_t rows, int32_t k, int32_t n, int32_t rank, int32_t groups, bool transposed) {
    if (!transposed && few_rows(rows, groups, rank)) return 0;
    int64_t bytes = 0;
    NORI_DISPATCH_FLOAT(dtype, DT, {
        by_rank(rank, [&](auto RP_) {
            using P = Packed<DT, decltype(RP_)::value>;
            bytes = groups * (P::first(k) + P::second(n)) * 16;
            return 0;
        });
    });
    return bytes;
}

// h and, where u.out is not null, out; the packed factors in `packed`, 16-byte aligned, or null
static void launch_update(Update u, int dtype, int64_t rows, bool transposed, void* packed, hipStream_t stream) {
    const int cus = device_cus(), groups = u.groups;
    const bool few = few_rows(rows, groups, u.rank);
    NORI_DISPATCH_FLOAT(dtype, DT, {
        by_rank(u.rank, [&](auto RP_) {
            constexpr int RP = decltype(RP_)::value;
            using P = Packed<DT, RP>;
            if (packed) {
                u.pa = packed;
                u.pb = reinterpret_cast<char*>(packed) + groups * P::first(u.k) * 16;
                const int64_t each = P::first(u.k) + P::second(u.n);
                hipLaunchKernelGGL((pack_kernel<DT, RP>), dim3((unsigned)((each + kThreads - 1) / kThreads), groups), dim3(kThreads),
                                   0, stream, u, transposed ? 1 : 0);
            }
            if (!few) {
                const auto launch = [&](auto R_) {
                    constexpr int R = decltype(R_)::value;
                    using L = UpdateLds<DT, RP, R>;
                    const int64_t tiles = rows / (64 * R) + groups;
                    hipLaunchKernelGGL((update_kernel<DT, RP, R>), dim3((unsigned)tiles), dim3(kThreads),
                                       unused_lds(rows / (64 * R), L::HELD, L::MORE, sizeof(L)), stream, u);
                };
                if constexpr (RP <= 32) {
                    launch(std::integral_constant<int, 1>{});
                } else if (short_round(rows, RP)) {
                    launch(std::integral_constant<int, 1>{});
                } else {
                    launch(std::integral_constant<int, 2>{});
                }
                return 0;
            }
            // out's columns are shared among as many workgroups, each with an h of its own, as take the least time: about
            // 1 us of latency for every 512 of k and every round of columns, and the cycles of a compute unit's address
            // units, twice the elements that its workgroups read (64 tables x 16 rows 1408 -> 999: 14 us at 4, 18 at
            // 8; 32 x 128 560 -> 1680: 22 us at 1, 15 at 3)
            const int64_t tiles = rows / 16 + groups;
            const int wide = 32 * kWaves, most = u.out ? (u.n + wide - 1) / wide : 1;
            int steps = most;
            for (int64_t split = 1, least = 0; split <= most; ++split) {
                const int64_t round = (most + split - 1) / split, each = (tiles * split + cus - 1) / cus;
                const int64_t cost = 2400 * (u.k / 512 + round) + each * 2 * (u.k * (P::RT + 1) + round * wide * (P::RT + 2));
                if (!least || cost < least) least = cost, steps = (int)round;
            }
            u.columns = steps * wide;
            // tiles in multiples of 8: a tile's workgroups stay on one XCD, whose L2 holds its x
            const dim3 grid((unsigned)((tiles + 7) / 8 * 8), (unsigned)((most + steps - 1) / steps));
            hipLaunchKernelGGL((update_few_kernel<DT, RP>), grid, dim3(kThreads), 0, stream, u);
            return 0;
        });
    });
}

extern "C" int64_t nori_low_rank_workspace_bytes(int dtype, int64_t rows, int32_t k, int32_t n, int32_t rank, int32_t groups) {
    if (!is_float(dtype) || rows <= 0 || k <= 0 || n <= 0 || rank <= 0 || groups <= 0) return 0;
    return packed_bytes(dtype, rows, k, n, rank, groups, false);
}

extern "C" int nori_low_rank_update(const void* x, int dtype, int64_t rows, int32_t k, int64_t x_row_stride, const void* y,
                                    int64_t y_row_stride, const void* a, const void* b, const float* scales, int32_t adapters,
                                    int32_t rank, int32_t n, const int32_t* order, const int32_t* starts, const int32_t* ids,
                                    int32_t groups, void* out, int64_t out_row_stride, float* h, void* workspace,
                                    int64_t workspace_bytes, void* stream_v) {
    clear_error();
    if (int rc = check("low_rank_update", dtype, rows, groups, k, n, rank, adapters)) return rc;
    if (rows == 0) return NORI_OK;
    if (!x || !a || !b || !order || !starts || !ids || !out || groups <= 0)
        return fail(NORI_ERR_INVALID, "low_rank_update: null pointer");
    if (out_row_stride < n && rows > 1) return fail(NORI_ERR_INVALID, "low_rank_update: rows of out overlap");
    if (out == y && out_row_stride != y_row_stride && rows > 1)
        return fail(NORI_ERR_INVALID, "low_rank_update: out is y, at another row stride");
    const int64_t need = nori_low_rank_workspace_bytes(dtype, rows, k, n, rank, groups);
    if (need && (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < need))
        return fail(NORI_ERR_INVALID, "low_rank_update: workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
                    (long long)need);
    const Update u{x,  y, a,   b,      x_row_stride, y_row_stride, out_row_stride, k, n, rank, adapters, scales, order, starts, ids,
                   groups, 0, out, h, nullptr, nullptr};
    launch_update(u, dtype, rows, false, need ? workspace : nullptr, (hipStream_t)stream_v);
    return launch_status("low_rank_update");
}

namespace {
// the backward pass's workspace: g [rows][rank], the packed factors, g and h as operands and their steps' powers of
// two, the partial sums of da and of db
struct Layout {
    int64_t packed, ops_a, ops_b, da, db, end;
    int part;
};

Layout layout_of(int dtype, int64_t rows, int32_t k, int32_t n, int32_t rank, int32_t groups, int64_t longest, bool need_x,
                 bool need_a, bool need_b) {
    auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
    Layout l;
    l.part = part_of(rows, longest, groups, (need_a ? chunks_of(k, dtype) : 0) + (need_b ? chunks_of(n, dtype) : 0), rank);
    const bool parts = longest > l.part;
    l.packed = up(need_a ? rows * rank * 4 : 0);
    l.ops_a = l.packed + up(need_x || need_a ? packed_bytes(dtype, rows, n, k, rank, groups, true) : 0);
    const int64_t ops = up(operand_bytes(rows, groups, rank)) + up((rows / kStep + groups) * 4);
    l.ops_b = l.ops_a + (need_a ? ops : 0);
    l.da = l.ops_b + (need_b ? ops : 0);
    l.db = l.da + up(need_a && parts ? partial_bytes(rows, l.part, k, rank) : 0);
    l.end = l.db + up(need_b && parts ? partial_bytes(rows, l.part, n, rank) : 0);
    return l;
}
}  // namespace

extern "C" int64_t nori_low_rank_backward_workspace_bytes(int dtype, int64_t rows, int32_t k, int32_t n, int32_t rank,
                                                          int32_t groups, int64_t longest, int32_t need_x, int32_t need_a,
                                                          int32_t need_b) {
    if (!is_float(dtype) || rows <= 0 || k <= 0 || n <= 0 || rank <= 0 || groups <= 0) return 0;
    return layout_of(dtype, rows, k, n, rank, groups, longest, need_x, need_a, need_b).end;
}

// grad_dtype: of da and db
static int backward(const void* x, int dtype, int64_t rows, int32_t k, int64_t x_row_stride, const void* dy, int32_t n,
                    int64_t dy_row_stride, const void* base, int64_t base_row_stride, const void* a, const void* b,
                    const float* scales, int32_t adapters, int32_t rank, const int32_t* order, const int32_t* starts,
                    const int32_t* ids, int32_t groups, int64_t longest, const float* h, void* dx, int64_t dx_row_stride, void* da,
                    void* db, int grad_dtype, void* workspace, int64_t workspace_bytes, void* stream_v) {
    clear_error();
    if (int rc = check("low_rank_backward", dtype, rows, groups, k, n, rank, adapters)) return rc;
    if (rows == 0 || (!dx && !da && !db)) return NORI_OK;
    if (!x || !dy || !a || !b || !order || !starts || !ids || (db && !h) || groups <= 0)
        return fail(NORI_ERR_INVALID, "low_rank_backward: null pointer");
    if (dx && dx_row_stride < k && rows > 1) return fail(NORI_ERR_INVALID, "low_rank_backward: rows of dx overlap");
    if (dx && dx == base && dx_row_stride != base_row_stride && rows > 1)
        return fail(NORI_ERR_INVALID, "low_rank_backward: dx is its base, at another row stride");
    if (longest < 0 || longest > rows)
        return fail(NORI_ERR_INVALID, "low_rank_backward: a longest group of %lld rows of %lld", (long long)longest, (long long)rows);
    const Layout l = layout_of(dtype, rows, k, n, rank, groups, longest, dx, da, db);
    if (l.end && (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < l.end))
        return fail(NORI_ERR_INVALID, "low_rank_backward: workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
                    (long long)l.end);
    char* at = reinterpret_cast<char*>(workspace);
    float* kept = reinterpret_cast<float*>(at);
    hipStream_t stream = (hipStream_t)stream_v;
    if (dx || da) {
        // dx = base + (s dy B) A: the update with the factors' roles swapped, g kept for da
        const Update u{dy, dx ? base : nullptr, b, a, dy_row_stride, base_row_stride, dx_row_stride, n, k, rank, adapters, scales, order,
                       starts, ids, groups, 0, dx, da ? kept : nullptr, nullptr, nullptr};
        launch_update(u, dtype, rows, true, at + l.packed, stream);
    }
    if (!da && !db) return launch_status("low_rank_backward");
    Grads q{};
    q.rank = rank;
    q.adapters = adapters;
    q.order = order;
    q.starts = starts;
    q.ids = ids;
    q.groups = groups;
    q.part = l.part;
    q.dt = grad_dtype;
    int tasks = 0;
    const int64_t exps = (operand_bytes(rows, groups, rank) + 255) / 256 * 256;
    auto task = [&](const void* t, const float* h, int64_t ops, int64_t ts, int cols, void* out, int64_t o_col, int64_t o_rank,
                    int64_t partial) {
        q.task[tasks++] = Task{t, h, at + ops, reinterpret_cast<int*>(at + ops + exps), ts, cols, chunks_of(cols, dtype), out, o_col,
                               o_rank, reinterpret_cast<float*>(at + partial)};
    };
    if (da) task(x, kept, l.ops_a, x_row_stride, k, da, 1, k, l.da);          // [adapters][rank][k]
    if (db) task(dy, h, l.ops_b, dy_row_stride, n, db, rank, 1, l.db);        // [adapters][n][rank]
    const unsigned slots = (unsigned)((rows / kStep + groups + kWaves - 1) / kWaves);
    NORI_DISPATCH_FLOAT(dtype, DT, {
        hipLaunchKernelGGL((pack_rows_kernel<DT>), dim3(slots, (unsigned)tasks), dim3(kThreads), 0, stream, q);
    });
    const int64_t parts = rows / q.part + groups;
    // the tasks whose rows are whole vectors together, the others by themselves
    auto go = [&](const Grads& some, bool narrow_rows) {
        const unsigned chunks = (unsigned)(some.task[0].chunks + some.task[1].chunks);
        NORI_DISPATCH_FLOAT(dtype, DT, {
            auto launch = [&](auto RT_, auto SHORT_) {
                constexpr int RT = decltype(RT_)::value;
                hipLaunchKernelGGL((grad_kernel<DT, RT, decltype(SHORT_)::value>),
                                   dim3((unsigned)parts, chunks, (unsigned)((rank + 16 * RT - 1) / (16 * RT))), dim3(kThreads), 0,
                                   stream, some);
            };
            if (narrow_rows) launch(std::integral_constant<int, 1>{}, std::true_type{});
            else if (grad_tiles(rank) == 1) launch(std::integral_constant<int, 1>{}, std::false_type{});
            else if (grad_tiles(rank) == 2) launch(std::integral_constant<int, 2>{}, std::false_type{});
            else launch(std::integral_constant<int, 4>{}, std::false_type{});
        });
    };
    const int vector = dtype == NORI_F32 ? 4 : 8;
    Grads many = q, single = q;
    many.task[0] = many.task[1] = Task{};
    int taken = 0;
    for (int i = 0; i < tasks; ++i) {
        if (q.task[i].cols >= vector) {
            many.task[taken++] = q.task[i];
        } else {
            single.task[0] = q.task[i];
            single.task[1] = Task{};
            go(single, true);
        }
    }
    if (taken) go(many, false);
    if (longest > q.part) {
        const int blocks0 = (int)(((int64_t)q.task[0].cols * rank + kThreads - 1) / kThreads);
        const int blocks1 = (int)(((int64_t)q.task[1].cols * rank + kThreads - 1) / kThreads);
        hipLaunchKernelGGL(grad_join_kernel, dim3((unsigned)(blocks0 + blocks1), groups), dim3(kThreads), 0, stream, q, blocks0);
    }
    return launch_status("low_rank_backward");
}

extern "C" int nori_low_rank_backward(const void* x, int dtype, int64_t rows, int32_t k, int64_t x_row_stride, const void* dy,
                                      int32_t n, int64_t dy_row_stride, const void* base, int64_t base_row_stride, const void* a,
                                      const void* b, const float* scales, int32_t adapters, int32_t rank, const int32_t* order,
                                      const int32_t* starts, const int32_t* ids, int32_t groups, int64_t longest, const float* h,
                                      void* dx, int64_t dx_row_stride, void* da, void* db, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
    return backward(x, dtype, rows, k, x_row_stride, dy, n, dy_row_stride, base, base_row_stride, a, b, scales, adapters, rank, order,
                    starts, ids, groups, longest, h, dx, dx_row_stride, da, db, dtype, workspace, workspace_bytes, stream);
}

extern "C" int nori_low_rank_backward_f32(const void* x, int dtype, int64_t rows, int32_t k, int64_t x_row_stride, const void* dy,
                                          int32_t n, int64_t dy_row_stride, const void* base, int64_t base_row_stride,
                                          const void* a, const void* b, const float* scales, int32_t adapters, int32_t rank,
                                          const int32_t* order, const int32_t* starts, const int32_t* ids, int32_t groups,
                                          int64_t longest, const float* h, void* dx, int64_t dx_row_stride, void* da, void* db,
                                          void* workspace, int64_t workspace_bytes, void* stream) {
    return backward(x, dtype, rows, k, x_row_stride, dy, n, dy_row_stride, base, base_row_stride, a, b, scales, adapters, rank, order,
                    starts, ids, groups, longest, h, dx, dx_row_stride, da, db, NORI_F32, workspace, workspace_bytes, stream);
}
