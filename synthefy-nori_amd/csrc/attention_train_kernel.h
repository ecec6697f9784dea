// The kernels of attention with gradients, instantiated by attention_train_<type>.hip (attention_train.h has the
// mathematics and the layout).
#pragma once

#include "attention_train.h"
#include "train_matrix.h"

namespace nori {
namespace attn_train {

using namespace train;

// Geometry of a head width padded to DK (a multiple of 16): DP is DK in whole products of 32 columns.
template <int DT, int DK> struct Geo {
    using E = El<DT>;
    using T = typename E::T;
    static constexpr int DP = (DK + 31) / 32 * 32;
    static constexpr int LS = DP + E::kPad;      // elements from one row of a tile to the next
    static constexpr int KS = DK / 16, MS = DP / 32, NS = E::kRows / 32;
};

// Left operand: row `row` (lane % 32 of a step's 32) of a tile, its columns 16 k + 8 h .. + 7.
template <int DT, int DK>
__device__ __forceinline__ typename El<DT>::Frag direct(const typename El<DT>::T* tile, int row, int k, int half) {
    const auto* p = tile + row * Geo<DT, DK>::LS + 16 * k + 8 * half;
    return *reinterpret_cast<const typename El<DT>::Frag*>(p);
}

// The operands that stay: columns 16 k + 8 h .. + 7 of the row at p, zeros past d or where the row is not there.
template <int DT, int DK, int W>
__device__ __forceinline__ void load_own(typename El<DT>::Frag (&f)[DK / 16], const typename El<DT>::T* p, bool there, int d, int half) {
    using E = El<DT>;
    typedef uint32_t Chunk __attribute__((ext_vector_type(W * sizeof(typename E::T) / 4)));
#pragma unroll
    for (int k = 0; k < DK / 16; ++k) {
        Chunk c[8 / W] = {};
#pragma unroll
        for (int j = 0; j < 8 / W; ++j) {
            const int at = 16 * k + 8 * half + W * j;
            if (there && at < d) c[j] = *reinterpret_cast<const Chunk*>(p + at);
        }
        f[k] = __builtin_bit_cast(typename E::Frag, c);
    }
}

// Writes 4 results, columns at .. at + 3 of a row.
template <int DT>
__device__ __forceinline__ void store4(typename El<DT>::T* p, const float (&x)[4]) {
    if constexpr (DT == NORI_F32) {
        *reinterpret_cast<f32x4*>(p) = f32x4{x[0], x[1], x[2], x[3]};
    } else {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = DT == NORI_F16 ? f32_to_f16(x[j]) : f32_to_bf16(x[j]);
        *reinterpret_cast<u32x2*>(p) = u32x2{w[0] | (w[1] << 16), w[2] | (w[3] << 16)};
    }
}

// Query row r of a unit: head and query.
struct Row { int64_t head, query; };
__device__ __forceinline__ Row row_of(const Args& p, int64_t unit_head, int r) {
    if (p.group == 1) return {unit_head, r};
    const int h = r / (int)p.a.nq;
    return {unit_head * p.group + h, r - h * (int)p.a.nq};
}

struct Block { int64_t tile, split, unit, b, hk; };
__device__ __forceinline__ Block block_of(const Args& p) {
    int64_t i = work_index(blockIdx.x, gridDim.x);
    Block w;
    w.tile = i % p.tiles;
    i /= p.tiles;
    w.split = i % p.splits;
    w.unit = i / p.splits;
    w.b = w.unit / p.a.kv_heads;
    w.hk = w.unit % p.a.kv_heads;
    return w;
}

// A tile of two tensors on its way to LDS: chunks of W elements in registers, asked for while the tile before is worked on.
// A thread's chunks are at the same places of every tile: 32-bit byte offsets from the tile's first row, which moves on
// uniformly (the host keeps strides to what that takes).
template <int DT, int DK, int W> struct Stage {
    using G = Geo<DT, DK>;
    using E = El<DT>;
    using T = typename E::T;
    typedef uint32_t Chunk __attribute__((ext_vector_type(W * sizeof(T) / 4)));
    static constexpr int CH = DK / W;                                       // chunks a row
    static constexpr int N = (E::kRows * CH + kThreads - 1) / kThreads;     // chunks a thread, a tile
    Chunk x[N], y[N];
    uint32_t ox[N], oy[N];
    int row[N];  // past every tile for chunks that no row has: they stay zero

    __device__ __forceinline__ void place(int d, int64_t x_stride, int64_t y_stride) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int idx = threadIdx.x + i * kThreads, r = idx / CH, col = W * (idx % CH);
            row[i] = r < E::kRows && col < d ? r : 1 << 30;
            ox[i] = (uint32_t)(r * (uint32_t)x_stride + col) * sizeof(T);
            oy[i] = (uint32_t)(r * (uint32_t)y_stride + col) * sizeof(T);
        }
    }
    // `left` rows from px and py on
    __device__ __forceinline__ void load(const T* px, const T* py, int left) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            x[i] = Chunk{};
            y[i] = Chunk{};
            if (row[i] < left) {
                x[i] = *reinterpret_cast<const Chunk*>(reinterpret_cast<const char*>(px) + ox[i]);
                y[i] = *reinterpret_cast<const Chunk*>(reinterpret_cast<const char*>(py) + oy[i]);
            }
        }
    }
    // the same where rows from `over` on lie wx and wy bytes further (the next head's)
    __device__ __forceinline__ void load_over(const T* px, const T* py, int left, int over, int64_t wx, int64_t wy) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            x[i] = Chunk{};
            y[i] = Chunk{};
            if (row[i] < left) {
                const bool next = row[i] >= over;
                x[i] = *reinterpret_cast<const Chunk*>(reinterpret_cast<const char*>(px) + ox[i] + (next ? wx : 0));
                y[i] = *reinterpret_cast<const Chunk*>(reinterpret_cast<const char*>(py) + oy[i] + (next ? wy : 0));
            }
        }
    }
    // rows anywhere
    template <class At>
    __device__ __forceinline__ void load_each(int left, At at) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            x[i] = Chunk{};
            y[i] = Chunk{};
            if (row[i] < left) {
                const T *px, *py;
                at(row[i], px, py);
                const int col = W * ((threadIdx.x + i * kThreads) % CH);
                x[i] = *reinterpret_cast<const Chunk*>(px + col);
                y[i] = *reinterpret_cast<const Chunk*>(py + col);
            }
        }
    }
    __device__ __forceinline__ void store(T* tx, T* ty) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int idx = threadIdx.x + i * kThreads, to = idx / CH * G::LS + W * (idx % CH);
            if (E::kRows * CH % kThreads == 0 || idx < E::kRows * CH) {
                *reinterpret_cast<Chunk*>(tx + to) = x[i];
                *reinterpret_cast<Chunk*>(ty + to) = y[i];
            }
        }
    }
};

// ---------------------------------------------------------------- forward
template <int DT, int DK, int W>
__global__ __launch_bounds__(kThreads, DK <= 64 ? 3 : 2) void forward_kernel(const Args p) {
    using E = El<DT>;
    using G = Geo<DT, DK>;
    using T = typename E::T;
    __shared__ __attribute__((aligned(16))) T ks[E::kRows * G::LS];
    __shared__ __attribute__((aligned(16))) T vs[E::kRows * G::LS];
    const auto& a = p.a;
    const Block w = block_of(p);
    const int lane = threadIdx.x & 63, half = lane >> 5, wave = threadIdx.x >> 6;
    const int64_t r64 = w.tile * kOwn + wave * 32 + (lane & 31);
    const bool there = r64 < p.rows;
    const int r = (int)r64;
    const Row row = there ? row_of(p, w.hk, r) : Row{w.hk * p.group, 0};
    const int length = length_of(a, w.b);
    const int begin = (int)(w.split * p.per_split);
    const int end = (int)min((int64_t)length, w.split * p.per_split + p.per_split);

    typename E::Frag qf[G::KS];
    load_own<DT, DK, W>(qf, reinterpret_cast<const T*>(a.q) + w.b * a.q_bg + row.query * a.q_row + row.head * a.q_head, there, a.d, half);
    const T* kv = reinterpret_cast<const T*>(a.kv) + w.b * a.kv_bg + w.hk * a.kv_head + begin * a.kv_row;
    // the running maximum wants a positive factor: a negative one changes signs first, one of 0 makes the logits 0
    const float c = p.c == 0.f ? 1.f : fabsf(p.c);
    if (p.c <= 0.f) {
        const float sign = p.c < 0.f ? -1.f : 0.f;
#pragma unroll
        for (int k = 0; k < G::KS; ++k)
#pragma unroll
            for (int j = 0; j < 8; ++j) at(qf[k], j) = at(qf[k], j) * sign;
    }

    float m = -INFINITY, l = 0.f;  // of this half-wave's keys
    f32x16 o[G::MS] = {};
    Stage<DT, DK, W> stage;
    stage.place(a.d, a.kv_row, a.kv_row);
    if (begin < end) stage.load(kv, kv + a.kv_half, end - begin);
    for (int first = begin; first < end; first += E::kRows) {
        __syncthreads();
        stage.store(ks, vs);
        __syncthreads();
        kv += E::kRows * a.kv_row;
        if (first + E::kRows < end) stage.load(kv, kv + a.kv_half, end - first - E::kRows);
        f32x16 s[G::NS];
#pragma unroll
        for (int sub = 0; sub < G::NS; ++sub) {
            s[sub] = f32x16{};
#pragma unroll
            for (int k = 0; k < G::KS; ++k) s[sub] = mma(direct<DT, DK>(ks, sub * 32 + (lane & 31), k, half), qf[k], s[sub]);
        }
        if (first + E::kRows > end) {
#pragma unroll
            for (int sub = 0; sub < G::NS; ++sub)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (first + sub * 32 + 8 * (i / 4) + 4 * half + i % 4 >= end) s[sub][i] = -INFINITY;
        }
        float top = s[0][0];
#pragma unroll
        for (int i = 1; i < 16 * G::NS; ++i) top = fmaxf(top, s[i / 16][i % 16]);
        top = fmaxf(top, other_half(top));
        // the maximum that p is taken against moves when one passes it by 2^kSlack: rarely, after the first tiles
        if (__any((top - m) * c > E::kSlack)) {
            const float next = fmaxf(m, top);
            const float shrink = next == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - next) * c);
            m = next;
            l *= shrink;
#pragma unroll
            for (int j = 0; j < G::MS; ++j) o[j] *= shrink;
        }
        const float off = E::kTop - (m == -INFINITY ? 0.f : m * c);  // (all keys so far at -inf: their p is 0)
#pragma unroll
        for (int sub = 0; sub < G::NS; ++sub) {
            float x[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                x[i] = __builtin_amdgcn_exp2f(fmaf(s[sub][i], c, off));
                l += x[i];
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const auto pf = rounded<DT>(x, t);
#pragma unroll
                for (int j = 0; j < G::MS; ++j) o[j] = mma(transposed<DT, G::LS>(vs, sub * 32 + 16 * t, 32 * j, lane), pf, o[j]);
            }
        }
    }
    if (!there) return;
    l += other_half(l);
    const float inv = begin < end ? 1.f / l : 0.f;
    const float lse2 = begin < end ? __builtin_amdgcn_logf(l) - E::kTop + m * c : -INFINITY;
    if (p.splits > 1) {
        const int64_t units = a.bg * a.kv_heads;
        const int64_t to = (w.split * units + w.unit) * p.rows + r;
        if (half == 0) p.part_lse[to] = lse2;
#pragma unroll
        for (int j = 0; j < G::MS; ++j)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int col = 32 * j + 2 * i + 4 * half;
                if (col < a.d) *reinterpret_cast<f32x4*>(p.part + to * a.d + col) = f32x4{o[j][i] * inv, o[j][i + 1] * inv, o[j][i + 2] * inv, o[j][i + 3] * inv};
            }
        return;
    }
    if (half == 0 && a.lse) a.lse[w.unit * p.rows + r] = lse2 * kLn2;
    T* out = reinterpret_cast<T*>(a.out) + ((w.b * a.nq + row.query) * a.heads + row.head) * a.d;
#pragma unroll
    for (int j = 0; j < G::MS; ++j)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int col = 32 * j + 2 * i + 4 * half;
            const float x[4] = {o[j][i] * inv, o[j][i + 1] * inv, o[j][i + 2] * inv, o[j][i + 3] * inv};
            if (col < a.d) store4<DT>(out + col, x);
        }
}

// ds in float16 carries a power of two a column (a query of dq, a key of dk): gradients of a mean over many rows lie below
// float16's range, those under a loss scale above it. The power brings the first values to 2^8 and falls where a later
// one would pass 2^15; what is summed so far is brought along. Exact, so the result does not go by it but for values
// 2^-22 of the column's largest.
struct Scale {
    float f = 0.f;  // 0: nothing but zeros so far

    // the values of this step with the factor on; acc takes a change of it
    template <int NS, int MS>
    __device__ __forceinline__ void apply(float (&x)[NS][16], f32x16 (&acc)[MS]) {
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 16 * NS; ++i) top = fmaxf(top, fabsf(x[i / 16][i % 16]));
        top = fmaxf(top, other_half(top));
        const bool change = f == 0.f ? top > 0.f : top * f > 32768.f;
        if (__any(change)) {
            float next = f;
            if (change) {
                int e = 8 + 127 - (int)(__float_as_uint(top) >> 23);  // top * 2^e in [2^8, 2^9)
                e = e > 120 ? 120 : (e < -100 ? -100 : e);
                next = __uint_as_float((uint32_t)(e + 127) << 23);
            }
            const float by = f == 0.f ? 1.f : next / f;  // (nothing is summed while f is 0)
#pragma unroll
            for (int j = 0; j < MS; ++j) acc[j] *= by;
            f = next;
        }
#pragma unroll
        for (int i = 0; i < 16 * NS; ++i) x[i / 16][i % 16] *= f;
    }
    __device__ __forceinline__ float inverse() const { return f == 0.f ? 1.f : 1.f / f; }
};

// ---------------------------------------------------------------- dq, and delta for dk and dv
template <int DT, int DK, int W>
__global__ __launch_bounds__(kThreads, DT == NORI_F32 && DK > 96 ? 1 : 2) void dq_kernel(const Args p) {
    using E = El<DT>;
    using G = Geo<DT, DK>;
    using T = typename E::T;
    __shared__ __attribute__((aligned(16))) T ks[E::kRows * G::LS];
    __shared__ __attribute__((aligned(16))) T vs[E::kRows * G::LS];
    const auto& a = p.a;
    const Block w = block_of(p);
    const int lane = threadIdx.x & 63, half = lane >> 5, wave = threadIdx.x >> 6;
    const int64_t r64 = w.tile * kOwn + wave * 32 + (lane & 31);
    const bool there = r64 < p.rows;
    const int r = (int)r64;
    const Row row = there ? row_of(p, w.hk, r) : Row{w.hk * p.group, 0};
    const int64_t unit_row = w.unit * p.rows + r;
    const int length = length_of(a, w.b);
    const int begin = (int)(w.split * p.per_split);
    const int end = a.dq ? (int)min((int64_t)length, w.split * p.per_split + p.per_split) : begin;

    typename E::Frag dof[G::KS], qf[G::KS];
    load_own<DT, DK, W>(dof, reinterpret_cast<const T*>(a.dout) + w.b * a.do_bg + row.query * a.do_row + row.head * a.do_head, there, a.d, half);
    load_own<DT, DK, W>(qf, reinterpret_cast<const T*>(a.out) + ((w.b * a.nq + row.query) * a.heads + row.head) * a.d, there, a.d, half);
    float delta = 0.f;
#pragma unroll
    for (int k = 0; k < G::KS; ++k) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if constexpr (DT == NORI_F32) delta = fmaf(dof[k].v[j], qf[k].v[j], delta);
            else delta = fmaf((float)dof[k][j], (float)qf[k][j], delta);
        }
    }
    delta += other_half(delta);
    if (there && half == 0 && w.split == 0) p.delta[unit_row] = delta;
    if (!a.dq) return;
    load_own<DT, DK, W>(qf, reinterpret_cast<const T*>(a.q) + w.b * a.q_bg + row.query * a.q_row + row.head * a.q_head, there, a.d, half);
    const float lse2 = there ? a.lse[unit_row] * kLog2e : 0.f;
    const T* kv = reinterpret_cast<const T*>(a.kv) + w.b * a.kv_bg + w.hk * a.kv_head + begin * a.kv_row;

    f32x16 dq[G::MS] = {};
    Scale scale;
    Stage<DT, DK, W> stage;
    stage.place(a.d, a.kv_row, a.kv_row);
    if (begin < end) stage.load(kv, kv + a.kv_half, end - begin);
    for (int first = begin; first < end; first += E::kRows) {
        __syncthreads();
        stage.store(ks, vs);
        __syncthreads();
        kv += E::kRows * a.kv_row;
        if (first + E::kRows < end) stage.load(kv, kv + a.kv_half, end - first - E::kRows);
        float ds[G::NS][16];
#pragma unroll
        for (int sub = 0; sub < G::NS; ++sub) {
            f32x16 s = {}, dp;
#pragma unroll
            for (int i = 0; i < 16; ++i) dp[i] = -delta;
#pragma unroll
            for (int k = 0; k < G::KS; ++k) {
                s = mma(direct<DT, DK>(ks, sub * 32 + (lane & 31), k, half), qf[k], s);
                dp = mma(direct<DT, DK>(vs, sub * 32 + (lane & 31), k, half), dof[k], dp);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) ds[sub][i] = __builtin_amdgcn_exp2f(fmaf(s[i], p.c, -lse2)) * dp[i];
        }
        if (first + E::kRows > end) {
#pragma unroll
            for (int sub = 0; sub < G::NS; ++sub)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (first + sub * 32 + 8 * (i / 4) + 4 * half + i % 4 >= end) ds[sub][i] = 0.f;
        }
        if constexpr (E::kScaled) scale.apply(ds, dq);
#pragma unroll
        for (int sub = 0; sub < G::NS; ++sub)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const auto f = rounded<DT>(ds[sub], t);
#pragma unroll
                for (int j = 0; j < G::MS; ++j) dq[j] = mma(transposed<DT, G::LS>(ks, sub * 32 + 16 * t, 32 * j, lane), f, dq[j]);
            }
    }
    if (!there) return;
    const float by = a.scale * (E::kScaled ? scale.inverse() : 1.f);
    T* out = reinterpret_cast<T*>(a.dq) + ((w.b * a.nq + row.query) * a.heads + row.head) * a.d;
    float* part = p.part + (w.split * a.bg * a.kv_heads * p.rows + unit_row) * a.d;
#pragma unroll
    for (int j = 0; j < G::MS; ++j)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int col = 32 * j + 2 * i + 4 * half;
            const float x[4] = {dq[j][i] * by, dq[j][i + 1] * by, dq[j][i + 2] * by, dq[j][i + 3] * by};
            if (col >= a.d) continue;
            if (p.splits > 1) *reinterpret_cast<f32x4*>(part + col) = f32x4{x[0], x[1], x[2], x[3]};
            else store4<DT>(out + col, x);
        }
}

// ---------------------------------------------------------------- dk and dv
template <int DT, int DK, int W>
__global__ __launch_bounds__(kThreads, DK <= 64 ? 2 : 1) void dkv_kernel(const Args p) {
    using E = El<DT>;
    using G = Geo<DT, DK>;
    using T = typename E::T;
    __shared__ __attribute__((aligned(16))) T qs[E::kRows * G::LS];
    __shared__ __attribute__((aligned(16))) T dos[E::kRows * G::LS];
    __shared__ __attribute__((aligned(16))) float off[E::kRows];    // kBias - log2 of the row's sum
    __shared__ __attribute__((aligned(16))) float deltas[E::kRows];  // negative: what the products of dout and v start from
    const auto& a = p.a;
    const Block w = block_of(p);
    const int lane = threadIdx.x & 63, half = lane >> 5, wave = threadIdx.x >> 6;
    const int64_t key64 = w.tile * kOwn + wave * 32 + (lane & 31);
    const int length = length_of(a, w.b);
    const bool there = key64 < length;
    const int key = (int)key64;
    const int begin = (int)(w.split * p.per_split);
    // (a tile behind the length has no products, its gradients are zeros)
    const int end = w.tile * kOwn < length ? (int)min(p.rows, w.split * p.per_split + p.per_split) : begin;

    typename E::Frag kf[G::KS], vf[G::KS];
    const T* kv = reinterpret_cast<const T*>(a.kv) + w.b * a.kv_bg + w.hk * a.kv_head + (there ? key * a.kv_row : 0);
    load_own<DT, DK, W>(kf, kv, there, a.d, half);
    load_own<DT, DK, W>(vf, kv + a.kv_half, there, a.d, half);
    const T* q = reinterpret_cast<const T*>(a.q) + w.b * a.q_bg + w.hk * p.group * a.q_head;
    const T* dout = reinterpret_cast<const T*>(a.dout) + w.b * a.do_bg + w.hk * p.group * a.do_head;
    const float* lse = a.lse + w.unit * p.rows;
    const float* delta = p.delta + w.unit * p.rows;
    // where a tile's first row is: head `at_head` of the unit's, query `at_query`
    const int nq = (int)a.nq;
    int at_head = begin < end ? begin / nq : 0, at_query = begin - at_head * nq;

    f32x16 dk[G::MS] = {}, dv[G::MS] = {};
    Scale scale;
    Stage<DT, DK, W> stage;
    stage.place(a.d, a.q_row, a.do_row);
    float next_off = 0.f, next_delta = 0.f;
    const auto load = [&](int first) {
        const int left = end - first;
        const T* px = q + at_head * a.q_head + at_query * a.q_row;
        const T* py = dout + at_head * a.do_head + at_query * a.do_row;
        if (at_query + E::kRows <= nq || p.group == 1) {
            stage.load(px, py, left);
        } else if (nq >= E::kRows) {
            stage.load_over(px, py, left, nq - at_query, (a.q_head - nq * a.q_row) * (int64_t)sizeof(T),
                            (a.do_head - nq * a.do_row) * (int64_t)sizeof(T));
        } else {
            stage.load_each(left, [&](int row, const T*& x, const T*& y) {
                const int h = (first + row) / nq, i = first + row - h * nq;
                x = q + h * a.q_head + i * a.q_row;
                y = dout + h * a.do_head + i * a.do_row;
            });
        }
        at_query += E::kRows;
        while (at_query >= nq) {
            at_query -= nq;
            ++at_head;
        }
        if (threadIdx.x < E::kRows) {
            const bool in = (int)threadIdx.x < left;
            next_off = in ? E::kBias - lse[first + threadIdx.x] * kLog2e : 0.f;
            next_delta = in ? -delta[first + threadIdx.x] : 0.f;
        }
    };
    if (begin < end) load(begin);
    for (int first = begin; first < end; first += E::kRows) {
        __syncthreads();
        stage.store(qs, dos);
        if (threadIdx.x < E::kRows) {
            off[threadIdx.x] = next_off;
            deltas[threadIdx.x] = next_delta;
        }
        __syncthreads();
        if (first + E::kRows < end) load(first + E::kRows);
#pragma unroll
        for (int sub = 0; sub < G::NS; ++sub) {
            f32x16 s = {}, dp;
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const f32x4 d4 = *reinterpret_cast<const f32x4*>(&deltas[sub * 32 + 2 * i + 4 * half]);
#pragma unroll
                for (int j = 0; j < 4; ++j) dp[i + j] = d4[j];
            }
#pragma unroll
            for (int k = 0; k < G::KS; ++k) {
                s = mma(direct<DT, DK>(qs, sub * 32 + (lane & 31), k, half), kf[k], s);
                dp = mma(direct<DT, DK>(dos, sub * 32 + (lane & 31), k, half), vf[k], dp);
            }
            float pr[16], ds[1][16];
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const f32x4 o4 = *reinterpret_cast<const f32x4*>(&off[sub * 32 + 2 * i + 4 * half]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    pr[i + j] = __builtin_amdgcn_exp2f(fmaf(s[i + j], p.c, o4[j]));
                    ds[0][i + j] = pr[i + j] * dp[i + j];
                }
            }
            if (first + E::kRows > end) {  // rows that are not there: 0, also beside keys that are not finite
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (first + sub * 32 + 8 * (i / 4) + 4 * half + i % 4 >= end) pr[i] = ds[0][i] = 0.f;
            }
            if constexpr (E::kScaled) scale.apply(ds, dk);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const auto pf = rounded<DT>(pr, t), f = rounded<DT>(ds[0], t);
#pragma unroll
                for (int j = 0; j < G::MS; ++j) {
                    dv[j] = mma(transposed<DT, G::LS>(dos, sub * 32 + 16 * t, 32 * j, lane), pf, dv[j]);
                    dk[j] = mma(transposed<DT, G::LS>(qs, sub * 32 + 16 * t, 32 * j, lane), f, dk[j]);
                }
            }
        }
    }
    if (key64 >= a.nk) return;
    constexpr float unbias = DT == NORI_F16 ? 0x1p-15f : 1.f;
    const float byk = there ? a.scale * unbias * (E::kScaled ? scale.inverse() : 1.f) : 0.f, byv = unbias;
    T* out = reinterpret_cast<T*>(a.dkv) + (((w.b * a.nk + key) * 2) * a.kv_heads + w.hk) * a.d;
    float* part = p.part + ((w.split * a.bg * a.kv_heads + w.unit) * a.nk + key) * 2 * a.d;
#pragma unroll
    for (int j = 0; j < G::MS; ++j)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int col = 32 * j + 2 * i + 4 * half;
            float x[4], y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[e] = there ? dk[j][i + e] * byk : 0.f;
                y[e] = there ? dv[j][i + e] * byv : 0.f;
            }
            if (col >= a.d) continue;
            if (p.splits > 1) {
                *reinterpret_cast<f32x4*>(part + col) = f32x4{x[0], x[1], x[2], x[3]};
                *reinterpret_cast<f32x4*>(part + a.d + col) = f32x4{y[0], y[1], y[2], y[3]};
            } else {
                store4<DT>(out + col, x);
                store4<DT>(out + (int64_t)a.kv_heads * a.d + col, y);
            }
        }
}

template <int DT, int DK, int W>
int launch(Kind kind, const Args& p, int64_t blocks, hipStream_t stream) {
    const dim3 grid((unsigned)blocks), threads(kThreads);
    switch (kind) {
        case kForward: hipLaunchKernelGGL((forward_kernel<DT, DK, W>), grid, threads, 0, stream, p); break;
        case kDq: hipLaunchKernelGGL((dq_kernel<DT, DK, W>), grid, threads, 0, stream, p); break;
        case kDkv: hipLaunchKernelGGL((dkv_kernel<DT, DK, W>), grid, threads, 0, stream, p); break;
    }
    return launch_status("attention_train");
}

template <int DT, int W>
int launch_width(Kind kind, const Args& p, int64_t blocks, hipStream_t stream) {
    const int d = p.a.d;
    if (d <= 32) return launch<DT, 32, W>(kind, p, blocks, stream);
    if (d <= 48) return launch<DT, 48, W>(kind, p, blocks, stream);
    if (d <= 64) return launch<DT, 64, W>(kind, p, blocks, stream);
    if (d <= 96) return launch<DT, 96, W>(kind, p, blocks, stream);
    return launch<DT, 128, W>(kind, p, blocks, stream);
}

// Chunks of 16 bytes, where the host found everything aligned to them, or of 4 elements.
template <int DT>
int launch_chunks(Kind kind, const Args& p, int64_t blocks, hipStream_t stream) {
    if constexpr (DT != NORI_F32)
        if (p.wide) return launch_width<DT, 8>(kind, p, blocks, stream);
    return launch_width<DT, 4>(kind, p, blocks, stream);
}

}  // namespace attn_train
}  // namespace nori
