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
    static constexpr int LS = DK + E::kPad;      // elements from one row of a tile to the next
    static constexpr int kTail = DP - DK;        // behind a tile: what the last products' columns past DK reach of its last row
    static constexpr int KS = DK / 16, MS = DP / 32;
};

// The order in which the compiler lays out `products` products, each with `reads` reads of its operand from LDS: the operands of
// `ahead` products first, then a product and the next operand's reads in turn. Left to itself it reads an operand right
// before its product, a latency every time.
template <int DT, int products, int reads, int ahead, int before = 0>
__device__ __forceinline__ void interleave() {
    if constexpr (DT != NORI_F32) {
        __builtin_amdgcn_sched_group_barrier(0x100, before + ahead * reads, 0);
#pragma unroll
        for (int i = 0; i < products - ahead; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, reads, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x8, ahead, 0);
    }
}

// Left operand: row `row` (lane % 32 of a step's 32) of a tile, its columns 16 k + 8 h .. + 7.
template <int DT, int DK>
__device__ __forceinline__ typename El<DT>::Frag direct(const typename El<DT>::T* tile, int row, int k, int half) {
    const auto* p = tile + row * Geo<DT, DK>::LS + 16 * k + 8 * half;
    return *reinterpret_cast<const typename El<DT>::Frag*>(p);
}

// Lane's row of a tile's 32-row step `sub`, of T16 sixteens: past them the last one, whose products are not used.
template <int T16>
__device__ __forceinline__ int row_in(int sub, int lane) {
    const int row = sub * 32 + (lane & 31);
    return 32 * sub + 32 > 16 * T16 ? min(row, 16 * T16 - 1) : row;
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

// Writes a column of a result, `by` times, as the d elements of a row: in the type, or fp32 of a part.
template <int DT, int MS, class Out>
__device__ __forceinline__ void store_row(Out* out, const f32x16 (&x)[MS], float by, int d, int half) {
#pragma unroll
    for (int j = 0; j < MS; ++j)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int col = 32 * j + 2 * i + 4 * half;
            if (col >= d) continue;
            f32x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = x[j][i + e] * by;
            if constexpr (sizeof(Out) == 4) {
                *reinterpret_cast<f32x4*>(out + col) = v;
            } else if constexpr (DT == NORI_F16) {
                typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
                *reinterpret_cast<f16x4*>(out + col) = __builtin_convertvector(v, f16x4);
            } else {
                typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
                *reinterpret_cast<bf16x4*>(out + col) = __builtin_convertvector(v, bf16x4);
            }
        }
}

// The same for the 32 rows of a wavefront's columns by way of LDS (its own 32 rows there): a lane's columns are apart in memory, 32
// lines an access, which the address units bound short scans by; from LDS rows go out side by side. to(row): where it begins.
// (Units of 33 x 33 of 44, fp16, 8,192 x 8: backward 487 us without, 404 so; x 10 of 51 x 51 of 56: 951 and 859.)
template <int DT, int DK, int W, int LS, int MS, class To>
__device__ __forceinline__ void store_rows(typename El<DT>::T* lds, const f32x16 (&x)[MS], float by, int d, int lane, int rows, To to) {
    using T = typename El<DT>::T;
    typedef uint32_t Chunk __attribute__((ext_vector_type(W * sizeof(T) / 4)));
    constexpr int CH = DK / W;
    if ((lane & 31) < rows) store_row<DT>(lds + (lane & 31) * LS, x, by, d, lane >> 5);  // (past them another's may begin)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < (32 * CH + 63) / 64; ++i) {
        const int idx = lane + 64 * i, row = idx / CH, col = W * (idx % CH);
        if (row < rows && col < d) *reinterpret_cast<Chunk*>(to(row) + col) = *reinterpret_cast<const Chunk*>(lds + row * LS + col);
    }
    __builtin_amdgcn_wave_barrier();
}

// Query row r of a unit: head and query.
struct Row { int64_t head, query; };
__device__ __forceinline__ Row row_of(const Args& p, int64_t unit_head, int r) {
    if (p.group == 1) return {unit_head, r};
    const int h = r / (int)p.a.nq;
    return {unit_head * p.group + h, r - h * (int)p.a.nq};
}

// Rows of a tile that passes a workgroup of NW wavefronts.
template <int DT, int NW>
constexpr int kTileOf = NW == 1 ? 32 : El<DT>::kRows;

// The work of a workgroup: part `split` of what passes by tile `tile` of what stays, in a unit.
// heads: the heads of one tile are neighbours and not the tiles of one head.
struct Block { int64_t tile, split, unit, b, hk; };
__device__ __forceinline__ Block block_of(const Args& p, bool heads = false) {
    int64_t i = work_index(blockIdx.x, gridDim.x);
    Block w;
    if (heads) {
        w.hk = i % p.a.kv_heads;
        i /= p.a.kv_heads;
        w.tile = i % p.tiles;
        i /= p.tiles;
        w.split = i % p.splits;
        w.b = i / p.splits;
        w.unit = w.b * p.a.kv_heads + w.hk;
        return w;
    }
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
template <int DT, int DK, int W, int TH, int ROWS> struct Stage {
    using G = Geo<DT, DK>;
    using E = El<DT>;
    using T = typename E::T;
    typedef uint32_t Chunk __attribute__((ext_vector_type(W * sizeof(T) / 4)));
    static constexpr int CH = DK / W;                                       // chunks a row
    static constexpr int N = (ROWS * CH + TH - 1) / TH;     // chunks a thread, a tile
    Chunk x[N], y[N];
    uint32_t ox[N], oy[N];
    int row[N];  // past every tile for chunks that no row has: they stay zero

    __device__ __forceinline__ void place(int d, int64_t x_stride, int64_t y_stride) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int idx = threadIdx.x + i * TH, r = idx / CH, col = W * (idx % CH);
            row[i] = r < ROWS && col < d ? r : 1 << 30;
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
                const int col = W * ((threadIdx.x + i * TH) % CH);
                x[i] = *reinterpret_cast<const Chunk*>(px + col);
                y[i] = *reinterpret_cast<const Chunk*>(py + col);
            }
        }
    }
    __device__ __forceinline__ void store(T* tx, T* ty) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int idx = threadIdx.x + i * TH, to = idx / CH * G::LS + W * (idx % CH);
            if (ROWS * CH % TH == 0 || idx < ROWS * CH) {
                *reinterpret_cast<Chunk*>(tx + to) = x[i];
                *reinterpret_cast<Chunk*>(ty + to) = y[i];
            }
        }
    }
};

// ---------------------------------------------------------------- forward
// One tile's part of the forward pass: `left` of its keys are there.
template <int DT, int DK, int NS>
__device__ __forceinline__ void forward_step(const typename El<DT>::T* ks, const typename El<DT>::T* vs, int left,
                                             const typename El<DT>::Frag (&qf)[DK / 16], f32x16 (&o)[Geo<DT, DK>::MS], float& m, float& l,
                                             float c, int lane) {
    using E = El<DT>;
    using G = Geo<DT, DK>;
    const int half = lane >> 5;
    f32x16 s[NS];
#pragma unroll
    for (int sub = 0; sub < NS; ++sub) {
        s[sub] = f32x16{};
#pragma unroll
        for (int k = 0; k < G::KS; ++k) s[sub] = mma(direct<DT, DK>(ks, sub * 32 + (lane & 31), k, half), qf[k], s[sub]);
    }
    if (left < 32 * NS) {
#pragma unroll
        for (int sub = 0; sub < NS; ++sub)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (sub * 32 + 8 * (i / 4) + i % 4 >= left - 4 * half) s[sub][i] = -INFINITY;
    }
    float top = s[0][0];
#pragma unroll
    for (int i = 1; i < 16 * NS; ++i) top = fmaxf(top, s[i / 16][i % 16]);
    top = fmaxf(top, other_half(top));
    // the maximum that p is taken against moves when one passes it by 2^kSlack: rarely, after the first tiles
    if (__any((top - m) * c > E::kSlack)) {
        const float next = fmaxf(m, top);
        const float shrink = next == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - next) * c);
        m = next;
        l *= shrink;
#pragma unroll
        for (int j = 0; j < 16 * G::MS; ++j) o[j / 16][j % 16] *= shrink;  // (whole vectors end up copied on every step)
    }
    const float off = E::kTop - (m == -INFINITY ? 0.f : m * c);  // (all keys so far at -inf: their p is 0)
#pragma unroll
    for (int sub = 0; sub < NS; ++sub) {
        float e[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            e[i] = __builtin_amdgcn_exp2f(fmaf(s[sub][i], c, off));
            l += e[i];
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const auto pf = rounded<DT>(e, t);
#pragma unroll
            for (int j = 0; j < G::MS; ++j) o[j] = mma(transposed<DT, G::LS>(vs, sub * 32 + 16 * t, 32 * j, lane), pf, o[j]);
        }
    }
}

// The magnitude of the logits' factor: the running maximum wants it positive, so a negative one changes the queries' signs, and one
// of 0 makes them 0 beside a factor of 1.
template <int DT, int KS>
__device__ __forceinline__ float positive(float c, typename El<DT>::Frag (&q)[KS]) {
    if (c <= 0.f) {
        const float sign = c < 0.f ? -1.f : 0.f;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int j = 0; j < 8; ++j) at(q[k], j) = at(q[k], j) * sign;
    }
    return c == 0.f ? 1.f : fabsf(c);
}

// Bound by the matrix instructions and the exponentials between them over many rows, by HBM over few. 9 x 2 heads of 64, 8,192 x
// 8,192, bf16: 398 us (777 TFLOP/s; the card settled, as all figures here); four wavefronts a SIMD spill. One row over 65,536 keys: 49 us
// (6.2 TB/s, keys in part still in the cache) and 10 for the parts.
template <int DT, int DK, int W, int NW>
__global__ __launch_bounds__(64 * NW, DK <= 64 && NW == 4 ? 3 : 2) void forward_kernel(const Args p) {
    using E = El<DT>;
    using G = Geo<DT, DK>;
    using T = typename E::T;
    constexpr int kRows = kTileOf<DT, NW>;
    __shared__ __attribute__((aligned(16))) T ks[kRows * G::LS + G::kTail];
    __shared__ __attribute__((aligned(16))) T vs[kRows * G::LS + G::kTail];
    const auto& a = p.a;
    const Block w = block_of(p);
    const int lane = threadIdx.x & 63, half = lane >> 5, wave = threadIdx.x >> 6;
    const int64_t r64 = w.tile * 32 * NW + wave * 32 + (lane & 31);
    const bool there = r64 < p.rows;
    const int r = (int)r64;
    const Row row = there ? row_of(p, w.hk, r) : Row{w.hk * p.group, 0};
    const int length = length_of(a, w.b);
    const int begin = (int)(w.split * p.per_split);
    const int end = (int)min((int64_t)length, w.split * p.per_split + p.per_split);

    typename E::Frag qf[G::KS];
    load_own<DT, DK, W>(qf, reinterpret_cast<const T*>(a.q) + w.b * a.q_bg + row.query * a.q_row + row.head * a.q_head, there, a.d, half);
    const float c = positive<DT>(p.c, qf);

    const T* kv = reinterpret_cast<const T*>(a.kv) + w.b * a.kv_bg + w.hk * a.kv_head + begin * a.kv_row;
    Stage<DT, DK, W, 64 * NW, kRows> stage;
    stage.place(a.d, a.kv_row, a.kv_row);
    if (begin < end) stage.load(kv, kv + a.kv_half, end - begin);
    float m = -INFINITY, l = 0.f;  // of this half-wave's keys
    f32x16 o[G::MS] = {};
    const auto finish = [&](const f32x16 (&x)[G::MS], float by, float lse2) {
        if (p.splits > 1) {
            const int64_t to = (w.split * a.bg * a.kv_heads + w.unit) * p.rows + r;
            if (half == 0) p.part_lse[to] = lse2;
            store_row<DT>(p.part + to * a.d, x, by, a.d, half);
            return;
        }
        if (half == 0 && a.lse) a.lse[w.unit * p.rows + r] = lse2 * kLn2;
        store_row<DT>(reinterpret_cast<T*>(a.out) + ((w.b * a.nq + row.query) * a.heads + row.head) * a.d, x, by, a.d, half);
    };
    if (begin >= end) {  // no keys: zeros. (On a path of its own: sums that the loop may skip would be copied on every step.)
        if (there) finish(o, 0.f, -INFINITY);
        return;
    }
    for (int first = begin; first < end; first += kRows) {
        __syncthreads();
        stage.store(ks, vs);
        __syncthreads();
        kv += kRows * a.kv_row;
        if (first + kRows < end) stage.load(kv, kv + a.kv_half, end - first - kRows);
        forward_step<DT, DK, kRows / 32>(ks, vs, end - first, qf, o, m, l, c, lane);
    }
    if (!there) return;
    l += other_half(l);
    finish(o, 1.f / l, __builtin_amdgcn_logf(l) - E::kTop + m * c);
}

// What takes kBias off again.
template <int DT>
constexpr float kUnbias = DT == NORI_F16 ? 0x1p-15f : 1.f;

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
            for (int j = 0; j < 16 * MS; ++j) acc[j / 16][j % 16] *= by;  // (whole vectors end up copied on every step)
            f = next;
        }
#pragma unroll
        for (int i = 0; i < 16 * NS; ++i) x[i / 16][i % 16] *= f;
    }
    __device__ __forceinline__ float inverse() const { return f == 0.f ? 1.f : 1.f / f; }
};

// ---------------------------------------------------------------- dq, and delta for dk and dv
// The sum of a row's products of dout and out.
template <int DT, int KS>
__device__ __forceinline__ float row_sum(typename El<DT>::Frag (&x)[KS], typename El<DT>::Frag (&y)[KS]) {
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j) sum = fmaf(at(x[k], j), at(y[k], j), sum);
    return sum + other_half(sum);
}

// One tile's part of dq: `left` of its keys are there.
template <int DT, int DK, int NS>
__device__ __forceinline__ void dq_step(const typename El<DT>::T* ks, const typename El<DT>::T* vs, int left,
                                        const typename El<DT>::Frag (&qf)[DK / 16], const typename El<DT>::Frag (&dof)[DK / 16],
                                        f32x16 (&dq)[Geo<DT, DK>::MS], Scale& scale, float c, float lse2, float delta, int lane) {
    using G = Geo<DT, DK>;
    const int half = lane >> 5;
    float ds[NS][16];
#pragma unroll
    for (int sub = 0; sub < NS; ++sub) {
        f32x16 s = {}, dp;
#pragma unroll
        for (int i = 0; i < 16; ++i) dp[i] = -delta;
#pragma unroll
        for (int k = 0; k < G::KS; ++k) {
            s = mma(direct<DT, DK>(ks, sub * 32 + (lane & 31), k, half), qf[k], s);
            dp = mma(direct<DT, DK>(vs, sub * 32 + (lane & 31), k, half), dof[k], dp);
        }
        interleave<DT, 2 * G::KS, 1, 4>();
#pragma unroll
        for (int i = 0; i < 16; ++i) ds[sub][i] = __builtin_amdgcn_exp2f(fmaf(s[i], c, -lse2)) * dp[i];
    }
    if (left < 32 * NS) {
#pragma unroll
        for (int sub = 0; sub < NS; ++sub)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (sub * 32 + 8 * (i / 4) + i % 4 >= left - 4 * half) ds[sub][i] = 0.f;
    }
    if constexpr (El<DT>::kScaled) scale.apply(ds, dq);
#pragma unroll
    for (int sub = 0; sub < NS; ++sub)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const auto f = rounded<DT>(ds[sub], t);
#pragma unroll
            for (int j = 0; j < G::MS; ++j) dq[j] = mma(transposed<DT, G::LS>(ks, sub * 32 + 16 * t, 32 * j, lane), f, dq[j]);
        }
}

// The same of rows whose keys are all in this tile, which takes delta = sum of p (dout v) from them: with few keys ds is a small
// difference, and delta of the result as it was rounded would be off by as much.
// T16: the sixteens of rows that the tile has.
template <int DT, int DK, int NS, int T16 = 2 * NS>
__device__ __forceinline__ void dq_whole(const typename El<DT>::T* ks, const typename El<DT>::T* vs, int left,
                                         const typename El<DT>::Frag (&qf)[DK / 16], const typename El<DT>::Frag (&dof)[DK / 16],
                                         f32x16 (&dq)[Geo<DT, DK>::MS], Scale& scale, float c, float lse2, float& delta, int lane) {
    using G = Geo<DT, DK>;
    const int half = lane >> 5;
    float pr[NS][16], ds[NS][16];
    delta = 0.f;
#pragma unroll
    for (int sub = 0; sub < NS; ++sub) {
        f32x16 s = {}, dp = {};
#pragma unroll
        for (int k = 0; k < G::KS; ++k) {
            s = mma(direct<DT, DK>(ks, row_in<T16>(sub, lane), k, half), qf[k], s);
            dp = mma(direct<DT, DK>(vs, row_in<T16>(sub, lane), k, half), dof[k], dp);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const bool in = 2 * sub + i / 8 < T16 && sub * 32 + 8 * (i / 4) + i % 4 < left - 4 * half;
            pr[sub][i] = in ? __builtin_amdgcn_exp2f(fmaf(s[i], c, -lse2)) : 0.f;
            if (sub == 0 && i == 0 && left == 1 && half == 0) pr[0][0] = fmaf(pr[0][0], 0.f, 1.f);  // one key: 1, so that ds is 0
            ds[sub][i] = in ? dp[i] : 0.f;
            delta = fmaf(pr[sub][i], ds[sub][i], delta);
        }
    }
    delta += other_half(delta);
#pragma unroll
    for (int sub = 0; sub < NS; ++sub)
#pragma unroll
        for (int i = 0; i < 16; ++i) ds[sub][i] = pr[sub][i] * (ds[sub][i] - delta);
    if constexpr (El<DT>::kScaled) scale.apply(ds, dq);
#pragma unroll
    for (int sub = 0; sub < NS; ++sub)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            if (2 * sub + t >= T16) continue;
            const auto f = rounded<DT>(ds[sub], t);
#pragma unroll
            for (int j = 0; j < G::MS; ++j) dq[j] = mma(transposed<DT, G::LS>(ks, sub * 32 + 16 * t, 32 * j, lane), f, dq[j]);
        }
}

// Three products of the pairs, bound as the forward pass over many rows: 9 x 2 heads of 64, 8,192 x 8,192, bf16:
// 487 us (952 TFLOP/s). Three wavefronts a SIMD spill.
template <int DT, int DK, int W, int NW>
__global__ __launch_bounds__(64 * NW, DT == NORI_F32 && DK > 96 ? 1 : 2) void dq_kernel(const Args p) {
    using E = El<DT>;
    using G = Geo<DT, DK>;
    using T = typename E::T;
    constexpr int kRows = kTileOf<DT, NW>;
    __shared__ __attribute__((aligned(16))) T ks[kRows * G::LS + G::kTail];
    __shared__ __attribute__((aligned(16))) T vs[kRows * G::LS + G::kTail];
    const auto& a = p.a;
    const Block w = block_of(p);
    const int lane = threadIdx.x & 63, half = lane >> 5, wave = threadIdx.x >> 6;
    const int64_t r64 = w.tile * 32 * NW + wave * 32 + (lane & 31);
    const bool there = r64 < p.rows;
    const int r = (int)r64;
    const Row row = there ? row_of(p, w.hk, r) : Row{w.hk * p.group, 0};
    const int64_t unit_row = w.unit * p.rows + r;
    const int length = length_of(a, w.b);
    const int begin = (int)(w.split * p.per_split);
    const bool whole = length <= kRows;  // all keys in the first part's first tile
    const int end = a.dq || whole ? (int)min((int64_t)length, w.split * p.per_split + p.per_split) : begin;

    typename E::Frag dof[G::KS], qf[G::KS];
    load_own<DT, DK, W>(dof, reinterpret_cast<const T*>(a.dout) + w.b * a.do_bg + row.query * a.do_row + row.head * a.do_head, there, a.d, half);
    load_own<DT, DK, W>(qf, reinterpret_cast<const T*>(a.out) + ((w.b * a.nq + row.query) * a.heads + row.head) * a.d, there, a.d, half);
    float delta = row_sum<DT>(dof, qf);
    if (there && half == 0 && w.split == 0 && !whole) p.delta[unit_row] = delta;
    if (begin >= end && !a.dq) return;
    load_own<DT, DK, W>(qf, reinterpret_cast<const T*>(a.q) + w.b * a.q_bg + row.query * a.q_row + row.head * a.q_head, there, a.d, half);
    const float lse2 = there ? a.lse[unit_row] * kLog2e : 0.f;

    const T* kv = reinterpret_cast<const T*>(a.kv) + w.b * a.kv_bg + w.hk * a.kv_head + begin * a.kv_row;
    Stage<DT, DK, W, 64 * NW, kRows> stage;
    stage.place(a.d, a.kv_row, a.kv_row);
    if (begin < end) stage.load(kv, kv + a.kv_half, end - begin);
    f32x16 dq[G::MS] = {};
    Scale scale;
    if (whole && begin < end) {
        stage.store(ks, vs);
        __syncthreads();
        dq_whole<DT, DK, kRows / 32>(ks, vs, length, qf, dof, dq, scale, p.c, lse2, delta, lane);
        if (there && half == 0) p.delta[unit_row] = delta;
        if (!a.dq) return;
    }
    for (int first = whole ? end : begin; first < end; first += kRows) {
        __syncthreads();
        stage.store(ks, vs);
        __syncthreads();
        kv += kRows * a.kv_row;
        if (first + kRows < end) stage.load(kv, kv + a.kv_half, end - first - kRows);
        dq_step<DT, DK, kRows / 32>(ks, vs, end - first, qf, dof, dq, scale, p.c, lse2, delta, lane);
    }
    if (!there) return;
    const float by = a.scale * (E::kScaled ? scale.inverse() : 1.f);
    if (p.splits > 1) store_row<DT>(p.part + (w.split * a.bg * a.kv_heads * p.rows + unit_row) * a.d, dq, by, a.d, half);
    else store_row<DT>(reinterpret_cast<T*>(a.dq) + ((w.b * a.nq + row.query) * a.heads + row.head) * a.d, dq, by, a.d, half);
}

// ---------------------------------------------------------------- dk and dv
// One tile's part of dk and dv: `left` of its rows are there. off: kBias - log2 of a row's sum, deltas: its -delta, what the
// products of dout and v start from.
template <int DT, int DK, int NS, int T16 = 2 * NS>
__device__ __forceinline__ void dkv_step(const typename El<DT>::T* qs, const typename El<DT>::T* dos, const float* off, const float* deltas,
                                         int left, const typename El<DT>::Frag (&kf)[DK / 16], const typename El<DT>::Frag (&vf)[DK / 16],
                                         f32x16 (&dk)[Geo<DT, DK>::MS], f32x16 (&dv)[Geo<DT, DK>::MS], Scale& scale, float c, int lane) {
    using G = Geo<DT, DK>;
    const int half = lane >> 5;
#pragma unroll
    for (int sub = 0; sub < NS; ++sub) {
        f32x16 s = {}, dp;
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const f32x4 d4 = *reinterpret_cast<const f32x4*>(&deltas[sub * 32 + 2 * i + 4 * half]);
#pragma unroll
            for (int j = 0; j < 4; ++j) dp[i + j] = d4[j];
        }
#pragma unroll
        for (int k = 0; k < G::KS; ++k) {
            s = mma(direct<DT, DK>(qs, row_in<T16>(sub, lane), k, half), kf[k], s);
            dp = mma(direct<DT, DK>(dos, row_in<T16>(sub, lane), k, half), vf[k], dp);
        }
        interleave<DT, 2 * G::KS, 1, 4, 4>();
        float pr[16], ds[1][16];
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const f32x4 o4 = *reinterpret_cast<const f32x4*>(&off[sub * 32 + 2 * i + 4 * half]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                pr[i + j] = __builtin_amdgcn_exp2f(fmaf(s[i + j], c, o4[j]));
                ds[0][i + j] = pr[i + j] * dp[i + j];
            }
        }
        if (left < 32 * NS) {  // rows that are not there: 0, also beside keys that are not finite
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (2 * sub + i / 8 >= T16 || sub * 32 + 8 * (i / 4) + i % 4 >= left - 4 * half) pr[i] = ds[0][i] = 0.f;
        }
        if constexpr (El<DT>::kScaled) scale.apply(ds, dk);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            if (2 * sub + t >= T16) continue;
            const auto pf = rounded<DT>(pr, t), f = rounded<DT>(ds[0], t);
#pragma unroll
            for (int j = 0; j < G::MS; ++j) {
                dv[j] = mma(transposed<DT, G::LS>(dos, sub * 32 + 16 * t, 32 * j, lane), pf, dv[j]);
                dk[j] = mma(transposed<DT, G::LS>(qs, sub * 32 + 16 * t, 32 * j, lane), f, dk[j]);
            }
        }
        interleave<DT, 4 * G::MS, 2, 2>();
    }
}

// Four products of the pairs; keys stay, so two sums of 32 x D a wavefront take the registers that a third wavefront would need. The
// same rows: 685 us (903 TFLOP/s).
// kRows: of the tile that passes. Up to 32 rows in all take one tile of 32; the time goes to keys in and out then, so every
// wavefront's results have room in LDS at once, and heads whose rows share lines of memory are neighbours. One row of 8 heads over 8,192
// keys, 64 times, dq, dk and dv together: bf16 heads of 64 700 us (4.6 TB/s; results by turns 790, neighbouring heads 752), fp16 of 44
// 757 (869 in tiles of 64 rows, 891 with a head's tiles as neighbours).
template <int DT, int DK, int W, int NW, int kRows>
__global__ __launch_bounds__(64 * NW, DK <= 64 ? 2 : 1) void dkv_kernel(const Args p) {
    using E = El<DT>;
    using G = Geo<DT, DK>;
    using T = typename E::T;
    constexpr bool kFewRows = kRows != kTileOf<DT, NW>;
    // rows of the tiles, or of the results on their way out
    constexpr int kRoom = !kFewRows ? kRows : (sizeof(T) == 2 && DK <= 64 ? 32 * NW : kTileOf<DT, NW>);
    __shared__ __attribute__((aligned(16))) T qs[kRoom * G::LS + G::kTail];
    __shared__ __attribute__((aligned(16))) T dos[kRoom * G::LS + G::kTail];
    __shared__ __attribute__((aligned(16))) float off[kRows];
    __shared__ __attribute__((aligned(16))) float deltas[kRows];
    const auto& a = p.a;
    const Block w = block_of(p, kFewRows && a.d * sizeof(T) % 128 != 0);
    const int lane = threadIdx.x & 63, half = lane >> 5, wave = threadIdx.x >> 6;
    const int64_t key64 = w.tile * 32 * NW + wave * 32 + (lane & 31);
    const int length = length_of(a, w.b);
    const bool there = key64 < length;
    const int key = (int)key64;
    const int begin = (int)(w.split * p.per_split);
    // (a tile behind the length has no products, its gradients are zeros)
    const int end = w.tile * 32 * NW < length ? (int)min(p.rows, w.split * p.per_split + p.per_split) : begin;

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
    Stage<DT, DK, W, 64 * NW, kRows> stage;
    stage.place(a.d, a.q_row, a.do_row);
    float next_off = 0.f, next_delta = 0.f;
    const auto load = [&](int first) {
        const int left = end - first;
        const T* px = q + at_head * a.q_head + at_query * a.q_row;
        const T* py = dout + at_head * a.do_head + at_query * a.do_row;
        if (at_query + kRows <= nq || p.group == 1) {
            stage.load(px, py, left);
        } else if (nq >= kRows) {
            stage.load_over(px, py, left, nq - at_query, (a.q_head - nq * a.q_row) * (int64_t)sizeof(T),
                            (a.do_head - nq * a.do_row) * (int64_t)sizeof(T));
        } else {
            stage.load_each(left, [&](int row, const T*& x, const T*& y) {
                const int h = (first + row) / nq, i = first + row - h * nq;
                x = q + h * a.q_head + i * a.q_row;
                y = dout + h * a.do_head + i * a.do_row;
            });
        }
        at_query += kRows;
        if (p.group > 1) {
            const int heads = at_query / nq;
            at_head += heads;
            at_query -= heads * nq;
        }
        if (threadIdx.x < kRows) {
            const bool in = (int)threadIdx.x < left;
            next_off = in ? E::kBias - lse[first + threadIdx.x] * kLog2e : 0.f;
            next_delta = in ? -delta[first + threadIdx.x] : 0.f;
        }
    };
    if (begin < end) load(begin);
    for (int first = begin; first < end; first += kRows) {
        __syncthreads();
        stage.store(qs, dos);
        if (threadIdx.x < kRows) {
            off[threadIdx.x] = next_off;
            deltas[threadIdx.x] = next_delta;
        }
        __syncthreads();
        if (first + kRows < end) load(first + kRows);
        dkv_step<DT, DK, kRows / 32>(qs, dos, off, deltas, end - first, kf, vf, dk, dv, scale, p.c, lane);
    }
    if (!there) {  // past the length
#pragma unroll
        for (int j = 0; j < G::MS; ++j) dk[j] = dv[j] = f32x16{};
    }
    const float byk = a.scale * kUnbias<DT> * (E::kScaled ? scale.inverse() : 1.f);
    if (p.splits > 1) {
        if (key64 >= a.nk) return;
        float* part = p.part + ((w.split * a.bg * a.kv_heads + w.unit) * a.nk + key) * 2 * a.d;
        store_row<DT>(part, dk, byk, a.d, half);
        store_row<DT>(part + a.d, dv, kUnbias<DT>, a.d, half);
        return;
    }
    // there is room for 32 rows of each of so many wavefronts at a time
    constexpr int kAtOnce = kRoom / 32;
    const int64_t from = w.tile * 32 * NW + wave * 32;
    T* to = reinterpret_cast<T*>(a.dkv) + ((w.b * a.nk + from) * 2 * a.kv_heads + w.hk) * a.d;
    const int left = (int)min((int64_t)32, a.nk - from);
#pragma unroll
    for (int turn = 0; turn < NW / kAtOnce; ++turn) {
        __syncthreads();
        if (wave / kAtOnce != turn) continue;
        const int mine = wave % kAtOnce * 32 * G::LS;
        store_rows<DT, DK, W, G::LS>(qs + mine, dk, byk, a.d, lane, left, [&](int i) { return to + (int64_t)i * 2 * a.kv_heads * a.d; });
        store_rows<DT, DK, W, G::LS>(dos + mine, dv, kUnbias<DT>, a.d, lane, left, [&](int i) { return to + ((int64_t)i * 2 + 1) * a.kv_heads * a.d; });
    }
}

// ---------------------------------------------------------------- few rows and few keys
// The forward pass of a unit of up to 32 NW rows and keys. One tile and no loop: half the registers of forward_kernel, so twice the
// wavefronts, which is what units this short go by: 8,192 x 8 units of 33 x 33 of 44, fp16, 188 us (4.0 TB/s).
template <int DT, int DK, int W, int NW>
__global__ __launch_bounds__(64 * NW, 4) void forward_few_kernel(const Args p) {
    using E = El<DT>;
    using G = Geo<DT, DK>;
    using T = typename E::T;
    __shared__ __attribute__((aligned(16))) T ks[32 * NW * G::LS + G::kTail];
    __shared__ __attribute__((aligned(16))) T vs[32 * NW * G::LS + G::kTail];
    const auto& a = p.a;
    const int64_t unit = work_index(blockIdx.x, gridDim.x), b = unit / a.kv_heads, hk = unit % a.kv_heads;
    const int lane = threadIdx.x & 63, half = lane >> 5, wave = threadIdx.x >> 6, own = wave * 32 + (lane & 31);
    const int length = length_of(a, b), rows = (int)p.rows;
    const T* kv = reinterpret_cast<const T*>(a.kv) + b * a.kv_bg + hk * a.kv_head;
    const bool there = own < rows;
    const Row row = there ? row_of(p, hk, own) : Row{hk * p.group, 0};
    typename E::Frag qf[G::KS];
    {
        Stage<DT, DK, W, 64 * NW, 32 * NW> keys;
        keys.place(a.d, a.kv_row, a.kv_row);
        keys.load(kv, kv + a.kv_half, length);
        load_own<DT, DK, W>(qf, reinterpret_cast<const T*>(a.q) + b * a.q_bg + row.query * a.q_row + row.head * a.q_head, there, a.d, half);
        keys.store(ks, vs);
    }
    const float c = positive<DT>(p.c, qf);
    __syncthreads();
    float m = -INFINITY, l = 0.f;
    f32x16 o[G::MS] = {};
    if (length > 0) forward_step<DT, DK, NW>(ks, vs, length, qf, o, m, l, c, lane);
    l += other_half(l);
    if (there && half == 0 && a.lse) a.lse[unit * p.rows + own] = length > 0 ? (__builtin_amdgcn_logf(l) - E::kTop + m * c) * kLn2 : -INFINITY;
    T* out = reinterpret_cast<T*>(a.out) + b * a.nq * a.heads * a.d;
    __syncthreads();  // the tile is everyone's until here
    store_rows<DT, DK, W, G::LS>(ks + wave * 32 * G::LS, o, length > 0 ? 1.f / l : 0.f, a.d, lane, rows - wave * 32, [&](int i) {
        const Row to = row_of(p, hk, wave * 32 + i);
        return out + (to.query * a.heads + to.head) * a.d;
    });
}

// The whole backward pass of such a unit: both sides in LDS, read from memory once, where the kernels above read them twice and the
// rows' sums pass through memory. (Keys first and queries in their place later take half the LDS and a wavefront a SIMD more, but
// read the queries twice: 8,192 x 8 units of 33 x 33 of 44, fp16, 656 us so, 557 this way.) ROWS is 48 where that holds both sides, for LDS
// that lets a wavefront a SIMD more in and a quarter less work: the same units 529 us with 64, 499 with 48. Now: 401 us (3.3 TB/s), bound
// by the instructions that tiles half empty take.
template <int DT, int DK, int W, int NW, int ROWS>
__global__ __launch_bounds__(64 * NW, 2) void backward_few_kernel(const Args p) {
    using E = El<DT>;
    using G = Geo<DT, DK>;
    using T = typename E::T;
    constexpr int kTile = ROWS * G::LS;
    __shared__ __attribute__((aligned(16))) T tiles[4 * kTile + G::kTail];
    __shared__ __attribute__((aligned(16))) float off[32 * NW];
    __shared__ __attribute__((aligned(16))) float deltas[32 * NW];
    T *ks = tiles, *vs = tiles + kTile, *qs = tiles + 2 * kTile, *dos = tiles + 3 * kTile;
    const auto& a = p.a;
    const int64_t unit = work_index(blockIdx.x, gridDim.x), b = unit / a.kv_heads, hk = unit % a.kv_heads;
    const int lane = threadIdx.x & 63, half = lane >> 5, wave = threadIdx.x >> 6, own = wave * 32 + (lane & 31), mine = row_in<ROWS / 16>(wave, lane);
    const int length = length_of(a, b), rows = (int)p.rows, nq = (int)a.nq;

    const T* kv = reinterpret_cast<const T*>(a.kv) + b * a.kv_bg + hk * a.kv_head;
    const T* q = reinterpret_cast<const T*>(a.q) + b * a.q_bg + hk * p.group * a.q_head;
    const T* dout = reinterpret_cast<const T*>(a.dout) + b * a.do_bg + hk * p.group * a.do_head;
    Stage<DT, DK, W, 64 * NW, ROWS> keys, queries;
    keys.place(a.d, a.kv_row, a.kv_row);
    keys.load(kv, kv + a.kv_half, length);
    queries.place(a.d, a.q_row, a.do_row);
    if (p.group == 1) queries.load(q, dout, rows);
    else queries.load_each(rows, [&](int r, const T*& x, const T*& y) {
        const int h = r / nq, i = r - h * nq;
        x = q + h * a.q_head + i * a.q_row;
        y = dout + h * a.do_head + i * a.do_row;
    });
    const bool there = own < rows;
    typename E::Frag x[G::KS], y[G::KS];
    const float lse2 = there ? a.lse[unit * p.rows + own] * kLog2e : 0.f;
    keys.store(ks, vs);
    queries.store(qs, dos);
    __syncthreads();
    f32x16 dq[G::MS] = {};
    Scale qscale;
    float delta = 0.f;
#pragma unroll
    for (int k = 0; k < G::KS; ++k) {
        x[k] = direct<DT, DK>(qs, mine, k, half);
        y[k] = direct<DT, DK>(dos, mine, k, half);
    }
    if (length > 0) dq_whole<DT, DK, NW, ROWS / 16>(ks, vs, length, x, y, dq, qscale, p.c, lse2, delta, lane);
    if (half == 0) {
        off[own] = there ? E::kBias - lse2 : 0.f;
        deltas[own] = there ? -delta : 0.f;
    }
    __syncthreads();
    // from here on a wavefront's 32 rows of ks and vs are its own
#pragma unroll
    for (int k = 0; k < G::KS; ++k) {
        x[k] = direct<DT, DK>(ks, mine, k, half);
        y[k] = direct<DT, DK>(vs, mine, k, half);
    }
    T *lk = ks + wave * 32 * G::LS, *lv = vs + wave * 32 * G::LS;
    T* to_q = reinterpret_cast<T*>(a.dq) + b * a.nq * a.heads * a.d;
    store_rows<DT, DK, W, G::LS>(lk, dq, a.scale * (E::kScaled ? qscale.inverse() : 1.f), a.d, lane, rows - wave * 32, [&](int i) {
        const Row to = row_of(p, hk, wave * 32 + i);
        return to_q + (to.query * a.heads + to.head) * a.d;
    });
    f32x16 dk[G::MS] = {}, dv[G::MS] = {};
    Scale scale;
    if (length > 0 && rows > 0) dkv_step<DT, DK, NW, ROWS / 16>(qs, dos, off, deltas, rows, x, y, dk, dv, scale, p.c, lane);
    if (own >= length) {
#pragma unroll
        for (int j = 0; j < G::MS; ++j) dk[j] = dv[j] = f32x16{};
    }
    T* to_k = reinterpret_cast<T*>(a.dkv) + ((b * a.nk + wave * 32) * 2 * a.kv_heads + hk) * a.d;
    const int left = (int)a.nk - wave * 32;
    store_rows<DT, DK, W, G::LS>(lk, dk, a.scale * kUnbias<DT> * (E::kScaled ? scale.inverse() : 1.f), a.d, lane, left,
                                 [&](int i) { return to_k + (int64_t)i * 2 * a.kv_heads * a.d; });
    store_rows<DT, DK, W, G::LS>(lv, dv, kUnbias<DT>, a.d, lane, left, [&](int i) { return to_k + ((int64_t)i * 2 + 1) * a.kv_heads * a.d; });
}

// ---------------------------------------------------------------- launches
template <int DT, int DK, int W, int NW>
void launch_one(Kind kind, const Args& p, dim3 grid, hipStream_t stream) {
    const dim3 threads(64 * NW);
    if (kind == kForward) hipLaunchKernelGGL((forward_kernel<DT, DK, W, NW>), grid, threads, 0, stream, p);
    else if (kind == kDq) hipLaunchKernelGGL((dq_kernel<DT, DK, W, NW>), grid, threads, 0, stream, p);
    else if (kind == kDkv && p.rows <= 32) hipLaunchKernelGGL((dkv_kernel<DT, DK, W, NW, 32>), grid, threads, 0, stream, p);
    else if (kind == kDkv) hipLaunchKernelGGL((dkv_kernel<DT, DK, W, NW, kTileOf<DT, NW>>), grid, threads, 0, stream, p);
    else if constexpr (few_fits(DT == NORI_F32, DK, NW)) {
        if (kind == kFewForward) hipLaunchKernelGGL((forward_few_kernel<DT, DK, W, NW>), grid, threads, 0, stream, p);
        else if (NW == 2 && p.rows <= 48 && p.a.nk <= 48)
            hipLaunchKernelGGL((backward_few_kernel<DT, DK, W, NW, NW == 2 ? 48 : 32>), grid, threads, 0, stream, p);
        else hipLaunchKernelGGL((backward_few_kernel<DT, DK, W, NW, 32 * NW>), grid, threads, 0, stream, p);
    }
}

template <int DT, int DK, int W>
void launch_waves(Kind kind, const Args& p, dim3 grid, hipStream_t stream) {
    if constexpr (DK <= kFewWidth) {
        if (p.waves == 1) return launch_one<DT, DK, W, 1>(kind, p, grid, stream);
        if (p.waves == 2) return launch_one<DT, DK, W, 2>(kind, p, grid, stream);
    }
    launch_one<DT, DK, W, 4>(kind, p, grid, stream);
}

template <int DT, int W>
int launch_width(Kind kind, const Args& p, int64_t blocks, hipStream_t stream) {
    const int d = p.a.d;
    const dim3 grid((unsigned)blocks);
    if (d <= 32) launch_waves<DT, 32, W>(kind, p, grid, stream);
    else if (d <= 48) launch_waves<DT, 48, W>(kind, p, grid, stream);
    else if (d <= 64) launch_waves<DT, 64, W>(kind, p, grid, stream);
    else if (d <= 96) launch_waves<DT, 96, W>(kind, p, grid, stream);
    else launch_waves<DT, 128, W>(kind, p, grid, stream);
    return launch_status("attention_train");
}

}  // namespace attn_train
}  // namespace nori
