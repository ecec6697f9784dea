// Attention with gradients (gfx950): what the kernels and the host side share.
//
// A unit is one (batch entry, key head): the R = group * nq query rows of the `group` heads that share the key head,
// row r being query r % nq of the unit's head r / nq, over the entry's keys, `length` of its nk. With c = scale * log2(e)
// and L = log2 of the sum of 2^(c s):
//     s = q k^T,  p = 2^(c s - L),  out = p v
//     dv = p^T dout,  ds = p (dout v^T - delta),  delta = rowsum(dout * out),  dq = scale ds k,  dk = scale ds^T q
// Three kernels walk one side of s in tiles through LDS while the other side's operands stay in registers, 32 rows or
// keys a wavefront, and recompute p from the statistics that the forward pass kept:
//     forward, dq:  query rows stay, keys and values pass       dk and dv:  keys and values stay, query rows pass
// so every sum has one owner and an order of its own: no atomics.
//
// Layout. The side that stays gives the columns of every product's result (lane % 32), so its statistics, its rescaling
// and its scales are one value a lane. Its result of one product is the next one's right operand as it lies: the matrix
// instruction leaves rows 8 (i / 4) + 4 h + i % 4 in register i of half-wave h, and the contraction over them takes the
// left operand's rows in that same order (transposed reads of four rows by 16 columns).
#pragma once

#include "nori_common.h"

namespace nori {
namespace attn_train {

constexpr int kFewWidth = 64;  // head widths to which workgroups of one and two wavefronts are built
// Whether both sides of a unit of 32 `waves` rows and keys fit a workgroup's LDS.
constexpr bool few_fits(bool f32, int d, int waves) { return waves <= 2 && d <= kFewWidth && (!f32 || waves == 1 || d <= 32); }
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct Args {
    nori_attention_train_args a;
    int group;            // query heads a key head
    int64_t rows;         // group * nq
    int waves;            // of a workgroup, 32 rows or keys that stay each
    int64_t tiles;        // of the side that stays, a unit
    int64_t splits;       // parts of the side that passes
    int64_t per_split;    // its rows a part, whole tiles
    float* part;          // partial results where splits > 1
    float* part_lse;
    float* delta;
    float c;              // scale * log2(e)
    bool wide;            // 16-byte chunks of the 16-bit types
};

// Keys of batch entry b.
__device__ __forceinline__ int length_of(const nori_attention_train_args& a, int64_t b) {
    if (!a.lengths) return (int)a.nk;
    const int64_t i = b / a.length_group;
    int64_t n = a.lengths_i64 ? reinterpret_cast<const int64_t*>(a.lengths)[i] : reinterpret_cast<const int32_t*>(a.lengths)[i];
    n = n < 0 ? 0 : n;
    return (int)(n < a.nk ? n : a.nk);
}

// Workgroups are dealt to the 8 XCDs in turn: neighbours in the work's order, which share keys or rows, go to one XCD
// and its L2.
__device__ __forceinline__ int64_t work_index(int64_t i, int64_t n) {
    const int64_t whole = n & ~(int64_t)7;
    return i < whole ? (i & 7) * (whole >> 3) + (i >> 3) : i;
}

// What a launch does; kFewForward, kFew: the forward and the whole backward pass of units of few rows and keys. Launches of the
// typed translation units, in chunks of 16 bytes or (narrow) of 4 elements.
enum Kind { kForward, kDq, kDkv, kFewForward, kFew };
int launch_f16(Kind kind, const Args& p, int64_t blocks, hipStream_t stream);
int launch_f16_narrow(Kind kind, const Args& p, int64_t blocks, hipStream_t stream);
int launch_bf16(Kind kind, const Args& p, int64_t blocks, hipStream_t stream);
int launch_bf16_narrow(Kind kind, const Args& p, int64_t blocks, hipStream_t stream);
int launch_f32(Kind kind, const Args& p, int64_t blocks, hipStream_t stream);

}  // namespace attn_train
}  // namespace nori
