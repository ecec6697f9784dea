// Attention with gradients: checks, launch plans and the kernels that join split axes (attention_train.h has the
// mathematics, attention_train_kernel.h the kernels).
#include <math.h>

#include <algorithm>

#include "attention_train.h"

using namespace nori;
using namespace nori::attn_train;

namespace {

constexpr int64_t kTileRows = 64;      // a multiple of every type's tile
constexpr int64_t kLeastRows = 256;    // of a part: below it, joining costs more than the idle units

// Element col of row `at` of a result: out or dq rows in a unit's order, or dk's and dv's (key, then K or V).
template <bool KV>
__device__ __forceinline__ int64_t place_of(const Args& p, int64_t at, int64_t col) {
    const auto& a = p.a;
    if constexpr (KV) {
        const int64_t unit = at / (2 * a.nk), row = at % (2 * a.nk);
        return ((unit / a.kv_heads * 2 * a.nk + row) * a.kv_heads + unit % a.kv_heads) * a.d + col;
    } else {
        const int64_t unit = at / p.rows, r = at % p.rows;
        const int64_t head = unit % a.kv_heads * p.group + r / a.nq;
        return ((unit / a.kv_heads * a.nq + r % a.nq) * a.heads + head) * a.d + col;
    }
}

// A row of a result from its parts by one workgroup: the parts are dealt to groups of d / 4 threads, whose sums are added in
// order. Forward parts are normalised over their own keys and weighed by their shares of the row's sum.
template <int DT, Kind KIND>
__global__ __launch_bounds__(256) void join_kernel(const Args p) {
    __shared__ float sums[256 * 4], totals[256], tops[4];
    const auto& a = p.a;
    const int64_t n = a.bg * a.kv_heads * (KIND == kDkv ? 2 * a.nk : p.rows);
    const int quads = a.d / 4, groups = 256 / quads, group = threadIdx.x / quads, col = 4 * (threadIdx.x % quads);
    for (int64_t at = blockIdx.x; at < n; at += gridDim.x) {
        float base = 0.f;
        if constexpr (KIND == kForward) {
            float top = -INFINITY;
            for (int64_t s = threadIdx.x; s < p.splits; s += 256) top = fmaxf(top, p.part_lse[s * n + at]);
            for (int i = 32; i > 0; i /= 2) top = fmaxf(top, __shfl_xor(top, i));
            if (threadIdx.x % 64 == 0) tops[threadIdx.x / 64] = top;
            __syncthreads();
            top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
            base = top == -INFINITY ? 0.f : top;
        }
        f32x4 sum = {};
        float total = 0.f;
        if (group < groups) {
#pragma unroll 4
            for (int64_t s = group; s < p.splits; s += groups) {
                const f32x4 x = *reinterpret_cast<const f32x4*>(p.part + (s * n + at) * a.d + col);
                if constexpr (KIND == kForward) {
                    const float l = p.part_lse[s * n + at];
                    const float w = __builtin_amdgcn_exp2f(l - base);
                    if (l != -INFINITY) {  // (no keys, or none that counts, in this part)
                        total += w;
                        sum += w * x;
                    }
                } else {
                    sum += x;
                }
            }
        }
        *reinterpret_cast<f32x4*>(&sums[4 * threadIdx.x]) = sum;
        totals[threadIdx.x] = total;
        __syncthreads();
        if (group == 0) {
            for (int g = 1; g < groups && g < p.splits; ++g) {
                sum += *reinterpret_cast<const f32x4*>(&sums[4 * (g * quads + threadIdx.x)]);
                total += totals[g * quads];
            }
            if constexpr (KIND == kForward) {
                if (total != 0.f) sum *= 1.f / total;
                else if (length_of(a, at / p.rows / a.kv_heads) > 0) sum = f32x4{} + NAN;  // every logit at -inf
                if (col == 0 && a.lse) a.lse[at] = (base + __builtin_amdgcn_logf(total)) * kLn2;
            }
            void* out = KIND == kForward ? a.out : (KIND == kDq ? a.dq : a.dkv);
            const int64_t to = place_of<KIND == kDkv>(p, at, col);
            for (int j = 0; j < 4; ++j) store_elem<DT>(out, to + j, sum[j]);
        }
        __syncthreads();
    }
}

int64_t part_rows(const Args& p, Kind kind) { return p.a.bg * p.a.kv_heads * (kind == kDkv ? 2 * p.a.nk : p.rows); }

// Tiles of the side that stays, and parts of the side that passes where the tiles alone leave compute units idle.
Args plan(const nori_attention_train_args& a, Kind kind) {
    Args p{};
    p.a = a;
    p.group = a.heads / a.kv_heads;
    p.rows = (int64_t)p.group * a.nq;
    p.c = a.scale * kLog2e;
    const int64_t stay = kind == kDkv ? a.nk : p.rows, pass = kind == kDkv ? p.rows : a.nk;
    p.waves = a.d > kFewWidth || stay > 64 ? 4 : (stay > 32 ? 2 : 1);
    p.tiles = (stay + 32 * p.waves - 1) / (32 * p.waves);
    const int64_t blocks = a.bg * a.kv_heads * p.tiles, want = 8 / p.waves * device_cus();
    int64_t splits = blocks > 0 && blocks < want ? (want + blocks - 1) / blocks : 1;
    splits = std::max<int64_t>(1, std::min(splits, pass / kLeastRows));
    p.per_split = std::max<int64_t>(kTileRows, ((pass + splits - 1) / splits + kTileRows - 1) / kTileRows * kTileRows);
    p.splits = std::max<int64_t>(1, (pass + p.per_split - 1) / p.per_split);
    return p;
}

// Wavefronts for a unit's rows and for its keys, where one workgroup takes it through a whole pass.
int few_waves(const nori_attention_train_args& a) { return (int)((std::max(a.nk, a.nq * (a.heads / a.kv_heads)) + 31) / 32); }
bool few(const nori_attention_train_args& a, bool backward) {
    return a.nk <= 64 && a.nq * (a.heads / a.kv_heads) <= 64 && few_fits(a.dtype == NORI_F32, a.d, few_waves(a)) && (!backward || (a.dq && a.dkv));
}

int64_t part_bytes(const Args& p, Kind kind) { return p.splits > 1 ? p.splits * part_rows(p, kind) * p.a.d * 4 : 0; }
int64_t aligned16(int64_t n) { return (n + 15) / 16 * 16; }

int launch_typed(Kind kind, const Args& p, hipStream_t stream) {
    const int64_t blocks = p.a.bg * p.a.kv_heads * p.tiles * p.splits;
    switch (p.a.dtype) {
        case NORI_F16: return p.wide ? launch_f16(kind, p, blocks, stream) : launch_f16_narrow(kind, p, blocks, stream);
        case NORI_BF16: return p.wide ? launch_bf16(kind, p, blocks, stream) : launch_bf16_narrow(kind, p, blocks, stream);
        default: return launch_f32(kind, p, blocks, stream);
    }
}

int launch_few(Kind kind, Args p, hipStream_t stream) {
    p.waves = std::max(1, few_waves(p.a));
    p.tiles = p.splits = 1;
    return launch_typed(kind, p, stream);
}

int join(Kind kind, const Args& p, hipStream_t stream) {
    const dim3 grid((unsigned)std::min<int64_t>(part_rows(p, kind), 32 * device_cus())), threads(256);
    NORI_DISPATCH_FLOAT(p.a.dtype, DT, {
        if (kind == kForward) hipLaunchKernelGGL((join_kernel<DT, kForward>), grid, threads, 0, stream, p);
        else if (kind == kDq) hipLaunchKernelGGL((join_kernel<DT, kDq>), grid, threads, 0, stream, p);
        else hipLaunchKernelGGL((join_kernel<DT, kDkv>), grid, threads, 0, stream, p);
    });
    return launch_status("attention_train join");
}

// A pointer and its strides, in elements: loads take n at once.
bool loads(const void* p, int size, std::initializer_list<int64_t> strides, int n = 4) {
    if (reinterpret_cast<uintptr_t>(p) % (n * size)) return false;
    return std::all_of(strides.begin(), strides.end(), [n](int64_t s) { return s % n == 0; });
}

// Whether everything that is read or written lies in 16-byte chunks of a 16-bit type.
bool wide(const nori_attention_train_args& a, bool backward) {
    return a.dtype != NORI_F32 && a.d % 8 == 0 && loads(a.q, 2, {a.q_bg, a.q_row, a.q_head}, 8) &&
           loads(a.kv, 2, {a.kv_bg, a.kv_row, a.kv_half, a.kv_head}, 8) && loads(a.out, 2, {}, 8) &&
           (!backward || (loads(a.dout, 2, {a.do_bg, a.do_row, a.do_head}, 8) && loads(a.dq, 2, {}, 8) && loads(a.dkv, 2, {}, 8)));
}

int check(const nori_attention_train_args* a, bool backward) {
    const char* what = backward ? "attention_train_backward" : "attention_train_forward";
    if (!a) return fail(NORI_ERR_INVALID, "%s: null arguments", what);
    if (a->dtype != NORI_F32 && a->dtype != NORI_F16 && a->dtype != NORI_BF16)
        return fail(NORI_ERR_UNSUPPORTED, "%s: unsupported dtype %s", what, dtype_name(a->dtype));
    if (a->bg < 0 || a->nq < 0 || a->nk < 0 || a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads)
        return fail(NORI_ERR_INVALID, "%s: %lld x %lld queries of %d heads over %lld keys of %d", what, (long long)a->bg, (long long)a->nq,
                    a->heads, (long long)a->nk, a->kv_heads);
    if (a->d < 4 || a->d > NORI_ATTENTION_TRAIN_WIDTH || a->d % 4)
        return fail(NORI_ERR_UNSUPPORTED, "%s: heads of %d; a multiple of 4 up to %d is taken", what, a->d, NORI_ATTENTION_TRAIN_WIDTH);
    constexpr int64_t most = 1LL << 30;
    if (a->nq > most || a->nk > most || a->nq * (a->heads / a->kv_heads) > most)
        return fail(NORI_ERR_UNSUPPORTED, "%s: up to 2^30 keys, and queries of heads that share one, are taken", what);
    if (a->bg > (1LL << 40) / ((int64_t)a->heads * std::max<int64_t>(1, std::max(a->nq, a->nk))))
        return fail(NORI_ERR_UNSUPPORTED, "%s: too many rows", what);
    const float c = a->scale * kLog2e;
    if (!(c - c == 0.f)) return fail(NORI_ERR_INVALID, "%s: the scale must be finite, times log2(e) too", what);
    if (a->lengths && (a->length_group < 1)) return fail(NORI_ERR_INVALID, "%s: lengths of %lld entries each", what, (long long)a->length_group);
    const int size = dtype_size(a->dtype);
    if (a->bg * a->nq > 0) {
        if (!a->q || !a->out || (backward && (!a->lse || !a->dout))) return fail(NORI_ERR_INVALID, "%s: null pointer", what);
        if (!loads(a->q, size, {a->q_bg, a->q_row, a->q_head}) || !loads(a->out, size, {}) ||
            (backward && (!loads(a->dout, size, {a->do_bg, a->do_row, a->do_head}) || !loads(a->dq, size, {}))))
            return fail(NORI_ERR_UNSUPPORTED, "%s: query rows not aligned to 4 elements", what);
    }
    if (a->bg * a->nk > 0) {
        if (!a->kv) return fail(NORI_ERR_INVALID, "%s: null pointer", what);
        if (!loads(a->kv, size, {a->kv_bg, a->kv_row, a->kv_half, a->kv_head}) || (backward && !loads(a->dkv, size, {})))
            return fail(NORI_ERR_UNSUPPORTED, "%s: key rows not aligned to 4 elements", what);
    }
    // a tile's rows are at 32-bit byte offsets from its first
    constexpr int64_t far = 1LL << 24;
    for (int64_t s : {a->q_row, a->kv_row, backward ? a->do_row : 0})
        if (s < 0 || s > far) return fail(NORI_ERR_UNSUPPORTED, "%s: a row stride of %lld; up to 2^24 is taken", what, (long long)s);
    const Kind kinds[3] = {kForward, kDq, kDkv};
    for (Kind k : kinds) {
        const Args p = plan(*a, k);
        if (!one_launch(a->bg * a->kv_heads * p.tiles * p.splits, 64 * p.waves))
            return fail(NORI_ERR_UNSUPPORTED, "%s: more workgroups than one launch has", what);
    }
    return NORI_OK;
}

int check_workspace(const nori_attention_train_args* a, bool backward) {
    const int64_t need = nori_attention_train_workspace_bytes(a, backward);
    if (need == 0) return NORI_OK;
    if (!a->workspace || a->workspace_bytes < need || reinterpret_cast<uintptr_t>(a->workspace) % 16)
        return fail(NORI_ERR_INVALID, "attention_train: a 16-byte aligned workspace of %lld bytes is needed", (long long)need);
    return NORI_OK;
}

}  // namespace

extern "C" int64_t nori_attention_train_workspace_bytes(const nori_attention_train_args* a, int32_t backward) {
    if (!a || a->heads < 1 || a->kv_heads < 1 || a->bg < 0 || a->nq < 0 || a->nk < 0) return 0;
    if (!backward) {
        const Args p = plan(*a, kForward);
        return p.splits > 1 ? aligned16(part_bytes(p, kForward)) + aligned16(p.splits * part_rows(p, kForward) * 4) : 0;
    }
    if (few(*a, true)) return 0;
    const Args q = plan(*a, kDq), kv = plan(*a, kDkv);
    return aligned16(part_rows(q, kDq) * 4) + std::max(a->dq ? part_bytes(q, kDq) : 0, a->dkv ? part_bytes(kv, kDkv) : 0);
}

extern "C" int nori_attention_train_forward(const nori_attention_train_args* a, void* stream_v) {
    clear_error();
    if (int rc = check(a, false)) return rc;
    if (a->bg * a->nq == 0) return NORI_OK;
    if (int rc = check_workspace(a, false)) return rc;
    hipStream_t stream = (hipStream_t)stream_v;
    Args p = plan(*a, kForward);
    p.wide = wide(*a, false);
    if (few(*a, false)) return launch_few(kFewForward, p, stream);
    p.part = reinterpret_cast<float*>(a->workspace);
    p.part_lse = reinterpret_cast<float*>(reinterpret_cast<char*>(a->workspace) + aligned16(part_bytes(p, kForward)));
    if (int rc = launch_typed(kForward, p, stream)) return rc;
    return p.splits > 1 ? join(kForward, p, stream) : NORI_OK;
}

extern "C" int nori_attention_train_backward(const nori_attention_train_args* a, void* stream_v) {
    clear_error();
    if (int rc = check(a, true)) return rc;
    if (a->bg == 0 || (!a->dq && !a->dkv)) return NORI_OK;
    if (int rc = check_workspace(a, true)) return rc;
    hipStream_t stream = (hipStream_t)stream_v;
    float* delta = reinterpret_cast<float*>(a->workspace);
    Args q = plan(*a, kDq);
    q.wide = wide(*a, true);
    if (few(*a, true)) return launch_few(kFew, q, stream);
    if (a->nq > 0) {
        if (!a->dq) q.splits = 1;  // the rows' sums alone
        q.delta = delta;
        q.part = reinterpret_cast<float*>(reinterpret_cast<char*>(a->workspace) + aligned16(part_rows(q, kDq) * 4));
        if (int rc = launch_typed(kDq, q, stream)) return rc;
        if (q.splits > 1)
            if (int rc = join(kDq, q, stream)) return rc;
    }
    if (!a->dkv || a->nk == 0) return NORI_OK;
    Args kv = plan(*a, kDkv);
    kv.wide = q.wide;
    kv.delta = delta;
    kv.part = reinterpret_cast<float*>(reinterpret_cast<char*>(a->workspace) + aligned16(part_rows(q, kDq) * 4));
    if (int rc = launch_typed(kDkv, kv, stream)) return rc;
    return kv.splits > 1 ? join(kDkv, kv, stream) : NORI_OK;
}
