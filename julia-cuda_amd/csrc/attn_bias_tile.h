// Device code that the forward and the backward pass of the biased attention share: f16 / bf16
// fragments, a row of the bias table in LDS, and the scores of a 64-key block.
#pragma once

#include "attn_bias.h"
#include "attn_tile.h"

namespace jh {

// What the kernels take: the attention in the units they work in. Scores run in the exp2 domain:
// without a cap the MFMA accumulates q . k + (bias / scale), and a weight is exp2 of that times
// `mul` = scale log2(e) less the row's log-sum; with one, a score is
//   cap log2(e) tanh(x) + bias log2(e) = (off + bias unit) - 2 off / (exp2(q . k pre) + 1)
// with x = scale q . k / cap, pre = 2 log2(e) scale / cap, off = cap log2(e) and unit = log2(e) (`mul` is 1).
struct BiasParams {
    const f16 *q, *k, *v;
    int64_t q_stride, kv_stride;
    f16* o;
    int64_t o_stride;
    int nq, nk, heads, kv_heads, each, q_first;
    float scale, mul, unit, off, pre;
    const float* table;
    const int32_t* bucket;
    int buckets, reach, row;  // row: floats of a head's padded distances in LDS
    const float* slopes;
    int window;
    const int32_t* span;
    float* lse;
    int chunks;
    float* ws;
    uint32_t* counters;
};

BiasParams bias_params(const AttnBias& a);

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float floatx2 __attribute__((ext_vector_type(2)));

// 16x16x32 MFMA of two fragments of f16 or bf16 bits.
template <bool BF>
__device__ __forceinline__ floatx4 mma(half8 a, half8 b, floatx4 c) {
    if (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    return mfma16(a, b, c);
}

// Two values rounded to nearest even, in one instruction.
template <bool BF>
__device__ __forceinline__ half2 pack2(float a, float b) {
    const floatx2 v = {a, b};
    if (BF) return __builtin_bit_cast(half2, __builtin_convertvector(v, bf16x2));
    return __builtin_convertvector(v, half2);
}
template <bool BF>
__device__ __forceinline__ half8 pack8(floatx4 lo, floatx4 hi) {
    const half2 a = pack2<BF>(lo[0], lo[1]), b = pack2<BF>(lo[2], lo[3]);
    const half2 c = pack2<BF>(hi[0], hi[1]), d = pack2<BF>(hi[2], hi[3]);
    return half8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
template <bool BF>
__device__ __forceinline__ half4 pack4(floatx4 v) {
    const half2 a = pack2<BF>(v[0], v[1]), b = pack2<BF>(v[2], v[3]);
    return half4{a[0], a[1], b[0], b[1]};
}
template <bool BF>
__device__ __forceinline__ float widen(f16 v) {
    if (BF) return __uint_as_float((uint32_t)__builtin_bit_cast(uint16_t, v) << 16);
    return (float)v;
}

__device__ __forceinline__ int wave_min(int v) {
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) v = min(v, __shfl_xor(v, s));
    return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int wave_max(int v) {
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) v = max(v, __shfl_xor(v, s));
    return __builtin_amdgcn_readfirstlane(v);
}

// The keys that query i sees, [lo, hi) within [0, nk); none: lo = hi = 0.
struct KeyRange {
    int lo, hi;
};
__device__ __forceinline__ KeyRange key_range(const BiasParams& p, int i) {
    int lo = 0, hi = p.nk;
    if (p.span) {
        const int2 s = *(const int2*)(p.span + 2 * (size_t)i);
        lo = max(s.x, 0), hi = min(s.y, p.nk);
    }
    if (p.window > 0) {  // (positions and windows are below 2^30)
        const int pos = p.q_first + i;
        lo = max(lo, pos - p.window), hi = min(hi, pos + p.window + 1);
    }
    return hi > lo ? KeyRange{lo, hi} : KeyRange{0, 0};
}

// A bias in the scores' units, plus the cap's offset. A finite one stays finite: where every key
// of a row has the lowest bias of the type, their weights are equal, as in the formula.
__device__ __forceinline__ float bias_value(const BiasParams& p, float b) {
    const float v = b * p.unit;
    return (fabsf(b) <= 3.4028234e38f ? fminf(fmaxf(v, -3.4028234e38f), 3.4028234e38f) : v) + p.off;
}

// The padded distances of `n` heads from `head` on into LDS: tab[x row + reach + BIAS_PAD + t] is
// the bias of head + x at distance t (key - query).
__device__ __forceinline__ void load_bias(const BiasParams& p, int head, int n, float* tab, int threads) {
    for (int i = threadIdx.x; i < p.row; i += threads) {
        const int t = min(max(i - BIAS_PAD, 0), 2 * p.reach);
        const int b = min(max(p.bucket[t], 0), p.buckets - 1);
        for (int x = 0; x < n; x++) tab[x * p.row + i] = bias_value(p, p.table[(size_t)b * p.heads + head + x]);
    }
}

// A row of f16 / bf16 (64 values) times another, for the paths that go key by key.
template <bool BF>
__device__ __forceinline__ float dot64(const f16* a, const f16* b) {
    float s = 0.0f;
    for (int c = 0; c < 64; c += 8) {
        const half8 x = *(const half8*)(a + c), y = *(const half8*)(b + c);
#pragma unroll
        for (int e = 0; e < 8; e++) s = fmaf(widen<BF>(x[e]), widen<BF>(y[e]), s);
    }
    return s;
}

// A score's weight in the exp2 domain (before the row's log-sum is taken off) from q . k, the
// tanh's slope in `slope` (1 without a cap). base: the bias in the scores' units plus the offset.
template <bool CAP>
__device__ __forceinline__ float score_of(const BiasParams& p, float qk, float base, float& slope) {
    if (CAP) {
        const float r = __builtin_amdgcn_rcpf(fast_exp2(qk * p.pre) + 1.0f);
        slope = 4.0f * fmaf(-r, r, r);
        return fmaf(-2.0f * p.off, r, base);
    }
    slope = 1.0f;
    return (qk + base) * p.mul;
}

// The bias of head h (tab: its row in LDS) at distance t, in the same units.
template <int BIAS>
__device__ __forceinline__ float bias_at(const BiasParams& p, const float* tab, float slope, int t) {
    if (BIAS == BIAS_TABLE) return tab[min(max(t, -p.reach), p.reach) + p.reach + BIAS_PAD];
    if (BIAS == BIAS_SLOPES) return fmaf(-slope, fabsf((float)t), p.off);
    return p.off;
}

}  // namespace jh
