// Device code that the forward and the backward pass of the biased attention share: f16 / bf16
// fragments, a row of the bias table in LDS, and the scores of a 64-key block.
#pragma once

#include "attn_bias.h"
#include "attn_tile.h"

namespace jh {

// Division by a number that the host knows, in five operations (the compiler's takes some 30, and a
// block does several before its first load): m = 2^32 / d rounded down, so the product's high word is
// the quotient or one less.
struct Div {
    uint32_t d, m;
    Div(uint32_t n = 1) : d(n), m(n > 1 ? (uint32_t)((uint64_t(1) << 32) / n) : 0xffffffffu) {}
};
struct Quotient {
    int q, r;
};
__device__ __forceinline__ Quotient divide(int n, Div by) {
    uint32_t q = __umulhi((uint32_t)n, by.m), r = (uint32_t)n - q * by.d;
    if (r >= by.d) q++, r -= by.d;
    return {(int)q, (int)r};
}

// What the kernels take: the attention in the units they work in. Scores run in the exp2 domain:
// without a cap the MFMA accumulates q . k + (bias / scale), and a weight is exp2 of that times
// `mul` = scale log2(e) less the row's log-sum; with one, a score is
//   cap log2(e) tanh(x) + bias log2(e) = off - 2 off / (exp2(q . k pre) + 1) + bias unit
// with x = scale q . k / cap, pre = 2 log2(e) scale / cap, off = cap log2(e) and unit = log2(e) (`mul` is
// 1). Where |x| <= 1/2 the tanh is x times a polynomial of x^2 instead (poly, in units of q . k and with off
// taken in; |q . k| <= small): exact to 2^-24 of itself, where the other form is to 2^-23 of 1, which `off`
// makes some 2^-17 of a score.
struct BiasParams {
    const f16 *q, *k, *v;
    int64_t q_stride, kv_stride;
    f16* o;
    int64_t o_stride;
    int nq, nk, heads, kv_heads, each, q_first;
    Div by_each, by_tiles, by_chunks;  // (by_tiles: the launch's tiles of a head)
    float scale, mul, unit, off, pre;
    float poly[5], small, per_off;  // (per_off: 1 / off)
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

// Least values without LDS (a shuffle's round trip is some 100 clocks, and a block takes several such
// results before its first product): of each 16 lanes by DPP, as group_sum, and of the wave from
// those by the lane swaps.
template <int CTRL>
__device__ __forceinline__ int dpp_int(int v) {
    return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xF, 0xF, true);
}
__device__ __forceinline__ int row_min(int v) {
    v = min(v, dpp_int<0xB1>(v)), v = min(v, dpp_int<0x4E>(v));
    v = min(v, dpp_int<0x141>(v));
    return min(v, dpp_int<0x140>(v));
}
__device__ __forceinline__ int rows_min(int v) {
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = min((int)a[0], (int)a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return __builtin_amdgcn_readfirstlane(min((int)b[0], (int)b[1]));
}
// The most of 16 lanes' values, none negative, to each of them.
__device__ __forceinline__ float row_max(float v) {
    v = fmaxf(v, dpp_move<0xB1>(v)), v = fmaxf(v, dpp_move<0x4E>(v));
    v = fmaxf(v, dpp_move<0x141>(v));
    return fmaxf(v, dpp_move<0x140>(v));
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
    if (p.window > 0) {  // (pos + window may pass 2^31)
        const int pos = p.q_first + i;
        lo = max(lo, pos - p.window);
        hi = (int)min((uint32_t)max(hi, 0), (uint32_t)pos + (uint32_t)p.window + 1);
    }
    return hi > lo ? KeyRange{lo, hi} : KeyRange{0, 0};
}

// The keys of a block's rows, a lane each (`real`: it is a row): those that any of the block's or of wave
// w's 16 sees lie in [k0, k1) or [lo, hi); every real row of the wave sees [flo, fhi), of the block
// [all_flo, all_fhi).
struct KeyBounds {
    int k0, k1, lo, hi, flo, fhi, all_flo, all_fhi;
};
__device__ __forceinline__ KeyBounds key_bounds(KeyRange r, bool real, int w) {
    const int a = row_min(r.hi > r.lo ? r.lo : 0x7fffffff), b = row_min(~r.hi);
    const int c = row_min(~(real ? r.lo : 0)), d = row_min(real ? r.hi : 0x7fffffff);
    return {rows_min(a), ~rows_min(b), __builtin_amdgcn_readlane(a, 16 * w), ~__builtin_amdgcn_readlane(b, 16 * w),
            ~__builtin_amdgcn_readlane(c, 16 * w), __builtin_amdgcn_readlane(d, 16 * w), ~rows_min(c), rows_min(d)};
}

// A bias in the scores' units. A finite one stays finite: where every key
// of a row has the lowest bias of the type, their weights are equal, as in the formula.
__device__ __forceinline__ float bias_value(const BiasParams& p, float b) {
    const float v = b * p.unit;
    return (fabsf(b) <= 3.4028234e38f ? fminf(fmaxf(v, -3.4028234e38f), 3.4028234e38f) : v);
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

// N x 4 capped scores in place from q . k, base in them; slope: the tanh's slope times `by`, into base.
// Whether every one of the wave's is small is asked first: those of a model usually are, and the
// polynomial takes 7 operations where the other takes 11 (an exponential and a reciprocal at four each).
template <int N, bool SLOPE>
__device__ __forceinline__ void cap_scores(const BiasParams& p, floatx4 (&sc)[N], floatx4 (&base)[N], float by) {
    float most = 0.0f;
#pragma unroll
    for (int t = 0; t < N; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) most = fmaxf(most, fabsf(sc[t][e]));
    if (__builtin_amdgcn_ballot_w64(!(most <= p.small)) == 0) {  // (NaN: the other form keeps it)
#pragma unroll
        for (int t = 0; t < N; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float z = sc[t][e] * sc[t][e];
                const float v = sc[t][e] * fmaf(z, fmaf(z, fmaf(z, fmaf(z, p.poly[4], p.poly[3]), p.poly[2]), p.poly[1]), p.poly[0]);
                sc[t][e] = v + base[t][e];
                if (SLOPE) {
                    const float y = v * p.per_off;
                    base[t][e] = by * fmaf(-y, y, 1.0f);
                }
            }
    } else {
        // (opaque, or the compiler computes this side ahead of the branch every time)
#pragma unroll
        for (int t = 0; t < N; t++) asm volatile("" : "+v"(sc[t]));
#pragma unroll
        for (int t = 0; t < N; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float r = __builtin_amdgcn_rcpf(fast_exp2(sc[t][e] * p.pre) + 1.0f);
                sc[t][e] = fmaf(-2.0f * p.off, r, base[t][e] + p.off);
                if (SLOPE) base[t][e] = (4.0f * by) * fmaf(-r, r, r);
            }
    }
}

// The biases of 16 N keys from kb on for a lane's query (S^T: keys kb + 16 t + 4 g + e): tab, the lane's
// distance 0; left, right: the table's ends; wq0, wql: the wave's first and last query.
template <int BIAS, int N>
__device__ __forceinline__ void block_bias(const BiasParams& p, const float* tab, float left, float right, float slope,
                                           int kb, int g, int qpos, int wq0, int wql, floatx4 (&base)[N]) {
    if (BIAS == BIAS_TABLE) {
        if (kb - wql >= p.reach || kb + 16 * N - 1 - wq0 <= -p.reach) {
            const float b0 = kb > wq0 ? right : left;
#pragma unroll
            for (int t = 0; t < N; t++) base[t] = floatx4{b0, b0, b0, b0};
        } else {
            const float* at = tab + (kb + 4 * g - qpos);
#pragma unroll
            for (int t = 0; t < N; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) base[t][e] = at[16 * t + e];
        }
    } else if (BIAS == BIAS_SLOPES) {
        const float x = (float)(kb + 4 * g - qpos);
        // (keys all after or all before the wave's queries: a line, one operation a score in place of two)
        if (N == 4 && (kb >= wql || kb + 16 * N - 1 <= wq0)) {
            const float s = kb >= wql ? -slope : slope, b0 = s * x;
#pragma unroll
            for (int t = 0; t < N; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) base[t][e] = fmaf(s, (float)(16 * t + e), b0);
            return;
        }
#pragma unroll
        for (int t = 0; t < N; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) base[t][e] = -slope * fabsf(x + (float)(16 * t + e));
    } else {
#pragma unroll
        for (int t = 0; t < N; t++) base[t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    }
}

// Before a step's reads: all of this wave's copies into LDS but the last N have landed, then every
// wave's, and every wave's reads of the last step are done. (__syncthreads waits for all copies, or for
// none: its fence does not count them, only the wave's own reads of them do.)
template <int N>
__device__ __forceinline__ void stage_barrier() {
    static_assert(N >= 0 && N < 16, "vmcnt field");
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(N | 0x0070);  // vmcnt N, lgkmcnt 0
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// The pairs of a product's 32 rows (16 (i / 4) + 4 (lane / 16) + i % 4, as pack8 lays them) that exist: 16 bits
// each, all set where seen(row) holds.
typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));
template <typename F>
__device__ __forceinline__ uintx4 seen_pairs(F&& seen) {
    const int g = (threadIdx.x & 63) >> 4;
    uintx4 m;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int c = 16 * (i >> 1) + 4 * g + 2 * (i & 1);
        m[i] = (seen(c) ? 0xffffu : 0u) | (seen(c + 1) ? 0xffff0000u : 0u);
    }
    return m;
}
// acc += a . w where a masked pair's value may be infinite or NaN (times a weight of 0 it would make the sum
// NaN): the finite values' product, and a second one that counts each sum's infinities of either sign, NaN
// as one of both. ANY: an infinity makes the sum NaN (its own weight is a difference that it made NaN). Only a
// block whose sums were not finite comes here.
template <bool BF, bool ANY>
__device__ __forceinline__ floatx4 careful_mma(half8 a, half8 w, uintx4 pairs, floatx4 acc) {
    constexpr uint32_t E = BF ? 0x7f80 : 0x7c00, ONE = BF ? 0x3f80 : 0x3c00, C64 = BF ? 0x4280 : 0x5400, C65 = BF ? 0x4282 : 0x5410;
    const uintx4 av = __builtin_bit_cast(uintx4, a), wv = __builtin_bit_cast(uintx4, w);
    uintx4 value, flag;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t v = 0, f = 0;
#pragma unroll
        for (int y = 0; y < 32; y += 16) {
            const uint32_t u = (av[i] >> y) & 0xffff;
            const uint32_t sort = ANY || (u & 0x7fff) > E ? C65 : u >> 15 ? C64 : ONE;
            v |= ((u & E) == E ? 0 : u) << y;
            f |= ((u & E) == E ? sort : 0) << y;
        }
        value[i] = v, flag[i] = f;
    }
    acc = mma<BF>(__builtin_bit_cast(half8, value), __builtin_bit_cast(half8, wv & pairs), acc);
    const floatx4 n = mma<BF>(__builtin_bit_cast(half8, flag), __builtin_bit_cast(half8, pairs & (ONE * 0x10001u)),
                              floatx4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
    for (int e = 0; e < 4; e++) {  // (32 rows at most of each sort: exact)
        const float neg = floorf(n[e] * 0.015625f);
        acc[e] += n[e] > 64.0f * neg ? INFINITY : 0.0f;
        acc[e] += neg > 0.0f ? -INFINITY : 0.0f;
    }
    __builtin_amdgcn_sched_barrier(0);  // (one product after the other: registers)
    return acc;
}
__device__ __forceinline__ bool finite4(floatx4 v) {
    return fabsf(v[0]) < INFINITY && fabsf(v[1]) < INFINITY && fabsf(v[2]) < INFINITY && fabsf(v[3]) < INFINITY;
}

}  // namespace jh
