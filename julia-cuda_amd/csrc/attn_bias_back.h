// The biased attention's backward pass (attn_bias.h). With P = exp(s - lse) and D_i = dO_i . o_i:
//   dV = P^T dO,  dS = P (dO V^T - D),  dbias[t] = the sum of dS over j - pos_i = t,
//   dA = scale dS (the tanh's slope),  dQ = dA K,  dK = dA^T Q.
//
// Two launches, each over the scores again (seven products in place of five), so that no block adds to
// another's results and the gradients are the same bits at every call:
// - dq_kernel: 16 NW queries of a head over their keys: dQ, the rows' constants for the other (-lse,
//   -D, their keys) and the block's sums of dS by distance.
// - dkv_kernel: 16 NG NW keys of a key head over the queries that see them: dK and dV; its first blocks
//   sum the distances' shares over the first launch's, and by bucket.
//
// - Both keep the scores where the next product wants them: a lane's column is its query (dQ) or its
//   key (dK, dV), and the transposed operand comes from LDS by the transposing read.
// - dO V^T starts from -D in the accumulators, the scores from the bias.
// - f16: dS is scaled by a power of two from |dO| (a query's own for dQ, the largest of the queries
//   that see a block for dK and dV), so that |dO| becomes 2^3 to 2^4 and dS keeps the type's
//   precision whatever the loss's scale: a weight of 2^-14 times a |v| of 1 is still a normal value. It
//   overflows where a weight near 1 meets |v| > 2^11; such a block is computed again at 2^-11 of it.
// - KS key groups (or groups of queries) of NW waves share a block, each with its own stages, where
//   the grid is small; their sums join in LDS in order.
// - The bias's gradient in 32 bits, before dS is rounded: a 64-key block past `reach` on one side adds
//   to one sum; else the 16 queries of a wave are summed along the diagonals with lane shifts (a
//   lane's four keys of a 16-key tile against its neighbours' queries) and added to rows of distances
//   in LDS that no other lane group adds to (64 documents in 18752 rows: dQ alone 61 us; with the sums
//   on masked additions 128, the groups joined by shifts and an MFMA with ones 110, so 98 to 104).
// - A block whose sums are not finite is computed again, its tiles with masked pairs pair by pair: a
//   masked infinity or NaN times a weight of 0 is NaN in the tiles' products. Twice the time at most.
//
// Both launches are bound by vector instructions and LDS reads between the products, at two (dK, dV) and
// three (dQ) waves a SIMD: 64 documents in 18752 rows take 207 us for 44 GFLOP and 231 MB.
#pragma once

#include <algorithm>
#include <stdexcept>
#include <string>

#include "attn_bias_tile.h"

namespace jh {

struct BiasBack {
    BiasParams p;
    const f16* dout;
    int64_t do_stride;
    f16 *dq, *dk, *dv;
    int64_t dq_stride, dkv_stride;
    float* dtable;
    // The workspace: per head and 64 (padded) rows -lse log2(e) (-inf: a row without keys), -D and the
    // rows' keys (first, number), a kilobyte together (`info`); per 16 NW rows the keys (least first, most past last, most first, least
    // past last), per 16 rows a head's largest |dO|^2, per (head, block) the distances' sums.
    float* info;
    int4* bounds;
    float *max_do, *part;
    int nqp, tiles, dkv_blocks;  // tiles: a head's blocks of the first launch
    int per;                     // of them to 64 rows: 4, 2 or 1
};

constexpr int DQ_STAGE = 16384;           // K and V of 64 keys
// The distances' sums in LDS: a row (and a spare) for each of a wave's four lane groups, so that no two lanes
// share a sum (rows a multiple of 64 and 12 apart: with the groups' 4 keys, on different banks); a row a
// wave for eight waves of four stages.
__host__ __device__ constexpr int hist_groups(int nw) { return nw == 2 ? 1 : 4; }
__host__ __device__ constexpr int hist_pitch(int reach) { return (2 * reach + 2 - 12 + 63) / 64 * 64 + 12; }
__host__ __device__ constexpr int dq_lds(int reach, int nw, int ks) {  // beside the stages
    return 4 * (2 * (reach + BIAS_PAD) + 1 + nw * ks * hist_groups(nw) * hist_pitch(reach));
}
constexpr int DKV_STAGE = 16384 + 1024;   // Q, dO and `info` of 64 queries

// Row i of head h's -lse log2(e); its -D is 64 floats on, its keys at 128 + i % 64 more.
__device__ __forceinline__ float* row_info(const BiasBack& b, int h, int i) {
    return b.info + ((size_t)h * (b.nqp / 64) + (i >> 6)) * 256 + (i & 63);
}

// The power of two that takes the root of `sq` to between 2^3 and 2^4 (1 where it is 0 or not finite).
__device__ __forceinline__ float grad_scale(float sq) {
    if (!(sq > 0.0f && sq < INFINITY)) return 1.0f;
    int e;
    frexpf(sqrtf(sq), &e);  // < 2^e
    return ldexpf(1.0f, 4 - e);
}

// out[x stride] = the sum of term(x, i) over i < n, for x < m, by a block: THREADS / (m rounded up to a
// power of two) threads share an x, each taking every so-manyth i, and join in order. sm: THREADS floats.
template <int THREADS, typename F>
__device__ __forceinline__ void sum_groups(int m, int n, float* sm, float* out, int stride, F&& term) {
    int wide = 1;
    while (wide < m && wide < THREADS) wide *= 2;
    const int parts = THREADS / wide, y = threadIdx.x / wide;
    for (int x0 = 0; x0 < m; x0 += wide) {
        const int x = x0 + threadIdx.x % wide;
        float a = 0.0f;
        if (x < m)
#pragma unroll 8
            for (int i = y; i < n; i += parts) a += term(x, i);
        sm[threadIdx.x] = a;
        __syncthreads();
        if (y == 0 && x < m) {
            for (int z = 1; z < parts; z++) a += sm[z * wide + threadIdx.x];
            out[(size_t)x * stride] = a;
        }
        __syncthreads();
    }
}

// Sums along the diagonals of a 16 x 16 tile S^T (lane (r16, g): query r16, keys 4 g + e): lane (r16, g) adds
// what its group has at distance (the tile's first key less its first query) + 4 g - r16 to `here`, and
// at 16 more to `next`. Key e of lane r16 is on the diagonal of key 0 of the lane e to the left, or 16 on
// where that leaves the 16 lanes.
__device__ __forceinline__ void diagonal_sums(floatx4 s, float& here, float& next) {
    here += s[0];
    here += dpp_move<0x101>(s[1]);
    here += dpp_move<0x102>(s[2]);
    here += dpp_move<0x103>(s[3]);
    next += dpp_move<0x11F>(s[1]);
    next += dpp_move<0x11E>(s[2]);
    next += dpp_move<0x11D>(s[3]);
}

// ---- dQ of 16 NW queries of a head --------------------------------------------------------------
template <bool BF, int BIAS, bool CAP, int NW, int KS>
__global__ __launch_bounds__(64 * NW * KS) void attn_bias_dq_kernel(BiasBack b) {
    const BiasParams& p = b.p;
    // (stages: as in the forward pass, arrays of their own)
    __shared__ __attribute__((aligned(16))) char stage0[KS * DQ_STAGE], stage1[KS * DQ_STAGE];
    extern __shared__ __attribute__((aligned(16))) float tab0[];
    constexpr int QB = 16 * NW, LOADS = 16 / NW, HG = hist_groups(NW);
    const Quotient ht = divide(xcd_task(blockIdx.x, gridDim.x), p.by_tiles);
    const int h = ht.q, tile = ht.r, q0 = QB * tile, kvh = divide(h, p.by_each).q;
    const int tid = threadIdx.x, l = tid & 63, r16 = l & 15, g = l >> 4;
    const int wk = __builtin_amdgcn_readfirstlane(tid >> 6), w = wk % NW, kg = wk / NW;
    const int j4 = r16 >> 2, q4 = r16 & 3;
    __shared__ uint32_t s_bad;
    if (tid == 0) s_bad = 0;
    const int dists = 2 * p.reach + 1;
    float* const hist0 = tab0 + p.row;
    const int pitch = hist_pitch(p.reach);
    float* const hist = hist0 + (wk * HG + (HG == 4 ? g : 0)) * pitch;  // the lane's row of distances

    // The keys of the block's rows (lane l: row q0 + l), then the lane's own row.
    KeyRange tr{0, 0};
    const bool listed = l < QB && q0 + l < p.nq;
    if (listed) tr = key_range(p, q0 + l);
    const int row = q0 + 16 * w + r16, qi = min(row, p.nq - 1), qpos = p.q_first + row;
    const bool real = row < p.nq;
    half8 qf[2], gf[2], of[2];
    {
        const f16* qp = p.q + (int64_t)qi * p.q_stride + h * 64 + 8 * g;
        const f16* gp = b.dout + (int64_t)qi * b.do_stride + h * 64 + 8 * g;
        const f16* op = p.o + (int64_t)qi * p.o_stride + h * 64 + 8 * g;
#pragma unroll
        for (int k2 = 0; k2 < 2; k2++)
            qf[k2] = *(const half8*)(qp + 32 * k2), gf[k2] = *(const half8*)(gp + 32 * k2), of[k2] = *(const half8*)(op + 32 * k2);
    }
    const float lse = p.lse[(size_t)h * p.nq + qi];
    const KeyBounds kb_ = key_bounds(tr, listed, w);
    const int k0 = kb_.k0, k1 = kb_.k1, wlo = kb_.lo, whi = kb_.hi, flo = kb_.flo, fhi = kb_.fhi;
    const int nblk = k1 > k0 ? (k1 - k0 + 63) >> 6 : 0;
    uint32_t doff[LOADS];
#pragma unroll
    for (int x = 0; x < LOADS; x++) {
        const int c = ((w + NW * x) & 7) * 64 + l, r = c >> 3, ch = (c & 7) ^ (r & 7);
        doff[x] = (uint32_t)(r * (int)p.kv_stride * 2 + ch * 16);
    }
    auto stage = [&](int bl, char* to) {
        const int kb = k0 + 64 * bl;
        const uint32_t bytes = (uint32_t)((min(k1 - kb, 64) - 1) * (int)p.kv_stride * 2 + 128);
        const auto rk = buffer_rsrc(p.k + (int64_t)kb * p.kv_stride + kvh * 64, bytes);
        const auto rv = buffer_rsrc(p.v + (int64_t)kb * p.kv_stride + kvh * 64, bytes);
#pragma unroll
        for (int x = 0; x < LOADS; x++)
            lds_bdma16<false>(x < LOADS / 2 ? rk : rv, doff[x], to + (x < LOADS / 2 ? 0 : 8192) + ((w + NW * x) & 7) * 1024);
    };
    auto has = [&](int s) { return kg + KS * s < nblk; };
    if (has(0)) stage(kg, stage0 + kg * DQ_STAGE);
    if (BIAS == BIAS_TABLE) {
        load_bias(p, h, 1, tab0, 64 * NW * KS);
        for (int i = tid; i < NW * KS * HG * pitch; i += 64 * NW * KS) hist0[i] = 0.0f;
    }

    // The row's constants.
    float d = 0.0f, sq = 0.0f;
#pragma unroll
    for (int k2 = 0; k2 < 2; k2++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float v = widen<BF>(gf[k2][e]);
            d = fmaf(v, widen<BF>(of[k2][e]), d);
            sq = fmaf(v, v, sq);
        }
    d = sum_xor32(sum_xor16(d)), sq = sum_xor32(sum_xor16(sq));
    if (!real) {
        sq = 0.0f;
#pragma unroll
        for (int k2 = 0; k2 < 2; k2++) qf[k2] = gf[k2] = half8{};
    }
    // (past 2^20 either way: a row of biases like the type's lowest value, its weights lost in lse's rounding)
    const float nl = !real || fabsf(lse) > 1048576.0f ? -INFINITY : lse * -1.4426950408889634f;
    const float dn = real ? -d : 0.0f;
    float sigma = BF ? 1.0f : grad_scale(sq);
    const KeyRange kr = {__shfl(tr.lo, 16 * w + r16), __shfl(tr.hi, 16 * w + r16)};
    if (kg == 0) {
        if (g == 0) {
            float* to = row_info(b, h, row);
            to[0] = nl, to[64] = dn;
            *(int2*)(to + 128 + (row & 63)) = make_int2(kr.lo, kr.hi - kr.lo);
        }
        const float m = row_max(sq);
        if (l == 0) {
            b.max_do[(size_t)h * (b.nqp / 16) + q0 / 16 + w] = m;
            if (h == 0 && w == 0) b.bounds[tile] = make_int4(k0, k1, kb_.all_flo, kb_.all_fhi);
        }
    }
    const int wq0 = p.q_first + q0 + 16 * w, wql = wq0 + 15;
    const uint32_t kspan = (uint32_t)(kr.hi - kr.lo);
    const float slope = BIAS == BIAS_SLOPES ? p.slopes[h] * p.unit : 0.0f;
    const float* const tab = tab0 + p.reach + BIAS_PAD;
    __syncthreads();
    const float left = BIAS == BIAS_TABLE ? tab[-p.reach] : 0.0f, right = BIAS == BIAS_TABLE ? tab[p.reach] : 0.0f;
    float far_left = 0.0f, far_right = 0.0f;

    int koff[2], toff[4];
#pragma unroll
    for (int k2 = 0; k2 < 2; k2++) koff[k2] = att_swz(r16, 4 * k2 + g);
#pragma unroll
    for (int dt = 0; dt < 4; dt++) toff[dt] = att_swz(4 * g + j4, 2 * dt + (q4 >> 1)) + (q4 & 1) * 8;

    floatx4 dq[4];
    auto step = [&](int s, auto st_, auto careful_) __attribute__((always_inline)) {
        constexpr int ST = decltype(st_)::value;
        constexpr bool careful = decltype(careful_)::value;  // (the second time, as in the forward pass)
        stage_barrier<0>();
        const int kb0 = k0 + 64 * (kg + KS * s);
        const char* st = (ST ? stage1 : stage0) + kg * DQ_STAGE;
        if (has(s + 1)) stage(kg + KS * (s + 1), (ST ? stage0 : stage1) + kg * DQ_STAGE);
        if (!has(s) || kb0 + 64 <= wlo || kb0 >= whi) return;
        float diag[3] = {0.0f, 0.0f, 0.0f};  // sums along diagonals; those that run into the next half's keys go on
#pragma unroll
        for (int hf = 0; hf < 2; hf++) {  // 32 keys: kb + 16 t + 4 g + e
            const int kb = kb0 + 32 * hf;
            floatx4 base[2], sc[2], ds[2];
            half8 kf[2][2], vf[2][2];
            half4 kt[4][2];
            auto columns = [&](int dt) {
#pragma unroll
                for (int y = 0; y < 2; y++) kt[dt][y] = lds_read_tr16(st + toff[dt] + 4096 * hf + 2048 * y);
            };
            block_bias<BIAS>(p, tab, left, right, slope, kb, g, qpos, wq0, wql, base);
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int k2 = 0; k2 < 2; k2++) {
                    kf[t][k2] = *(const half8*)(st + koff[k2] + 4096 * hf + 2048 * t);
                    vf[t][k2] = *(const half8*)(st + 8192 + koff[k2] + 4096 * hf + 2048 * t);
                }
#pragma unroll
            for (int dt = 0; dt < 4; dt++)
                if (!careful) columns(dt);
#pragma unroll
            for (int t = 0; t < 2; t++) {
                sc[t] = CAP ? floatx4{0.0f, 0.0f, 0.0f, 0.0f} : base[t];
                ds[t] = floatx4{dn, dn, dn, dn};
#pragma unroll
                for (int k2 = 0; k2 < 2; k2++) sc[t] = mma<BF>(kf[t][k2], qf[k2], sc[t]);
#pragma unroll
                for (int k2 = 0; k2 < 2; k2++) ds[t] = mma<BF>(vf[t][k2], gf[k2], ds[t]);
            }
            if (CAP) cap_scores<2, true>(p, sc, base, sigma);
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) ds[t][e] *= fast_exp2(CAP ? sc[t][e] + nl : fmaf(sc[t][e], p.mul, nl));
            if (!(kb >= flo && kb + 32 <= fhi)) {  // (whatever a masked pair's score was)
                const int at = kb + 4 * g - kr.lo;
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++) ds[t][e] = (uint32_t)(at + 16 * t + e) < kspan ? ds[t][e] : 0.0f;
            }
            if (BIAS == BIAS_TABLE && !careful) {
                const bool far = kb - wql >= p.reach || kb + 31 - wq0 <= -p.reach;
                if (far) {
                    const float v = ((ds[0][0] + ds[0][1]) + (ds[0][2] + ds[0][3])) + ((ds[1][0] + ds[1][1]) + (ds[1][2] + ds[1][3]));
                    if (kb > wq0) far_right += v;
                    else far_left += v;
                } else {
#pragma unroll
                    for (int t = 0; t < 2; t++) diagonal_sums(ds[t], diag[t], diag[t + 1]);
                }
                if (!far || hf == 1) {
                    const int x0 = kb - wq0 + 4 * g - r16;
                    float* const to = hist + x0 + p.reach;
                    const bool within = kb - wql >= -p.reach && kb + 47 + 12 - wq0 <= p.reach;
                    if (HG == 4) {
                        // (read, add, write: an LDS addition of f32 takes its lanes one by one)
                        float was[3];
                        int at[3];
#pragma unroll
                        for (int t = 0; t < 2 + hf; t++) {
                            const int x = x0 + 16 * t;
                            at[t] = within || (x >= -p.reach && x <= p.reach) ? 16 * t : dists - x0 - p.reach;  // (or the spare)
                            was[t] = to[at[t]];
                            if (!within) {
                                far_left += x < -p.reach ? diag[t] : 0.0f;
                                far_right += x > p.reach ? diag[t] : 0.0f;
                            }
                        }
#pragma unroll
                        for (int t = 0; t < 2 + hf; t++) to[at[t]] = was[t] + diag[t];
                    } else {
#pragma unroll
                        for (int t = 0; t < 2 + hf; t++) {
                            const int x = x0 + 16 * t;
                            far_left += x < -p.reach ? diag[t] : 0.0f;
                            far_right += x > p.reach ? diag[t] : 0.0f;
                            // one group of lanes after the other: no two lanes of an addition share a distance
#pragma unroll
                            for (int y = 0; y < 4; y++) {
                                if (g == y && x >= -p.reach && x <= p.reach)
                                    __hip_atomic_fetch_add(to + 16 * t, diag[t], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT);
                                __builtin_amdgcn_wave_barrier();
                            }
                        }
                    }
                    diag[0] = diag[2];
                    diag[1] = diag[2] = 0.0f;
                }
            }
            if (CAP || !BF) {
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++) ds[t][e] *= CAP ? base[t][e] : sigma;
            }
            const bool by_pair = careful && !(kb >= flo && kb + 32 <= fhi);
            const uintx4 pairs = by_pair ? seen_pairs([&](int c) { return (uint32_t)(kb + c - kr.lo) < kspan; }) : uintx4{};
            const half8 sf = pack8<BF>(ds[0], ds[1]);
#pragma unroll
            for (int dt = 0; dt < 4; dt++) {
                if (careful) columns(dt);
                const half4 lo = kt[dt][0], hi = kt[dt][1];
                const half8 ka = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                dq[dt] = by_pair ? careful_mma<BF, true>(ka, sf, pairs, dq[dt]) : mma<BF>(ka, sf, dq[dt]);
            }
        }
    };
    const int nsteps = (nblk + KS - 1) / KS;
    auto all_keys = [&](auto careful) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < 4; t++) dq[t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int s = 0; s < nsteps; s += 2) {
            step(s, std::integral_constant<int, 0>{}, careful);
            if (s + 1 < nsteps) step(s + 1, std::integral_constant<int, 1>{}, careful);
        }
    };
    all_keys(std::false_type{});
    if (!(finite4(dq[0]) && finite4(dq[1]) && finite4(dq[2]) && finite4(dq[3])) && real) s_bad = 1;
    __syncthreads();
    if (__builtin_expect(__builtin_amdgcn_readfirstlane(s_bad), 0)) {
        if (!BF) sigma *= 0x1p-11f;
        if (has(0)) stage(kg, stage0 + kg * DQ_STAGE);
        all_keys(std::true_type{});
    }

    if (BIAS == BIAS_TABLE) {
        far_left = wave_sum(far_left), far_right = wave_sum(far_right);
        if (l == 0) {
            hist[0] += far_left;
            hist[dists - 1] += far_right;
        }
    }
    __syncthreads();
    if (BIAS == BIAS_TABLE) {
        float* to = b.part + ((size_t)h * b.tiles + tile) * dists;
        for (int i = tid; i < dists; i += 64 * NW * KS) {
            float s = hist0[i];
#pragma unroll
            for (int x = 1; x < NW * KS * HG; x++) s += hist0[x * pitch + i];
            to[i] = s;
        }
    }
    if (KS > 1) {
        if (kg > 0) {
            float* mg = (float*)stage0 + ((kg - 1) * NW + w) * 16 * 64;
#pragma unroll
            for (int f = 0; f < 16; f++) mg[f * 64 + l] = dq[f >> 2][f & 3];
        }
        __syncthreads();
        if (kg > 0) return;
#pragma unroll
        for (int k = 1; k < KS; k++) {
            const float* mg = (const float*)stage0 + ((k - 1) * NW + w) * 16 * 64;
#pragma unroll
            for (int f = 0; f < 16; f++) dq[f >> 2][f & 3] += mg[f * 64 + l];
        }
    }

    const float back = p.scale / sigma;
    if (real) {
        f16* to = b.dq + (int64_t)row * b.dq_stride + h * 64 + 4 * g;
#pragma unroll
        for (int dt = 0; dt < 4; dt++) *(half4*)(to + 16 * dt) = pack4<BF>(dq[dt] * back);
    }
}

// ---- dK and dV of 16 NG NW keys -----------------------------------------------------------------
// (Two waves a SIMD for the blocks of one group: without the bound the compiler took registers for one.)
template <bool BF, int BIAS, bool CAP, int NG, int NW, int KS>
__global__ __launch_bounds__(64 * NW * KS, KS == 1 ? 2 : 1) void attn_bias_dkv_kernel(BiasBack b) {
    const BiasParams& p = b.p;
    // Two stages, or three where the LDS has room: with two, a step waited for copies that it had seen
    // issued only one step before (the batch's copies and barriers alone, without the products, took
    // 51 of its 101 us).
    constexpr int NS = KS == 1 ? 3 : 2;
    __shared__ __attribute__((aligned(16))) char stage0[KS * DKV_STAGE], stage1[KS * DKV_STAGE];
    __shared__ __attribute__((aligned(16))) char stage2[NS == 3 ? KS * DKV_STAGE : 16];
    extern __shared__ __attribute__((aligned(16))) float tab0[];
    constexpr int WK = 16 * NG, KB = WK * NW, LOADS = 16 / NW;
    const int first = BIAS == BIAS_TABLE ? p.heads : 0;
    if ((int)blockIdx.x < first) {  // (first, so that they are done long before the others)
        const int h = blockIdx.x, dists = 2 * p.reach + 1;
        const float* from = b.part + (size_t)h * b.tiles * dists;
        float *sm = (float*)stage0, *sums = sm + 64 * NW * KS;
        int* bucket = (int*)(sums + dists);
        sum_groups<64 * NW * KS>(dists, b.tiles, sm, sums, 1, [&](int x, int i) { return from[(size_t)i * dists + x]; });
        for (int i = threadIdx.x; i < dists; i += 64 * NW * KS) bucket[i] = min(max(p.bucket[i], 0), p.buckets - 1);
        __syncthreads();
        sum_groups<64 * NW * KS>(p.buckets, dists, sm, b.dtable + h, p.heads,
                                 [&](int x, int i) { return bucket[i] == x ? sums[i] : 0.0f; });
        return;
    }
    const Quotient ht = divide(xcd_task(blockIdx.x - first, b.dkv_blocks), p.by_tiles);
    const int kvh = ht.q, kb = ht.r * KB;
    const int tid = threadIdx.x, l = tid & 63, r16 = l & 15, g = l >> 4;
    const int wk = __builtin_amdgcn_readfirstlane(tid >> 6), w = wk % NW, kg = wk / NW;
    const int j4 = r16 >> 2, q4 = r16 & 3;
    const int qt = b.nqp / 64;

    // This wave's keys: kw .. + WK - 1, the lane's the r16th of each 16.
    const int kw = kb + WK * w;
    half8 kf[NG][2], vf[NG][2];
    int key[NG];
#pragma unroll
    for (int x = 0; x < NG; x++) {
        key[x] = kw + 16 * x + r16;
        const int64_t at = (int64_t)min(key[x], p.nk - 1) * p.kv_stride + kvh * 64 + 8 * g;
#pragma unroll
        for (int k2 = 0; k2 < 2; k2++) {
            kf[x][k2] = *(const half8*)(p.k + at + 32 * k2);
            vf[x][k2] = *(const half8*)(p.v + at + 32 * k2);
        }
    }
    if (BIAS == BIAS_TABLE) load_bias(p, kvh * p.each, p.each, tab0, 64 * NW * KS);
    // 64 queries' keys
    auto tile_bounds = [&](int t) {
        int4 r = make_int4(0x7fffffff, 0, 0, 0x7fffffff);
        if (t < qt) {
            if (b.per == 1) return b.bounds[t];
            for (int x = 0; x < b.per; x++) {
                const int4 y = b.bounds[b.per * t + x];
                r.x = min(r.x, y.x), r.y = max(r.y, y.y), r.z = max(r.z, y.z), r.w = min(r.w, y.w);
            }
        }
        return r;
    };
    float sigma = 1.0f;
#pragma unroll
    for (int x = 0; x < NG; x++)
        if (key[x] >= p.nk) kf[x][0] = kf[x][1] = vf[x][0] = vf[x][1] = half8{};
    floatx4 dk[NG][4], dv[NG][4];
    __shared__ uint32_t s_bad;
    if (tid == 0) s_bad = 0;

    uint32_t off[LOADS];
#pragma unroll
    for (int x = 0; x < LOADS; x++) {  // 8 rows of Q (the first half of the copies) or dO
        const int c = ((w + NW * x) & 7) * 64 + l, r = c >> 3, ch = (c & 7) ^ (r & 7);
        off[x] = (uint32_t)(r * (int)(x < LOADS / 2 ? p.q_stride : b.do_stride) * 2 + ch * 16);
    }
    auto stage = [&](int h, int t, char* to) {
        const int q0 = 64 * t, n = min(p.nq - q0, 64);
        const auto rq = buffer_rsrc(p.q + (int64_t)q0 * p.q_stride + h * 64, (uint32_t)((n - 1) * (int)p.q_stride * 2 + 128));
        const auto rg = buffer_rsrc(b.dout + (int64_t)q0 * b.do_stride + h * 64, (uint32_t)((n - 1) * (int)b.do_stride * 2 + 128));
        const auto ri = buffer_rsrc(b.info + ((size_t)h * qt + t) * 256, 1024);
#pragma unroll
        for (int x = 0; x < LOADS; x++)
            lds_bdma16<false>(x < LOADS / 2 ? rq : rg, off[x], to + (x < LOADS / 2 ? 0 : 8192) + ((w + NW * x) & 7) * 1024);
#pragma unroll
        for (int x = 0; x < 4 / NW; x++)  // (a quarter of `info` each)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                ri, (__attribute__((address_space(3))) void*)(to + 16384 + 256 * (w + NW * x)), 4, l * 4 + 256 * (w + NW * x), 0, 0, 0);
    };
    int aoff[2], toff[4];
#pragma unroll
    for (int k2 = 0; k2 < 2; k2++) aoff[k2] = att_swz(r16, 4 * k2 + g);
#pragma unroll
    for (int dt = 0; dt < 4; dt++) toff[dt] = att_swz(4 * g + j4, 2 * dt + (q4 >> 1)) + (q4 & 1) * 8;

    // 64 tiles of 64 queries at a time (the bounds of 256 loaded together): those that see some of the
    // block's keys, for each query head; group kg of the block takes every KS-th.
    int4 ahead[4];
    auto all_queries = [&](auto careful_) __attribute__((always_inline)) {
        constexpr bool careful = decltype(careful_)::value;  // (the second time, as in the forward pass)
#pragma unroll
        for (int x = 0; x < NG; x++)
#pragma unroll
            for (int t = 0; t < 4; t++) dk[x][t] = dv[x][t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int t0 = 0; t0 < qt; t0 += 64) {
            if ((t0 & 255) == 0) {
#pragma unroll
                for (int x = 0; x < 4; x++) ahead[x] = tile_bounds(t0 + 64 * x + l);
            }
            const int4 bd = ahead[0];
            ahead[0] = ahead[1], ahead[1] = ahead[2], ahead[2] = ahead[3];
            const uint64_t seen = __builtin_amdgcn_ballot_w64(bd.x < kb + KB && bd.y > kb);
            if (seen == 0) continue;
            const int steps = p.each * __builtin_popcountll(seen);
            int sub = 0;
            uint64_t rest = seen;
            auto skip = [&](int n) {  // (query head, tile) n further on
                for (; n > 0; n--) {
                    rest &= rest - 1;
                    if (rest == 0) rest = seen, sub++;
                }
            };
            auto has = [&](int s) { return kg + KS * s < steps; };
            struct Step {
                int sub, t;
            };
            auto at_step = [&]() { return Step{sub, t0 + __builtin_ctzll(rest)}; };
            skip(kg);
            Step now = at_step(), then = now;  // (then: the step after, of three stages)
            __syncthreads();  // the table; the stages of the last 64 tiles are no longer read
            if (has(0)) stage(kvh * p.each + now.sub, now.t, stage0 + kg * DKV_STAGE);
            if (NS == 3 && has(1)) {
                skip(KS);
                then = at_step();
                stage(kvh * p.each + then.sub, then.t, stage1 + kg * DKV_STAGE);
            }
            if (!BF) {
                float m = 0.0f;
                if ((seen >> l) & 1)
                    for (int s = 0; s < p.each; s++) {
                        const floatx4 d = *(const floatx4*)(b.max_do + (size_t)(kvh * p.each + s) * (b.nqp / 16) + 4 * (t0 + l));
                        m = fmaxf(m, fmaxf(fmaxf(d[0], d[1]), fmaxf(d[2], d[3])));
                    }
                const float was = sigma;
                sigma = grad_scale(max_xor32(max_xor16(row_max(m)))) * (careful ? 0x1p-11f : 1.0f);
                if (sigma != was) {
#pragma unroll
                    for (int x = 0; x < NG; x++)
#pragma unroll
                        for (int t = 0; t < 4; t++) dk[x][t] = dk[x][t] * (sigma / was);
                }
            }
            auto step = [&](int s, auto st_) __attribute__((always_inline)) {
                constexpr int ST = decltype(st_)::value;
                // (all but the next step's copies have landed)
                if (NS == 3 && has(s + 1)) stage_barrier<NS == 3 ? LOADS + 4 / NW : 0>();
                else stage_barrier<0>();
                if (!has(s)) return;
                const char* st = (ST == 0 ? stage0 : ST == 1 ? stage1 : stage2) + kg * DKV_STAGE;
                const int hx = now.sub, pos0 = p.q_first + 64 * now.t, h = kvh * p.each + hx, at_t = now.t - t0;
                const int lo = __builtin_amdgcn_readlane(bd.x, at_t), hi = __builtin_amdgcn_readlane(bd.y, at_t);
                const int flo = __builtin_amdgcn_readlane(bd.z, at_t), fhi = __builtin_amdgcn_readlane(bd.w, at_t);
                const bool act = kw < hi && kw + WK > lo, full = kw >= flo && kw + WK <= fhi;
                const float slope = BIAS == BIAS_SLOPES ? p.slopes[h] * p.unit : 0.0f;
                const float* tab = tab0 + (BIAS == BIAS_TABLE ? hx * p.row + p.reach + BIAS_PAD : 0);
                const float* nl = (const float*)(st + 16384);
                const float* dn = (const float*)(st + 16384 + 256);
                const int2* rg = (const int2*)(st + 16384 + 512);
                now = then;
                if (has(s + NS - 1)) {
                    skip(KS);
                    then = at_step();
                    constexpr int TO = (ST + NS - 1) % NS;
                    stage(kvh * p.each + then.sub, then.t, (TO == 0 ? stage0 : TO == 1 ? stage1 : stage2) + kg * DKV_STAGE);
                }
                if (NS == 2) now = then;
                if (!act) return;
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {  // 32 queries: rows 32 hf + 16 t + 4 g + e of the tile, column key[x]
                    half8 qa[2][2], ga[2][2];
                    floatx4 l4[2], d4[2], base[2 * NG], sc[2 * NG], ds[2 * NG];
#pragma unroll
                    for (int t = 0; t < 2; t++) {
                        const int at = 32 * hf + 16 * t;
#pragma unroll
                        for (int k2 = 0; k2 < 2; k2++) {
                            qa[t][k2] = *(const half8*)(st + aoff[k2] + 128 * at);
                            ga[t][k2] = *(const half8*)(st + 8192 + aoff[k2] + 128 * at);
                        }
                        l4[t] = *(const floatx4*)(nl + at + 4 * g);
                        d4[t] = *(const floatx4*)(dn + at + 4 * g);
                    }
                    if (BIAS == BIAS_TABLE) {
                        // distances from kw - (pos0 + 32 hf + 31) to kw + WK - 1 - (pos0 + 32 hf)
                        const int z = kw - pos0 - 32 * hf;
                        if (z - 31 >= p.reach || z + WK - 1 <= -p.reach) {
                            const float b0 = z > 0 ? tab[p.reach] : tab[-p.reach];
#pragma unroll
                            for (int y = 0; y < 2 * NG; y++) base[y] = floatx4{b0, b0, b0, b0};
                        } else {
                            const float* from = tab + (z + r16 - 4 * g);
#pragma unroll
                            for (int x = 0; x < NG; x++)
#pragma unroll
                                for (int t = 0; t < 2; t++)
#pragma unroll
                                    for (int e = 0; e < 4; e++) base[2 * x + t][e] = from[16 * x - 16 * t - e];
                        }
                    } else if (BIAS == BIAS_SLOPES) {
                        const float y = (float)(kw + r16 - pos0 - 32 * hf - 4 * g);
#pragma unroll
                        for (int x = 0; x < NG; x++)
#pragma unroll
                            for (int t = 0; t < 2; t++)
#pragma unroll
                                for (int e = 0; e < 4; e++) base[2 * x + t][e] = -slope * fabsf(y + (float)(16 * x - 16 * t - e));
                    } else {
#pragma unroll
                        for (int y = 0; y < 2 * NG; y++) base[y] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
                    }
#pragma unroll
                    for (int x = 0; x < NG; x++)
#pragma unroll
                        for (int t = 0; t < 2; t++) {
                            const int y = 2 * x + t;
                            sc[y] = CAP ? floatx4{0.0f, 0.0f, 0.0f, 0.0f} : base[y];
                            ds[y] = d4[t];
#pragma unroll
                            for (int k2 = 0; k2 < 2; k2++) sc[y] = mma<BF>(qa[t][k2], kf[x][k2], sc[y]);
#pragma unroll
                            for (int k2 = 0; k2 < 2; k2++) ds[y] = mma<BF>(ga[t][k2], vf[x][k2], ds[y]);
                        }
                    if (CAP) cap_scores<2 * NG, true>(p, sc, base, sigma);
                    if (!full) {
#pragma unroll
                        for (int t = 0; t < 2; t++)
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                const int2 k = rg[32 * hf + 16 * t + 4 * g + e];
#pragma unroll
                                for (int x = 0; x < NG; x++) {
                                    const bool ok = (uint32_t)(key[x] - k.x) < (uint32_t)k.y;
                                    sc[2 * x + t][e] = ok ? sc[2 * x + t][e] : -INFINITY;
                                    ds[2 * x + t][e] = ok ? ds[2 * x + t][e] : 0.0f;
                                }
                            }
                    }
                    half4 gt[4][2], qt4[4][2];
                    auto columns = [&](int dt) {
#pragma unroll
                        for (int y = 0; y < 2; y++) {
                            gt[dt][y] = lds_read_tr16(st + 8192 + toff[dt] + 4096 * hf + 2048 * y);
                            qt4[dt][y] = lds_read_tr16(st + toff[dt] + 4096 * hf + 2048 * y);
                        }
                    };
#pragma unroll
                    for (int dt = 0; dt < 4; dt++)
                        if (!careful) columns(dt);
                    half8 pf[NG], sf[NG];
#pragma unroll
                    for (int x = 0; x < NG; x++) {
#pragma unroll
                        for (int t = 0; t < 2; t++)
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                const int y = 2 * x + t;
                                sc[y][e] = fast_exp2(CAP ? sc[y][e] + l4[t][e] : fmaf(sc[y][e], p.mul, l4[t][e]));
                                ds[y][e] *= sc[y][e];
                                if (CAP || !BF) ds[y][e] *= CAP ? base[y][e] : sigma;
                            }
                        pf[x] = pack8<BF>(sc[2 * x], sc[2 * x + 1]);
                        sf[x] = pack8<BF>(ds[2 * x], ds[2 * x + 1]);
                    }
                    if (careful && !full) {
#pragma unroll
                        for (int x = 0; x < NG; x++) {
                            const uintx4 pairs = seen_pairs([&](int c) {
                                const int2 k = rg[32 * hf + c];
                                return (uint32_t)(key[x] - k.x) < (uint32_t)k.y;
                            });
#pragma unroll
                            for (int dt = 0; dt < 4; dt++) {
                                columns(dt);
                                const half8 a = {gt[dt][0][0], gt[dt][0][1], gt[dt][0][2], gt[dt][0][3], gt[dt][1][0], gt[dt][1][1], gt[dt][1][2], gt[dt][1][3]};
                                const half8 c = {qt4[dt][0][0], qt4[dt][0][1], qt4[dt][0][2], qt4[dt][0][3], qt4[dt][1][0], qt4[dt][1][1], qt4[dt][1][2], qt4[dt][1][3]};
                                dv[x][dt] = careful_mma<BF, false>(a, pf[x], pairs, dv[x][dt]);
                                dk[x][dt] = careful_mma<BF, true>(c, sf[x], pairs, dk[x][dt]);
                            }
                        }
                        continue;
                    }
#pragma unroll
                    for (int dt = 0; dt < 4; dt++) {
                        if (careful) columns(dt);
                        const half8 a = {gt[dt][0][0], gt[dt][0][1], gt[dt][0][2], gt[dt][0][3], gt[dt][1][0], gt[dt][1][1], gt[dt][1][2], gt[dt][1][3]};
                        const half8 c = {qt4[dt][0][0], qt4[dt][0][1], qt4[dt][0][2], qt4[dt][0][3], qt4[dt][1][0], qt4[dt][1][1], qt4[dt][1][2], qt4[dt][1][3]};
#pragma unroll
                        for (int x = 0; x < NG; x++) {
                            dv[x][dt] = mma<BF>(a, pf[x], dv[x][dt]);
                            dk[x][dt] = mma<BF>(c, sf[x], dk[x][dt]);
                        }
                    }
                }
            };
            const int nsteps = (steps + KS - 1) / KS;
            for (int s = 0; s < nsteps; s += NS) {
                step(s, std::integral_constant<int, 0>{});
                if (s + 1 < nsteps) step(s + 1, std::integral_constant<int, 1>{});
                if (NS == 3 && s + 2 < nsteps) step(s + 2, std::integral_constant<int, NS - 1>{});
            }
        }
    };
    all_queries(std::false_type{});
    bool fine = true;
#pragma unroll
    for (int x = 0; x < NG; x++)
#pragma unroll
        for (int t = 0; t < 4; t++) fine = fine && (key[x] >= p.nk || (finite4(dk[x][t]) && finite4(dv[x][t])));
    if (!fine) s_bad = 1;
    __syncthreads();
    if (__builtin_expect(__builtin_amdgcn_readfirstlane(s_bad), 0)) all_queries(std::true_type{});

    if (KS > 1) {
        __syncthreads();
        if (kg > 0) {
            float* mg = (float*)stage0 + ((kg - 1) * NW + w) * 32 * NG * 64;
#pragma unroll
            for (int x = 0; x < NG; x++)
#pragma unroll
                for (int f = 0; f < 16; f++) {
                    mg[(32 * x + f) * 64 + l] = dk[x][f >> 2][f & 3];
                    mg[(32 * x + 16 + f) * 64 + l] = dv[x][f >> 2][f & 3];
                }
        }
        __syncthreads();
        if (kg > 0) return;
#pragma unroll
        for (int k = 1; k < KS; k++) {
            const float* mg = (const float*)stage0 + ((k - 1) * NW + w) * 32 * NG * 64;
#pragma unroll
            for (int x = 0; x < NG; x++)
#pragma unroll
                for (int f = 0; f < 16; f++) {
                    dk[x][f >> 2][f & 3] += mg[(32 * x + f) * 64 + l];
                    dv[x][f >> 2][f & 3] += mg[(32 * x + 16 + f) * 64 + l];
                }
        }
    }
    const float back = p.scale / sigma;
#pragma unroll
    for (int x = 0; x < NG; x++) {
        if (key[x] >= p.nk) continue;
        const int64_t at = (int64_t)key[x] * b.dkv_stride + kvh * 64 + 4 * g;
#pragma unroll
        for (int dt = 0; dt < 4; dt++) {
            *(half4*)(b.dk + at + 16 * dt) = pack4<BF>(dk[x][dt] * back);
            *(half4*)(b.dv + at + 16 * dt) = pack4<BF>(dv[x][dt]);
        }
    }
}

// ---- launching ----------------------------------------------------------------------------------
// The tiles of a call: 16 dq_nw queries, 16 ng nw keys a block, in ks groups.
struct GradPlan {
    int dq_nw, dq_ks, ng, nw, ks;
};

constexpr int LDS_BYTES = 160 * 1024 - 64;  // (the rest: a flag)

[[noreturn]] inline void grad_fail(const std::string& m) { throw std::runtime_error("attention_bias_backward: " + m); }

template <bool BF, int BIAS, bool CAP, int NW, int KS>
void launch_dq(BiasBack b, hipStream_t st) {
    constexpr int waves = NW * KS;
    static std::atomic<uint64_t> devices{0};
    if (!dynamic_lds(devices, reinterpret_cast<const void*>(attn_bias_dq_kernel<BF, BIAS, CAP, NW, KS>),
                     std::min(dq_lds(BIAS_MAX_REACH, NW, KS), LDS_BYTES - 2 * KS * DQ_STAGE)))
        grad_fail("a kernel cannot have its LDS");
    const size_t lds = BIAS == BIAS_TABLE ? dq_lds(b.p.reach, NW, KS) : 0;
    b.p.by_tiles = Div(b.tiles);
    hipLaunchKernelGGL((attn_bias_dq_kernel<BF, BIAS, CAP, NW, KS>), dim3(b.tiles * b.p.heads), dim3(64 * waves), lds, st, b);
}

template <bool BF, int BIAS, bool CAP, int NG, int NW, int KS>
void launch_dkv(BiasBack b, hipStream_t st) {
    static std::atomic<uint64_t> devices{0};
    if (!dynamic_lds(devices, reinterpret_cast<const void*>(attn_bias_dkv_kernel<BF, BIAS, CAP, NG, NW, KS>), 4 * BIAS_MAX_TABLE))
        grad_fail("a kernel cannot have its LDS");
    const int tiles = (b.p.nk + 16 * NG * NW - 1) / (16 * NG * NW);
    b.dkv_blocks = tiles * b.p.kv_heads, b.p.by_tiles = Div(std::max(tiles, 1));
    const int blocks = b.dkv_blocks + (BIAS == BIAS_TABLE ? b.p.heads : 0);
    const size_t lds = BIAS == BIAS_TABLE ? 4 * (size_t)b.p.each * b.p.row : 0;
    if (blocks) hipLaunchKernelGGL((attn_bias_dkv_kernel<BF, BIAS, CAP, NG, NW, KS>), dim3(blocks), dim3(64 * NW * KS), lds, st, b);
}

template <bool BF, int BIAS, bool CAP>
void grad_kernels(const BiasBack& b, const GradPlan& plan, hipStream_t st) {
    if (b.p.nq > 0) {
        if (plan.dq_nw == 1) launch_dq<BF, BIAS, CAP, 1, 4>(b, st);
        else if (plan.dq_nw == 2) launch_dq<BF, BIAS, CAP, 2, 4>(b, st);
        else if (plan.dq_ks == 2) launch_dq<BF, BIAS, CAP, 4, 2>(b, st);
        else launch_dq<BF, BIAS, CAP, 4, 1>(b, st);
    }
    if (plan.nw == 1) launch_dkv<BF, BIAS, CAP, 1, 1, 4>(b, st);
    else if (plan.ng == 1) launch_dkv<BF, BIAS, CAP, 1, 2, 4>(b, st);
    else if (plan.nw == 2) launch_dkv<BF, BIAS, CAP, 2, 2, 4>(b, st);
    else if (plan.ks == 2) launch_dkv<BF, BIAS, CAP, 2, 4, 2>(b, st);
    else launch_dkv<BF, BIAS, CAP, 2, 4, 1>(b, st);
}

// (f16: attn_bias_back.hip; bf16: attn_bias_back_bf16.hip, so that they compile side by side)
template <bool BF>
void grad_launch(const BiasBack& b, const GradPlan& plan, int bias, bool cap, hipStream_t st) {
    if (bias == BIAS_TABLE) cap ? grad_kernels<BF, BIAS_TABLE, true>(b, plan, st) : grad_kernels<BF, BIAS_TABLE, false>(b, plan, st);
    else if (bias == BIAS_SLOPES) cap ? grad_kernels<BF, BIAS_SLOPES, true>(b, plan, st) : grad_kernels<BF, BIAS_SLOPES, false>(b, plan, st);
    else cap ? grad_kernels<BF, BIAS_NONE, true>(b, plan, st) : grad_kernels<BF, BIAS_NONE, false>(b, plan, st);
}
void grad_launch_bf16(const BiasBack& b, const GradPlan& plan, int bias, bool cap, hipStream_t st);

}  // namespace jh
