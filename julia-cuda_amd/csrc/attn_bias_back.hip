// The biased attention's backward pass (attn_bias.h). With P = exp(s - lse) and
// D_i = dO_i . o_i:
//   dV = P^T dO,  dS = P (dO V^T - D),  dbias[t] = the sum of dS over j - pos_i = t,
//   dA = scale dS (the tanh's slope),  dQ = dA K,  dK = dA^T Q.
//
// Three launches: a row's constants (rows_kernel), the products (grad_kernel's two roles: a block
// takes 64 NG keys of a key head and goes over the queries that see them, for dK and dV; or 64 queries
// of a head and goes over their keys, for dQ and the bias's gradient) and the table's sums
// (table_kernel). Each role computes the scores again, seven products in place of five, so that no
// block adds to another's results: the gradients are the same bits at every call.
//
// - Both roles keep the scores where the next product wants them: lane r16's column is its key (dK,
//   dV) or its query (dQ), and the transposed operand comes from LDS by the transposing read.
// - dO V^T starts from -D in the accumulators, the scores from the bias.
// - f16: dS is scaled by a power of two a key head, from the largest |dO_i| and |v_j|, so that it
//   neither overflows nor loses its small values (|dS_ij| <= 2 |dO_i| |v_j| at most); taken off at the end.
// - The bias's gradient in 32 bits, before dS is rounded: a 64-key block past `reach` on one side adds
//   to one sum; else the 16 queries of a wave are summed along the diagonals with lane shifts (a
//   lane's four keys of a 16-key tile against its neighbours' queries) and added to the wave's own
//   row of distances in LDS.
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
    // the workspace: per head and (padded) row -lse log2(e) (-inf: a row without keys) and -D, per row
    // its keys (first, number), per 64 rows (least first, most past last, most first, least past last),
    // per 16 rows the largest |dO|^2 a head and |v|^2 a key head, per (head, 64 rows) the distances' sums
    float *nl, *dn;
    int2* range;
    int4* bounds;
    float *max_do, *max_v, *part;
    int nqp, qt, pb;
};

constexpr int PREP_ROWS = 16;

// Rows 16 b .. of the queries and of the keys, a wave four of them.
template <bool BF>
__global__ __launch_bounds__(256) void attn_bias_rows_kernel(BiasBack b) {
    const BiasParams& p = b.p;
    extern __shared__ float sm[];  // [4][heads + kv_heads]
    const int tid = threadIdx.x, l = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int width = p.heads + p.kv_heads;
    float* mine = sm + w * width;
    for (int i = l; i < width; i += 64) mine[i] = 0.0f;
    const int r0 = blockIdx.x * PREP_ROWS;
    // (a head's eight lanes keep its maximum over the wave's rows: written once a row by one lane)
    for (int x = 0; x < PREP_ROWS / 4; x++) {
        const int i = r0 + 4 * x + w;
        if (i < b.nqp) {
            for (int c = l; c < p.heads * 8; c += 64) {
                float d = 0.0f, sq = 0.0f;
                if (i < p.nq) {
                    const half8 g = *(const half8*)(b.dout + (int64_t)i * b.do_stride + c * 8);
                    const half8 o = *(const half8*)(p.o + (int64_t)i * p.o_stride + c * 8);
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const float v = widen<BF>(g[e]);
                        d = fmaf(v, widen<BF>(o[e]), d);
                        sq = fmaf(v, v, sq);
                    }
                }
                d = group_sum<8>(d), sq = group_sum<8>(sq);
                const int h = c >> 3;
                if ((l & 7) == 0) {
                    const float lse = i < p.nq ? p.lse[(size_t)h * p.nq + i] : -INFINITY;
                    // (a row of biases like the type's lowest value: its weights are lost in lse's rounding)
                    b.nl[(size_t)h * b.nqp + i] = fabsf(lse) > 1048576.0f ? -INFINITY : lse * -1.4426950408889634f;
                    b.dn[(size_t)h * b.nqp + i] = -d;
                    mine[h] = fmaxf(mine[h], sq);
                }
            }
        }
        if (i < p.nk)
            for (int c = l; c < p.kv_heads * 8; c += 64) {
                const half8 v = *(const half8*)(p.v + (int64_t)i * p.kv_stride + c * 8);
                float sq = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; e++) sq = fmaf(widen<BF>(v[e]), widen<BF>(v[e]), sq);
                sq = group_sum<8>(sq);
                if ((l & 7) == 0) mine[p.heads + (c >> 3)] = fmaxf(mine[p.heads + (c >> 3)], sq);
            }
    }
    __syncthreads();
    for (int i = tid; i < width; i += 256) {
        const float m = fmaxf(fmaxf(sm[i], sm[width + i]), fmaxf(sm[2 * width + i], sm[3 * width + i]));
        if (i < p.heads) b.max_do[(size_t)i * b.pb + blockIdx.x] = m;
        else b.max_v[(size_t)(i - p.heads) * b.pb + blockIdx.x] = m;
    }
    if (blockIdx.x % 4 == 0 && w == 0 && r0 < b.nqp) {
        const int i = r0 + l;
        const KeyRange r = i < p.nq ? key_range(p, i) : KeyRange{0, 0};
        b.range[i] = make_int2(r.lo, r.hi - r.lo);
        const bool some = r.hi > r.lo;
        const int lo = wave_min(some ? r.lo : 0x7fffffff), hi = wave_max(r.hi);
        const int flo = wave_max(r.lo), fhi = wave_min(i < p.nq ? r.hi : 0x7fffffff);
        if (l == 0) b.bounds[r0 / 64] = make_int4(lo, hi, flo, fhi);
    }
}

// The power of two that dS of a key head is scaled by (f16), so that 2 |dO| |v| is at most 2^15.
__device__ __forceinline__ float grad_scale(const BiasBack& b, int kvh) {
    const int l = threadIdx.x & 63;
    float d = 0.0f, v = 0.0f;
    for (int i = l; i < b.pb; i += 64) {
        for (int x = 0; x < b.p.each; x++) d = fmaxf(d, b.max_do[(size_t)(kvh * b.p.each + x) * b.pb + i]);
        v = fmaxf(v, b.max_v[(size_t)kvh * b.pb + i]);
    }
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) d = fmaxf(d, __shfl_xor(d, s)), v = fmaxf(v, __shfl_xor(v, s));
    const float m = sqrtf(d) * sqrtf(v);
    if (!(m > 0.0f && m < INFINITY)) return 1.0f;
    int e;
    frexpf(m, &e);  // m < 2^e
    return ldexpf(1.0f, min(max(14 - e, -100), 100));
}

// One key's share of a row's gradient, for the paths that go value by value: the weight and
// dA (without the scale) of query i (head h) and key j.
template <bool BF, int BIAS, bool CAP>
__device__ __forceinline__ void grad_pair(const BiasBack& b, const float* tab, float slope, int h, int kvh, int i, int j,
                                          float& w, float& da) {
    const BiasParams& p = b.p;
    float cap;
    const float qk = dot64<BF>(p.q + (int64_t)i * p.q_stride + h * 64, p.k + (int64_t)j * p.kv_stride + kvh * 64);
    const float s = score_of<CAP>(p, qk, bias_at<BIAS>(p, tab, slope, j - (p.q_first + i)), cap);
    w = fast_exp2(s + b.nl[(size_t)h * b.nqp + i]);
    const float dp = dot64<BF>(b.dout + (int64_t)i * b.do_stride + h * 64, p.v + (int64_t)j * p.kv_stride + kvh * 64);
    da = w * (dp + b.dn[(size_t)h * b.nqp + i]) * cap;
}

// ---- dK and dV of 64 NG keys ------------------------------------------------------------------
constexpr int GRAD_STAGE = 16384 + 1024;  // Q, dO, -lse, -D and the key ranges of 64 queries

template <bool BF, int BIAS, bool CAP, int NG>
__global__ __launch_bounds__(256) void attn_bias_dkv_kernel(BiasBack b) {
    const BiasParams& p = b.p;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    constexpr int KB = 64 * NG;
    const int tiles = (p.nk + KB - 1) / KB;
    const int task = xcd_task(blockIdx.x, tiles * p.kv_heads);
    const int kvh = task / tiles, kb = (task % tiles) * KB;
    const int tid = threadIdx.x, l = tid & 63, r16 = l & 15, g = l >> 4;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int j4 = r16 >> 2, q4 = r16 & 3;
    float* const tab0 = (float*)(lds + 2 * GRAD_STAGE);
    if (BIAS == BIAS_TABLE) load_bias(p, kvh * p.each, p.each, tab0, 256);
    const float sigma = BF ? 1.0f : grad_scale(b, kvh);

    // This wave's keys: group x's are kb + 64 x + 16 w .. + 15, the lane's the r16th.
    half8 kf[NG][2], vf[NG][2];
    int key[NG];
#pragma unroll
    for (int x = 0; x < NG; x++) {
        key[x] = kb + 64 * x + 16 * w + r16;
        const int64_t at = (int64_t)min(key[x], p.nk - 1) * p.kv_stride + kvh * 64 + 8 * g;
#pragma unroll
        for (int k2 = 0; k2 < 2; k2++) {
            kf[x][k2] = *(const half8*)(p.k + at + 32 * k2);
            vf[x][k2] = *(const half8*)(p.v + at + 32 * k2);
            if (key[x] >= p.nk) kf[x][k2] = vf[x][k2] = half8{};
        }
    }
    floatx4 dk[NG][4], dv[NG][4];
#pragma unroll
    for (int x = 0; x < NG; x++)
#pragma unroll
        for (int t = 0; t < 4; t++) dk[x][t] = dv[x][t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};

    uint32_t qoff[4], goff[4];
#pragma unroll
    for (int x = 0; x < 4; x++) {  // copy x of Q (x < 2) or dO: 8 rows each
        const int I = (w + 4 * x) & 7, c = I * 64 + l, r = c >> 3, ch = (c & 7) ^ (r & 7);
        qoff[x] = (uint32_t)(r * (int)p.q_stride * 2 + ch * 16);
        goff[x] = (uint32_t)(r * (int)b.do_stride * 2 + ch * 16);
    }
    auto stage = [&](int h, int t, int st) {
        char* to = lds + st * GRAD_STAGE;
        const int q0 = 64 * t, n = min(p.nq - q0, 64);
        const auto rq = buffer_rsrc(p.q + (int64_t)q0 * p.q_stride + h * 64, (uint32_t)((n - 1) * (int)p.q_stride * 2 + 128));
        const auto rg = buffer_rsrc(b.dout + (int64_t)q0 * b.do_stride + h * 64, (uint32_t)((n - 1) * (int)b.do_stride * 2 + 128));
#pragma unroll
        for (int x = 0; x < 2; x++) lds_bdma16<false>(rq, qoff[x], to + ((w + 4 * x) & 7) * 1024);
#pragma unroll
        for (int x = 2; x < 4; x++) lds_bdma16<false>(rg, goff[x], to + 8192 + ((w + 4 * x) & 7) * 1024);
        const void* src = w == 0 ? (const void*)(b.nl + (size_t)h * b.nqp + q0)
                        : w == 1 ? (const void*)(b.dn + (size_t)h * b.nqp + q0)
                                 : (const void*)((const int*)(b.range + q0) + 64 * (w - 2));
        __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer_rsrc(src, 256),
            (__attribute__((address_space(3))) void*)(to + 16384 + 256 * w), 4, l * 4, 0, 0, 0);
    };

    int aoff[2], toff[4];
#pragma unroll
    for (int k2 = 0; k2 < 2; k2++) aoff[k2] = att_swz(r16, 4 * k2 + g);
#pragma unroll
    for (int dt = 0; dt < 4; dt++) toff[dt] = att_swz(4 * g + j4, 2 * dt + (q4 >> 1)) + (q4 & 1) * 8;
    __syncthreads();  // (the table)

    // 64 tiles of 64 queries at a time: those that see some of the keys, for each query head.
    for (int t0 = 0; t0 < b.qt; t0 += 64) {
        int4 bd = make_int4(0, 0, 0, 0);
        if (t0 + l < b.qt) bd = b.bounds[t0 + l];
        const uint64_t seen = __builtin_amdgcn_ballot_w64(bd.x < kb + KB && bd.y > kb);
        if (seen == 0) continue;
        int sub = 0;
        uint64_t rest = seen;
        const int steps = p.each * __builtin_popcountll(seen);
        auto next = [&](int& h, int& t) {  // the next (query head, tile)
            if (rest == 0) rest = seen, sub++;
            t = t0 + __builtin_ctzll(rest);
            h = sub;
            rest &= rest - 1;
        };
        int hx, tx, hn = 0, tn = 0;
        next(hx, tx);
        __syncthreads();  // the stages of the last group of tiles are no longer read
        stage(kvh * p.each + hx, tx, 0);
        for (int s = 0; s < steps; s++) {
            wait_vmcnt<0>();
            __builtin_amdgcn_s_barrier();
            const char* st = lds + (s & 1) * GRAD_STAGE;
            const bool more = s + 1 < steps;
            if (more) next(hn, tn);
            const int q0 = 64 * tx, pos0 = p.q_first + q0;
            const int flo = __builtin_amdgcn_readlane(bd.z, tx - t0), fhi = __builtin_amdgcn_readlane(bd.w, tx - t0);
            const bool full = kb >= flo && kb + KB <= fhi;
            const int h = kvh * p.each + hx;
            const float slope = BIAS == BIAS_SLOPES ? p.slopes[h] * p.unit : 0.0f;
            const float* tab = tab0 + (BIAS == BIAS_TABLE ? hx * p.row + p.reach + BIAS_PAD : 0);
            const float* nl = (const float*)(st + 16384);
            const float* dn = (const float*)(st + 16384 + 256);
            const int2* rg = (const int2*)(st + 16384 + 512);
#pragma unroll
            for (int hf = 0; hf < 2; hf++) {  // 32 queries: rows q0 + 32 hf + 16 t + 4 g + e, column key[x]
                half8 qa[2][2], ga[2][2];
                floatx4 l4[2], d4[2], base[NG][2];
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    const int at = 32 * hf + 16 * t + 4 * g;
#pragma unroll
                    for (int k2 = 0; k2 < 2; k2++) {
                        qa[t][k2] = *(const half8*)(st + aoff[k2] + 4096 * hf + 2048 * t);
                        ga[t][k2] = *(const half8*)(st + 8192 + aoff[k2] + 4096 * hf + 2048 * t);
                    }
                    l4[t] = *(const floatx4*)(nl + at);
                    d4[t] = *(const floatx4*)(dn + at);
#pragma unroll
                    for (int x = 0; x < NG; x++) {
                        if (BIAS == BIAS_TABLE) {
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                base[x][t][e] = tab[min(max(key[x] - pos0 - at - e, -p.reach), p.reach)];
                        } else if (BIAS == BIAS_SLOPES) {
                            const float y = (float)(key[x] - pos0 - at);
#pragma unroll
                            for (int e = 0; e < 4; e++) base[x][t][e] = fmaf(-slope, fabsf(y - (float)e), p.off);
                        } else {
                            const float y = CAP ? p.off : 0.0f;
                            base[x][t] = floatx4{y, y, y, y};
                        }
                    }
                }
                floatx4 sc[NG][2], ds[NG][2];
#pragma unroll
                for (int x = 0; x < NG; x++)
#pragma unroll
                    for (int t = 0; t < 2; t++) {
                        sc[x][t] = CAP ? floatx4{0.0f, 0.0f, 0.0f, 0.0f} : base[x][t];
                        ds[x][t] = d4[t];
#pragma unroll
                        for (int k2 = 0; k2 < 2; k2++) {
                            sc[x][t] = mma<BF>(qa[t][k2], kf[x][k2], sc[x][t]);
                            ds[x][t] = mma<BF>(ga[t][k2], vf[x][k2], ds[x][t]);
                        }
                    }
                if (!full) {
#pragma unroll
                    for (int t = 0; t < 2; t++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const int2 k = rg[32 * hf + 16 * t + 4 * g + e];
#pragma unroll
                            for (int x = 0; x < NG; x++) {
                                const bool ok = (uint32_t)(key[x] - k.x) < (uint32_t)k.y;
                                // (with a cap the mask goes on after it: a score of -inf there is -cap)
                                if (CAP) base[x][t][e] = ok ? base[x][t][e] : -INFINITY;
                                else sc[x][t][e] = ok ? sc[x][t][e] : -INFINITY;
                                ds[x][t][e] = ok ? ds[x][t][e] : 0.0f;
                            }
                        }
                }
                half4 gt[4][2], qt[4][2];
#pragma unroll
                for (int dt = 0; dt < 4; dt++)
#pragma unroll
                    for (int y = 0; y < 2; y++) {
                        gt[dt][y] = lds_read_tr16(st + 8192 + toff[dt] + 4096 * hf + 2048 * y);
                        qt[dt][y] = lds_read_tr16(st + toff[dt] + 4096 * hf + 2048 * y);
                    }
                if (hf == 1) {
                    __builtin_amdgcn_sched_barrier(0);
                    if (more) stage(kvh * p.each + hn, tn, (s + 1) & 1);
                    __builtin_amdgcn_sched_barrier(0);
                }
                half8 pf[NG], sf[NG];
#pragma unroll
                for (int x = 0; x < NG; x++) {
#pragma unroll
                    for (int t = 0; t < 2; t++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            float by = sigma;
                            if (CAP) {
                                const float r = __builtin_amdgcn_rcpf(fast_exp2(sc[x][t][e] * p.pre) + 1.0f);
                                sc[x][t][e] = fmaf(-2.0f * p.off, r, base[x][t][e]);
                                by = (4.0f * sigma) * fmaf(-r, r, r);
                            }
                            sc[x][t][e] = fast_exp2(CAP ? sc[x][t][e] + l4[t][e] : fmaf(sc[x][t][e], p.mul, l4[t][e]));
                            ds[x][t][e] *= sc[x][t][e];
                            if (CAP || !BF) ds[x][t][e] *= by;
                        }
                    pf[x] = pack8<BF>(sc[x][0], sc[x][1]);
                    sf[x] = pack8<BF>(ds[x][0], ds[x][1]);
                }
#pragma unroll
                for (int dt = 0; dt < 4; dt++) {
                    const half8 a = {gt[dt][0][0], gt[dt][0][1], gt[dt][0][2], gt[dt][0][3], gt[dt][1][0], gt[dt][1][1], gt[dt][1][2], gt[dt][1][3]};
                    const half8 c = {qt[dt][0][0], qt[dt][0][1], qt[dt][0][2], qt[dt][0][3], qt[dt][1][0], qt[dt][1][1], qt[dt][1][2], qt[dt][1][3]};
#pragma unroll
                    for (int x = 0; x < NG; x++) {
                        dv[x][dt] = mma<BF>(a, pf[x], dv[x][dt]);
                        dk[x][dt] = mma<BF>(c, sf[x], dk[x][dt]);
                    }
                }
            }
            hx = hn, tx = tn;
        }
    }

    const float back = p.scale / sigma;
#pragma unroll
    for (int x = 0; x < NG; x++) {
        bool bad = false;
#pragma unroll
        for (int dt = 0; dt < 4; dt++) {
            dk[x][dt] = dk[x][dt] * back;
#pragma unroll
            for (int e = 0; e < 4; e++) bad |= !(fabsf(dk[x][dt][e]) < INFINITY) || !(fabsf(dv[x][dt][e]) < INFINITY);
        }
        uint64_t again = __builtin_amdgcn_ballot_w64(bad && key[x] < p.nk);
        again = (again | again >> 32) & 0xffffffffull;
        again = (again | again >> 16) & 0xffffull;
        if (key[x] < p.nk && !((again >> r16) & 1)) {
            const int64_t at = (int64_t)key[x] * b.dkv_stride + kvh * 64 + 4 * g;
#pragma unroll
            for (int dt = 0; dt < 4; dt++) {
                *(half4*)(b.dk + at + 16 * dt) = pack4<BF>(dk[x][dt]);
                *(half4*)(b.dv + at + 16 * dt) = pack4<BF>(dv[x][dt]);
            }
        }
        // Rows whose sums are not finite again, over the queries that see the key alone (a row of q or
        // dO that does not may hold infinities or NaN). Lane l: dimension l.
        while (again) {
            const int y = __builtin_ctzll(again);
            again &= again - 1;
            const int j = kb + 64 * x + 16 * w + y;
            float ak = 0.0f, av = 0.0f;
            for (int sub = 0; sub < p.each; sub++) {
                const int h = kvh * p.each + sub;
                const float slope = BIAS == BIAS_SLOPES ? p.slopes[h] * p.unit : 0.0f;
                for (int i0 = 0; i0 < p.nq; i0 += 64) {
                    const int i = i0 + l;
                    float pw = 0.0f, da = 0.0f;
                    bool ok = false;
                    if (i < p.nq) {
                        const int2 r = b.range[i];
                        ok = (uint32_t)(j - r.x) < (uint32_t)r.y;
                        if (ok) grad_pair<BF, BIAS, CAP>(b, tab0 + sub * p.row, slope, h, kvh, i, j, pw, da);
                    }
                    uint64_t some = __builtin_amdgcn_ballot_w64(ok);
                    while (some) {
                        const int z = __builtin_ctzll(some);
                        some &= some - 1;
                        av = fmaf(__shfl(pw, z), widen<BF>(b.dout[(int64_t)(i0 + z) * b.do_stride + h * 64 + l]), av);
                        ak = fmaf(__shfl(da, z), widen<BF>(p.q[(int64_t)(i0 + z) * p.q_stride + h * 64 + l]), ak);
                    }
                }
            }
            const int64_t at = (int64_t)j * b.dkv_stride + kvh * 64 + l;
            b.dk[at] = pack2<BF>(ak * p.scale, 0.0f)[0];
            b.dv[at] = pack2<BF>(av, 0.0f)[0];
        }
    }
}

// ---- dQ of 64 queries, and the bias's gradient -------------------------------------------------
template <bool BF, int BIAS, bool CAP>
__global__ __launch_bounds__(256) void attn_bias_dq_kernel(BiasBack b) {
    const BiasParams& p = b.p;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int task = xcd_task(blockIdx.x, b.qt * p.heads);
    const int h = task / b.qt, tile = task % b.qt, q0 = 64 * tile, kvh = h / p.each;
    const int tid = threadIdx.x, l = tid & 63, r16 = l & 15, g = l >> 4;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int j4 = r16 >> 2, q4 = r16 & 3;
    const int dists = 2 * p.reach + 1;
    float* const tab0 = (float*)(lds + 32768);
    float* const hist = tab0 + p.row + w * dists;
    if (BIAS == BIAS_TABLE) {
        load_bias(p, h, 1, tab0, 256);
        for (int i = l; i < dists; i += 64) hist[i] = 0.0f;
    }
    const float sigma = BF ? 1.0f : grad_scale(b, kvh);

    const int4 bd = b.bounds[tile];
    const int k0 = bd.x, k1 = bd.y;
    const int row = q0 + 16 * w + r16, qi = min(row, p.nq - 1), qpos = p.q_first + row;
    const int wq0 = p.q_first + q0 + 16 * w, wql = wq0 + 15;
    const int2 kr = b.range[row];
    const int wlo = wave_min(kr.y ? kr.x : 0x7fffffff), whi = wave_max(kr.x + kr.y);
    const int flo = wave_max(kr.x), fhi = wave_min(row < p.nq ? kr.x + kr.y : 0x7fffffff);
    const float nl = b.nl[(size_t)h * b.nqp + row], dn = b.dn[(size_t)h * b.nqp + row];
    half8 qf[2], gf[2];
    {
        const f16* qp = p.q + (int64_t)qi * p.q_stride + h * 64 + 8 * g;
        const f16* gp = b.dout + (int64_t)qi * b.do_stride + h * 64 + 8 * g;
#pragma unroll
        for (int k2 = 0; k2 < 2; k2++) {
            qf[k2] = *(const half8*)(qp + 32 * k2), gf[k2] = *(const half8*)(gp + 32 * k2);
            if (row >= p.nq) qf[k2] = gf[k2] = half8{};
        }
    }
    const float slope = BIAS == BIAS_SLOPES ? p.slopes[h] * p.unit : 0.0f;
    const float* const tab = tab0 + p.reach + BIAS_PAD;
    __syncthreads();
    const float left = BIAS == BIAS_TABLE ? tab[-p.reach] : 0.0f, right = BIAS == BIAS_TABLE ? tab[p.reach] : 0.0f;
    float far_left = 0.0f, far_right = 0.0f;

    const int nblk = k1 > k0 ? (k1 - k0 + 63) >> 6 : 0;
    uint32_t doff[4];
#pragma unroll
    for (int x = 0; x < 4; x++) {
        const int c = ((w + 4 * x) & 7) * 64 + l, r = c >> 3, ch = (c & 7) ^ (r & 7);
        doff[x] = (uint32_t)(r * (int)p.kv_stride * 2 + ch * 16);
    }
    auto stage = [&](int bl, int st) {
        char* to = lds + st * 16384;
        const int kb = k0 + 64 * bl;
        const uint32_t bytes = (uint32_t)((min(k1 - kb, 64) - 1) * (int)p.kv_stride * 2 + 128);
        const auto rk = buffer_rsrc(p.k + (int64_t)kb * p.kv_stride + kvh * 64, bytes);
        const auto rv = buffer_rsrc(p.v + (int64_t)kb * p.kv_stride + kvh * 64, bytes);
#pragma unroll
        for (int x = 0; x < 4; x++)
            lds_bdma16<false>(x < 2 ? rk : rv, doff[x], to + (x < 2 ? 0 : 8192) + ((w + 4 * x) & 7) * 1024);
    };
    int koff[2], toff[4];
#pragma unroll
    for (int k2 = 0; k2 < 2; k2++) koff[k2] = att_swz(r16, 4 * k2 + g);
#pragma unroll
    for (int dt = 0; dt < 4; dt++) toff[dt] = att_swz(4 * g + j4, 2 * dt + (q4 >> 1)) + (q4 & 1) * 8;

    floatx4 dq[4];
#pragma unroll
    for (int t = 0; t < 4; t++) dq[t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    if (nblk > 0) stage(0, 0);
    for (int bl = 0; bl < nblk; bl++) {
        wait_vmcnt<0>();
        __builtin_amdgcn_s_barrier();
        const int kb = k0 + 64 * bl;
        const bool act = !(kb + 64 <= wlo || kb >= whi);
        const char* st = lds + (bl & 1) * 16384;
        const bool far = kb - wql >= p.reach || kb + 63 - wq0 <= -p.reach;  // (a table's)
        floatx4 base[4], sc[4], ds[4];
        half4 kt[2][4][2];
        if (act) {
#pragma unroll
            for (int t = 0; t < 4; t++) {
                if (BIAS == BIAS_TABLE) {
                    if (far) {
                        const float b0 = kb > wq0 ? right : left;
                        base[t] = floatx4{b0, b0, b0, b0};
                    } else {
                        const float* at = tab + (kb + 4 * g - qpos);
#pragma unroll
                        for (int e = 0; e < 4; e++) base[t][e] = at[16 * t + e];
                    }
                } else if (BIAS == BIAS_SLOPES) {
                    const float x = (float)(kb + 4 * g - qpos);
#pragma unroll
                    for (int e = 0; e < 4; e++) base[t][e] = fmaf(-slope, fabsf(x + (float)(16 * t + e)), p.off);
                } else {
                    const float y = CAP ? p.off : 0.0f;
                    base[t] = floatx4{y, y, y, y};
                }
                sc[t] = CAP ? floatx4{0.0f, 0.0f, 0.0f, 0.0f} : base[t];
                ds[t] = floatx4{dn, dn, dn, dn};
#pragma unroll
                for (int k2 = 0; k2 < 2; k2++) {
                    sc[t] = mma<BF>(*(const half8*)(st + koff[k2] + 2048 * t), qf[k2], sc[t]);
                    ds[t] = mma<BF>(*(const half8*)(st + 8192 + koff[k2] + 2048 * t), gf[k2], ds[t]);
                }
            }
#pragma unroll
            for (int hf = 0; hf < 2; hf++)
#pragma unroll
                for (int dt = 0; dt < 4; dt++)
#pragma unroll
                    for (int y = 0; y < 2; y++) kt[hf][dt][y] = lds_read_tr16(st + toff[dt] + 4096 * hf + 2048 * y);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (bl + 1 < nblk) stage(bl + 1, (bl + 1) & 1);
        __builtin_amdgcn_sched_barrier(0);
        if (!act) continue;
        if (!(kb >= flo && kb + 64 <= fhi)) {
            const int at = kb + 4 * g - kr.x;
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const bool ok = (uint32_t)(at + 16 * t + e) < (uint32_t)kr.y;
                    if (CAP) base[t][e] = ok ? base[t][e] : -INFINITY;
                    else sc[t][e] = ok ? sc[t][e] : -INFINITY;
                    ds[t][e] = ok ? ds[t][e] : 0.0f;
                }
        }
        // dS; `base` keeps the tanh's slope
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (CAP) {
                    const float r = __builtin_amdgcn_rcpf(fast_exp2(sc[t][e] * p.pre) + 1.0f);
                    sc[t][e] = fmaf(-2.0f * p.off, r, base[t][e]);
                    base[t][e] = (4.0f * sigma) * fmaf(-r, r, r);
                }
                ds[t][e] *= fast_exp2(CAP ? sc[t][e] + nl : fmaf(sc[t][e], p.mul, nl));
            }
        if (BIAS == BIAS_TABLE) {
            if (far) {
                float v = 0.0f;
#pragma unroll
                for (int t = 0; t < 4; t++) v += (ds[t][0] + ds[t][1]) + (ds[t][2] + ds[t][3]);
                if (kb > wq0) far_right += v;
                else far_left += v;
            } else {
                // diag[t], lane (r16, g): the sum at distance kb + 16 t + 4 g - (wq0 + r16). A lane's
                // e-th key is at its query's distance + e, which is the diagonal of the lane e to the
                // left: those that leave the 16 lanes belong to the next 16 keys' diagonals.
                float diag[5] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    diag[t] += ds[t][0];
                    diag[t] += dpp_move<0x101>(ds[t][1]);
                    diag[t] += dpp_move<0x102>(ds[t][2]);
                    diag[t] += dpp_move<0x103>(ds[t][3]);
                    diag[t + 1] += dpp_move<0x11F>(ds[t][1]);
                    diag[t + 1] += dpp_move<0x11E>(ds[t][2]);
                    diag[t + 1] += dpp_move<0x11D>(ds[t][3]);
                }
#pragma unroll
                for (int t = 0; t < 5; t++) {
                    const int d = kb + 16 * t + 4 * g - qpos;
                    far_left += d < -p.reach ? diag[t] : 0.0f;
                    far_right += d > p.reach ? diag[t] : 0.0f;
                    // (one group of 16 lanes after the other: distinct distances in each)
#pragma unroll
                    for (int y = 0; y < 4; y++)
                    {
                        if (g == y && d >= -p.reach && d <= p.reach) hist[d + p.reach] += diag[t];
                        __builtin_amdgcn_wave_barrier();
                    }
                }
            }
        }
        if (CAP || !BF) {
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) ds[t][e] *= CAP ? base[t][e] : sigma;
        }
#pragma unroll
        for (int hf = 0; hf < 2; hf++) {
            const half8 sf = pack8<BF>(ds[2 * hf], ds[2 * hf + 1]);
#pragma unroll
            for (int dt = 0; dt < 4; dt++) {
                const half4 lo = kt[hf][dt][0], hi = kt[hf][dt][1];
                const half8 kf = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                dq[dt] = mma<BF>(kf, sf, dq[dt]);
            }
        }
    }

    const float back = p.scale / sigma;
    bool bad = false;
#pragma unroll
    for (int dt = 0; dt < 4; dt++) {
        dq[dt] = dq[dt] * back;
#pragma unroll
        for (int e = 0; e < 4; e++) bad |= !(fabsf(dq[dt][e]) < INFINITY);
    }
    uint64_t again = __builtin_amdgcn_ballot_w64(bad && row < p.nq);
    again = (again | again >> 32) & 0xffffffffull;
    again = (again | again >> 16) & 0xffffull;
    if (row < p.nq && !((again >> r16) & 1)) {
        f16* to = b.dq + (int64_t)row * b.dq_stride + h * 64 + 4 * g;
#pragma unroll
        for (int dt = 0; dt < 4; dt++) *(half4*)(to + 16 * dt) = pack4<BF>(dq[dt]);
    }
    // (as in dK and dV: a row's gradient over the keys that it sees alone)
    while (again) {
        const int y = __builtin_ctzll(again);
        again &= again - 1;
        const int i = q0 + 16 * w + y;
        const int2 r = b.range[i];
        float acc = 0.0f;
        for (int j0 = r.x; j0 < r.x + r.y; j0 += 64) {
            float pw = 0.0f, da = 0.0f;
            const int n = min(64, r.x + r.y - j0);
            if (l < n) grad_pair<BF, BIAS, CAP>(b, tab0, slope, h, kvh, i, j0 + l, pw, da);
            for (int z = 0; z < n; z++)
                acc = fmaf(__shfl(da, z), widen<BF>(p.k[(int64_t)(j0 + z) * p.kv_stride + kvh * 64 + l]), acc);
        }
        b.dq[(int64_t)i * b.dq_stride + h * 64 + l] = pack2<BF>(acc * p.scale, 0.0f)[0];
    }

    if (BIAS == BIAS_TABLE) {
        far_left = wave_sum(far_left), far_right = wave_sum(far_right);
        if (l == 0) hist[0] += far_left;
        __builtin_amdgcn_wave_barrier();
        if (l == 0) hist[dists - 1] += far_right;
        __syncthreads();
        float* to = b.part + ((size_t)h * b.qt + tile) * dists;
        const float* from = tab0 + p.row;
        for (int i = tid; i < dists; i += 256)
            to[i] = (from[i] + from[dists + i]) + (from[2 * dists + i] + from[3 * dists + i]);
    }
}

// dtable[b][h]: the distances' sums over the tiles, in order, then those of each bucket.
__global__ __launch_bounds__(1024) void attn_bias_table_kernel(BiasBack b) {
    const int dists = 2 * b.p.reach + 1, h = blockIdx.x, tid = threadIdx.x;
    extern __shared__ float sums[];  // [4][dists], then their buckets
    int* const bucket = (int*)(sums + 4 * dists);
    const int part = tid >> 8, t0 = part * b.qt / 4, t1 = (part + 1) * b.qt / 4;
    for (int i = tid & 255; i < dists; i += 256) {
        const float* from = b.part + (size_t)h * b.qt * dists + i;
        float s = 0.0f;
        for (int t = t0; t < t1; t++) s += from[(size_t)t * dists];
        sums[part * dists + i] = s;
        if (part == 0) bucket[i] = min(max(b.p.bucket[i], 0), b.p.buckets - 1);
    }
    __syncthreads();
    for (int i = tid; i < dists; i += 1024)
        sums[i] = (sums[i] + sums[dists + i]) + (sums[2 * dists + i] + sums[3 * dists + i]);
    __syncthreads();
    for (int x = tid; x < b.p.buckets; x += 1024) {
        float s = 0.0f;
        for (int i = 0; i < dists; i++) s += bucket[i] == x ? sums[i] : 0.0f;
        b.dtable[(size_t)x * b.p.heads + h] = s;
    }
}

// ---- the host side ----------------------------------------------------------------------------
namespace {

[[noreturn]] void fail(const std::string& m) { throw std::runtime_error("attention_bias_backward: " + m); }

constexpr int NG = 2;  // key groups of 64 a block, dK and dV

// The workspace's parts, in floats, each on 256 bytes.
struct Layout {
    size_t nl, dn, range, bounds, max_do, max_v, part, all;
};

Layout layout(const AttnBias& a, int& nqp, int& pb) {
    nqp = (a.nq + 63) / 64 * 64;
    pb = (std::max(nqp, a.nk) + PREP_ROWS - 1) / PREP_ROWS;
    Layout y{};
    auto take = [&](size_t floats) {
        const size_t at = y.all;
        y.all += (floats + 63) / 64 * 64;
        return at;
    };
    y.nl = take((size_t)a.heads * nqp), y.dn = take((size_t)a.heads * nqp);
    y.range = take(2 * (size_t)nqp), y.bounds = take(4 * (size_t)(nqp / 64));
    y.max_do = take((size_t)a.heads * pb), y.max_v = take((size_t)a.kv_heads * pb);
    y.part = take(a.table ? (size_t)a.heads * (nqp / 64) * (2 * a.reach + 1) : 0);
    return y;
}

template <typename K>
void lds_limit(K kernel, int bytes) {
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess)
        fail("a kernel cannot have its LDS");
}

template <bool BF, int BIAS, bool CAP>
void launch(const BiasBack& b, hipStream_t st) {
    const BiasParams& p = b.p;
    static const bool ok = [] {
        lds_limit(attn_bias_dkv_kernel<BF, BIAS, CAP, NG>, 2 * GRAD_STAGE + 4 * BIAS_MAX_TABLE);
        lds_limit(attn_bias_dq_kernel<BF, BIAS, CAP>, 32768 + 4 * (bias_row(BIAS_MAX_REACH) + 4 * (2 * BIAS_MAX_REACH + 1)));
        return true;
    }();
    (void)ok;
    hipLaunchKernelGGL((attn_bias_rows_kernel<BF>), dim3(b.pb), dim3(256), 4 * (p.heads + p.kv_heads) * 4, st, b);
    const size_t tab = BIAS == BIAS_TABLE ? 4 * (size_t)p.row : 0;
    if (p.nk > 0)
        hipLaunchKernelGGL((attn_bias_dkv_kernel<BF, BIAS, CAP, NG>), dim3((p.nk + 64 * NG - 1) / (64 * NG) * p.kv_heads), dim3(256),
                           2 * GRAD_STAGE + p.each * tab, st, b);
    const int dists = 2 * p.reach + 1;
    if (p.nq > 0)
        hipLaunchKernelGGL((attn_bias_dq_kernel<BF, BIAS, CAP>), dim3(b.qt * p.heads), dim3(256),
                           32768 + tab + (BIAS == BIAS_TABLE ? 16 * (size_t)dists : 0), st, b);
    if (BIAS == BIAS_TABLE)
        hipLaunchKernelGGL(attn_bias_table_kernel, dim3(p.heads), dim3(1024), 20 * (size_t)dists, st, b);
}

template <bool BF>
void launch_type(const BiasBack& b, int bias, bool cap, hipStream_t st) {
    if (bias == BIAS_TABLE) cap ? launch<BF, BIAS_TABLE, true>(b, st) : launch<BF, BIAS_TABLE, false>(b, st);
    else if (bias == BIAS_SLOPES) cap ? launch<BF, BIAS_SLOPES, true>(b, st) : launch<BF, BIAS_SLOPES, false>(b, st);
    else cap ? launch<BF, BIAS_NONE, true>(b, st) : launch<BF, BIAS_NONE, false>(b, st);
}

}  // namespace

ScratchSize attn_bias_backward_scratch(const AttnBias& a, int) {
    int nqp, pb;
    return {layout(a, nqp, pb).all, 0};
}

void attn_bias_backward_launch(const AttnBias& a, const AttnBiasGrads& g, const Scratch& s, hipStream_t st) {
    attn_bias_check(a, &g);
    if (a.nq == 0 && a.nk == 0 && !g.dtable) return;
    BiasBack b{};
    const Layout y = layout(a, b.nqp, b.pb);
    if (y.all > s.ws_floats)
        fail("the scratch has " + std::to_string(s.ws_floats) + " floats, not " + std::to_string(y.all));
    b.p = bias_params(a);
    b.qt = b.nqp / 64;
    b.dout = (const f16*)g.dout, b.do_stride = g.do_stride;
    b.dq = (f16*)g.dq, b.dk = (f16*)g.dk, b.dv = (f16*)g.dv;
    b.dq_stride = g.dq_stride, b.dkv_stride = g.dkv_stride, b.dtable = g.dtable;
    b.nl = s.ws + y.nl, b.dn = s.ws + y.dn, b.range = (int2*)(s.ws + y.range), b.bounds = (int4*)(s.ws + y.bounds);
    b.max_do = s.ws + y.max_do, b.max_v = s.ws + y.max_v, b.part = s.ws + y.part;
    const int bias = a.table ? BIAS_TABLE : a.slopes ? BIAS_SLOPES : BIAS_NONE;
    if (b.pb > 0) a.bf16 ? launch_type<true>(b, bias, a.cap > 0.0f, st) : launch_type<false>(b, bias, a.cap > 0.0f, st);
    else hipLaunchKernelGGL(attn_bias_table_kernel, dim3(a.heads), dim3(1024), 20 * (2 * a.reach + 1), st, b);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) fail(hipGetErrorString(e));
}

}  // namespace jh
