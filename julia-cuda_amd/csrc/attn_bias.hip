// The biased attention's forward pass (attn_bias.h). The tile is the streaming attention's
// (attn_tile.h): a block takes 16 NW rows of a key head, K and V go 64 keys at a time through two
// LDS stages, S^T = K . Q^T leaves a lane one query's scores, and O^T += V^T . P^T takes the weights
// straight from them.
//
// - A row is a (query, query head) pair: the heads that share a key head are neighbours, so a block
//   reads K and V once for all of them, and one token's heads fill a tile's rows.
// - Without a cap the bias is the MFMAs' initial accumulator, in units of 1 / scale: a table's values
//   are read from LDS into the accumulators at addresses that differ by constants (the table is
//   padded, so no distance is clamped), and blocks past `reach` on one side take one value.
// - Few rows and many keys: `chunks` blocks share a tile's keys; the last to arrive joins their
//   maxima, sums and outputs in order.
//
// Bound by the softmax's vector instructions: 8192 rows with slopes take 301 us (685 TFLOP/s, half of what a
// large f16 product reaches), 64 documents in 18752 rows with a table 57.6 (its bytes: 16).
#include <algorithm>
#include <cmath>
#include <limits>
#include <stdexcept>
#include <string>

#include "attn_bias_tile.h"

namespace jh {

constexpr int BIAS_STAGE = 16384;  // 64 keys: K, then V
constexpr int BIAS_CHUNKS = 16;    // blocks that share a tile's keys, at most

// (Four waves a SIMD without a cap: 128 registers. At three the batch took 63 us in place of 57.6; with the
// cap's operations 128 registers would spill.)
template <bool BF, int BIAS, bool CAP, int NW, int KS>
__global__ __launch_bounds__(64 * NW * KS, NW == 4 && !CAP ? 4 : 1) void attn_bias_kernel(BiasParams p) {
    // The two stages are arrays of their own, so that the compiler can tell a copy into one from the reads
    // of the other: in one array every LDS read waits for every copy in flight.
    __shared__ __attribute__((aligned(16))) char stage0[KS * BIAS_STAGE], stage1[KS * BIAS_STAGE];
    extern __shared__ __attribute__((aligned(16))) float tab0[];
    __shared__ uint32_t s_last, s_bad;
    constexpr int QB = 16 * NW, LOADS = 16 / NW;
    const int rows = p.nq * p.each;
    const Quotient ct = divide(xcd_task(blockIdx.x, gridDim.x), p.by_chunks), ht = divide(ct.q, p.by_tiles);
    const int chunk = ct.r, tile = ct.q, kvh = ht.q, r0 = ht.r * QB;
    const int tid = threadIdx.x, l = tid & 63, r16 = l & 15, g = l >> 4;
    const int wk = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int w = wk % NW, kg = wk / NW;
    const int j4 = r16 >> 2, q4 = r16 & 3;

    // The keys of the block's rows (lane l: row r0 + l), of this wave's 16 and of the lane's own.
    const int mine = r0 + l;
    const bool real = l < QB && mine < rows;
    KeyRange tr{0, 0};
    if (real) tr = key_range(p, divide(mine, p.by_each).q);
    const int row = r0 + 16 * w + r16;
    const Quotient qh = divide(min(row, rows - 1), p.by_each);
    const int qi = qh.q, hh = qh.r, h = kvh * p.each + hh;
    const int qpos = p.q_first + qi;
    const f16* const qp = p.q + (int64_t)qi * p.q_stride + h * 64;
    const half8 qf[2] = {*(const half8*)(qp + 8 * g), *(const half8*)(qp + 32 + 8 * g)};
    const KeyBounds kb_ = key_bounds(tr, real, w);
    const int k0 = kb_.k0, k1 = kb_.k1, wlo = kb_.lo, whi = kb_.hi, flo = kb_.flo, fhi = kb_.fhi;
    const KeyRange kr = {__shfl(tr.lo, 16 * w + r16), __shfl(tr.hi, 16 * w + r16)};
    const uint32_t kspan = (uint32_t)(kr.hi - kr.lo);
    const int wq0 = __builtin_amdgcn_readfirstlane(qpos), wql = __builtin_amdgcn_readlane(qpos, 15);
    const float slope = BIAS == BIAS_SLOPES ? p.slopes[h] * p.unit : 0.0f;
    const float* const tab = tab0 + (BIAS == BIAS_TABLE ? hh * p.row + p.reach + BIAS_PAD : 0);  // distance 0
    const int blocks = k1 > k0 ? (k1 - k0 + 63) >> 6 : 0;
    int c0 = 0, nblk = blocks;
    if (p.chunks > 1) {  // (blocks are below 2^24, chunks up to 256)
        c0 = (uint32_t)(chunk * blocks) / (uint32_t)p.chunks;
        nblk = (uint32_t)((chunk + 1) * blocks) / (uint32_t)p.chunks - c0;
    }

    uint32_t doff[LOADS];
#pragma unroll
    for (int qq = 0; qq < LOADS; qq++) {
        const int c = ((w + NW * qq) & 7) * 64 + l, r = c >> 3, ch = (c & 7) ^ (r & 7);
        doff[qq] = (uint32_t)(r * (int)p.kv_stride * 2 + ch * 16);
    }
    auto stage = [&](int b, char* dst) {
        const int kb = k0 + 64 * (c0 + b);
        const uint32_t bytes = (uint32_t)((min(k1 - kb, 64) - 1) * (int)p.kv_stride * 2 + 128);
        const auto rk = buffer_rsrc(p.k + (int64_t)kb * p.kv_stride + kvh * 64, bytes);
        const auto rv = buffer_rsrc(p.v + (int64_t)kb * p.kv_stride + kvh * 64, bytes);
#pragma unroll
        for (int qq = 0; qq < LOADS; qq++) {
            const bool kk = qq < LOADS / 2;
            const int I = (w + NW * qq) & 7;
            lds_bdma16<false>(kk ? rk : rv, doff[qq], dst + (kk ? 0 : 8192) + I * 1024);
        }
    };

    int koff[2], voff[4];
#pragma unroll
    for (int k2 = 0; k2 < 2; k2++) koff[k2] = att_swz(r16, 4 * k2 + g);
#pragma unroll
    for (int dt = 0; dt < 4; dt++) voff[dt] = 8192 + att_swz(4 * g + j4, 2 * dt + (q4 >> 1)) + (q4 & 1) * 8;

    // exp2(fma(score, mul, -(max mul))) scales all weights by two to the rounding of max mul, which the
    // sum takes off again: nothing while |max mul| is up to 2^20. Past that (every key of a row has a
    // bias like the type's lowest value) `big` blocks subtract first.
    float top, mx, neg, sum;
    bool big;
    floatx4 o[4];

    float left = 0.0f, right = 0.0f;  // a table's ends
    const int nsteps = (nblk + KS - 1) / KS;
    auto has = [&](int b) { return kg + KS * b < nblk; };
    auto step = [&](int b, auto st_, auto careful_) __attribute__((always_inline)) {
        constexpr int ST = decltype(st_)::value;
        constexpr bool careful = decltype(careful_)::value;  // (the second time over the keys)
        stage_barrier<0>();
        const int kb = k0 + 64 * (c0 + kg + KS * b);
        const bool act = has(b) && !(kb + 64 <= wlo || kb >= whi);
        const char* st = (ST ? stage1 : stage0) + kg * BIAS_STAGE;
        if (has(b + 1)) stage(kg + KS * (b + 1), (ST ? stage0 : stage1) + kg * BIAS_STAGE);
        if (!act) return;
        floatx4 sc[4], base[4];  // (base: the scores' initial values; with a cap, what is added after it)
        half4 vlo[2][4], vhi[2][4];
        auto columns = [&](int hf, int dt) {
            vlo[hf][dt] = lds_read_tr16(st + voff[dt] + 4096 * hf);
            vhi[hf][dt] = lds_read_tr16(st + voff[dt] + 4096 * hf + 2048);
        };
        {
            block_bias<BIAS>(p, tab, left, right, slope, kb, g, qpos, wq0, wql, base);
            half8 kf[4][2];
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int k2 = 0; k2 < 2; k2++) kf[t][k2] = *(const half8*)(st + koff[k2] + 2048 * t);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int t = 0; t < 4; t++) {
                sc[t] = CAP ? floatx4{0.0f, 0.0f, 0.0f, 0.0f} : base[t];
#pragma unroll
                for (int k2 = 0; k2 < 2; k2++) sc[t] = mma<BF>(kf[t][k2], qf[k2], sc[t]);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int hf = 0; hf < 2; hf++)
#pragma unroll
                for (int dt = 0; dt < 4; dt++)
                    if (!careful) columns(hf, dt);
        }
        if (CAP) cap_scores<4, false>(p, sc, base, 1.0f);
        if (!(kb >= flo && kb + 64 <= fhi)) {
            const int at = kb + 4 * g - kr.lo;
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    sc[t][e] = (uint32_t)(at + 16 * t + e) < kspan ? sc[t][e] : -INFINITY;
        }
#pragma unroll
        for (int t = 0; t < 4; t++) asm volatile("" : "+v"(sc[t]));
        float bm = -INFINITY;
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) bm = fmaxf(bm, sc[t][e]);
        const float mul = CAP ? 1.0f : p.mul;
        if (__builtin_amdgcn_ballot_w64(bm > top) != 0) {
            top = fmaxf(top, max_xor32(max_xor16(bm)));
            const float m = top * mul, b0 = m == -INFINITY ? 0.0f : m;
            const float alpha = fast_exp2(mx - b0);
            mx = m;
            neg = -b0;
            if (!CAP) big = __builtin_amdgcn_ballot_w64(fabsf(b0) > 1048576.0f) != 0;
            sum *= alpha;
#pragma unroll
            for (int dt = 0; dt < 4; dt++) o[dt] = o[dt] * alpha;
        }
        float rs = 0.0f;
        if (!CAP && big) {
            const float from = top == -INFINITY ? 0.0f : top;
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) sc[t][e] = (sc[t][e] - from) * mul;
        } else {
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) sc[t][e] = CAP ? sc[t][e] + neg : fmaf(sc[t][e], mul, neg);
        }
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                sc[t][e] = fast_exp2(sc[t][e]);
                rs += sc[t][e];
            }
        sum += rs;
        const bool by_pair = careful && !(kb >= flo && kb + 64 <= fhi);
#pragma unroll
        for (int hf = 0; hf < 2; hf++) {
            const half8 pf = pack8<BF>(sc[2 * hf], sc[2 * hf + 1]);
            const uintx4 pairs = by_pair ? seen_pairs([&](int c) { return (uint32_t)(kb + 32 * hf + c - kr.lo) < kspan; }) : uintx4{};
#pragma unroll
            for (int dt = 0; dt < 4; dt++) {
                if (careful) columns(hf, dt);
                const half4 lo = vlo[hf][dt], hi = vhi[hf][dt];
                const half8 vf = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                o[dt] = by_pair ? careful_mma<BF, false>(vf, pf, pairs, o[dt]) : mma<BF>(vf, pf, o[dt]);
            }
        }
    };
    if (tid == 0) s_bad = 0;
    auto all_keys = [&](auto careful) __attribute__((always_inline)) {
        top = mx = -INFINITY, neg = sum = 0.0f, big = false;
#pragma unroll
        for (int t = 0; t < 4; t++) o[t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        // (the first copy goes out ahead of the table's two dependent loads)
        if (has(0)) stage(kg, stage0 + kg * BIAS_STAGE);
        if (BIAS == BIAS_TABLE && !careful) {
            load_bias(p, kvh * p.each, p.each, tab0, 64 * NW * KS);
            __syncthreads();
            left = tab[-p.reach], right = tab[p.reach];
        }
        for (int b = 0; b < nsteps; b += 2) {
            step(b, std::integral_constant<int, 0>{}, careful);
            if (b + 1 < nsteps) step(b + 1, std::integral_constant<int, 1>{}, careful);
        }
    };
    all_keys(std::false_type{});
    // Sums that are not finite: a V that a row does not see may have made them so. Again, with the blocks
    // that have masked pairs pair by pair (code of its own: as a branch of the first loop it cost that 15 %).
    if (!(finite4(o[0]) && finite4(o[1]) && finite4(o[2]) && finite4(o[3])) && row < rows) s_bad = 1;
    __syncthreads();
    if (__builtin_expect(__builtin_amdgcn_readfirstlane(s_bad), 0)) all_keys(std::true_type{});

    // The key groups' maxima, sums and outputs, through LDS to group 0, in group order.
    auto merge = [&](float mk, float sk, const floatx4 (&ok)[4]) {
        const float m = fmaxf(mx, mk), base = m == -INFINITY ? 0.0f : m;
        const float a = fast_exp2(mx - base), b = fast_exp2(mk - base);
        mx = m;
        sum = sum * a + sk * b;
#pragma unroll
        for (int dt = 0; dt < 4; dt++) o[dt] = o[dt] * a + ok[dt] * b;
    };
    auto merge_groups = [&]() {
        if (KS == 1) return;
        __syncthreads();
        if (kg > 0) {
            float* mg = (float*)stage0 + ((kg - 1) * NW + w) * 18 * 64;
            mg[16 * 64 + l] = mx;
            mg[17 * 64 + l] = sum;
#pragma unroll
            for (int f = 0; f < 16; f++) mg[f * 64 + l] = o[f >> 2][f & 3];
        }
        __syncthreads();
        if (kg == 0)
            for (int k = 1; k < KS; k++) {
                const float* mg = (const float*)stage0 + ((k - 1) * NW + w) * 18 * 64;
                floatx4 ok[4];
#pragma unroll
                for (int f = 0; f < 16; f++) ok[f >> 2][f & 3] = mg[f * 64 + l];
                merge(mg[16 * 64 + l], mg[17 * 64 + l], ok);
            }
    };
    merge_groups();
    if (NW == 1 && p.chunks > 1) {
        // A chunk's part: a lane's outputs as four 16-byte pieces, its maximum and its sum; the lanes of rows
        // that there are. The last block's waves load all of their chunks' parts at once.
        constexpr uint32_t PART = 18 * 64 * NW * 4;
        constexpr int AT_ONCE = BIAS_CHUNKS / KS;
        const auto slots = buffer_rsrc(p.ws + (size_t)tile * p.chunks * (PART / 4), PART * p.chunks);
        const uint32_t lane16 = (w * 64 + l) * 16, lane8 = 64 * NW * 64 + (w * 64 + l) * 8;
        const bool real = row < rows;
        if (kg == 0) {
            if (real) {
                const uint32_t at = PART * chunk;
#pragma unroll
                for (int dt = 0; dt < 4; dt++)
                    bstore16f(slots, at + dt * 1024 * NW + lane16, make_float4(o[dt][0], o[dt][1], o[dt][2], o[dt][3]));
                bstore8(slots, at + lane8, make_float2(mx, sum));
            }
            release_wait();
        }
        __syncthreads();
        if (tid == 0) {
            const uint32_t last = atomic_add_agent(p.counters + tile, 1u) == (uint32_t)(p.chunks - 1);
            if (last) atomic_store_agent(p.counters + tile, 0u);
            s_last = last;
        }
        __syncthreads();
        if (s_last == 0) return;
        mx = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int dt = 0; dt < 4; dt++) o[dt] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        if (real)
            for (int z = kg; z < p.chunks; z += AT_ONCE * KS) {
                float4 part[AT_ONCE][4];
                float2 ms[AT_ONCE];
#pragma unroll
                for (int x = 0; x < AT_ONCE; x++) {
                    const uint32_t at = PART * min(z + x * KS, p.chunks - 1);
#pragma unroll
                    for (int dt = 0; dt < 4; dt++) part[x][dt] = bload16f(slots, at + dt * 1024 * NW + lane16);
                    ms[x] = bload8<true>(slots, at + lane8);
                }
#pragma unroll
                for (int x = 0; x < AT_ONCE; x++) {
                    if (z + x * KS >= p.chunks) break;
                    floatx4 ok[4];
#pragma unroll
                    for (int dt = 0; dt < 4; dt++) ok[dt] = floatx4{part[x][dt].x, part[x][dt].y, part[x][dt].z, part[x][dt].w};
                    merge(ms[x].x, ms[x].y, ok);
                }
            }
        merge_groups();
    }
    if (kg > 0) return;

    const float total = sum_xor32(sum_xor16(sum));
    const float inv = total > 0.0f || total != total ? 1.0f / total : 0.0f;
    if (row < rows) {
        f16* op = p.o + (int64_t)qi * p.o_stride + h * 64 + 4 * g;
#pragma unroll
        for (int dt = 0; dt < 4; dt++) *(half4*)(op + 16 * dt) = pack4<BF>(o[dt] * inv);
        if (p.lse && g == 0)
            p.lse[(size_t)h * p.nq + qi] =
                total > 0.0f || total != total ? (mx + __builtin_amdgcn_logf(total)) * 0.69314718055994531f : -INFINITY;
    }
}

// ---- the host side ----------------------------------------------------------------------------
namespace {

[[noreturn]] void fail(const std::string& m) { throw std::runtime_error("attention_bias: " + m); }

bool aligned(const void* p, size_t to) { return (uintptr_t)p % to == 0; }

void check_rows(const char* what, const void* p, int64_t stride, int width) {
    if (!p || !aligned(p, 16)) fail(std::string(what) + " must be a 16-byte aligned device address");
    if (stride < width || stride % 8 || stride > (1 << 22))
        fail(std::string(what) + " rows of " + std::to_string(width) + " cannot be " + std::to_string(stride) +
             " apart (a multiple of 8 up to 2^22)");
}

}  // namespace

bool dynamic_lds(std::atomic<uint64_t>& devices, const void* kernel, int bytes) {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return false;
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (devices.load(std::memory_order_relaxed) & bit) return true;
    if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess) return false;
    devices.fetch_or(bit, std::memory_order_relaxed);
    return true;
}

void attn_bias_check(const AttnBias& a, const AttnBiasGrads* g) {
    if (a.nq < 0 || a.nk < 0 || a.nq > (1 << 24) || a.nk >= (1 << 30)) fail("a bad number of queries or keys");
    if (a.heads < 1 || a.heads > 256 || a.kv_heads < 1 || a.heads % a.kv_heads)
        fail(std::to_string(a.heads) + " heads cannot share " + std::to_string(a.kv_heads) + " key heads (up to 256 heads)");
    const int each = a.heads / a.kv_heads;
    if ((int64_t)a.nq * a.heads > (1 << 30)) fail("more than 2^30 rows of heads");
    if ((int64_t)a.nk * a.kv_heads > (1 << 30)) fail("more than 2^30 keys of heads");
    if (a.q_first < 0 || a.q_first >= (1 << 30)) fail("q_first must be from 0 to 2^30");
    if (!(a.scale >= 1e-6f && a.scale <= 1e6f)) fail("the scale must be from 1e-6 to 1e6");
    if (!(a.cap == 0.0f || (a.cap >= 1e-3f && a.cap <= 1e6f))) fail("the cap must be 0 or from 1e-3 to 1e6");
    if (a.cap > 0.0f && a.scale > 1e3f * a.cap) fail("the scale must be up to 1000 caps");
    if (a.window < 0 || a.window >= (1 << 30)) fail("the window must be from 0 to 2^30");
    if (a.table && a.slopes) fail("a bias table or slopes, not both");
    if (a.table) {
        if (!a.bucket) fail("a bias table needs its buckets");
        if (a.buckets < 1 || a.buckets > 1024) fail("1 to 1024 buckets");
        if (a.reach < 0 || a.reach > BIAS_MAX_REACH) fail("the table's reach must be up to " + std::to_string(BIAS_MAX_REACH));
        if (each * bias_row(a.reach) > BIAS_MAX_TABLE)
            fail("the table of " + std::to_string(each) + " heads to a key head is too long for a reach of " + std::to_string(a.reach));
        if (!aligned(a.table, 4) || !aligned(a.bucket, 4)) fail("the table and its buckets must be 4-byte aligned");
    }
    if (a.slopes && !aligned(a.slopes, 4)) fail("the slopes must be 4-byte aligned");
    if (a.span && !aligned(a.span, 8)) fail("span must be 8-byte aligned");
    if (a.nq > 0) {
        check_rows("q", a.q, a.q_stride, 64 * a.heads);
        check_rows("o", a.o, a.o_stride, 64 * a.heads);
        if (a.nk > 0) {
            check_rows("k", a.k, a.kv_stride, 64 * a.kv_heads);
            check_rows("v", a.v, a.kv_stride, 64 * a.kv_heads);
        }
        if (a.lse && !aligned(a.lse, 4)) fail("lse must be 4-byte aligned");
    }
    if (!g) return;
    if (a.nq > 0 && !a.lse) fail("the gradients need lse of the forward pass");
    if (a.nq > 0) {
        check_rows("dout", g->dout, g->do_stride, 64 * a.heads);
        check_rows("dq", g->dq, g->dq_stride, 64 * a.heads);
    }
    if (a.nk > 0) {
        check_rows("k", a.k, a.kv_stride, 64 * a.kv_heads);
        check_rows("v", a.v, a.kv_stride, 64 * a.kv_heads);
        check_rows("dk", g->dk, g->dkv_stride, 64 * a.kv_heads);
        check_rows("dv", g->dv, g->dkv_stride, 64 * a.kv_heads);
    }
    if ((g->dtable != nullptr) != (a.table != nullptr)) fail("dtable goes with a table");
    if (g->dtable && !aligned(g->dtable, 4)) fail("dtable must be 4-byte aligned");
}

BiasParams bias_params(const AttnBias& a) {
    const double log2e = 1.4426950408889634;
    BiasParams p{};
    p.q = (const f16*)a.q, p.k = (const f16*)a.k, p.v = (const f16*)a.v, p.o = (f16*)a.o;
    p.q_stride = a.q_stride, p.kv_stride = a.kv_stride, p.o_stride = a.o_stride;
    p.nq = a.nq, p.nk = a.nk, p.heads = a.heads, p.kv_heads = a.kv_heads, p.each = a.heads / a.kv_heads;
    p.by_each = Div(p.each);
    p.q_first = a.q_first, p.scale = a.scale;
    if (a.cap > 0.0f) {
        p.mul = 1.0f, p.unit = (float)log2e, p.off = (float)(a.cap * log2e), p.pre = (float)(2.0 * log2e * a.scale / a.cap);
        // tanh(x) / x over 0 <= x^2 <= 1/4 by a polynomial of x^2 with the least relative error
        // (a weighted least squares fit over Chebyshev points, reweighted until it is level: 1.3e-8)
        const double c[5] = {0.9999999868719406, -0.3333306939409053, 0.13324779312866444, -0.05298607478007015, 0.01713500531796541};
        const double x = (double)a.scale / a.cap;  // of q . k
        for (int i = 0; i < 5; i++) p.poly[i] = (float)(c[i] * a.cap * log2e * pow(x, 2 * i + 1));
        p.small = (float)(0.5 / x), p.per_off = (float)(1.0 / (a.cap * log2e));
    } else
        p.mul = (float)(a.scale * log2e), p.unit = (float)(1.0 / a.scale), p.off = 0.0f, p.pre = 0.0f;
    p.table = a.table, p.bucket = a.bucket, p.buckets = a.buckets, p.reach = a.reach, p.row = a.table ? bias_row(a.reach) : 0;
    p.slopes = a.slopes, p.window = a.window, p.span = a.span, p.lse = a.lse;
    p.chunks = 1;
    return p;
}

namespace {

// The tile of a forward call: 16 NW rows a block, KS key groups, `chunks` blocks a tile.
struct BiasPlan {
    int nw, ks, chunks;
    long tiles;
};

// Key groups while the grid is small (MI355X, d = 768, us; nw x ks): 293 rows 1x4 6.2, 2x4 6.4; 448 rows
// 2x4 6.9, 4x4 8.3, 4x1 9.0; 600 rows 2x4 8.2; 1024 rows 4x4 12.4, 4x2 13.5, 4x1 16.3; 2029 rows 4x2 33.4,
// 4x1 36.4; 2900 rows 4x1 56.7, 4x2 62.7.
BiasPlan bias_plan(const AttnBias& a, int cus) {
    const long rows = (long)a.nq * (a.heads / a.kv_heads);
    const long t16 = (rows + 15) / 16 * a.kv_heads, t32 = (rows + 31) / 32 * a.kv_heads, t64 = (rows + 63) / 64 * a.kv_heads;
    if (t16 > cus) {
        if (t32 <= cus) return {2, 4, 1, t32};
        return {4, t64 <= cus ? 4 : t64 <= 2L * cus ? 2 : 1, 1, t64};
    }
    // a block for every 256 keys at most, and few enough that their arrivals at the tile's counter, one
    // after the other, cost less than their keys (one row, 4 key heads: 8192 keys in 32 chunks 11.9 us, in
    // 16 9.6, in 8 11.0; 16384 keys in 64 16.8, in 32 12.3, in 16 12.0)
    const long most = std::max(1L, std::min({(a.nk + 255L) / 256, (long)cus / std::max(1L, t16), (long)BIAS_CHUNKS}));
    return {1, 4, (int)most, t16};
}

template <bool BF, int BIAS, bool CAP, int NW, int KS>
void launch_tile(const BiasParams& p, long tiles, hipStream_t st) {
    static std::atomic<uint64_t> devices{0};
    if (!dynamic_lds(devices, reinterpret_cast<const void*>(attn_bias_kernel<BF, BIAS, CAP, NW, KS>), 4 * BIAS_MAX_TABLE))
        fail("the kernel cannot have its LDS");
    const size_t lds = BIAS == BIAS_TABLE ? 4 * (size_t)p.each * p.row : 0;
    hipLaunchKernelGGL((attn_bias_kernel<BF, BIAS, CAP, NW, KS>), dim3((unsigned)(tiles * p.chunks)), dim3(64 * NW * KS), lds, st, p);
}

template <bool BF, int BIAS, bool CAP>
void launch_plan(const BiasParams& p, const BiasPlan& plan, hipStream_t st) {
    if (plan.nw == 1) launch_tile<BF, BIAS, CAP, 1, 4>(p, plan.tiles, st);
    else if (plan.nw == 2) launch_tile<BF, BIAS, CAP, 2, 4>(p, plan.tiles, st);
    else if (plan.ks == 4) launch_tile<BF, BIAS, CAP, 4, 4>(p, plan.tiles, st);
    else if (plan.ks == 2) launch_tile<BF, BIAS, CAP, 4, 2>(p, plan.tiles, st);
    else launch_tile<BF, BIAS, CAP, 4, 1>(p, plan.tiles, st);
}

template <bool BF>
void launch_type(const BiasParams& p, const BiasPlan& plan, int bias, bool cap, hipStream_t st) {
    if (bias == BIAS_TABLE) cap ? launch_plan<BF, BIAS_TABLE, true>(p, plan, st) : launch_plan<BF, BIAS_TABLE, false>(p, plan, st);
    else if (bias == BIAS_SLOPES) cap ? launch_plan<BF, BIAS_SLOPES, true>(p, plan, st) : launch_plan<BF, BIAS_SLOPES, false>(p, plan, st);
    else cap ? launch_plan<BF, BIAS_NONE, true>(p, plan, st) : launch_plan<BF, BIAS_NONE, false>(p, plan, st);
}

size_t plan_floats(const BiasPlan& plan) { return plan.chunks > 1 ? (size_t)plan.tiles * plan.chunks * 18 * 64 * plan.nw : 0; }

}  // namespace

ScratchSize attn_bias_forward_scratch(const AttnBias& a, int cus) {
    const BiasPlan plan = bias_plan(a, cus);
    return {plan_floats(plan), plan.chunks > 1 ? (size_t)plan.tiles : 0};
}

void attn_bias_launch(const AttnBias& a, const Scratch& s, hipStream_t st) {
    attn_bias_check(a, nullptr);
    if (a.nq == 0) return;
    const int cus = device_cus();
    const BiasPlan plan = bias_plan(a, cus);
    const ScratchSize need = attn_bias_forward_scratch(a, cus);
    if (need.floats > s.ws_floats || need.counters > s.n_counters)
        fail("the scratch has " + std::to_string(s.ws_floats) + " floats and " + std::to_string(s.n_counters) + " counters, not " +
             std::to_string(need.floats) + " and " + std::to_string(need.counters));
    BiasParams p = bias_params(a);
    p.by_tiles = Div((uint32_t)(plan.tiles / a.kv_heads)), p.by_chunks = Div(plan.chunks);
    p.chunks = plan.chunks, p.ws = s.ws, p.counters = s.counters;
    const int bias = a.table ? BIAS_TABLE : a.slopes ? BIAS_SLOPES : BIAS_NONE;
    a.bf16 ? launch_type<true>(p, plan, bias, a.cap > 0.0f, st) : launch_type<false>(p, plan, bias, a.cap > 0.0f, st);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) fail(hipGetErrorString(e));
}

}  // namespace jh
