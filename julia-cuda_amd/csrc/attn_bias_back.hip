// The biased attention's gradients (attn_bias_back.h): the plan, the workspace and the f16 kernels.
#include "attn_bias_back.h"

namespace jh {

namespace {

// More groups to a block, and smaller blocks, while the grid is about a block a CU or less (MI355X, d =
// 768, us for the whole pass with the other launch as it is; nw x ks for dQ, ng x nw x ks for dK and dV):
//    448 rows  dQ 2x4 20.3, 4x1 25.1, 1x4 26.2             dK, dV 1x2x4 25.2, 1x4x2 27.5, 2x4x1 33.2
//   1024 rows  dQ 4x2 45.8, 4x4 46.9, 4x1 52.8             dK, dV 2x2x4 45.5, 1x4x2 47.1, 2x4x1 59.0
//   1345 rows  dQ 4x1 86.0, 4x2 89.7                       dK, dV 2x4x2 74.1, 2x2x4 81.7, 2x4x1 85.4
//   2029 rows  dQ 4x1 120, 4x2 123                         dK, dV 2x4x2 102, 2x2x4 111, 2x4x1 120
//   2029 rows, prefix, capped, 4 key heads: dQ 4x2 115, 4x1 126;  dK, dV 1x2x4 128, 2x2x4 154, 2x4x1 286
//   64 documents in 18752 rows: dQ 4x1 203, 4x2 264        dK, dV 2x4x1 205, 1x4x1 234, 2x4x2 241
// (dQ's groups need rows of distances to the table's reach in LDS.)
GradPlan grad_plan(const AttnBias& a, int cus) {
    const long q16 = (long)(a.nq + 15) / 16 * a.heads, q32 = (long)(a.nq + 31) / 32 * a.heads, q64 = (long)(a.nq + 63) / 64 * a.heads;
    const long k16 = (long)(a.nk + 15) / 16 * a.kv_heads;
    GradPlan y{4, 1, 2, 4, 1};
    auto room = [&](int nw, int ks) { return 2 * ks * DQ_STAGE + (a.table ? dq_lds(a.reach, nw, ks) : 0) <= LDS_BYTES; };
    if (q16 <= cus && room(1, 4)) y.dq_nw = 1, y.dq_ks = 4;
    else if (q32 <= cus && room(2, 4)) y.dq_nw = 2, y.dq_ks = 4;
    else if (2 * q64 <= 3L * cus && room(4, 2)) y.dq_ks = 2;
    if (k16 <= cus) y.ng = 1, y.nw = 1, y.ks = 4;
    else if (k16 <= 2L * cus) y.ng = 1, y.nw = 2, y.ks = 4;
    else if (k16 <= 3L * cus) y.nw = 2, y.ks = 4;
    else if (k16 <= 8L * cus) y.ks = 2;
    return y;
}

// The workspace's parts, in floats, each on 256 bytes.
struct Layout {
    size_t info, bounds, max_do, part, all;
    int nqp, tiles;
};

Layout layout(const AttnBias& a, const GradPlan& plan) {
    Layout y{};
    y.nqp = (a.nq + 63) / 64 * 64;
    y.tiles = y.nqp / (16 * plan.dq_nw);
    auto take = [&](size_t floats) {
        const size_t at = y.all;
        y.all += (floats + 63) / 64 * 64;
        return at;
    };
    y.info = take(4 * (size_t)a.heads * y.nqp), y.bounds = take(4 * (size_t)y.tiles);
    y.max_do = take((size_t)a.heads * (y.nqp / 16));
    y.part = take(a.table ? (size_t)a.heads * y.tiles * (2 * a.reach + 1) : 0);
    return y;
}

}  // namespace

ScratchSize attn_bias_backward_scratch(const AttnBias& a, int cus) {
    return {layout(a, grad_plan(a, cus)).all, 0};
}

void attn_bias_backward_launch(const AttnBias& a, const AttnBiasGrads& g, const Scratch& s, hipStream_t st) {
    attn_bias_check(a, &g);
    const GradPlan plan = grad_plan(a, device_cus());
    const Layout y = layout(a, plan);
    if (y.all > s.ws_floats) grad_fail("the scratch has " + std::to_string(s.ws_floats) + " floats, not " + std::to_string(y.all));
    BiasBack b{};
    b.p = bias_params(a);
    b.nqp = y.nqp, b.tiles = y.tiles, b.per = 4 / plan.dq_nw;
    b.dout = (const f16*)g.dout, b.do_stride = g.do_stride;
    b.dq = (f16*)g.dq, b.dk = (f16*)g.dk, b.dv = (f16*)g.dv;
    b.dq_stride = g.dq_stride, b.dkv_stride = g.dkv_stride, b.dtable = g.dtable;
    b.info = s.ws + y.info, b.bounds = (int4*)(s.ws + y.bounds);
    b.max_do = s.ws + y.max_do, b.part = s.ws + y.part;
    const int bias = a.table ? BIAS_TABLE : a.slopes ? BIAS_SLOPES : BIAS_NONE;
    (a.bf16 ? grad_launch_bf16 : grad_launch<false>)(b, plan, bias, a.cap > 0.0f, st);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) grad_fail(hipGetErrorString(e));
}

}  // namespace jh
