// The C ABI of the operators for encoders with relative positions and for their gradients
// (include/julia_hip.h, parts 2 and 3): the biased attention, layer norm, and the tables a program
// makes for them on the host.
#include <math.h>

#include <stdexcept>

#include "attn_bias.h"
#include "capi.h"

using namespace jh;

namespace {

AttnBias to_bias(const julia_hip_attention_bias_args* a) {
    if (!a) throw std::runtime_error("attention_bias: no arguments");
    if (a->type != JULIA_HIP_F16 && a->type != JULIA_HIP_BF16) throw std::runtime_error("attention_bias: f16 or bf16");
    AttnBias x{};
    x.bf16 = a->type == JULIA_HIP_BF16;
    x.q = (const jh_half*)a->q, x.k = (const jh_half*)a->k, x.v = (const jh_half*)a->v, x.o = (jh_half*)a->o;
    x.q_stride = a->q_stride, x.kv_stride = a->kv_stride, x.o_stride = a->o_stride;
    x.nq = a->nq, x.nk = a->nk, x.heads = a->heads, x.kv_heads = a->kv_heads, x.q_first = a->q_first;
    x.scale = a->scale, x.cap = a->cap;
    x.table = a->table, x.bucket = a->bucket, x.buckets = a->buckets, x.reach = a->reach;
    x.slopes = a->slopes, x.window = a->window, x.span = a->span, x.lse = a->lse;
    return x;
}

AttnBiasGrads to_grads(const julia_hip_attention_bias_grads* g) {
    if (!g) throw std::runtime_error("attention_bias_backward: no gradients");
    AttnBiasGrads x{};
    x.dout = (const jh_half*)g->dout, x.do_stride = g->do_stride;
    x.dq = (jh_half*)g->dq, x.dk = (jh_half*)g->dk, x.dv = (jh_half*)g->dv;
    x.dq_stride = g->dq_stride, x.dkv_stride = g->dkv_stride, x.dtable = g->dtable;
    return x;
}

Norm to_norm(int type, const void* x, int64_t x_stride, int rows, int d, const float* gamma, void* y, int64_t y_stride,
             float* stats) {
    Norm n{};
    n.type = type, n.rows = rows, n.d = d, n.x = x, n.x_stride = x_stride, n.gamma = gamma;
    n.y = y, n.y_stride = y_stride, n.stats = stats;
    return n;
}

}  // namespace

extern "C" {

int julia_hip_attention_bias_scratch(const julia_hip_attention_bias_args* a, int backward, size_t* ws_floats,
                                     size_t* counters, char* err, size_t err_len) {
    return guarded(err, err_len, [&] {
        if (!ws_floats || !counters) throw std::runtime_error("attention_bias: nowhere to put the sizes");
        const AttnBias x = to_bias(a);
        attn_bias_check(x, nullptr);
        const ScratchSize s = backward ? attn_bias_backward_scratch(x, device_cus()) : attn_bias_forward_scratch(x, device_cus());
        *ws_floats = s.floats, *counters = s.counters;
    });
}

int julia_hip_attention_bias_check(const julia_hip_attention_bias_args* a, const julia_hip_attention_bias_grads* g,
                                   char* err, size_t err_len) {
    return guarded(err, err_len, [&] {
        const AttnBias x = to_bias(a);
        if (g) {
            const AttnBiasGrads y = to_grads(g);
            attn_bias_check(x, &y);
        } else {
            attn_bias_check(x, nullptr);
        }
    });
}

int julia_hip_attention_bias(const julia_hip_attention_bias_args* a, const julia_hip_scratch* s, void* stream,
                             char* err, size_t err_len) {
    return guarded(err, err_len, [&] { attn_bias_launch(to_bias(a), scratch_of(s), (hipStream_t)stream); });
}

int julia_hip_attention_bias_backward(const julia_hip_attention_bias_args* a, const julia_hip_attention_bias_grads* g,
                                      const julia_hip_scratch* s, void* stream, char* err, size_t err_len) {
    return guarded(err, err_len, [&] {
        attn_bias_backward_launch(to_bias(a), to_grads(g), scratch_of(s), (hipStream_t)stream);
    });
}

int julia_hip_layer_norm(int type, const void* x, int64_t x_stride, int rows, int d, const float* gamma, const float* beta,
                         float eps, void* y, int64_t y_stride, float* stats, void* stream, char* err, size_t err_len) {
    return guarded(err, err_len, [&] {
        Norm n = to_norm(type, x, x_stride, rows, d, gamma, y, y_stride, stats);
        n.beta = beta, n.eps = eps;
        norm_launch(n, (hipStream_t)stream);
    });
}

int julia_hip_layer_norm_scratch(int rows, int d, size_t* ws_floats, size_t* counters, char* err, size_t err_len) {
    return guarded(err, err_len, [&] {
        if (!ws_floats || !counters) throw std::runtime_error("layer_norm: nowhere to put the sizes");
        const ScratchSize s = norm_scratch(rows, d, device_cus());
        *ws_floats = s.floats, *counters = s.counters;
    });
}

int julia_hip_layer_norm_backward(int type, const void* x, int64_t x_stride, const void* dy, int64_t dy_stride, int rows,
                                  int d, const float* gamma, const float* stats, void* dx, int64_t dx_stride,
                                  float* dgamma, float* dbeta, const julia_hip_scratch* s, void* stream, char* err,
                                  size_t err_len) {
    return guarded(err, err_len, [&] {
        Norm n = to_norm(type, x, x_stride, rows, d, gamma, dx, dx_stride, const_cast<float*>(stats));
        n.dy = dy, n.dy_stride = dy_stride, n.dgamma = dgamma, n.dbeta = dbeta;
        norm_backward_launch(n, scratch_of(s), (hipStream_t)stream);
    });
}

int julia_hip_prep_relative_buckets(int buckets, int max_distance, int both, int reach, int32_t* bucket, char* err,
                                    size_t err_len) {
    return guarded(err, err_len, [&] {
        auto fail = [](const char* m) { throw std::runtime_error(std::string("relative_buckets: ") + m); };
        if (!bucket) fail("nowhere to put them");
        if (reach < 0 || reach > BIAS_MAX_REACH) fail("the reach must be from 0 to 512");
        const int side = both ? buckets / 2 : buckets, exact = side / 2;
        if (buckets > 1024 || exact < 1 || (both && buckets % 2)) fail("at least 2 buckets a side, an even number for both sides, up to 1024");
        if (max_distance <= exact) fail("max_distance must be past the buckets of one distance each");
        for (int t = -reach; t <= reach; t++) {
            const int a = both ? abs(t) : t < 0 ? -t : 0;
            int b = a;
            if (a >= exact) {
                // (a distance on a range's border, where the quotient of the logarithms is whole, opens it)
                const double x = (side - exact) * log((double)a / exact) / log((double)max_distance / exact);
                b = std::min(side - 1, exact + (int)floor(x + 1e-9));
            }
            bucket[t + reach] = b + (both && t > 0 ? side : 0);
        }
    });
}

int julia_hip_prep_spans(const size_t* lens, const size_t* prefix, size_t documents, int32_t* span, char* err,
                         size_t err_len) {
    return guarded(err, err_len, [&] {
        size_t at = 0;
        if (documents && (!lens || !span)) throw std::runtime_error("spans: no lengths, or nowhere to put them");
        for (size_t d = 0; d < documents; d++) {
            if (lens[d] >= (size_t(1) << 30) || at + lens[d] >= (size_t(1) << 30)) throw std::runtime_error("spans: 2^30 rows or more");
            if (prefix && prefix[d] > lens[d]) throw std::runtime_error("spans: a prefix longer than its document");
            for (size_t i = 0; i < lens[d]; i++) {
                span[2 * (at + i)] = (int32_t)at;
                span[2 * (at + i) + 1] = (int32_t)(at + (prefix ? std::max(i + 1, prefix[d]) : lens[d]));
            }
            at += lens[d];
        }
    });
}

}  // extern "C"
