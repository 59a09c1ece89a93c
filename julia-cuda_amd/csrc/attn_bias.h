// Attention whose scores may be capped by a tanh, get a bias that depends on the distance and are
// masked by a range of keys a query, with its gradients: what the host and the kernels share
// (attn_bias.hip: forward; attn_bias_back.h: backward). Heads of 64, f16 or bf16.
//
//   s_ij = a_ij + b(j - pos_i),  a_ij = scale q_i . k_j, or cap tanh(scale q_i . k_j / cap)
//   o_i  = sum_j exp(s_ij - lse_i) v_j over the keys that query i sees, lse_i = log sum_j exp(s_ij)
#pragma once

#include <hip/hip_runtime_api.h>
#include <stddef.h>
#include <stdint.h>

#include <atomic>

#include "kernels.h"

namespace jh {

// Lets a kernel have `bytes` of dynamic LDS on the current device, asked for once a device (`devices`: a
// bit each, the kernel's own).
bool dynamic_lds(std::atomic<uint64_t>& devices, const void* kernel, int bytes);

enum { BIAS_NONE = 0, BIAS_TABLE = 1, BIAS_SLOPES = 2 };

// What an attention computes (include/julia_hip.h, julia_hip_attention_bias_args).
struct AttnBias {
    int bf16;
    const jh_half *q, *k, *v;
    int64_t q_stride, kv_stride;  // elements between rows
    jh_half* o;
    int64_t o_stride;
    int nq, nk, heads, kv_heads, q_first;
    float scale, cap;
    const float* table;     // [buckets][heads]
    const int32_t* bucket;  // [2 reach + 1]
    int buckets, reach;
    const float* slopes;  // [heads]
    int window;
    const int32_t* span;  // [nq][2]
    float* lse;           // [heads][nq]
};

struct AttnBiasGrads {
    const jh_half* dout;
    int64_t do_stride;
    jh_half *dq, *dk, *dv;
    int64_t dq_stride, dkv_stride;
    float* dtable;  // [buckets][heads]
};

// A table's distances in LDS are padded by this much on either side with its end values, so that
// a 64-key block that reaches into [-reach, reach] for a wave's 16 queries needs no clamp (its
// distances go up to 78 past either end).
constexpr int BIAS_PAD = 80;
constexpr int BIAS_MAX_REACH = 512;
// LDS for the tables of the query heads that share a key head, in floats.
constexpr int BIAS_MAX_TABLE = 6000;
inline int bias_row(int reach) { return 2 * (reach + BIAS_PAD) + 1; }

struct ScratchSize {
    size_t floats, counters;
};

// Throws std::runtime_error when `a` (and `g`, for the backward pass) break what the kernels assume.
void attn_bias_check(const AttnBias& a, const AttnBiasGrads* g);
ScratchSize attn_bias_forward_scratch(const AttnBias& a, int cus);
ScratchSize attn_bias_backward_scratch(const AttnBias& a, int cus);
void attn_bias_launch(const AttnBias& a, const Scratch& s, hipStream_t stream);
void attn_bias_backward_launch(const AttnBias& a, const AttnBiasGrads& g, const Scratch& s, hipStream_t stream);

// Layer norm over rows of d values (norm.hip).
enum { NORM_F16 = 0, NORM_BF16 = 1, NORM_F32 = 2 };
constexpr int NORM_MAX_D = 8192;
struct Norm {
    int type, rows, d;
    const void* x;
    int64_t x_stride;
    const float* gamma;
    const float* beta;  // forward, nullable
    float eps;          // forward
    void* y;            // forward: the result; backward: dx
    int64_t y_stride;
    float* stats;  // [rows][2] (mean, 1 / sqrt(var + eps)): forward: written, nullable; backward: read
    const void* dy;
    int64_t dy_stride;
    float *dgamma, *dbeta;
};
void norm_check(const Norm& n, bool backward);
ScratchSize norm_scratch(int rows, int d, int cus);
void norm_launch(const Norm& n, hipStream_t stream);
void norm_backward_launch(const Norm& n, const Scratch& s, hipStream_t stream);

}  // namespace jh
