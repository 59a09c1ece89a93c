// Layer norm over rows of d values, forward and backward (attn_bias.h, Norm), in f16, bf16 or f32 with
// 32-bit statistics and weights:
//   y = (x - mean) rstd gamma + beta,  rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   dx = rstd (g - mean(g) - xh mean(g xh)),  g = dy gamma,  xh = (x - mean) rstd
//   dgamma = the sum over rows of dy xh,  dbeta = of dy.
#include <algorithm>
#include <stdexcept>
#include <string>

#include "attn_bias_tile.h"

namespace jh {

struct NormParams {
    const void *x, *dy;
    void* y;
    int64_t x_stride, dy_stride, y_stride;
    const float *gamma, *beta;
    float* stats;
    float* part;  // [blocks][2][d]
    int rows, d;
    float eps, inv_d;
};

// Four consecutive values of a row, in 32 bits: f16, bf16 (T = 0, 1: 8 bytes) or f32 (16 bytes). VEC:
// the rows are aligned to that and d is a multiple of four; otherwise one by one, zeros past d.
template <int T, bool VEC>
__device__ __forceinline__ floatx4 norm_load(const void* row, int c, int d) {
    if (VEC) {
        if (T == NORM_F32) return *(const floatx4*)((const float*)row + c);
        const half4 v = *(const half4*)((const f16*)row + c);
        return floatx4{widen<T == NORM_BF16>(v[0]), widen<T == NORM_BF16>(v[1]), widen<T == NORM_BF16>(v[2]), widen<T == NORM_BF16>(v[3])};
    }
    floatx4 r = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (c + e < d) r[e] = T == NORM_F32 ? ((const float*)row)[c + e] : widen<T == NORM_BF16>(((const f16*)row)[c + e]);
    return r;
}

template <int T, bool VEC>
__device__ __forceinline__ void norm_store(void* row, int c, int d, floatx4 v) {
    if (VEC) {
        if (T == NORM_F32) *(floatx4*)((float*)row + c) = v;
        else *(half4*)((f16*)row + c) = pack4<T == NORM_BF16>(v);
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (c + e < d) {
            if (T == NORM_F32) ((float*)row)[c + e] = v[e];
            else ((f16*)row)[c + e] = pack2<T == NORM_BF16>(v[e], v[e])[0];
        }
}

template <int T>
__device__ __forceinline__ const void* norm_row(const void* base, int64_t at) {
    return (const char*)base + at * (T == NORM_F32 ? 4 : 2);
}

// The sums of W waves' values, to all of their lanes (W == 1: no barrier).
template <int W>
__device__ __forceinline__ float2 norm_sums(float a, float b, float2* sm) {
    a = wave_sum(a), b = wave_sum(b);
    if (W == 1) return make_float2(a, b);
    __syncthreads();  // (the last sums have been read)
    if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = make_float2(a, b);
    __syncthreads();
    float2 s = sm[0];
#pragma unroll
    for (int w = 1; w < W; w++) s.x += sm[w].x, s.y += sm[w].y;
    return s;
}

// A row by W waves (1, four rows a block; or 4), NC chunks of four values a lane.
template <int T, bool VEC, int W, int NC>
__global__ __launch_bounds__(256) void norm_kernel(NormParams p) {
    __shared__ float2 sm[4];
    const int lane = W == 1 ? threadIdx.x & 63 : threadIdx.x;
    const int row = W == 1 ? blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
    if (row >= p.rows) return;  // (whole waves; with W = 4 never)
    const void* x = norm_row<T>(p.x, row * p.x_stride);
    floatx4 v[NC];
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < NC; j++) {
        const int c = 4 * (lane + 64 * W * j);
        v[j] = c < p.d ? norm_load<T, VEC>(x, c, p.d) : floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        s += (v[j][0] + v[j][1]) + (v[j][2] + v[j][3]);
    }
    const float mean = norm_sums<W>(s, 0.0f, sm).x * p.inv_d;
    float q = 0.0f;
#pragma unroll
    for (int j = 0; j < NC; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int c = 4 * (lane + 64 * W * j) + e;
            v[j][e] -= mean;
            q += c < p.d ? v[j][e] * v[j][e] : 0.0f;
        }
    const float rstd = 1.0f / sqrtf(norm_sums<W>(q, 0.0f, sm).x * p.inv_d + p.eps);
    void* y = const_cast<void*>(norm_row<T>(p.y, row * p.y_stride));
#pragma unroll
    for (int j = 0; j < NC; j++) {
        const int c = 4 * (lane + 64 * W * j);
        if (c < p.d) {
            floatx4 o = v[j] * rstd * norm_load<NORM_F32, VEC>(p.gamma, c, p.d);
            if (p.beta) o += norm_load<NORM_F32, VEC>(p.beta, c, p.d);
            norm_store<T, VEC>(y, c, p.d, o);
        }
    }
    if (p.stats && lane == 0) *(float2*)(p.stats + 2 * (size_t)row) = make_float2(mean, rstd);
}

// Rows blockIdx.x, + gridDim.x, ... (W = 4) or four of them at a time (W = 1); a lane's columns stay
// its own, so its shares of dgamma and dbeta stay in registers until the block's are written.
template <int T, bool VEC, int W, int NC>
__global__ __launch_bounds__(256) void norm_back_kernel(NormParams p) {
    extern __shared__ float red[];
    __shared__ float2 sm[4];
    const int lane = W == 1 ? threadIdx.x & 63 : threadIdx.x;
    const int wave = threadIdx.x >> 6;
    floatx4 dg[NC], db[NC], gm[NC];
#pragma unroll
    for (int j = 0; j < NC; j++) {
        const int c = 4 * (lane + 64 * W * j);
        dg[j] = db[j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        gm[j] = c < p.d ? norm_load<NORM_F32, VEC>(p.gamma, c, p.d) : floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const int step = gridDim.x * (W == 1 ? 4 : 1);
    for (int row = W == 1 ? blockIdx.x * 4 + wave : blockIdx.x; row < p.rows; row += step) {
        const void *x = norm_row<T>(p.x, row * p.x_stride), *dy = norm_row<T>(p.dy, row * p.dy_stride);
        const float2 st = *(const float2*)(p.stats + 2 * (size_t)row);
        floatx4 xh[NC], g[NC];
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int j = 0; j < NC; j++) {
            const int c = 4 * (lane + 64 * W * j);
            xh[j] = g[j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
            if (c < p.d) xh[j] = norm_load<T, VEC>(x, c, p.d), g[j] = norm_load<T, VEC>(dy, c, p.d);
        }
#pragma unroll
        for (int j = 0; j < NC; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int c = 4 * (lane + 64 * W * j) + e;
                xh[j][e] = c < p.d ? (xh[j][e] - st.x) * st.y : 0.0f;
                dg[j][e] = fmaf(g[j][e], xh[j][e], dg[j][e]);
                db[j][e] += g[j][e];
                g[j][e] *= gm[j][e];
                s1 += g[j][e];
                s2 = fmaf(g[j][e], xh[j][e], s2);
            }
        const float2 s = norm_sums<W>(s1, s2, sm);
        const float m1 = s.x * p.inv_d, m2 = s.y * p.inv_d;
        void* dx = const_cast<void*>(norm_row<T>(p.y, row * p.y_stride));
#pragma unroll
        for (int j = 0; j < NC; j++) {
            const int c = 4 * (lane + 64 * W * j);
            if (c < p.d) norm_store<T, VEC>(dx, c, p.d, st.y * (g[j] - m1 - xh[j] * m2));
        }
    }
    float* part = p.part + (size_t)blockIdx.x * 2 * p.d;
    if (W == 1) {  // the four waves' shares, through LDS
#pragma unroll
        for (int j = 0; j < NC; j++) {
            *(floatx4*)(red + ((wave * 2 + 0) * NC + j) * 256 + 4 * lane) = dg[j];
            *(floatx4*)(red + ((wave * 2 + 1) * NC + j) * 256 + 4 * lane) = db[j];
        }
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * NC * 64; i += 256) {
            const int l = i & 63, j = (i >> 6) % NC, which = (i >> 6) / NC, c = 4 * (l + 64 * j);
            floatx4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < 4; w++) v += *(const floatx4*)(red + ((w * 2 + which) * NC + j) * 256 + 4 * l);
            if (c < p.d) norm_store<NORM_F32, VEC>(part + which * p.d, c, p.d, v);
        }
    } else {
#pragma unroll
        for (int j = 0; j < NC; j++) {
            const int c = 4 * (lane + 256 * j);
            if (c < p.d) {
                norm_store<NORM_F32, VEC>(part, c, p.d, dg[j]);
                norm_store<NORM_F32, VEC>(part + p.d, c, p.d, db[j]);
            }
        }
    }
}

// The blocks' shares of 64 columns of dgamma and dbeta end to end, summed in order.
__global__ __launch_bounds__(1024) void norm_sum_kernel(const float* part, int blocks, int d, float* dgamma, float* dbeta) {
    __shared__ float sm[16][64];
    const int l = threadIdx.x & 63, w = threadIdx.x >> 6, c = blockIdx.x * 64 + l;
    float s = 0.0f;
    if (c < 2 * d)
        for (int b = w; b < blocks; b += 16) s += part[(size_t)b * 2 * d + c];
    sm[w][l] = s;
    __syncthreads();
    if (w == 0 && c < 2 * d) {
#pragma unroll
        for (int i = 1; i < 16; i++) s += sm[i][l];
        if (c < d) dgamma[c] = s;
        else if (dbeta) dbeta[c - d] = s;
    }
}

// ---- the host side ----------------------------------------------------------------------------
namespace {

[[noreturn]] void fail(const std::string& m) { throw std::runtime_error("layer_norm: " + m); }

void check_rows(const char* what, const void* p, int64_t stride, const Norm& n) {
    if (!p || (uintptr_t)p % (n.type == NORM_F32 ? 4 : 2)) fail(std::string(what) + " must be a device address aligned to its type");
    if (stride < n.d || stride > (int64_t(1) << 40)) fail(std::string(what) + " rows of " + std::to_string(n.d) + " cannot be " + std::to_string(stride) + " apart");
}

int norm_blocks(int rows, int d, int cus) {
    const long work = d <= 2048 ? (rows + 3) / 4 : rows;  // (a block's rows at a time)
    return (int)std::max(1L, std::min(work, 2L * cus));
}

NormParams norm_params(const Norm& n) {
    NormParams p{};
    p.x = n.x, p.dy = n.dy, p.y = n.y, p.x_stride = n.x_stride, p.dy_stride = n.dy_stride, p.y_stride = n.y_stride;
    p.gamma = n.gamma, p.beta = n.beta, p.stats = n.stats, p.rows = n.rows, p.d = n.d, p.eps = n.eps;
    p.inv_d = (float)(1.0 / n.d);
    return p;
}

template <int T, bool VEC, int W, int NC>
void run(const NormParams& p, bool back, int blocks, hipStream_t st) {
    if (back) {
        const size_t lds = W == 1 ? (size_t)8 * NC * 256 * 4 : 0;
        hipLaunchKernelGGL((norm_back_kernel<T, VEC, W, NC>), dim3(blocks), dim3(256), lds, st, p);
    } else {
        hipLaunchKernelGGL((norm_kernel<T, VEC, W, NC>), dim3(W == 1 ? (p.rows + 3) / 4 : p.rows), dim3(256), 0, st, p);
    }
}

template <int T, bool VEC>
void run_width(const NormParams& p, bool back, int blocks, hipStream_t st) {
    const int c = (p.d + 255) / 256;  // chunks of a wave's lane
    if (c <= 1) run<T, VEC, 1, 1>(p, back, blocks, st);
    else if (c <= 2) run<T, VEC, 1, 2>(p, back, blocks, st);
    else if (c <= 3) run<T, VEC, 1, 3>(p, back, blocks, st);
    else if (c <= 4) run<T, VEC, 1, 4>(p, back, blocks, st);
    else if (c <= 6) run<T, VEC, 1, 6>(p, back, blocks, st);
    else if (c <= 8) run<T, VEC, 1, 8>(p, back, blocks, st);
    else if (c <= 16) run<T, VEC, 4, 4>(p, back, blocks, st);
    else run<T, VEC, 4, 8>(p, back, blocks, st);
}

void run_type(const Norm& n, const NormParams& p, bool back, int blocks, hipStream_t st) {
    const size_t to = n.type == NORM_F32 ? 16 : 8;
    auto fits = [&](const void* a, int64_t stride) { return !a || ((uintptr_t)a % to == 0 && stride % 4 == 0); };
    const bool vec = n.d % 4 == 0 && fits(p.x, p.x_stride) && fits(p.y, p.y_stride) && fits(p.dy, p.dy_stride) &&
                     (uintptr_t)p.gamma % 16 == 0 && (uintptr_t)p.beta % 16 == 0;
    if (n.type == NORM_F32) vec ? run_width<NORM_F32, true>(p, back, blocks, st) : run_width<NORM_F32, false>(p, back, blocks, st);
    else if (n.type == NORM_BF16) vec ? run_width<NORM_BF16, true>(p, back, blocks, st) : run_width<NORM_BF16, false>(p, back, blocks, st);
    else vec ? run_width<NORM_F16, true>(p, back, blocks, st) : run_width<NORM_F16, false>(p, back, blocks, st);
}

void check_launch() {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) fail(hipGetErrorString(e));
}

}  // namespace

void norm_check(const Norm& n, bool back) {
    if (n.type != NORM_F16 && n.type != NORM_BF16 && n.type != NORM_F32) fail("unknown type " + std::to_string(n.type));
    if (n.rows < 0 || n.rows > (1 << 28)) fail("a bad number of rows");
    if (n.d < 1 || n.d > NORM_MAX_D) fail("rows of " + std::to_string(n.d) + " values (1 to " + std::to_string(NORM_MAX_D) + ")");
    if (back) {
        if (!n.dgamma || (uintptr_t)n.dgamma % 4 || (uintptr_t)n.dbeta % 4) fail("dgamma and dbeta must be 4-byte aligned, dgamma not null");
    } else if (!(n.eps >= 0.0f && n.eps < 1e30f)) {
        fail("eps must be 0 or more");
    }
    if (n.rows == 0) return;
    check_rows("x", n.x, n.x_stride, n);
    check_rows(back ? "dx" : "y", n.y, n.y_stride, n);
    if (!n.gamma || (uintptr_t)n.gamma % 4 || (uintptr_t)n.beta % 4) fail("gamma and beta must be 4-byte aligned, gamma not null");
    if ((uintptr_t)n.stats % 8 || (back && !n.stats)) fail("stats must be 8-byte aligned, and not null for the gradients");
    if (back) check_rows("dy", n.dy, n.dy_stride, n);
}

ScratchSize norm_scratch(int rows, int d, int cus) {
    if (rows < 0 || d < 1 || d > NORM_MAX_D) fail("bad sizes");
    return {(size_t)norm_blocks(rows, d, cus) * 2 * d, 0};
}

void norm_launch(const Norm& n, hipStream_t st) {
    norm_check(n, false);
    if (n.rows == 0) return;
    run_type(n, norm_params(n), false, 0, st);
    check_launch();
}

void norm_backward_launch(const Norm& n, const Scratch& s, hipStream_t st) {
    norm_check(n, true);
    const int blocks = n.rows == 0 ? 0 : norm_blocks(n.rows, n.d, device_cus());
    if ((size_t)blocks * 2 * n.d > s.ws_floats)
        fail("the scratch has " + std::to_string(s.ws_floats) + " floats, not " + std::to_string((size_t)blocks * 2 * n.d));
    NormParams p = norm_params(n);
    p.part = s.ws;
    if (blocks) run_type(n, p, true, blocks, st);
    hipLaunchKernelGGL(norm_sum_kernel, dim3((2 * n.d + 63) / 64), dim3(1024), 0, st, p.part, blocks, n.d, n.dgamma, n.dbeta);
    check_launch();
}

}  // namespace jh
