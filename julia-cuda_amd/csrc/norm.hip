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

// Up to NORM_ONE_ROWS rows the gradients take one launch of up to NORM_ONE_LAUNCH blocks.
constexpr int NORM_ONE_ROWS = 512, NORM_ONE_LAUNCH = 16;

struct NormParams {
    const void *x, *dy;
    void* y;
    int64_t x_stride, dy_stride, y_stride;
    const float *gamma, *beta;
    float* stats;
    float* part;  // [blocks][2][d]
    float *dgamma, *dbeta;
    uint32_t* counter;
    int rows, d;
    float eps, inv_d;
};

// E consecutive values of a row as they lie: 16 bytes (eight f16 or bf16, four f32), or four of 16 bits. VEC:
// rows are aligned to that and d is a multiple of E; otherwise four, one by one, zeros past d.
template <int T, int E, bool VEC>
struct NormChunk {
    static constexpr bool BF = T == NORM_BF16;
    floatx4 f;  // (f32, or one by one)
    half8 h;
    __device__ __forceinline__ void load(const void* row, int c, int d) {
        if (!VEC) {
#pragma unroll
            for (int e = 0; e < 4; e++)
                f[e] = c + e >= d ? 0.0f : T == NORM_F32 ? ((const float*)row)[c + e] : widen<BF>(((const f16*)row)[c + e]);
        } else if (T == NORM_F32) {
            f = *(const floatx4*)((const float*)row + c);
        } else if (E == 8) {
            h = *(const half8*)((const f16*)row + c);
        } else {
            const half4 v = *(const half4*)((const f16*)row + c);
            h = half8{v[0], v[1], v[2], v[3]};
        }
    }
    __device__ __forceinline__ void clear() { f = floatx4{}, h = half8{}; }
    __device__ __forceinline__ float operator[](int e) const { return !VEC || T == NORM_F32 ? f[e & 3] : widen<BF>(h[e]); }
};

template <int T, int E, bool VEC>
__device__ __forceinline__ void norm_store(void* row, int c, int d, const float (&v)[E]) {
    constexpr bool BF = T == NORM_BF16;
    if (!VEC) {
#pragma unroll
        for (int e = 0; e < E; e++)
            if (c + e < d) {
                if (T == NORM_F32) ((float*)row)[c + e] = v[e];
                else ((f16*)row)[c + e] = pack2<BF>(v[e], v[e])[0];
            }
    } else if (T == NORM_F32) {
        *(floatx4*)((float*)row + c) = floatx4{v[0], v[1], v[2], v[3]};
    } else if (E == 8) {
        *(half8*)((f16*)row + c) = pack8<BF>(floatx4{v[0], v[1], v[2], v[3]}, floatx4{v[E - 4], v[E - 3], v[E - 2], v[E - 1]});
    } else {
        *(half4*)((f16*)row + c) = pack4<BF>(floatx4{v[0], v[1], v[2], v[3]});
    }
}

// E of gamma or beta.
template <int E, bool VEC>
__device__ __forceinline__ void norm_weights(const float* w, int c, int d, float (&v)[E]) {
#pragma unroll
    for (int q = 0; q < E / 4; q++) {
        NormChunk<NORM_F32, 4, VEC> x;
        x.load(w, c + 4 * q, d);
#pragma unroll
        for (int e = 0; e < 4; e++) v[4 * q + e] = x[e];
    }
}

template <int T>
__device__ __forceinline__ const void* norm_row(const void* base, int64_t at) {
    return (const char*)base + at * (T == NORM_F32 ? 4 : 2);
}

// The sums over the LR lanes of a row, or (LR = 256) the block's four waves.
template <int LR>
__device__ __forceinline__ float2 norm_sums(float a, float b, float2* sm) {
    a = group_sum<(LR < 64 ? LR : 64)>(a), b = group_sum<(LR < 64 ? LR : 64)>(b);
    if (LR <= 64) return make_float2(a, b);
    __syncthreads();  // (the last sums have been read)
    if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = make_float2(a, b);
    __syncthreads();
    float2 s = sm[0];
#pragma unroll
    for (int w = 1; w < 4; w++) s.x += sm[w].x, s.y += sm[w].y;
    return s;
}

// LR lanes a row, NC chunks a lane, R rows to those lanes: their loads go out together, and gamma and
// beta, in 32 bits twice a row's bytes, are read once for them.
template <int T, int E, bool VEC, int LR, int NC, int R>
__global__ __launch_bounds__(256) void norm_kernel(NormParams p) {
    __shared__ float2 sm[4];
    const int lane = threadIdx.x % LR;
    const int row0 = (blockIdx.x * (256 / LR) + threadIdx.x / LR) * R;
    NormChunk<T, E, VEC> x[R][NC];
#pragma unroll
    for (int r = 0; r < R; r++) {
        const void* from = norm_row<T>(p.x, min(row0 + r, p.rows - 1) * p.x_stride);
#pragma unroll
        for (int j = 0; j < NC; j++) {
            const int c = E * (lane + LR * j);
            if (c < p.d) x[r][j].load(from, c, p.d);
            else x[r][j].clear();
        }
    }
    float gm[NC][E], bt[NC][E];
#pragma unroll
    for (int j = 0; j < NC; j++) {
        const int c = E * (lane + LR * j);
#pragma unroll
        for (int e = 0; e < E; e++) gm[j][e] = bt[j][e] = 0.0f;
        if (c < p.d) {
            norm_weights<E, VEC>(p.gamma, c, p.d, gm[j]);
            if (p.beta) norm_weights<E, VEC>(p.beta, c, p.d, bt[j]);
        }
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int row = row0 + r;
        float v[NC][E], s = 0.0f, q = 0.0f;
#pragma unroll
        for (int j = 0; j < NC; j++)
#pragma unroll
            for (int e = 0; e < E; e++) s += v[j][e] = x[r][j][e];
        const float mean = norm_sums<LR>(s, 0.0f, sm).x * p.inv_d;
#pragma unroll
        for (int j = 0; j < NC; j++)
#pragma unroll
            for (int e = 0; e < E; e++) {
                v[j][e] -= mean;
                q += E * (lane + LR * j) + e < p.d ? v[j][e] * v[j][e] : 0.0f;
            }
        const float rstd = 1.0f / sqrtf(norm_sums<LR>(q, 0.0f, sm).x * p.inv_d + p.eps);
        if (row >= p.rows) continue;  // (LR = 256 has one row, which there is)
        void* to = const_cast<void*>(norm_row<T>(p.y, row * p.y_stride));
#pragma unroll
        for (int j = 0; j < NC; j++) {
            const int c = E * (lane + LR * j);
#pragma unroll
            for (int e = 0; e < E; e++) v[j][e] = fmaf(v[j][e] * rstd, gm[j][e], bt[j][e]);
            if (c < p.d) norm_store<T, E, VEC>(to, c, p.d, v[j]);
        }
        if (p.stats && lane == 0) *(float2*)(p.stats + 2 * (size_t)row) = make_float2(mean, rstd);
    }
}

// A column's sum over the blocks' shares is its dgamma, or its dbeta past d.
__device__ __forceinline__ void norm_column(const NormParams& p, int c, float s) {
    if (c < p.d) p.dgamma[c] = s;
    else if (p.dbeta) p.dbeta[c - p.d] = s;
}

// Rows blockIdx.x (512 / LR) + ..., + gridDim.x (512 / LR), ...: a lane's columns stay its own, so its shares of
// dgamma and dbeta stay in registers until the block's are written. The next row's loads go out ahead of
// this one's arithmetic. ONE: the last block to arrive sums the shares (a few blocks); else norm_sum_kernel.
template <int T, int E, bool VEC, int LR, int NC>
__global__ __launch_bounds__(LR == 256 ? 256 : 512) void norm_back_kernel(NormParams p, int one) {
    extern __shared__ float red[];  // [waves][2][d], or the columns' sums
    __shared__ float2 sm[4];
    __shared__ uint32_t s_last;
    constexpr int THREADS = LR == 256 ? 256 : 512, GROUPS = THREADS / LR;
    const int lane = threadIdx.x % LR;
    float dg[NC][E], db[NC][E], gm[NC][E];
#pragma unroll
    for (int j = 0; j < NC; j++) {
        const int c = E * (lane + LR * j);
#pragma unroll
        for (int e = 0; e < E; e++) dg[j][e] = db[j][e] = gm[j][e] = 0.0f;
        if (c < p.d) norm_weights<E, VEC>(p.gamma, c, p.d, gm[j]);
    }
    NormChunk<T, E, VEC> x[NC], g[NC];
    float2 st;
    auto load = [&](int row) {
        row = min(row, p.rows - 1);
        const void *xr = norm_row<T>(p.x, row * p.x_stride), *gr = norm_row<T>(p.dy, row * p.dy_stride);
        st = *(const float2*)(p.stats + 2 * (size_t)row);
#pragma unroll
        for (int j = 0; j < NC; j++) {
            const int c = E * (lane + LR * j);
            if (c < p.d) x[j].load(xr, c, p.d), g[j].load(gr, c, p.d);
            else x[j].clear(), g[j].clear();
        }
    };
    const int step = gridDim.x * GROUPS, first = blockIdx.x * GROUPS + threadIdx.x / LR;
    const int turns = first / GROUPS * GROUPS < p.rows ? (p.rows - first / GROUPS * GROUPS + step - 1) / step : 0;  // (the block's)
    if (turns > 0) load(first);
    for (int t = 0; t < turns; t++) {
        const int row = first + t * step;
        const bool real = row < p.rows;
        float xh[NC][E], gy[NC][E], s1 = 0.0f, s2 = 0.0f;
        const float rstd = st.y;
#pragma unroll
        for (int j = 0; j < NC; j++)
#pragma unroll
            for (int e = 0; e < E; e++) {
                const bool in = real && E * (lane + LR * j) + e < p.d;
                xh[j][e] = in ? (x[j][e] - st.x) * rstd : 0.0f;
                const float v = in ? g[j][e] : 0.0f;
                dg[j][e] = fmaf(v, xh[j][e], dg[j][e]);
                db[j][e] += v;
                gy[j][e] = v * gm[j][e];
                s1 += gy[j][e];
                s2 = fmaf(gy[j][e], xh[j][e], s2);
            }
        if (t + 1 < turns) load(row + step);
        const float2 s = norm_sums<LR>(s1, s2, sm);
        const float m1 = s.x * p.inv_d, m2 = s.y * p.inv_d;
        if (real) {
            void* dx = const_cast<void*>(norm_row<T>(p.y, row * p.y_stride));
#pragma unroll
            for (int j = 0; j < NC; j++) {
                const int c = E * (lane + LR * j);
#pragma unroll
                for (int e = 0; e < E; e++) gy[j][e] = rstd * (gy[j][e] - m1 - xh[j][e] * m2);
                if (c < p.d) norm_store<T, E, VEC>(dx, c, p.d, gy[j]);
            }
        }
    }
    // The block's shares: of the rows side by side in a wave by lane swaps, of the waves through LDS.
    float* part = p.part + (size_t)blockIdx.x * 2 * p.d;
    const int wave = threadIdx.x >> 6, waves = LR == 256 ? 1 : THREADS / 64;
#pragma unroll
    for (int j = 0; j < NC; j++)
#pragma unroll
        for (int e = 0; e < E; e++) {
            if (LR <= 8) dg[j][e] += __shfl_xor(dg[j][e], 8), db[j][e] += __shfl_xor(db[j][e], 8);
            if (LR <= 16) dg[j][e] = sum_xor16(dg[j][e]), db[j][e] = sum_xor16(db[j][e]);
            if (LR <= 32) dg[j][e] = sum_xor32(dg[j][e]), db[j][e] = sum_xor32(db[j][e]);
        }
    if (LR == 256 || (threadIdx.x & 63) < LR) {
        float* to = red + (LR == 256 ? 0 : wave * 2 * p.d);
#pragma unroll
        for (int j = 0; j < NC; j++)
#pragma unroll
            for (int e = 0; e < E; e++) {
                const int c = E * (lane + LR * j) + e;
                if (c < p.d) to[c] = dg[j][e], to[p.d + c] = db[j][e];
            }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * p.d; c += THREADS) {
        float s = red[c];
        for (int w = 1; w < waves; w++) s += red[w * 2 * p.d + c];
        if (gridDim.x == 1) norm_column(p, c, s);
        else if (one) xstore32(part + c, s);
        else part[c] = s;
    }
    if (!one || gridDim.x == 1) return;
    release_wait();
    __syncthreads();
    if (threadIdx.x == 0) {
        const uint32_t last = atomic_add_agent(p.counter, 1u) == gridDim.x - 1;
        if (last) atomic_store_agent(p.counter, 0u);
        s_last = last;
    }
    __syncthreads();
    if (s_last == 0) return;
    for (int c = threadIdx.x; c < 2 * p.d; c += THREADS) {
        float v[NORM_ONE_LAUNCH], s = 0.0f;
#pragma unroll
        for (int b = 0; b < NORM_ONE_LAUNCH; b++) v[b] = xload32(p.part + (size_t)min(b, (int)gridDim.x - 1) * 2 * p.d + c);
#pragma unroll
        for (int b = 0; b < NORM_ONE_LAUNCH; b++) s += b < (int)gridDim.x ? v[b] : 0.0f;
        norm_column(p, c, s);
    }
}

// 32 columns a block: its 32 half waves take every 32nd share each, and join in order.
__global__ __launch_bounds__(1024) void norm_sum_kernel(NormParams p, int blocks) {
    __shared__ float sm[1024];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31);
    float s = 0.0f;
    if (c < 2 * p.d)
#pragma unroll 8
        for (int b = threadIdx.x >> 5; b < blocks; b += 32) s += p.part[(size_t)b * 2 * p.d + c];
    sm[threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.x < 32 && c < 2 * p.d) {
        for (int i = 1; i < 32; i++) s += sm[32 * i + threadIdx.x];
        norm_column(p, c, s);
    }
}

// ---- the host side ----------------------------------------------------------------------------
namespace {

[[noreturn]] void fail(const std::string& m) { throw std::runtime_error("layer_norm: " + m); }

void check_rows(const char* what, const void* p, int64_t stride, const Norm& n) {
    if (!p || (uintptr_t)p % (n.type == NORM_F32 ? 4 : 2)) fail(std::string(what) + " must be a device address aligned to its type");
    if (stride < n.d || stride > (int64_t(1) << 40)) fail(std::string(what) + " rows of " + std::to_string(n.d) + " cannot be " + std::to_string(stride) + " apart");
}

// How a call's rows are taken: E values a chunk, LR lanes a row, NC chunks a lane.
struct NormPlan {
    int e, lr, nc;
    bool vec;
};

// 16-byte chunks where rows, strides and d allow, else four values of 16 bits at a time, or one by one;
// the fewest lanes to a row that hold it in at most four chunks of 16 bytes (a wave's loads are then
// full, and its rows share a load of gamma): 18752 rows of 768 bf16 14.3 -> 11.4 us against a wave a row
// in 8-byte chunks. Past four chunks of a wave's lanes a block takes a row.
NormPlan norm_plan(const Norm& n, bool back) {
    const int size = n.type == NORM_F32 ? 4 : 2;
    auto fits = [&](int e) {
        auto ok = [&](const void* a, int64_t stride) { return !a || ((uintptr_t)a % (e * size) == 0 && stride % e == 0); };
        return n.d % e == 0 && ok(n.x, n.x_stride) && ok(n.y, n.y_stride) && (!back || ok(n.dy, n.dy_stride)) &&
               (uintptr_t)n.gamma % 16 == 0 && (back || (uintptr_t)n.beta % 16 == 0);
    };
    NormPlan y{4, 64, 0, false};
    if (fits(16 / size)) y.e = 16 / size, y.vec = true;
    else if (fits(4)) y.vec = true;
    if (n.d > 256 * y.e) {
        y.e = 4, y.lr = 256;
    } else if (y.vec && y.e * size == 16) {
        while (y.lr > 8 && y.lr / 2 * (y.lr == 64 ? 4 : 3) * y.e >= n.d) y.lr /= 2;
    }
    y.nc = (n.d + y.e * y.lr - 1) / (y.e * y.lr);
    return y;
}

// Blocks of the gradients (each leaves a share of dgamma and dbeta): one a CU, or few enough for the
// last of them to sum their shares.
int norm_blocks(int rows, int d, int cus) {
    const int per = d > 1024 ? 1 : 8;  // (rows of a block at a time, at least)
    const int most = rows <= NORM_ONE_ROWS ? NORM_ONE_LAUNCH : cus;
    return std::max(1, std::min((rows + per - 1) / per, most));
}
NormParams norm_params(const Norm& n) {
    NormParams p{};
    p.x = n.x, p.dy = n.dy, p.y = n.y, p.x_stride = n.x_stride, p.dy_stride = n.dy_stride, p.y_stride = n.y_stride;
    p.gamma = n.gamma, p.beta = n.beta, p.stats = n.stats, p.rows = n.rows, p.d = n.d, p.eps = n.eps;
    p.inv_d = (float)(1.0 / n.d), p.dgamma = n.dgamma, p.dbeta = n.dbeta;
    return p;
}

template <int T, int E, bool VEC, int LR, int NC>
void run(const NormParams& p, bool back, int blocks, hipStream_t st) {
    if (back) {
        const int threads = LR == 256 ? 256 : 512;
        const size_t lds = std::max<size_t>((size_t)(LR == 256 ? 1 : 8) * 2 * p.d * 4, threads * 4);
        static std::atomic<uint64_t> devices{0};
        if (!dynamic_lds(devices, reinterpret_cast<const void*>(norm_back_kernel<T, E, VEC, LR, NC>), 8 * 2 * 2048 * 4))
            fail("the kernel cannot have its LDS");
        hipLaunchKernelGGL((norm_back_kernel<T, E, VEC, LR, NC>), dim3(blocks), dim3(threads), lds, st, p, blocks <= NORM_ONE_LAUNCH);
        return;
    }
    constexpr int G = 256 / LR, R = LR == 256 ? 1 : 2;
    // (two rows to a group of lanes once the grid is several blocks a CU anyway)
    if (R == 2 && p.rows >= 4 * device_cus() * G)
        hipLaunchKernelGGL((norm_kernel<T, E, VEC, LR, NC, R>), dim3((p.rows + R * G - 1) / (R * G)), dim3(256), 0, st, p);
    else
        hipLaunchKernelGGL((norm_kernel<T, E, VEC, LR, NC, 1>), dim3((p.rows + G - 1) / G), dim3(256), 0, st, p);
}

template <int T, int E, bool VEC, int LR>
void run_chunks(const NormParams& p, int nc, bool back, int blocks, hipStream_t st) {
    if constexpr (LR == 256) {
        if (nc <= 2) run<T, E, VEC, LR, 2>(p, back, blocks, st);
        else if (nc <= 4) run<T, E, VEC, LR, 4>(p, back, blocks, st);
        else run<T, E, VEC, LR, 8>(p, back, blocks, st);
    } else {
        if (nc <= 1) run<T, E, VEC, LR, 1>(p, back, blocks, st);
        else if (nc <= 2) run<T, E, VEC, LR, 2>(p, back, blocks, st);
        else if (nc <= 3) run<T, E, VEC, LR, 3>(p, back, blocks, st);
        else run<T, E, VEC, LR, 4>(p, back, blocks, st);
    }
}

template <int T>
void run_type(const NormParams& p, const NormPlan& y, bool back, int blocks, hipStream_t st) {
    constexpr int E = T == NORM_F32 ? 4 : 8;
    if (y.lr == 256) return y.vec ? run_chunks<T, 4, true, 256>(p, y.nc, back, blocks, st) : run_chunks<T, 4, false, 256>(p, y.nc, back, blocks, st);
    if (!y.vec) return run_chunks<T, 4, false, 64>(p, y.nc, back, blocks, st);
    if (y.e != E) return run_chunks<T, 4, true, 64>(p, y.nc, back, blocks, st);
    if (y.lr == 8) return run_chunks<T, E, true, 8>(p, y.nc, back, blocks, st);
    if (y.lr == 16) return run_chunks<T, E, true, 16>(p, y.nc, back, blocks, st);
    if (y.lr == 32) return run_chunks<T, E, true, 32>(p, y.nc, back, blocks, st);
    run_chunks<T, E, true, 64>(p, y.nc, back, blocks, st);
}

void run_any(const Norm& n, const NormParams& p, bool back, int blocks, hipStream_t st) {
    const NormPlan y = norm_plan(n, back);
    if (n.type == NORM_F32) run_type<NORM_F32>(p, y, back, blocks, st);
    else if (n.type == NORM_BF16) run_type<NORM_BF16>(p, y, back, blocks, st);
    else run_type<NORM_F16>(p, y, back, blocks, st);
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
    return {(size_t)norm_blocks(rows, d, cus) * 2 * d, 1};
}

void norm_launch(const Norm& n, hipStream_t st) {
    norm_check(n, false);
    if (n.rows == 0) return;
    run_any(n, norm_params(n), false, 0, st);
    check_launch();
}

void norm_backward_launch(const Norm& n, const Scratch& s, hipStream_t st) {
    norm_check(n, true);
    const int blocks = n.rows == 0 ? 0 : norm_blocks(n.rows, n.d, device_cus());
    if ((size_t)blocks * 2 * n.d > s.ws_floats || (blocks > 0 && s.n_counters < 1))
        fail("the scratch has " + std::to_string(s.ws_floats) + " floats and " + std::to_string(s.n_counters) + " counters, not " +
             std::to_string((size_t)blocks * 2 * n.d) + " and 1");
    NormParams p = norm_params(n);
    p.part = s.ws, p.counter = s.counters;
    if (blocks) run_any(n, p, true, blocks, st);
    if (blocks == 0 || blocks > NORM_ONE_LAUNCH)
        hipLaunchKernelGGL(norm_sum_kernel, dim3((2 * n.d + 31) / 32), dim3(1024), 0, st, p, blocks);
    check_launch();
}

}  // namespace jh
