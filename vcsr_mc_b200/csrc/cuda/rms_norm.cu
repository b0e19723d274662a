// Residual addition with root-mean-square norm, written as a microscaled (MX) matrix, and its
// backward pass. For a row of O columns:
//   s = round(x + residual)              (to the residual's type; the next residual)
//   inv = 1 / sqrt(mean(s^2) + eps)
//   Q = MX(s * inv * w)                  (mx.cuh)
// and with dy the gradient of the values that Q stands for (the element's rounding counts as identity):
//   g = dy * w
//   dx = d_residual + inv * g - s * inv^3 * mean(g * s)
//   dw = sum over rows of dy * s * inv
// The square sums are held in 64 bits: fp32 would overflow for |s| above 2^64, which bf16 and fp32 can
// hold. Both passes read each input once and write each output once (the row stays in registers up to
// O = 32768, and is read a second time beyond), so HBM bounds them except for a few rows.
#include <cuda_runtime.h>

#include <algorithm>

#include "mx.cuh"
#include "mx.hpp"
#include "vcsrmc.h"

namespace vcsrmc {
namespace dev {
namespace {

// A row is held by kL lanes of a warp (kL in 4 .. 32), kC chunks of 8 columns per lane, or, for
// kL = 0, by a whole block. kC = 0: any width, the row is read twice.
constexpr int kWarpRowThreads = 256;  // threads per block where a row fits a warp

__device__ __forceinline__ float load_weight(const void* w, int dtype, int64_t i) {
    if (dtype == VCSRMC_F32) return static_cast<const float*>(w)[i];
    if (dtype == VCSRMC_F16) return __half2float(static_cast<const __half*>(w)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
}

// Sum over the kL lanes of a row, or over the block (kL = 0); every thread gets the result. The order
// of the additions depends on the thread count alone.
template <int kL>
__device__ __forceinline__ double row_sum(double v, double* smem) {
    constexpr int kW = kL == 0 ? 32 : kL;
#pragma unroll
    for (int d = kW / 2; d >= 1; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    if constexpr (kL == 0) {
        const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
        __syncthreads();  // smem may still be read from the row before
        if (lane == 0) smem[threadIdx.x >> 5] = v;
        __syncthreads();
        v = lane < warps ? smem[lane] : 0.0;
#pragma unroll
        for (int d = 16; d >= 1; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    }
    return v;
}

struct NormShape {
    int64_t rows;
    int O;
    bool vec_x, vec_r, vec_o, vec_q;  // rows aligned for 16-byte loads and stores, Q for its full store
};

// The sum s of eight columns, rounded to the residual's type.
template <typename XT, typename RT>
__device__ __forceinline__ void load_sum(const RmsNormArgs& a, const NormShape& sh, int64_t row, int c, int nv, float (&s)[8]) {
    load8(static_cast<const XT*>(a.x.p) + row * a.x.ld + c, nv, sh.vec_x, s);
    if (a.residual.p) {
        float r[8];
        load8(static_cast<const RT*>(a.residual.p) + row * a.residual.ld + c, nv, sh.vec_r, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i] += r[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = to_f32(from_f32<RT>(s[i]));
}

template <typename XT, typename RT, int kL, int kC>
__global__ void __launch_bounds__(kL ? kWarpRowThreads : 1024) rms_norm_kernel(RmsNormArgs a, NormShape sh) {
    __shared__ double smem[32];
    const int per_row = kL ? kL : int(blockDim.x);
    const int sl = kL ? int(threadIdx.x) % (kL ? kL : 1) : int(threadIdx.x);
    // rows of a block move together: every thread takes part in the reductions of a row past the end
    const int in_block = kL ? kWarpRowThreads / (kL ? kL : 1) : 1;
    const int64_t row = int64_t(blockIdx.x) * in_block + (kL ? int(threadIdx.x) / (kL ? kL : 1) : 0);
    const bool live = row < sh.rows;
    const int O = live ? sh.O : 0;
    constexpr int kHeld = kC ? kC : 1;
    const int chunks = kC ? kC : (sh.O + 8 * per_row - 1) / (8 * per_row);
    float s[kHeld][8];
    double sum = 0.0;
    // forward over the chunks; with kC = 0 only the sum is kept
    auto first = [&](int k, float (&v)[8]) {
        const int c = 8 * (k * per_row + sl);
        const int nv = max(0, min(8, O - c));
        load_sum<XT, RT>(a, sh, row, c, nv, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += double(v[i]) * double(v[i]);
    };
    if constexpr (kC > 0) {
#pragma unroll
        for (int k = 0; k < kC; ++k) first(k, s[k]);
    } else {
        for (int k = 0; k < chunks; ++k) first(k, s[0]);
    }
    sum = row_sum<kL>(sum, smem);
    const float inv = float(1.0 / sqrt(sum / double(sh.O) + double(a.eps)));
    if (live && sl == 0 && a.inv_rms) a.inv_rms[row] = inv;
    auto second = [&](int k, float (&v)[8]) {
        const int c = 8 * (k * per_row + sl);
        const int nv = max(0, min(8, O - c));
        if constexpr (kC == 0) load_sum<XT, RT>(a, sh, row, c, nv, v);
        if (a.residual_out.p) store8(static_cast<RT*>(a.residual_out.p) + row * a.residual_out.ld + c, nv, sh.vec_o, v);
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = i < nv ? v[i] * inv * load_weight(a.weight, a.w_dtype, c + i) : 0.f;
        mx_store_block(y, nv, a.out.q4, a.out.q + row * a.out.ldq + (a.out.q4 ? c / 2 : c), a.out.s + row * a.out.lds + c / kMxBlock,
                       sh.vec_q);
    };
    if constexpr (kC > 0) {
#pragma unroll
        for (int k = 0; k < kC; ++k) second(k, s[k]);
    } else {
        for (int k = 0; k < chunks; ++k) second(k, s[0]);
    }
}

template <typename XT, typename RT, int kL, int kC>
cudaError_t launch_norm(const RmsNormArgs& a, const NormShape& sh, int threads, cudaStream_t st) {
    const int64_t in_block = kL ? kWarpRowThreads / (kL ? kL : 1) : 1;
    const int64_t blocks = (sh.rows + in_block - 1) / in_block;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
    rms_norm_kernel<XT, RT, kL, kC><<<unsigned(blocks), kL ? kWarpRowThreads : threads, 0, st>>>(a, sh);
    return cudaGetLastError();
}

bool aligned(const void* p, int64_t ld_bytes, int64_t to) {
    return reinterpret_cast<uintptr_t>(p) % to == 0 && ld_bytes % to == 0;
}

template <typename XT, typename RT>
cudaError_t norm_t(const RmsNormArgs& a, cudaStream_t st) {
    NormShape sh;
    sh.rows = a.rows;
    sh.O = a.O;
    sh.vec_x = aligned(a.x.p, a.x.ld * int64_t(sizeof(XT)), 16);
    sh.vec_r = aligned(a.residual.p, a.residual.ld * int64_t(sizeof(RT)), 16);
    sh.vec_o = aligned(a.residual_out.p, a.residual_out.ld * int64_t(sizeof(RT)), 16);
    sh.vec_q = aligned(a.out.q, a.out.ldq, a.out.q4 ? 4 : 8);
    const int O = a.O;
    if (O <= 32) return launch_norm<XT, RT, 4, 1>(a, sh, 0, st);
    if (O <= 64) return launch_norm<XT, RT, 8, 1>(a, sh, 0, st);
    if (O <= 128) return launch_norm<XT, RT, 16, 1>(a, sh, 0, st);
    if (O <= 256) return launch_norm<XT, RT, 32, 1>(a, sh, 0, st);
    if (O <= 512) return launch_norm<XT, RT, 32, 2>(a, sh, 0, st);
    if (O <= 1024) return launch_norm<XT, RT, 32, 4>(a, sh, 0, st);
    int threads = 128;
    while (threads < 1024 && 8 * threads * 4 < O) threads *= 2;
    if (O <= 8 * threads * 2) return launch_norm<XT, RT, 0, 2>(a, sh, threads, st);
    if (O <= 8 * threads * 4) return launch_norm<XT, RT, 0, 4>(a, sh, threads, st);
    return launch_norm<XT, RT, 0, 0>(a, sh, 1024, st);
}

// ---- backward --------------------------------------------------------------------------------------
struct GradShape {
    int64_t rows;
    int O;
    bool vec_dy, vec_dr, vec_h, vec_dx;
};

// Persistent blocks over the rows; each thread keeps the weight gradient of its columns in registers
// and the block writes one row of partial sums to the workspace, in which a second kernel adds the
// blocks up in their order.
template <typename DT, typename RT, int kL, int kC>
__global__ void __launch_bounds__(kL ? kWarpRowThreads : 1024) rms_norm_grad_kernel(RmsNormGradArgs a, GradShape sh) {
    __shared__ double smem[32];
    __shared__ float fold[kL ? kWarpRowThreads : 1][kL ? 8 : 1];
    const int per_row = kL ? kL : int(blockDim.x);
    const int sl = kL ? int(threadIdx.x) % (kL ? kL : 1) : int(threadIdx.x);
    const int in_block = kL ? kWarpRowThreads / (kL ? kL : 1) : 1;
    const int my = kL ? int(threadIdx.x) / (kL ? kL : 1) : 0;
    constexpr int kHeld = kC ? kC : 1;
    const int chunks = kC ? kC : (sh.O + 8 * per_row - 1) / (8 * per_row);
    float* part = a.workspace + int64_t(blockIdx.x) * sh.O;
    float dw[kHeld][8] = {};
    for (int64_t r0 = int64_t(blockIdx.x) * in_block; r0 < sh.rows; r0 += int64_t(gridDim.x) * in_block) {
        const int64_t row = r0 + my;
        const bool live = row < sh.rows;
        const int O = live ? sh.O : 0;
        const float inv = live ? a.inv_rms[row] : 0.f;
        float dy[kHeld][8], h[kHeld][8];
        double dot = 0.0;
        auto first = [&](int k, float (&vy)[8], float (&vh)[8]) {
            const int c = 8 * (k * per_row + sl);
            const int nv = max(0, min(8, O - c));
            load8(static_cast<const DT*>(a.dy.p) + row * a.dy.ld + c, nv, sh.vec_dy, vy);
            load8(static_cast<const RT*>(a.hidden.p) + row * a.hidden.ld + c, nv, sh.vec_h, vh);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < nv) dot += double(vy[i] * load_weight(a.weight, a.w_dtype, c + i)) * double(vh[i]);
        };
        if constexpr (kC > 0) {
#pragma unroll
            for (int k = 0; k < kC; ++k) first(k, dy[k], h[k]);
        } else {
            for (int k = 0; k < chunks; ++k) first(k, dy[0], h[0]);
        }
        dot = row_sum<kL>(dot, smem);
        // inv^2 * mean(g * s), in 64 bits: its factors may leave fp32's range where the product does not
        const float m = float(dot * double(inv) * double(inv) / double(sh.O));
        auto second = [&](int k, float (&vy)[8], float (&vh)[8], float (&vw)[8]) {
            const int c = 8 * (k * per_row + sl);
            const int nv = max(0, min(8, O - c));
            if constexpr (kC == 0) {
                load8(static_cast<const DT*>(a.dy.p) + row * a.dy.ld + c, nv, sh.vec_dy, vy);
                load8(static_cast<const RT*>(a.hidden.p) + row * a.hidden.ld + c, nv, sh.vec_h, vh);
            }
            float dx[8];
            if (a.d_residual.p) load8(static_cast<const RT*>(a.d_residual.p) + row * a.d_residual.ld + c, nv, sh.vec_dr, dx);
            else
#pragma unroll
                for (int i = 0; i < 8; ++i) dx[i] = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < nv) {
                    dx[i] += inv * (vy[i] * load_weight(a.weight, a.w_dtype, c + i) - vh[i] * m);
                    vw[i] += vy[i] * (vh[i] * inv);
                }
            store8(static_cast<RT*>(a.dx.p) + row * a.dx.ld + c, nv, sh.vec_dx, dx);
        };
        if constexpr (kC > 0) {
#pragma unroll
            for (int k = 0; k < kC; ++k) second(k, dy[k], h[k], dw[k]);
        } else {
            for (int k = 0; k < chunks; ++k) {
                // the block's own row of the workspace carries the sums of a row wider than its registers
                const int c = 8 * (k * per_row + sl);
                const int nv = max(0, min(8, O - c));
                float w[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = i < nv && r0 != int64_t(blockIdx.x) ? part[c + i] : 0.f;
                second(k, dy[0], h[0], w);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i < nv) part[c + i] = w[i];
            }
        }
    }
    if constexpr (kC == 0) return;
    if constexpr (kL > 0) {
        // sum over the rows of the block, in their order
#pragma unroll
        for (int k = 0; k < kC; ++k) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 8; ++i) fold[threadIdx.x][i] = dw[k][i];
            __syncthreads();
            for (int t = int(threadIdx.x); t < kL * 8; t += kWarpRowThreads) {
                const int c = 8 * (k * kL + t / 8) + t % 8;
                float v = 0.f;
                for (int g = 0; g < kWarpRowThreads / (kL ? kL : 1); ++g) v += fold[g * kL + t / 8][t % 8];
                if (c < sh.O) part[c] = v;
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < kHeld; ++k) {
            const int c = 8 * (k * per_row + sl);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < sh.O) part[c + i] = dw[k][i];
        }
    }
}

// dweight[c] = sum over the blocks' partial rows: 32 columns per block, 8 warps over the rows.
__global__ void __launch_bounds__(256) rms_norm_dweight_kernel(const float* __restrict__ part, int n, int O, float* __restrict__ dw) {
    __shared__ float s[8][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int c = int(blockIdx.x) * 32 + lane;
    float v = 0.f;
    if (c < O)
        for (int i = warp; i < n; i += 8) v += part[int64_t(i) * O + c];
    s[warp][lane] = v;
    __syncthreads();
    if (warp == 0 && c < O) {
#pragma unroll
        for (int k = 1; k < 8; ++k) v += s[k][lane];
        dw[c] = v;
    }
}

// Rows that a block holds at once, for a width.
int rows_in_block(int O) {
    if (O > 1024) return 1;
    int lanes = 4;
    while (lanes < 32 && 8 * lanes < O) lanes *= 2;
    return kWarpRowThreads / lanes;
}
// Blocks of the backward pass: two for every SM, or one for every group of rows where there are fewer.
int64_t grad_blocks(int64_t rows, int O, int sms) {
    const int64_t groups = (rows + rows_in_block(O) - 1) / rows_in_block(O);
    return std::max<int64_t>(1, std::min<int64_t>(groups, int64_t(sms) * (O > 1024 ? 2 : 8)));
}

template <typename DT, typename RT, int kL, int kC>
cudaError_t launch_grad(const RmsNormGradArgs& a, const GradShape& sh, int threads, int64_t blocks, cudaStream_t st) {
    rms_norm_grad_kernel<DT, RT, kL, kC><<<unsigned(blocks), kL ? kWarpRowThreads : threads, 0, st>>>(a, sh);
    return cudaGetLastError();
}

template <typename DT, typename RT>
cudaError_t grad_t(const RmsNormGradArgs& a, int64_t blocks, cudaStream_t st) {
    GradShape sh;
    sh.rows = a.rows;
    sh.O = a.O;
    sh.vec_dy = aligned(a.dy.p, a.dy.ld * int64_t(sizeof(DT)), 16);
    sh.vec_dr = aligned(a.d_residual.p, a.d_residual.ld * int64_t(sizeof(RT)), 16);
    sh.vec_h = aligned(a.hidden.p, a.hidden.ld * int64_t(sizeof(RT)), 16);
    sh.vec_dx = aligned(a.dx.p, a.dx.ld * int64_t(sizeof(RT)), 16);
    const int O = a.O;
    if (O <= 32) return launch_grad<DT, RT, 4, 1>(a, sh, 0, blocks, st);
    if (O <= 64) return launch_grad<DT, RT, 8, 1>(a, sh, 0, blocks, st);
    if (O <= 128) return launch_grad<DT, RT, 16, 1>(a, sh, 0, blocks, st);
    if (O <= 256) return launch_grad<DT, RT, 32, 1>(a, sh, 0, blocks, st);
    if (O <= 512) return launch_grad<DT, RT, 32, 2>(a, sh, 0, blocks, st);
    if (O <= 1024) return launch_grad<DT, RT, 32, 4>(a, sh, 0, blocks, st);
    int threads = 256;
    while (threads < 1024 && 8 * threads * 2 < O) threads *= 2;
    if (O <= 8 * threads * 2) return launch_grad<DT, RT, 0, 2>(a, sh, threads, blocks, st);
    return launch_grad<DT, RT, 0, 0>(a, sh, 1024, blocks, st);
}

}  // namespace

cudaError_t add_rms_norm(const RmsNormArgs& a, cudaStream_t st) {
    const int x = a.x.dtype, r = a.residual_out.dtype;
    if (x == VCSRMC_F16) return norm_t<__half, __half>(a, st);
    if (x == VCSRMC_BF16) return norm_t<__nv_bfloat16, __nv_bfloat16>(a, st);
    if (r == VCSRMC_F16) return norm_t<float, __half>(a, st);
    if (r == VCSRMC_BF16) return norm_t<float, __nv_bfloat16>(a, st);
    return norm_t<float, float>(a, st);
}

int64_t rms_norm_grad_workspace(int64_t rows, int O, int sms) { return grad_blocks(rows, O, sms) * O * int64_t(sizeof(float)); }

cudaError_t add_rms_norm_backward(const RmsNormGradArgs& a, int sms, cudaStream_t st) {
    const int64_t blocks = grad_blocks(a.rows, a.O, sms);
    const int d = a.dy.dtype, r = a.hidden.dtype;
    cudaError_t e;
    if (d == VCSRMC_F16) e = grad_t<__half, __half>(a, blocks, st);
    else if (d == VCSRMC_BF16) e = grad_t<__nv_bfloat16, __nv_bfloat16>(a, blocks, st);
    else if (r == VCSRMC_F16) e = grad_t<float, __half>(a, blocks, st);
    else if (r == VCSRMC_BF16) e = grad_t<float, __nv_bfloat16>(a, blocks, st);
    else e = grad_t<float, float>(a, blocks, st);
    if (e != cudaSuccess) return e;
    rms_norm_dweight_kernel<<<unsigned((a.O + 31) / 32), 256, 0, st>>>(a.workspace, int(blocks), a.O, a.dweight);
    return cudaGetLastError();
}

}  // namespace dev
}  // namespace vcsrmc
