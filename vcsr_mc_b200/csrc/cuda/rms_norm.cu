// Residual addition with root-mean-square norm and its backward pass (rms_norm.cuh): the choice of the element
// widths and the last step of the weight's gradient.
#include <cuda_runtime.h>

#include <algorithm>

#include "rms_norm.cuh"

namespace vcsrmc {
namespace dev {
namespace {

// dweight[c] = sum over the blocks' partial rows: 32 columns per block, 32 warps over the rows, eight in flight. (Eight
// warps with four in flight took half of the backward pass of 8192 rows of 1000.)
constexpr int kSumWarps = 32, kSumFlight = 8;
__global__ void __launch_bounds__(kSumWarps * 32) rms_norm_dweight_kernel(const float* __restrict__ part, int n, int O, float* __restrict__ dw) {
    __shared__ float s[kSumWarps][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int c = int(blockIdx.x) * 32 + lane;
    float v[kSumFlight] = {};
    wait_for_launch_before();  // the partial sums
    if (c < O) {
        for (int i = warp; i < n; i += kSumWarps * kSumFlight) {
#pragma unroll
            for (int k = 0; k < kSumFlight; ++k)
                if (i + k * kSumWarps < n) v[k] += part[int64_t(i + k * kSumWarps) * O + c];
        }
    }
#pragma unroll
    for (int d = 1; d < kSumFlight; d *= 2)
#pragma unroll
        for (int k = 0; k < kSumFlight; k += 2 * d) v[k] += v[k + d];
    s[warp][lane] = v[0];
    __syncthreads();
    // warp w adds up column w's 32 sums
    float t = s[lane][warp];
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) t += __shfl_xor_sync(0xffffffffu, t, d);
    const int column = int(blockIdx.x) * 32 + warp;
    if (lane == 0 && column < O) dw[column] = t;
}

// Blocks of the backward pass: enough to fill every SM with about 1024 threads, or one for every row (or
// group of rows that a block holds) where there are fewer. The same for both access forms, so that the
// workspace depends on the shape alone.
int64_t grad_blocks(int64_t rows, int O, int sms) {
    if (O <= 256) {
        int lanes = 4;
        while (8 * lanes < O) lanes *= 2;
        const int64_t in_block = 256 / lanes;
        return std::max<int64_t>(1, std::min(int64_t(sms) * 4, (rows + in_block - 1) / in_block));
    }
    return std::max<int64_t>(1, std::min(rows, int64_t(sms) * (1024 / norm::grad_threads(O))));
}

}  // namespace

cudaError_t add_rms_norm(const RmsNormArgs& args, cudaStream_t st) {
    RmsNormArgs a = args;
    a.vec_w = reinterpret_cast<uintptr_t>(a.weight) % 16 == 0;
    a.vec_q = norm::aligned(a.out.q, a.out.ldq, a.out.q4 ? 4 : 8);
    if (a.x.dtype != VCSRMC_F32) return norm::forward<false, false>(a, st);
    return a.residual_out.dtype == VCSRMC_F32 ? norm::forward<true, true>(a, st) : norm::forward<true, false>(a, st);
}

int64_t rms_norm_grad_workspace(int64_t rows, int O, int sms) { return grad_blocks(rows, O, sms) * O * int64_t(sizeof(float)); }

cudaError_t add_rms_norm_backward(const RmsNormGradArgs& args, int sms, cudaStream_t st) {
    RmsNormGradArgs a = args;
    a.vec_w = reinterpret_cast<uintptr_t>(a.weight) % 16 == 0;
    const int64_t blocks = grad_blocks(a.rows, a.O, sms);
    const cudaError_t e = a.dy.dtype != VCSRMC_F32          ? norm::backward<false, false>(a, blocks, st)
                          : a.hidden.dtype == VCSRMC_F32 ? norm::backward<true, true>(a, blocks, st)
                                                         : norm::backward<true, false>(a, blocks, st);
    if (e != cudaSuccess) return e;
    LaunchAfter L(dim3(unsigned((a.O + 31) / 32), 1, 1), dim3(kSumWarps * 32, 1, 1), st);
    return cudaLaunchKernelEx(&L.cfg, rms_norm_dweight_kernel, static_cast<const float*>(a.workspace), int(blocks), a.O, a.dweight);
}

}  // namespace dev
}  // namespace vcsrmc
