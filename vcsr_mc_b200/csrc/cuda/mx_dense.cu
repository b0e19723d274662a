// Quantisation of a dense matrix to the microscaled format, and back (mx.cuh has the format).
//
// Both are one pass over memory: per element they move the dense value (2 or 4 bytes) and 1 or 1/2
// byte of element plus 1/32 byte of scale, so HBM bounds them. A thread owns eight consecutive columns
// (16 or 32 bytes of the dense side in flight), four neighbouring threads a block of 32.
#include <cuda_runtime.h>

#include <algorithm>

#include "mx.cuh"
#include "mx.hpp"
#include "vcsrmc.h"

namespace vcsrmc {
namespace dev {
namespace {

constexpr int kThreads = 256;

// Work is numbered (row, group of 8 columns), padded to whole blocks of four groups; a launch covers
// rows whose numbers fit 31 bits.
struct Shape {
    int rows, O, groups;  // groups = 4 * blocks of a row
    bool vec_x, vec_q;
};

template <typename T>
__global__ void __launch_bounds__(kThreads) mx_quantize_kernel(const T* __restrict__ X, int64_t ldx, Shape sh, MxView Q) {
    const int i = int(blockIdx.x) * kThreads + int(threadIdx.x);
    const int row = i / sh.groups, g = i - row * sh.groups, c = 8 * g;
    const int nv = row < sh.rows ? max(0, min(8, sh.O - c)) : 0;
    float v[8];
    load8(X + int64_t(row) * ldx + c, nv, sh.vec_x, v);
    mx_store_block(v, nv, Q.q4, Q.q + int64_t(row) * Q.ldq + (Q.q4 ? c / 2 : c), Q.s + int64_t(row) * Q.lds + c / kMxBlock, sh.vec_q);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) mx_dequantize_kernel(MxView Q, Shape sh, T* __restrict__ Y, int64_t ldy) {
    const int i = int(blockIdx.x) * kThreads + int(threadIdx.x);
    const int row = i / sh.groups, g = i - row * sh.groups, c = 8 * g;
    if (row >= sh.rows || c >= sh.O) return;
    const int nv = min(8, sh.O - c);
    const uint8_t* q = Q.q + int64_t(row) * Q.ldq + (Q.q4 ? c / 2 : c);
    const float scale = mx_scale_value(Q.s[int64_t(row) * Q.lds + c / kMxBlock]);
    const int bytes = Q.q4 ? (nv + 1) / 2 : nv;
    uint32_t w[2] = {0u, 0u};
    if (sh.vec_q && nv == 8) {
        if (Q.q4) w[0] = *reinterpret_cast<const uint32_t*>(q);
        else *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(q);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k < bytes) w[k >> 2] |= uint32_t(q[k]) << (8 * (k & 3));
    }
    float v[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float2 f = mx_f16x2_to_f32(Q.q4 ? mx_decode2_e2m1((w[0] >> (8 * k)) & 0xffu)
                                              : mx_decode2_e4m3((w[k >> 1] >> (16 * (k & 1))) & 0xffffu));
        v[2 * k] = f.x * scale;
        v[2 * k + 1] = f.y * scale;
    }
    store8(Y + int64_t(row) * ldy + c, nv, sh.vec_x, v);
}

template <typename T>
bool rows_aligned(const void* p, int64_t ld_bytes, T bytes) {
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && ld_bytes % bytes == 0;
}

// Calls launch(first row, shape, blocks) for slices of rows whose work numbers fit 31 bits.
template <typename T, class Fn>
cudaError_t sliced(const DenseView& X, int64_t rows, int O, const MxView& Q, Fn&& launch) {
    Shape sh;
    sh.O = O;
    sh.groups = 4 * ((O + kMxBlock - 1) / kMxBlock);
    sh.vec_x = rows_aligned(X.p, X.ld * int64_t(sizeof(T)), 16);
    sh.vec_q = rows_aligned(Q.q, Q.ldq, Q.q4 ? 4 : 8);
    const int64_t most = std::max<int64_t>(1, int64_t(0x7fff0000) / sh.groups);
    for (int64_t r = 0; r < rows; r += most) {
        sh.rows = int(std::min(most, rows - r));
        const int64_t n = int64_t(sh.rows) * sh.groups;
        launch(r, sh, unsigned((n + kThreads - 1) / kThreads));
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

MxView from_row(MxView Q, int64_t r) {
    Q.q += r * Q.ldq;
    Q.s += r * Q.lds;
    return Q;
}

template <typename T>
cudaError_t quantize_t(const DenseView& X, int64_t rows, int O, const MxView& Q, cudaStream_t st) {
    return sliced<T>(X, rows, O, Q, [&](int64_t r, const Shape& sh, unsigned blocks) {
        mx_quantize_kernel<T><<<blocks, kThreads, 0, st>>>(static_cast<const T*>(X.p) + r * X.ld, X.ld, sh, from_row(Q, r));
    });
}

template <typename T>
cudaError_t dequantize_t(const MxView& Q, int64_t rows, int O, const DenseView& Y, cudaStream_t st) {
    return sliced<T>(Y, rows, O, Q, [&](int64_t r, const Shape& sh, unsigned blocks) {
        mx_dequantize_kernel<T><<<blocks, kThreads, 0, st>>>(from_row(Q, r), sh, static_cast<T*>(Y.p) + r * Y.ld, Y.ld);
    });
}

}  // namespace

cudaError_t mx_quantize(const DenseView& X, int64_t rows, int O, const MxView& Q, cudaStream_t st) {
    if (X.dtype == VCSRMC_F32) return quantize_t<float>(X, rows, O, Q, st);
    if (X.dtype == VCSRMC_F16) return quantize_t<__half>(X, rows, O, Q, st);
    return quantize_t<__nv_bfloat16>(X, rows, O, Q, st);
}

cudaError_t mx_dequantize(const MxView& Q, int64_t rows, int O, const DenseView& Y, cudaStream_t st) {
    if (Y.dtype == VCSRMC_F32) return dequantize_t<float>(Q, rows, O, Y, st);
    if (Y.dtype == VCSRMC_F16) return dequantize_t<__half>(Q, rows, O, Y, st);
    return dequantize_t<__nv_bfloat16>(Q, rows, O, Y, st);
}

}  // namespace dev
}  // namespace vcsrmc
