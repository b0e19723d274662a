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

// i / d for 0 <= i < 2^31 by a multiplication: m = ceil(2^(31 + bits) / d) with 2^(bits - 1) < d <= 2^bits.
// m * d - 2^(31 + bits) < d <= 2^bits, so i * m / 2^(31 + bits) is above i / d by less than 1 / d.
struct Divisor {
    uint64_t m;
    int shift;
    explicit Divisor(int d) {
        int bits = 0;
        while ((int64_t(1) << bits) < d) ++bits;
        shift = 31 + bits;
        m = ((uint64_t(1) << shift) + uint64_t(d) - 1) / uint64_t(d);
    }
    __device__ int operator()(int i) const { return int((uint64_t(uint32_t(i)) * m) >> shift); }
};

// A launch covers rows whose work numbers fit 31 bits. Aligned rows of whole groups of eight columns: a
// number is (row, group), padded to whole blocks of four groups, and a thread takes two of them half the work
// apart, so that two loads are in flight. Every other layout: a number is (row, block) and a warp's, one
// column per lane, so that its loads and stores stay coalesced.
struct Shape {
    int rows, O, per_row, half;  // numbers of a row; numbers of a thread's first part
    Divisor by_row;
};

template <typename T>
__global__ void __launch_bounds__(kThreads) mx_quantize_kernel(const T* __restrict__ X, int64_t ldx, Shape sh, MxView Q) {
    float v[2][8];
    int row[2], c[2], nv[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int i = int(blockIdx.x) * kThreads + int(threadIdx.x) + k * sh.half;
        row[k] = sh.by_row(i);
        c[k] = 8 * (i - row[k] * sh.per_row);
        nv[k] = i - k * sh.half < sh.half && row[k] < sh.rows && c[k] < sh.O ? 8 : 0;
        load8(X + int64_t(row[k]) * ldx + c[k], nv[k], true, v[k]);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k)
        mx_store_block(v[k], nv[k], Q.q4, Q.q + int64_t(row[k]) * Q.ldq + (Q.q4 ? c[k] / 2 : c[k]),
                       Q.s + int64_t(row[k]) * Q.lds + c[k] / kMxBlock, true);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) mx_quantize_columns_kernel(const T* __restrict__ X, int64_t ldx, Shape sh, MxView Q) {
    const int lane = threadIdx.x & 31;
    float v[4];
    int row[4], c[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int i = (int(blockIdx.x) * (kThreads / 32) + int(threadIdx.x >> 5)) * 4 + k;
        row[k] = sh.by_row(i);
        c[k] = kMxBlock * (i - row[k] * sh.per_row) + lane;
        if (row[k] >= sh.rows) c[k] = sh.O;
        v[k] = c[k] < sh.O ? to_f32(X[int64_t(row[k]) * ldx + c[k]]) : 0.f;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
        mx_store_column(v[k], c[k] < sh.O, c[k] + 1 < sh.O, Q.q4, Q.q + int64_t(row[k]) * Q.ldq + (Q.q4 ? c[k] / 2 : c[k]),
                        Q.s + int64_t(row[k]) * Q.lds + c[k] / kMxBlock);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) mx_dequantize_kernel(MxView Q, Shape sh, T* __restrict__ Y, int64_t ldy) {
    uint32_t w[2][2];
    float scale[2];
    int row[2], c[2];
    bool live[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int i = int(blockIdx.x) * kThreads + int(threadIdx.x) + k * sh.half;
        row[k] = sh.by_row(i);
        c[k] = 8 * (i - row[k] * sh.per_row);
        live[k] = i - k * sh.half < sh.half && row[k] < sh.rows && c[k] < sh.O;
        if (!live[k]) continue;
        const uint8_t* q = Q.q + int64_t(row[k]) * Q.ldq + (Q.q4 ? c[k] / 2 : c[k]);
        if (Q.q4) w[k][0] = __ldcs(reinterpret_cast<const uint32_t*>(q));
        else *reinterpret_cast<uint2*>(w[k]) = __ldcs(reinterpret_cast<const uint2*>(q));
        scale[k] = mx_scale_value(Q.s[int64_t(row[k]) * Q.lds + c[k] / kMxBlock]);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        if (!live[k]) continue;
        float v[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = mx_f16x2_to_f32(Q.q4 ? mx_decode2_e2m1((w[k][0] >> (8 * j)) & 0xffu)
                                                  : mx_decode2_e4m3((w[k][j >> 1] >> (16 * (j & 1))) & 0xffffu));
            v[2 * j] = f.x * scale[k];
            v[2 * j + 1] = f.y * scale[k];
        }
        store8(Y + int64_t(row[k]) * ldy + c[k], 8, true, v);
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) mx_dequantize_columns_kernel(MxView Q, Shape sh, T* __restrict__ Y, int64_t ldy) {
    const int lane = threadIdx.x & 31;
    uint32_t w[4];
    float scale[4];
    int row[4], c[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int i = (int(blockIdx.x) * (kThreads / 32) + int(threadIdx.x >> 5)) * 4 + k;
        row[k] = sh.by_row(i);
        c[k] = kMxBlock * (i - row[k] * sh.per_row) + lane;
        if (row[k] >= sh.rows) c[k] = sh.O;
        if (c[k] >= sh.O) continue;
        w[k] = Q.q[int64_t(row[k]) * Q.ldq + (Q.q4 ? c[k] / 2 : c[k])];
        scale[k] = mx_scale_value(Q.s[int64_t(row[k]) * Q.lds + c[k] / kMxBlock]);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (c[k] >= sh.O) continue;
        const float2 f = mx_f16x2_to_f32(Q.q4 ? mx_decode2_e2m1(w[k]) : mx_decode2_e4m3(w[k]));
        Y[int64_t(row[k]) * ldy + c[k]] = from_f32<T>((Q.q4 && (c[k] & 1) ? f.y : f.x) * scale[k]);
    }
}

bool rows_aligned(const void* p, int64_t ld_bytes, int64_t bytes) {
    return reinterpret_cast<uintptr_t>(p) % uintptr_t(bytes) == 0 && ld_bytes % bytes == 0;
}

// Calls launch(first row, shape, blocks, whole groups?) for slices of rows whose work numbers fit 31 bits.
template <typename T, class Fn>
cudaError_t sliced(const DenseView& X, int64_t rows, int O, const MxView& Q, Fn&& launch) {
    const int blocks = (O + kMxBlock - 1) / kMxBlock;
    const bool groups = O % 8 == 0 && rows_aligned(X.p, X.ld * int64_t(sizeof(T)), 16) && rows_aligned(Q.q, Q.ldq, Q.q4 ? 4 : 8);
    const int per_row = groups ? 4 * blocks : blocks;
    const int64_t most = std::max<int64_t>(1, int64_t(0x7ff00000) / per_row);
    for (int64_t r = 0; r < rows; r += most) {
        const int64_t n = std::min(most, rows - r);
        const int64_t numbers = n * per_row;
        const int64_t per_block = groups ? kThreads : kThreads / 32 * 4;
        const int64_t half = (numbers / 4 + 1) / 2 * 4;  // whole blocks of four groups
        const int64_t grid = ((groups ? half : numbers) + per_block - 1) / per_block;
        launch(r, Shape{int(n), O, per_row, int(half), Divisor(per_row)}, unsigned(grid), groups);
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
    return sliced<T>(X, rows, O, Q, [&](int64_t r, const Shape& sh, unsigned blocks, bool groups) {
        const T* x = static_cast<const T*>(X.p) + r * X.ld;
        if (groups) mx_quantize_kernel<T><<<blocks, kThreads, 0, st>>>(x, X.ld, sh, from_row(Q, r));
        else mx_quantize_columns_kernel<T><<<blocks, kThreads, 0, st>>>(x, X.ld, sh, from_row(Q, r));
    });
}

template <typename T>
cudaError_t dequantize_t(const MxView& Q, int64_t rows, int O, const DenseView& Y, cudaStream_t st) {
    return sliced<T>(Y, rows, O, Q, [&](int64_t r, const Shape& sh, unsigned blocks, bool groups) {
        T* y = static_cast<T*>(Y.p) + r * Y.ld;
        if (groups) mx_dequantize_kernel<T><<<blocks, kThreads, 0, st>>>(from_row(Q, r), sh, y, Y.ld);
        else mx_dequantize_columns_kernel<T><<<blocks, kThreads, 0, st>>>(from_row(Q, r), sh, y, Y.ld);
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
