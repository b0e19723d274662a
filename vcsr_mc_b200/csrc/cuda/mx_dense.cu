// Quantisation of a dense matrix to the microscaled format, and back (mx.cuh has the format).
//
// Both are one pass over memory: per element they move the dense value (2 or 4 bytes) and 1 or 1/2
// byte of element plus 1/32 byte of scale, so HBM bounds them: 2^20 x 128 fp16 to E2M1 and back to bf16 take 129 us in
// all on a B200 (675 MB with the 4-bit matrix in between, 5.2 TB/s; copies run at 6.5), 131072 x 512 fp32 to E4M3
// 52 us (6.6 TB/s, part of it from L2). Rows that are not aligned move a column per load and are bound by those: x 501
// bf16 to E4M3 64 us and back 82 us (floor 30). A thread owns eight consecutive columns (16 or 32 bytes of the dense
// side in flight), four neighbouring threads a block of 32.
#include <cuda_runtime.h>

#include <algorithm>

#include "mx.cuh"
#include "mx.hpp"
#include "vcsrmc.h"

namespace vcsrmc {
namespace dev {
namespace {

constexpr int kThreads = 256;
// Groups of a thread: reading 4-bit elements takes four to have as much in flight as two of a dense type.
constexpr int kQuantizeParts = 2, kDequantizeParts = 4;

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

// A launch covers rows whose work numbers fit 31 bits. A number is (row, group of eight columns), padded to whole
// spans of kL groups; a thread takes kParts of them, `part` apart, so that as many loads are in flight. Aligned rows
// (O a multiple of 8): kL = 4, a block. Every other layout: kL (4 .. 32, a row's groups at most) neighbouring threads
// deal a span's columns out over them for coalesced single accesses, and turn them in shared memory.
struct Shape {
    int rows, O, per_row, part;  // per_row: numbers of a row
    Divisor by_row;
    bool vec_q;                  // Q's rows are aligned to the stores of eight elements
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 8) mx_quantize_kernel(const T* __restrict__ X, int64_t ldx, Shape sh, MxView Q) {
    float v[kQuantizeParts][8];
    int row[kQuantizeParts], c[kQuantizeParts], nv[kQuantizeParts];
#pragma unroll
    for (int k = 0; k < kQuantizeParts; ++k) {
        const int i = int(blockIdx.x) * kThreads + int(threadIdx.x) + k * sh.part;
        row[k] = sh.by_row(i);
        c[k] = 8 * (i - row[k] * sh.per_row);
        nv[k] = i - k * sh.part < sh.part && row[k] < sh.rows && c[k] < sh.O ? 8 : 0;
        load8(X + int64_t(row[k]) * ldx + c[k], nv[k], true, v[k]);
    }
#pragma unroll
    for (int k = 0; k < kQuantizeParts; ++k)
        mx_store_block(v[k], nv[k], Q.q4, Q.q + int64_t(row[k]) * Q.ldq + (Q.q4 ? c[k] / 2 : c[k]),
                       Q.s + int64_t(row[k]) * Q.lds + c[k] / kMxBlock, true);
}

template <typename T, int kL>
__global__ void __launch_bounds__(kThreads) mx_quantize_columns_kernel(const T* __restrict__ X, int64_t ldx, Shape sh, MxView Q) {
    __shared__ __align__(16) float turn[8 * kThreads];
    const int sl = threadIdx.x % kL;
    float t[kQuantizeParts][8];
    int row[kQuantizeParts], c[kQuantizeParts];
#pragma unroll
    for (int k = 0; k < kQuantizeParts; ++k) {
        const int i = int(blockIdx.x) * kThreads + int(threadIdx.x) + k * sh.part;
        row[k] = sh.by_row(i);
        c[k] = 8 * (i - row[k] * sh.per_row);
        if (i - k * sh.part >= sh.part || row[k] >= sh.rows) c[k] = sh.O + 8 * sl;  // nothing exists
        const int first = c[k] - 8 * sl;
        const T* p = X + int64_t(row[k]) * ldx + first + sl;
#pragma unroll
        for (int j = 0; j < 8; ++j) t[k][j] = first + j * kL + sl < sh.O ? to_f32(p[j * kL]) : 0.f;
    }
#pragma unroll
    for (int k = 0; k < kQuantizeParts; ++k) {
        float v[8];
        turn_to_groups<kL>(t[k], v, turn + 8 * (threadIdx.x - sl), sl);
        mx_store_block(v, max(0, min(8, sh.O - c[k])), Q.q4, Q.q + int64_t(row[k]) * Q.ldq + (Q.q4 ? c[k] / 2 : c[k]),
                       Q.s + int64_t(row[k]) * Q.lds + c[k] / kMxBlock, sh.vec_q);
    }
}

// Eight elements from byte q on as fp32, times their block's scale; nv of them exist.
__device__ __forceinline__ void decode8(const uint8_t* q, const uint8_t* s, bool q4, int nv, bool vec, float (&v)[8]) {
    uint32_t w[2] = {0u, 0u};
    if (vec && nv == 8) {
        if (q4) w[0] = __ldcs(reinterpret_cast<const uint32_t*>(q));
        else *reinterpret_cast<uint2*>(w) = __ldcs(reinterpret_cast<const uint2*>(q));
    } else {
        const int bytes = q4 ? (nv + 1) / 2 : nv;
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k < bytes) w[k >> 2] |= uint32_t(q[k]) << (8 * (k & 3));
    }
    const float scale = nv > 0 ? mx_scale_value(*s) : 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 f = mx_f16x2_to_f32(q4 ? mx_decode2_e2m1((w[0] >> (8 * j)) & 0xffu) : mx_decode2_e4m3((w[j >> 1] >> (16 * (j & 1))) & 0xffffu));
        v[2 * j] = f.x * scale;
        v[2 * j + 1] = f.y * scale;
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) mx_dequantize_kernel(MxView Q, Shape sh, T* __restrict__ Y, int64_t ldy) {
    float v[kDequantizeParts][8];
    int row[kDequantizeParts], c[kDequantizeParts];
    bool live[kDequantizeParts];
#pragma unroll
    for (int k = 0; k < kDequantizeParts; ++k) {
        const int i = int(blockIdx.x) * kThreads + int(threadIdx.x) + k * sh.part;
        row[k] = sh.by_row(i);
        c[k] = 8 * (i - row[k] * sh.per_row);
        live[k] = i - k * sh.part < sh.part && row[k] < sh.rows && c[k] < sh.O;
        if (live[k])
            decode8(Q.q + int64_t(row[k]) * Q.ldq + (Q.q4 ? c[k] / 2 : c[k]), Q.s + int64_t(row[k]) * Q.lds + c[k] / kMxBlock, Q.q4, 8, true, v[k]);
    }
#pragma unroll
    for (int k = 0; k < kDequantizeParts; ++k)
        if (live[k]) store8(Y + int64_t(row[k]) * ldy + c[k], v[k]);
}

template <typename T, int kL>
__global__ void __launch_bounds__(kThreads) mx_dequantize_columns_kernel(MxView Q, Shape sh, T* __restrict__ Y, int64_t ldy) {
    __shared__ __align__(16) float turn[8 * kThreads];
    const int sl = threadIdx.x % kL;
    float v[kDequantizeParts][8];
    int row[kDequantizeParts], c[kDequantizeParts];
#pragma unroll
    for (int k = 0; k < kDequantizeParts; ++k) {
        const int i = int(blockIdx.x) * kThreads + int(threadIdx.x) + k * sh.part;
        row[k] = sh.by_row(i);
        c[k] = 8 * (i - row[k] * sh.per_row);
        if (i - k * sh.part >= sh.part || row[k] >= sh.rows) c[k] = sh.O + 8 * sl;  // nothing exists
        decode8(Q.q + int64_t(row[k]) * Q.ldq + (Q.q4 ? c[k] / 2 : c[k]), Q.s + int64_t(row[k]) * Q.lds + c[k] / kMxBlock, Q.q4,
                max(0, min(8, sh.O - c[k])), sh.vec_q, v[k]);
    }
#pragma unroll
    for (int k = 0; k < kDequantizeParts; ++k) {
        float t[8];
        turn_to_columns<kL>(v[k], t, turn + 8 * (threadIdx.x - sl), sl);
        const int first = c[k] - 8 * sl;
        T* p = Y + int64_t(row[k]) * ldy + first + sl;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (first + j * kL + sl < sh.O) p[j * kL] = from_f32<T>(t[j]);
    }
}

bool rows_aligned(const void* p, int64_t ld_bytes, int64_t bytes) {
    return reinterpret_cast<uintptr_t>(p) % uintptr_t(bytes) == 0 && ld_bytes % bytes == 0;
}

// Calls launch(first row, shape, blocks, lanes) for slices of rows whose work numbers fit 31 bits; lanes = 0: aligned
// rows, else the kL of the other form.
template <typename T, class Fn>
cudaError_t sliced(const DenseView& X, int64_t rows, int O, const MxView& Q, int parts, Fn&& launch) {
    const bool vec_q = rows_aligned(Q.q, Q.ldq, Q.q4 ? 4 : 8);
    const bool vec = O % 8 == 0 && rows_aligned(X.p, X.ld * int64_t(sizeof(T)), 16) && vec_q;
    int span = 4;  // groups of eight columns
    if (!vec)
        while (span < 32 && 8 * span < O) span *= 2;
    const int per_row = (O + 8 * span - 1) / (8 * span) * span;
    const int64_t most = std::max<int64_t>(1, int64_t(0x7f000000) / per_row);
    for (int64_t r = 0; r < rows; r += most) {
        const int64_t n = std::min(most, rows - r);
        const int64_t part = (n * per_row / span + parts - 1) / parts * span;  // whole spans
        launch(r, Shape{int(n), O, per_row, int(part), Divisor(per_row), vec_q}, unsigned((part + kThreads - 1) / kThreads), vec ? 0 : span);
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
    return sliced<T>(X, rows, O, Q, kQuantizeParts, [&](int64_t r, const Shape& sh, unsigned blocks, int lanes) {
        const T* x = static_cast<const T*>(X.p) + r * X.ld;
        const MxView q = from_row(Q, r);
        if (lanes == 0) mx_quantize_kernel<T><<<blocks, kThreads, 0, st>>>(x, X.ld, sh, q);
        else if (lanes == 4) mx_quantize_columns_kernel<T, 4><<<blocks, kThreads, 0, st>>>(x, X.ld, sh, q);
        else if (lanes == 8) mx_quantize_columns_kernel<T, 8><<<blocks, kThreads, 0, st>>>(x, X.ld, sh, q);
        else if (lanes == 16) mx_quantize_columns_kernel<T, 16><<<blocks, kThreads, 0, st>>>(x, X.ld, sh, q);
        else mx_quantize_columns_kernel<T, 32><<<blocks, kThreads, 0, st>>>(x, X.ld, sh, q);
    });
}

template <typename T>
cudaError_t dequantize_t(const MxView& Q, int64_t rows, int O, const DenseView& Y, cudaStream_t st) {
    return sliced<T>(Y, rows, O, Q, kDequantizeParts, [&](int64_t r, const Shape& sh, unsigned blocks, int lanes) {
        T* y = static_cast<T*>(Y.p) + r * Y.ld;
        const MxView q = from_row(Q, r);
        if (lanes == 0) mx_dequantize_kernel<T><<<blocks, kThreads, 0, st>>>(q, sh, y, Y.ld);
        else if (lanes == 4) mx_dequantize_columns_kernel<T, 4><<<blocks, kThreads, 0, st>>>(q, sh, y, Y.ld);
        else if (lanes == 8) mx_dequantize_columns_kernel<T, 8><<<blocks, kThreads, 0, st>>>(q, sh, y, Y.ld);
        else if (lanes == 16) mx_dequantize_columns_kernel<T, 16><<<blocks, kThreads, 0, st>>>(q, sh, y, Y.ld);
        else mx_dequantize_columns_kernel<T, 32><<<blocks, kThreads, 0, st>>>(q, sh, y, Y.ld);
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
