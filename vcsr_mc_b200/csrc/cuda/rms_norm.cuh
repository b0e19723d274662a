// Residual addition with root-mean-square norm, written as a microscaled (MX) matrix, and its
// backward pass. For a row of O columns:
//   s = round(x + residual)              (to the residual's type; the next residual)
//   inv = 1 / sqrt(mean(s^2) + eps)
//   Q = MX(s * inv * w)                  (mx.cuh)
// and with dy the gradient of the values that Q stands for (the element's rounding counts as identity),
// n = s * inv and g = dy * w:
//   dx = d_residual + inv * (g - n * mean(g * n))
//   dw = sum over rows of dy * n
// The square sums are held in 64 bits: fp32 would overflow for |s| above 2^64, which bf16 and fp32 can
// hold; the backward pass sums products of the normalised n, which cannot. Both passes read each input
// once and write each output once (a row is held up to 16384 columns forward and 8192 backward, and is read a second
// time beyond), so HBM bounds them except for a few rows, and for 4097 to 8192 columns backward: sixteen columns a
// thread do not fit its 64 registers there (504 to 912 bytes of spills) and the row goes through local memory. On a B200
// (copies run at 6.5 TB/s): forward, 2^20 rows of 128, fp32 X and fp16 residual to E4M3, 191 us (6.4 TB/s); 16384 rows of
// 4096 in bf16, 90 us (5.2 TB/s); both up to 27 us more where one of the last rows has a block that rewrite_block takes;
// 20011 rows of 1009 (single columns, bound by instructions), 43 us (4.2 TB/s); one row of 4096, 4.4 us.
// Backward, 32768 rows of 4096 in bf16, 187 us (5.7 TB/s); 16384 rows of 8192, 526 us (2.0 TB/s), of 5001 (single
// columns), 720 us; 2^20 rows of 128, fp32 dY, fp16 else, 244 us (5.5 TB/s); 4096 rows of 128, 8.4 us.
#pragma once
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "mx.cuh"
#include "mx.hpp"
#include "vcsrmc.h"

namespace vcsrmc {
namespace dev {
namespace norm {

// How a row lies over threads: kN columns per thread, in groups of eight, on kL lanes of a warp or, for kL = 0, on
// the whole block. kN = 0: any width in steps of 8, the row is read twice. kV = 8: a group is eight consecutive
// columns (16-byte loads and stores; O is a multiple of 8 and every row aligned). kV = 1, for every other layout:
// the columns of neighbouring threads' groups are dealt out over them in turn, so that single loads and stores are
// coalesced; a block of scales needs them turned into consecutive ones (turn_to_groups).
template <int kV_, int kL_, int kN_, int kThreads_ = 256>
struct Span {
    static constexpr int kV = kV_, kL = kL_;
    static constexpr bool kAny = kN_ == 0;
    static constexpr int kN = kAny ? 8 : kN_;      // columns held at once
    static constexpr int kThreads = kThreads_;     // per block, at most
    static constexpr int kRows = kL_ ? 256 / (kL_ ? kL_ : 1) : 1;  // rows in a block
    static constexpr int kW = kL_ ? kL_ : 32;      // threads whose groups are neighbours
    // forward blocks per SM that the registers are held to: with eight columns a thread, all of an SM's threads (2^20
    // rows of 128: 191 against 202 us); with 16 in blocks of up to 512, three blocks (16384 rows of 4096, with a late block
    // that is written again: 110 against 115 us with four and 122 with two)
    static constexpr int kForwardBlocks = !kAny && kN == 8 ? 2048 / kThreads : kThreads == 512 ? 3 : 1;
    static_assert(kN % 8 == 0, "whole groups");
    __device__ static int per_row() { return kL ? kL : int(blockDim.x); }
    __device__ static int slot() { return kL ? int(threadIdx.x) % (kL ? kL : 1) : int(threadIdx.x); }
    __device__ static int row_in_block() { return kL ? int(threadIdx.x) / (kL ? kL : 1) : 0; }
    // first column of this thread's group g, `step` kN-wide steps into the row
    __device__ static int group(int g, int step = 0) { return 8 * ((step * (kN / 8) + g) * per_row() + slot()); }
    // column of its element i
    __device__ static int column(int i, int step = 0) {
        if (kV == 8) return group(i / 8, step) + i % 8;
        return group(i / 8, step) - 8 * (slot() % kW) + (i % 8) * kW + slot() % kW;
    }
};

// A thread's columns as they were read; converted when they are used, so that all loads are in flight first.
// kWide: fp32, else fp16 or bf16 (two to a word where a thread holds groups of eight).
template <class S, bool kWide>
struct Held {
    static constexpr int kPer = S::kV == 8 && !kWide ? 2 : 1;  // elements per word
    uint32_t w[S::kN / kPer];
};

template <class S, bool kWide>
__device__ __forceinline__ void load(Held<S, kWide>& r, const DenseView& v, int64_t row, int O, int step = 0) {
    using T = typename std::conditional<kWide, uint32_t, unsigned short>::type;
    const T* p = static_cast<const T*>(v.p) + row * v.ld;
#pragma unroll
    for (int i = 0; i < S::kN; i += S::kV) {
        const int c = S::column(i, step);
        if constexpr (S::kV == 8) {
#pragma unroll
            for (int k = 0; k < (kWide ? 2 : 1); ++k) {
                const uint4 a = c < O ? __ldcs(reinterpret_cast<const uint4*>(p + c) + k) : make_uint4(0, 0, 0, 0);
                uint32_t* w = r.w + i / Held<S, kWide>::kPer + 4 * k;
                w[0] = a.x;
                w[1] = a.y;
                w[2] = a.z;
                w[3] = a.w;
            }
        } else {
            r.w[i] = c < O ? p[c] : 0u;
        }
    }
}

// Calls fn with the element type of a dense dtype (kWide says which are possible). The type is uniform, so this
// is one branch around the loops of a row and not one in them.
template <bool kWide, class Fn>
__device__ __forceinline__ void with_type(int dtype, Fn&& fn) {
    if constexpr (kWide) fn(float{});
    else if (dtype == VCSRMC_F16) fn(__half{});
    else fn(__nv_bfloat16{});
}

template <class S, bool kWide>
__device__ __forceinline__ void to_floats(const Held<S, kWide>& r, int dtype, float (&v)[S::kN]) {
    with_type<kWide>(dtype, [&](auto t) {
        using T = decltype(t);
#pragma unroll
        for (int i = 0; i < S::kN; ++i) v[i] = to_f32(reinterpret_cast<const T*>(&r.w[i / Held<S, kWide>::kPer])[i % Held<S, kWide>::kPer]);
    });
}

template <class S, bool kWide>
__device__ __forceinline__ void store(const float (&v)[S::kN], const DenseView& d, int64_t row, int O, int step = 0) {
    with_type<kWide>(d.dtype, [&](auto t) {
        using T = decltype(t);
        T* p = static_cast<T*>(d.p) + row * d.ld;
#pragma unroll
        for (int i = 0; i < S::kN; i += S::kV) {
            const int c = S::column(i, step);
            if (c >= O) continue;
            if constexpr (S::kV == 8) {
                float u[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) u[k] = v[i + k];
                store8(p + c, u);
            } else {
                p[c] = from_f32<T>(v[i]);
            }
        }
    });
}

// The weights of a thread's columns (0 past the row's end).
template <class S>
__device__ __forceinline__ void load_weights(float (&w)[S::kN], const void* weight, int dtype, bool vec, int O, int step = 0) {
    auto read = [&](auto t) {
        using T = decltype(t);
        const T* p = static_cast<const T*>(weight);
#pragma unroll
        for (int i = 0; i < S::kN; i += S::kV) {
            const int c = S::column(i, step);
            if constexpr (S::kV == 8) {
                float u[8];
                load8(p + c, c < O ? 8 : 0, vec, u);
#pragma unroll
                for (int k = 0; k < 8; ++k) w[i + k] = u[k];
            } else {
                w[i] = c < O ? to_f32(p[c]) : 0.f;
            }
        }
    };
    if (dtype == VCSRMC_F32) read(float{});
    else with_type<false>(dtype, read);
}

// Sum over the lanes of a row, or over the block (kL = 0); every thread gets the result. The order of the
// additions depends on the thread count alone.
template <class S, typename T>
__device__ __forceinline__ T row_sum(T v, T* smem) {
    constexpr int kW = S::kL == 0 ? 32 : S::kL;
#pragma unroll
    for (int d = kW / 2; d >= 1; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    if constexpr (S::kL == 0) {
        const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
        __syncthreads();  // smem may still be read from the row before
        if (lane == 0) smem[threadIdx.x >> 5] = v;
        __syncthreads();
        v = lane < warps ? smem[lane] : T(0);
#pragma unroll
        for (int d = 16; d >= 1; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    }
    return v;
}

// 1 / sqrt(v): the hardware's estimate and a Newton step in 64 bits (its error squared,
// below 2^-40), or 64-bit operations where v leaves the estimate's range.
__device__ __forceinline__ double inverse_root(double v) {
    if (v > 1e-30 && v < 1e30) {
        const double r = double(rsqrtf(float(v)));
        return r * (1.5 - 0.5 * v * r * r);
    }
    return 1.0 / sqrt(v);
}

__device__ __forceinline__ float read_as(const DenseView& d, int64_t row, int c) {
    const int64_t i = row * d.ld + c;
    if (d.dtype == VCSRMC_F32) return static_cast<const volatile float*>(d.p)[i];
    const unsigned short h = static_cast<const volatile unsigned short*>(d.p)[i];
    return d.dtype == VCSRMC_F16 ? __half2float(__ushort_as_half(h)) : __bfloat162float(__ushort_as_bfloat16(h));
}

// Writes the block from column c on again, its scale from the largest |s * root * w| in 64 bits: for a block whose
// largest value in fp32 is next to a border between scales. One thread, from memory, and a call of its own: a block
// in a million needs it, and in the kernel's registers it would cost all of them (218 against 191 us for 2^20 rows
// of 128). The call takes about 25 us, which shows where it falls to one of the last rows (the same rows: 191 and 215 us;
// 16384 rows of 4096: 90 and up to 116 us).
static __device__ __noinline__ void rewrite_block(const RmsNormArgs& a, int64_t row, int c, double root) {
    const float inv = float(root);
    const DenseView weight{const_cast<void*>(a.weight), a.w_dtype, 0};
    const int n = min(kMxBlock, a.O - c);
    auto sum = [&](int i) {
        if (a.residual_out.p) return read_as(a.residual_out, row, c + i);
        const float v = read_as(a.x, row, c + i) + (a.residual.p ? read_as(a.residual, row, c + i) : 0.f);
        if (a.residual_out.dtype == VCSRMC_F32) return v;
        return a.residual_out.dtype == VCSRMC_F16 ? __half2float(__float2half_rn(v)) : __bfloat162float(__float2bfloat16_rn(v));
    };
    double exact = 0.0;
    float amax = 0.f;
    for (int i = 0; i < n; ++i) {
        const float v = sum(i), w = read_as(weight, 0, c + i);
        exact = fmax(exact, fabs(double(v) * root * double(w)));
        amax = fmaxf(amax, fabsf(v * inv * w));
    }
    const uint32_t border = (__float_as_uint(amax) & 0x7f800000u) | (a.out.q4 ? 0x400000u : 0x600000u);
    const uint32_t code = mx_scale_code(exact > double(__uint_as_float(border)) ? border + 1u : border, a.out.q4);
    const float scale = mx_inverse_scale(code);
    uint8_t* q = a.out.q + row * a.out.ldq;
    a.out.s[row * a.out.lds + c / kMxBlock] = uint8_t(code);
    for (int i = 0; i < n; i += 2) {
        float y[2] = {0.f, 0.f};
        for (int k = 0; k < 2 && i + k < n; ++k) y[k] = sum(i + k) * inv * read_as(weight, 0, c + i + k) * scale;
        if (a.out.q4) {
            q[(c + i) / 2] = uint8_t(mx_encode2_e2m1(y[0], y[1]));
        } else {
            const uint32_t two = mx_encode2_e4m3(y[0], y[1]);
            q[c + i] = uint8_t(two);
            if (i + 1 < n) q[c + i + 1] = uint8_t(two >> 8);
        }
    }
}

template <class S, bool kXWide, bool kRWide>
__global__ void __launch_bounds__(S::kThreads, S::kForwardBlocks) rms_norm_kernel(const __grid_constant__ RmsNormArgs a) {
    __shared__ double smem[32], roots[S::kL ? S::kRows : 32];
    extern __shared__ __align__(16) float turn[];  // kV = 1: eight floats a thread
    const int64_t row = int64_t(blockIdx.x) * S::kRows + S::row_in_block();
    const bool live = row < a.rows;  // every thread takes part in the reductions of a row past the end
    const int O = live ? a.O : 0;
    const int r_dtype = a.residual_out.dtype;
    const int steps = S::kAny ? (a.O + S::kN * S::per_row() - 1) / (S::kN * S::per_row()) : 1;
    float s[S::kN];
    auto load_sum = [&](int step) {
        Held<S, kXWide> x;
        Held<S, kRWide> r;
        load(x, a.x, row, O, step);
        if (a.residual.p) {
            load(r, a.residual, row, O, step);
            float t[S::kN];
            to_floats(x, a.x.dtype, s);
            to_floats(r, r_dtype, t);
#pragma unroll
            for (int i = 0; i < S::kN; ++i) s[i] += t[i];
        } else {
            to_floats(x, a.x.dtype, s);
        }
        with_type<kRWide>(r_dtype, [&](auto t) {
#pragma unroll
            for (int i = 0; i < S::kN; ++i) s[i] = to_f32(from_f32<decltype(t)>(s[i]));
        });
    };
    double sum = 0.0;
    for (int k = 0; k < steps; ++k) {
        load_sum(k);
#pragma unroll
        for (int i = 0; i < S::kN; ++i) sum = fma(double(s[i]), double(s[i]), sum);
    }
    sum = row_sum<S>(sum, smem);
    const double root = inverse_root(sum / double(a.O) + double(a.eps));
    const float inv = float(root);
    // for rewrite_block, kept out of the registers; one for a warp's own use where it shares a row
    const int root_at = S::kL ? S::row_in_block() : int(threadIdx.x >> 5);
    if (S::slot() % 32 == 0) roots[root_at] = root;
    if (live && S::slot() == 0 && a.inv_rms) a.inv_rms[row] = inv;
    uint8_t* q = a.out.q + row * a.out.ldq;
    uint8_t* scales = a.out.s + row * a.out.lds;
    for (int k = 0; k < steps; ++k) {
        if constexpr (S::kAny) load_sum(k);
        if (a.residual_out.p) store<S, kRWide>(s, a.residual_out, row, O, k);
        float w[S::kN];
        load_weights<S>(w, a.weight, a.w_dtype, a.vec_w, O, k);
        uint32_t again = 0;  // groups whose block is next to a border between scales
#pragma unroll
        for (int i = 0; i < S::kN; i += 8) {
            float y[8], t[8];
            bool near;
#pragma unroll
            for (int j = 0; j < 8; ++j) t[j] = s[i + j] * inv * w[i + j];
            const int c = S::group(i / 8, k);
            if constexpr (S::kV == 1) {
                turn_to_groups<S::kW>(t, y, turn + 8 * (threadIdx.x - S::slot() % S::kW), S::slot() % S::kW);
                near = mx_store_block(y, max(0, min(8, O - c)), a.out.q4, q + (a.out.q4 ? c / 2 : c), scales + c / kMxBlock, a.vec_q);
            } else {
                near = mx_store_block(t, c < O ? 8 : 0, a.out.q4, q + (a.out.q4 ? c / 2 : c), scales + c / kMxBlock, true);
            }
            if (near) again |= 1u << (i / 8);
        }
        if (__any_sync(0xffffffffu, again != 0)) {
            __syncwarp();  // the block's values and first bytes are written
            if (S::slot() % 4 == 0)
                for (int g = 0; g < S::kN / 8; ++g)
                    if ((again >> g) & 1u) rewrite_block(a, row, S::group(g, k), roots[root_at]);
        }
    }
}

// ---- backward --------------------------------------------------------------------------------------
// Persistent blocks over the rows; each thread keeps the weight gradient of its columns in registers
// and the block writes one row of partial sums to the workspace, in which a second kernel adds the
// blocks up in their order. Registers are held to 64 a thread: the pass waits for memory, and 1024 threads per SM
// hide it better than 512 with more registers (rows of 128: 233 against 265 us, of 4096: 234 against 347 us). With sixteen
// columns a thread that bound spills (see the top); the other side of it is not measured there.
template <class S, bool kYWide, bool kRWide>
__global__ void __launch_bounds__(S::kThreads, S::kL ? 4 : 2) rms_norm_grad_kernel(RmsNormGradArgs a) {
    __shared__ float smem[32];
    __shared__ float fold[S::kL ? 8 : 1][S::kL ? 257 : 1];
    const int steps = S::kAny ? (a.O + S::kN * S::per_row() - 1) / (S::kN * S::per_row()) : 1;
    float* part = a.workspace + int64_t(blockIdx.x) * a.O;
    float dw[S::kN] = {}, w[S::kN];
    if constexpr (!S::kAny) load_weights<S>(w, a.weight, a.w_dtype, a.vec_w, a.O);
    const int64_t stride = int64_t(gridDim.x) * S::kRows;
    Held<S, kYWide> dy;
    Held<S, kRWide> h, dr;
    float inv = 0.f;
    // the inputs of a row's step; rows past the end read nothing and count as zeros
    auto load_row = [&](int64_t row, int k, bool residual) {
        const int O = row < a.rows ? a.O : 0;
        inv = row < a.rows ? a.inv_rms[row] : 0.f;
        load(dy, a.dy, row, O, k);
        load(h, a.hidden, row, O, k);
        if (residual && a.d_residual.p) load(dr, a.d_residual, row, O, k);
    };
    int64_t row = int64_t(blockIdx.x) * S::kRows + S::row_in_block();
    // a block's row: the next row's inputs are loaded over this one's reduction and stores (rows of 4096: 189
    // against 235 us); warps' rows overlap one another, and the registers would cost more (rows of 128: 334
    // against 236 us)
    constexpr bool kAhead = !S::kAny && S::kL == 0;
    if constexpr (kAhead) load_row(row, 0, true);
    for (int64_t r0 = int64_t(blockIdx.x) * S::kRows; r0 < a.rows; r0 += stride, row += stride) {
        const int O = row < a.rows ? a.O : 0;
        float vy[S::kN], vh[S::kN], dx[S::kN] = {};
        // the gradient g = dy * w is 0 past the row's end, where w is, and so are its products
        float dot = 0.f;
        for (int k = 0; k < steps; ++k) {
            if constexpr (!kAhead) load_row(row, k, !S::kAny);
            if constexpr (S::kAny) load_weights<S>(w, a.weight, a.w_dtype, a.vec_w, O, k);
            to_floats(dy, a.dy.dtype, vy);
            to_floats(h, a.hidden.dtype, vh);
#pragma unroll
            for (int i = 0; i < S::kN; ++i) {
                vh[i] *= inv;
                dot = fmaf(vy[i] * w[i], vh[i], dot);
            }
        }
        const float inv_row = inv;
        if constexpr (kAhead) {
            if (a.d_residual.p) to_floats(dr, a.hidden.dtype, dx);
            load_row(row + stride, 0, true);
        }
        const float m = row_sum<S>(dot, smem) / float(a.O);
        for (int k = 0; k < steps; ++k) {
            if constexpr (S::kAny) {
                load_row(row, k, true);
                load_weights<S>(w, a.weight, a.w_dtype, a.vec_w, O, k);
                to_floats(dy, a.dy.dtype, vy);
                to_floats(h, a.hidden.dtype, vh);
#pragma unroll
                for (int i = 0; i < S::kN; ++i) vh[i] *= inv;
            }
            if (!kAhead && a.d_residual.p) to_floats(dr, a.hidden.dtype, dx);
#pragma unroll
            for (int i = 0; i < S::kN; ++i) {
                dx[i] = fmaf(inv_row, fmaf(vy[i], w[i], -(vh[i] * m)), dx[i]);
                if constexpr (S::kAny) {
                    const int c = S::column(i, k);
                    if (c < O) part[c] = fmaf(vy[i], vh[i], r0 == int64_t(blockIdx.x) ? 0.f : part[c]);
                } else {
                    dw[i] = fmaf(vy[i], vh[i], dw[i]);
                }
            }
            store<S, kRWide>(dx, a.dx, row, O, k);
            if constexpr (S::kAny) {
#pragma unroll
                for (int i = 0; i < S::kN; ++i) dx[i] = 0.f;
            }
        }
    }
    if constexpr (!S::kAny && S::kL > 0) {
        // sum over the rows of the block, in their order, eight elements of every thread at a time
#pragma unroll
        for (int i0 = 0; i0 < S::kN; i0 += 8) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 8; ++i) fold[i][threadIdx.x] = dw[i0 + i];
            __syncthreads();
            for (int t = int(threadIdx.x); t < S::kL * 8; t += 256) {
                const int i = t / S::kL, slot = t % S::kL;
                const int c = i0 * S::kL + (S::kV == 8 ? 8 * slot + i : i * S::kL + slot);
                if (c < a.O) {
                    float v = 0.f;
                    for (int g = 0; g < S::kRows; ++g) v += fold[i][g * S::kL + slot];
                    part[c] = v;
                }
            }
        }
    } else if constexpr (!S::kAny) {
#pragma unroll
        for (int i = 0; i < S::kN; ++i)
            if (S::column(i) < a.O) part[S::column(i)] = dw[i];
    }
}

inline bool aligned(const void* p, int64_t ld_bytes, int64_t to) {
    return reinterpret_cast<uintptr_t>(p) % uintptr_t(to) == 0 && ld_bytes % to == 0;
}
inline bool aligned16(const DenseView& v) { return aligned(v.p, v.ld * (v.dtype == VCSRMC_F32 ? 4 : 2), 16); }

// Threads that hold O columns, n each, in whole warps.
inline int threads_for(int O, int n) { return ((O + n - 1) / n + 31) / 32 * 32; }
// Threads of a backward block that holds one row (O > 256): 8 columns each up to 4096 columns, 16 up to 8192 (512
// threads of 8 hold 4096).
inline int grad_threads(int O) { return std::min(512, threads_for(O, O <= 4096 ? 8 : 16)); }

template <class S, bool kXWide, bool kRWide>
cudaError_t launch_norm(const RmsNormArgs& a, int threads, cudaStream_t st) {
    const int64_t blocks = (a.rows + S::kRows - 1) / S::kRows;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
    const int n = S::kL ? 256 : threads;
    rms_norm_kernel<S, kXWide, kRWide><<<unsigned(blocks), n, S::kV == 1 ? 8 * n * sizeof(float) : 0, st>>>(a);
    return cudaGetLastError();
}

template <class S, bool kYWide, bool kRWide>
cudaError_t launch_grad(const RmsNormGradArgs& a, int threads, int64_t blocks, cudaStream_t st) {
    rms_norm_grad_kernel<S, kYWide, kRWide><<<unsigned(blocks), S::kL ? 256 : threads, 0, st>>>(a);
    return cudaGetLastError();
}

template <int kV, bool kXWide, bool kRWide>
cudaError_t forward_spans(const RmsNormArgs& a, cudaStream_t st) {
    const int O = a.O;
    if (O <= 32) return launch_norm<Span<kV, 4, 8>, kXWide, kRWide>(a, 0, st);
    if (O <= 64) return launch_norm<Span<kV, 8, 8>, kXWide, kRWide>(a, 0, st);
    if (O <= 128) return launch_norm<Span<kV, 16, 8>, kXWide, kRWide>(a, 0, st);
    if (O <= 256) return launch_norm<Span<kV, 32, 8>, kXWide, kRWide>(a, 0, st);
    if (O <= 512) return launch_norm<Span<kV, 32, 16>, kXWide, kRWide>(a, 0, st);
    if (O <= 1024) return launch_norm<Span<kV, 0, 8, 128>, kXWide, kRWide>(a, threads_for(O, 8), st);
    // 16 columns a thread: 8 in twice the threads take 103 against 90 us on 16384 rows of 4096, 68 against 65 us on rows
    // of 2048, and as long on one row
    if (O <= 8 * 1024) return launch_norm<Span<kV, 0, 16, 512>, kXWide, kRWide>(a, threads_for(O, 16), st);
    if (O <= 16 * 1024) return launch_norm<Span<kV, 0, 16, 1024>, kXWide, kRWide>(a, threads_for(O, 16), st);
    return launch_norm<Span<kV, 0, 0, 1024>, kXWide, kRWide>(a, 1024, st);
}

template <int kV, bool kYWide, bool kRWide>
cudaError_t backward_spans(const RmsNormGradArgs& a, int64_t blocks, cudaStream_t st) {
    const int O = a.O, threads = grad_threads(O);
    if (O <= 32) return launch_grad<Span<kV, 4, 8>, kYWide, kRWide>(a, 0, blocks, st);
    if (O <= 64) return launch_grad<Span<kV, 8, 8>, kYWide, kRWide>(a, 0, blocks, st);
    if (O <= 128) return launch_grad<Span<kV, 16, 8>, kYWide, kRWide>(a, 0, blocks, st);
    if (O <= 256) return launch_grad<Span<kV, 32, 8>, kYWide, kRWide>(a, 0, blocks, st);
    if (O <= 4096) return launch_grad<Span<kV, 0, 8, 512>, kYWide, kRWide>(a, threads, blocks, st);
    if (O <= 8192) return launch_grad<Span<kV, 0, 16, 512>, kYWide, kRWide>(a, threads, blocks, st);
    return launch_grad<Span<kV, 0, 0, 512>, kYWide, kRWide>(a, threads, blocks, st);
}

// The launches of one pair of element widths (X or dY, residual); each pair is a translation unit.
template <bool kXWide, bool kRWide>
cudaError_t forward(const RmsNormArgs& a, cudaStream_t st) {
    const bool vec = a.O % 8 == 0 && aligned16(a.x) && (!a.residual.p || aligned16(a.residual)) &&
                     (!a.residual_out.p || aligned16(a.residual_out)) && a.vec_q;
    return vec ? forward_spans<8, kXWide, kRWide>(a, st) : forward_spans<1, kXWide, kRWide>(a, st);
}

template <bool kYWide, bool kRWide>
cudaError_t backward(const RmsNormGradArgs& a, int64_t blocks, cudaStream_t st) {
    const bool vec = a.O % 8 == 0 && aligned16(a.dy) && aligned16(a.hidden) && aligned16(a.dx) && (!a.d_residual.p || aligned16(a.d_residual));
    return vec ? backward_spans<8, kYWide, kRWide>(a, blocks, st) : backward_spans<1, kYWide, kRWide>(a, blocks, st);
}

extern template cudaError_t forward<true, true>(const RmsNormArgs&, cudaStream_t);
extern template cudaError_t forward<true, false>(const RmsNormArgs&, cudaStream_t);
extern template cudaError_t forward<false, false>(const RmsNormArgs&, cudaStream_t);
extern template cudaError_t backward<true, true>(const RmsNormGradArgs&, int64_t, cudaStream_t);
extern template cudaError_t backward<true, false>(const RmsNormGradArgs&, int64_t, cudaStream_t);
extern template cudaError_t backward<false, false>(const RmsNormGradArgs&, int64_t, cudaStream_t);

}  // namespace norm
}  // namespace dev
}  // namespace vcsrmc
