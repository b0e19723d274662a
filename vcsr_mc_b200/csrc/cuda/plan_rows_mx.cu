// The rows plan with a microscaled (MX) dense operand: C (+)= A * B, B's rows held as E4M3 or E2M1
// elements with one power-of-two scale per 32 columns (mx.cuh).
//
//   C[i, c] (+)= scale * sum_j a_ij * elem[j, c] * 2^(S[j, c / 32] - 127)      sums in fp32
//
// A group of eight lanes owns one work unit of the row view (plan_rows.hpp) and one 128-column slab
// of C; a lane holds 16 columns (16 bytes of E4M3, 8 of E2M1: half a scale block). Entries are staged
// eight at a time in shared memory as (column, a * 2^e for each of the slab's four blocks), so the
// scale is applied once per entry and block and not in every lane. The four groups of a warp take
// their steps together (the trip count is the warp's largest), which keeps the warp converged.
// A row of C has one owner and is written once at its last entry; a chunk of a split row goes to a row
// of the workspace, and the chunks are added up in their order afterwards: the result does not
// depend on the order in which the groups run.
#include <cuda_runtime.h>

#include <algorithm>

#include "mx.cuh"
#include "mx.hpp"
#include "plan_rows.hpp"

namespace vcsrmc {
namespace dev {
namespace {

constexpr int kWarps = 4;           // per block
constexpr int kGroup = 8;           // lanes per unit
constexpr int kGroups = 32 / kGroup;
constexpr int kCols = 16;           // columns per lane
constexpr int kBatch = 8;           // entries staged and gathered at once
constexpr int kSlab = kGroup * kCols;
constexpr unsigned kFull = 0xffffffffu;
constexpr int kNever = 0x7fffffff;

struct alignas(16) StagedBatch {
    float4 a[kBatch];  // A value times the scale of each of the slab's four blocks
    int col[kBatch];
};

// acc (two columns) += a * b, both columns in one instruction
__device__ __forceinline__ void fma2(float2& acc, float a, float2 b) {
    unsigned long long d = *reinterpret_cast<unsigned long long*>(&acc);
    const float2 aa = make_float2(a, a);
    asm("fma.rn.f32x2 %0, %1, %2, %0;"
        : "+l"(d)
        : "l"(*reinterpret_cast<const unsigned long long*>(&aa)), "l"(*reinterpret_cast<const unsigned long long*>(&b)));
    acc = *reinterpret_cast<float2*>(&d);
}

// One lane's 16 elements of a row: kW 32-bit words.
template <bool k4>
struct Raw {
    static constexpr int kW = k4 ? 2 : 4;
    uint32_t w[kW];
};

// kWhole: p is aligned to the whole load and all its bytes belong to the row. Otherwise the row's
// `bytes` bytes from p are read as aligned 32-bit words, each of which holds at least one of them, and
// shifted into place.
template <bool k4, bool kWhole>
__device__ __forceinline__ Raw<k4> load_raw(const uint8_t* p, int bytes) {
    Raw<k4> r;
    if constexpr (kWhole) {
        if constexpr (k4) {
            const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
            r.w[0] = v.x;
            r.w[1] = v.y;
        } else {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
            r.w[0] = v.x;
            r.w[1] = v.y;
            r.w[2] = v.z;
            r.w[3] = v.w;
        }
    } else {
        const int m = int(reinterpret_cast<uintptr_t>(p) & 3);
        const uint32_t* q = reinterpret_cast<const uint32_t*>(p - m);
        uint32_t t[Raw<k4>::kW + 1];
#pragma unroll
        for (int i = 0; i <= Raw<k4>::kW; ++i) t[i] = 4 * i < m + bytes ? __ldg(q + i) : 0u;
#pragma unroll
        for (int i = 0; i < Raw<k4>::kW; ++i) r.w[i] = __funnelshift_r(t[i], t[i + 1], 8 * m);
    }
    return r;
}

template <bool k4>
__device__ __forceinline__ void fma_raw(float2 (&acc)[8], float a, const Raw<k4>& r) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t h = k4 ? mx_decode2_e2m1((r.w[k4 ? i >> 2 : 0] >> (8 * (i & 3))) & 0xffu)
                              : mx_decode2_e4m3((r.w[k4 ? 0 : i >> 1] >> (16 * (i & 1))) & 0xffffu);
        fma2(acc[i], a, mx_f16x2_to_f32(h));
    }
}

// Writes a lane's 16 columns (nv of them exist) times `scale`; kAdd adds them to C, whose row has this
// one writer.
template <bool kVec, bool kAdd>
__device__ __forceinline__ void write_row(float* dst, const float2 (&acc)[8], float scale, int nv) {
    const float* a = reinterpret_cast<const float*>(acc);
    if (kVec && nv == kCols) {
#pragma unroll
        for (int i = 0; i < kCols; i += 4) {
            const float4 v = make_float4(a[i] * scale, a[i + 1] * scale, a[i + 2] * scale, a[i + 3] * scale);
            if constexpr (kAdd) atomicAdd(reinterpret_cast<float4*>(dst + i), v);
            else __stcs(reinterpret_cast<float4*>(dst + i), v);
        }
    } else {
#pragma unroll
        for (int i = 0; i < kCols; ++i) {
            if (i < nv) {
                if constexpr (kAdd) atomicAdd(dst + i, a[i] * scale);
                else dst[i] = a[i] * scale;
            }
        }
    }
}

struct RowsMxArgs {
    const int4* units;
    int64_t n_units;
    const int* rp;
    const int* cols;
    const int* hot_cols;
    MxView B;
    int O;
    float* C;
    int64_t ldc;
    float scale;
    float* partial;
    bool scale_words;  // scale rows are 4-byte aligned
};

template <bool k4, bool kWhole, bool kVec, bool kAdd, typename VT>
__global__ void __launch_bounds__(kWarps * 32) rows_mx_kernel(RowsMxArgs P, const VT* __restrict__ vals) {
    __shared__ StagedBatch stage_all[kWarps * kGroups];
    const int lane = threadIdx.x & 31, sub = lane / kGroup, sl = lane % kGroup;
    StagedBatch& stage = stage_all[(threadIdx.x >> 5) * kGroups + sub];
    const int64_t unit = (int64_t(blockIdx.x) * kWarps + (threadIdx.x >> 5)) * kGroups + sub;
    const int4 u = unit < P.n_units ? P.units[unit] : make_int4(0, 0, 0, 0);
    const bool chunk = (u.y & 0x80000000) != 0;
    const int64_t pb = u.z;
    const int n = u.w - u.z;  // entries; positions below count from the unit's first
    const int slab = int(blockIdx.y) * kSlab;
    const int c0 = slab + kCols * sl;
    const int nv = max(0, min(kCols, P.O - c0));
    // a lane past the last column gathers the row's first columns and stores nothing
    const int cl = nv > 0 ? c0 : slab;
    const int bytes = k4 ? (min(kCols, P.O - cl) + 1) / 2 : min(kCols, P.O - cl);
    const uint8_t* q_base = P.B.q + (k4 ? cl / 2 : cl);
    const int block = nv > 0 ? sl / 2 : 0;  // scale block of the slab
    const uint8_t* s_base = P.B.s + slab / kMxBlock;
    const int blocks = min(4, (P.O - slab + kMxBlock - 1) / kMxBlock);
    const int ldq = int(P.B.ldq), lds = int(P.B.lds);

    int row = u.x;
    const int row_end = chunk ? row + 1 : (u.y & 0x7fffffff);
    // where the current row ends, and where the one after it does
    int end = row < row_end ? (chunk ? n : int(P.rp[row + 1] - pb)) : kNever;
    int end_next = row < row_end ? (chunk ? n : int(P.rp[min(row + 2, row_end)] - pb)) : kNever;
    float2 acc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = make_float2(0.f, 0.f);
    // stores the rows that end at position `at`: the open one, and the empty ones behind it
    auto close = [&](int at) {
        while (end == at) {
            if (chunk) write_row<false, false>(P.partial + unit * P.O + c0, acc, 1.f, nv);
            else write_row<kVec, kAdd>(P.C + int64_t(row) * P.ldc + c0, acc, P.scale, nv);
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] = make_float2(0.f, 0.f);
            ++row;
            end = row < row_end ? end_next : kNever;
            if (row < row_end) end_next = int(P.rp[min(row + 2, row_end)] - pb);
        }
    };
    close(0);

    // entry at position e: its column, A value and scale bytes
    auto load_entry = [&](int e, int& c, float& v) {
        c = 0;
        v = 0.f;
        if (e < n) {
            c = __ldcs(P.cols + pb + e);
            if constexpr (sizeof(VT) == 2) v = __half2float(__ushort_as_half(__ldcs(reinterpret_cast<const unsigned short*>(vals + pb + e))));
            else v = __ldcs(vals + pb + e);
        }
    };
    auto load_scales = [&](int e, int& c) -> uint32_t {
        if (e >= n) return 0u;
        if (c < 0) c = __ldg(P.hot_cols + ~c);  // a ranked hot column
        const uint8_t* s = s_base + int64_t(c) * lds;
        if (P.scale_words) return __ldg(reinterpret_cast<const uint32_t*>(s));
        uint32_t w = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b)
            if (b < blocks) w |= uint32_t(__ldg(s + b)) << (8 * b);
        return w;
    };
    int c_now, c_next;
    float v_now, v_next;
    load_entry(sl, c_now, v_now);
    load_entry(kBatch + sl, c_next, v_next);
    uint32_t s_now = load_scales(sl, c_now);
    const int longest = __reduce_max_sync(kFull, n);
    for (int q = 0; q < longest; q += kBatch) {
        float4 a;
        const bool live = q + sl < n;
        a.x = live ? v_now * mx_scale_value(s_now & 0xffu) : 0.f;
        a.y = live ? v_now * mx_scale_value((s_now >> 8) & 0xffu) : 0.f;
        a.z = live ? v_now * mx_scale_value((s_now >> 16) & 0xffu) : 0.f;
        a.w = live ? v_now * mx_scale_value(s_now >> 24) : 0.f;
        __syncwarp();
        stage.a[sl] = a;
        stage.col[sl] = c_now;
        __syncwarp();
        c_now = c_next;
        v_now = v_next;
        s_now = load_scales(q + kBatch + sl, c_now);
        load_entry(q + 2 * kBatch + sl, c_next, v_next);
        Raw<k4> raw[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) raw[j] = load_raw<k4, kWhole>(q_base + int64_t(stage.col[j]) * ldq, bytes);
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            fma_raw<k4>(acc, reinterpret_cast<const float*>(&stage.a[j])[block], raw[j]);
            close(q + j + 1);
        }
    }
}

// C's split rows: the sum of their chunks, in order. One block per (split row, 128 columns); its eight
// warps take every eighth chunk.
__global__ void __launch_bounds__(256) join_chunks_kernel(const int4* __restrict__ units, int n_chunks, const int* __restrict__ split_rows,
                                                          const float* __restrict__ partial, int O, float* __restrict__ C, int64_t ldc,
                                                          float scale, int accumulate) {
    __shared__ float part[8][128];
    const int row = split_rows[blockIdx.x];
    // first chunk of the row: units are listed by row
    int lo = 0, hi = n_chunks;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (units[mid].x < row) lo = mid + 1;
        else hi = mid;
    }
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int k = 0; k < 4; ++k) {
        const int c = int(blockIdx.y) * 128 + 32 * k + lane;
        float v = 0.f;
        if (c < O)
            for (int i = lo + warp; i < n_chunks && units[i].x == row; i += 8) v += partial[int64_t(i) * O + c];
        part[warp][32 * k + lane] = v;
    }
    __syncthreads();
    const int c = int(blockIdx.y) * 128 + int(threadIdx.x);
    if (threadIdx.x < 128 && c < O) {
        float v = 0.f;
        for (int i = 0; i < 8; ++i) v += part[i][threadIdx.x];
        float* dst = C + int64_t(row) * ldc + c;
        *dst = accumulate ? *dst + v * scale : v * scale;
    }
}

template <bool k4, bool kWhole, bool kVec, typename VT>
cudaError_t launch(const RowsMxArgs& a, const VT* vals, bool accumulate, cudaStream_t st) {
    const int64_t per_block = kWarps * kGroups;
    const int64_t blocks = (a.n_units + per_block - 1) / per_block;
    const int slabs = (a.O + kSlab - 1) / kSlab;
    if (blocks > 0x7fffffffLL || slabs > 65535) return cudaErrorInvalidValue;
    const dim3 grid(unsigned(blocks), unsigned(slabs), 1);
    if (accumulate) rows_mx_kernel<k4, kWhole, kVec, true, VT><<<grid, kWarps * 32, 0, st>>>(a, vals);
    else rows_mx_kernel<k4, kWhole, kVec, false, VT><<<grid, kWarps * 32, 0, st>>>(a, vals);
    return cudaGetLastError();
}

template <bool k4, typename VT>
cudaError_t launch_v(const RowsMxArgs& a, const VT* vals, bool accumulate, cudaStream_t st) {
    const int64_t full = k4 ? 8 : 16;
    const bool whole = a.O % kCols == 0 && reinterpret_cast<uintptr_t>(a.B.q) % full == 0 && a.B.ldq % full == 0;
    const bool vec = reinterpret_cast<uintptr_t>(a.C) % 16 == 0 && a.ldc % 4 == 0;
    if (whole) return vec ? launch<k4, true, true>(a, vals, accumulate, st) : launch<k4, true, false>(a, vals, accumulate, st);
    return vec ? launch<k4, false, true>(a, vals, accumulate, st) : launch<k4, false, false>(a, vals, accumulate, st);
}

}  // namespace

cudaError_t spmm_rows_mx(const RowPlanView& P, const MxView& B, int O, float* C, int64_t ldc, bool accumulate,
                         float* partial, cudaStream_t st) {
    if (P.n_units == 0) {
        if (!accumulate && P.M > 0) return cudaMemset2DAsync(C, size_t(ldc) * 4, 0, size_t(O) * 4, size_t(P.M), st);
        return cudaSuccess;
    }
    RowsMxArgs a;
    a.units = P.units;
    a.n_units = P.n_units;
    a.rp = P.rp;
    a.cols = P.cols;
    a.hot_cols = P.hot.hot_cols;
    a.B = B;
    a.O = O;
    a.C = C;
    a.ldc = ldc;
    a.scale = P.scale;
    a.partial = partial;
    a.scale_words = reinterpret_cast<uintptr_t>(B.s) % 4 == 0 && B.lds % 4 == 0;
    cudaError_t e;
    if (P.vals_f16) {
        const __half* v = static_cast<const __half*>(P.vals);
        e = B.q4 ? launch_v<true>(a, v, accumulate, st) : launch_v<false>(a, v, accumulate, st);
    } else {
        const float* v = static_cast<const float*>(P.vals);
        e = B.q4 ? launch_v<true>(a, v, accumulate, st) : launch_v<false>(a, v, accumulate, st);
    }
    if (e != cudaSuccess || P.n_split_rows == 0) return e;
    join_chunks_kernel<<<dim3(unsigned(P.n_split_rows), unsigned((O + 127) / 128)), 256, 0, st>>>(
        P.units, int(P.n_chunks), P.split_rows, partial, O, C, ldc, P.scale, accumulate ? 1 : 0);
    return cudaGetLastError();
}

}  // namespace dev
}  // namespace vcsrmc
