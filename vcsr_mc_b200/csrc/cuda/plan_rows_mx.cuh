// The rows plan with a microscaled (MX) dense operand: C (+)= A * B, B's rows held as E4M3 or E2M1
// elements with one power-of-two scale per 32 columns (mx.cuh).
//
//   C[i, c] (+)= scale * sum_j a_ij * elem[j, c] * 2^(S[j, c / 32] - 127)      sums in fp32
//
// A group of 4, 8 or 16 lanes owns one work unit of the row view (plan_rows.hpp) and one slab of 32, 64 or
// 128 columns of C; a lane holds 8 or 16 columns. Entries are staged 8 or 16 at a time in shared memory as
// (column, a * 2^e for each of the slab's blocks), so the scale is applied once per entry and block and not in
// every lane. The groups of a warp take their steps together (the trip count is the warp's largest), which keeps the
// warp converged. A row of C has one owner and is written once at its last entry; a chunk of a split row goes
// to a row of the workspace, and the chunks are added up in their order afterwards (join_chunks_kernel):
// the result does not depend on the order in which the groups run.
//
// On a B200, O = 128 and E2M1, issue bounds both of the large cases: the 27-point stencil on 100^3 (26.5 M entries)
// takes 0.411 ms, 51 instructions per warp for four entries, 30 of them decoding and multiplying, at 2.99 per clock
// and SM; the 2^20-row R-MAT (16.2 M entries) 0.400 ms, 72 for four entries at 2.83, because a warp takes as many steps as
// the longest of its groups (1.28 per entry, by its units). L2 is at 37 and 44 % of its throughput, DRAM at 24 and 23 %;
// A and C move once, and 739 and 706 MB would take 0.113 and 0.108 ms at the copy rate.
#pragma once
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "mx.cuh"
#include "mx.hpp"
#include "plan_rows.hpp"

namespace vcsrmc {
namespace dev {
namespace rows_mx {

constexpr int kWarps = 4;  // per block
constexpr unsigned kFull = 0xffffffffu;
constexpr int kNever = 0x7fffffff;

// How a slab of C is laid over lanes: kGroup lanes own a work unit and kGroup * kCols columns, kCols
// of them per lane; kFlight entries are gathered at once.
template <int kGroup_, int kCols_, int kFlight_>
struct Lanes {
    static constexpr int kGroup = kGroup_, kCols = kCols_, kFlight = kFlight_;
    static constexpr int kGroups = 32 / kGroup;            // units per warp
    static constexpr int kSlab = kGroup * kCols;           // columns
    static constexpr int kBlocks = kSlab / kMxBlock;       // scale blocks of the slab
    static constexpr int kBatch = kGroup > 8 ? kGroup : 8;  // entries staged at once
    static constexpr int kPer = kBatch / kGroup;           // entries a lane stages
};

// A batch of entries as a group stages it: columns, and for each of the slab's blocks the A values times
// the block's scale, in fp16 (in the first half of the place) or fp32.
template <int kBlocks, int kBatch>
struct alignas(16) Stage {
    int col[kBatch];
    uint32_t a[kBlocks][kBatch];
    __device__ unsigned short* half(int block) { return reinterpret_cast<unsigned short*>(a[block]); }
};

// Two E2M1 or E4M3 elements of a word as f16x2: its byte or half `i`.
template <bool k4>
__device__ __forceinline__ uint32_t decode2(uint32_t w, int i) {
    uint32_t r;
    if constexpr (k4) {
        // the byte is picked by unpacking the word: shifts and masks would cost as much as the conversion
        if (i == 0) asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\t}" : "=r"(r) : "r"(w));
        if (i == 1) asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b;\n\t}" : "=r"(r) : "r"(w));
        if (i == 2) asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, c;\n\t}" : "=r"(r) : "r"(w));
        if (i == 3) asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, d;\n\t}" : "=r"(r) : "r"(w));
    } else {
        if (i == 0) asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\t}" : "=r"(r) : "r"(w));
        if (i == 1) asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, b;\n\t}" : "=r"(r) : "r"(w));
    }
    return r;
}

// acc (two columns) += a * b, in fp32, both columns in one instruction
__device__ __forceinline__ void fma2(float2& acc, float a, float2 b) {
    unsigned long long d = *reinterpret_cast<unsigned long long*>(&acc);
    const float2 aa = make_float2(a, a);
    asm("fma.rn.f32x2 %0, %1, %2, %0;"
        : "+l"(d)
        : "l"(*reinterpret_cast<const unsigned long long*>(&aa)), "l"(*reinterpret_cast<const unsigned long long*>(&b)));
    acc = *reinterpret_cast<float2*>(&d);
}
// acc (two columns) += a * b with fp16 factors and fp32 sums: half `i` of the word a, both halves of b
__device__ __forceinline__ void fma2_f16(float2& acc, uint32_t a, int i, uint32_t b) {
    if (i == 0)
        asm("{\n\t.reg .b16 a0, a1, b0, b1;\n\tmov.b32 {a0, a1}, %2;\n\tmov.b32 {b0, b1}, %3;\n\t"
            "fma.rn.f32.f16 %0, a0, b0, %0;\n\tfma.rn.f32.f16 %1, a0, b1, %1;\n\t}" : "+f"(acc.x), "+f"(acc.y) : "r"(a), "r"(b));
    else
        asm("{\n\t.reg .b16 a0, a1, b0, b1;\n\tmov.b32 {a0, a1}, %2;\n\tmov.b32 {b0, b1}, %3;\n\t"
            "fma.rn.f32.f16 %0, a1, b0, %0;\n\tfma.rn.f32.f16 %1, a1, b1, %1;\n\t}" : "+f"(acc.x), "+f"(acc.y) : "r"(a), "r"(b));
}

// acc (two columns) *= f
__device__ __forceinline__ void mul2(float2& acc, float f) {
    unsigned long long d = *reinterpret_cast<unsigned long long*>(&acc);
    const float2 ff = make_float2(f, f);
    asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(d) : "l"(*reinterpret_cast<const unsigned long long*>(&ff)));
    acc = *reinterpret_cast<float2*>(&d);
}

// Element pair i of a lane's columns.
template <bool k4, int kW>
__device__ __forceinline__ uint32_t pair_of(const uint32_t (&r)[kW], int i) {
    return k4 ? decode2<k4>(r[k4 ? i >> 2 : 0], i & 3) : decode2<k4>(r[k4 ? 0 : i >> 1], i & 1);
}

// How a lane reads its elements. kWhole: its consecutive columns in one aligned load. kPadded: the same for rows
// that end inside a load but are far enough apart; the operand's last row is then read word by word, as what
// follows it may not be the operand's. Else word by word, the words of a row dealt out over the group's lanes in
// turn, so that a load of the group is one stretch of the row: kWords reads aligned words, kBytes two aligned ones
// that are shifted into place.
enum class Access { kWhole, kPadded, kWords, kBytes };

// The columns of a lane: kW words of kIn columns each.
template <bool k4, class L, Access kAccess>
struct Columns {
    static constexpr int kIn = k4 ? 8 : 4;
    static constexpr int kW = L::kCols / kIn;
    static constexpr bool kWhole = kAccess == Access::kWhole || kAccess == Access::kPadded;
    static constexpr int kScales = kWhole ? 1 : kW;  // scale blocks a lane may touch
    static constexpr int kRun = kWhole ? L::kCols : kIn;  // consecutive columns
    // first column of word i, from the slab's first
    __device__ static int of(int sl, int i) { return kWhole ? sl * L::kCols + i * kIn : (sl + i * L::kGroup) * kIn; }
};

// The lane's words of the row at `row`, word i from byte at[i], bytes[i] bytes of which are the row's (and
// may be read: every aligned word that is read holds one of them).
template <Access kAccess, int kW, int kAt>
__device__ __forceinline__ void load_raw(const uint8_t* row, const int (&at)[kAt], const int (&bytes)[kAt], bool last, uint32_t (&r)[kW]) {
    if constexpr (kAccess == Access::kWhole || kAccess == Access::kPadded) {
        const uint8_t* p = row + at[0];
        if (kAccess == Access::kPadded && last && bytes[0] < 4 * kW) {
#pragma unroll
            for (int i = 0; i < kW; ++i) r[i] = 4 * i < bytes[0] ? __ldg(reinterpret_cast<const uint32_t*>(p) + i) : 0u;
        } else if constexpr (kW == 1) {
            r[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
        } else if constexpr (kW == 2) {
            const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
            r[0] = v.x;
            r[1] = v.y;
        } else {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
            r[0] = v.x;
            r[1] = v.y;
            r[2] = v.z;
            r[3] = v.w;
        }
    } else if constexpr (kAccess == Access::kWords) {
#pragma unroll
        for (int i = 0; i < kW; ++i) r[i] = __ldg(reinterpret_cast<const uint32_t*>(row + at[i]));
    } else {
        const int m = int(reinterpret_cast<uintptr_t>(row + at[0]) & 3);  // of every word: they are whole words apart
#pragma unroll
        for (int i = 0; i < kW; ++i) {
            const uint32_t* q = reinterpret_cast<const uint32_t*>(row + at[i] - m);
            const uint32_t lo = __ldg(q), hi = m + bytes[i] > 4 ? __ldg(q + 1) : 0u;
            r[i] = __funnelshift_r(lo, hi, 8 * m);
        }
    }
}

// Writes a lane's columns of a row of C, or adds them: the row has this one writer, so either is one operation
// on every value. kVec: the row is 16-byte aligned and its columns are whole groups of four.
template <class M, bool kVec, int kPairs>
__device__ __forceinline__ void write_row(float* dst, const float2 (&acc)[kPairs], int sl, int exist, bool add) {
    if constexpr (kVec) {
#pragma unroll
        for (int f = 0; f < 2 * kPairs; f += 4) {
            const int c = M::of(sl, f / M::kIn) + f % M::kIn;
            const float4 v = make_float4(acc[f / 2].x, acc[f / 2].y, acc[f / 2 + 1].x, acc[f / 2 + 1].y);
            if (c < exist) {
                if (add) atomicAdd(reinterpret_cast<float4*>(dst + c), v);
                else __stcs(reinterpret_cast<float4*>(dst + c), v);
            }
        }
    } else if (add) {
#pragma unroll
        for (int f = 0; f < 2 * kPairs; ++f) {
            const int c = M::of(sl, f / M::kIn) + f % M::kIn;
            if (c < exist) atomicAdd(dst + c, f & 1 ? acc[f / 2].y : acc[f / 2].x);
        }
    } else {
#pragma unroll
        for (int f = 0; f < 2 * kPairs; ++f) {
            const int c = M::of(sl, f / M::kIn) + f % M::kIn;
            if (c < exist) dst[c] = f & 1 ? acc[f / 2].y : acc[f / 2].x;
        }
    }
}

struct Args {
    const int4* units;
    int64_t n_units;
    const int* rp;
    const int* cols;
    const void* vals;
    const int* hot_cols;
    MxView B;
    int N, O;
    float* C;
    int64_t ldc;
    float scale;
    float* partial;
    int direct;        // split rows up to this many entries are one group's after all
    bool scale_words;  // a slab's scales can be read at once
    bool acc16;        // the format's scale leaves room for the fp16 form
    bool add;          // C += A * B
    bool vec;          // C's rows take 16-byte stores
    int64_t pitch;     // floats from one partial row to the next, whole groups of four
};

// Two scales of a word's low (0) or high (1) half as fp32 (255 is NaN).
__device__ __forceinline__ float2 scale_pair(uint32_t w, int half) {
    uint32_t r;
    if (half == 0) asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.rn.bf16x2.ue8m0x2 %0, a;\n\t}" : "=r"(r) : "r"(w));
    else asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.rn.bf16x2.ue8m0x2 %0, b;\n\t}" : "=r"(r) : "r"(w));
    return make_float2(__uint_as_float(r << 16), __uint_as_float(r & 0xffff0000u));
}

// Product with fp32's subnormals as zero. Blocks of zeros have code 0, 2^-127: it would keep their entries
// from the fp16 form below for nothing.
__device__ __forceinline__ float mul_ftz(float a, float b) {
    float r;
    asm("mul.ftz.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// kAcc16 (the FP16 format): the products are formed as fp16 x fp16 with fp32 sums, which needs no conversion
// of the elements to fp32 (121 against 79 elements per clock and SM in a loop of nothing else). An A value
// times its block's scale has the A value's 11 bits; 2^-shift, fixed for a block by the unit's first batch,
// brings it into fp16's range, where it stays exact over 30 binades. A batch with a value that is not exact
// there (checked for each) brings the sums back to their own scale, and it and what follows in the unit that
// does not fit either is multiplied in fp32: the products are exact in both forms, so the form shows in no bit
// but those of sums that leave fp32's normal range.
template <bool k4, class L, Access kAccess, bool kVec, typename VT>
__global__ void __launch_bounds__(kWarps * 32) rows_mx_kernel(Args P) {
    constexpr bool kAcc16 = sizeof(VT) == 2;
    using M = Columns<k4, L, kAccess>;
    constexpr int kPairs = L::kCols / 2, kBlocks = L::kBlocks, kPer = L::kPer, kFlight = L::kFlight, kBatch = L::kBatch;
    constexpr int kW = M::kW, kScales = M::kScales;
    __shared__ Stage<kBlocks, kBatch> stage_all[2][kWarps * L::kGroups];
    __shared__ int ends_all[kWarps * L::kGroups][kUnitRows + 1];
    const VT* vals = static_cast<const VT*>(P.vals);
    const int lane = threadIdx.x & 31, sub = lane / L::kGroup, sl = lane % L::kGroup;
    const int group = (threadIdx.x >> 5) * L::kGroups + sub;
    const int64_t unit = int64_t(blockIdx.x) * (kWarps * L::kGroups) + group;
    const int4 u = unit < P.n_units ? P.units[unit] : make_int4(0, 0, 0, 0);
    const int slab = int(blockIdx.y) * L::kSlab;
    const int exist = P.O - slab;  // columns from the slab's first on
    // bytes of the lane's words in a row, and how many of them are the row's; a word past the last column is
    // read as the slab's first and not stored
    int at[kScales], bytes[kScales], block[kScales];
#pragma unroll
    for (int i = 0; i < kScales; ++i) {
        int c = M::of(sl, i);
        if (c >= exist) c = 0;
        const int n = min(M::kWhole ? L::kCols : M::kIn, exist - c);
        at[i] = k4 ? (slab + c) / 2 : slab + c;
        bytes[i] = k4 ? (n + 1) / 2 : n;
        block[i] = c / kMxBlock;
    }
    const uint8_t* s_base = P.B.s + slab / kMxBlock;
    const int blocks = min(kBlocks, (exist + kMxBlock - 1) / kMxBlock);
    // What stands behind a row's last scale is nobody's, and no part of the choice between the fp16 and the fp32 form
    // below. Cut at the scales' use and not at their load, which the warp would wait for (R-MAT 420 against 400 us), and
    // not in the form that reads elements byte by byte, whose registers it does not fit (O = 101: 203 against 181 us).
    constexpr bool kCut = kBlocks == 4 && kAccess != Access::kBytes;
    const uint32_t existing = 0xffffffffu >> (8 * (4 - blocks));
    const uint32_t ldq = uint32_t(P.B.ldq), lds = uint32_t(P.B.lds);

    // the unit's entries (positions below count from its first) and rows
    int64_t pb = u.z;
    int n = u.w - u.z;
    bool chunk = (u.y & 0x80000000) != 0;
    int rows = chunk ? 1 : u.y - u.x;
    if (chunk) {
        const int64_t first = P.rp[u.x];
        const int len = int(P.rp[u.x + 1] - first);
        if (len <= P.direct) {  // the row's first chunk takes all of it
            chunk = false;
            n = pb == first ? len : 0;
            rows = pb == first ? 1 : 0;
        }
    }
    // where each row ends
    int* ends = ends_all[group];
#pragma unroll
    for (int k = 0; k < (kUnitRows + L::kGroup - 1) / L::kGroup; ++k) {
        const int r = sl + k * L::kGroup;
        ends[r] = r >= rows ? kNever : rows == 1 ? n : int(P.rp[u.x + r + 1] - pb);
    }
    if (sl == 0) ends[kUnitRows] = kNever;
    __syncwarp();
    int end = ends[0];
    float* dst = chunk ? P.partial + unit * P.pitch + slab : P.C + int64_t(u.x) * P.ldc + slab;
    const bool add = P.add && !chunk;

    float2 acc[kPairs];
#pragma unroll
    for (int i = 0; i < kPairs; ++i) acc[i] = make_float2(0.f, 0.f);
    float unshift[kScales];  // 2^shift of the blocks of this lane's words
    float to_f16[kBlocks];   // 2^-shift of each block of the slab
#pragma unroll
    for (int i = 0; i < kScales; ++i) unshift[i] = 1.f;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) to_f16[b] = 1.f;
    constexpr int kPairsPer = kPairs / kScales;
    // stores the rows that end at position `at_entry`: the open one, and the empty ones behind it
    auto close = [&](int at_entry) {
        do {
#pragma unroll
            for (int i = 0; i < kPairs; ++i) mul2(acc[i], unshift[i / kPairsPer] * P.scale);
            write_row<M, kVec>(dst, acc, sl, exist, add);
#pragma unroll
            for (int i = 0; i < kPairs; ++i) acc[i] = make_float2(0.f, 0.f);
            dst += P.ldc;
            end = *++ends;
        } while (end == at_entry);
    };
    if (end == 0) close(0);

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
        const uint8_t* s = s_base + uint64_t(uint32_t(c)) * lds;
        if constexpr (kBlocks == 1) return __ldg(s);
        // In one word where it ends with the slab's blocks or before the operand does (`kCut`: the rest of it is cut off
        // when it is used), else byte by byte.
        if (P.scale_words && (blocks == kBlocks || (kCut && c != P.N - 1))) {
            if constexpr (kBlocks == 4) return __ldg(reinterpret_cast<const uint32_t*>(s));
            else return __ldg(reinterpret_cast<const unsigned short*>(s));
        }
        uint32_t w = 0;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
            if (b < blocks) w |= uint32_t(__ldg(s + b)) << (8 * b);
        return w;
    };
    int c_now[kPer], c_next[kPer];
    float v_now[kPer], v_next[kPer];
    uint32_t s_now[kPer];
#pragma unroll
    for (int k = 0; k < kPer; ++k) load_entry(sl + k * L::kGroup, c_now[k], v_now[k]);
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        load_entry(kBatch + sl + k * L::kGroup, c_next[k], v_next[k]);
        s_now[k] = load_scales(sl + k * L::kGroup, c_now[k]);
    }
    const int longest = __reduce_max_sync(kFull, n);
    for (int q = 0; q < longest; q += kBatch) {
        Stage<kBlocks, kBatch>& stage = stage_all[(q / kBatch) & 1][group];
        // A values times the scale of each block; 0 past the unit's end, where the A value and code are 0
        float a[kPer][kBlocks];
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            const uint32_t codes = kAcc16 && kCut ? s_now[k] & existing : s_now[k];
            const float2 s01 = scale_pair(codes, 0);
            a[k][0] = mul_ftz(v_now[k], s01.x);
            if constexpr (kBlocks > 1) a[k][1] = mul_ftz(v_now[k], s01.y);
            if constexpr (kBlocks > 2) {
                const float2 s23 = scale_pair(codes, 1);
                a[k][2] = mul_ftz(v_now[k], s23.x);
                a[k][3] = mul_ftz(v_now[k], s23.y);
            }
        }
        bool in_f32 = true;
        if constexpr (kAcc16) {
            if (q == 0 && P.acc16) {
                // the largest exponent of each block's products goes to 2^6: 9 binades above, 20 below stay exact
                uint32_t t = 0;
#pragma unroll
                for (int k = 0; k < kPer; ++k) {
                    uint32_t w = 0;
#pragma unroll
                    for (int b = 0; b < kBlocks; ++b) w |= ((__float_as_uint(a[k][b]) >> 23) & 0xffu) << (8 * b);
                    t = __vmaxu4(t, w);
                }
#pragma unroll
                for (int d = 1; d < L::kGroup; d *= 2) t = __vmaxu4(t, __shfl_xor_sync(kFull, t, d));
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) {
                    const int e = int((t >> (8 * b)) & 0xffu);
                    const int shift = e == 0 ? 0 : max(73, min(193, e)) - 133;
                    to_f16[b] = __uint_as_float(uint32_t(127 - shift) << 23);
#pragma unroll
                    for (int i = 0; i < kScales; ++i)
                        if (b == block[i]) unshift[i] = __uint_as_float(uint32_t(127 + shift) << 23);
                }
            }
            bool inexact = !P.acc16;
            uint32_t h[kPer][(kBlocks + 1) / 2];
#pragma unroll
            for (int k = 0; k < kPer; ++k) {
#pragma unroll
                for (int b = 0; b < kBlocks; b += 2) {
                    const float x = a[k][b] * to_f16[b], y = kBlocks > 1 ? a[k][b + (kBlocks > 1)] * to_f16[b + (kBlocks > 1)] : 0.f;
                    const __half2 xy = __floats2half2_rn(x, y);
                    const float2 back = __half22float2(xy);
                    inexact |= !(back.x == x && back.y == y);
                    h[k][b / 2] = *reinterpret_cast<const uint32_t*>(&xy);
                }
            }
            in_f32 = __any_sync(kFull, inexact);
            if (!in_f32) {
#pragma unroll
                for (int k = 0; k < kPer; ++k)
#pragma unroll
                    for (int b = 0; b < kBlocks; ++b) stage.half(b)[sl + k * L::kGroup] = (unsigned short)(h[k][b / 2] >> (16 * (b & 1)));
            }
        }
        if (in_f32) {
            if (kAcc16) {
#pragma unroll
                for (int i = 0; i < kPairs; ++i) mul2(acc[i], unshift[i / kPairsPer]);
#pragma unroll
                for (int i = 0; i < kScales; ++i) unshift[i] = 1.f;
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) to_f16[b] = 1.f;
            }
#pragma unroll
            for (int k = 0; k < kPer; ++k)
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) stage.a[b][sl + k * L::kGroup] = __float_as_uint(a[k][b]);
        }
#pragma unroll
        for (int k = 0; k < kPer; ++k) stage.col[sl + k * L::kGroup] = c_now[k];
        __syncwarp();  // the other buffer's reads ended before this batch's values were staged
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            c_now[k] = c_next[k];
            v_now[k] = v_next[k];
            s_now[k] = load_scales(q + kBatch + sl + k * L::kGroup, c_now[k]);
            load_entry(q + 2 * kBatch + sl + k * L::kGroup, c_next[k], v_next[k]);
        }
#pragma unroll
        for (int j0 = 0; j0 < kBatch; j0 += kFlight) {
            uint32_t raw[kFlight][kW];
#pragma unroll
            for (int j = 0; j < kFlight; j += 4) {
                const int4 c = *reinterpret_cast<const int4*>(stage.col + j0 + j);
                const int cj[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) load_raw<kAccess>(P.B.q + uint64_t(uint32_t(cj[k])) * ldq, at, bytes, cj[k] == P.N - 1, raw[j + k]);
            }
            // no group has a row's end among these entries: no test for one after each
            const bool straight = !__any_sync(kFull, end <= q + j0 + kFlight);
            if (!in_f32) {
                uint32_t w[kScales][kFlight / 2];
#pragma unroll
                for (int i = 0; i < kScales; ++i)
#pragma unroll
                    for (int j = 0; j < kFlight / 2; j += 2) {
                        const uint2 t = *reinterpret_cast<const uint2*>(stage.half(block[i]) + j0 + 2 * j);
                        w[i][j] = t.x;
                        w[i][j + 1] = t.y;
                    }
                auto entry = [&](int j) {
#pragma unroll
                    for (int i = 0; i < kPairs; ++i) fma2_f16(acc[i], w[i / kPairsPer][j >> 1], j & 1, pair_of<k4, kW>(raw[j], i));
                };
                if (straight) {
#pragma unroll
                    for (int j = 0; j < kFlight; ++j) entry(j);
                } else {
#pragma unroll
                    for (int j = 0; j < kFlight; ++j) {
                        entry(j);
                        if (end == q + j0 + j + 1) close(q + j0 + j + 1);
                    }
                }
            } else {
                float w[kScales][kFlight];
#pragma unroll
                for (int i = 0; i < kScales; ++i)
#pragma unroll
                    for (int j = 0; j < kFlight; j += 4) {
                        const float4 t = *reinterpret_cast<const float4*>(stage.a[block[i]] + j0 + j);
                        w[i][j] = t.x;
                        w[i][j + 1] = t.y;
                        w[i][j + 2] = t.z;
                        w[i][j + 3] = t.w;
                    }
                auto entry = [&](int j) {
#pragma unroll
                    for (int i = 0; i < kPairs; ++i) fma2(acc[i], w[i / kPairsPer][j], mx_f16x2_to_f32(pair_of<k4, kW>(raw[j], i)));
                };
                if (!kAcc16 && straight) {
#pragma unroll
                    for (int j = 0; j < kFlight; ++j) entry(j);
                } else {
#pragma unroll
                    for (int j = 0; j < kFlight; ++j) {
                        entry(j);
                        if (end == q + j0 + j + 1) close(q + j0 + j + 1);
                    }
                }
            }
        }
    }
}

template <bool k4, class L, Access kAccess, typename VT>
cudaError_t launch(Args a, cudaStream_t st) {
    const int64_t per_block = kWarps * L::kGroups;
    const int64_t blocks = (a.n_units + per_block - 1) / per_block;
    const int slabs = (a.O + L::kSlab - 1) / L::kSlab;
    if (blocks > 0x7fffffffLL || slabs > 65535) return cudaErrorInvalidValue;
    a.scale_words = reinterpret_cast<uintptr_t>(a.B.s) % L::kBlocks == 0 && a.B.lds % L::kBlocks == 0;
    const dim3 grid(unsigned(blocks), unsigned(slabs), 1);
    if (a.vec) rows_mx_kernel<k4, L, kAccess, true, VT><<<grid, kWarps * 32, 0, st>>>(a);
    else rows_mx_kernel<k4, L, kAccess, false, VT><<<grid, kWarps * 32, 0, st>>>(a);
    return cudaGetLastError();
}

// One load for a lane's columns, where every row is aligned to it; the row stride, a multiple of it, then pads a row that
// ends inside a load. True where that holds; the launch's result is in e.
template <bool k4, class L, typename VT>
bool launch_whole(const Args& a, cudaStream_t st, cudaError_t& e) {
    const int64_t full = k4 ? L::kCols / 2 : L::kCols;
    if (reinterpret_cast<uintptr_t>(a.B.q) % uintptr_t(full) || a.B.ldq % full) return false;
    e = a.O % L::kCols == 0 ? launch<k4, L, Access::kWhole, VT>(a, st) : launch<k4, L, Access::kPadded, VT>(a, st);
    return true;
}

// Words, Bytes: the forms for rows that are read word by word, aligned to words or not.
template <bool k4, class Words, class Bytes, typename VT>
cudaError_t launch_words(const Args& a, cudaStream_t st) {
    if (reinterpret_cast<uintptr_t>(a.B.q) % 4 == 0 && a.B.ldq % 4 == 0) return launch<k4, Words, Access::kWords, VT>(a, st);
    return launch<k4, Bytes, Access::kBytes, VT>(a, st);
}

template <bool k4, typename VT>
cudaError_t product_columns(const Args& a, cudaStream_t st) {
    // Columns per lane and entries in flight as measured on 262144 rows of 16 entries, O = 32: 4 lanes of 8 columns 60
    // (E2M1) and 60 us (E4M3, four in flight; eight: 71), 2 lanes of 16: 74 and 75; O = 64: 8 lanes of 8 columns 67,
    // 4 of 16 85 us; O = 128: 16 lanes of 8 columns 96, as 8 of 16, but 468 against 409 us on the stencil.
    cudaError_t e;
    if (a.O <= 32) {
        using L = Lanes<4, 8, k4 ? 8 : 4>;
        return launch_whole<k4, L, VT>(a, st, e) ? e : launch_words<k4, L, L, VT>(a, st);
    }
    if (a.O <= 64) {
        using L = Lanes<8, 8, 8>;
        return launch_whole<k4, L, VT>(a, st, e) ? e : launch_words<k4, L, L, VT>(a, st);
    }
    using Wide = Lanes<8, 16, 8>;
    using Narrow = Lanes<16, 8, 8>;
    if (launch_whole<k4, Wide, VT>(a, st, e)) return e;
    // E4M3 rows at multiples of 8 bytes: 8 columns in one load, O = 120, 104 against 138 us word by word (stencil 482
    // against 635, R-MAT 448 against 618; eight entries in flight: 109, 509, 457)
    if constexpr (!k4)
        if (launch_whole<k4, Lanes<16, 8, 4>, VT>(a, st, e)) return e;
    // Word by word, 8 columns against 16: O = 300 in 4 bits 381 against 438 us; O = 100 in 8 bits 121 against 134 us,
    // fp32 A 129 against 149 us; but O = 101 in 8 bits, fp16 A, 195 against 180 us.
    return launch_words<k4, Narrow, typename std::conditional<k4 || sizeof(VT) == 4, Narrow, Wide>::type, VT>(a, st);
}

// One pair of element and A value types; each pair is a translation unit. Up to 64 columns behind the last whole slab
// of 128 go to a launch of their own, whose lanes they fill, where that takes less than the launch.
template <bool k4, typename VT>
cudaError_t product(const Args& a, cudaStream_t st) {
    const int rest = a.O % 128;
    if (a.O < 128 || rest == 0 || rest > 64 || a.n_units < 8192) return product_columns<k4, VT>(a, st);
    Args b = a;
    const int c = a.O - rest;
    b.O = rest;
    b.B.q += k4 ? c / 2 : c;
    b.B.s += c / kMxBlock;
    b.C += c;
    b.partial += c;
    Args head = a;
    head.O = c;
    const cudaError_t e = product_columns<k4, VT>(head, st);
    return e != cudaSuccess ? e : product_columns<k4, VT>(b, st);
}

extern template cudaError_t product<true, __half>(const Args&, cudaStream_t);
extern template cudaError_t product<true, float>(const Args&, cudaStream_t);
extern template cudaError_t product<false, __half>(const Args&, cudaStream_t);
extern template cudaError_t product<false, float>(const Args&, cudaStream_t);

}  // namespace rows_mx
}  // namespace dev
}  // namespace vcsrmc
