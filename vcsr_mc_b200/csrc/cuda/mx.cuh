// Microscaled (MX) elements: 32 consecutive columns of a row share one power-of-two scale.
//   element  E4M3 (8 bits, largest 448 = 1.75 * 2^8) or E2M1 (4 bits, largest 6 = 1.5 * 2^2)
//   scale    E8M0, one byte: 2^(code - 127), 255 = NaN
// The scale is the smallest power of two (from 2^-127) under which the block's largest magnitude
// fits the element type, so no element is clipped; x * 2^-e is exact (a power of two) but for results
// below fp32's normal range, which round to zero anyway, and the one rounding is the element's, to
// nearest with ties to even. A block that holds an infinity or a NaN gets scale 255 and zero elements.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace vcsrmc {
namespace dev {

constexpr int kMxBlock = 32;       // columns per scale
constexpr uint32_t kMxNan = 255u;  // scale code of a block with an infinity or a NaN

// Scale code of a block from the bits of its largest |x| (a NaN's bits are above infinity's): the exponent, one
// more where the mantissa is above the element type's largest (the sum carries into the exponent), less the
// exponent of that largest. A subnormal clamps to code 0.
__device__ __forceinline__ uint32_t mx_scale_code(uint32_t amax_bits, bool q4) {
    const int code = int((amax_bits + (q4 ? 0x3fffffu : 0x1fffffu)) >> 23) - (q4 ? 2 : 8);
    return amax_bits >= 0x7f800000u ? kMxNan : uint32_t(max(code, 0));
}
// 2^-e of a finite block's code (codes reach 253 at most, so this is a normal number).
__device__ __forceinline__ float mx_inverse_scale(uint32_t code) { return __uint_as_float((254u - code) << 23); }
// 2^(code - 127); code 0 is subnormal, code 255 NaN.
__device__ __forceinline__ float mx_scale_value(uint32_t code) {
    const uint32_t bits = code == 0 ? 0x00400000u : code << 23;
    return __uint_as_float(code == kMxNan ? 0x7fffffffu : bits);
}

// Two elements as f16x2 (exact), the low half of the input first.
__device__ __forceinline__ uint32_t mx_decode2_e2m1(uint32_t byte) {
    uint32_t r;
    asm("{\n\t.reg .b8 t;\n\tcvt.u8.u32 t, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, t;\n\t}" : "=r"(r) : "r"(byte));
    return r;
}
__device__ __forceinline__ uint32_t mx_decode2_e4m3(uint32_t half) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((unsigned short)half));
    return r;
}
__device__ __forceinline__ float2 mx_f16x2_to_f32(uint32_t h) {
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// ---- a launch that starts while the one before it in the stream ends ----------------------------
// The host side's attribute lets it start, and its blocks wait here for the other's results.
__device__ __forceinline__ void wait_for_launch_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ---- dense elements (fp32, fp16, bf16) ---------------------------------------------------------
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Eight consecutive elements; `vec`: p is 16-byte aligned and all eight exist, else the first nv are
// read one by one and the others are 0.
template <typename T>
__device__ __forceinline__ void load8(const T* p, int nv, bool vec, float (&v)[8]) {
    if (vec && nv == 8) {
        if constexpr (sizeof(T) == 4) {
            const float4 a = __ldcs(reinterpret_cast<const float4*>(p)), b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
            v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
            const uint4 a = __ldcs(reinterpret_cast<const uint4*>(p));
            const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const T* h = reinterpret_cast<const T*>(&w[i]);
                v[2 * i] = to_f32(h[0]);
                v[2 * i + 1] = to_f32(h[1]);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < nv ? to_f32(p[i]) : 0.f;
    }
}
// Stores eight consecutive elements; p is 16-byte aligned.
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        __stcs(reinterpret_cast<float4*>(p), make_float4(v[0], v[1], v[2], v[3]));
        __stcs(reinterpret_cast<float4*>(p) + 1, make_float4(v[4], v[5], v[6], v[7]));
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            T* h = reinterpret_cast<T*>(&w[i]);
            h[0] = from_f32<T>(v[2 * i]);
            h[1] = from_f32<T>(v[2 * i + 1]);
        }
        __stcs(reinterpret_cast<uint4*>(p), make_uint4(w[0], w[1], w[2], w[3]));
    }
}

// Two elements, `lo` in the low half of the result (8 bits of it for E2M1, 16 for E4M3).
__device__ __forceinline__ uint32_t mx_encode2_e2m1(float lo, float hi) {
    uint32_t r;
    asm("{\n\t.reg .b8 t;\n\tcvt.rn.satfinite.e2m1x2.f32 t, %2, %1;\n\tcvt.u32.u8 %0, t;\n\t}" : "=r"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ uint32_t mx_encode2_e4m3(float lo, float hi) {
    unsigned short r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(r) : "f"(lo), "f"(hi));
    return r;
}

// Largest |x| of the two and `m`; a NaN wins.
__device__ __forceinline__ float max3_abs(float m, float x, float y) {
    asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(x), "f"(y));
    return m;
}

// Quantises and stores eight columns of a block held by four neighbouring lanes (8 columns each; all
// 32 lanes of the warp take part). `q` is the eight columns' place in the row (byte c for E4M3, c / 2 for
// E2M1), `s` the block's scale; nv of the eight columns exist (0: nothing is stored), the others are zeros.
// `vec`: q is aligned to its full store (8 bytes for E4M3, 4 for E2M1). True where the block's largest magnitude
// is within four units of the last place of a border between two scales: a y that was rounded on its way may then
// stand on the wrong side of it (one block in a million).
__device__ __forceinline__ bool mx_store_block(const float (&y)[8], int nv, bool q4, uint8_t* q, uint8_t* s, bool vec) {
    uint32_t amax = __float_as_uint(max3_abs(max3_abs(max3_abs(max3_abs(0.f, y[0], y[1]), y[2], y[3]), y[4], y[5]), y[6], y[7]));
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const bool near = (amax & 0x7fffffu) - ((q4 ? 0x400000u : 0x600000u) - 4u) <= 8u;
    if (nv <= 0) return false;
    const uint32_t code = mx_scale_code(amax, q4);
    if ((threadIdx.x & 3) == 0) *s = uint8_t(code);
    const float inv = mx_inverse_scale(code);  // of no use in a block with the NaN scale
    if (q4) {
        uint32_t w = 0;
        if (code != kMxNan)
            asm("{\n\t.reg .b8 a, b, c, d;\n\t"
                "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
                "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
                "mov.b32 %0, {a, b, c, d};\n\t}"
                : "=r"(w)
                : "f"(y[0] * inv), "f"(y[1] * inv), "f"(y[2] * inv), "f"(y[3] * inv), "f"(y[4] * inv), "f"(y[5] * inv), "f"(y[6] * inv),
                  "f"(y[7] * inv));
        if (vec && nv == 8) {
            *reinterpret_cast<uint32_t*>(q) = w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (2 * i < nv) q[i] = uint8_t(w >> (8 * i));
        }
    } else {
        uint32_t w[2] = {0u, 0u};
        if (code != kMxNan) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
                asm("{\n\t.reg .b16 a, b;\n\tcvt.rn.satfinite.e4m3x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 b, %4, %3;\n\t"
                    "mov.b32 %0, {a, b};\n\t}"
                    : "=r"(w[i])
                    : "f"(y[4 * i] * inv), "f"(y[4 * i + 1] * inv), "f"(y[4 * i + 2] * inv), "f"(y[4 * i + 3] * inv));
        }
        if (vec && nv == 8) {
            *reinterpret_cast<uint2*>(q) = make_uint2(w[0], w[1]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < nv) q[i] = uint8_t(w[i >> 2] >> (8 * (i & 3)));
        }
    }
    return near;
}

// From columns dealt out over kL neighbouring lanes (t[j] is column j * kL + lane of a span of 8 * kL, as coalesced
// single loads give them) to eight consecutive columns per lane, or back. `span`: 8 * kL floats of shared memory
// that are the lanes' own, 16-byte aligned. All lanes of the warp take part.
template <int kL>
__device__ __forceinline__ void turn_to_groups(const float (&t)[8], float (&v)[8], float* span, int sl) {
    __syncwarp();  // the span may still be read
#pragma unroll
    for (int j = 0; j < 8; ++j) span[j * kL + sl] = t[j];
    __syncwarp();
    const float4 a = *reinterpret_cast<const float4*>(span + 8 * sl), b = *reinterpret_cast<const float4*>(span + 8 * sl + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <int kL>
__device__ __forceinline__ void turn_to_columns(const float (&v)[8], float (&t)[8], float* span, int sl) {
    __syncwarp();
    *reinterpret_cast<float4*>(span + 8 * sl) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(span + 8 * sl + 4) = make_float4(v[4], v[5], v[6], v[7]);
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = span[j * kL + sl];
}

}  // namespace dev
}  // namespace vcsrmc
