// The rows plan with a microscaled operand (plan_rows_mx.cuh): the choice of the types, and the split rows' last
// step.
#include <cuda_runtime.h>

#include <algorithm>

#include "plan_rows_mx.cuh"

namespace vcsrmc {
namespace dev {
namespace {

constexpr int kJoinWarps = 8;   // per block
constexpr int kJoinFlight = 8;  // chunks in flight per warp

// C's split rows: the sums of their chunks, in an order that their number alone decides. kPerRow warps add up every
// kPerRow-th chunk of a row each, 128 columns; rows of up to direct_chunks chunks were written by one group.
template <int kPerRow>
__global__ void __launch_bounds__(kJoinWarps * 32) join_chunks_kernel(const int* __restrict__ split_rows, int n_split,
                                                                      const int* __restrict__ chunk_start, const float* __restrict__ partial,
                                                                      int64_t pitch, int O, float* __restrict__ C, int64_t ldc,
                                                                      bool accumulate, int first_column, int direct_chunks) {
    __shared__ float4 part[kJoinWarps][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, of_row = warp % kPerRow;
    const int i = int(blockIdx.x) * (kJoinWarps / kPerRow) + warp / kPerRow;
    const int c = first_column + int(blockIdx.y) * 128 + 4 * lane;
    const int n = max(0, min(4, O - c));
    const int lo = i < n_split ? chunk_start[i] : 0, hi = i < n_split ? chunk_start[i + 1] : 0;
    const int row = i < n_split ? split_rows[i] : 0;
    const bool live = hi - lo > direct_chunks && n > 0;
    wait_for_launch_before();  // the chunks
    float4 v[kJoinFlight];
#pragma unroll
    for (int k = 0; k < kJoinFlight; ++k) v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (live) {
        for (int q = lo + of_row; q < hi; q += kJoinFlight * kPerRow) {
#pragma unroll
            for (int k = 0; k < kJoinFlight; ++k) {
                if (q + k * kPerRow < hi) {
                    const float4 t = *reinterpret_cast<const float4*>(partial + int64_t(q + k * kPerRow) * pitch + c);
                    v[k].x += t.x;
                    v[k].y += t.y;
                    v[k].z += t.z;
                    v[k].w += t.w;
                }
            }
        }
    }
#pragma unroll
    for (int d = 1; d < kJoinFlight; d *= 2)
#pragma unroll
        for (int k = 0; k < kJoinFlight; k += 2 * d)
            v[k] = make_float4(v[k].x + v[k + d].x, v[k].y + v[k + d].y, v[k].z + v[k + d].z, v[k].w + v[k + d].w);
    part[warp][lane] = v[0];
    __syncthreads();
    if (of_row == 0 && live) {
        float4 t = v[0];
#pragma unroll
        for (int k = 1; k < kPerRow; ++k) {
            const float4 u = part[warp + k][lane];
            t = make_float4(t.x + u.x, t.y + u.y, t.z + u.z, t.w + u.w);
        }
        float* dst = C + int64_t(row) * ldc + c;
        const float w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (k < n) dst[k] = accumulate ? dst[k] + w[k] : w[k];
    }
}

}  // namespace

// Split rows of up to this many entries are computed by one group after all: it takes them less time than the
// second launch (4096 rows of about 16 entries: 10.5 against 13.6 us). Longer rows would leave the other groups of
// their warp idle (rows of up to 1024 entries on the 2^20-row R-MAT: 481 against 403 us). A matrix whose rows are
// all within it needs no workspace.
constexpr int kDirect = 64;

int64_t rows_mx_chunks(const RowPlanView& P) { return P.most_chunks > kDirect / P.unit_nnz ? P.n_chunks : 0; }

int64_t rows_mx_pitch(int O) { return (int64_t(O) + 3) / 4 * 4; }

cudaError_t spmm_rows_mx(const RowPlanView& P, const MxView& B, int O, float* C, int64_t ldc, bool accumulate,
                         float* partial, cudaStream_t st) {
    if (P.n_units == 0) return cudaSuccess;  // no rows: every row, empty ones too, is a unit's
    rows_mx::Args a;
    a.units = P.units;
    a.n_units = P.n_units;
    a.rp = P.rp;
    a.cols = P.cols;
    a.vals = P.vals;
    a.hot_cols = P.hot.hot_cols;
    a.B = B;
    a.N = P.N;
    a.O = O;
    a.C = C;
    a.ldc = ldc;
    a.scale = P.scale;
    a.partial = partial;
    a.direct = kDirect / P.unit_nnz * P.unit_nnz;  // whole chunks, as the rows' chunk counts tell them
    a.scale_words = false;
    // the sums' scale and the format's are multiplied: both within 2^60
    a.acc16 = P.scale >= 0x1p-60f && P.scale <= 0x1p60f;
    a.add = accumulate;
    a.vec = O % 4 == 0 && reinterpret_cast<uintptr_t>(C) % 16 == 0 && ldc % 4 == 0;
    a.pitch = rows_mx_pitch(O);
    cudaError_t e;
    if (P.vals_f16) e = B.q4 ? rows_mx::product<true, __half>(a, st) : rows_mx::product<false, __half>(a, st);
    else e = B.q4 ? rows_mx::product<true, float>(a, st) : rows_mx::product<false, float>(a, st);
    if (e != cudaSuccess || rows_mx_chunks(P) == 0) return e;
    const int slabs = (O + 127) / 128;
    // Few rows may be long and get a block each (8 rows of 4000 entries: 14.5 against 24.2 us with two warps each); for
    // many it makes no difference (4465 rows of the power law: 129.3 and 128.6 us; the R-MAT's: 398 and 396) and two
    // warps each take fewer blocks.
    const bool few = P.n_split_rows <= 8192;
    const int per_block = few ? 1 : kJoinWarps / 2;
    const unsigned blocks = unsigned((P.n_split_rows + per_block - 1) / per_block);
    for (int t = 0; t < slabs && e == cudaSuccess; t += 65535) {  // a grid's y extent
        LaunchAfter L(dim3(blocks, unsigned(std::min(65535, slabs - t)), 1), dim3(kJoinWarps * 32, 1, 1), st);
        e = cudaLaunchKernelEx(&L.cfg, few ? join_chunks_kernel<kJoinWarps> : join_chunks_kernel<2>, P.split_rows, P.n_split_rows,
                               P.chunk_start, static_cast<const float*>(partial), a.pitch, O, C, ldc, accumulate, 128 * t, a.direct / P.unit_nnz);
    }
    return e;
}

}  // namespace dev
}  // namespace vcsrmc
