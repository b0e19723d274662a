// Launchers of the microscaled (MX) operators: quantise, dequantise, residual addition with RMS norm
// and its backward pass, and the rows plan with an MX operand (see mx.cuh for the format).
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "plan_rows.hpp"

namespace vcsrmc {
namespace dev {

// Configuration of a launch whose blocks may start before the launch ahead of them in the stream has ended (they
// wait for it themselves, wait_for_launch_before in mx.cuh).
struct LaunchAfter {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[1];
    LaunchAfter(dim3 grid, dim3 block, cudaStream_t st) {
        cfg.gridDim = grid;
        cfg.blockDim = block;
        cfg.stream = st;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
    }
};

// A strided row-major matrix of fp32, fp16 or bf16 (VCSRMC_F32, _F16, _BF16); ld in elements.
struct DenseView {
    void* p = nullptr;
    int dtype = 0;
    int64_t ld = 0;
};

// An MX matrix: element rows ldq bytes apart, scale rows lds bytes apart.
struct MxView {
    uint8_t* q = nullptr;
    int64_t ldq = 0;
    uint8_t* s = nullptr;
    int64_t lds = 0;
    bool q4 = false;
};

cudaError_t mx_quantize(const DenseView& X, int64_t rows, int O, const MxView& Q, cudaStream_t st);
cudaError_t mx_dequantize(const MxView& Q, int64_t rows, int O, const DenseView& Y, cudaStream_t st);

// s = round(x + residual) to residual_out's type; Q = MX(s * inv_rms * weight). residual.p and
// residual_out.p and inv_rms may be null (no addition, nothing stored).
struct RmsNormArgs {
    DenseView x, residual, residual_out;
    const void* weight = nullptr;
    int w_dtype = 0;
    bool vec_w = false;  // the weight is 16-byte aligned (set by the launcher)
    float eps = 0.f;
    int64_t rows = 0;
    int O = 0;
    MxView out;
    bool vec_q = false;  // out's rows are aligned to the stores of eight elements (set by the launcher)
    float* inv_rms = nullptr;
};
cudaError_t add_rms_norm(const RmsNormArgs& a, cudaStream_t st);

struct RmsNormGradArgs {
    DenseView dy, d_residual, hidden, dx;
    const void* weight = nullptr;
    int w_dtype = 0;
    bool vec_w = false;  // the weight is 16-byte aligned (set by the launcher)
    const float* inv_rms = nullptr;
    int64_t rows = 0;
    int O = 0;
    float* dweight = nullptr;
    float* workspace = nullptr;  // rms_norm_grad_workspace(rows, O) bytes
};
int64_t rms_norm_grad_workspace(int64_t rows, int O, int sms);
cudaError_t add_rms_norm_backward(const RmsNormGradArgs& a, int sms, cudaStream_t st);

// C (+)= A * B with an MX operand B over the row view. `partial`: rows_mx_chunks(P) rows of rows_mx_pitch(O)
// floats, 16-byte aligned (null when there are none), one for every chunk of a split row; they are summed in
// chunk order.
int64_t rows_mx_chunks(const RowPlanView& P);
int64_t rows_mx_pitch(int O);
cudaError_t spmm_rows_mx(const RowPlanView& P, const MxView& B, int O, float* C, int64_t ldc, bool accumulate,
                         float* partial, cudaStream_t st);

}  // namespace dev
}  // namespace vcsrmc
