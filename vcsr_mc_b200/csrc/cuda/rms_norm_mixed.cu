// The norm's kernels for fp32 X, 16-bit residual (rms_norm.cuh).
#include "rms_norm.cuh"

namespace vcsrmc {
namespace dev {
namespace norm {

template cudaError_t forward<true, false>(const RmsNormArgs&, cudaStream_t);
template cudaError_t backward<true, false>(const RmsNormGradArgs&, int64_t, cudaStream_t);

}  // namespace norm
}  // namespace dev
}  // namespace vcsrmc
