// The norm's kernels for fp32 X and residual (rms_norm.cuh).
#include "rms_norm.cuh"

namespace vcsrmc {
namespace dev {
namespace norm {

template cudaError_t forward<true, true>(const RmsNormArgs&, cudaStream_t);
template cudaError_t backward<true, true>(const RmsNormGradArgs&, int64_t, cudaStream_t);

}  // namespace norm
}  // namespace dev
}  // namespace vcsrmc
