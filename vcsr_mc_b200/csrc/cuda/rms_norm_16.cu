// The norm's kernels for 16-bit X and residual (rms_norm.cuh).
#include "rms_norm.cuh"

namespace vcsrmc {
namespace dev {
namespace norm {

template cudaError_t forward<false, false>(const RmsNormArgs&, cudaStream_t);
template cudaError_t backward<false, false>(const RmsNormGradArgs&, int64_t, cudaStream_t);

}  // namespace norm
}  // namespace dev
}  // namespace vcsrmc
