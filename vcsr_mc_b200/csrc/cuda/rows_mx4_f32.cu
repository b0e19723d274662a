// The rows plan's kernels for E2M1 elements, fp32 A values (plan_rows_mx.cuh).
#include "plan_rows_mx.cuh"

namespace vcsrmc {
namespace dev {
namespace rows_mx {

template cudaError_t product<true, float>(const Args&, cudaStream_t);

}  // namespace rows_mx
}  // namespace dev
}  // namespace vcsrmc
