// The leaky recurrence for x of type __nv_bfloat16.
#include "b200_leaky.cuh"

namespace b200 {
namespace leaky {

cudaError_t forward_bf16(cudaStream_t s, const Form &f, const Args &a) {
    return launch_narrow<__nv_bfloat16>(s, f, a, false);
}
cudaError_t backward_bf16(cudaStream_t s, const Form &f, const Args &a) {
    return launch_narrow<__nv_bfloat16>(s, f, a, true);
}
cudaError_t step_bf16(cudaStream_t s, const Form &f, const StepArgs &a, dim3 grid) {
    return step_narrow<__nv_bfloat16>(s, f, a, grid);
}

}  // namespace leaky
}  // namespace b200
