// The leaky recurrence for x of type __half.
#include "b200_leaky.cuh"

namespace b200 {
namespace leaky {

cudaError_t forward_f16(cudaStream_t s, const Form &f, const Args &a) {
    return launch_narrow<__half>(s, f, a, false);
}
cudaError_t backward_f16(cudaStream_t s, const Form &f, const Args &a) {
    return launch_narrow<__half>(s, f, a, true);
}
cudaError_t step_f16(cudaStream_t s, const Form &f, const StepArgs &a, dim3 grid) {
    return step_narrow<__half>(s, f, a, grid);
}

}  // namespace leaky
}  // namespace b200
