// The leaky recurrence for x of type float.
#include "b200_leaky.cuh"

namespace b200 {
namespace leaky {

cudaError_t forward_f32(cudaStream_t s, const Form &f, const Args &a) {
    return launch_wide<float>(s, f, a, false);
}
cudaError_t backward_f32(cudaStream_t s, const Form &f, const Args &a) {
    return launch_wide<float>(s, f, a, true);
}
cudaError_t step_f32(cudaStream_t s, const Form &f, const StepArgs &a, dim3 grid) {
    return step_wide<float>(s, f, a, grid);
}

}  // namespace leaky
}  // namespace b200
