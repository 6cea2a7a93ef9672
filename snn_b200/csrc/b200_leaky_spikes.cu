// The leaky recurrence for x of type Spike.
#include "b200_leaky.cuh"

namespace b200 {
namespace leaky {

cudaError_t forward_spikes(cudaStream_t s, const Form &f, const Args &a) {
    return launch_wide<Spike>(s, f, a, false);
}
cudaError_t backward_spikes(cudaStream_t s, const Form &f, const Args &a) {
    return launch_wide<Spike>(s, f, a, true);
}
cudaError_t step_spikes(cudaStream_t s, const Form &f, const StepArgs &a, dim3 grid) {
    return step_wide<Spike>(s, f, a, grid);
}

}  // namespace leaky
}  // namespace b200
