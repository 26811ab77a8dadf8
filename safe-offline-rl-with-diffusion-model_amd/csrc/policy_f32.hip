// The policy loss on float32 log-probabilities.
#include "policy.inl"

namespace trebi {
hipError_t launch_policy_f32(const PolicyP& p, int blocks, hipStream_t st) { return launch_policy_t<float>(p, blocks, st); }
}  // namespace trebi
