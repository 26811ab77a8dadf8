// The policy loss on float16 log-probabilities.
#include "policy.inl"

namespace trebi {
hipError_t launch_policy_f16(const PolicyP& p, int blocks, hipStream_t st) { return launch_policy_t<f16_t>(p, blocks, st); }
}  // namespace trebi
