// The policy loss on bfloat16 log-probabilities.
#include "policy.inl"

namespace trebi {
hipError_t launch_policy_bf16(const PolicyP& p, int blocks, hipStream_t st) { return launch_policy_t<bf16_t>(p, blocks, st); }
}  // namespace trebi
