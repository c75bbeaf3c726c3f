// Policy losses over rows of f16 logits (the kernels are in policy_loss_rows.cuh).
#include "policy_loss_rows.cuh"

namespace ob200 {
int launch_policy_rows_f16(int kind, const PolicyRows& r, cudaStream_t st) { return launch_policy_rows<__half>(kind, r, st); }
}  // namespace ob200
