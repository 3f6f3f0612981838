// Masked attention's kernels for bf16.
#include "attention_masked.hpp"

namespace dlm {

int am_run_bf16(const AmParams& p, const AmPlan& pl, bool cap, hipStream_t s) { return am_run<__bf16>(p, pl, cap, s); }

}  // namespace dlm
