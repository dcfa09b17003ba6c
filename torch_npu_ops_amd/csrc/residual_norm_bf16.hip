// bf16 instances of the block-to-block norm kernels (residual_norm.h).
#include "residual_norm.h"

namespace xk {
namespace resnorm {
int run_fwd_bf16(const FwdParams& p, hipStream_t s) { return run_fwd<bf16>(p, s); }
int run_bwd_bf16(const BwdParams& p, hipStream_t s) { return run_bwd<bf16>(p, s); }
}  // namespace resnorm
}  // namespace xk
