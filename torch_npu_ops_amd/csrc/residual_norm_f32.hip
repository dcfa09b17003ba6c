// f32 instances of the block-to-block norm kernels (residual_norm.h).
#include "residual_norm.h"

namespace xk {
namespace resnorm {
int run_fwd_f32(const FwdParams& p, hipStream_t s) { return run_fwd<float>(p, s); }
int run_bwd_f32(const BwdParams& p, hipStream_t s) { return run_bwd<float>(p, s); }
}  // namespace resnorm
}  // namespace xk
