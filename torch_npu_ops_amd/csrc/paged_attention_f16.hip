// fp16 instances of the paged attention kernels (paged_attention.h).
#include "paged_attention.h"

namespace xk {
namespace paged {
int run_f16(Params& p, int tiles, hipStream_t s) { return run<f16, f16>(p, tiles, s); }
}  // namespace paged
}  // namespace xk
