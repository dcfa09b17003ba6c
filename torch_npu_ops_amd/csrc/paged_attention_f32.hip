// fp32 instances of the paged attention kernels (paged_attention.h).
#include "paged_attention.h"

namespace xk {
namespace paged {
int run_f32(Params& p, int tiles, hipStream_t s) { return run<float, float>(p, tiles, s); }
}  // namespace paged
}  // namespace xk
