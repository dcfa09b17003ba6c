// bf16 instances of the paged attention kernels (paged_attention.h).
#include "paged_attention.h"

namespace xk {
namespace paged {
int run_bf16(Params& p, int tiles, hipStream_t s) { return run<bf16, bf16>(p, tiles, s); }
}  // namespace paged
}  // namespace xk
