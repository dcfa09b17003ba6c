// fp16 queries, e4m3 cache: instances of the paged attention kernels (paged_attention.h).
#include "paged_attention.h"

namespace xk {
namespace paged {
int run_f16_f8(Params& p, int tiles, hipStream_t s) { return run<f16, f8>(p, tiles, s); }
}  // namespace paged
}  // namespace xk
