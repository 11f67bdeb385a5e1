// tq_batch_attn_v2.hip -- the batch attention kernels for 2-bit values.
#include "tq_batch_attn_kernel.h"

namespace tq {
template void ba_launch<2>(const BaArgs&, int, bool, bool, int, int, unsigned, hipStream_t);
}  // namespace tq
