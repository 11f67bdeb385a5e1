// tq_batch_attn_v4.hip -- the batch attention kernels for 4-bit values.
#include "tq_batch_attn_kernel.h"

namespace tq {
template void ba_launch<4>(const BaArgs&, int, bool, bool, int, int, unsigned, hipStream_t);
}  // namespace tq
