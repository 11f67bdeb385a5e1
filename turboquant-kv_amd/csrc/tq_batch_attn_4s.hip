// tq_batch_attn_4s.hip -- the batch attention kernels for 4-bit values in 16-token sub-blocks.
#include "tq_batch_attn_kernel.h"

namespace tq {
BA_LAUNCH(4, true)
}  // namespace tq
