// tq_batch_attn_3s.hip -- the batch attention kernels for 3-bit values in 16-token sub-blocks.
#include "tq_batch_attn_kernel.h"

namespace tq {
BA_LAUNCH(3, true)
}  // namespace tq
