// tq_batch_attn_2s.hip -- the batch attention kernels for 2-bit values in 16-token sub-blocks.
#include "tq_batch_attn_kernel.h"

namespace tq {
BA_LAUNCH(2, true)
}  // namespace tq
