// tq_batch_attn_3t.hip -- the batch attention kernels for 3-bit values in 64-token tiles.
#include "tq_batch_attn_kernel.h"

namespace tq {
BA_LAUNCH(3, false)
}  // namespace tq
