// tq_batch_attn_4t.hip -- the batch attention kernels for 4-bit values in 64-token tiles.
#include "tq_batch_attn_kernel.h"

namespace tq {
BA_LAUNCH(4, false)
}  // namespace tq
