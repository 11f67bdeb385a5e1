// tq_batch_attn_2t.hip -- the batch attention kernels for 2-bit values in 64-token tiles.
#include "tq_batch_attn_kernel.h"

namespace tq {
BA_LAUNCH(2, false)
}  // namespace tq
