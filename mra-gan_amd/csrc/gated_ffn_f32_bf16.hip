// Gated feed-forward block on fp32 tensors as bf16 planes.
#include "gated_ffn.h"

namespace mragan {
MRAGAN_FFN_ENTRIES(f32_bf16, __bf16, float)
}
