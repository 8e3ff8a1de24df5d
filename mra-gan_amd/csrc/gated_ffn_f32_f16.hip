// Gated feed-forward block on fp32 tensors as one fp16 plane.
#include "gated_ffn.h"

namespace mragan {
MRAGAN_FFN_ENTRIES(f32_f16, _Float16, float)
}
