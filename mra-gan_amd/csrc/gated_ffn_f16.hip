// Gated feed-forward block on fp16 tensors.
#include "gated_ffn.h"

namespace mragan {
MRAGAN_FFN_ENTRIES(f16, _Float16, _Float16)
}
