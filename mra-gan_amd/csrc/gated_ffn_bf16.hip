// Gated feed-forward block on bf16 tensors.
#include "gated_ffn.h"

namespace mragan {
MRAGAN_FFN_ENTRIES(bf16, __bf16, __bf16)
}
