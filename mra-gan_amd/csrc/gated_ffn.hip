// Gated feed-forward block: the choice of operand planes by element type and precision mode.
// The kernels are in gated_ffn.h, instantiated once per (plane type, tensor type).
#include "prec.h"
#include "token_ops.h"

namespace mragan {

#define MRAGAN_FFN_DECLARE(name)                                                                                            \
  size_t ffn_ws_##name(const FfnArgs&, int planes, int pack, int backward, int recompute);                                  \
  size_t ffn_bwd_bytes_##name(const FfnArgs&, int planes, int pack, const void* dy, const void* kept, const FfnGrads&);     \
  int ffn_fwd_##name(const FfnArgs&, int planes, int pack, void* y, void* kept, void* ws, hipStream_t);                     \
  int ffn_bwd_##name(const FfnArgs&, int planes, int pack, const void* dy, const void* kept, const FfnGrads&, void* ws, hipStream_t);
MRAGAN_FFN_DECLARE(bf16)
MRAGAN_FFN_DECLARE(f16)
MRAGAN_FFN_DECLARE(f32_bf16)
MRAGAN_FFN_DECLARE(f32_f16)

// 16-bit tensors are their own plane; fp32 ones become planes by the process's precision mode: three
// bf16 planes (f32), two (bf16x3), one bf16 or one fp16
#define MRAGAN_FFN_DISPATCH(f, pmode, call)                                                         \
  f.dtype == kBF16   ? call(bf16, 1, 0)                                                             \
  : f.dtype == kF16  ? call(f16, 1, 0)                                                              \
  : pmode == kPrecF16 ? call(f32_f16, 1, 1)                                                         \
                      : call(f32_bf16, (pmode == kPrecBf16 ? 1 : pmode == kPrecBf16x3 ? 2 : 3), 1)

size_t gated_ffn_ws_bytes(const FfnArgs& f, int pmode, int backward, int recompute) {
#define MRAGAN_FFN_WS(name, planes, pack) ffn_ws_##name(f, planes, pack, backward, recompute)
  return MRAGAN_FFN_DISPATCH(f, pmode, MRAGAN_FFN_WS);
}
size_t gated_ffn_bwd_bytes(const FfnArgs& f, int pmode, const void* dy, const void* kept, const FfnGrads& o) {
#define MRAGAN_FFN_BYTES(name, planes, pack) ffn_bwd_bytes_##name(f, planes, pack, dy, kept, o)
  return MRAGAN_FFN_DISPATCH(f, pmode, MRAGAN_FFN_BYTES);
}
int gated_ffn_fwd(const FfnArgs& f, int pmode, void* y, void* kept, void* ws, hipStream_t st) {
#define MRAGAN_FFN_FWD(name, planes, pack) ffn_fwd_##name(f, planes, pack, y, kept, ws, st)
  return MRAGAN_FFN_DISPATCH(f, pmode, MRAGAN_FFN_FWD);
}
int gated_ffn_bwd(const FfnArgs& f, int pmode, const void* dy, const void* kept, const FfnGrads& o, void* ws, hipStream_t st) {
#define MRAGAN_FFN_BWD(name, planes, pack) ffn_bwd_##name(f, planes, pack, dy, kept, o, ws, st)
  return MRAGAN_FFN_DISPATCH(f, pmode, MRAGAN_FFN_BWD);
}

}  // namespace mragan
