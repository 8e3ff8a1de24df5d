// Internal interface between the token-block entry points (token_capi.hip) and their kernel files.
#pragma once
#include "token.h"

namespace mragan {

size_t layer_norm_bwd_ws_bytes(int64_t rows, int C, int dtype);
int layer_norm_fwd(const void* x, int64_t rows, int C, int dtype, const void* w, const void* b, int wdtype, float eps, void* y,
                   float* mean, float* rstd, hipStream_t st);
int layer_norm_bwd(const void* x, const float* mean, const float* rstd, const void* dy, int64_t rows, int C, int dtype,
                   const void* w, int wdtype, void* dx, void* dw, void* db, float* part, hipStream_t st);

struct RecurArgs {
  const void* x; int64_t x_sb, x_st;
  const void* decay; int64_t d_sb, d_st;
  const void* gate; int64_t g_sb, g_st;     // null: y = h
  int64_t B, T;
  int C, dtype, reverse;
};
int64_t recurrence_carries(int64_t T);
int64_t recurrence_threads(int64_t B, int64_t T, int C);   // of the largest launch
size_t recurrence_ws_bytes(int64_t B, int64_t T, int C);
int recurrence_fwd(const RecurArgs& r, const float* h0, void* y, float* last, float* carry, float* ws, hipStream_t st);
int recurrence_bwd(const RecurArgs& r, const float* carry, const void* dy, int64_t dy_sb, int64_t dy_st, const float* dlast,
                   void* dx, void* dd, void* dz, float* dh0, float* ws, hipStream_t st);

struct FfnArgs {
  const void* x; int64_t M; int C, F, O, dtype;
  const void *wg, *wu, *wd, *bg, *bu, *bd;   // biases may be null
  int act;
};
struct FfnGrads {                            // each may be null
  void *dx, *dwg, *dwu, *dwd, *dbg, *dbu, *dbd;
};
size_t gated_ffn_ws_bytes(const FfnArgs& f, int pmode, int backward, int recompute);
// what gated_ffn_bwd takes of its workspace for these gradients
size_t gated_ffn_bwd_bytes(const FfnArgs& f, int pmode, const void* dy, const void* kept, const FfnGrads& o);
int gated_ffn_fwd(const FfnArgs& f, int pmode, void* y, void* kept, void* ws, hipStream_t st);
int gated_ffn_bwd(const FfnArgs& f, int pmode, const void* dy, const void* kept, const FfnGrads& o, void* ws, hipStream_t st);

}  // namespace mragan
