// extern "C" entry points of the token-block operators: argument checks, then the launches of
// layernorm.hip, gated_ffn.hip and recurrence.hip.  Nothing here throws or allocates.
#include "../../include/mragan_hip.h"
#include <initializer_list>

#include "token_ops.h"

using namespace mragan;

namespace {
constexpr int64_t kMaxThreads = (int64_t)1 << 32;         // of a launch, exclusive
constexpr int64_t kMaxChannels = (int64_t)1 << 30;        // of a normalized row: strided walks stay in an int
constexpr int64_t kMaxSide = ((int64_t)1 << 22) - 64;     // row length of an FFN operand: 256 rows below 2^31 bytes
constexpr int64_t kMaxRows = (int64_t)1 << 30;

bool all_aligned(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if (!aligned_to(p, 16)) return false;
  return true;
}
}  // namespace

extern "C" {

int mragan_layer_norm_fwd(const void* x, int64_t rows, int C, int dtype, const void* weight, const void* bias, int wdtype,
                          float eps, void* y, float* mean, float* rstd, void* stream) {
  MRAGAN_CHECK_ARG(rows >= 0 && C > 0, "layer_norm: bad shape [%lld][%d]", (long long)rows, C);
  MRAGAN_CHECK_ARG(rows == 0 || (x && y && mean && rstd), "layer_norm: null pointer");
  MRAGAN_CHECK_ARG(dtype_ok(dtype) && (wdtype == dtype || wdtype == kF32), "layer_norm: bad types %d / %d", dtype, wdtype);
  MRAGAN_CHECK_ARG(eps >= 0.f, "layer_norm: eps must not be negative");
  MRAGAN_CHECK_ARG(rows < kMaxRows * 2 && C <= kMaxChannels, "layer_norm: too many rows or channels (rows from 2^31 on, C above 2^30)");
  return layer_norm_fwd(x, rows, C, dtype, weight, bias, wdtype, eps, y, mean, rstd, static_cast<hipStream_t>(stream));
}

size_t mragan_layer_norm_bwd_workspace(int64_t rows, int C, int dtype) {
  return rows > 0 && C > 0 && dtype_ok(dtype) ? layer_norm_bwd_ws_bytes(rows, C, dtype) : 0;
}

int mragan_layer_norm_bwd(const void* x, const float* mean, const float* rstd, const void* dy, int64_t rows, int C,
                          int dtype, const void* weight, int wdtype, void* dx, void* dweight, void* dbias, void* ws,
                          size_t ws_bytes, void* stream) {
  MRAGAN_CHECK_ARG(rows >= 0 && C > 0, "layer_norm_bwd: bad shape [%lld][%d]", (long long)rows, C);
  MRAGAN_CHECK_ARG(rows == 0 || (x && mean && rstd && dy), "layer_norm_bwd: null pointer");
  MRAGAN_CHECK_ARG(dtype_ok(dtype) && (wdtype == dtype || wdtype == kF32), "layer_norm_bwd: bad types %d / %d", dtype, wdtype);
  MRAGAN_CHECK_ARG(rows < kMaxRows * 2 && C <= kMaxChannels, "layer_norm_bwd: too many rows or channels (rows from 2^31 on, C above 2^30)");
  if (!dx && !dweight && !dbias) return kOk;
  if (dweight || dbias) {
    const size_t need = rows ? layer_norm_bwd_ws_bytes(rows, C, dtype) : 0;
    if (need && (!ws || ws_bytes < need)) {
      set_error("layer_norm_bwd: workspace %zu < %zu bytes (query mragan_layer_norm_bwd_workspace)", ws_bytes, need);
      return kWorkspace;
    }
  }
  return layer_norm_bwd(x, mean, rstd, dy, rows, C, dtype, weight, wdtype, dx, dweight, dbias, static_cast<float*>(ws),
                        static_cast<hipStream_t>(stream));
}

static int ffn_shape(int64_t M, int C, int F, int O, int dtype, int act) {
  MRAGAN_CHECK_ARG(M >= 0 && C > 0 && F > 0 && O > 0, "gated_ffn: bad shape M %lld, C %d, F %d, O %d", (long long)M, C, F, O);
  MRAGAN_CHECK_ARG(M <= kMaxRows && C <= kMaxSide && F <= kMaxSide && O <= kMaxSide,
                   "gated_ffn: more than 2^30 rows, or C, F, O: a side above 2^22 - 64");
  MRAGAN_CHECK_ARG(dtype_ok(dtype), "gated_ffn: unknown dtype %d", dtype);
  MRAGAN_CHECK_ARG(act >= MRAGAN_ACT_NONE && act <= MRAGAN_ACT_GELU, "gated_ffn: unknown activation %d", act);
  return kOk;
}

size_t mragan_gated_ffn_workspace(int64_t M, int C, int F, int O, int dtype, int backward, int recompute) {
  if (M <= 0 || C <= 0 || F <= 0 || O <= 0 || !dtype_ok(dtype)) return 0;
  const FfnArgs f{nullptr, M, C, F, O, dtype, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, 0};
  return gated_ffn_ws_bytes(f, mragan_get_conv_precision(), backward, recompute);
}

int mragan_gated_ffn_fwd(const void* x, int64_t M, int C, int F, int O, int dtype, const void* w_gate, const void* w_up,
                         const void* w_down, const void* b_gate, const void* b_up, const void* b_down, int act, void* y,
                         void* kept, void* ws, size_t ws_bytes, void* stream) {
  if (int rc = ffn_shape(M, C, F, O, dtype, act)) return rc;
  if (M == 0) return kOk;
  MRAGAN_CHECK_ARG(x && w_gate && w_up && w_down && y, "gated_ffn: null pointer");
  MRAGAN_CHECK_ARG(all_aligned({x, w_gate, w_up, w_down, b_gate, b_up, b_down, y, kept, ws}),
                   "gated_ffn: tensors must be 16-byte aligned");
  const FfnArgs f{x, M, C, F, O, dtype, w_gate, w_up, w_down, b_gate, b_up, b_down, act};
  const int mode = mragan_get_conv_precision();
  const size_t need = gated_ffn_ws_bytes(f, mode, 0, 0);
  if (!ws || ws_bytes < need) {
    set_error("gated_ffn: workspace %zu < %zu bytes (query mragan_gated_ffn_workspace)", ws_bytes, need);
    return kWorkspace;
  }
  return gated_ffn_fwd(f, mode, y, kept, ws, static_cast<hipStream_t>(stream));
}

int mragan_gated_ffn_bwd(const void* x, int64_t M, int C, int F, int O, int dtype, const void* w_gate, const void* w_up,
                         const void* w_down, const void* b_gate, const void* b_up, int act, const void* dy,
                         const void* kept, void* dx, void* dw_gate, void* dw_up, void* dw_down, void* db_gate, void* db_up,
                         void* db_down, void* ws, size_t ws_bytes, void* stream) {
  if (int rc = ffn_shape(M, C, F, O, dtype, act)) return rc;
  MRAGAN_CHECK_ARG(M > 0, "gated_ffn_bwd: no rows (the gradients are zeros)");
  MRAGAN_CHECK_ARG(x && w_gate && w_up && w_down && dy, "gated_ffn_bwd: null pointer");
  MRAGAN_CHECK_ARG(all_aligned({x, w_gate, w_up, w_down, b_gate, b_up, dy, kept, dx, dw_gate, dw_up, dw_down, db_gate, db_up,
                                db_down, ws}),
                   "gated_ffn_bwd: tensors must be 16-byte aligned");
  const FfnGrads o{dx, dw_gate, dw_up, dw_down, db_gate, db_up, db_down};
  if (!dx && !dw_gate && !dw_up && !dw_down && !db_gate && !db_up && !db_down) return kOk;
  const FfnArgs f{x, M, C, F, O, dtype, w_gate, w_up, w_down, b_gate, b_up, nullptr, act};
  const int mode = mragan_get_conv_precision();
  const size_t need = gated_ffn_bwd_bytes(f, mode, dy, kept, o);
  if (!ws || ws_bytes < need) {
    set_error("gated_ffn_bwd: workspace %zu < %zu bytes (query mragan_gated_ffn_workspace)", ws_bytes, need);
    return kWorkspace;
  }
  return gated_ffn_bwd(f, mode, dy, kept, o, ws, static_cast<hipStream_t>(stream));
}

int64_t mragan_linear_recurrence_carries(int64_t T, int C) { return C > 0 ? recurrence_carries(T) : 0; }
size_t mragan_linear_recurrence_workspace(int64_t B, int64_t T, int C, int backward) {
  (void)backward;
  return C > 0 ? recurrence_ws_bytes(B, T, C) : 0;
}

// Channels of a recurrence, exclusive: a lane's offset in its chunk, up to 120 rows and a tile of 64 channels,
// stays below 2³² elements.
constexpr int64_t kMaxRecurChannels = (int64_t)1 << 25;
// Time strides: rows that follow each other, or less than 2²² apart.  A single step has none.
static bool time_stride_ok(int64_t T, int64_t st, int C) { return T == 1 || st == C || (st >= 0 && st < ((int64_t)1 << 22)); }

static int recur_check(const RecurArgs& r, const void* ws, size_t ws_bytes) {
  MRAGAN_CHECK_ARG(r.B >= 0 && r.T > 0 && r.C > 0, "linear_recurrence: bad shape [%lld][%lld][%d]", (long long)r.B,
                   (long long)r.T, r.C);
  MRAGAN_CHECK_ARG(dtype_ok(r.dtype), "linear_recurrence: unknown dtype %d", r.dtype);
  MRAGAN_CHECK_ARG(r.reverse == 0 || r.reverse == 1, "linear_recurrence: reverse must be 0/1");
  if (r.B == 0) return kOk;
  MRAGAN_CHECK_ARG(r.x && r.decay, "linear_recurrence: null pointer");
  MRAGAN_CHECK_ARG(r.C < kMaxRecurChannels && time_stride_ok(r.T, r.x_st, r.C) && time_stride_ok(r.T, r.d_st, r.C) &&
                       (!r.gate || time_stride_ok(r.T, r.g_st, r.C)),
                   "linear_recurrence: C must be below 2^25, time strides C or in [0, 2^22)");
  MRAGAN_CHECK_ARG(r.B <= kMaxThreads && recurrence_threads(r.B, r.T, r.C) < kMaxThreads, "linear_recurrence: too many sequences");
  const size_t need = recurrence_ws_bytes(r.B, r.T, r.C);
  if (need && (!ws || ws_bytes < need)) {
    set_error("linear_recurrence: workspace %zu < %zu bytes (query mragan_linear_recurrence_workspace)", ws_bytes, need);
    return kWorkspace;
  }
  return kOk;
}

int mragan_linear_recurrence_fwd(const void* x, int64_t x_sb, int64_t x_st, const void* decay, int64_t d_sb, int64_t d_st,
                                 const void* gate, int64_t g_sb, int64_t g_st, const float* h0, int64_t B, int64_t T, int C,
                                 int dtype, int reverse, void* y, float* last, float* carry, void* ws, size_t ws_bytes,
                                 void* stream) {
  const RecurArgs r{x, x_sb, x_st, decay, d_sb, d_st, gate, g_sb, g_st, B, T, C, dtype, reverse};
  if (int rc = recur_check(r, ws, ws_bytes)) return rc;
  if (B == 0) return kOk;
  MRAGAN_CHECK_ARG(y && last, "linear_recurrence: null pointer");
  return recurrence_fwd(r, h0, y, last, carry, static_cast<float*>(ws), static_cast<hipStream_t>(stream));
}

int mragan_linear_recurrence_bwd(const void* x, int64_t x_sb, int64_t x_st, const void* decay, int64_t d_sb, int64_t d_st,
                                 const void* gate, int64_t g_sb, int64_t g_st, const float* carry, const void* dy,
                                 int64_t dy_sb, int64_t dy_st, const float* dlast, int64_t B, int64_t T, int C, int dtype,
                                 int reverse, void* dx, void* ddecay, void* dgate, float* dh0, void* ws, size_t ws_bytes,
                                 void* stream) {
  const RecurArgs r{x, x_sb, x_st, decay, d_sb, d_st, gate, g_sb, g_st, B, T, C, dtype, reverse};
  if (int rc = recur_check(r, ws, ws_bytes)) return rc;
  if (B == 0 || (!dx && !ddecay && !dgate && !dh0)) return kOk;
  MRAGAN_CHECK_ARG(carry && dy, "linear_recurrence_bwd: null pointer");
  MRAGAN_CHECK_ARG(time_stride_ok(T, dy_st, C), "linear_recurrence_bwd: time strides must be C or in [0, 2^22)");
  MRAGAN_CHECK_ARG(gate || !dgate, "linear_recurrence_bwd: dgate without a gate");
  return recurrence_bwd(r, carry, dy, dy_sb, dy_st, dlast, dx, ddecay, dgate, dh0, static_cast<float*>(ws),
                        static_cast<hipStream_t>(stream));
}

}  // extern "C"
