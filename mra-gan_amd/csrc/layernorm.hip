// LayerNorm over the channels of channels-last rows, forward and backward.
//
//   fwd   μ = mean_c x,  rstd = (mean_c (x − μ)² + eps)^−½,  y = (x − μ)·rstd·w + b
//   bwd   p = dy·w,  x̂ = (x − μ)·rstd,  dx = rstd·(p − mean_c p − x̂·mean_c(p·x̂)),
//         dw = Σ_rows dy·x̂,  db = Σ_rows dy
//
// Both directions read and write each tensor once, fwd x and y, bwd x, dy and dx, and HBM is the bound of fwd and
// of bwd over short rows; over rows that a block shares, bwd waits for the block's barriers, three a row.  So a row lives in the registers of the G lanes that own it (G = 4 … 64 lanes of a wave, or a
// block of 256 / 1024 threads), every sum is taken from there (the variance as the mean of squared
// deviations, exact for rows far from zero), a block walks over rows with the next row's loads in
// flight, and w and b are loaded once per block.  The weight's gradient is summed per lane over the
// rows of its block in fp32, then over the block's row groups in LDS, then over the blocks by a
// second launch: a fixed order, no atomics.
// Measured: 524288 rows of 32 fp32 channels 27 us forward (134 MB, 5.0 TB/s), 33 + 4 us backward (201 MB, 6.1 TB/s:
// x comes from the cache); 8192 rows of 2048 bf16 channels 14.3 us forward (67 MB, 4.7 TB/s), 28.6 + 4.3 us backward
// (101 MB, 3.5 TB/s).  A copy of 256 MB moves 5.4 TB/s.
#include "token_ops.h"

// Columns that two lanes share (kOverlap) are formed in different slots of theirs and written by both, so their
// bits have to be the same in each: the compiler joins no product and sum by itself, fma says where one rounding
// is meant.
#pragma clang fp contract(off)

namespace mragan {
namespace {

constexpr int kThreads = 256;

// A lane's 16 bytes of a row.  Rows of any channel count start at any element; gfx950 takes global
// accesses of any alignment.  How a row ends:
//   kExact    C is a multiple of N: a vector is inside the row or behind it
//   kOverlap  the last vector of a row is moved back to end with it; what it shares with the one before
//             is left out of the sums and written twice, with the same value
//   kTiny     C < N: element by element
enum RowEnd : int { kExact = 0, kOverlap = 1, kTiny = 2 };
template <typename T>
constexpr int vec_len() { return 16 / sizeof(T); }

// vector of the columns from `col`: where it is loaded, and how many of its elements to skip (N: all)
struct Slot {
  int at, skip;
};
template <int N, int END>
__device__ __forceinline__ Slot slot(int col, int C) {
  if (col >= C) return {0, N};
  if (END == kOverlap && col + N > C) return {C - N, col + N - C};
  return {col, 0};
}
template <int N, int END, typename T>
__device__ __forceinline__ Words<T, N> vec_load(const T* row, Slot s, int C) {
  Words<T, N> r{};
  if constexpr (END == kTiny) {
#pragma unroll
    for (int i = 0; i < N; i++) r.set(i, s.skip == 0 && i < C ? (float)row[i] : 0.f);
  } else {
    if (s.skip < N) __builtin_memcpy(&r, row + s.at, sizeof(r));
  }
  return r;
}
template <int N, int END, typename T>
__device__ __forceinline__ void vec_store(T* row, Slot s, int C, const Words<T, N>& r) {
  if constexpr (END == kTiny) {
#pragma unroll
    for (int i = 0; i < N; i++)
      if (s.skip == 0 && i < C) row[i] = (T)r.get(i);
  } else {
    if (s.skip < N) __builtin_memcpy(row + s.at, &r, sizeof(r));
  }
}
// whether element j of a vector counts
template <int N, int END>
__device__ __forceinline__ bool counts(Slot s, int j, int C) {
  if constexpr (END == kTiny) return s.skip == 0 && j < C;
  else if constexpr (END == kExact) return s.skip == 0;
  else return j >= s.skip;
}

// sum over the G lanes of a row; G > 64: over the block's waves through `red` (one slot per wave),
// which the caller must not reuse before its next barrier
template <int G>
__device__ __forceinline__ float row_sum(float v, float* red) {
  if constexpr (G <= 64) {
    return group_sum<G>(v);
  } else {
    v = group_sum<64>(v);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < G / 64; i++) s += red[i];
    return s;
  }
}

template <typename T, typename W, int G, int NV, int END>
__global__ __launch_bounds__(kThreads) void ln_fwd_kernel(const T* x, int64_t rows, int C, const W* w, const W* b, float eps, T* y,
                                                          float* mean, float* rstd) {
  constexpr int N = vec_len<T>();
  __shared__ float red[2][16];
  const int lane = threadIdx.x % G;
  const int64_t step = (int64_t)gridDim.x * (kThreads / G);
  int64_t row = (int64_t)blockIdx.x * (kThreads / G) + threadIdx.x / G;
  const float inv = 1.f / (float)C;
  Slot at[NV];
  Words<W, N> wv[NV], bv[NV];                                        // held for all rows of the block
  Words<T, N> cur[NV], nxt[NV];
#pragma unroll
  for (int i = 0; i < NV; i++) {
    at[i] = slot<N, END>((i * G + lane) * N, C);
    if (row < rows) cur[i] = vec_load<N, END>(x + row * C, at[i], C);
    if (w) wv[i] = vec_load<N, END>(w, at[i], C);
    if (b) bv[i] = vec_load<N, END>(b, at[i], C);
  }
  for (; row < rows; row += step) {
    if (row + step < rows) {
#pragma unroll
      for (int i = 0; i < NV; i++) nxt[i] = vec_load<N, END>(x + (row + step) * C, at[i], C);
    }
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
      for (int j = 0; j < N; j++)                                      // vectors behind the row hold zeros
        if (END != kOverlap || counts<N, END>(at[i], j, C)) s += cur[i].get(j);
    const float mu = row_sum<G>(s, red[0]) * inv;
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
      for (int j = 0; j < N; j++) {
        const float d = cur[i].get(j) - mu;
        q = counts<N, END>(at[i], j, C) ? fma(d, d, q) : q;
      }
    const float r = rsqrtf(row_sum<G>(q, red[1]) * inv + eps);
#pragma unroll
    for (int i = 0; i < NV; i++) {
      Words<T, N> o;
#pragma unroll
      for (int j = 0; j < N; j++) {
        float v = (cur[i].get(j) - mu) * r;
        if (w) v *= wv[i].get(j);
        if (b) v += bv[i].get(j);
        o.set(j, v);
      }
      vec_store<N, END>(y + row * C, at[i], C, o);
    }
    if (lane == 0) {
      mean[row] = mu;
      rstd[row] = r;
    }
    if constexpr (G > 64) __syncthreads();                           // red is read before the next row writes it
#pragma unroll
    for (int i = 0; i < NV; i++) cur[i] = nxt[i];
  }
}

// part: [gridDim.x][2][C] fp32 sums of this block's rows (Σ dy·x̂, Σ dy), or null
template <typename T, typename W, int G, int NV, int END>
__global__ __launch_bounds__(G > kThreads ? G : kThreads) void ln_bwd_kernel(const T* x, const float* mean, const float* rstd,
                                                                             const T* dy, int64_t rows, int C, const W* w,
                                                                             T* dx, float* part) {
  constexpr int N = vec_len<T>(), BT = G > kThreads ? G : kThreads, E = NV * N;
  __shared__ float red[2][16];
  __shared__ float acc_s[G <= 64 ? BT / 64 : 1][G <= 64 ? G * E + 1 : 1];
  const int lane = threadIdx.x % G;
  const int64_t step = (int64_t)gridDim.x * (BT / G);
  int64_t row = (int64_t)blockIdx.x * (BT / G) + threadIdx.x / G;
  const float inv = 1.f / (float)C;
  Slot at[NV];
  Words<W, N> wv[NV];
  Words<T, N> cx[NV], cd[NV], nx[NV], nd[NV];
  float aw[NV][N], ab[NV][N], mu = 0.f, r = 0.f, nmu = 0.f, nr = 0.f;
#pragma unroll
  for (int i = 0; i < NV; i++) {
    at[i] = slot<N, END>((i * G + lane) * N, C);
    if (row < rows) {
      cx[i] = vec_load<N, END>(x + row * C, at[i], C);
      cd[i] = vec_load<N, END>(dy + row * C, at[i], C);
    }
    if (w) wv[i] = vec_load<N, END>(w, at[i], C);
#pragma unroll
    for (int j = 0; j < N; j++) aw[i][j] = ab[i][j] = 0.f;
  }
  if (row < rows) mu = mean[row], r = rstd[row];
  for (; row < rows; row += step) {
    if (row + step < rows) {
#pragma unroll
      for (int i = 0; i < NV; i++) {
        nx[i] = vec_load<N, END>(x + (row + step) * C, at[i], C);
        nd[i] = vec_load<N, END>(dy + (row + step) * C, at[i], C);
      }
      nmu = mean[row + step];
      nr = rstd[row + step];
    }
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
      for (int j = 0; j < N; j++) {                                  // dy is zero behind the row
        const float d = cd[i].get(j), xh = (cx[i].get(j) - mu) * r, p = w ? d * wv[i].get(j) : d;
        if (END != kOverlap || counts<N, END>(at[i], j, C)) {
          s1 += p;
          s2 = fma(p, xh, s2);
        }
        aw[i][j] = fma(d, xh, aw[i][j]);
        ab[i][j] += d;
      }
    if (dx) {
      const float m1 = row_sum<G>(s1, red[0]) * inv, m2 = row_sum<G>(s2, red[1]) * inv;
#pragma unroll
      for (int i = 0; i < NV; i++) {
        Words<T, N> o;
#pragma unroll
        for (int j = 0; j < N; j++) {
          const float d = cd[i].get(j), xh = (cx[i].get(j) - mu) * r, p = w ? d * wv[i].get(j) : d;
          o.set(j, r * fma(-xh, m2, p - m1));
        }
        vec_store<N, END>(dx + row * C, at[i], C, o);
      }
      if constexpr (G > 64) __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < NV; i++) {
      cx[i] = nx[i];
      cd[i] = nd[i];
    }
    mu = nmu;
    r = nr;
  }
  if (!part) return;
  float* out = part + (int64_t)blockIdx.x * 2 * C;
  if constexpr (G > 64) {                                            // one row group: nothing to join
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
      for (int j = 0; j < N; j++)
        if (counts<N, END>(at[i], j, C)) {
          out[at[i].at + j] = aw[i][j];
          out[C + at[i].at + j] = ab[i][j];
        }
  } else {
    const int wave = threadIdx.x >> 6;
#pragma unroll
    for (int k = 0; k < 2; k++) {                                    // dw, then db through the same LDS
      if (k) __syncthreads();
#pragma unroll
      for (int i = 0; i < NV; i++)
#pragma unroll
        for (int j = 0; j < N; j++) {
          float v = k ? ab[i][j] : aw[i][j];
          // the row groups of a wave: lanes that differ in the bits above G
          if constexpr (G <= 4) v += __shfl_xor(v, 4);
          if constexpr (G <= 8) v += __shfl_xor(v, 8);
          if constexpr (G <= 16) v += __shfl_xor(v, 16);
          if constexpr (G <= 32) v += __shfl_xor(v, 32);
          if ((threadIdx.x & 63) < G && counts<N, END>(at[i], j, C)) acc_s[wave][at[i].at + j] = v;
        }
      __syncthreads();
      for (int col = threadIdx.x; col < C; col += BT) {
        float v = 0.f;
#pragma unroll
        for (int q = 0; q < BT / 64; q++) v += acc_s[q][col];
        out[k * C + col] = v;
      }
    }
  }
}

// Σ over the nb blocks' partials: a block takes 32 of the 2C columns with 32 threads each, then the next
// 32 behind those of the launch's other blocks
template <typename W>
__global__ __launch_bounds__(1024) void ln_param_reduce_kernel(const float* part, int nb, int C, W* dw, W* db) {
  __shared__ float s[32][33];
  const int cl = threadIdx.x & 31, slot = threadIdx.x >> 5;
  const int64_t n = 2 * (int64_t)C, step = (int64_t)gridDim.x * 32;
  for (int64_t c0 = (int64_t)blockIdx.x * 32; c0 < n; c0 += step) {
    const int64_t col = c0 + cl;
    float v = 0.f;
    if (col < n) {
#pragma unroll 8
      for (int k = slot; k < nb; k += 32) v += part[k * n + col];
    }
    s[slot][cl] = v;
    __syncthreads();
    if (slot == 0 && col < n) {
      v = 0.f;
#pragma unroll
      for (int k = 0; k < 32; k++) v += s[k][cl];
      if (col < C) {
        if (dw) dw[col] = (W)v;
      } else if (db) {
        db[col - C] = (W)v;
      }
    }
    if (c0 + step < n) __syncthreads();                                // s is read before the next columns write it
  }
}

// Rows of more channels than the registers of a block hold (C > kMaxRow): the block walks the row
// in memory, once per sum; the parameter gradients take a column per thread over a run of rows.  Loads of single
// elements: 4096 rows of 16384 bf16 channels take 124 us forward (268 MB, floor 53) and 252 backward (403 MB, 79).
template <typename T, typename W>
__global__ __launch_bounds__(1024) void ln_fwd_long_kernel(const T* x, int64_t rows, int C, const W* w, const W* b, float eps,
                                                           T* y, float* mean, float* rstd) {
  __shared__ float red[2][16];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + row * C;
    float s = 0.f, q = 0.f;
    for (int c = threadIdx.x; c < C; c += 1024) s += (float)xr[c];
    const float mu = row_sum<1024>(s, red[0]) / (float)C;
    for (int c = threadIdx.x; c < C; c += 1024) {
      const float d = (float)xr[c] - mu;
      q = fma(d, d, q);
    }
    const float r = rsqrtf(row_sum<1024>(q, red[1]) / (float)C + eps);
    for (int c = threadIdx.x; c < C; c += 1024)
      y[row * C + c] = (T)(((float)xr[c] - mu) * r * (w ? (float)w[c] : 1.f) + (b ? (float)b[c] : 0.f));
    if (threadIdx.x == 0) {
      mean[row] = mu;
      rstd[row] = r;
    }
    __syncthreads();                                                 // red is read before the next row writes it
  }
}
template <typename T, typename W>
__global__ __launch_bounds__(1024) void ln_bwd_long_kernel(const T* x, const float* mean, const float* rstd, const T* dy,
                                                           int64_t rows, int C, const W* w, T* dx) {
  __shared__ float red[2][16];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const float mu = mean[row], r = rstd[row];
    float s1 = 0.f, s2 = 0.f;
    for (int c = threadIdx.x; c < C; c += 1024) {
      const float p = (float)dy[row * C + c] * (w ? (float)w[c] : 1.f);
      s1 += p;
      s2 = fma(p, ((float)x[row * C + c] - mu) * r, s2);
    }
    const float m1 = row_sum<1024>(s1, red[0]) / (float)C, m2 = row_sum<1024>(s2, red[1]) / (float)C;
    for (int c = threadIdx.x; c < C; c += 1024) {
      const float xh = ((float)x[row * C + c] - mu) * r, p = (float)dy[row * C + c] * (w ? (float)w[c] : 1.f);
      dx[row * C + c] = (T)(r * fma(-xh, m2, p - m1));
    }
    __syncthreads();
  }
}
// part: [gridDim.y][2][C], rows dealt to gridDim.y in runs of `per`
template <typename T>
__global__ __launch_bounds__(256) void ln_param_long_kernel(const T* x, const float* mean, const float* rstd, const T* dy,
                                                            int64_t rows, int64_t per, int C, float* part) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= C) return;
  const int64_t k0 = blockIdx.y * per, k1 = k0 + per < rows ? k0 + per : rows;
  float sw = 0.f, sb = 0.f;
#pragma unroll 8
  for (int64_t k = k0; k < k1; k++) {
    const float d = (float)dy[k * C + c];
    sw = fma(d, ((float)x[k * C + c] - mean[k]) * rstd[k], sw);
    sb += d;
  }
  float* out = part + (int64_t)blockIdx.y * 2 * C;
  out[c] = sw;
  out[C + c] = sb;
}

// The largest row that a block holds: 16 channels a thread of 512 (backward: their 256 registers also
// carry the next row, the weight and two accumulators), 32 a thread of 256 (forward).
constexpr int kMaxRow = 8192;
// A launch takes fewer than 2^32 threads, and says nothing of more (it leaves some of its blocks out): at most
// 2^16 blocks of 1024, of the longer rows' kernels and of the parameter sums
unsigned bounded_grid(int64_t blocks) { return (unsigned)(blocks < 65536 ? blocks : 65536); }
// Most blocks of a backward launch: four on each of the 256 CUs, whose partial sums the second launch reads
constexpr int kMaxBwdBlocks = 1024;

// Lanes per row and 16-byte vectors per lane.  A wave or a part of one per row as long as `most`
// channels a lane suffice, else the block.  Rows of more than 64 vectors take a block each where there
// are no more than `few`, so that more CUs share the loads.
struct Shape {
  int G, NV;
};
Shape pick(int64_t rows, int C, int N, int most, int few) {
  const int V = ceil_div(C, N);
  for (int g = 4; g <= 64; g *= 2)
    if (V <= g) return {g, 1};
  for (int g : {64, 256}) {
    if (g == 64 && rows <= few) continue;
    for (int nv = 1; nv * N <= most; nv *= 2)
      if (V <= g * nv) return {g, nv};
  }
  return {512, 16 / N};
}

template <typename T, typename W>
int ln_fwd(const void* x, int64_t rows, int C, const void* w, const void* b, float eps, void* y, float* mean, float* rstd,
           hipStream_t st) {
  constexpr int N = vec_len<T>();
  const T* xt = static_cast<const T*>(x);
  const W *wt = static_cast<const W*>(w), *bt = static_cast<const W*>(b);
  T* yt = static_cast<T*>(y);
  if (C > kMaxRow) {
    ln_fwd_long_kernel<T, W><<<bounded_grid(rows), 1024, 0, st>>>(xt, rows, C, wt, bt, eps, yt, mean, rstd);
    return check_launch("layer_norm_fwd_long");
  }
  // bf16, 2048 channels: 64 rows take 2.6 us with a block each, 3.3 with a wave; 1024 channels: 256 rows
  // 2.5 and 2.7, 1024 rows 3.3 and 3.0
  const Shape s = pick(rows, C, N, 32, 512);
  const int64_t per = kThreads / s.G, blocks = (rows + per - 1) / per, most = 2048;
  const unsigned grid = (unsigned)(blocks < most ? blocks : most);
#define LN_END(G_, NV_, END_)                                                                                            \
  ln_fwd_kernel<T, W, G_, NV_, END_><<<grid, kThreads, 0, st>>>(xt, rows, C, wt, bt, eps, yt, mean, rstd)
#define LN_RUN(G_, NV_)                                                   \
  if constexpr (NV_ * N <= 32) {                                          \
    if (s.G == G_ && s.NV == NV_) {                                       \
      if (C % N == 0) LN_END(G_, NV_, kExact);                            \
      else LN_END(G_, NV_, kOverlap);                                     \
      return check_launch("layer_norm_fwd");                              \
    }                                                                     \
  }
  if (C < N) {
    LN_END(4, 1, kTiny);
    return check_launch("layer_norm_fwd");
  }
  LN_RUN(4, 1) LN_RUN(8, 1) LN_RUN(16, 1) LN_RUN(32, 1) LN_RUN(64, 1) LN_RUN(64, 2) LN_RUN(64, 4) LN_RUN(64, 8)
  LN_RUN(256, 1) LN_RUN(256, 2) LN_RUN(256, 4) LN_RUN(256, 8)
#undef LN_RUN
#undef LN_END
  set_error("layer_norm_fwd: no kernel for C = %d", C);
  return kUnsupported;
}

// Half the forward's channels a lane: 8192 rows of 2048 bf16 channels take 27.7 us with a block a row,
// 29.2 with 32 channels a lane of a wave.  No block a row for few rows: each block's sums are as long as
// a row, and 1024 rows of 1024 channels take 14.5 us with 1024 such blocks, 7.3 with a wave a row.
Shape bwd_shape(int C, int N) { return pick(0, C, N, 16, -1); }
// As many blocks as the chip holds, but at least eight row groups each where that leaves one block for
// every CU, as each block adds 8·C bytes of sums: 2048 rows of 2048 bf16 channels take 15.2 us, 17.0 with
// four groups each, 24.8 with one.
int bwd_blocks(int64_t rows, int C, int N) {
  const Shape s = bwd_shape(C, N);
  const int per = s.G > kThreads ? 1 : kThreads / s.G;
  const int64_t groups = (rows + per - 1) / per, most = s.G > kThreads ? kMaxBwdBlocks / 2 : kMaxBwdBlocks;
  const int64_t few = groups < 256 ? groups : 256, blocks = groups / 8 > few ? groups / 8 : few;
  return (int)(blocks < most ? blocks : most);
}

// row runs of the long rows' parameter sums, 64 rows each up to 64 runs
int long_chunks(int64_t rows) { return rows > 64 * 64 ? 64 : (int)((rows + 63) / 64); }

template <typename T, typename W>
int ln_bwd(const void* x, const float* mean, const float* rstd, const void* dy, int64_t rows, int C, const void* w, void* dx,
           void* dw, void* db, float* part, hipStream_t st) {
  constexpr int N = vec_len<T>();
  const T *xt = static_cast<const T*>(x), *dyt = static_cast<const T*>(dy);
  const W* wt = static_cast<const W*>(w);
  T* dxt = static_cast<T*>(dx);
  W *dwt = static_cast<W*>(dw), *dbt = static_cast<W*>(db);
  const bool params = dw || db;
  if (C > kMaxRow) {
    if (dx) {
      ln_bwd_long_kernel<T, W><<<bounded_grid(rows), 1024, 0, st>>>(xt, mean, rstd, dyt, rows, C, wt, dxt);
      if (int rc = check_launch("layer_norm_bwd_long")) return rc;
    }
    if (!params) return kOk;
    const int chunks = long_chunks(rows);
    ln_param_long_kernel<T><<<dim3(ceil_div(C, 256), chunks), 256, 0, st>>>(xt, mean, rstd, dyt, rows, (rows + chunks - 1) / chunks, C,
                                                                            part);
    if (int rc = check_launch("layer_norm_param_long")) return rc;
    ln_param_reduce_kernel<W><<<bounded_grid(ceil_div(2 * (int64_t)C, 32)), 1024, 0, st>>>(part, chunks, C, dwt, dbt);
    return check_launch("layer_norm_param_reduce");
  }
  const Shape s = bwd_shape(C, N);
  const unsigned grid = bwd_blocks(rows, C, N);
  if (!params) part = nullptr;
  int rc = kUnsupported;
#define LN_END(G_, NV_, END_)                                                                                            \
  ln_bwd_kernel<T, W, G_, NV_, END_><<<grid, G_ > kThreads ? G_ : kThreads, 0, st>>>(xt, mean, rstd, dyt, rows, C, wt, dxt, part)
#define LN_RUN(G_, NV_)                                                   \
  if constexpr (NV_ * N <= 16) {                                          \
    if (C >= N && s.G == G_ && s.NV == NV_) {                             \
      if (C % N == 0) LN_END(G_, NV_, kExact);                            \
      else LN_END(G_, NV_, kOverlap);                                     \
      rc = check_launch("layer_norm_bwd");                                \
    }                                                                     \
  }
  if (C < N) {
    LN_END(4, 1, kTiny);
    rc = check_launch("layer_norm_bwd");
  }
  LN_RUN(4, 1) LN_RUN(8, 1) LN_RUN(16, 1) LN_RUN(32, 1) LN_RUN(64, 1) LN_RUN(64, 2) LN_RUN(64, 4)
  LN_RUN(256, 1) LN_RUN(256, 2) LN_RUN(256, 4) LN_RUN(512, 16 / N)
#undef LN_RUN
#undef LN_END
  if (rc) return rc;
  if (params) {
    ln_param_reduce_kernel<W><<<bounded_grid(ceil_div(2 * (int64_t)C, 32)), 1024, 0, st>>>(part, (int)grid, C, dwt, dbt);
    return check_launch("layer_norm_param_reduce");
  }
  return kOk;
}

template <typename W>
__global__ void ln_zero_kernel(W* dw, W* db, int C) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= C) return;
  if (dw) dw[c] = (W)0.f;
  if (db) db[c] = (W)0.f;
}

}  // namespace

size_t layer_norm_bwd_ws_bytes(int64_t rows, int C, int dtype) {
  if (rows == 0) return 0;
  return (size_t)(C > kMaxRow ? long_chunks(rows) : bwd_blocks(rows, C, dtype == kF32 ? 4 : 8)) * 2 * C * sizeof(float);
}

int layer_norm_fwd(const void* x, int64_t rows, int C, int dtype, const void* w, const void* b, int wdtype, float eps, void* y,
                   float* mean, float* rstd, hipStream_t st) {
  if (rows == 0) return kOk;
  MRAGAN_DTYPE_DISPATCH(dtype, T, {
    if (wdtype == kF32) return ln_fwd<T, float>(x, rows, C, w, b, eps, y, mean, rstd, st);
    return ln_fwd<T, T>(x, rows, C, w, b, eps, y, mean, rstd, st);
  })
  return kOk;
}

int layer_norm_bwd(const void* x, const float* mean, const float* rstd, const void* dy, int64_t rows, int C, int dtype,
                   const void* w, int wdtype, void* dx, void* dw, void* db, float* part, hipStream_t st) {
  if (rows == 0) {                                                   // empty sums
    if (!dw && !db) return kOk;
    MRAGAN_DTYPE_DISPATCH(wdtype, W, {
      ln_zero_kernel<W><<<ceil_div(C, 256), 256, 0, st>>>(static_cast<W*>(dw), static_cast<W*>(db), C);
    })
    return check_launch("layer_norm_zero");
  }
  MRAGAN_DTYPE_DISPATCH(dtype, T, {
    if (wdtype == kF32) return ln_bwd<T, float>(x, mean, rstd, dy, rows, C, w, dx, dw, db, part, st);
    return ln_bwd<T, T>(x, mean, rstd, dy, rows, C, w, dx, dw, db, part, st);
  })
  return kOk;
}

}  // namespace mragan
