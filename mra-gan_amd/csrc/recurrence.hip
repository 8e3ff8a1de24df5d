// Gated linear recurrence along the time axis of [B][T][C] tensors, forward and backward.
//
//   a_t = σ(d_t), i_t = σ(−d_t)      h_t = a_t·h_{t−1} + i_t·x_t      y_t = h_t·silu(z_t)  (or h_t)
//   G_t = dy_t·silu(z_t) + Q_{t+1},  Q_t = a_t·G_t  (Q_T = dlast, dh0 = Q_0)
//   dx_t = G_t·i_t,  dd_t = G_t·(h_{t−1} − x_t)·a_t·i_t,  dz_t = dy_t·h_t·silu'(z_t)
//
// Both recursions are products of affine maps s ↦ P·s + E, which compose associatively, so time is
// split: a lane takes S steps of kVC channels in order, the LT time lanes of a block join their
// (P, E) through LDS (a chunk of kChunk = LT·S steps), and a block walks over the chunks with the
// state of 64 channels in fp32.  HBM is the bound: each tensor is read or written once.  Where B and
// C give too few blocks to fill the chip, the chunks are also split into segments over blocks: a
// first launch reduces each segment to its (P, E), the second starts each segment from the fold
// of the ones before it (its inputs then come a second time, as a rule from the 256 MB cache).
// The forward leaves the fp32 state entering each chunk; the backward recomputes the states of a
// chunk from it in registers and walks the chunks backwards, so that no state is read or written.
#include "token_ops.h"

namespace mragan {
namespace {

constexpr int kVC = 4;          // channels a lane
constexpr int kChunk = 128;     // steps between two carried states
constexpr int kLC = 16;         // channel lanes: 64 channels, 128 bytes of a 16-bit row
constexpr int kCT = kLC * kVC;
constexpr int kShort = 16;      // sequences up to this long: a thread walks the whole sequence

template <typename T>
struct Strided {                // element (b, t, c) at p[b·sb + t·st + c]
  const T* p;
  int64_t sb, st;
};

// kVC channels of one step; lanes past C hold zeros
template <typename T>
struct Quad {
  T v[kVC];
};
template <typename T>
__device__ __forceinline__ Quad<T> quad_load(const T* p, int n) {    // n: channels left, ≥ 1
  Quad<T> r;
  if (n >= kVC) {
    __builtin_memcpy(&r, p, sizeof(r));
  } else {
#pragma unroll
    for (int i = 0; i < kVC; i++) r.v[i] = i < n ? p[i] : (T)0.f;
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void quad_store(T* p, int n, const Quad<T>& r) {
  if (n >= kVC) {
    __builtin_memcpy(p, &r, sizeof(r));
  } else {
#pragma unroll
    for (int i = 0; i < kVC; i++)
      if (i < n) p[i] = r.v[i];
  }
}

__device__ __forceinline__ float silu(float z) {
  float s, n;
  sigmoid_pair(z, s, n);
  return z * s;
}
// z·σ(z) and its derivative σ(z)·(1 + z·σ(−z))
__device__ __forceinline__ void silu_pair(float z, float& f, float& df) {
  float s, n;
  sigmoid_pair(z, s, n);
  f = z * s;
  df = s * (1.f + z * n);
}

struct Geo {
  int64_t B, T;
  int C, reverse;
  int tiles;                    // channel tiles
  int64_t chunks, per_seg;      // chunks of a sequence, chunks of a segment
  int segs;
  __device__ __forceinline__ int64_t at(int64_t t) const { return reverse ? T - 1 - t : t; }
};

// this block's (sequence, segment, first channel)
struct Place {
  int64_t b, k0, k1;
  int seg, c0;
};
__device__ __forceinline__ Place place(const Geo& g) {
  Place p;
  int64_t id = blockIdx.x;
  p.c0 = (int)(id % g.tiles) * kCT;
  id /= g.tiles;
  p.seg = (int)(id % g.segs);
  p.b = id / g.segs;
  p.k0 = p.seg * g.per_seg;
  p.k1 = p.k0 + g.per_seg < g.chunks ? p.k0 + g.per_seg : g.chunks;
  return p;
}

// ---- segment maps: (P, E) of each segment, agg [B][segs][2][C] --------------------------------
// Each time lane walks one contiguous span of the segment, so the lanes join once, at its end.
// BWD: the map of Q from the segment's end to its start (E from dy, z); else that of h (E from x).
template <typename T, bool BWD, int LT>
__global__ __launch_bounds__(kLC* LT) void recur_segment_kernel(Strided<T> e, Strided<T> d, Strided<T> z, Geo g, float* agg) {
  __shared__ float sP[LT][kCT], sE[LT][kCT];
  const Place pl = place(g);
  const int cl = threadIdx.x % kLC, lt = threadIdx.x / kLC, c = pl.c0 + cl * kVC, n = g.C - c;
  const int64_t first = pl.k0 * kChunk, end = pl.k1 * kChunk < g.T ? pl.k1 * kChunk : g.T;
  const int64_t span = (end - first + LT - 1) / LT;
  const int64_t t0 = first + lt * span, t1 = t0 + span < end ? t0 + span : end;
  float P[kVC], E[kVC];
#pragma unroll
  for (int v = 0; v < kVC; v++) P[v] = 1.f, E[v] = 0.f;
  if (n > 0) {
    const T *ep = e.p + pl.b * e.sb + c, *dp = d.p + pl.b * d.sb + c, *zp = z.p ? z.p + pl.b * z.sb + c : nullptr;
    constexpr int U = 8;
    for (int64_t t = t0; t < t1; t += U) {
      Quad<T> qe[U], qd[U], qz[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        int64_t k = t + u < t1 ? t + u : t1 - 1;
        if constexpr (BWD) k = t0 + t1 - 1 - k;                       // from the span's end to its start
        k = g.at(k);
        qe[u] = quad_load(ep + k * e.st, n);
        qd[u] = quad_load(dp + k * d.st, n);
        if (BWD && zp) qz[u] = quad_load(zp + k * z.st, n);
      }
#pragma unroll
      for (int u = 0; u < U; u++)
        if (t + u < t1) {
#pragma unroll
          for (int v = 0; v < kVC; v++) {
            float a, i;
            sigmoid_pair((float)qd[u].v[v], a, i);
            const float in = (float)qe[u].v[v];
            if constexpr (BWD) E[v] = a * (E[v] + (zp ? in * silu((float)qz[u].v[v]) : in));
            else E[v] = a * E[v] + i * in;
            P[v] *= a;
          }
        }
    }
  }
#pragma unroll
  for (int v = 0; v < kVC; v++) sP[lt][cl * kVC + v] = P[v], sE[lt][cl * kVC + v] = E[v];
  __syncthreads();
  for (int ch = threadIdx.x; ch < kCT; ch += kLC * LT) {
    if (pl.c0 + ch >= g.C) continue;
    float p = 1.f, s = 0.f;
#pragma unroll
    for (int j = 0; j < LT; j++) {
      const int l = BWD ? LT - 1 - j : j;
      s = sP[l][ch] * s + sE[l][ch];
      p *= sP[l][ch];
    }
    float* out = agg + ((pl.b * g.segs + pl.seg) * 2) * g.C + pl.c0 + ch;
    out[0] = p;
    out[g.C] = s;
  }
}

// the state entering this block's segment: `s` run through the maps before it
template <bool BWD>
__device__ __forceinline__ float enter_segment(const float* agg, const Geo& g, const Place& pl, int ch, float s) {
  const float* q = agg + pl.b * g.segs * 2 * (int64_t)g.C + pl.c0 + ch;
  if constexpr (BWD) {
    for (int k = g.segs - 1; k > pl.seg; k--) s = q[2 * (int64_t)k * g.C] * s + q[(2 * (int64_t)k + 1) * g.C];
  } else {
    for (int k = 0; k < pl.seg; k++) s = q[2 * (int64_t)k * g.C] * s + q[(2 * (int64_t)k + 1) * g.C];
  }
  return s;
}

// ---- forward ----------------------------------------------------------------------------------
template <typename T, int LT>
__global__ __launch_bounds__(kLC* LT) void recur_fwd_kernel(Strided<T> x, Strided<T> d, Strided<T> z, const float* h0, Geo g,
                                                            const float* agg, T* y, float* last, float* carry) {
  constexpr int S = kChunk / LT;
  // two sets: a chunk's maps are written while slower waves still read those of the chunk before
  __shared__ __attribute__((aligned(16))) float sP[2][LT][kCT], sE[2][LT][kCT], sH[2][kCT];
  const Place pl = place(g);
  const int cl = threadIdx.x % kLC, lt = threadIdx.x / kLC, c = pl.c0 + cl * kVC, n = g.C - c;
  if (threadIdx.x < kCT) {
    const int ch = pl.c0 + threadIdx.x;
    float s = 0.f;
    if (ch < g.C) {
      if (h0) s = h0[pl.b * g.C + ch];
      if (agg) s = enter_segment<false>(agg, g, pl, threadIdx.x, s);
    }
    sH[pl.k0 & 1][threadIdx.x] = s;
  }
  const T *xp = x.p + pl.b * x.sb + c, *dp = d.p + pl.b * d.sb + c, *zp = z.p ? z.p + pl.b * z.sb + c : nullptr;
  T* yp = y + pl.b * g.T * g.C + c;
  for (int64_t k = pl.k0; k < pl.k1; k++) {
    const int par = k & 1;
    const int64_t t0 = k * kChunk + lt * S;
    Quad<T> qx[S], qd[S], qz[S];
    if (n > 0) {
#pragma unroll
      for (int s = 0; s < S; s++)
        if (t0 + s < g.T) {
          const int64_t t = g.at(t0 + s);
          qx[s] = quad_load(xp + t * x.st, n);
          qd[s] = quad_load(dp + t * d.st, n);
          if (zp) qz[s] = quad_load(zp + t * z.st, n);
        }
    }
    float A[S][kVC], Bx[S][kVC], P[kVC], E[kVC];
#pragma unroll
    for (int v = 0; v < kVC; v++) P[v] = 1.f, E[v] = 0.f;
#pragma unroll
    for (int s = 0; s < S; s++) {
      const bool in = n > 0 && t0 + s < g.T;                          // past the end: the identity
#pragma unroll
      for (int v = 0; v < kVC; v++) {
        float a, i;
        sigmoid_pair((float)qd[s].v[v], a, i);
        A[s][v] = in ? a : 1.f;
        Bx[s][v] = in ? i * (float)qx[s].v[v] : 0.f;
        E[v] = A[s][v] * E[v] + Bx[s][v];
        P[v] *= A[s][v];
      }
    }
#pragma unroll
    for (int v = 0; v < kVC; v++) sP[par][lt][cl * kVC + v] = P[v], sE[par][lt][cl * kVC + v] = E[v];
    __syncthreads();
    float h[kVC];
#pragma unroll
    for (int v = 0; v < kVC; v++) h[v] = sH[par][cl * kVC + v];
    if (carry && lt == 0) {
#pragma unroll
      for (int v = 0; v < kVC; v++)
        if (v < n) carry[(pl.b * g.chunks + k) * g.C + c + v] = h[v];
    }
    for (int j = 0; j < lt; j++)
#pragma unroll
      for (int v = 0; v < kVC; v++) h[v] = sP[par][j][cl * kVC + v] * h[v] + sE[par][j][cl * kVC + v];
#pragma unroll
    for (int s = 0; s < S; s++) {
      Quad<T> o;
#pragma unroll
      for (int v = 0; v < kVC; v++) {
        h[v] = A[s][v] * h[v] + Bx[s][v];
        o.v[v] = (T)(zp ? h[v] * silu((float)qz[s].v[v]) : h[v]);
      }
      if (n > 0 && t0 + s < g.T) quad_store(yp + g.at(t0 + s) * g.C, n, o);
    }
    if (lt == LT - 1) {
#pragma unroll
      for (int v = 0; v < kVC; v++) {
        sH[par ^ 1][cl * kVC + v] = h[v];
        if (k == g.chunks - 1 && v < n) last[pl.b * g.C + c + v] = h[v];
      }
    }
  }
}

// ---- backward ---------------------------------------------------------------------------------
template <typename T, int LT>
__global__ __launch_bounds__(kLC* LT) void recur_bwd_kernel(Strided<T> x, Strided<T> d, Strided<T> z, Strided<T> dy,
                                                            const float* carry, const float* dlast, Geo g, const float* agg,
                                                            T* dx, T* dd, T* dz, float* dh0) {
  constexpr int S = kChunk / LT;
  __shared__ __attribute__((aligned(16))) float sP[2][LT][kCT], sE[2][LT][kCT], sQ[2][LT][kCT], sG[2][kCT];
  const Place pl = place(g);
  const int cl = threadIdx.x % kLC, lt = threadIdx.x / kLC, c = pl.c0 + cl * kVC, n = g.C - c;
  if (threadIdx.x < kCT) {
    const int ch = pl.c0 + threadIdx.x;
    float s = 0.f;
    if (ch < g.C) {
      if (dlast) s = dlast[pl.b * g.C + ch];
      if (agg) s = enter_segment<true>(agg, g, pl, threadIdx.x, s);
    }
    sG[(pl.k1 - 1) & 1][threadIdx.x] = s;
  }
  const T *xp = x.p + pl.b * x.sb + c, *dp = d.p + pl.b * d.sb + c, *yp = dy.p + pl.b * dy.sb + c;
  const T* zp = z.p ? z.p + pl.b * z.sb + c : nullptr;
  const int64_t ob = pl.b * g.T * g.C + c;
  for (int64_t k = pl.k1 - 1; k >= pl.k0; k--) {
    const int par = k & 1;
    const int64_t t0 = k * kChunk + lt * S;
    Quad<T> qx[S], qd[S], qz[S], qy[S];
    float hin[kVC];
#pragma unroll
    for (int v = 0; v < kVC; v++) hin[v] = 0.f;
    if (n > 0) {
#pragma unroll
      for (int s = 0; s < S; s++)
        if (t0 + s < g.T) {
          const int64_t t = g.at(t0 + s);
          qx[s] = quad_load(xp + t * x.st, n);
          qd[s] = quad_load(dp + t * d.st, n);
          qy[s] = quad_load(yp + t * dy.st, n);
          if (zp) qz[s] = quad_load(zp + t * z.st, n);
        }
#pragma unroll
      for (int v = 0; v < kVC; v++)
        if (v < n) hin[v] = carry[(pl.b * g.chunks + k) * g.C + c + v];
    }
    float A[S][kVC], P[kVC], E[kVC], Q[kVC];
#pragma unroll
    for (int v = 0; v < kVC; v++) P[v] = 1.f, E[v] = 0.f, Q[v] = 0.f;
#pragma unroll
    for (int s = 0; s < S; s++) {
      const bool in = n > 0 && t0 + s < g.T;
#pragma unroll
      for (int v = 0; v < kVC; v++) {
        float a, i;
        sigmoid_pair((float)qd[s].v[v], a, i);
        A[s][v] = in ? a : 1.f;
        E[v] = A[s][v] * E[v] + (in ? i * (float)qx[s].v[v] : 0.f);
        P[v] *= A[s][v];
      }
    }
#pragma unroll
    for (int s = S - 1; s >= 0; s--) {
      const bool in = n > 0 && t0 + s < g.T;
#pragma unroll
      for (int v = 0; v < kVC; v++) {
        float top = (float)qy[s].v[v];
        if (zp) top *= silu((float)qz[s].v[v]);
        Q[v] = A[s][v] * (Q[v] + (in ? top : 0.f));
      }
    }
#pragma unroll
    for (int v = 0; v < kVC; v++) {
      sP[par][lt][cl * kVC + v] = P[v];
      sE[par][lt][cl * kVC + v] = E[v];
      sQ[par][lt][cl * kVC + v] = Q[v];
    }
    __syncthreads();
    float q[kVC];
#pragma unroll
    for (int v = 0; v < kVC; v++) q[v] = sG[par][cl * kVC + v];
    for (int j = 0; j < lt; j++)
#pragma unroll
      for (int v = 0; v < kVC; v++) hin[v] = sP[par][j][cl * kVC + v] * hin[v] + sE[par][j][cl * kVC + v];
    for (int j = LT - 1; j > lt; j--)
#pragma unroll
      for (int v = 0; v < kVC; v++) q[v] = sP[par][j][cl * kVC + v] * q[v] + sQ[par][j][cl * kVC + v];
    float H[S][kVC];                                                   // the state before each step
#pragma unroll
    for (int s = 0; s < S; s++)
#pragma unroll
      for (int v = 0; v < kVC; v++) {
        float a, i;
        sigmoid_pair((float)qd[s].v[v], a, i);
        H[s][v] = hin[v];
        hin[v] = A[s][v] * hin[v] + i * (float)qx[s].v[v];
      }
#pragma unroll
    for (int s = S - 1; s >= 0; s--) {
      const bool in = n > 0 && t0 + s < g.T;
      Quad<T> ox, od, oz;
#pragma unroll
      for (int v = 0; v < kVC; v++) {
        float a, i, f = 1.f, df = 0.f;
        sigmoid_pair((float)qd[s].v[v], a, i);
        const float xv = (float)qx[s].v[v], yv = (float)qy[s].v[v];
        if (zp) silu_pair((float)qz[s].v[v], f, df);
        const float G = q[v] + yv * f;
        ox.v[v] = (T)(G * i);
        od.v[v] = (T)(G * (H[s][v] - xv) * a * i);
        oz.v[v] = (T)(yv * (a * H[s][v] + i * xv) * df);
        if (in) q[v] = a * G;
      }
      if (in) {
        const int64_t o = ob + g.at(t0 + s) * g.C;
        if (dx) quad_store(dx + o, n, ox);
        if (dd) quad_store(dd + o, n, od);
        if (dz) quad_store(dz + o, n, oz);
      }
    }
    if (lt == 0) {
#pragma unroll
      for (int v = 0; v < kVC; v++) {
        sG[par ^ 1][cl * kVC + v] = q[v];
        if (k == 0 && dh0 && v < n) dh0[pl.b * g.C + c + v] = q[v];
      }
    }
  }
}

// ---- short sequences --------------------------------------------------------------------------
// A thread walks kVC channels of a whole sequence (T ≤ kShort, one position of a stream above all):
// no joins, B·C/kVC threads.
template <typename T>
__global__ __launch_bounds__(128) void recur_fwd_short_kernel(Strided<T> x, Strided<T> d, Strided<T> z, const float* h0, Geo g,
                                                              T* y, float* last, float* carry) {
  const int64_t id = (int64_t)blockIdx.x * 128 + threadIdx.x, b = id / g.tiles;
  if (b >= g.B) return;
  const int c = (int)(id % g.tiles) * kVC, n = g.C - c;
  float h[kVC];
#pragma unroll
  for (int v = 0; v < kVC; v++) {
    h[v] = h0 && v < n ? h0[b * g.C + c + v] : 0.f;
    if (carry && v < n) carry[b * g.C + c + v] = h[v];
  }
  for (int64_t k = 0; k < g.T; k++) {
    const int64_t t = g.at(k);
    const Quad<T> qx = quad_load(x.p + b * x.sb + t * x.st + c, n), qd = quad_load(d.p + b * d.sb + t * d.st + c, n);
    Quad<T> qz, o;
    if (z.p) qz = quad_load(z.p + b * z.sb + t * z.st + c, n);
#pragma unroll
    for (int v = 0; v < kVC; v++) {
      float a, i;
      sigmoid_pair((float)qd.v[v], a, i);
      h[v] = a * h[v] + i * (float)qx.v[v];
      o.v[v] = (T)(z.p ? h[v] * silu((float)qz.v[v]) : h[v]);
    }
    quad_store(y + (b * g.T + t) * g.C + c, n, o);
  }
#pragma unroll
  for (int v = 0; v < kVC; v++)
    if (v < n) last[b * g.C + c + v] = h[v];
}

template <typename T>
__global__ __launch_bounds__(128) void recur_bwd_short_kernel(Strided<T> x, Strided<T> d, Strided<T> z, Strided<T> dy,
                                                              const float* carry, const float* dlast, Geo g, T* dx, T* dd,
                                                              T* dz, float* dh0) {
  const int64_t id = (int64_t)blockIdx.x * 128 + threadIdx.x, b = id / g.tiles;
  if (b >= g.B) return;
  const int c = (int)(id % g.tiles) * kVC, n = g.C - c;
  float H[kShort][kVC], h[kVC], q[kVC];
#pragma unroll
  for (int v = 0; v < kVC; v++) {
    h[v] = v < n ? carry[b * g.C + c + v] : 0.f;
    q[v] = dlast && v < n ? dlast[b * g.C + c + v] : 0.f;
  }
#pragma unroll
  for (int k = 0; k < kShort; k++)
    if (k < g.T) {
      const int64_t t = g.at(k);
      const Quad<T> qx = quad_load(x.p + b * x.sb + t * x.st + c, n), qd = quad_load(d.p + b * d.sb + t * d.st + c, n);
#pragma unroll
      for (int v = 0; v < kVC; v++) {
        float a, i;
        sigmoid_pair((float)qd.v[v], a, i);
        H[k][v] = h[v];
        h[v] = a * h[v] + i * (float)qx.v[v];
      }
    }
#pragma unroll
  for (int k = kShort - 1; k >= 0; k--)
    if (k < g.T) {
      const int64_t t = g.at(k);
      const Quad<T> qx = quad_load(x.p + b * x.sb + t * x.st + c, n), qd = quad_load(d.p + b * d.sb + t * d.st + c, n),
                    qy = quad_load(dy.p + b * dy.sb + t * dy.st + c, n);
      Quad<T> qz, ox, od, oz;
      if (z.p) qz = quad_load(z.p + b * z.sb + t * z.st + c, n);
#pragma unroll
      for (int v = 0; v < kVC; v++) {
        float a, i, f = 1.f, df = 0.f;
        sigmoid_pair((float)qd.v[v], a, i);
        const float xv = (float)qx.v[v], yv = (float)qy.v[v];
        if (z.p) silu_pair((float)qz.v[v], f, df);
        const float G = q[v] + yv * f;
        ox.v[v] = (T)(G * i);
        od.v[v] = (T)(G * (H[k][v] - xv) * a * i);
        oz.v[v] = (T)(yv * (a * H[k][v] + i * xv) * df);
        q[v] = a * G;
      }
      const int64_t o = (b * g.T + t) * g.C + c;
      if (dx) quad_store(dx + o, n, ox);
      if (dd) quad_store(dd + o, n, od);
      if (dz) quad_store(dz + o, n, oz);
    }
  if (dh0) {
#pragma unroll
    for (int v = 0; v < kVC; v++)
      if (v < n) dh0[b * g.C + c + v] = q[v];
  }
}

// Segments: none once sequences × channel tiles give each of the 256 CUs a block; else as many as
// bring the launch to about four blocks a CU, each at least four chunks long.
Geo geometry(int64_t B, int64_t T, int C, int reverse) {
  Geo g{};
  g.B = B, g.T = T, g.C = C, g.reverse = reverse;
  g.chunks = (T + kChunk - 1) / kChunk;
  g.tiles = T <= kShort ? ceil_div(C, kVC) : ceil_div(C, kCT);
  const int64_t base = B * g.tiles;
  int64_t segs = base >= 256 ? 1 : (1024 + base - 1) / base;
  if (segs > g.chunks / 4) segs = g.chunks / 4 > 0 ? g.chunks / 4 : 1;
  g.per_seg = (g.chunks + segs - 1) / segs;
  g.segs = (int)((g.chunks + g.per_seg - 1) / g.per_seg);
  return g;
}

template <typename T>
Strided<T> strided(const void* p, int64_t sb, int64_t st) {
  return {static_cast<const T*>(p), sb, st};
}

}  // namespace

int64_t recurrence_carries(int64_t T) { return T <= 0 ? 0 : (T + kChunk - 1) / kChunk; }
int64_t recurrence_blocks(int64_t B, int64_t T, int C) {
  const Geo g = geometry(B, T, C, 0);
  return T <= kShort ? (B * g.tiles + 127) / 128 : B * g.tiles * g.segs;
}

size_t recurrence_ws_bytes(int64_t B, int64_t T, int C) {
  if (B <= 0 || T <= kShort) return 0;
  const Geo g = geometry(B, T, C, 0);
  return g.segs > 1 ? (size_t)B * g.segs * 2 * C * sizeof(float) : 0;
}

int recurrence_fwd(const RecurArgs& r, const float* h0, void* y, float* last, float* carry, float* ws, hipStream_t st) {
  const Geo g = geometry(r.B, r.T, r.C, r.reverse);
  const unsigned grid = (unsigned)recurrence_blocks(r.B, r.T, r.C);
  MRAGAN_DTYPE_DISPATCH(r.dtype, T, {
    const auto x = strided<T>(r.x, r.x_sb, r.x_st), d = strided<T>(r.decay, r.d_sb, r.d_st), z = strided<T>(r.gate, r.g_sb, r.g_st);
    T* yt = static_cast<T*>(y);
    if (r.T <= kShort) {
      recur_fwd_short_kernel<T><<<grid, 128, 0, st>>>(x, d, z, h0, g, yt, last, carry);
      return check_launch("recurrence_fwd_short");
    }
    if (g.segs > 1) {
      recur_segment_kernel<T, false, 16><<<grid, kLC * 16, 0, st>>>(x, d, z, g, ws);
      if (int rc = check_launch("recurrence_segment")) return rc;
    }
    recur_fwd_kernel<T, 16><<<grid, kLC * 16, 0, st>>>(x, d, z, h0, g, g.segs > 1 ? ws : nullptr, yt, last, carry);
    return check_launch("recurrence_fwd");
  })
  return kOk;
}

int recurrence_bwd(const RecurArgs& r, const float* carry, const void* dy, int64_t dy_sb, int64_t dy_st, const float* dlast,
                   void* dx, void* dd, void* dz, float* dh0, float* ws, hipStream_t st) {
  const Geo g = geometry(r.B, r.T, r.C, r.reverse);
  const unsigned grid = (unsigned)recurrence_blocks(r.B, r.T, r.C);
  MRAGAN_DTYPE_DISPATCH(r.dtype, T, {
    const auto x = strided<T>(r.x, r.x_sb, r.x_st), d = strided<T>(r.decay, r.d_sb, r.d_st), z = strided<T>(r.gate, r.g_sb, r.g_st),
               gy = strided<T>(dy, dy_sb, dy_st);
    T *dxt = static_cast<T*>(dx), *ddt = static_cast<T*>(dd), *dzt = static_cast<T*>(dz);
    if (r.T <= kShort) {
      recur_bwd_short_kernel<T><<<grid, 128, 0, st>>>(x, d, z, gy, carry, dlast, g, dxt, ddt, dzt, dh0);
      return check_launch("recurrence_bwd_short");
    }
    if (g.segs > 1) {
      recur_segment_kernel<T, true, 16><<<grid, kLC * 16, 0, st>>>(gy, d, z, g, ws);
      if (int rc = check_launch("recurrence_segment")) return rc;
    }
    recur_bwd_kernel<T, 32><<<grid, kLC * 32, 0, st>>>(x, d, z, gy, carry, dlast, g, g.segs > 1 ? ws : nullptr, dxt, ddt, dzt, dh0);
    return check_launch("recurrence_bwd");
  })
  return kOk;
}

}  // namespace mragan
