// Gated linear recurrence along the time axis of [B][T][C] tensors, forward and backward.
//
//   a_t = σ(d_t), i_t = σ(−d_t)      h_t = a_t·h_{t−1} + i_t·x_t      y_t = h_t·silu(z_t)  (or h_t)
//   G_t = dy_t·silu(z_t) + Q_{t+1},  Q_t = a_t·G_t  (Q_T = dlast, dh0 = Q_0)
//   dx_t = G_t·i_t,  dd_t = G_t·(h_{t−1} − x_t)·a_t·i_t,  dz_t = dy_t·h_t·silu'(z_t)
//
// Both recursions are products of affine maps s ↦ P·s + E, which compose associatively, so time is
// split: a lane takes S = 8 steps of two channels in order, the time lanes of a wave join their maps
// in registers and the waves of a block through LDS (a chunk of 128 steps), and a block walks over
// the chunks with the fp32 state of its channels in registers, the next chunk's loads in
// flight.  HBM is the bound: each tensor is read or written once.  Where B and C give too few blocks to
// fill the chip, the chunks are also split into segments over blocks: a first launch reduces each segment
// to its (P, E), the second starts each segment from the fold of the ones before it (its inputs then come
// a second time, as a rule from the 256 MB cache).
// Steps behind the end of a sequence enter as d = +inf, x = 0: the identity.
// The forward leaves the fp32 state entering each chunk; the backward recomputes the states of a
// chunk from it in registers and walks the chunks backwards, so that no state is read or written.
// Measured: 16 × 2048 × 1024 bf16 with gate 69 us forward (268 MB, 3.9 TB/s) and 107 us backward (470 MB,
// 4.4 TB/s), one block of 8 waves a CU; 2 × 32768 × 128 fp32 in segments 15 + 18 us forward (67 MB read
// twice, 34 MB written) and 17 + 34 us backward.
#include "token_ops.h"

// A channel may be formed in either slot of a lane, by lanes moved back beside its own (see place), and on a
// guarded or a whole path.  Its bits have to be the same in each, so the compiler joins no product and sum by
// itself: where one rounding is meant for both, the code says fma.
#pragma clang fp contract(off)

namespace mragan {
namespace {

constexpr int kVC = 2;                    // channels a lane
constexpr int kS = 8;                     // steps of a time lane
constexpr int kLT = 16;                   // time lanes of a block
constexpr int kChunk = kLT * kS;          // 128 steps between two carried states
// A block's LC channel lanes: 32 (64 channels, 8 waves of 2 time lanes) or 16 (32 channels, 4 waves of 4)
template <int LC>
struct Shape {
  static constexpr int kCT = LC * kVC, kThreads = LC * kLT, kWaves = kThreads / 64;
};
constexpr int kShort = 16;                // sequences up to this long: a thread walks the whole sequence
constexpr int kShortVC = 4;               // of this many channels

template <typename T>
struct Strided {                // element (b, t, c) at p[b·sb + t·st + c]
  const T* p;
  int64_t sb, st;
};

// N channels of one step; those past the row's end (n channels left) read `fill` and are not written
template <int N, typename T>
__device__ __forceinline__ Words<T, N> group_load(const T* p, int n, float fill = 0.f) {
  Words<T, N> r;
  if (n >= N) {
    __builtin_memcpy(&r, p, sizeof(r));
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) r.set(i, i < n ? (float)p[i] : fill);
  }
  return r;
}
template <int N, typename T>
__device__ __forceinline__ void group_store(T* p, int n, const Words<T, N>& r) {
  if (n >= N) {
    __builtin_memcpy(p, &r, sizeof(r));
  } else {
#pragma unroll
    for (int i = 0; i < N; i++)
      if (i < n) p[i] = (T)r.get(i);
  }
}

__device__ __forceinline__ float silu(float z) { return z * __builtin_amdgcn_rcpf(1.f + __expf(-z)); }
// z·σ(z) and its derivative σ(z)·(1 + z·(1 − σ(z)))
__device__ __forceinline__ void silu_pair(float z, float& f, float& df) {
  const float s = __builtin_amdgcn_rcpf(1.f + __expf(-z));
  f = z * s;
  df = s * fma(z, 1.f - s, 1.f);
}

template <bool V>
struct Bool {
  static constexpr bool value = V;
};

struct Geo {
  int64_t B, T;
  int C, reverse;
  int lc, tiles;                // channel lanes of a block, channel tiles
  int64_t chunks, per_seg;      // chunks of a sequence, chunks of a segment
  int segs;
  __device__ __forceinline__ int64_t at(int64_t t) const { return reverse ? T - 1 - t : t; }
};

// This block's (sequence, segment, first channel) and this thread's channels and time lane.  Lanes that
// would pass the last channel are moved back to end with it and compute and write channels of their
// neighbours again, with the same values: no tile has another path for its channels (B = 4, T = 49191, 117
// bf16 channels, forward and backward: 181 us instead of 237).  Only a single channel, less than a lane's, is guarded.
struct Place {
  int64_t b, k0, k1;
  int seg, c0, wave, half, odd, lt, cl, c, n;                       // half, odd: bits of the time lane in its wave
  int last;                                                         // the last lane's first channel
  // the channel of slot `i` of the tile (slot cl + v: this lane's channel c + v)
  __device__ __forceinline__ int channel(int i) const {
    const int c = c0 + i / kVC * kVC;
    return (c < last ? c : last) + i % kVC;
  }
};
template <int LC>
__device__ __forceinline__ Place place(const Geo& g) {
  Place p;
  int64_t id = blockIdx.x;
  p.last = g.C > kVC ? g.C - kVC : 0;
  p.c0 = (int)(id % g.tiles) * Shape<LC>::kCT;
  p.c0 = p.c0 < p.last ? p.c0 : p.last;
  id /= g.tiles;
  p.seg = (int)(id % g.segs);
  p.b = id / g.segs;
  p.k0 = p.seg * g.per_seg;
  p.k1 = p.k0 + g.per_seg < g.chunks ? p.k0 + g.per_seg : g.chunks;
  p.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  p.half = (threadIdx.x >> 5) & 1;
  p.odd = (threadIdx.x >> 4) & 1;
  p.lt = threadIdx.x / LC;
  p.cl = (threadIdx.x % LC) * kVC;
  p.c = p.channel(p.cl);
  p.n = g.C - p.c;
  return p;
}

// Where this lane's steps of chunk k lie: a wave-uniform address per step (of the chunk's lowest
// position in memory, which a chunk cut off by the sequence's end may place before the tensor) plus
// one 32-bit offset of the lane: per-lane 64-bit addresses of every step and tensor would take more registers than
// there are.  Steps behind the end (and C = 1's second channel) read as `fill` and are not written.
template <typename T>
struct Steps {
  T* base;                                                           // step 0 of time lane 0 (reverse: of the last)
  unsigned off;
  int64_t step;
  __device__ __forceinline__ Steps(T* q, int64_t sb, int64_t st, const Geo& g, const Place& p, int64_t k) {
    const int64_t low = g.reverse ? g.T - (k + 1) * kChunk + kS - 1 : k * kChunk;
    base = q + (p.b * sb + low * st + p.c0);
    off = (unsigned)(g.reverse ? kLT - 1 - p.lt : p.lt) * (unsigned)(kS * st) + (unsigned)(p.c - p.c0);
    step = g.reverse ? -st : st;
  }
  __device__ __forceinline__ T* at(int s) const { return base + s * step + off; }
};
template <bool WHOLE, typename T>
__device__ __forceinline__ void load_steps(const Strided<T>& q, const Geo& g, const Place& p, int64_t k, float fill,
                                           Words<T, kVC> (&r)[kS]) {
  const Steps<const T> a(q.p, q.sb, q.st, g, p, k);
  const int64_t left = g.T - (k * kChunk + p.lt * kS);
#pragma unroll
  for (int s = 0; s < kS; s++) {
    if (WHOLE || (s < left && p.n >= kVC)) {
      __builtin_memcpy(&r[s], a.at(s), sizeof(r[s]));
    } else {
#pragma unroll
      for (int v = 0; v < kVC; v++) r[s].set(v, s < left && v < p.n ? (float)a.at(s)[v] : fill);
    }
  }
}
template <bool WHOLE, typename T>
__device__ __forceinline__ void store_step(const Steps<T>& a, const Geo& g, const Place& p, int64_t k, int s,
                                           const Words<T, kVC>& r) {
  if (WHOLE) __builtin_memcpy(a.at(s), &r, sizeof(r));
  else if (k * kChunk + p.lt * kS + s < g.T && p.n > 0) group_store<kVC>(a.at(s), p.n, r);
}
// chunks from k0 on that lie inside the sequence: the loop over them has no other path, whose merges
// would wait for the loads in flight
__device__ __forceinline__ int64_t whole_chunks_end(const Geo& g, const Place& p) {
  const int64_t e = g.C >= kVC ? g.T / kChunk : p.k0;
  return e < p.k0 ? p.k0 : e < p.k1 ? e : p.k1;
}

// of each two neighbouring rows of 16 lanes, or of the two half waves: the lower's and the upper's value
__device__ __forceinline__ void rows16(float v, float& lo, float& hi) {
  const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
  lo = __builtin_bit_cast(float, (unsigned)r[0]);
  hi = __builtin_bit_cast(float, (unsigned)r[1]);
}
__device__ __forceinline__ void halves(float v, float& lo, float& hi) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
  lo = __builtin_bit_cast(float, (unsigned)r[0]);
  hi = __builtin_bit_cast(float, (unsigned)r[1]);
}

// ---- segment maps: (P, E) of each segment, agg [B][segs][2][C] --------------------------------
// Each time lane walks one contiguous span of the segment, so the lanes join once, at its end.
// BWD: the map of Q from the segment's end to its start (E from dy, z); else that of h (E from x).
template <typename T, bool BWD, int LC>
__global__ __launch_bounds__(Shape<LC>::kThreads) void recur_segment_kernel(Strided<T> e, Strided<T> d, Strided<T> z, Geo g,
                                                                            float* agg) {
  constexpr int kCT = Shape<LC>::kCT;
  __shared__ float sP[kLT][kCT], sE[kLT][kCT];
  const Place p = place<LC>(g);
  const int64_t first = p.k0 * kChunk, end = p.k1 * kChunk < g.T ? p.k1 * kChunk : g.T;
  const int64_t span = (end - first + kLT - 1) / kLT;
  const int64_t t0 = first + p.lt * span, t1 = t0 + span < end ? t0 + span : end;
  float P[kVC], E[kVC];
#pragma unroll
  for (int v = 0; v < kVC; v++) P[v] = 1.f, E[v] = 0.f;
  if (p.n > 0) {
    const T *ep = e.p + p.b * e.sb + p.c, *dp = d.p + p.b * d.sb + p.c, *zp = z.p ? z.p + p.b * z.sb + p.c : nullptr;
    constexpr int U = 8;
    for (int64_t t = t0; t < t1; t += U) {
      Words<T, kVC> qe[U], qd[U], qz[U];
#pragma unroll
      for (int w = 0; w < U; w++) {
        int64_t k = t + w < t1 ? t + w : t1 - 1;
        if constexpr (BWD) k = t0 + t1 - 1 - k;                       // from the span's end to its start
        k = g.at(k);
        qe[w] = group_load<kVC>(ep + k * e.st, p.n);
        qd[w] = group_load<kVC>(dp + k * d.st, p.n);
        if (BWD && zp) qz[w] = group_load<kVC>(zp + k * z.st, p.n);
      }
#pragma unroll
      for (int w = 0; w < U; w++)
        if (t + w < t1) {
#pragma unroll
          for (int v = 0; v < kVC; v++) {
            float a, i;
            sigmoid_pair(qd[w].get(v), a, i);
            const float in = qe[w].get(v);
            if constexpr (BWD) E[v] = a * (zp ? fma(in, silu(qz[w].get(v)), E[v]) : E[v] + in);
            else E[v] = fma(a, E[v], i * in);
            P[v] *= a;
          }
        }
    }
  }
#pragma unroll
  for (int v = 0; v < kVC; v++) sP[p.lt][p.cl + v] = P[v], sE[p.lt][p.cl + v] = E[v];
  __syncthreads();
  const int ch = threadIdx.x;
  if (ch < kCT && p.channel(ch) < g.C) {
    float m = 1.f, s = 0.f;
#pragma unroll
    for (int j = 0; j < kLT; j++) {
      const int l = BWD ? kLT - 1 - j : j;
      s = fma(sP[l][ch], s, sE[l][ch]);
      m *= sP[l][ch];
    }
    float* out = agg + ((p.b * g.segs + p.seg) * 2) * g.C + p.channel(ch);
    out[0] = m;
    out[g.C] = s;
  }
}

// The state entering this block's segment in each lane's channels: `s0` [B][C] (or null: 0) run
// through the maps of the segments before it (BWD: behind it).  Eight threads a channel take a
// contiguous part of those maps each.
template <bool BWD, int LC>
__device__ __forceinline__ void enter(const float* s0, const float* agg, const Geo& g, const Place& p, float (&state)[kVC]) {
  constexpr int kCT = Shape<LC>::kCT, kParts = Shape<LC>::kThreads / kCT;
  __shared__ float fP[kParts][kCT], fE[kParts][kCT];
#pragma unroll
  for (int v = 0; v < kVC; v++) state[v] = s0 && v < p.n ? s0[p.b * g.C + p.c + v] : 0.f;
  if (!agg) return;
  const int ch = threadIdx.x % kCT, at = threadIdx.x / kCT;
  const int lo = BWD ? p.seg + 1 : 0, cnt = BWD ? g.segs - 1 - p.seg : p.seg;
  const int part = (cnt + kParts - 1) / kParts, j0 = at * part, j1 = j0 + part < cnt ? j0 + part : cnt;
  float m = 1.f, s = 0.f;
  if (p.channel(ch) < g.C) {
    const float* q = agg + (p.b * g.segs + lo) * 2 * (int64_t)g.C + p.channel(ch);
#pragma unroll 4
    for (int j = j0; j < j1; j++) {
      const int64_t o = 2 * (int64_t)(BWD ? cnt - 1 - j : j) * g.C;
      const float pj = q[o], ej = q[o + g.C];
      s = fma(pj, s, ej);
      m *= pj;
    }
  }
  fP[at][ch] = m;
  fE[at][ch] = s;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kParts; w++)
#pragma unroll
    for (int v = 0; v < kVC; v++) state[v] = fma(fP[w][p.cl + v], state[v], fE[w][p.cl + v]);
}

// ---- forward ----------------------------------------------------------------------------------
template <typename T, bool GATE, int LC>
__global__ __launch_bounds__(Shape<LC>::kThreads) void recur_fwd_kernel(Strided<T> x, Strided<T> d, Strided<T> z, const float* h0,
                                                                        Geo g, const float* agg, T* y, float* last,
                                                                        float* carry) {
  constexpr int kCT = Shape<LC>::kCT, kWaves = Shape<LC>::kWaves;
  // two sets: a chunk's maps are written while slower waves still read those of the chunk before
  __shared__ float sP[2][kWaves][kCT], sE[2][kWaves][kCT];
  const Place p = place<LC>(g);
  float state[kVC];                                                   // entering the chunk
  enter<false, LC>(h0, agg, g, p, state);
  struct Raw {                                                        // a chunk's operands as loaded
    Words<T, kVC> x[kS], d[kS], z[GATE ? kS : 1];
  };
  auto fetch = [&](auto whole, int64_t k, Raw& n) {
    constexpr bool W = decltype(whole)::value;
    load_steps<W>(x, g, p, k, 0.f, n.x);
    load_steps<W>(d, g, p, k, __builtin_inff(), n.d);
    if constexpr (GATE) load_steps<W>(z, g, p, k, 0.f, n.z);
  };
  const int64_t whole_end = whole_chunks_end(g, p);
  auto chunk = [&](auto whole, int64_t k, Raw& n) {
    constexpr bool W = decltype(whole)::value;
    const int par = k & 1;
    float A[kS][kVC], I[kS][kVC], F[kS][kVC], P[kVC], E[kVC];
#pragma unroll
    for (int v = 0; v < kVC; v++) P[v] = 1.f, E[v] = 0.f;
#pragma unroll
    for (int s = 0; s < kS; s++)
#pragma unroll
      for (int v = 0; v < kVC; v++) {
        sigmoid_pair(n.d[s].get(v), A[s][v], I[s][v]);
        I[s][v] *= n.x[s].get(v);
        E[v] = fma(A[s][v], E[v], I[s][v]);
        P[v] *= A[s][v];
        if constexpr (GATE) F[s][v] = n.z[s].get(v);
      }
    if (W && k + 1 < whole_end) fetch(whole, k + 1, n);
    // maps of the lower row of 16 and of the lower half: what enters the rows and the half above them
    float Pa[kVC], Ea[kVC], Pl[kVC], El[kVC];
#pragma unroll
    for (int v = 0; v < kVC; v++) {
      float Ph, Eh;
      if constexpr (LC == 16) {
        rows16(P[v], Pa[v], Ph);
        rows16(E[v], Ea[v], Eh);
        P[v] = Pa[v] * Ph;
        E[v] = fma(Ph, Ea[v], Eh);
      }
      halves(P[v], Pl[v], Ph);
      halves(E[v], El[v], Eh);
      if (threadIdx.x % 64 < LC) {
        sP[par][p.wave][p.cl + v] = Pl[v] * Ph;
        sE[par][p.wave][p.cl + v] = fma(Ph, El[v], Eh);
      }
    }
    __syncthreads();
    if (carry && threadIdx.x < LC) {
#pragma unroll
      for (int v = 0; v < kVC; v++)
        if (v < p.n) carry[(p.b * g.chunks + k) * g.C + p.c + v] = state[v];
    }
    float h[kVC];
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
#pragma unroll
      for (int v = 0; v < kVC; v++) {
        if (w == p.wave) h[v] = state[v];
        state[v] = fma(sP[par][w][p.cl + v], state[v], sE[par][w][p.cl + v]);
      }
    }
#pragma unroll
    for (int v = 0; v < kVC; v++) {
      h[v] = p.half ? fma(Pl[v], h[v], El[v]) : h[v];
      if constexpr (LC == 16) h[v] = p.odd ? fma(Pa[v], h[v], Ea[v]) : h[v];
    }
    const Steps<T> at(y, g.T * g.C, g.C, g, p, k);
#pragma unroll
    for (int s = 0; s < kS; s++) {
      Words<T, kVC> o;
#pragma unroll
      for (int v = 0; v < kVC; v++) {
        h[v] = fma(A[s][v], h[v], I[s][v]);
        o.set(v, GATE ? h[v] * silu(F[s][v]) : h[v]);
      }
      store_step<W>(at, g, p, k, s, o);
    }
  };
  Raw n;
  if (p.k0 < whole_end) fetch(Bool<true>{}, p.k0, n);
  for (int64_t k = p.k0; k < whole_end; k++) chunk(Bool<true>{}, k, n);
  for (int64_t k = whole_end; k < p.k1; k++) {
    fetch(Bool<false>{}, k, n);
    chunk(Bool<false>{}, k, n);
  }
  if (p.k1 == g.chunks && threadIdx.x < LC) {
#pragma unroll
    for (int v = 0; v < kVC; v++)
      if (v < p.n) last[p.b * g.C + p.c + v] = state[v];
  }
}

// ---- backward ---------------------------------------------------------------------------------
template <typename T, bool GATE, int LC>
__global__ __launch_bounds__(Shape<LC>::kThreads) void recur_bwd_kernel(Strided<T> x, Strided<T> d, Strided<T> z, Strided<T> dy,
                                                                        const float* carry, const float* dlast, Geo g,
                                                                        const float* agg, T* dx, T* dd, T* dz, float* dh0) {
  constexpr int kCT = Shape<LC>::kCT, kWaves = Shape<LC>::kWaves;
  // a and i of a step stay in registers where those suffice, else are computed again from d
  constexpr bool kHold = sizeof(T) == 2;
  __shared__ float sP[2][kWaves][kCT], sE[2][kWaves][kCT], sQ[2][kWaves][kCT];
  const Place p = place<LC>(g);
  float state[kVC];                                                   // Q entering the chunk from its end
  enter<true, LC>(dlast, agg, g, p, state);
  struct Raw {
    Words<T, kVC> x[kS], d[kS], y[kS], z[GATE ? kS : 1];
    float h[kVC];
  };
  auto fetch = [&](auto whole, int64_t k, Raw& n) {
    constexpr bool W = decltype(whole)::value;
    load_steps<W>(x, g, p, k, 0.f, n.x);
    load_steps<W>(d, g, p, k, __builtin_inff(), n.d);
    load_steps<W>(dy, g, p, k, 0.f, n.y);
    if constexpr (GATE) load_steps<W>(z, g, p, k, 0.f, n.z);
#pragma unroll
    for (int v = 0; v < kVC; v++) n.h[v] = W || v < p.n ? carry[(p.b * g.chunks + k) * g.C + p.c + v] : 0.f;
  };
  const int64_t whole_end = whole_chunks_end(g, p);
  auto chunk = [&](auto whole, int64_t k, Raw& n) {
    constexpr bool W = decltype(whole)::value;
    const int par = k & 1;
    Words<T, kVC> cx[kS], cd[kHold ? 1 : kS];
    float A[kHold ? kS : 1][kVC], I[kHold ? kS : 1][kVC], top[kS][kVC], yf[kS][kVC], P[kVC], E[kVC], Q[kVC], h[kVC];
    auto pair = [&](int s, int v, float& a, float& i) {
      if constexpr (kHold) a = A[s][v], i = I[s][v];
      else {
        float t = cd[s].get(v);
        asm volatile("" : "+v"(t));                                    // else the first pair is kept after all
        sigmoid_pair(t, a, i);
      }
    };
#pragma unroll
    for (int v = 0; v < kVC; v++) P[v] = 1.f, E[v] = Q[v] = 0.f, h[v] = n.h[v];
#pragma unroll
    for (int s = 0; s < kS; s++) {
      cx[s] = n.x[s];
      if constexpr (!kHold) cd[s] = n.d[s];
#pragma unroll
      for (int v = 0; v < kVC; v++) {
        float a, i;
        sigmoid_pair(n.d[s].get(v), a, i);
        if constexpr (kHold) A[s][v] = a, I[s][v] = i;
        E[v] = fma(a, E[v], i * n.x[s].get(v));
        P[v] *= a;
        const float g_out = n.y[s].get(v);
        if constexpr (GATE) {
          float f, df;
          silu_pair(n.z[s].get(v), f, df);
          top[s][v] = g_out * f;
          yf[s][v] = g_out * df;
        } else {
          top[s][v] = g_out;
        }
      }
    }
    if (W && k > p.k0) fetch(whole, k - 1, n);
#pragma unroll
    for (int s = kS - 1; s >= 0; s--)
#pragma unroll
      for (int v = 0; v < kVC; v++) {
        float a, i;
        pair(s, v, a, i);
        Q[v] = a * (Q[v] + top[s][v]);
      }
    float Pa[kVC], Ea[kVC], Pb[kVC], Qb[kVC], Pl[kVC], El[kVC], Ph[kVC], Qh[kVC];
#pragma unroll
    for (int v = 0; v < kVC; v++) {
      float Eh, Ql;
      if constexpr (LC == 16) {
        rows16(P[v], Pa[v], Pb[v]);
        rows16(E[v], Ea[v], Eh);
        rows16(Q[v], Ql, Qb[v]);
        P[v] = Pa[v] * Pb[v];
        E[v] = fma(Pb[v], Ea[v], Eh);
        Q[v] = fma(Pa[v], Qb[v], Ql);
      }
      halves(P[v], Pl[v], Ph[v]);
      halves(E[v], El[v], Eh);
      halves(Q[v], Ql, Qh[v]);
      if (threadIdx.x % 64 < LC) {
        sP[par][p.wave][p.cl + v] = Pl[v] * Ph[v];
        sE[par][p.wave][p.cl + v] = fma(Ph[v], El[v], Eh);
        sQ[par][p.wave][p.cl + v] = fma(Pl[v], Qh[v], Ql);
      }
    }
    __syncthreads();
    float q[kVC];
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
#pragma unroll
      for (int v = 0; v < kVC; v++) {
        if (w < p.wave) h[v] = fma(sP[par][w][p.cl + v], h[v], sE[par][w][p.cl + v]);
        const int r = kWaves - 1 - w;
        if (r == p.wave) q[v] = state[v];
        state[v] = fma(sP[par][r][p.cl + v], state[v], sQ[par][r][p.cl + v]);
      }
    }
#pragma unroll
    for (int v = 0; v < kVC; v++) {
      h[v] = p.half ? fma(Pl[v], h[v], El[v]) : h[v];
      q[v] = p.half ? q[v] : fma(Ph[v], q[v], Qh[v]);
      if constexpr (LC == 16) {
        h[v] = p.odd ? fma(Pa[v], h[v], Ea[v]) : h[v];
        q[v] = p.odd ? q[v] : fma(Pb[v], q[v], Qb[v]);
      }
    }
    float H[kS][kVC];                                                  // the state before each step
#pragma unroll
    for (int s = 0; s < kS; s++)
#pragma unroll
      for (int v = 0; v < kVC; v++) {
        float a, i;
        pair(s, v, a, i);
        H[s][v] = h[v];
        h[v] = fma(a, h[v], i * cx[s].get(v));
      }
    const int64_t sb = g.T * g.C;
    const Steps<T> ax(dx, sb, g.C, g, p, k), ad(dd, sb, g.C, g, p, k), az(dz, sb, g.C, g, p, k);
#pragma unroll
    for (int s = kS - 1; s >= 0; s--) {
      Words<T, kVC> ox, od, oz;
#pragma unroll
      for (int v = 0; v < kVC; v++) {
        float a, i;
        pair(s, v, a, i);
        const float xv = cx[s].get(v), G = q[v] + top[s][v], Gi = G * i;
        ox.set(v, Gi);
        od.set(v, Gi * (H[s][v] - xv) * a);
        if constexpr (GATE) oz.set(v, yf[s][v] * fma(a, H[s][v], i * xv));
        q[v] = a * G;
      }
      if (dx) store_step<W>(ax, g, p, k, s, ox);
      if (dd) store_step<W>(ad, g, p, k, s, od);
      if constexpr (GATE)
        if (dz) store_step<W>(az, g, p, k, s, oz);
    }
  };
  Raw n;
  for (int64_t k = p.k1 - 1; k >= whole_end; k--) {
    fetch(Bool<false>{}, k, n);
    chunk(Bool<false>{}, k, n);
  }
  if (p.k0 < whole_end) fetch(Bool<true>{}, whole_end - 1, n);
  for (int64_t k = whole_end - 1; k >= p.k0; k--) chunk(Bool<true>{}, k, n);
  if (p.k0 == 0 && dh0 && threadIdx.x < LC) {
#pragma unroll
    for (int v = 0; v < kVC; v++)
      if (v < p.n) dh0[p.b * g.C + p.c + v] = state[v];
  }
}

// ---- short sequences --------------------------------------------------------------------------
// A thread walks kShortVC channels of a whole sequence (T ≤ MAXT, kShort or a single position of a stream):
// no joins, B·C/kShortVC threads.  Latency is the bound, so the loads of U steps are issued together,
// those past the sequence's end at its last step.
template <typename T, int MAXT>
__global__ __launch_bounds__(128) void recur_fwd_short_kernel(Strided<T> x, Strided<T> d, Strided<T> z, const float* h0, Geo g,
                                                              T* y, float* last, float* carry) {
  using Q = Words<T, kShortVC>;
  constexpr int U = MAXT < 4 ? MAXT : 4;
  const int64_t id = (int64_t)blockIdx.x * 128 + threadIdx.x, b = id / g.tiles;
  if (b >= g.B) return;
  const int c = (int)(id % g.tiles) * kShortVC, n = g.C - c;
  float h[kShortVC];
#pragma unroll
  for (int v = 0; v < kShortVC; v++) {
    h[v] = h0 && v < n ? h0[b * g.C + c + v] : 0.f;
    if (carry && v < n) carry[b * g.C + c + v] = h[v];
  }
  auto walk = [&](auto whole, auto gated) {
    const int m = decltype(whole)::value ? kShortVC : n;
    for (int64_t k0 = 0; k0 < g.T; k0 += U) {
      Q qx[U], qd[U], qz[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int64_t t = g.at(k0 + u < g.T ? k0 + u : g.T - 1);
        qx[u] = group_load<kShortVC>(x.p + b * x.sb + t * x.st + c, m);
        qd[u] = group_load<kShortVC>(d.p + b * d.sb + t * d.st + c, m);
        if (decltype(gated)::value) qz[u] = group_load<kShortVC>(z.p + b * z.sb + t * z.st + c, m);
      }
#pragma unroll
      for (int u = 0; u < U; u++)
        if (k0 + u < g.T) {
          Q o;
#pragma unroll
          for (int v = 0; v < kShortVC; v++) {
            float a, i;
            sigmoid_pair(qd[u].get(v), a, i);
            h[v] = fma(a, h[v], i * qx[u].get(v));
            o.set(v, decltype(gated)::value ? h[v] * silu(qz[u].get(v)) : h[v]);
          }
          group_store<kShortVC>(y + (b * g.T + g.at(k0 + u)) * g.C + c, m, o);
        }
    }
  };
  auto gate = [&](auto whole) {
    if (z.p) walk(whole, Bool<true>{});
    else walk(whole, Bool<false>{});
  };
  if (n >= kShortVC) gate(Bool<true>{});
  else gate(Bool<false>{});
#pragma unroll
  for (int v = 0; v < kShortVC; v++)
    if (v < n) last[b * g.C + c + v] = h[v];
}

template <typename T, int MAXT>
__global__ __launch_bounds__(128) void recur_bwd_short_kernel(Strided<T> x, Strided<T> d, Strided<T> z, Strided<T> dy,
                                                              const float* carry, const float* dlast, Geo g, T* dx, T* dd,
                                                              T* dz, float* dh0) {
  using Q = Words<T, kShortVC>;
  constexpr int U = MAXT < 4 ? MAXT : 4;
  const int64_t id = (int64_t)blockIdx.x * 128 + threadIdx.x, b = id / g.tiles;
  if (b >= g.B) return;
  const int c = (int)(id % g.tiles) * kShortVC, n = g.C - c;
  float H[MAXT][kShortVC], h[kShortVC], q[kShortVC];
#pragma unroll
  for (int v = 0; v < kShortVC; v++) {
    h[v] = v < n ? carry[b * g.C + c + v] : 0.f;
    q[v] = dlast && v < n ? dlast[b * g.C + c + v] : 0.f;
  }
  auto walk = [&](auto whole, auto gated) {
    const int m = decltype(whole)::value ? kShortVC : n;
#pragma unroll
    for (int k0 = 0; k0 < MAXT; k0 += U)
      if (k0 < g.T) {
        Q qx[U], qd[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
          const int64_t t = g.at(k0 + u < g.T ? k0 + u : g.T - 1);
          qx[u] = group_load<kShortVC>(x.p + b * x.sb + t * x.st + c, m);
          qd[u] = group_load<kShortVC>(d.p + b * d.sb + t * d.st + c, m);
        }
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
          for (int v = 0; v < kShortVC; v++) {                       // states behind the end are not used
            float a, i;
            sigmoid_pair(qd[u].get(v), a, i);
            H[k0 + u][v] = h[v];
            h[v] = fma(a, h[v], i * qx[u].get(v));
          }
      }
#pragma unroll
    for (int k0 = MAXT - U; k0 >= 0; k0 -= U)
      if (k0 < g.T) {
        Q qx[U], qd[U], qz[U], qy[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
          const int64_t t = g.at(k0 + u < g.T ? k0 + u : g.T - 1);
          qx[u] = group_load<kShortVC>(x.p + b * x.sb + t * x.st + c, m);
          qd[u] = group_load<kShortVC>(d.p + b * d.sb + t * d.st + c, m);
          qy[u] = group_load<kShortVC>(dy.p + b * dy.sb + t * dy.st + c, m);
          if (decltype(gated)::value) qz[u] = group_load<kShortVC>(z.p + b * z.sb + t * z.st + c, m);
        }
#pragma unroll
        for (int u = U - 1; u >= 0; u--)
          if (k0 + u < g.T) {
            Q ox, od, oz;
#pragma unroll
            for (int v = 0; v < kShortVC; v++) {
              float a, i, f = 1.f, df = 0.f;
              sigmoid_pair(qd[u].get(v), a, i);
              const float xv = qx[u].get(v), yv = qy[u].get(v), hv = H[k0 + u][v];
              if (decltype(gated)::value) silu_pair(qz[u].get(v), f, df);
              const float G = fma(yv, f, q[v]);
              ox.set(v, G * i);
              od.set(v, G * (hv - xv) * a * i);
              if (decltype(gated)::value) oz.set(v, yv * fma(a, hv, i * xv) * df);
              q[v] = a * G;
            }
            const int64_t o = (b * g.T + g.at(k0 + u)) * g.C + c;
            if (dx) group_store<kShortVC>(dx + o, m, ox);
            if (dd) group_store<kShortVC>(dd + o, m, od);
            if (decltype(gated)::value && dz) group_store<kShortVC>(dz + o, m, oz);
          }
      }
  };
  auto gate = [&](auto whole) {
    if (z.p) walk(whole, Bool<true>{});
    else walk(whole, Bool<false>{});
  };
  if (n >= kShortVC) gate(Bool<true>{});
  else gate(Bool<false>{});
  if (dh0) {
#pragma unroll
    for (int v = 0; v < kShortVC; v++)
      if (v < n) dh0[b * g.C + c + v] = q[v];
  }
}

// Tiles of 64 channels, of 32 where C has no more (fp32, 16384 steps of 32 channels,
// 16 sequences with gate: 35 us forward and 59 backward against 51 and 96 with half the lanes idle).
// Segments: none once sequences × channel tiles give each of the 256 CUs a block; else as many as
// bring the launch up to two blocks a CU (B = 3, T = 9705, 680 fp16 channels, forward and backward: 201 us, 229
// with 16 blocks more), each at least four chunks long.
Geo geometry(int64_t B, int64_t T, int C, int reverse) {
  Geo g{};
  g.B = B, g.T = T, g.C = C, g.reverse = reverse;
  g.chunks = (T + kChunk - 1) / kChunk;
  g.lc = C <= 32 ? 16 : 32;
  g.tiles = T <= kShort ? ceil_div(C, kShortVC) : ceil_div(C, g.lc * kVC);
  const int64_t base = B * g.tiles;
  int64_t segs = base >= 256 ? 1 : 512 / base;
  if (segs > g.chunks / 4) segs = g.chunks / 4 > 0 ? g.chunks / 4 : 1;
  g.per_seg = (g.chunks + segs - 1) / segs;
  g.segs = (int)((g.chunks + g.per_seg - 1) / g.per_seg);
  return g;
}

int64_t blocks_of(const Geo& g) { return g.T <= kShort ? (g.B * g.tiles + 127) / 128 : g.B * g.tiles * g.segs; }

// run the statement block with the channel lanes as LC
#define MRAGAN_RECUR_LC(lc, ...) \
  if (lc == 32) {                \
    constexpr int LC = 32;       \
    __VA_ARGS__;                 \
  } else {                       \
    constexpr int LC = 16;       \
    __VA_ARGS__;                 \
  }

template <typename T>
Strided<T> strided(const void* p, int64_t sb, int64_t st) {
  return {static_cast<const T*>(p), sb, st};
}

}  // namespace

int64_t recurrence_carries(int64_t T) { return T <= 0 ? 0 : (T + kChunk - 1) / kChunk; }
int64_t recurrence_threads(int64_t B, int64_t T, int C) {
  const Geo g = geometry(B, T, C, 0);
  return blocks_of(g) * (T <= kShort ? 128 : g.lc * kLT);
}

size_t recurrence_ws_bytes(int64_t B, int64_t T, int C) {
  if (B <= 0 || T <= kShort) return 0;
  const Geo g = geometry(B, T, C, 0);
  return g.segs > 1 ? (size_t)B * g.segs * 2 * C * sizeof(float) : 0;
}

int recurrence_fwd(const RecurArgs& r, const float* h0, void* y, float* last, float* carry, float* ws, hipStream_t st) {
  const Geo g = geometry(r.B, r.T, r.C, r.reverse);
  const unsigned grid = (unsigned)blocks_of(g);
  MRAGAN_DTYPE_DISPATCH(r.dtype, T, {
    const auto x = strided<T>(r.x, r.x_sb, r.x_st), d = strided<T>(r.decay, r.d_sb, r.d_st), z = strided<T>(r.gate, r.g_sb, r.g_st);
    T* yt = static_cast<T*>(y);
    if (r.T <= kShort) {
      if (r.T == 1) recur_fwd_short_kernel<T, 1><<<grid, 128, 0, st>>>(x, d, z, h0, g, yt, last, carry);
      else recur_fwd_short_kernel<T, kShort><<<grid, 128, 0, st>>>(x, d, z, h0, g, yt, last, carry);
      return check_launch("recurrence_fwd_short");
    }
    const float* agg = g.segs > 1 ? ws : nullptr;
    MRAGAN_RECUR_LC(g.lc, {
      constexpr int N = Shape<LC>::kThreads;
      if (agg) {
        recur_segment_kernel<T, false, LC><<<grid, N, 0, st>>>(x, d, z, g, ws);
        if (int rc = check_launch("recurrence_segment")) return rc;
      }
      if (r.gate) recur_fwd_kernel<T, true, LC><<<grid, N, 0, st>>>(x, d, z, h0, g, agg, yt, last, carry);
      else recur_fwd_kernel<T, false, LC><<<grid, N, 0, st>>>(x, d, z, h0, g, agg, yt, last, carry);
    })
    return check_launch("recurrence_fwd");
  })
  return kOk;
}

int recurrence_bwd(const RecurArgs& r, const float* carry, const void* dy, int64_t dy_sb, int64_t dy_st, const float* dlast,
                   void* dx, void* dd, void* dz, float* dh0, float* ws, hipStream_t st) {
  const Geo g = geometry(r.B, r.T, r.C, r.reverse);
  const unsigned grid = (unsigned)blocks_of(g);
  MRAGAN_DTYPE_DISPATCH(r.dtype, T, {
    const auto x = strided<T>(r.x, r.x_sb, r.x_st), d = strided<T>(r.decay, r.d_sb, r.d_st), z = strided<T>(r.gate, r.g_sb, r.g_st),
               gy = strided<T>(dy, dy_sb, dy_st);
    T *dxt = static_cast<T*>(dx), *ddt = static_cast<T*>(dd), *dzt = static_cast<T*>(dz);
    if (r.T <= kShort) {
      if (r.T == 1) recur_bwd_short_kernel<T, 1><<<grid, 128, 0, st>>>(x, d, z, gy, carry, dlast, g, dxt, ddt, dzt, dh0);
      else recur_bwd_short_kernel<T, kShort><<<grid, 128, 0, st>>>(x, d, z, gy, carry, dlast, g, dxt, ddt, dzt, dh0);
      return check_launch("recurrence_bwd_short");
    }
    const float* agg = g.segs > 1 ? ws : nullptr;
    MRAGAN_RECUR_LC(g.lc, {
      constexpr int N = Shape<LC>::kThreads;
      if (agg) {
        recur_segment_kernel<T, true, LC><<<grid, N, 0, st>>>(gy, d, z, g, ws);
        if (int rc = check_launch("recurrence_segment")) return rc;
      }
      if (r.gate) recur_bwd_kernel<T, true, LC><<<grid, N, 0, st>>>(x, d, z, gy, carry, dlast, g, agg, dxt, ddt, dzt, dh0);
      else recur_bwd_kernel<T, false, LC><<<grid, N, 0, st>>>(x, d, z, gy, carry, dlast, g, agg, dxt, ddt, dzt, dh0);
    })
    return check_launch("recurrence_bwd");
  })
  return kOk;
}

}  // namespace mragan
