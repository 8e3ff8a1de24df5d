// Gated feed-forward block, forward and backward, on MFMA.
//
//   g = x·Wgᵀ + bg, u = x·Wuᵀ + bu, h = act(g)·u, y = h·Wdᵀ + bd
//   dh = dy·Wd, dg = dh·u·act'(g), du = dh·act(g), dx = dg·Wg + du·Wu,
//   dWg = dgᵀ·x, dWu = duᵀ·x, dWd = dyᵀ·h, db = column sums
//
// Every product runs through one kernel, D[m][n] = Σ_s Σ_k A_s(m, k)·B_s(n, k) over a list of
// operand pairs s of 16-bit words.  An operand lies in memory as the tensor does: with k contiguous
// (x, the weights of the forward, dy, dg, du as left operands), or with its rows contiguous and k
// the slow axis (the weights of the data gradients, both operands of the weight gradients); the
// latter are transposed on their way from LDS into registers, so that no transposed copy exists.
// That one kernel covers
//   * fp32 tensors: an operand is split into bf16 planes x = x0 + x1 + x2 and the product is the list
//     of plane pairs (six pairs with three planes, three with two, one in the one-plane modes);
//   * dx: the two weights' products are two pairs of one list;
//   * both projections of the forward: a block's B tile is half gate rows, half up rows, so that a
//     lane ends with g and u of the same (m, n) and act(g)·u never leaves the registers.
// The forward keeps h, act'(g)·u and act(g) for the backward, whose epilogue is then two products
// with dh; h is the operand of dWd as it stands.
// Roundings of 16-bit tensors: h, dg and du are operands of the next products and are rounded to the type for
// them.  A second plane of each would double those products (2.5 of the 4.4 ms below); without one the outputs are
// off by 0.0023 of their size in bf16, results rounded only once by 0.0017.
// The matrix units are the bound.  Measured on 16384 rows, 2048 → 8192 → 2048, bf16 (a library product of
// these sides: 1.3 … 1.6 PFLOP/s): gate and up 1078 us (1.02 PFLOP/s; the epilogue writes 1.07 GB of
// kept tensors, which one block a CU does not overlap), down 425 us (1.29), dg and du 787 us (0.70; its epilogue
// reads 805 MB and writes 537), dx 851 us (1.29), dWg and dWu 820 us (1.34), dWd 400 us (1.37).
#pragma once
#include <type_traits>

#include "prec.h"
#include "token_ops.h"

namespace mragan {
namespace {

using prec::bf16x8;                       // eight 16-bit words; fp16 planes travel in it too
using prec::f16x8;
using prec::f32x4;
constexpr int kBK = 64;                   // k elements of a stage: 128-byte rows of 8 16-byte chunks
constexpr int kMaxPairs = 12;
enum Epi : int { kEpiStore = 0, kEpiGate = 1, kEpiGateBwd = 2 };

inline int64_t round_k(int64_t k) { return (k + kBK - 1) / kBK * kBK; }

// ---- activations ------------------------------------------------------------------------------
enum GateAct : int { kActSilu = 5, kActGelu = 6 };

__device__ __forceinline__ void gate_act_pair(float g, int act, float& f, float& df) {
  float s, n;
  switch (act) {
    case kActSilu: sigmoid_pair(g, s, n); f = g * s; df = s * (1.f + g * n); return;
    case kActGelu: {
      const float c = 0.5f * (1.f + erff(g * 0.70710678118654752f));
      f = g * c;
      df = c + g * 0.39894228040143268f * __expf(-0.5f * g * g);
      return;
    }
    case kActSigmoid: sigmoid_pair(g, s, n); f = s; df = s * n; return;
    case kActRelu: f = g > 0.f ? g : 0.f; df = g > 0.f ? 1.f : 0.f; return;
    case kActLrelu: f = g > 0.f ? g : g * kLreluSlope; df = g > 0.f ? 1.f : kLreluSlope; return;
    case kActTanh: f = tanhf(g); df = 1.f - f * f; return;
    default: f = g; df = 1.f; return;
  }
}

// ---- planes -----------------------------------------------------------------------------------
// v as the sum of up to three 16-bit words, each the rounding (RNE) of what the ones before leave;
// an infinite or NaN word ends the sum
template <typename H>
__device__ __forceinline__ void split_planes(float v, int planes, H (&out)[3]) {
  out[0] = (H)v;
  float r = v - (float)out[0];
  if (!(fabsf((float)out[0]) < __builtin_inff())) r = 0.f;
  out[1] = (H)r;
  out[2] = planes > 2 ? (H)(r - (float)out[1]) : (H)0.f;
}

// src [R][K] (any type) → 16-bit planes dst [planes][R][ld], zeros from K to ld; several tensors a launch,
// kPackQuads groups of four elements a block and pass.  At most kPackBlocks blocks: a launch of 2^32 threads and
// more would leave some out without a word.
constexpr int kPackQuads = 1024, kMaxPacks = 8, kPackBlocks = 65536;
struct PackJob {
  const void* src;
  void* dst;
  int64_t R, K, ld;
  int64_t first;                  // its first block
};
struct PackArgs {
  PackJob job[kMaxPacks];
  int jobs, planes;
  int64_t blocks;                 // of all jobs
};
template <typename T, typename H>
__global__ __launch_bounds__(256) void ffn_pack_kernel(const PackArgs a) {
  for (int64_t block = blockIdx.x; block < a.blocks; block += gridDim.x) {
    int j = 0;
    while (j + 1 < a.jobs && block >= a.job[j + 1].first) j++;
    const PackJob& q = a.job[j];
    const T* src = static_cast<const T*>(q.src);
    const int64_t quads = q.ld / 4, total = q.R * quads, plane = q.R * q.ld, i0 = (block - q.first) * kPackQuads;
#pragma unroll
    for (int n = 0; n < kPackQuads / 256; n++) {
      const int64_t i = i0 + n * 256 + threadIdx.x;
      if (i >= total) break;
      const int64_t r = total >> 32 ? i / quads : (uint32_t)i / (uint32_t)quads, k = (i - r * quads) * 4;
      float v[4];
      if (k + 4 <= q.K) {                                              // of any alignment where K is odd
        T t[4];
        __builtin_memcpy(t, src + r * q.K + k, sizeof(t));
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = (float)t[e];
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = k + e < q.K ? (float)src[r * q.K + k + e] : 0.f;
      }
      H w[4][3];
#pragma unroll
      for (int e = 0; e < 4; e++) split_planes<H>(v[e], a.planes, w[e]);
#pragma unroll
      for (int p = 0; p < 3; p++)
        if (p < a.planes) {
          Pack<H, 4> o;
#pragma unroll
          for (int e = 0; e < 4; e++) o.v[e] = w[e][p];
          *reinterpret_cast<Pack<H, 4>*>(static_cast<H*>(q.dst) + p * plane + r * q.ld + k) = o;
        }
    }
  }
}

// Σ over chunk blockIdx.y of the rows of src [rows][cols] → part [chunks][cols]: a thread per column and
// every fourth row of the chunk
template <typename T>
__global__ __launch_bounds__(256) void ffn_col_sum_kernel(const T* src, int64_t rows, int cols, int64_t per_chunk, float* part) {
  __shared__ float s[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
  const int64_t r0 = blockIdx.y * per_chunk, r1 = r0 + per_chunk < rows ? r0 + per_chunk : rows;
  float v = 0.f;
  if (c < cols) {
#pragma unroll 8
    for (int64_t r = r0 + wave; r < r1; r += 4) v += (float)src[r * cols + c];
  }
  s[wave][lane] = v;
  __syncthreads();
  if (wave == 0 && c < cols) part[(int64_t)blockIdx.y * cols + c] = s[0][lane] + s[1][lane] + s[2][lane] + s[3][lane];
}

// out[i] = Σ_s part[s][i] (+ bias[i mod N]), and of a second set of parts → out2: 64 elements a block, SLOTS threads each that take every
// SLOTS-th part and join in order
template <typename TO, int SLOTS>
__global__ __launch_bounds__(64 * SLOTS) void ffn_reduce_kernel(const float* part, int parts, int64_t total, int N, const TO* bias,
                                                                TO* out, TO* out2) {
  if (blockIdx.y) part += parts * total, out = out2;
  __shared__ float s[SLOTS][64];
  const int lane = threadIdx.x & 63, slot = threadIdx.x >> 6;
  const int64_t i = (int64_t)blockIdx.x * 64 + lane;
  float v = 0.f;
  if (i < total) {
#pragma unroll 8
    for (int p = slot; p < parts; p += SLOTS) v += part[p * total + i];
  }
  s[slot][lane] = v;
  __syncthreads();
  if (slot == 0 && i < total) {
    v = 0.f;
#pragma unroll
    for (int k = 0; k < SLOTS; k++) v += s[k][lane];
    if (bias) v += (float)bias[i % N];
    out[i] = (TO)v;
  }
}

// the same for few parts of many elements: four elements a thread (total and N multiples of 4)
template <typename TO>
__global__ __launch_bounds__(256) void ffn_reduce4_kernel(const float* part, int parts, int64_t total, int N, const TO* bias,
                                                          TO* out, TO* out2) {
  if (blockIdx.y) part += parts * total, out = out2;
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= total) return;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int p = 0; p < parts; p++) {
    float t[4];
    load_vec<float, 4>(part + p * total + i, t);
#pragma unroll
    for (int q = 0; q < 4; q++) v[q] += t[q];
  }
  if (bias) {
    const int n = (int)(i % N);
#pragma unroll
    for (int q = 0; q < 4; q++) v[q] += (float)bias[n + q];
  }
  store_vec<TO, 4>(out + i, v);
}

// db of both projections from the column sums [rows][2][F] of the dg / du launch
template <typename TO>
__global__ __launch_bounds__(1024) void ffn_bias_reduce_kernel(const float* part, int rows, int F, TO* dbg, TO* dbu) {
  __shared__ float s[16][64];
  const int lane = threadIdx.x & 63, slot = threadIdx.x >> 6;
  const int64_t i = (int64_t)blockIdx.x * 64 + lane, total = 2 * (int64_t)F;
  float v = 0.f;
  if (i < total) {
#pragma unroll 8
    for (int p = slot; p < rows; p += 16) v += part[p * total + i];
  }
  s[slot][lane] = v;
  __syncthreads();
  if (slot == 0 && i < total) {
    v = 0.f;
#pragma unroll
    for (int k = 0; k < 16; k++) v += s[k][lane];
    if (i < F) {
      if (dbg) dbg[i] = (TO)v;
    } else if (dbu) {
      dbu[i - F] = (TO)v;
    }
  }
}

// ---- the product ------------------------------------------------------------------------------
struct GemmArgs {
  const void* A[kMaxPairs];       // k contiguous: [M][lda]; rows contiguous: [K][lda]
  const void* A2[kMaxPairs];      // of a second product with the same B (batches = 2), to out2
  const void* B[kMaxPairs];       // [N][ldb] or [K][ldb]; kEpiGate: the gate weight
  const void* B2[kMaxPairs];      // kEpiGate: the up weight
  int pairs, ktiles, batches;     // operand pairs (NP > 1: of first planes), stages of kBK of one pair
  int64_t lda, ldb, K;            // elements
  int64_t plane_a, plane_b;       // bytes from an operand's plane to its next
  int M, N;
  int tiles_m, tiles_n, splits, per_split;   // stages of all pairs cut into `splits` runs of per_split
  // kEpiStore: out[m][n] (+ bias[n]); splits > 1: fp32 partials [batch][split][M][N]
  void *out, *out2;
  const void* bias;
  float* partial;
  // kEpiGate / kEpiGateBwd: 16-bit planes of [M][ldf]
  const void *bias_g, *bias_u;
  int act, planes;
  void* kept;                     // [M][N] layers (see store_kept): written by kEpiGate if given, read by kEpiGateBwd
  float* col_part;                // kEpiGateBwd, or null: [tiles_m·WM][2][N] column sums of dg and du
  void *h, *dg, *du;
  int64_t ldf;
};

// A wave's 64 × 16 bytes from a buffer straight into LDS at `lds` + 16·lane.  As assembly, with the
// waits below: after the builtin the compiler waits for every such load before any transposed LDS
// read, whichever stage it reads, and the loads of the next stages would never be in flight.  The
// nops cover the wait states of a descriptor register that a vector instruction wrote (5) and of m0.
typedef int i32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void load_to_lds(i32x4 rsrc, unsigned lds, unsigned voffset) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(voffset), "s"(rsrc)
               : "memory", "m0");
}
// all but the N newest of this wave's loads have landed, its LDS reads are done, and so for every wave
template <int N>
__device__ __forceinline__ void wait_and_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(N) : "memory");
}
__device__ __forceinline__ i32x4 descriptor(const void* p, uint32_t bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(p);
  return i32x4{(int)__builtin_amdgcn_readfirstlane((uint32_t)a), (int)__builtin_amdgcn_readfirstlane((uint32_t)(a >> 32) & 0xffffu),
               (int)__builtin_amdgcn_readfirstlane(bytes), 0x00020000};
}
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
// 16 lanes give the addresses of a 4 (k) × 16 block, lane l the quad of columns l & 3 in row l >> 2;
// lane l receives column l: its four k
__device__ __forceinline__ s16x4 read_transposed(const char* l) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)const_cast<char*>(l));
}

template <typename H>
__device__ __forceinline__ f32x4 mfma16(const bf16x8& a, const bf16x8& b, f32x4 c) {
  if constexpr (__is_same(H, _Float16))
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Addresses of the epilogue: a wave-uniform pointer and the lane's offset in elements (below 2³² bytes), so
// that the rows and layers a lane visits cost no address registers.
template <typename TO>
__device__ __forceinline__ TO* lane_ptr(TO* uniform, unsigned lane) {
  return reinterpret_cast<TO*>(reinterpret_cast<char*>(const_cast<std::remove_const_t<TO>*>(uniform)) + (size_t)(lane * (unsigned)sizeof(TO)));
}
// eight consecutive values of a row, `left` of them before its end; `vec`: rows of whole, aligned groups of eight
template <typename TO>
__device__ __forceinline__ void store8(TO* p, unsigned lane, int left, bool vec, const float (&v)[8]) {
  TO* q = lane_ptr(p, lane);
  if (vec) {
    if (left > 0) store_vec<TO, 8>(q, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (i < left) q[i] = (TO)v[i];
  }
}
template <typename TO>
__device__ __forceinline__ void load8(const TO* row, int left, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = i < left ? (float)row[i] : 0.f;
}
template <int V>
struct IntConst {
  static constexpr int value = V;
};

// What the forward keeps for the backward, as layers [M][N] of TO: h, then P = act'(g)·u and f = act(g).
// fp32 tensors: a layer each.  16-bit tensors: P and f with 24 bits of their fp32 form (rounding them to
// the type would cost dg and du as much again as their own rounding): a layer of the upper halves
// each, and one with the next byte of both.
constexpr int kept_layers(size_t element) { return element == 4 ? 3 : 4; }
template <typename TO>
__device__ __forceinline__ void store_kept(TO* k, unsigned lane, int64_t layer, int left, bool vec, const float (&h)[8],
                                           const float (&P)[8], const float (&f)[8]) {
  store8<TO>(k, lane, left, vec, h);
  if constexpr (sizeof(TO) == 4) {
    store8<TO>(k + layer, lane, left, vec, P);
    store8<TO>(k + 2 * layer, lane, left, vec, f);
  } else {
    Pack<uint16_t, 8> w[3];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const uint32_t bp = __builtin_bit_cast(uint32_t, P[i]) + 0x80u, bf = __builtin_bit_cast(uint32_t, f[i]) + 0x80u;
      w[0].v[i] = bp >> 16;
      w[1].v[i] = bf >> 16;
      w[2].v[i] = (bp >> 8 & 0xffu) | (bf & 0xff00u);
    }
#pragma unroll
    for (int l = 0; l < 3; l++) {
      uint16_t* q = lane_ptr(reinterpret_cast<uint16_t*>(k) + (l + 1) * layer, lane);
      if (vec) {
        if (left > 0) __builtin_nontemporal_store(__builtin_bit_cast(i32x4, w[l]), reinterpret_cast<i32x4*>(q));
      } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
          if (i < left) q[i] = w[l].v[i];
      }
    }
  }
}
// eight values of P and f as they lie in memory (aligned rows), and as fp32
template <typename TO>
struct KeptRaw {
  uint4 v[sizeof(TO) == 4 ? 4 : 3];
  __device__ __forceinline__ void load(const TO* k, unsigned lane, int64_t layer) {
    if constexpr (sizeof(TO) == 4) {
      const uint4 *p = reinterpret_cast<const uint4*>(lane_ptr(k + layer, lane)),
                  *q = reinterpret_cast<const uint4*>(lane_ptr(k + 2 * layer, lane));
      v[0] = p[0], v[1] = p[1], v[2] = q[0], v[3] = q[1];
    } else {
#pragma unroll
      for (int i = 0; i < 3; i++)
        v[i] = __builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const i32x4*>(lane_ptr(k + (i + 1) * layer, lane))));
    }
  }
  __device__ __forceinline__ void get(float (&P)[8], float (&f)[8]) const {
    if constexpr (sizeof(TO) == 4) {
      const float4 a = __builtin_bit_cast(float4, v[0]), b = __builtin_bit_cast(float4, v[1]), c = __builtin_bit_cast(float4, v[2]),
                   d = __builtin_bit_cast(float4, v[3]);
      P[0] = a.x, P[1] = a.y, P[2] = a.z, P[3] = a.w, P[4] = b.x, P[5] = b.y, P[6] = b.z, P[7] = b.w;
      f[0] = c.x, f[1] = c.y, f[2] = c.z, f[3] = c.w, f[4] = d.x, f[5] = d.y, f[6] = d.z, f[7] = d.w;
    } else {
      const uint32_t hp[4] = {v[0].x, v[0].y, v[0].z, v[0].w}, hf[4] = {v[1].x, v[1].y, v[1].z, v[1].w},
                     lo[4] = {v[2].x, v[2].y, v[2].z, v[2].w};
#pragma unroll
      for (int i = 0; i < 4; i++) {
        P[2 * i] = __builtin_bit_cast(float, hp[i] << 16 | (lo[i] & 0xffu) << 8);
        P[2 * i + 1] = __builtin_bit_cast(float, (hp[i] & 0xffff0000u) | (lo[i] >> 8 & 0xff00u));
        f[2 * i] = __builtin_bit_cast(float, hf[i] << 16 | (lo[i] & 0xff00u));
        f[2 * i + 1] = __builtin_bit_cast(float, (hf[i] & 0xffff0000u) | (lo[i] >> 16 & 0xff00u));
      }
    }
  }
};
template <typename TO>
__device__ __forceinline__ void load_kept(const TO* k, int64_t layer, int left, float (&P)[8], float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i++) {
    P[i] = f[i] = 0.f;
    if (i < left) {
      if constexpr (sizeof(TO) == 4) {
        P[i] = k[layer + i], f[i] = k[2 * layer + i];
      } else {
        const uint16_t* q = reinterpret_cast<const uint16_t*>(k) + layer + i;
        const uint32_t lo = q[2 * layer];
        P[i] = __builtin_bit_cast(float, (uint32_t)q[0] << 16 | (lo & 0xffu) << 8);
        f[i] = __builtin_bit_cast(float, (uint32_t)q[layer] << 16 | (lo & 0xff00u));
      }
    }
  }
}
// planes of eight values (rows of whole groups of eight)
template <typename H>
__device__ __forceinline__ void store_planes8(H* base, unsigned lane, int64_t plane, int planes, const float (&v)[8]) {
  H w[8][3];
#pragma unroll
  for (int i = 0; i < 8; i++) split_planes<H>(v[i], planes, w[i]);
#pragma unroll
  for (int p = 0; p < 3; p++)
    if (p < planes) {
      Pack<H, 8> q;
#pragma unroll
      for (int i = 0; i < 8; i++) q.v[i] = w[i][p];
      *reinterpret_cast<Pack<H, 8>*>(lane_ptr(base + p * plane, lane)) = q;
    }
}

// Tile images in LDS.  Loads write LDS linearly (16 bytes a lane), so a permutation of the 16-byte
// chunks of a row, which spreads the fragment reads over the banks, is made on the global address.
//   k contiguous:    [rows][8 chunks], chunk ^ swz(row).  A: row & 7, fragments read 16 successive
//                    rows.  B: fragment rows are fours 8 apart (see `nrow`), so row & 3 and bit 3.
//   rows contiguous: [64 k][ROWS / 8 chunks], chunk ^ swz_t(k).  A cycle serves 16 lanes of a transposed
//                    read: four k rows (k & 3) of four 8-byte quads, in one chunk pair (A) or four
//                    chunks (B); k & 3 moves them by four chunks, onto sixteen different ones.  With 64
//                    rows two LDS rows span all banks: bit 0 of k is in the address, bit 1 moves.
template <int ROWS, bool T>
struct TileMap {
  static constexpr int kChunks = T ? ROWS / 8 : 8;               // per LDS row
  static constexpr int kRowsPerLoad = 64 / kChunks;
};
template <int ROWS>
__device__ __forceinline__ int swz_t(int k) {
  return ROWS == 64 ? (k >> 1 & 1) << 2 | (k >> 3 & 3) : (k & 3) << 2 | (k >> 3 & 3);
}

// One block: a BM×BN tile of D (kEpiGate: BM×BN/2 of g and of u), WM×WN waves of 16×16×32 MFMAs, k in
// stages of kBK that travel from HBM straight into LDS through a ring of NS stages; one barrier a stage.  Rows past an operand's
// edge and k past its end are outside the buffer descriptor and arrive as zeros.  The right
// operand's fragment is the first MFMA operand, and its fragment rows are chosen so that a lane ends
// with eight consecutive n of a row m, four lanes with 32 (nrow): the epilogue moves 16 bytes a lane, 64
// a row, at a time.
// NP > 1: a stage holds that k run of NP planes of both operands and enters all their products that count,
// p + q < NP, so each tile is loaded once for several products (NP = 1: plane pairs are pairs like others).
template <int P>
struct PlaneProducts;
template <>
struct PlaneProducts<1> {
  static constexpr int n = 1, a[1] = {0}, b[1] = {0};
};
template <>
struct PlaneProducts<2> {                                        // the small products first
  static constexpr int n = 3, a[3] = {0, 1, 0}, b[3] = {1, 0, 0};
};
template <>
struct PlaneProducts<3> {
  static constexpr int n = 6, a[6] = {0, 1, 2, 0, 1, 0}, b[6] = {2, 1, 0, 1, 0, 0};
};
template <typename H, typename TO, int EPI, bool TA, bool TB, int BM, int BN, int WM, int WN, int NS, int NP = 1>
__global__ __launch_bounds__(64 * WM * WN) __attribute__((amdgpu_waves_per_eu(2))) void ffn_gemm_kernel(const GemmArgs a) {
  constexpr int kWaves = WM * WN, FM = BM / WM / 16, FN = BN / WN / 16;
  constexpr int NF = EPI == kEpiGate ? FN / 2 : FN;              // n fragments of one output
  constexpr int LA = BM / 8 / kWaves, LB = BN / 8 / kWaves;      // loads of a wave per stage
  static_assert(NF == 4 || NF == 2, "");
  constexpr int kImage = (BM + BN) * 128, kSlot = NP * kImage;    // bytes of a plane's two tiles, of a stage
  __shared__ uint4 lds[NS][kSlot / 16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;

  // Blocks are dealt to the 8 XCDs in turn: give each XCD a contiguous run of tiles, walked in
  // columns of 8 row tiles, so that its L2 sees the same operand rows again.
  int id = blockIdx.x;
  {
    const int total = gridDim.x, q = total / 8, r = total % 8, xcd = id % 8;
    id = xcd * q + (xcd < r ? xcd : r) + id / 8;
  }
  const int tiles = a.tiles_m * a.tiles_n;
  const int split = id / tiles % a.splits, batch = id / tiles / a.splits;
  id %= tiles;
  const int group = id / (8 * a.tiles_n), first_m = group * 8;
  const int rows_in = a.tiles_m - first_m < 8 ? a.tiles_m - first_m : 8, in_group = id - group * 8 * a.tiles_n;
  const int m0 = (first_m + in_group % rows_in) * BM;
  const int n0 = in_group / rows_in * (EPI == kEpiGate ? BN / 2 : BN);

  int kt = split * a.per_split;
  const int kend = kt + a.per_split < a.pairs * a.ktiles ? kt + a.per_split : a.pairs * a.ktiles;

  // this lane's byte offsets inside a stage, from its first row and k
  unsigned offA[LA], offB[LB];
#pragma unroll
  for (int i = 0; i < LA; i++) {
    constexpr int C = TileMap<BM, TA>::kChunks;
    const int r = (wave * LA + i) * TileMap<BM, TA>::kRowsPerLoad + lane / C, ch = (lane % C) ^ (TA ? swz_t<BM>(r) : r & 7);
    offA[i] = (unsigned)r * (unsigned)a.lda * 2 + ch * 16;
  }
#pragma unroll
  for (int i = 0; i < LB; i++) {
    constexpr int C = TileMap<BN, TB>::kChunks;
    int r = (wave * LB + i) * TileMap<BN, TB>::kRowsPerLoad + lane / C;
    const int ch = (lane % C) ^ (TB ? swz_t<BN>(r) : (r & 3) | ((r >> 3 & 1) << 2));
    if (EPI == kEpiGate) r %= BN / 2;
    offB[i] = (unsigned)r * (unsigned)a.ldb * 2 + ch * 16;
  }
  // An operand from the next stage's first row and k to its end: the base and size of its descriptor.
  // They move on by a constant inside a pair and are set anew at the next one.
  struct Window {
    const char* p;
    int64_t left;                                                  // bytes
    __device__ __forceinline__ i32x4 rsrc() const {
      return descriptor(p, left <= 0 ? 0u : left > 0x7ffffff0 ? 0x7ffffff0u : (uint32_t)left);
    }
  };
  auto window = [&](const void* q, bool trans, int64_t ld, int64_t rows, int r0, int64_t k) {
    const int64_t first = trans ? k * ld + r0 : r0 * ld + k;
    return Window{static_cast<const char*>(q) + first * 2, ((trans ? a.K : rows) * ld - first) * 2};
  };
  const int64_t stepA = kBK * 2 * (TA ? a.lda : 1), stepB = kBK * 2 * (TB ? a.ldb : 1);
  Window wa, wb, wb2;
  // The row tiles of a group start their (circular) walk over the stages two apart: rows of whole
  // multiples of 4 KB have the same k in the same channel of the L2, and in step all blocks would ask
  // that one channel.  Blocks of one row tile stay in step and share its rows.
  const int kfirst = kt;
  int cur = kt + (kt < kend ? in_group % rows_in * 2 % (kend - kt) : 0), pair = cur / a.ktiles, in_pair = cur - pair * a.ktiles;
  auto open = [&] {
    const int64_t k = (int64_t)in_pair * kBK;
    wa = window(batch ? a.A2[pair] : a.A[pair], TA, a.lda, a.M, m0, k);
    wb = window(a.B[pair], TB, a.ldb, a.N, n0, k);
    if constexpr (EPI == kEpiGate) wb2 = window(a.B2[pair], TB, a.ldb, a.N, n0, k);
  };
  auto advance = [&] {
    in_pair++;
    if (++cur == kend || in_pair == a.ktiles) {
      if (cur == kend) cur = kfirst;
      pair = cur / a.ktiles, in_pair = cur - pair * a.ktiles;
      open();
    } else {
      wa.p += stepA, wa.left -= stepA;
      wb.p += stepB, wb.left -= stepB;
      if constexpr (EPI == kEpiGate) wb2.p += stepB, wb2.left -= stepB;
    }
  };
  const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)&lds[0][0];
  // load `n` of this wave's NP·(LA + LB) of a stage, into the ring's slot
  auto issue = [&](int n, int slot) {
    const int p = n / (LA + LB), i = n % (LA + LB);
    const unsigned l = lds0 + slot * kSlot + p * kImage;
    auto of = [&](const Window& w, int64_t plane) { return Window{w.p + p * plane, w.left}.rsrc(); };
    if (i < LA) {
      load_to_lds(of(wa, a.plane_a), l + (wave * LA + i) * 1024, offA[i < LA ? i : 0]);
    } else {
      const int j = i - LA;
      const bool up = EPI == kEpiGate && (wave * LB + j) * 8 >= BN / 2;
      load_to_lds(of(up ? wb2 : wb, a.plane_b), l + BM * 128 + (wave * LB + j) * 1024, offB[j < 0 ? 0 : j]);
    }
  };

  f32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; i++)
#pragma unroll
    for (int j = 0; j < FN; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int fr = lane & 15, fk = lane >> 4;
  // tile row of row r of n fragment j
  auto nrow = [&](int j, int r) {
    const int up = EPI == kEpiGate && j >= NF ? BN / 2 : 0;
    return up + wn * (16 * NF) + (j % NF) / 2 * 32 + (r >> 2) * 8 + (j & 1) * 4 + (r & 3);
  };
  // A fragment of a tile whose rows are contiguous: `at` addresses this lane's quad of the wave's first
  // fragment in the k rows fk·8 + fr / 4; other fragments differ in bits of the chunk only, which the
  // permutation leaves a difference by exclusive or, other k rows by a multiple of 4 (no change to it).
  auto frag_t = [&](auto tile_rows, unsigned at, unsigned other, int image, int ks) {
    constexpr int rows = decltype(tile_rows)::value;
    s16x4 half[2];
#pragma unroll
    for (int hb = 0; hb < 2; hb++)
      half[hb] = read_transposed(reinterpret_cast<const char*>(lds) + ((at ^ other) + image) + (ks * 32 + hb * 4) * rows * 2);
    return __builtin_bit_cast(bf16x8, (s16x8)__builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7));
  };
  unsigned atA = 0, atB = 0;
  {
    const int k = fk * 8 + (fr >> 2);
    if constexpr (TA) atA = k * BM * 2 + (((wm * (BM / WM / 8) + ((fr & 3) >> 1)) ^ swz_t<BM>(k)) << 4) + (fr & 1) * 8;
    if constexpr (TB) atB = BM * 128 + k * BN * 2 + (((wn * (2 * NF) + (fr & 3)) ^ swz_t<BN>(k)) << 4);
  }
  struct Frags {
    bf16x8 a[NP][FM], b[NP][FN];
  };
  // fragment `n` of NP·(FN + FM) of k step ks in a slot
  auto read = [&](int slot, int ks, int n, Frags& f) {
    const int p = n / (FN + FM), i = n % (FN + FM), image = slot * kSlot + p * kImage;
    const uint4* la = &lds[0][0] + image / 16;
    const uint4* lb = la + BM * 8;
    if (i < FN) {
      if constexpr (TB) {
        f.b[p][i] = frag_t(IntConst<BN>{}, atB, (i >> 1) * 64 + (i & 1) * 8, image, ks);
      } else {
        const int r = nrow(i, fr);
        f.b[p][i] = __builtin_bit_cast(bf16x8, lb[r * 8 + ((ks * 4 + fk) ^ ((r & 3) | ((r >> 3 & 1) << 2)))]);
      }
    } else {
      if constexpr (TA) f.a[p][i - FN] = frag_t(IntConst<BM>{}, atA, (i - FN) * 32, image, ks);
      else f.a[p][i - FN] = __builtin_bit_cast(bf16x8, la[(wm * (BM / WM) + (i - FN) * 16 + fr) * 8 + ((ks * 4 + fk) ^ (fr & 7))]);
    }
  };
  // the products of a k step come in S groups: by rows of fragments (NP = 1) or by plane pairs
  constexpr int S = NP == 1 ? FM : PlaneProducts<NP>::n;
  auto products = [&](int s, const Frags& f) {
    const int p = NP == 1 ? 0 : PlaneProducts<NP>::a[NP == 1 ? 0 : s], q = NP == 1 ? 0 : PlaneProducts<NP>::b[NP == 1 ? 0 : s];
#pragma unroll
    for (int i = NP == 1 ? s : 0; i < (NP == 1 ? s + 1 : FM); i++)
#pragma unroll
      for (int j = 0; j < FN; j++) acc[i][j] = mfma16<H>(f.b[q][j], f.a[p][i], acc[i][j]);
  };

  // A stage is two k steps of 32.  A k step's products go group by group, and between the groups
  // go the reads of the next step's fragments and, in the second step, the loads of stage kt + NS (the
  // matrix unit runs on while the wave issues them; sched_barrier keeps the order).  Between the two
  // steps all waves meet: the next stage has landed for each, and the slot of this one, read by all,
  // is free for the loads.
  constexpr int L = NP * (LA + LB), NR = NP * (FM + FN);
  static_assert(kBK == 64, "");
  int get = 0;
  if (kt < kend) {
    open();
#pragma unroll
    for (int s = 0; s < NS; s++)
      if (kt + s < kend) {
#pragma unroll
        for (int i = 0; i < L; i++) issue(i, s);
        advance();
      }
    Frags f0, f1;
    if (kt + NS - 1 < kend) wait_and_barrier<(NS - 1) * L>();
    else wait_and_barrier<0>();
#pragma unroll
    for (int i = 0; i < NR; i++) read(0, 0, i, f0);
    auto both_steps = [&](auto more_c, auto load_c) {                // stages kt + 1, kt + NS follow
      constexpr bool more = decltype(more_c)::value, load = decltype(load_c)::value;
      // each fragment's address is an exclusive or away: not to be kept in a register over the loop
      if constexpr (TA) asm volatile("" : "+v"(atA), "+v"(atB));
#pragma unroll
      for (int s = 0; s < S; s++) {
        products(s, f0);
#pragma unroll
        for (int r = s * NR / S; r < (s + 1) * NR / S; r++) read(get, 1, r, f1);
        __builtin_amdgcn_sched_barrier(0);
      }
      const int slot = get;
      if constexpr (more) {
        if (load || kt + NS - 1 < kend) wait_and_barrier<(NS - 2) * L>();
        else wait_and_barrier<0>();
        get = get + 1 == NS ? 0 : get + 1;
      }
#pragma unroll
      for (int s = 0; s < S; s++) {
        products(s, f1);
        if constexpr (more) {
#pragma unroll
          for (int r = s * NR / S; r < (s + 1) * NR / S; r++) read(get, 0, r, f0);
        }
        if constexpr (load) {
#pragma unroll
          for (int r = s * L / S; r < (s + 1) * L / S; r++) issue(r, slot);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (load) advance();
    };
    for (; kt + NS < kend; kt++) both_steps(IntConst<1>{}, IntConst<1>{});
    for (; kt + 1 < kend; kt++) both_steps(IntConst<1>{}, IntConst<0>{});
    both_steps(IntConst<0>{}, IntConst<0>{});
  }

  // ---- epilogue: lane holds n = un + j·16 + ln … + 7 (j even) of the rows m = um + i·16 + fr --------
  const int um = m0 + wm * (BM / WM), un = n0 + wn * (16 * NF), ln = fk * 8;
  const bool vec = (a.N & 7) == 0;
  const unsigned lane_n = (unsigned)fr * (unsigned)a.N + ln, lane_f = (unsigned)fr * (unsigned)a.ldf + ln;
  auto at_n = [&](int i, int j) { return (int64_t)(um + i * 16) * a.N + un + j * 16; };
  auto at_f = [&](int i, int j) { return (um + i * 16) * a.ldf + un + j * 16; };
  if constexpr (EPI == kEpiStore) {
    TO* out = static_cast<TO*>(batch ? a.out2 : a.out);
    float* partial = a.partial ? a.partial + ((int64_t)batch * a.splits + split) * a.M * a.N : nullptr;
#pragma unroll
    for (int j = 0; j < NF; j += 2) {
      const int left = a.N - (un + j * 16 + ln);
      float b[8];
#pragma unroll
      for (int q = 0; q < 8; q++) b[q] = 0.f;
      if (a.bias && !partial) load8<TO>(static_cast<const TO*>(a.bias) + un + j * 16 + ln, left, b);
#pragma unroll
      for (int i = 0; i < FM; i++) {
        float v[8];
#pragma unroll
        for (int q = 0; q < 8; q++) v[q] = acc[i][j + q / 4][q % 4] + b[q];
        if (um + i * 16 + fr < a.M) {
          if (partial) store8<float>(partial + at_n(i, j), lane_n, left, vec, v);
          else store8<TO>(out + at_n(i, j), lane_n, left, vec, v);
        }
      }
    }
  } else if constexpr (EPI == kEpiGate) {
    const int64_t layer = (int64_t)a.M * a.N, plane = (int64_t)a.M * a.ldf;
#pragma unroll
    for (int j = 0; j < NF; j += 2) {
      const int n = un + j * 16 + ln;
      if (a.bias_g) {
        float b[8];
        load8<TO>(static_cast<const TO*>(a.bias_g) + n, a.N - n, b);
#pragma unroll
        for (int i = 0; i < FM; i++)
#pragma unroll
          for (int q = 0; q < 8; q++) acc[i][j + q / 4][q % 4] += b[q];
      }
      if (a.bias_u) {
        float b[8];
        load8<TO>(static_cast<const TO*>(a.bias_u) + n, a.N - n, b);
#pragma unroll
        for (int i = 0; i < FM; i++)
#pragma unroll
          for (int q = 0; q < 8; q++) acc[i][j + NF + q / 4][q % 4] += b[q];
      }
    }
    auto finish = [&](auto act) {                                // one unrolled body per activation
#pragma unroll
      for (int i = 0; i < FM; i++) {
#pragma unroll
        for (int j = 0; j < NF; j += 2) {
          const int left = a.N - (un + j * 16 + ln);
          float h[8], du[8], f[8];
#pragma unroll
          for (int q = 0; q < 8; q++) {
            const float g = acc[i][j + q / 4][q % 4], u = acc[i][j + NF + q / 4][q % 4];
            float df;
            gate_act_pair(g, decltype(act)::value, f[q], df);
            h[q] = q < left ? f[q] * u : 0.f;
            du[q] = df * u;
          }
          if (um + i * 16 + fr < a.M) {
            if (a.kept) store_kept<TO>(static_cast<TO*>(a.kept) + at_n(i, j), lane_n, layer, left, vec, h, du, f);
            if (a.h && a.N - left < a.ldf) store_planes8<H>(static_cast<H*>(a.h) + at_f(i, j), lane_f, plane, a.planes, h);
          }
        }
      }
    };
    switch (a.act) {
      case kActNone: finish(IntConst<kActNone>{}); break;
      case kActRelu: finish(IntConst<kActRelu>{}); break;
      case kActLrelu: finish(IntConst<kActLrelu>{}); break;
      case kActTanh: finish(IntConst<kActTanh>{}); break;
      case kActSigmoid: finish(IntConst<kActSigmoid>{}); break;
      case kActGelu: finish(IntConst<kActGelu>{}); break;
      default: finish(IntConst<kActSilu>{}); break;
    }
  } else {
    const TO* k = static_cast<const TO*>(a.kept);
    H *dg = static_cast<H*>(a.dg), *du = static_cast<H*>(a.du);
    const int64_t layer = (int64_t)a.M * a.N, plane = (int64_t)a.M * a.ldf;
    const bool inside = vec && m0 + BM <= a.M && n0 + BN <= a.N;      // no row or column of the tile is cut
#pragma unroll
    for (int j = 0; j < NF; j += 2) {
      const int left = a.N - (un + j * 16 + ln);
      float sg[8], su[8];
#pragma unroll
      for (int q = 0; q < 8; q++) sg[q] = su[q] = 0.f;
      auto finish = [&](int i, float (&P)[8], float (&f)[8]) {        // dg = dh·P, du = dh·act
#pragma unroll
        for (int q = 0; q < 8; q++) {
          const float dh = acc[i][j + q / 4][q % 4];
          P[q] *= dh;
          f[q] *= dh;
          sg[q] += P[q];
          su[q] += f[q];
        }
        store_planes8<H>(dg + at_f(i, j), lane_f, plane, a.planes, P);
        store_planes8<H>(du + at_f(i, j), lane_f, plane, a.planes, f);
      };
      if (inside) {
        constexpr int G = 2;                                          // rows whose loads are in flight together
#pragma unroll
        for (int i0 = 0; i0 < FM; i0 += G) {
          KeptRaw<TO> raw[G];
#pragma unroll
          for (int i = 0; i < G; i++) raw[i].load(k + at_n(i0 + i, j), lane_n, layer);
#pragma unroll
          for (int i = 0; i < G; i++) {
            float P[8], f[8];
            raw[i].get(P, f);
            finish(i0 + i, P, f);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < FM; i++) {
          if (um + i * 16 + fr < a.M && a.N - left < a.ldf) {
            float P[8], f[8];
            load_kept<TO>(lane_ptr(k + at_n(i, j), lane_n), layer, left, P, f);   // zeros past N: so are dg and du there
#pragma unroll
            for (int q = 0; q < 8; q++)
              if (q >= left) acc[i][j + q / 4][q % 4] = 0.f;
            finish(i, P, f);
          }
        }
      }
      if (a.col_part) {
        // over the 16 rows of a fragment: lanes of a row of 16 (a whole wave takes part in the sums)
        float* part = a.col_part + (int64_t)(m0 / BM * WM + wm) * 2 * a.N + un + j * 16 + ln;
#pragma unroll
        for (int q = 0; q < 8; q++) {
          sg[q] = group_sum<16>(sg[q]);
          su[q] = group_sum<16>(su[q]);
          if (fr == 0 && q < left) {
            part[q] = sg[q];
            part[a.N + q] = su[q];
          }
        }
      }
    }
  }
}

// ---- few rows ---------------------------------------------------------------------------------
// Up to kSkinnyRows rows in inference: the time is that of reading the weights once, so nothing is
// staged.  A block takes 16 rows of a weight, its waves split k; a lane loads 16 bytes of a weight row
// and of each 16 rows of x straight into MFMA fragments, the waves' sums meet in LDS.  h is rounded to the
// tensors' type between the two launches, as the products of more rows take it (16 bits: the second launch
// reads it once per 16 columns; two planes of it took 39 us instead of 31.6 for 16 rows, 2048 → 8192 → 2048).
// The larger products instead read x once for 128 columns of a block, not once for 16, but have fewer
// blocks and a chain of C / 64 stages each: their time over this form's falls as M·F grows, and they take
// 16-bit tensors from kSkinnyArea on (bf16: 16 rows, C = 1024, F = 4096 15.4 us here and 17.4 there, F =
// 8192, C = 2048 31.6 and 30.1; 64 rows, F = 1024, C = 4096 31.9 and 44.9, F = 2048, C = 512 17.7 and 14.2).
// fp32 weights would have to be split into planes in memory first (64 rows, 2048 → 8192: 122 us and 243).
constexpr int kSkinnyRows = 64, kSkinnyArea = 65536;

// Eight elements from k on, zeros behind K and where `live` is not set: by a load from inside the row and
// a selection, as a branch around each load would wait for one before the next.  ODD (K ≥ 8 no multiple of
// eight): the row's last eight elements are loaded as they end with it, and those before k are zeros; the
// other operand's are moved alike.
template <bool ODD, typename T>
__device__ __forceinline__ Words<T, 8> load_words8(const T* row, int64_t k, int64_t K, bool live = true) {
  Words<T, 8> r;
  if constexpr (ODD) {
    const int64_t at = live && k + 8 <= K ? k : K - 8;
    const int skip = live && k < K ? (int)(k - at) : 8;
    __builtin_memcpy(&r, row + at, sizeof(r));
#pragma unroll
    for (int i = 0; i < (int)(sizeof(r) / 4); i++) {
      if constexpr (sizeof(T) == 4) r.w[i] = i >= skip ? r.w[i] : 0u;
      else r.w[i] &= 2 * i >= skip ? ~0u : 2 * i + 1 >= skip ? 0xffff0000u : 0u;
    }
  } else {
    const bool in = live && k < K;
    __builtin_memcpy(&r, row + (in ? k : 0), sizeof(r));
#pragma unroll
    for (int i = 0; i < (int)(sizeof(r) / 4); i++) r.w[i] = in ? r.w[i] : 0u;
  }
  return r;
}
// the same as the fragments of P planes
template <typename H, typename T, int P>
__device__ __forceinline__ void split_frags(const Words<T, 8>& r, bf16x8 (&out)[P]) {
  if constexpr (sizeof(T) == 2 && P == 1) {
    out[0] = __builtin_bit_cast(bf16x8, r);
  } else {
    Pack<H, 8> w[3];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      H e[3];
      split_planes<H>(r.get(i), P, e);
#pragma unroll
      for (int p = 0; p < 3; p++) w[p].v[i] = e[p];
    }
#pragma unroll
    for (int p = 0; p < P; p++) out[p] = __builtin_bit_cast(bf16x8, w[p]);
  }
}

__device__ __forceinline__ float gate_act(float g, int act) {
  float f, df;
  gate_act_pair(g, act, f, df);
  return f;
}

// Up to kDotRows rows: a wave per column and plain fp32 products, so that every CU takes part in reading
// the weight (the MFMA form below gives N / 16 blocks).  Lanes walk the column's weight row 16 bytes at a
// time.  bf16, 1024 → 4096 → 1024: 6.6 us with one row and 10.4 with four, against 11.8 and 12.8;
// 2048 → 8192 → 2048, 100 MB of weights: 18.5 us, 5.4 TB/s.
constexpr int kDotRows = 4;
// h stays in fp32 between the two launches (TX, TY: the types of x and of the result).
// ROUND: operands rounded to H, as the one-plane modes of fp32 tensors have them
template <typename H, typename TX, typename TO, typename TY, int NB, int MR, bool ROUND, bool ODD>
__global__ __launch_bounds__(256) void ffn_dot_kernel(const TX* x, int M, int64_t K, const TO* w0, const TO* w1, const TO* b0,
                                                      const TO* b1, int N, int act, TY* out) {
  auto in = [](float v) { return ROUND ? (float)(H)v : v; };
  constexpr int U = 8 / NB / MR;                                   // loads of a weight row in flight
  const int lane = threadIdx.x & 63, n = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (n >= N) return;
  const TO* w[2] = {w0 + n * K, NB == 2 ? w1 + n * K : nullptr};
  float acc[NB][MR];
#pragma unroll
  for (int b = 0; b < NB; b++)
#pragma unroll
    for (int m = 0; m < MR; m++) acc[b][m] = 0.f;
  for (int64_t k0 = lane * 8; k0 < K; k0 += 512 * U) {
    Words<TO, 8> wv[U][NB];
    Words<TX, 8> xv[U][MR];
#pragma unroll
    for (int u = 0; u < U; u++) {
#pragma unroll
      for (int b = 0; b < NB; b++) wv[u][b] = load_words8<ODD>(w[b], k0 + u * 512, K);
#pragma unroll
      for (int m = 0; m < MR; m++) xv[u][m] = load_words8<ODD>(x + (int64_t)(m < M ? m : M - 1) * K, k0 + u * 512, K);
    }
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int m = 0; m < MR; m++)
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
          for (int i = 0; i < 8; i++) acc[b][m] += in(xv[u][m].get(i)) * in(wv[u][b].get(i));
  }
#pragma unroll
  for (int m = 0; m < MR; m++) {
    float v[NB];
#pragma unroll
    for (int b = 0; b < NB; b++) v[b] = group_sum<64>(acc[b][m]);
    if (lane == 0 && m < M) {
      float r = v[0] + (b0 ? (float)b0[n] : 0.f);
      if constexpr (NB == 2) r = gate_act(r, act) * (v[1] + (b1 ? (float)b1[n] : 0.f));
      out[(int64_t)m * N + n] = (TY)r;
    }
  }
}

// NB weights (gate and up, or down alone) times x [M][K], both as P planes: h = act(g)·u (NB = 2) or y
template <typename H, typename TO, int NB, int MF, int P, int WAVES, bool ODD>
__global__ __launch_bounds__(64 * WAVES) void ffn_skinny_kernel(const TO* x, int M, int64_t K, const TO* w0, const TO* w1,
                                                                const TO* b0, const TO* b1, int N, int act, TO* out) {
  constexpr int kLoads = (NB + MF) * (int)sizeof(TO) / 2;             // 16-byte loads a k step
  constexpr int U = kLoads <= 4 ? 4 : kLoads <= 8 ? 2 : 1;            // k steps whose loads are in flight
  __shared__ f32x4 part[WAVES][NB * MF][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 15, fk = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int64_t row = n0 + fr < N ? n0 + fr : N - 1;
  const TO* w[2] = {w0 + row * K, NB == 2 ? w1 + row * K : nullptr};
  f32x4 acc[NB][MF];
#pragma unroll
  for (int b = 0; b < NB; b++)
#pragma unroll
    for (int m = 0; m < MF; m++) acc[b][m] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int64_t steps = (K + 31) / 32, per = (steps + WAVES - 1) / WAVES, s1 = (wave + 1) * per < steps ? (wave + 1) * per : steps;
  for (int64_t s = wave * per; s < s1; s += U) {
    Words<TO, 8> qw[U][NB];
    Words<TO, 8> qx[U][MF];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int64_t k = (s + u) * 32 + fk * 8;
      const bool live = s + u < s1;
#pragma unroll
      for (int b = 0; b < NB; b++) qw[u][b] = load_words8<ODD>(w[b], k, K, live);
#pragma unroll
      for (int m = 0; m < MF; m++) qx[u][m] = load_words8<ODD>(x + (int64_t)(m * 16 + fr < M ? m * 16 + fr : M - 1) * K, k, K, live);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      bf16x8 fw[NB][P];
#pragma unroll
      for (int b = 0; b < NB; b++) split_frags<H>(qw[u][b], fw[b]);
#pragma unroll
      for (int m = 0; m < MF; m++) {
        bf16x8 fx[P];
        split_frags<H>(qx[u][m], fx);
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
          for (int o = P - 1; o >= 0; o--)                           // the small products first
#pragma unroll
            for (int i = 0; i <= o; i++) acc[b][m] = mfma16<H>(fw[b][o - i], fx[i], acc[b][m]);
      }
    }
  }
#pragma unroll
  for (int b = 0; b < NB; b++)
#pragma unroll
    for (int m = 0; m < MF; m++) part[wave][b * MF + m][lane] = acc[b][m];
  __syncthreads();
  // wave m joins the rows m·16 …: lane holds columns n0 + 4·fk … + 3 of row m·16 + fr
  const int m = wave * 16 + fr;
  if (wave < MF && m < M) {
    f32x4 v[NB];
#pragma unroll
    for (int b = 0; b < NB; b++) {
      v[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int q = 0; q < WAVES; q++) v[b] += part[q][b * MF + wave][lane];
    }
#pragma unroll
    for (int q = 0; q < 4; q++) {
      const int n = n0 + fk * 4 + q;
      if (n < N) {
        float r = v[0][q] + (b0 ? (float)b0[n] : 0.f);
        if constexpr (NB == 2) r = gate_act(r, act) * (v[1][q] + (b1 ? (float)b1[n] : 0.f));
        out[(int64_t)m * N + n] = (TO)r;
      }
    }
  }
}

// ---- host -------------------------------------------------------------------------------------
// How the operands become 16-bit planes
struct Mode {
  int planes;
  bool pack;                     // fp32: always; 16-bit tensors only where their rows do not fit the loads
};

// plane pairs of a product, the small terms first; pairs below the last kept order are left out
int plane_pairs(int planes, int (&pa)[6], int (&pb)[6]) {
  int n = 0;
  for (int s = planes - 1; s >= 0; s--)
    for (int i = 0; i <= s; i++) {
      pa[n] = i;
      pb[n++] = s - i;
    }
  return n;
}

// an operand in product form: planes of [rows][ld], zeros from the tensor's row end to ld
struct Operand {
  const char* p = nullptr;
  int64_t rows = 0, ld = 0;
};

struct Bump {                    // the caller's workspace, cut in order (base null: sizes only)
  char* base;
  size_t used = 0;
  void* take(size_t n) {
    char* p = base ? base + used : nullptr;
    used += (n + 255) / 256 * 256;
    return p;
  }
};

constexpr size_t kPartialCap = (size_t)256 << 20;   // bytes of split-K partials at most
constexpr int kColChunks = 64;                      // row chunks of a column sum at most

struct Tiling {
  int bm, bn, tiles_m, tiles_n, splits, per_split;   // bn: columns of the output
};
// The largest of three tiles that still gives the 256 CUs a block each: 256×256, 128×128 (two blocks a
// CU), 64×64 (kEpiGate: half as many columns of g and of u each, 64×64 with 64).  `stages`: of one plane
// pair; `products`: plane pairs.  Small tiles take all planes of a k run in one stage (NP): they are bound
// by their loads (fp32 8192 rows, 128 → 512 → 128: forward and backward 145 … 150 us back to back, 181 with a plane
// pair a stage; the forward takes 48 us, 55 with such stages in place of the 128×128 tiles too).
// A product of small tiles whose partial sums may be stored splits k into runs of at least 4 stages (2 of
// all planes): up to two blocks a CU where there is not one (one with three planes, whose stages fill its
// LDS: 512 × 128 from 8192, 21.2 us, 23.6 with two), and with one plane up to three for 64 stages and more,
// over which one block a CU waits longer than the sums cost (8192 × 128, 96 stages: 37.8 us unsplit, 32
// split; 48 stages: 18.9 and 21).
Tiling tile(int64_t M, int64_t N, int batches, int stages, int products, bool gate, bool may_split) {
  Tiling t{};
  for (int b : {256, 128, 64}) {
    t.bm = b, t.bn = gate && b > 64 ? b / 2 : b;
    t.tiles_m = (int)((M + t.bm - 1) / t.bm), t.tiles_n = (int)((N + t.bn - 1) / t.bn);
    if ((int64_t)t.tiles_m * t.tiles_n * batches >= 224) break;
  }
  if (t.bm > 64) stages *= products;
  t.splits = 1;
  const int64_t tiles = (int64_t)t.tiles_m * t.tiles_n * batches;
  if (may_split && t.bm == 64 && (tiles < 224 || (products == 1 && stages >= 64 && tiles < 512))) {
    int64_t s = (products > 3 ? 256 : tiles < 224 ? 512 : 768) / tiles;
    const int run = products > 1 ? 2 : 4;
    if (s > stages / run) s = stages / run;
    const int64_t cap = (int64_t)(kPartialCap / ((size_t)M * N * batches * 4));
    if (s > cap) s = cap;
    if (s > 1) t.splits = (int)s;
  }
  t.per_split = (stages + t.splits - 1) / t.splits;
  t.splits = (stages + t.per_split - 1) / t.per_split;
  return t;
}
size_t partial_bytes(const Tiling& t, int64_t M, int64_t N, int batches) {
  return t.splits > 1 ? (size_t)t.splits * M * N * batches * sizeof(float) : 0;
}
// One call: the same walk over the steps sizes the workspace (dry: no base pointer) and launches.
template <typename H, typename TO>
struct Ffn {
  const FfnArgs& f;
  const Mode mode;
  const int planes;
  Bump ws;
  const bool dry;
  hipStream_t st;

  Ffn(const FfnArgs& fa, Mode m, void* w, hipStream_t s)
      : f(fa), mode(m), planes(m.planes), ws{static_cast<char*>(w)}, dry(!w), st(s) {}

  struct Packed {
    const void* src;
    int64_t K;
    Operand o;
  };
  PackArgs packs{};
  int64_t pack_blocks = 0;
  Packed packed[kMaxPacks];
  int done = 0;

  int npairs() const { return planes * (planes + 1) / 2; }
  Operand planes_of(int64_t rows, int64_t cols) {
    Operand o;
    o.rows = rows;
    o.ld = round_k(cols);
    o.p = static_cast<const char*>(ws.take((size_t)planes * rows * o.ld * 2));
    return o;
  }

  // `src` [R][K] in product form: itself where its rows are whole stages (k contiguous) or whole
  // 16-byte chunks (k the slow axis), else packed into the workspace, once a call, by the next flush()
  Operand operand(const void* src, int64_t R, int64_t K, bool k_slow) {
    Operand o;
    if (!mode.pack && K % (k_slow ? 8 : kBK) == 0) {
      o.p = static_cast<const char*>(src), o.rows = R, o.ld = K;
      return o;
    }
    for (int i = 0; i < done; i++)
      if (packed[i].src == src && packed[i].o.rows == R && packed[i].K == K) return packed[i].o;
    o = planes_of(R, K);
    packed[done++] = {src, K, o};
    PackJob& j = packs.job[packs.jobs++];
    j = {src, const_cast<char*>(o.p), R, K, o.ld, pack_blocks};
    pack_blocks += (R * o.ld / 4 + kPackQuads - 1) / kPackQuads;
    return o;
  }
  int flush() {
    packs.planes = planes;
    const int n = packs.jobs;
    const int64_t blocks = pack_blocks;
    packs.jobs = 0, pack_blocks = 0;
    if (!n || dry) return kOk;
    const PackArgs a = [&] { PackArgs c = packs; c.jobs = n, c.blocks = blocks; return c; }();
    ffn_pack_kernel<TO, H><<<(unsigned)(blocks < kPackBlocks ? blocks : kPackBlocks), 256, 0, st>>>(a);
    return check_launch("ffn_pack");
  }

  // the plane pairs of A·B into the list; K: extent of k, rows of a slow-axis operand
  void pairs(GemmArgs& a, const Operand& A, const Operand* A2, const Operand& B, const Operand* B2, int64_t K) {
    int pa[6], pb[6];
    const int n = plane_pairs(planes, pa, pb);
    for (int i = 0; i < n; i++, a.pairs++) {
      a.A[a.pairs] = A.p + pa[i] * A.rows * A.ld * 2;
      a.A2[a.pairs] = A2 ? A2->p + pa[i] * A2->rows * A2->ld * 2 : nullptr;
      a.B[a.pairs] = B.p + pb[i] * B.rows * B.ld * 2;
      a.B2[a.pairs] = B2 ? B2->p + pb[i] * B2->rows * B2->ld * 2 : nullptr;
    }
    a.lda = A.ld, a.ldb = B.ld, a.K = K;
    a.plane_a = A.rows * A.ld * 2, a.plane_b = B.rows * B.ld * 2;
    a.ktiles = (int)(round_k(K) / kBK);
    a.batches = A2 ? 2 : 1;
  }

  template <int EPI, bool TA, bool TB>
  int gemm(GemmArgs& a, const Tiling& t, void* partial) {
    a.tiles_m = t.tiles_m, a.tiles_n = t.tiles_n, a.splits = t.splits, a.per_split = t.per_split;
    a.partial = t.splits > 1 ? static_cast<float*>(partial) : nullptr;
    const unsigned grid = (unsigned)t.tiles_m * t.tiles_n * t.splits * a.batches;
    constexpr int SN = EPI == kEpiGate ? 128 : 64;           // LDS columns of the smallest tile
    constexpr int GM = EPI == kEpiGate ? 4 : 2;              // waves along m: 128-byte rows of the gate's outputs a wave
    if (t.bm == 256) ffn_gemm_kernel<H, TO, EPI, TA, TB, 256, 256, GM, 8 / GM, 2><<<grid, 512, 0, st>>>(a);
    else if (t.bm == 128) ffn_gemm_kernel<H, TO, EPI, TA, TB, 128, 128, 2, 2, 2><<<grid, 256, 0, st>>>(a);
    else if (planes == 1) ffn_gemm_kernel<H, TO, EPI, TA, TB, 64, SN, 2, 2, 3><<<grid, 256, 0, st>>>(a);
    else if constexpr (sizeof(TO) == 4 && !__is_same(H, _Float16)) {   // fp32 as two or three bf16 planes
      const int n = npairs();
      a.pairs /= n;
      for (int g = 0; g < a.pairs; g++) {                              // the last of a run of pairs is that of the first planes
        const int k = g * n + n - 1;
        a.A[g] = a.A[k], a.A2[g] = a.A2[k], a.B[g] = a.B[k], a.B2[g] = a.B2[k];
      }
      if (planes == 2) ffn_gemm_kernel<H, TO, EPI, TA, TB, 64, SN, 2, 2, 2, 2><<<grid, 256, 0, st>>>(a);
      else ffn_gemm_kernel<H, TO, EPI, TA, TB, 64, SN, 2, 2, 2, 3><<<grid, 256, 0, st>>>(a);
    }
    static constexpr const char* names[3][3] = {{"ffn_gemm_64", "ffn_gemm_128", "ffn_gemm_256"},
                                                {"ffn_gemm_gate_64", "ffn_gemm_gate_128", "ffn_gemm_gate_256"},
                                                {"ffn_gemm_gate_bwd_64", "ffn_gemm_gate_bwd_128", "ffn_gemm_gate_bwd_256"}};
    if (int rc = check_launch(names[EPI][t.bm / 128])) return rc;
    if (t.splits > 1) {
      const int64_t total = (int64_t)a.M * a.N;
      return reduce(a.partial, t.splits, total, a.N, a.bias, a.out, a.batches == 2 ? a.out2 : nullptr);
    }
    return kOk;
  }

  // many parts of few elements: more threads an element
  int reduce(const float* part, int parts, int64_t total, int N, const void* bias, void* out, void* out2 = nullptr) {
    const dim3 grid((unsigned)((total + 63) / 64), out2 ? 2 : 1);
    const TO* b = static_cast<const TO*>(bias);
    TO *o = static_cast<TO*>(out), *o2 = static_cast<TO*>(out2);
    if (N % 4 == 0 && (parts <= 8 || total >= (1 << 18)))
      ffn_reduce4_kernel<TO><<<dim3((unsigned)((total / 4 + 255) / 256), grid.y), 256, 0, st>>>(part, parts, total, N, b, o, o2);
    else if (parts > 8) ffn_reduce_kernel<TO, 16><<<grid, 1024, 0, st>>>(part, parts, total, N, b, o, o2);
    else ffn_reduce_kernel<TO, 4><<<grid, 256, 0, st>>>(part, parts, total, N, b, o, o2);
    return check_launch("ffn_reduce");
  }

  struct GateIn {
    Operand x, wg, wu;
  };
  GateIn gate_operands() {
    GateIn g;
    g.x = operand(f.x, f.M, f.C, false);
    g.wg = operand(f.wg, f.F, f.C, false);
    g.wu = operand(f.wu, f.F, f.C, false);
    return g;
  }
  // h (planes) and / or kept of all rows
  int gate(const GateIn& in, const Operand& h, void* kept) {
    if (dry) return kOk;
    GemmArgs a{};
    pairs(a, in.x, nullptr, in.wg, &in.wu, f.C);
    a.M = (int)f.M, a.N = f.F;
    a.bias_g = f.bg, a.bias_u = f.bu, a.act = f.act, a.planes = planes;
    a.kept = kept;
    a.h = const_cast<char*>(h.p), a.ldf = h.ld;
    return gemm<kEpiGate, false, false>(a, tile(f.M, f.F, 1, a.ktiles, npairs(), true, false), nullptr);
  }

  // One launch for few rows, x [M][K]: NB = 2 gate, up → h; NB = 1 down → y.  P: planes of the operands.
  template <int NB, int P, bool ODD>
  int skinny(const void* x, int64_t K, const void* w0, const void* w1, const void* b0, const void* b1, int N, void* out) {
    const TO *xt = static_cast<const TO*>(x), *v0 = static_cast<const TO*>(w0), *v1 = static_cast<const TO*>(w1),
             *c0 = static_cast<const TO*>(b0), *c1 = static_cast<const TO*>(b1);
    TO* o = static_cast<TO*>(out);
    const int M = (int)f.M;
    constexpr int W = 8;
    const unsigned grid = (unsigned)ceil_div(N, 16);
    if (M <= 16) ffn_skinny_kernel<H, TO, NB, 1, P, W, ODD><<<grid, 64 * W, 0, st>>>(xt, M, K, v0, v1, c0, c1, N, f.act, o);
    else if (M <= 32) ffn_skinny_kernel<H, TO, NB, 2, P, W, ODD><<<grid, 64 * W, 0, st>>>(xt, M, K, v0, v1, c0, c1, N, f.act, o);
    else ffn_skinny_kernel<H, TO, NB, 4, P, W, ODD><<<grid, 64 * W, 0, st>>>(xt, M, K, v0, v1, c0, c1, N, f.act, o);
    return check_launch("ffn_skinny");
  }
  template <int NB, int P, bool ODD, typename TX, typename TY>
  int dot(const void* x, int64_t K, const void* w0, const void* w1, const void* b0, const void* b1, int N, TY* out) {
    constexpr bool R = sizeof(TO) == 4 && P == 1;
    const TX* xt = static_cast<const TX*>(x);
    const TO *v0 = static_cast<const TO*>(w0), *v1 = static_cast<const TO*>(w1), *c0 = static_cast<const TO*>(b0),
             *c1 = static_cast<const TO*>(b1);
    const int M = (int)f.M;
    const unsigned grid = (unsigned)ceil_div(N, 4);
    if (M == 1) ffn_dot_kernel<H, TX, TO, TY, NB, 1, R, ODD><<<grid, 256, 0, st>>>(xt, M, K, v0, v1, c0, c1, N, f.act, out);
    else if (M == 2) ffn_dot_kernel<H, TX, TO, TY, NB, 2, R, ODD><<<grid, 256, 0, st>>>(xt, M, K, v0, v1, c0, c1, N, f.act, out);
    else ffn_dot_kernel<H, TX, TO, TY, NB, 4, R, ODD><<<grid, 256, 0, st>>>(xt, M, K, v0, v1, c0, c1, N, f.act, out);
    return check_launch("ffn_dot");
  }
  template <int P, bool ODD>
  int first(void* h) {
    if (f.M <= kDotRows) return dot<2, P, ODD, TO>(f.x, f.C, f.wg, f.wu, f.bg, f.bu, f.F, static_cast<float*>(h));
    return skinny<2, P, ODD>(f.x, f.C, f.wg, f.wu, f.bg, f.bu, f.F, h);
  }
  template <int P, bool ODD>
  int second(const void* h, void* y) {
    if (f.M <= kDotRows) return dot<1, P, ODD, float>(h, f.F, f.wd, nullptr, f.bd, nullptr, f.O, static_cast<TO*>(y));
    return skinny<1, P, ODD>(h, f.F, f.wd, nullptr, f.bd, nullptr, f.O, y);
  }
  template <int P>
  int few_rows(void* y, void* h) {
    if (int rc = f.C % 8 ? first<P, true>(h) : first<P, false>(h)) return rc;
    return f.F % 8 ? second<P, true>(h, y) : second<P, false>(h, y);
  }

  int forward(void* y, void* kept) {
    const bool area = sizeof(TO) == 4 || f.M * f.F <= kSkinnyArea || f.M <= kDotRows;
    if (!kept && f.M <= kSkinnyRows && area && f.C >= 8 && f.F >= 8) {
      void* h = ws.take((size_t)f.M * f.F * (f.M <= kDotRows ? sizeof(float) : sizeof(TO)));
      if (dry) return kOk;
      if constexpr (sizeof(TO) == 2) return few_rows<1>(y, h);
      else return planes == 3 ? few_rows<3>(y, h) : planes == 2 ? few_rows<2>(y, h) : few_rows<1>(y, h);
    }
    // kept's first layer is h as the next product takes it, unless that needs planes or padding
    const bool direct = !mode.pack && f.F % kBK == 0;
    Operand h = planes_of(f.M, f.F);
    if (direct && kept) h.p = static_cast<const char*>(kept);
    const GateIn in = gate_operands();
    const Operand wd = operand(f.wd, f.O, f.F, false);
    if (int rc = flush()) return rc;
    if (int rc = gate(in, direct && kept ? Operand{} : h, kept)) return rc;
    const Tiling t = tile(f.M, f.O, 1, (int)(h.ld / kBK), npairs(), false, true);
    void* partial = ws.take(partial_bytes(t, f.M, f.O, 1));
    if (dry) return kOk;
    GemmArgs a{};
    pairs(a, h, nullptr, wd, nullptr, f.F);
    a.M = (int)f.M, a.N = f.O;
    a.out = y, a.bias = f.bd;
    return gemm<kEpiStore, false, false>(a, t, partial);
  }

  int column_sums(const void* src, int64_t rows, int cols, void* out) {
    const int64_t per = rows > 64 * kColChunks ? (rows + kColChunks - 1) / kColChunks : 64, chunks = (rows + per - 1) / per;
    float* part = static_cast<float*>(ws.take((size_t)chunks * cols * sizeof(float)));
    if (dry) return kOk;
    ffn_col_sum_kernel<TO><<<dim3(ceil_div(cols, 64), (unsigned)chunks), 256, 0, st>>>(static_cast<const TO*>(src), rows, cols, per,
                                                                                       part);
    if (int rc = check_launch("ffn_col_sum")) return rc;
    return reduce(part, (int)chunks, cols, cols, nullptr, out);
  }

  int backward(const void* dy, const void* kept, const FfnGrads& o) {
    const bool inner = o.dx || o.dwg || o.dwu || o.dbg || o.dbu, weights = o.dwg || o.dwu;
    const bool again = !kept;                                // h, act'·u and act are computed again
    GateIn in;
    if (again) {
      in = gate_operands();
      kept = ws.take((size_t)kept_layers(sizeof(TO)) * f.M * f.F * sizeof(TO));
    }
    Operand dyr, dyk, wd, wg, wu, x, h, dg, du;
    if (inner) dyr = operand(dy, f.M, f.O, false), wd = operand(f.wd, f.O, f.F, true);
    if (o.dx) wg = operand(f.wg, f.F, f.C, true), wu = operand(f.wu, f.F, f.C, true);
    if (weights) x = operand(f.x, f.M, f.C, true);
    if (o.dwd) dyk = operand(dy, f.M, f.O, true);
    if (o.dwd && !again) h = operand(kept, f.M, f.F, true);  // the first layer of kept
    if (int rc = flush()) return rc;
    if (again) {
      if (int rc = gate(in, Operand{}, const_cast<void*>(kept))) return rc;
      if (o.dwd) {
        h = operand(kept, f.M, f.F, true);
        if (int rc = flush()) return rc;
      }
    }
    if (inner) {
      dg = planes_of(f.M, f.F), du = planes_of(f.M, f.F);
      const Tiling t = tile(f.M, f.F, 1, (int)(round_k(f.O) / kBK), npairs(), false, false);
      const int rows = t.tiles_m * 2;                        // two waves along m in every tile
      float* part = o.dbg || o.dbu ? static_cast<float*>(ws.take((size_t)rows * 2 * f.F * sizeof(float))) : nullptr;
      if (!dry) {
        GemmArgs a{};
        pairs(a, dyr, nullptr, wd, nullptr, f.O);
        a.M = (int)f.M, a.N = f.F;
        a.planes = planes, a.kept = const_cast<void*>(kept);
        a.dg = const_cast<char*>(dg.p), a.du = const_cast<char*>(du.p), a.ldf = dg.ld;
        a.col_part = part;
        if (int rc = gemm<kEpiGateBwd, false, true>(a, t, nullptr)) return rc;
        if (part) {
          ffn_bias_reduce_kernel<TO><<<(unsigned)ceil_div(2 * (int64_t)f.F, 64), 1024, 0, st>>>(
              part, rows, f.F, static_cast<TO*>(o.dbg), static_cast<TO*>(o.dbu));
          if (int rc = check_launch("ffn_bias_reduce")) return rc;
        }
      }
    }
    if (o.dx) {
      const Tiling t = tile(f.M, f.C, 1, 2 * (int)(dg.ld / kBK), npairs(), false, true);
      void* partial = ws.take(partial_bytes(t, f.M, f.C, 1));
      if (!dry) {
        GemmArgs a{};
        pairs(a, dg, nullptr, wg, nullptr, f.F);
        pairs(a, du, nullptr, wu, nullptr, f.F);
        a.M = (int)f.M, a.N = f.C;
        a.out = o.dx;
        if (int rc = gemm<kEpiStore, false, true>(a, t, partial)) return rc;
      }
    }
    if (weights) {
      const int both = o.dwg && o.dwu ? 2 : 1;
      const int stages = (int)(round_k(f.M) / kBK);
      const Tiling t = tile(f.F, f.C, both, stages, npairs(), false, true);
      // one product has half the tiles of two and may split k where those do not: room for either, so that the
      // size asked for with both gradients holds for one
      size_t bytes = 0;
      for (int n : {1, 2}) {
        const size_t b = partial_bytes(tile(f.F, f.C, n, stages, npairs(), false, true), f.F, f.C, n);
        bytes = b > bytes ? b : bytes;
      }
      void* partial = ws.take(bytes);
      if (!dry) {
        GemmArgs a{};
        pairs(a, o.dwg ? dg : du, both == 2 ? &du : nullptr, x, nullptr, f.M);
        a.M = f.F, a.N = f.C;
        a.out = o.dwg ? o.dwg : o.dwu, a.out2 = o.dwu;
        if (int rc = gemm<kEpiStore, true, true>(a, t, partial)) return rc;
      }
    }
    if (o.dwd) {
      const Tiling t = tile(f.O, f.F, 1, (int)(round_k(f.M) / kBK), npairs(), false, true);
      void* partial = ws.take(partial_bytes(t, f.O, f.F, 1));
      if (!dry) {
        GemmArgs a{};
        pairs(a, dyk, nullptr, h, nullptr, f.M);
        a.M = f.O, a.N = f.F;
        a.out = o.dwd;
        if (int rc = gemm<kEpiStore, true, true>(a, t, partial)) return rc;
      }
    }
    if (o.dbd)
      if (int rc = column_sums(dy, f.M, f.O, o.dbd)) return rc;
    return kOk;
  }
};

template <typename H, typename TO>
size_t ffn_ws(const FfnArgs& shape, Mode mode, int backward, int recompute) {
  static char t[8];              // distinct tensors, none of them packed once for two
  FfnArgs f = shape;
  f.x = t, f.wg = t + 1, f.wu = t + 2, f.wd = t + 3;
  Ffn<H, TO> r(f, mode, nullptr, nullptr);
  if (backward) {
    r.backward(t + 4, recompute ? nullptr : t + 5, FfnGrads{t, t, t, t, t, t, t});
    return r.ws.used;
  }
  r.forward(t, t + 6);           // with kept, and without: the larger
  Ffn<H, TO> q(f, mode, nullptr, nullptr);
  q.forward(t, nullptr);
  return r.ws.used > q.ws.used ? r.ws.used : q.ws.used;
}

}  // namespace

// Entry points of one (plane type, tensor type): each is instantiated in a file of its own.
#define MRAGAN_FFN_ENTRIES(name, H, TO)                                                                                       \
  size_t ffn_ws_##name(const FfnArgs& f, int planes, int pack, int backward, int recompute) {                                 \
    return ffn_ws<H, TO>(f, Mode{planes, pack != 0}, backward, recompute);                                                    \
  }                                                                                                                           \
  size_t ffn_bwd_bytes_##name(const FfnArgs& f, int planes, int pack, const void* dy, const void* kept, const FfnGrads& o) {  \
    Ffn<H, TO> r(f, Mode{planes, pack != 0}, nullptr, nullptr);                                                               \
    r.backward(dy, kept, o);                                                                                                  \
    return r.ws.used;                                                                                                         \
  }                                                                                                                           \
  int ffn_fwd_##name(const FfnArgs& f, int planes, int pack, void* y, void* kept, void* ws, hipStream_t st) {                 \
    return Ffn<H, TO>(f, Mode{planes, pack != 0}, ws, st).forward(y, kept);                                                   \
  }                                                                                                                           \
  int ffn_bwd_##name(const FfnArgs& f, int planes, int pack, const void* dy, const void* kept, const FfnGrads& o, void* ws,   \
                     hipStream_t st) {                                                                                        \
    return Ffn<H, TO>(f, Mode{planes, pack != 0}, ws, st).backward(dy, kept, o);                                              \
  }

}  // namespace mragan
