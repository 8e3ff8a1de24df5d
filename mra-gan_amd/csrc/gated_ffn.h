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
#pragma once
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

// src [R][K] (any type) → 16-bit planes dst [planes][R][ld], zeros from K to ld
template <typename T, typename H>
__global__ __launch_bounds__(256) void ffn_pack_kernel(const T* src, int64_t R, int64_t K, int planes, H* dst, int64_t ld) {
  const int64_t quads = ld / 4, total = R * quads, step = (int64_t)gridDim.x * 256, plane = R * ld;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += step) {
    const int64_t r = i / quads, k = (i - r * quads) * 4;
    H w[4][3];
#pragma unroll
    for (int q = 0; q < 4; q++) split_planes<H>(k + q < K ? (float)src[r * K + k + q] : 0.f, planes, w[q]);
#pragma unroll
    for (int p = 0; p < 3; p++)
      if (p < planes) {
        Pack<H, 4> o;
#pragma unroll
        for (int q = 0; q < 4; q++) o.v[q] = w[q][p];
        *reinterpret_cast<Pack<H, 4>*>(dst + p * plane + r * ld + k) = o;
      }
  }
}

// Σ over a chunk of rows of the columns of planes [planes][rows][ld] → part [chunks][cols]; a thread
// takes four columns, the waves of a block every fourth row
template <typename H>
__global__ __launch_bounds__(256) void ffn_col_sum_kernel(const H* src, int64_t rows, int cols, int64_t ld, int planes,
                                                          int64_t per_chunk, float* part) {
  __shared__ float s[4][256];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = blockIdx.x * 256 + lane * 4;
  const int64_t r0 = blockIdx.y * per_chunk, r1 = r0 + per_chunk < rows ? r0 + per_chunk : rows;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  if (c < ld)
    for (int p = 0; p < planes; p++)
#pragma unroll 4
      for (int64_t r = r0 + wave; r < r1; r += 4) {
        float t[4];
        load_vec<H, 4>(src + (p * rows + r) * ld + c, t);
#pragma unroll
        for (int q = 0; q < 4; q++) v[q] += t[q];
      }
#pragma unroll
  for (int q = 0; q < 4; q++) s[wave][lane * 4 + q] = v[q];
  __syncthreads();
  const int col = blockIdx.x * 256 + threadIdx.x;
  if (col < cols) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < 4; w++) t += s[w][threadIdx.x];
    part[(int64_t)blockIdx.y * cols + col] = t;
  }
}

// out[i] = Σ_s part[s][i] in order (+ bias[i mod N])
template <typename TO>
__global__ __launch_bounds__(256) void ffn_reduce_kernel(const float* part, int parts, int64_t total, int N, const TO* bias,
                                                         TO* out) {
  const int64_t step = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += step) {
    float v = 0.f;
    for (int s = 0; s < parts; s++) v += part[s * total + i];
    if (bias) v += (float)bias[i % N];
    out[i] = (TO)v;
  }
}

// ---- the product ------------------------------------------------------------------------------
struct GemmArgs {
  const void* A[kMaxPairs];       // k contiguous: [M][lda]; rows contiguous: [K][lda]
  const void* A2[kMaxPairs];      // of a second product with the same B (batches = 2), to out2
  const void* B[kMaxPairs];       // [N][ldb] or [K][ldb]; kEpiGate: the gate weight
  const void* B2[kMaxPairs];      // kEpiGate: the up weight
  int pairs, ktiles, batches;     // operand pairs, stages of kBK of one pair
  int64_t lda, ldb, K;            // elements
  int M, N;
  int tiles_m, tiles_n, splits, per_split;   // stages of all pairs cut into `splits` runs of per_split
  // kEpiStore: out[m][n] (+ bias[n]); splits > 1: fp32 partials [batch][split][M][N]
  void *out, *out2;
  const void* bias;
  float* partial;
  // kEpiGate / kEpiGateBwd: 16-bit planes of [M][ldf]
  const void *bias_g, *bias_u;
  int act, planes;
  void* kept;                     // [3][M][N] (h, act'·u, act): written by kEpiGate if given, read by kEpiGateBwd
  void *h, *dg, *du;
  int64_t ldf;
};

// A wave's 64 × 16 bytes from a buffer straight into LDS at `lds` + 16·lane.  As assembly, with the
// waits below: after the builtin the compiler waits for every such load before any transposed LDS
// read, whichever stage it reads, and the loads of the next stages would never be in flight.
typedef int i32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void load_to_lds(i32x4 rsrc, unsigned lds, unsigned voffset) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(voffset), "s"(rsrc)
               : "memory");
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

// eight consecutive values of a row from column n; `vec`: rows of whole, aligned groups of eight
template <typename TO>
__device__ __forceinline__ void store8(TO* row, int n, int N, bool vec, const float (&v)[8]) {
  if (vec) {
    if (n < N) store_vec<TO, 8>(row + n, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (n + i < N) row[n + i] = (TO)v[i];
  }
}
template <typename TO>
__device__ __forceinline__ void load8(const TO* row, int n, int N, bool vec, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = 0.f;
  if (vec) {
    if (n < N) load_vec<TO, 8>(row + n, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (n + i < N) v[i] = (float)row[n + i];
  }
}
// planes of eight values at element `off` of each plane (rows of whole groups of eight)
template <typename H>
__device__ __forceinline__ void store_planes8(void* base, int64_t off, int64_t plane, int planes, const float (&v)[8]) {
  H w[8][3];
#pragma unroll
  for (int i = 0; i < 8; i++) split_planes<H>(v[i], planes, w[i]);
#pragma unroll
  for (int p = 0; p < 3; p++)
    if (p < planes) {
      Pack<H, 8> q;
#pragma unroll
      for (int i = 0; i < 8; i++) q.v[i] = w[i][p];
      *reinterpret_cast<Pack<H, 8>*>(static_cast<H*>(base) + p * plane + off) = q;
    }
}

template <int V>
struct IntConst {
  static constexpr int value = V;
};

// Tile images in LDS.  Loads write LDS linearly (16 bytes a lane), so a permutation of the 16-byte
// chunks of a row, which spreads the fragment reads over the banks, is made on the global address.
//   k contiguous:    [rows][8 chunks], chunk ^ swz(row).  A: row & 7, fragments read 16 successive
//                    rows.  B: fragment rows are 4·NF apart in fours (see `nrow`), so row & 3 and the
//                    lowest bit of that distance.
//   rows contiguous: [64 k][ROWS / 8 chunks], chunk ^ (k & 3 | (k >> 3 & 3) << 2): the 16 k rows that
//                    a wave's transposed reads touch land on 16 different chunks.
template <int ROWS, bool T>
struct TileMap {
  static constexpr int kChunks = T ? ROWS / 8 : 8;               // per LDS row
  static constexpr int kRowsPerLoad = 64 / kChunks;
};
__device__ __forceinline__ int swz_t(int k) { return (k & 3) | ((k >> 3 & 3) << 2); }

// One block: a BM×BN tile of D (kEpiGate: BM×BN/2 of g and of u), WM×WN waves of 16×16×32 MFMAs, k in
// stages of kBK that travel from HBM straight into LDS through a ring of NS stages, NS − 1 of them in
// flight while one is multiplied; one barrier a stage.  Rows past an operand's
// edge and k past its end are outside the buffer descriptor and arrive as zeros.  The right
// operand's fragment is the first MFMA operand, and its fragment rows are chosen so that a lane ends
// with 4·NF consecutive n of one row m (nrow), which the epilogue moves 16 bytes at a time.
template <typename H, typename TO, int EPI, bool TA, bool TB, int BM, int BN, int WM, int WN, int NS>
__global__ __launch_bounds__(64 * WM * WN) void ffn_gemm_kernel(const GemmArgs a) {
  constexpr int kWaves = WM * WN, FM = BM / WM / 16, FN = BN / WN / 16;
  constexpr int NF = EPI == kEpiGate ? FN / 2 : FN;              // n fragments of one output
  constexpr int LA = BM / 8 / kWaves, LB = BN / 8 / kWaves;      // loads of a wave per stage
  constexpr int kNBit = NF == 4 ? 4 : 3;                         // log2(4·NF)
  static_assert(NF == 4 || NF == 2, "");
  __shared__ uint4 lds[NS][(BM + BN) * 8];
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
    const int r = (wave * LA + i) * TileMap<BM, TA>::kRowsPerLoad + lane / C, ch = (lane % C) ^ (TA ? swz_t(r) : r & 7);
    offA[i] = (unsigned)r * (unsigned)a.lda * 2 + ch * 16;
  }
#pragma unroll
  for (int i = 0; i < LB; i++) {
    constexpr int C = TileMap<BN, TB>::kChunks;
    int r = (wave * LB + i) * TileMap<BN, TB>::kRowsPerLoad + lane / C;
    const int ch = (lane % C) ^ (TB ? swz_t(r) : (r & 3) | ((r >> kNBit & 1) << 2));
    if (EPI == kEpiGate) r %= BN / 2;
    offB[i] = (unsigned)r * (unsigned)a.ldb * 2 + ch * 16;
  }
  // descriptor of an operand from its row r0 and the k of stage t on, to its end
  auto window = [&](const void* p, bool trans, int64_t ld, int64_t rows, int r0, int64_t k) {
    const int64_t first = trans ? k * ld + r0 : r0 * ld + k, all = (trans ? a.K : rows) * ld;
    int64_t left = (all - first) * 2;
    if (left < 0) left = 0;
    if (left > 0x7ffffff0) left = 0x7ffffff0;
    return descriptor(static_cast<const char*>(p) + first * 2, (uint32_t)left);
  };
  const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)&lds[0][0];
  auto stage = [&](int t, int buf) {
    const int p = t / a.ktiles;
    const int64_t k = (int64_t)(t - p * a.ktiles) * kBK;
    const i32x4 ra = window(batch ? a.A2[p] : a.A[p], TA, a.lda, a.M, m0, k);
    const i32x4 rb = window(a.B[p], TB, a.ldb, a.N, n0, k);
    const unsigned la = lds0 + buf * ((BM + BN) * 128) + wave * (LA * 1024);
    const unsigned lb = lds0 + buf * ((BM + BN) * 128) + BM * 128 + wave * (LB * 1024);
#pragma unroll
    for (int i = 0; i < LA; i++) load_to_lds(ra, la + i * 1024, offA[i]);
    if constexpr (EPI == kEpiGate) {
      const i32x4 rb2 = window(a.B2[p], TB, a.ldb, a.N, n0, k);
#pragma unroll
      for (int i = 0; i < LB; i++) load_to_lds((wave * LB + i) * 8 >= BN / 2 ? rb2 : rb, lb + i * 1024, offB[i]);
    } else {
#pragma unroll
      for (int i = 0; i < LB; i++) load_to_lds(rb, lb + i * 1024, offB[i]);
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
    return up + wn * (16 * NF) + (r >> 2) * (4 * NF) + (j % NF) * 4 + (r & 3);
  };
  auto frag_t = [&](const char* base, int rows, int ks, int col) {
    s16x4 half[2];
#pragma unroll
    for (int hb = 0; hb < 2; hb++) {
      const int k = ks * 32 + fk * 8 + hb * 4 + (fr >> 2);
      half[hb] = read_transposed(base + k * rows * 2 + (((col >> 3) ^ swz_t(k)) << 4) + (col & 4) * 2);
    }
    return __builtin_bit_cast(bf16x8, (s16x8)__builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7));
  };
  auto compute = [&](int buf) {
    const uint4* la = lds[buf];
    const uint4* lb = lds[buf] + BM * 8;
#pragma unroll
    for (int ks = 0; ks < kBK / 32; ks++) {
      bf16x8 fa[FM], fb[FN];
#pragma unroll
      for (int i = 0; i < FM; i++) {
        const int r0 = wm * (BM / WM) + i * 16;
        if constexpr (TA) fa[i] = frag_t(reinterpret_cast<const char*>(la), BM, ks, r0 + (fr & 3) * 4);
        else fa[i] = __builtin_bit_cast(bf16x8, la[(r0 + fr) * 8 + ((ks * 4 + fk) ^ (fr & 7))]);
      }
#pragma unroll
      for (int j = 0; j < FN; j++) {
        if constexpr (TB) {
          fb[j] = frag_t(reinterpret_cast<const char*>(lb), BN, ks, nrow(j, (fr & 3) * 4));
        } else {
          const int r = nrow(j, fr);
          fb[j] = __builtin_bit_cast(bf16x8, lb[r * 8 + ((ks * 4 + fk) ^ ((r & 3) | ((r >> kNBit & 1) << 2)))]);
        }
      }
#pragma unroll
      for (int i = 0; i < FM; i++)
#pragma unroll
        for (int j = 0; j < FN; j++) acc[i][j] = mfma16<H>(fb[j], fa[i], acc[i][j]);
    }
  };

  // iteration kt: stage kt has landed for every wave, and every wave is done with stage kt − 1, whose
  // slot takes stage kt + NS − 1
  int put = 0, get = 0;
#pragma unroll
  for (int i = 0; i < NS - 1; i++)
    if (kt + i < kend) stage(kt + i, put++);
  for (; kt < kend; kt++) {
    if (kt + NS - 2 < kend) wait_and_barrier<(NS - 2) * (LA + LB)>();
    else wait_and_barrier<0>();
    if (kt + NS - 1 < kend) {
      stage(kt + NS - 1, put);
      put = put + 1 == NS ? 0 : put + 1;
    }
    compute(get);
    get = get + 1 == NS ? 0 : get + 1;
  }

  // ---- epilogue: lane holds n = nb … nb + 4·NF − 1 of the rows m = … + i·16 + fr ----------------
  const int nb = n0 + wn * (16 * NF) + fk * (4 * NF), mb = m0 + wm * (BM / WM) + fr;
  const bool vec = (a.N & 7) == 0;
  if constexpr (EPI == kEpiStore) {
#pragma unroll
    for (int j = 0; j < NF; j += 2) {
      const int n = nb + j * 4;
      float b[8];
      load8<TO>(static_cast<const TO*>(a.bias), n, a.bias && !a.partial ? a.N : 0, false, b);
#pragma unroll
      for (int i = 0; i < FM; i++) {
        const int m = mb + i * 16;
        float v[8];
#pragma unroll
        for (int q = 0; q < 8; q++) v[q] = acc[i][j + q / 4][q % 4] + b[q];
        if (m < a.M) {
          if (a.partial) store8<float>(a.partial + (((int64_t)batch * a.splits + split) * a.M + m) * a.N, n, a.N, vec, v);
          else store8<TO>(static_cast<TO*>(batch ? a.out2 : a.out) + (int64_t)m * a.N, n, a.N, vec, v);
        }
      }
    }
  } else if constexpr (EPI == kEpiGate) {
    const int64_t arr = (int64_t)a.M * a.N;
#pragma unroll
    for (int j = 0; j < NF; j += 2) {
      const int n = nb + j * 4;
      float bg[8], bu[8];
      load8<TO>(static_cast<const TO*>(a.bias_g), n, a.bias_g ? a.N : 0, false, bg);
      load8<TO>(static_cast<const TO*>(a.bias_u), n, a.bias_u ? a.N : 0, false, bu);
#pragma unroll
      for (int i = 0; i < FM; i++)
#pragma unroll
        for (int q = 0; q < 8; q++) {
          acc[i][j + q / 4][q % 4] += bg[q];
          acc[i][j + NF + q / 4][q % 4] += bu[q];
        }
    }
    auto finish = [&](auto act) {                                // one unrolled body per activation
#pragma unroll
      for (int i = 0; i < FM; i++) {
        const int m = mb + i * 16;
#pragma unroll
        for (int j = 0; j < NF; j += 2) {
          const int n = nb + j * 4;
          float h[8], du[8], f[8];
#pragma unroll
          for (int q = 0; q < 8; q++) {
            const float g = acc[i][j + q / 4][q % 4], u = acc[i][j + NF + q / 4][q % 4];
            float df;
            gate_act_pair(g, decltype(act)::value, f[q], df);
            h[q] = n + q < a.N ? f[q] * u : 0.f;
            du[q] = df * u;
          }
          if (m < a.M) {
            if (a.kept) {
              TO* k = static_cast<TO*>(a.kept) + (int64_t)m * a.N;
              store8<TO>(k, n, a.N, vec, h);
              store8<TO>(k + arr, n, a.N, vec, du);
              store8<TO>(k + 2 * arr, n, a.N, vec, f);
            }
            if (a.h && n < a.ldf) store_planes8<H>(a.h, (int64_t)m * a.ldf + n, (int64_t)a.M * a.ldf, a.planes, h);
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
    const TO* k = static_cast<const TO*>(a.kept) + (int64_t)a.M * a.N;
    const int64_t arr = (int64_t)a.M * a.N, plane = (int64_t)a.M * a.ldf;
#pragma unroll
    for (int i = 0; i < FM; i++) {
      const int m = mb + i * 16;
#pragma unroll
      for (int j = 0; j < NF; j += 2) {
        const int n = nb + j * 4;
        if (m < a.M && n < a.ldf) {
          float du[8], f[8];
          load8<TO>(k + (int64_t)m * a.N, n, a.N, vec, du);      // zeros past N: so are dg and du there
          load8<TO>(k + arr + (int64_t)m * a.N, n, a.N, vec, f);
#pragma unroll
          for (int q = 0; q < 8; q++) {
            const float dh = n + q < a.N ? acc[i][j + q / 4][q % 4] : 0.f;
            du[q] *= dh;
            f[q] *= dh;
          }
          store_planes8<H>(a.dg, (int64_t)m * a.ldf + n, plane, a.planes, du);
          store_planes8<H>(a.du, (int64_t)m * a.ldf + n, plane, a.planes, f);
        }
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
  int bm, tiles_m, tiles_n, splits, per_split;
};
// 256×256 tiles where they give each of the 256 CUs one, else 128×128 (two blocks a CU); a product
// of fewer tiles than CUs splits k into runs of at least 4 stages, up to about two blocks a CU.
Tiling tile(int64_t M, int64_t N, int batches, int stages, bool gate, bool may_split) {
  Tiling t{};
  const int64_t big = ((M + 255) / 256) * ((N * (gate ? 2 : 1) + 255) / 256) * batches;
  t.bm = big >= 224 ? 256 : 128;
  t.tiles_m = (int)((M + t.bm - 1) / t.bm);
  t.tiles_n = (int)((N + (gate ? t.bm / 2 : t.bm) - 1) / (gate ? t.bm / 2 : t.bm));
  t.splits = 1;
  const int64_t tiles = (int64_t)t.tiles_m * t.tiles_n * batches;
  if (may_split && tiles < 256) {
    int64_t s = 512 / tiles;
    if (s > stages / 4) s = stages / 4;
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
unsigned grid_of(int64_t items) {
  const int64_t b = (items + 255) / 256;
  return (unsigned)(b < 8192 ? b : 8192);
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

  int npairs() const { return planes * (planes + 1) / 2; }
  Operand planes_of(int64_t rows, int64_t cols) {
    Operand o;
    o.rows = rows;
    o.ld = round_k(cols);
    o.p = static_cast<const char*>(ws.take((size_t)planes * rows * o.ld * 2));
    return o;
  }

  // `src` [R][K] in product form: itself where its rows are whole stages (k contiguous) or whole
  // 16-byte chunks (k the slow axis), else packed into the workspace
  int operand(const void* src, int64_t R, int64_t K, bool k_slow, Operand& o) {
    if (!mode.pack && K % (k_slow ? 8 : kBK) == 0) {
      o.p = static_cast<const char*>(src), o.rows = R, o.ld = K;
      return kOk;
    }
    o = planes_of(R, K);
    if (dry) return kOk;
    ffn_pack_kernel<TO, H><<<grid_of(R * o.ld / 4), 256, 0, st>>>(static_cast<const TO*>(src), R, K, planes,
                                                                  reinterpret_cast<H*>(const_cast<char*>(o.p)), o.ld);
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
    a.ktiles = (int)(round_k(K) / kBK);
    a.batches = A2 ? 2 : 1;
  }

  template <int EPI, bool TA, bool TB>
  int gemm(GemmArgs& a, const Tiling& t, void* partial) {
    a.tiles_m = t.tiles_m, a.tiles_n = t.tiles_n, a.splits = t.splits, a.per_split = t.per_split;
    a.partial = t.splits > 1 ? static_cast<float*>(partial) : nullptr;
    const unsigned grid = (unsigned)t.tiles_m * t.tiles_n * t.splits * a.batches;
    if (t.bm == 256) ffn_gemm_kernel<H, TO, EPI, TA, TB, 256, 256, 2, 4, 2><<<grid, 512, 0, st>>>(a);
    else if (grid >= 512) ffn_gemm_kernel<H, TO, EPI, TA, TB, 128, 128, 2, 2, 2><<<grid, 256, 0, st>>>(a);
    else ffn_gemm_kernel<H, TO, EPI, TA, TB, 128, 128, 2, 2, 4><<<grid, 256, 0, st>>>(a);
    if (int rc = check_launch(EPI == kEpiStore ? "ffn_gemm" : EPI == kEpiGate ? "ffn_gemm_gate" : "ffn_gemm_gate_bwd")) return rc;
    if (t.splits > 1) {
      const int64_t total = (int64_t)a.M * a.N;
      for (int b = 0; b < a.batches; b++) {
        ffn_reduce_kernel<TO><<<grid_of(total), 256, 0, st>>>(a.partial + b * t.splits * total, t.splits, total, a.N,
                                                              static_cast<const TO*>(a.bias),
                                                              static_cast<TO*>(b ? a.out2 : a.out));
        if (int rc = check_launch("ffn_reduce")) return rc;
      }
    }
    return kOk;
  }

  // h (planes) and / or kept of all rows
  int gate(const Operand& h, void* kept) {
    Operand x, wg, wu;
    if (int rc = operand(f.x, f.M, f.C, false, x)) return rc;
    if (int rc = operand(f.wg, f.F, f.C, false, wg)) return rc;
    if (int rc = operand(f.wu, f.F, f.C, false, wu)) return rc;
    if (dry) return kOk;
    GemmArgs a{};
    pairs(a, x, nullptr, wg, &wu, f.C);
    a.M = (int)f.M, a.N = f.F;
    a.bias_g = f.bg, a.bias_u = f.bu, a.act = f.act, a.planes = planes;
    a.kept = kept;
    a.h = const_cast<char*>(h.p), a.ldf = h.ld;
    return gemm<kEpiGate, false, false>(a, tile(f.M, f.F, 1, a.pairs * a.ktiles, true, false), nullptr);
  }

  int forward(void* y, void* kept) {
    Operand h = planes_of(f.M, f.F), wd;
    if (int rc = gate(h, kept)) return rc;
    if (int rc = operand(f.wd, f.O, f.F, false, wd)) return rc;
    const Tiling t = tile(f.M, f.O, 1, npairs() * (int)(h.ld / kBK), false, true);
    void* partial = ws.take(partial_bytes(t, f.M, f.O, 1));
    if (dry) return kOk;
    GemmArgs a{};
    pairs(a, h, nullptr, wd, nullptr, f.F);
    a.M = (int)f.M, a.N = f.O;
    a.out = y, a.bias = f.bd;
    return gemm<kEpiStore, false, false>(a, t, partial);
  }

  int column_sums(const Operand& o, int cols, void* out) {
    const int64_t per = (o.rows + kColChunks - 1) / kColChunks, chunks = (o.rows + per - 1) / per;
    float* part = static_cast<float*>(ws.take((size_t)chunks * cols * sizeof(float)));
    if (dry) return kOk;
    ffn_col_sum_kernel<H><<<dim3(ceil_div(cols, 256), (unsigned)chunks), 256, 0, st>>>(reinterpret_cast<const H*>(o.p), o.rows, cols,
                                                                                       o.ld, planes, per, part);
    if (int rc = check_launch("ffn_col_sum")) return rc;
    ffn_reduce_kernel<TO><<<grid_of(cols), 256, 0, st>>>(part, (int)chunks, cols, cols, static_cast<const TO*>(nullptr),
                                                         static_cast<TO*>(out));
    return check_launch("ffn_reduce");
  }

  int backward(const void* dy, const void* kept, const FfnGrads& o) {
    if (!kept) {                                             // recomputed
      void* k = ws.take((size_t)3 * f.M * f.F * sizeof(TO));
      if (int rc = gate(Operand{}, k)) return rc;
      kept = k;
    }
    const bool inner = o.dx || o.dwg || o.dwu || o.dbg || o.dbu;
    Operand dg, du;
    if (inner) {
      Operand dyo, wd;
      dg = planes_of(f.M, f.F), du = planes_of(f.M, f.F);
      if (int rc = operand(dy, f.M, f.O, false, dyo)) return rc;
      if (int rc = operand(f.wd, f.O, f.F, true, wd)) return rc;
      if (!dry) {
        GemmArgs a{};
        pairs(a, dyo, nullptr, wd, nullptr, f.O);
        a.M = (int)f.M, a.N = f.F;
        a.planes = planes, a.kept = const_cast<void*>(kept);
        a.dg = const_cast<char*>(dg.p), a.du = const_cast<char*>(du.p), a.ldf = dg.ld;
        if (int rc = gemm<kEpiGateBwd, false, true>(a, tile(f.M, f.F, 1, a.pairs * a.ktiles, false, false), nullptr)) return rc;
      }
    }
    if (o.dx) {
      Operand wg, wu;
      if (int rc = operand(f.wg, f.F, f.C, true, wg)) return rc;
      if (int rc = operand(f.wu, f.F, f.C, true, wu)) return rc;
      const Tiling t = tile(f.M, f.C, 1, 2 * npairs() * (int)(dg.ld / kBK), false, true);
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
    if (o.dwg || o.dwu) {
      Operand x;
      if (int rc = operand(f.x, f.M, f.C, true, x)) return rc;
      const int both = o.dwg && o.dwu ? 2 : 1;
      const Tiling t = tile(f.F, f.C, both, npairs() * (int)(round_k(f.M) / kBK), false, true);
      void* partial = ws.take(partial_bytes(t, f.F, f.C, both));
      if (!dry) {
        GemmArgs a{};
        pairs(a, o.dwg ? dg : du, both == 2 ? &du : nullptr, x, nullptr, f.M);
        a.M = f.F, a.N = f.C;
        a.out = o.dwg ? o.dwg : o.dwu, a.out2 = o.dwu;
        if (int rc = gemm<kEpiStore, true, true>(a, t, partial)) return rc;
      }
    }
    if (o.dbg)
      if (int rc = column_sums(dg, f.F, o.dbg)) return rc;
    if (o.dbu)
      if (int rc = column_sums(du, f.F, o.dbu)) return rc;
    if (o.dwd || o.dbd) {
      Operand dyo;
      if (int rc = operand(dy, f.M, f.O, true, dyo)) return rc;
      if (o.dwd) {
        Operand h;
        if (int rc = operand(kept, f.M, f.F, true, h)) return rc;
        const Tiling t = tile(f.O, f.F, 1, npairs() * (int)(round_k(f.M) / kBK), false, true);
        void* partial = ws.take(partial_bytes(t, f.O, f.F, 1));
        if (!dry) {
          GemmArgs a{};
          pairs(a, dyo, nullptr, h, nullptr, f.M);
          a.M = f.O, a.N = f.F;
          a.out = o.dwd;
          if (int rc = gemm<kEpiStore, true, true>(a, t, partial)) return rc;
        }
      }
      if (o.dbd)
        if (int rc = column_sums(dyo, f.O, o.dbd)) return rc;
    }
    return kOk;
  }
};

template <typename H, typename TO>
size_t ffn_ws(const FfnArgs& f, Mode mode, int backward, int recompute) {
  static char any;
  Ffn<H, TO> r(f, mode, nullptr, nullptr);
  if (backward) r.backward(&any, recompute ? nullptr : &any, FfnGrads{&any, &any, &any, &any, &any, &any, &any});
  else r.forward(&any, nullptr);
  return r.ws.used;
}

}  // namespace

// Entry points of one (plane type, tensor type): each is instantiated in a file of its own.
#define MRAGAN_FFN_ENTRIES(name, H, TO)                                                                                       \
  size_t ffn_ws_##name(const FfnArgs& f, int planes, int pack, int backward, int recompute) {                                 \
    return ffn_ws<H, TO>(f, Mode{planes, pack != 0}, backward, recompute);                                                    \
  }                                                                                                                           \
  int ffn_fwd_##name(const FfnArgs& f, int planes, int pack, void* y, void* kept, void* ws, hipStream_t st) {                 \
    return Ffn<H, TO>(f, Mode{planes, pack != 0}, ws, st).forward(y, kept);                                                   \
  }                                                                                                                           \
  int ffn_bwd_##name(const FfnArgs& f, int planes, int pack, const void* dy, const void* kept, const FfnGrads& o, void* ws,   \
                     hipStream_t st) {                                                                                        \
    return Ffn<H, TO>(f, Mode{planes, pack != 0}, ws, st).backward(dy, kept, o);                                              \
  }

}  // namespace mragan
