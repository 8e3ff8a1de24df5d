// Shared by the token-block kernels (layer norm, gated feed-forward, linear recurrence): the
// element types, vector loads and stores between them and fp32, and wave reductions.
#pragma once
#include "common.h"

namespace mragan {

enum DType : int { kF32 = 0, kBF16 = 1, kF16 = 2 };
inline size_t dtype_size(int dt) { return dt == kF32 ? 4 : 2; }
inline bool dtype_ok(int dt) { return dt == kF32 || dt == kBF16 || dt == kF16; }

// n elements of T moved as one access
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};

template <typename T, int N>
__device__ __forceinline__ void load_vec(const T* p, float (&out)[N]) {
  const Pack<T, N> r = *reinterpret_cast<const Pack<T, N>*>(p);
#pragma unroll
  for (int i = 0; i < N; i++) out[i] = (float)r.v[i];
}
// the one rounding of a result to its tensor's type (RNE)
template <typename T, int N>
__device__ __forceinline__ void store_vec(T* p, const float (&in)[N]) {
  Pack<T, N> r;
#pragma unroll
  for (int i = 0; i < N; i++) r.v[i] = (T)in[i];
  *reinterpret_cast<Pack<T, N>*>(p) = r;
}

// N elements of T held as the 32-bit words they were loaded as (16-bit elements kept apart would take a
// register each while they wait), read element by element
template <typename T, int N>
struct Words {
  static_assert(sizeof(T) * N % 4 == 0, "");
  uint32_t w[sizeof(T) * N / 4];
  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 4) {
      return __builtin_bit_cast(float, w[i]);
    } else if constexpr (__is_same(T, __bf16)) {
      return __builtin_bit_cast(float, i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    } else {
      return (float)__builtin_bit_cast(T, (uint16_t)(w[i / 2] >> (i & 1) * 16));
    }
  }
  __device__ __forceinline__ void set(int i, float v) {           // rounds to T; elements in order from 0
    if constexpr (sizeof(T) == 4) {
      w[i] = __builtin_bit_cast(uint32_t, v);
    } else {
      const uint32_t b = __builtin_bit_cast(uint16_t, (T)v);
      w[i / 2] = i & 1 ? w[i / 2] | b << 16 : b;
    }
  }
};

// a·b + c with one rounding
__device__ __forceinline__ float fma(float a, float b, float c) { return __builtin_fmaf(a, b, c); }

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xF, 0xF, false));
}
// Sum over aligned groups of G lanes (G a power of two ≤ 64), the same value in every lane of the
// group: DPP inside 16 lanes, the gfx950 permlane swaps across them (no LDS round trip).  Each step
// adds two equal spans, so the order of the additions is a fixed tree.
template <int G>
__device__ __forceinline__ float group_sum(float v) {
  if constexpr (G >= 2) v += dpp<0xB1>(v);    // lane ^ 1
  if constexpr (G >= 4) v += dpp<0x4E>(v);    // lane ^ 2
  if constexpr (G >= 8) v += dpp<0x141>(v);   // mirror in 8 lanes: the other quad
  if constexpr (G >= 16) v += dpp<0x140>(v);  // mirror in 16 lanes: the other 8
  if constexpr (G >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    v = __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
  }
  if constexpr (G >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    v = __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
  }
  return v;
}

// logistic function of d and of −d, exact at ±inf (1 and 0), without overflow: exp of −|d| only
__device__ __forceinline__ void sigmoid_pair(float d, float& s, float& s_neg) {
  const float e = __expf(-fabsf(d));
  const float r = __builtin_amdgcn_rcpf(1.f + e), er = e * r;
  s = d >= 0.f ? r : er;
  s_neg = d >= 0.f ? er : r;
}

inline bool aligned_to(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// run the statement block with the type of `dt` as T
#define MRAGAN_DTYPE_DISPATCH(dt, T, ...)     \
  switch (dt) {                               \
    case ::mragan::kBF16: {                   \
      using T = __bf16;                       \
      __VA_ARGS__;                            \
      break;                                  \
    }                                         \
    case ::mragan::kF16: {                    \
      using T = _Float16;                     \
      __VA_ARGS__;                            \
      break;                                  \
    }                                         \
    default: {                                \
      using T = float;                        \
      __VA_ARGS__;                            \
      break;                                  \
    }                                         \
  }

}  // namespace mragan
