// Microscaled blocks: 32 neighbours of a row share one power of two, kept as its exponent + 127 in a byte
// (0: 2^-127; 255: the block holds NaN or an infinity, and all of its values are NaN).
//
// 8 bits (activations kept for the backward): a value is code * 2^(E - 6), code in -127 .. 127; codes dense
//   [rows][cols], bytes [rows][ceil(cols / 32)].
// 4 bits (operands of the 4-bit product): a value is one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign, times
//   2^E; codes [rows][Kp / 2], Kp = cols up to a multiple of 256, the even column in the low half of a byte,
//   zeros past cols; bytes in tiles of 64 rows x 8 blocks, in the order in which a wave's lanes take them
//   (mx4_scale_at).
//
// E is the exponent of the block's largest magnitude after that is rounded to the significand a code has
// (7 bits, or 2): so the largest value is off by at most half a step like every other, and no code
// saturates, except at the end of the f32 range, where E stops at 127 (8 bits) and 125 (4 bits: 6 * 2^126
// is no f32 value). x 2^-E is exact, so codes are the nearest ones, ties to even, in 32-bit arithmetic.
#pragma once
#include "vec.h"

namespace reels {

constexpr int kMxBlock = 32;

// the byte of a block whose largest magnitude has these bits (NaN and infinities are the largest)
template <int BITS> __device__ __forceinline__ uint32_t mx_exponent(uint32_t top) {
  constexpr int DOWN = BITS == 2 ? 2 : 0, MOST = BITS == 2 ? 252 : 254;
  if (top >= 0x7f800000u) return 255u;
  const int e = (int)((top + (1u << (23 - BITS))) >> 23) - DOWN;
  return (uint32_t)(e < 0 ? 0 : e > MOST ? MOST : e);
}

// the largest of N lanes' values (4 or 8 neighbours, all lanes active)
template <int N> __device__ __forceinline__ uint32_t mx_top(uint32_t v) {
  static_assert(N == 4 || N == 8, "");
  auto up = [&](uint32_t o) { v = v > o ? v : o; };
  up((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true));   // lanes l ^ 1
  up((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true));   // l ^ 2
  if constexpr (N == 8) up((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, true));  // the other four of eight
  return v;
}
// the largest magnitude of V values (v_maximum3: NaN stays)
template <int V> __device__ __forceinline__ uint32_t mx_top_of(const float (&f)[V]) {
  float t = fabsf(f[0]);
#pragma unroll
  for (int j = 1; j < V; j += 2) t = __builtin_elementwise_maximum(t, __builtin_elementwise_maximum(fabsf(f[j]), fabsf(f[j + 1 < V ? j + 1 : j])));
  return __float_as_uint(t);
}

// ---- 8 bits --------------------------------------------------------------------------------------
// V codes in V / 4 words. Adding 1.5 * 2^23 rounds to a whole number, ties to even, and leaves it in the
// low byte.
template <int V> __device__ __forceinline__ void mx8_codes(const float (&f)[V], uint32_t byte, uint32_t (&word)[V / 4]) {
  uint32_t c[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const float t = __builtin_amdgcn_fmed3f(__builtin_amdgcn_ldexpf(f[j], 133 - (int)byte), -127.0f, 127.0f);
    c[j] = __float_as_uint(t + 12582912.0f);
  }
#pragma unroll
  for (int i = 0; i < V / 4; ++i) {
    const uint32_t lo = __builtin_amdgcn_perm(c[4 * i + 1], c[4 * i], 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(c[4 * i + 3], c[4 * i + 2], 0x04000c0cu);
    word[i] = byte == 255u ? 0u : lo | hi;
  }
}
// 2^(E - 6), NaN for 255 (an f32 value, subnormal for the smallest)
__device__ __forceinline__ float mx8_unit(uint32_t byte) {
  return byte == 255u ? __builtin_nanf("") : __builtin_amdgcn_ldexpf(1.0f, (int)byte - 133);
}

// V codes at p, the first `left` of which exist; the row has cols codes: a part of V is its last V codes
// shifted down
template <int V> struct Codes {
  uint32_t d[V / 4];
  float unit;
  __device__ __forceinline__ float get(int j) const { return (float)(int8_t)(d[j / 4] >> (8 * (j % 4))) * unit; }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) d[i] = 0u;
    unit = 0.0f;
  }
  __device__ __forceinline__ void shift_down(int by) {  // by whole codes
    if constexpr (V == 8) {
      const uint64_t u = (((uint64_t)d[1] << 32) | d[0]) >> (8 * by);
      d[0] = (uint32_t)u;
      d[1] = (uint32_t)(u >> 32);
    } else {
      d[0] >>= 8 * by;
    }
  }
  __device__ __forceinline__ void load(const int8_t* p, int left, int cols) {
    struct Pack { uint32_t w[V / 4]; };
    if (left >= V) {
      const Pack k = load_any<Pack>(p);
#pragma unroll
      for (int i = 0; i < V / 4; ++i) d[i] = k.w[i];
    } else if (cols >= V) {
      const Pack k = load_any<Pack>(p + left - V);
#pragma unroll
      for (int i = 0; i < V / 4; ++i) d[i] = k.w[i];
      shift_down(V - left);
    } else {
#pragma unroll
      for (int i = 0; i < V / 4; ++i) d[i] = 0u;
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (j < left) d[j / 4] |= (uint32_t)(uint8_t)p[j] << (8 * (j % 4));
    }
  }
};

template <int V> __device__ __forceinline__ void mx8_store(int8_t* q, int left, const uint32_t (&word)[V / 4]) {
  struct Pack { uint32_t w[V / 4]; };
  if (left >= V) {
    Pack p;
#pragma unroll
    for (int i = 0; i < V / 4; ++i) p.w[i] = word[i];
    store_any(q, p);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < left) q[j] = (int8_t)(word[j / 4] >> (8 * (j % 4)));
  }
}

// ---- 4 bits --------------------------------------------------------------------------------------
__device__ __forceinline__ float mx4_unit(uint32_t byte) {
  return byte == 255u ? __builtin_nanf("") : byte == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23);
}
// V codes, V / 8 words (V = 4: the low half of one). v_cvt_scalef32_pk_fp4_f32 divides by the scale and
// rounds to the nearest value, ties to the even code, saturating at 6.
template <int V> __device__ __forceinline__ uint32_t mx4_codes(const float (&f)[V], uint32_t byte) {
  static_assert(V == 4 || V == 8, "");
  const float unit = byte == 255u ? 1.0f : mx4_unit(byte);
  uint32_t w = 0u;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[0], f[1], unit, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[2], f[3], unit, 1);
  if constexpr (V == 8) {
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[4], f[5], unit, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[6], f[7], unit, 3);
  }
  return byte == 255u ? 0u : w;
}
// where the byte of a block stands; tiles: of blocks, Kp / 256
__device__ __forceinline__ int64_t mx4_scale_at(int64_t row, int block, int tiles) {
  return ((row >> 6) * tiles + (block >> 3)) * 512 + ((block & 1) * 32 + (int)(row & 31)) * 8 + ((block >> 1) & 3) * 2 + (int)((row >> 5) & 1);
}

}  // namespace reels
