// Vectors of elements as the operators around the linears read and write them: any element-aligned
// address (gfx950 serves unaligned vector accesses), f32 values inside.
#pragma once
#include "common.h"

namespace reels {

// T<ELT>: the stored type of an element code and its conversions
template <int ELT> struct Store;
template <> struct Store<REELS_HIP_F32> {
  typedef uint32_t raw;
  static __device__ __forceinline__ float get(raw v) { return __uint_as_float(v); }
  static __device__ __forceinline__ raw put(float f) { return __float_as_uint(f); }
};
template <> struct Store<REELS_HIP_BF16> {
  typedef uint16_t raw;
  static __device__ __forceinline__ float get(raw v) { return bf16_to_f32(v); }
  // v_cvt_pk_bf16_f32: nearest even, NaN stays NaN (the integer formula of common.h carries a NaN
  // of small payload into an infinity)
  static __device__ __forceinline__ raw put(float f) { return __builtin_bit_cast(uint16_t, (__bf16)f); }
};
template <> struct Store<REELS_HIP_F16> {
  typedef uint16_t raw;
  static __device__ __forceinline__ float get(raw v) { return (float)__builtin_bit_cast(_Float16, v); }
  static __device__ __forceinline__ raw put(float f) { return __builtin_bit_cast(uint16_t, (_Float16)f); }
};

constexpr int elt_bytes(int elt) { return elt == REELS_HIP_F32 ? 4 : 2; }

// a T at any address that its elements are aligned to
template <typename T> __device__ __forceinline__ T load_any(const void* p) {
  T v;
  __builtin_memcpy(&v, p, sizeof(T));
  return v;
}
template <typename T> __device__ __forceinline__ void store_any(void* p, const T& v) { __builtin_memcpy(p, &v, sizeof(T)); }

// V elements at p, the first `left` of which exist (zeros past them)
template <int ELT, int V> __device__ __forceinline__ void load_vec(const void* p, int left, float (&f)[V]) {
  typedef typename Store<ELT>::raw raw;
  struct Pack { raw e[V]; };
  const raw* r = reinterpret_cast<const raw*>(p);
  if (left >= V) {
    const Pack v = load_any<Pack>(r);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = Store<ELT>::get(v.e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = i < left ? Store<ELT>::get(r[i]) : 0.0f;
  }
}

template <int ELT, int V> __device__ __forceinline__ void store_vec(void* p, int left, const float (&f)[V]) {
  typedef typename Store<ELT>::raw raw;
  struct Pack { raw e[V]; };
  raw* r = reinterpret_cast<raw*>(p);
  if (left >= V) {
    Pack v;
#pragma unroll
    for (int i = 0; i < V; ++i) v.e[i] = Store<ELT>::put(f[i]);
    store_any(r, v);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < left) r[i] = Store<ELT>::put(f[i]);
  }
}

// calls f(std::integral_constant<int, ELT>) for a checked element code
template <typename F> inline void with_any_elt(int elt, F&& f) {
  if (elt == REELS_HIP_F32) f(std::integral_constant<int, REELS_HIP_F32>{});
  else if (elt == REELS_HIP_F16) f(std::integral_constant<int, REELS_HIP_F16>{});
  else f(std::integral_constant<int, REELS_HIP_BF16>{});
}
inline bool known_elt(int elt) { return elt == REELS_HIP_F32 || elt == REELS_HIP_BF16 || elt == REELS_HIP_F16; }

// sum and maximum over groups of G lanes (a power of two up to 64), every lane gets the result
template <int G> __device__ __forceinline__ double group_sum(double v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
template <int G> __device__ __forceinline__ double group_max(double v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v = fmax(v, __shfl_xor(v, o, 64));
  return v;
}

}  // namespace reels
