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

// 16 bytes of elements as they are stored, for kernels that keep a row in registers: unpacked at each
// use (one operation an element or less), which takes half the registers of the f32 values
template <int ELT> struct Chunk {
  static constexpr int V = 16 / elt_bytes(ELT);
  u32x4 d;
  __device__ __forceinline__ float get(int i) const {
    if constexpr (ELT == REELS_HIP_F32) return __uint_as_float(d[i]);
    else return (i & 1) ? Elt<ELT>::hi(d[i / 2]) : Elt<ELT>::lo(d[i / 2]);
  }
  __device__ __forceinline__ void unpack(float (&f)[V]) const {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = get(i);
  }
  __device__ __forceinline__ void pack(const float (&f)[V]) {
    if constexpr (ELT == REELS_HIP_F32) {
#pragma unroll
      for (int i = 0; i < V; ++i) d[i] = __float_as_uint(f[i]);
    } else {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) d[i] = Elt<ELT>::pack2_fast(f[2 * i], f[2 * i + 1]);
    }
  }
  // the first `left` elements at p, zeros past them
  __device__ __forceinline__ void load(const void* p, int left) {
    if (left >= V) {
      d = load_any<u32x4>((const typename Store<ELT>::raw*)p);
    } else {
      float f[V];
      load_vec<ELT, V>(p, left, f);
      pack(f);
    }
  }
  __device__ __forceinline__ void store(void* p, int left) const {
    if (left >= V) {
      store_any((typename Store<ELT>::raw*)p, d);
    } else {
      float f[V];
      unpack(f);
      store_vec<ELT, V>(p, left, f);
    }
  }
  __device__ __forceinline__ void zero() { d = u32x4{0u, 0u, 0u, 0u}; }
  // values unpacked before this are not kept for the uses after it
  __device__ __forceinline__ void hold() { asm volatile("" : "+v"(d)); }
};

// calls f(std::integral_constant<int, ELT>) for a checked element code
template <typename F> inline void with_any_elt(int elt, F&& f) {
  if (elt == REELS_HIP_F32) f(std::integral_constant<int, REELS_HIP_F32>{});
  else if (elt == REELS_HIP_F16) f(std::integral_constant<int, REELS_HIP_F16>{});
  else f(std::integral_constant<int, REELS_HIP_BF16>{});
}
// A launch holds less than 2^32 threads
inline bool grid_fits(int64_t blocks, int threads) { return blocks < ((int64_t)1 << 32) / threads; }
inline bool known_elt(int elt) { return elt == REELS_HIP_F32 || elt == REELS_HIP_BF16 || elt == REELS_HIP_F16; }

// Sum or maximum over groups of G lanes (16 or 64, all of them active), the same bits in every lane:
// within 16 lanes by DPP, then by lane swaps, both cheaper than a trip through the LDS crossbar.
// a + b == b + a, so the lanes' different orders do not show.
template <int CTRL> __device__ __forceinline__ double dpp_move(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xf, 0xf, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xf, 0xf, true);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <bool MAX> __device__ __forceinline__ double join(double a, double b) { return MAX ? fmax(a, b) : a + b; }
template <int G, bool MAX> __device__ __forceinline__ double group_reduce(double v) {
  static_assert(G == 16 || G == 64, "");
  v = join<MAX>(v, dpp_move<0xB1>(v));   // lanes l ^ 1
  v = join<MAX>(v, dpp_move<0x4E>(v));   // l ^ 2
  v = join<MAX>(v, dpp_move<0x141>(v));  // the other four of eight
  v = join<MAX>(v, dpp_move<0x140>(v));  // the other eight of sixteen
  if constexpr (G == 64) {
    uint64_t u = __builtin_bit_cast(uint64_t, v);
    const auto l16 = __builtin_amdgcn_permlane16_swap((uint32_t)u, (uint32_t)u, false, false);
    const auto h16 = __builtin_amdgcn_permlane16_swap((uint32_t)(u >> 32), (uint32_t)(u >> 32), false, false);
    v = join<MAX>(__builtin_bit_cast(double, (uint64_t)h16[0] << 32 | l16[0]), __builtin_bit_cast(double, (uint64_t)h16[1] << 32 | l16[1]));
    u = __builtin_bit_cast(uint64_t, v);
    const auto l32 = __builtin_amdgcn_permlane32_swap((uint32_t)u, (uint32_t)u, false, false);
    const auto h32 = __builtin_amdgcn_permlane32_swap((uint32_t)(u >> 32), (uint32_t)(u >> 32), false, false);
    v = join<MAX>(__builtin_bit_cast(double, (uint64_t)h32[0] << 32 | l32[0]), __builtin_bit_cast(double, (uint64_t)h32[1] << 32 | l32[1]));
  }
  return v;
}

// 1 / sqrt(x) and 1 / x in 64 bits: the hardware's estimate and two Newton steps (0, infinity and NaN
// as the estimate has them)
__device__ __forceinline__ double rsqrt64(double x) {
  const double y0 = __builtin_amdgcn_rsq(x);
  double y = y0;
#pragma unroll
  for (int i = 0; i < 2; ++i) y = fma(y * 0.5, fma(-x * y, y, 1.0), y);
  return __builtin_isfinite(y) ? y : y0;
}
__device__ __forceinline__ double rcp64(double x) {
  const double y0 = __builtin_amdgcn_rcp(x);
  double y = y0;
#pragma unroll
  for (int i = 0; i < 2; ++i) y = fma(y, fma(-x, y, 1.0), y);
  return __builtin_isfinite(y) ? y : y0;
}

}  // namespace reels
