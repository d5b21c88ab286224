// Rows of a matrix in registers, as the root-mean-square norm holds them (norm.hip; the modulated norm has its
// own form, modnorm.h, whose threads walk several rows): a group of TPR threads has a row, NCH chunks of 16 bytes
// each.
#pragma once
#include "vec.h"

namespace reels {
namespace {

// sum (or maximum) over the TPR threads of a row's group; slot: per-block LDS, one per wave
template <int TPR, bool MAX> __device__ __forceinline__ double row_reduce(double v, double* slot) {
  constexpr int G = TPR < 64 ? TPR : 64;
  v = group_reduce<G, MAX>(v);
  if constexpr (TPR > 64) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) slot[wave] = v;
    __syncthreads();
    const int first = wave / (TPR / 64) * (TPR / 64);
    v = slot[first];
#pragma unroll
    for (int i = 1; i < TPR / 64; ++i) v = join<MAX>(v, slot[first + i]);
  }
  return v;
}

template <int ELT, int V> __device__ __forceinline__ void load_weight(const void* w, int w_f32, int64_t c, int left, float (&f)[V]) {
  if (w == nullptr) {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = 1.0f;
  } else if (w_f32) {
    load_vec<REELS_HIP_F32, V>((const float*)w + c, left, f);
  } else {
    load_vec<ELT, V>((const uint8_t*)w + c * elt_bytes(ELT), left, f);
  }
}

// Where a thread's chunks of a row lie: chunk i at element col(i). Chunks are read without a branch, so
// that all loads of a row are in flight together: a thread without a chunk reads the row's first one
// (and zeroes it), and where the row's length is no multiple of V its last V elements stand for the
// partial chunk, shifted down. Rows shorter than V are read by elements.
template <int ELT, int TPR, int NCH> struct Row {
  static constexpr int V = Chunk<ELT>::V, EB = elt_bytes(ELT);
  int cols, lane, base;
  bool live;  // a group past the last row takes part in the barriers
  __device__ __forceinline__ Row(int64_t n, bool l) : cols((int)n), live(l) {
    lane = threadIdx.x % TPR;
    // the wave's first chunk, in a scalar register: chunks that no lane of the wave has are skipped
    base = TPR > 64 ? __builtin_amdgcn_readfirstlane(lane & ~63) : 0;
  }
  __device__ __forceinline__ int col(int i) const { return (lane + TPR * i) * V; }
  __device__ __forceinline__ bool some(int i) const { return (base + TPR * i) * V < cols; }
  __device__ __forceinline__ bool full(int i) const { return live && col(i) + V <= cols; }
  __device__ __forceinline__ bool part(int i) const { return live && col(i) < cols && col(i) + V > cols; }
  __device__ __forceinline__ int left(int i) const { return cols - col(i); }
  template <int E> __device__ __forceinline__ void load(const void* row, Chunk<E> (&d)[NCH]) const {
    const uint8_t* p = (const uint8_t*)row;
    if (cols < V) {
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        d[i].zero();
        if (part(i)) d[i].load(p + (int64_t)col(i) * EB, left(i));
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int at = full(i) ? col(i) : part(i) ? cols - V : 0;
      if (some(i)) d[i].d = load_any<u32x4>((const typename Store<E>::raw*)(p + (int64_t)at * EB));
    }
    if (cols % V != 0) {
#pragma unroll
      for (int i = 0; i < NCH; ++i)
        if (some(i) && part(i))
          d[i].d = __builtin_bit_cast(u32x4, __builtin_bit_cast(unsigned __int128, d[i].d) >> (8 * EB * (V - left(i))));
    }
#pragma unroll
    for (int i = 0; i < NCH; ++i)
      if (!some(i) || !(full(i) || part(i))) d[i].zero();
  }
  // weights as f32, ones without any, by the same places
  __device__ __forceinline__ void load_w(const void* w, int w_f32, float (&f)[NCH][V]) const {
    if (w == nullptr) {
#pragma unroll
      for (int i = 0; i < NCH; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) f[i][j] = 1.0f;
      return;
    }
    if (cols < V) {
#pragma unroll
      for (int i = 0; i < NCH; ++i)
        if (part(i)) load_weight<ELT, V>(w, w_f32, col(i), left(i), f[i]);
      return;
    }
    if (w_f32) {
#pragma unroll
      for (int i = 0; i < NCH; ++i)
        if (some(i)) load_vec<REELS_HIP_F32, V>((const float*)w + (full(i) ? col(i) : part(i) ? cols - V : 0), V, f[i]);
    } else {
#pragma unroll
      for (int i = 0; i < NCH; ++i)
        if (some(i)) load_vec<ELT, V>((const uint8_t*)w + (int64_t)(full(i) ? col(i) : part(i) ? cols - V : 0) * EB, V, f[i]);
    }
    if (cols % V != 0) {
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        if (!some(i)) continue;
        const int by = part(i) ? V - left(i) : 0;  // down by so many elements, in steps of 4, 2 and 1
#pragma unroll
        for (int sh = V / 2; sh > 0; sh /= 2)
#pragma unroll
          for (int j = 0; j < V; ++j) f[i][j] = (by & sh) ? (j + sh < V ? f[i][j + sh] : 0.0f) : f[i][j];
      }
    }
  }
  __device__ __forceinline__ void store(void* row, int i, const Chunk<ELT>& d) const {
    uint8_t* p = (uint8_t*)row + (int64_t)col(i) * EB;
    if (full(i)) store_any((typename Store<ELT>::raw*)p, d.d);
    else if (part(i)) d.store(p, left(i));
  }
};

template <int N> using Int = std::integral_constant<int, N>;

}  // namespace
}  // namespace reels
