// What the forward and the backward of the modulated norm share.
#pragma once
#include "microscale.h"

#include <cmath>

namespace reels {

// Who has a row: 16 lanes (tpr 16; rows of up to 256 elements), a wave (tpr 64; up to 512), or a workgroup of
// `threads` (tpr 0), with nch chunks of 16 bytes a thread. 8 elements a thread up to four waves (three waves
// at 1536 leave no lane idle), then 16, up to 16 waves. Where there are rows enough a wave has up to 1024
// elements, 16 a lane: 58514 x 700 bf16 75 us and 98 with two waves to a row, to 4 bits 78 and 94; 3000 x 700
// forward 10.1 and 9.8, backward 20 and 24; 300 x 700 7.4 and 6.5, 16 and 15. A wave to a narrow row is bound
// by the row's instructions: 131040 x 64 bf16 70 us, with 16 lanes 22; 131040 x 200 72 and 38.
struct ModForm { int tpr, nch, threads; };
constexpr int64_t kModCols = 16384;  // the longest row
inline ModForm mod_form(int elt, int64_t rows, int64_t cols) {
  const int64_t waves = ceil_div(cols, 512);
  const int per = elt == REELS_HIP_F32 ? 2 : 1;
  if (cols <= 256) return {16, cols <= 128 ? per : 2 * per, 256};
  if (waves <= 1) return {64, per, 256};
  if (waves == 2 && rows >= 2048) return {64, 2 * per, 256};
  if (waves <= 4) return {0, per, (int)waves * 64};
  return {0, 2 * per, (int)ceil_div(waves, 2) * 64};
}
// rows of a workgroup at once
inline int64_t mod_walkers(ModForm f) { return f.tpr == 0 ? 1 : f.threads / f.tpr; }
// How the chunks of a row fall on its threads: every thread has whole ones, or some have a part or none, or
// the row is shorter than a chunk
enum ModKind { kEven = 0, kAny = 1, kTiny = 2 };

// calls g(tpr, nch, most threads of a workgroup, kind) as integral constants
template <int N> using ModInt = std::integral_constant<int, N>;
template <int ELT, typename F> void with_mod_form(ModForm f, int64_t cols, F&& g) {
  constexpr int P = ELT == REELS_HIP_F32 ? 2 : 1, V = Chunk<ELT>::V;
  auto kind = [&](auto tpr, auto nch, auto nt) {
    if (cols == (int64_t)(f.tpr == 0 ? f.threads : f.tpr) * f.nch * V) g(tpr, nch, nt, ModInt<kEven>{});
    else g(tpr, nch, nt, ModInt<kAny>{});
  };
  if (cols < V) g(ModInt<16>{}, ModInt<P>{}, ModInt<256>{}, ModInt<kTiny>{});
  else if (f.tpr == 16 && f.nch == P) kind(ModInt<16>{}, ModInt<P>{}, ModInt<256>{});
  else if (f.tpr == 16) kind(ModInt<16>{}, ModInt<2 * P>{}, ModInt<256>{});
  else if (f.tpr == 64 && f.nch == P) kind(ModInt<64>{}, ModInt<P>{}, ModInt<256>{});
  else if (f.tpr == 64) kind(ModInt<64>{}, ModInt<2 * P>{}, ModInt<256>{});
  else if (f.nch == P) kind(ModInt<0>{}, ModInt<P>{}, ModInt<256>{});
  else if (f.threads <= 512) kind(ModInt<0>{}, ModInt<2 * P>{}, ModInt<512>{});
  else kind(ModInt<0>{}, ModInt<2 * P>{}, ModInt<1024>{});
}

namespace {

// a and b summed over a row's threads in 64 bits: 16 lanes', a wave's, or a workgroup's of at most 16 waves through LDS,
// wave by wave in one order. slots: one of two in turn, so that a wave may enter the next row's sums while
// another still reads this one's. The barrier leaves loads in flight.
template <int TPR> __device__ __forceinline__ void row_sums(double& a, double& b, double (&slots)[16][2]) {
  constexpr int G = TPR == 16 ? 16 : 64;
  a = group_reduce<G, false>(a);
  b = group_reduce<G, false>(b);
  if constexpr (TPR == 0) {
    if ((threadIdx.x & 63) == 0) {
      slots[threadIdx.x >> 6][0] = a;
      slots[threadIdx.x >> 6][1] = b;
    }
    asm volatile("" ::: "memory");  // the slots are written on this side of the barrier
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    const int i = threadIdx.x & 15;
    const bool in = i < (int)(blockDim.x >> 6);
    a = group_reduce<16, false>(in ? slots[i][0] : 0.0);
    b = group_reduce<16, false>(in ? slots[i][1] : 0.0);
  }
}

// What n = (s - mean) rstd of a row's elements is formed with: fmaf(s - hi, rstd, k), the mean in two parts.
// Elements are at most sqrt(cols) spreads from the mean, so s - hi can pass the f32 range only where rstd is
// below `far` = sqrt(cols) 2^-128 (and 1 / 32 more, for values kept in 7 bits). Such a row's mean is taken off in k
// alone: |mean| rstd < 1.04 sqrt(cols) there, and n is off by half a step of that.
struct ModUnit { float hi, k; };
__device__ __forceinline__ ModUnit mod_unit(float hi, float lo, float rstd, float far) {
  const float k = -lo * rstd;
  const bool over = rstd < far;
  return {over ? 0.0f : hi, over ? fmaf(-hi, rstd, k) : k};
}
inline float mod_far(int64_t cols) { return (float)(std::sqrt((double)cols) * 0x1.08p-128); }

// A thread's chunks of a row: chunk i at element col(i). They are read without a branch, so that all loads of
// a row are in flight together: a thread without a chunk reads the row's first one, and where the row's
// length is no multiple of V its last V elements stand for the partial chunk; `trim` puts that right once the
// data is there, in the waves that have such threads. Rows shorter than a chunk are
// read by elements.
template <int ELT, int TPR, int NCH, int KIND> struct ModRow {
  static constexpr int V = Chunk<ELT>::V, EB = elt_bytes(ELT);
  int cols, lane, base;
  __device__ __forceinline__ static int threads() {
    if constexpr (TPR == 0) return (int)blockDim.x;
    else return TPR;
  }
  __device__ __forceinline__ explicit ModRow(int64_t n) : cols((int)n) {
    lane = TPR == 0 ? threadIdx.x : threadIdx.x % (TPR == 0 ? 64 : TPR);
    base = TPR == 0 ? __builtin_amdgcn_readfirstlane(lane & ~63) : 0;
  }
  __device__ __forceinline__ int col(int i) const { return (lane + threads() * i) * V; }
  __device__ __forceinline__ int left(int i) const { return cols - col(i); }
  // of the whole wave, in scalar registers: whether a lane has a chunk i, and whether all have whole ones
  __device__ __forceinline__ bool some(int i) const { return KIND == kEven || (base + threads() * i) * V < cols; }
  __device__ __forceinline__ bool all(int i) const {
    return KIND == kEven || (KIND == kAny && (base + threads() * i + (TPR == 16 ? 16 : 64)) * V <= cols);
  }
  __device__ __forceinline__ void load(const void* row, Chunk<ELT> (&d)[NCH]) const {
    const uint8_t* p = (const uint8_t*)row;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int l = left(i);
      if constexpr (KIND == kTiny) {
        d[i].zero();
        if (l > 0) d[i].load(p + (int64_t)col(i) * EB, l);
      } else {
        const int at = KIND == kEven || l >= V ? col(i) : l > 0 ? cols - V : 0;
        d[i].d = load_any<u32x4>((const typename Store<ELT>::raw*)(p + (uint32_t)(at * EB)));  // 32-bit offsets from a scalar base
      }
    }
  }
  __device__ __forceinline__ void trim(Chunk<ELT> (&d)[NCH]) const {
    if constexpr (KIND != kAny) return;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      if (all(i)) continue;
      const int l = left(i);
      const unsigned __int128 u = __builtin_bit_cast(unsigned __int128, d[i].d);
      if (l < V) d[i].d = __builtin_bit_cast(u32x4, l > 0 ? u >> (8 * EB * (V - l)) : (unsigned __int128)0);
    }
  }
  __device__ __forceinline__ void store(void* row, int i, const Chunk<ELT>& d) const {
    uint8_t* p = (uint8_t*)row + (uint32_t)(col(i) * EB);
    if (all(i)) store_any((typename Store<ELT>::raw*)p, d.d);
    else if (left(i) > 0) d.store(p, left(i));
  }
  // the same in f32
  __device__ __forceinline__ void store(float* row, int i, const float (&f)[V]) const {
    if (all(i)) store_vec<REELS_HIP_F32, V>(row + (uint32_t)col(i), V, f);
    else if (left(i) > 0) store_vec<REELS_HIP_F32, V>(row + (uint32_t)col(i), left(i), f);
  }
  // a row of modulations in f32 (or the rows' type), zeros where the thread has no element; read like the rows
  __device__ __forceinline__ void mods(const void* p, int64_t ld, int f32, int64_t group, float (&f)[NCH][V]) const {
    const uint8_t* r = (const uint8_t*)p + group * ld * (f32 ? 4 : EB);
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      int l = left(i);
      asm volatile("" : "+v"(l));  // what follows from it is not kept between rows
      const uint32_t at = KIND == kEven || l >= V ? (uint32_t)(cols - l) : KIND == kAny && l > 0 ? (uint32_t)(cols - V) : KIND == kTiny && l > 0 ? (uint32_t)(cols - l) : 0u;
      const int n = KIND == kTiny ? (l < 0 ? 0 : l) : V;
      if (f32) load_vec<REELS_HIP_F32, V>((const float*)r + at, n, f[i]);
      else load_vec<ELT, V>(r + at * EB, n, f[i]);
    }
    if constexpr (KIND != kAny) return;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      if (all(i)) continue;
      const int l = left(i), by = l < V ? V - l : 0;
#pragma unroll
      for (int s = V / 2; s > 0; s /= 2)
#pragma unroll
        for (int j = 0; j < V; ++j) f[i][j] = by & s ? (j + s < V ? f[i][j + s] : 0.0f) : f[i][j];
#pragma unroll
      for (int j = 0; j < V; ++j) f[i][j] = l > 0 ? f[i][j] : 0.0f;
    }
  }
};

inline int mod_check(const char* fn, int dtype, int m_dtype, int64_t rows, int64_t cols, int64_t rpg) {
  if (!known_elt(dtype) || (m_dtype != dtype && m_dtype != REELS_HIP_F32))
    return fail(REELS_HIP_EDTYPE, std::string(fn) + ": dtype must be f32, bf16 or f16, and m_dtype the same or f32");
  if (rows < 0 || cols <= 0 || cols > kModCols || rows > ((int64_t)1 << 31) - 1)
    return fail(REELS_HIP_EINVAL, std::string(fn) + ": 0 <= rows < 2^31 and 0 < cols <= 16384 required");
  if (rpg <= 0 || rows % rpg != 0)
    return fail(REELS_HIP_EINVAL, std::string(fn) + ": rows must be a multiple of rows_per_group, which is positive");
  return REELS_HIP_OK;
}

}  // namespace
}  // namespace reels
