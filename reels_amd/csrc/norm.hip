// Root-mean-square norm with the residual's addition, its output as int8 rows with scales, and its
// backward (the reference's rmsnorm, src/layers/normalization.jl:10-24, and the residual addition
// before it in one pass).
//
//   s = rnd(x + residual) (x itself without one);  rstd = (mean_c s^2 + eps)^(-1/2)
//   y = rnd(s rstd w)                                  (w = 1 where there is none)
//   int8: scale = max_c |s w| rstd / 127, q = round_ties_even(127 s w / max_c |s w|); rstd cancels in
//         q, so a code depends on the row's own ratios alone (formed in 64 bits). A zero row has
//         scale 1; a row whose scale is not finite has scale NaN and zero codes, so its values are
//         NaN, as y's would be.
//   backward, g = dy w: dx = rnd(rstd (g - s rstd^2 mean_c(g s)) + dsum);  dw = sum_m dy s rstd (f32)
//
// All of it is bound by memory: each kernel reads its operands once and keeps the row, as stored, in
// registers between the reduction and the output (the backward without dw also spills a few there: 7 of
// 128 at 5120 bf16, at most 11; f32 rows of 16384 with dw 26). A row belongs to a group of TPR threads
// that hold NCH 16-byte chunks each: TPR is the smallest of 16, 64 and 256 whose threads need at most four chunks, or
// 512 (f32: or 1024) with three or four, so short rows (one head) share a wave and long ones have many
// loads in flight. Rows past 16384 elements run the loop form, which reads them again from L2. Squares
// and products are summed in 64 bits (MI355X adds those at the rate of 32-bit ones), so the squares of
// large values do not leave the range; rstd itself is kept in 32 bits.
//
// 32760 x 5120 bf16: forward 120-125 us (5.4-5.6 TB/s), with the residual 237 us (5.7), backward 205-242 us
// (4.2-4.9), with dw and dsum 261 us (5.1), int8 rows with the residual 209-240 us (4.9-5.6); a copy of
// 1 GiB runs at 5.3 TB/s.
#include "vec.h"

namespace reels {
namespace {

constexpr int kLongThreads = 1024;

struct NormArgs {
  const void* x;
  const void* res;   // or nullptr
  const void* w;     // or nullptr
  void* sum;         // written when res is set
  void* y;
  float* rstd;
  int8_t* q;
  float* scales;
  int64_t ld_x, ld_r, rows, cols;
  double per_col;    // 1 / cols
  float eps;
  int w_f32;         // w holds f32 (else the row's type)
};

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

// What a row's codes take from it: the largest |s w| in 64 bits and its quotients' factors. even: every
// weight is below 1e20 (and none is NaN).
struct Quant {
  double top, inv;  // codes are 127 p / top = p inv
  float f1, f2;     // in f32: (s f1) w f2
  bool zero, fast;
  float scale;
  __device__ __forceinline__ Quant(double t, double rstd, bool even) : top(t) {
    const double size = top * rstd;  // the row's largest value
    scale = (float)(size * (1.0 / 127.0));
    // rstd is 0 or NaN where the row holds an infinity or NaN: top may have lost it, where its weight
    // is zero and the product NaN
    const bool whole = __builtin_isfinite(scale) && rstd > 0.0;
    if (!whole) scale = __builtin_nanf("");
    else if (top == 0.0) scale = 1.0f;
    zero = !whole || top == 0.0;
    inv = 127.0 * rcp64(top);
    f1 = (float)rstd;
    f2 = (float)(127.0 * rcp64(size));
    // In f32 the factors and the products that matter keep all their bits: a value (s rstd) that has
    // lost some is below 2^-126, its product with an even weight below 1e-17, its code 0
    fast = even && size > 1e-10 && size < 1e30 && rstd > 1e-30 && rstd < 1e30;
  }
};

// the largest |s w| may be infinite: NaN counts as infinity, which the maximum keeps
__device__ __forceinline__ double quant_abs(double p) {
  const double a = fabs(p);
  return a <= 1.7976931348623157e308 ? a : __builtin_inf();
}
// the largest |w| and |s w| of a chunk. wide: NaN stays (v_maximum3); the products in f32 where they
// are exact, two 16-bit significands (the range is looked at by the caller), else in 64 bits
template <bool EXACT32, int V>
__device__ __forceinline__ void quant_top(const float (&s)[V], const float (&w)[V], double& top, float& wide) {
  if constexpr (EXACT32) {
    float t = 0.0f;
#pragma unroll
    for (int j = 0; j < V; j += 2) t = fmaxf(t, fmaxf(fabsf(s[j] * w[j]), fabsf(s[j + 1] * w[j + 1])));
    top = fmax(top, (double)t);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) top = fmax(top, fabs((double)s[j] * (double)w[j]));
  }
#pragma unroll
  for (int j = 0; j < V; j += 2)
    wide = __builtin_elementwise_maximum(wide, __builtin_elementwise_maximum(fabsf(w[j]), fabsf(w[j + 1])));
}

// round_ties_even(127 p / top) of a product formed in 64 bits: p inv is within 2^-50 of the quotient,
// so only values next to a border take the division
__device__ __forceinline__ int quant_exact(float s, float w, const Quant& q) {
  const double p = (double)s * (double)w, t = p * q.inv;
  double k = rint(t);
  if (fabs(t - k) > 0.4999999999) k = rint(127.0 * p / q.top);
  return (int)k;
}

// The codes of a chunk, four to a word. In f32 the quotient has at most five roundings, 127 * 5 * 2^-24 = 3.8e-5: a chunk
// with a value within 2^-14 of a border (6% of a wave's) is formed in 64 bits. Adding 1.5 * 2^23
// rounds to a whole number, ties to even, and leaves it in the low byte.
template <bool EXACT32, int V>
__device__ __forceinline__ void quant_chunk(const float (&s)[V], const float (&w)[V], const Quant& q, uint32_t (&word)[V / 4]) {
  float far = q.fast ? 0.0f : 1.0f;
  uint32_t c[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const float p = EXACT32 ? s[j] * w[j] : s[j] * q.f1 * w[j], f = EXACT32 ? (float)q.inv : q.f2;
    const float m = fmaf(p, f, 12582912.0f);
    far = fmaxf(far, fabsf(fmaf(p, f, -(m - 12582912.0f))));
    c[j] = __float_as_uint(m);
  }
  if (far > 0.5f - 0x1p-14f) {
#pragma unroll
    for (int j = 0; j < V; ++j) c[j] = (uint32_t)quant_exact(s[j], w[j], q);
  }
#pragma unroll
  for (int i = 0; i < V / 4; ++i) {
    const uint32_t lo = __builtin_amdgcn_perm(c[4 * i + 1], c[4 * i], 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(c[4 * i + 3], c[4 * i + 2], 0x04000c0cu);
    word[i] = q.zero ? 0u : lo | hi;
  }
}

template <int V> __device__ __forceinline__ void store_codes(int8_t* q, int left, const uint32_t (&word)[V / 4]) {
  struct Pack { int8_t e[V]; };
  const Pack p = __builtin_bit_cast(Pack, word);
  if (left >= V) {
    store_any(q, p);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < left) q[i] = p.e[i];
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

// MODE 0: y; 1: int8 rows; 2: the same with 16-bit values and weights (or none)
template <int ELT, int TPR, int NCH, int MODE>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void norm_kernel(NormArgs a) {
  constexpr int V = Chunk<ELT>::V, EB = elt_bytes(ELT), NT = TPR < 256 ? 256 : TPR;
  constexpr bool QUANT = MODE > 0, EXACT32 = MODE == 2;
  __shared__ double slots[2][NT / 64];
  const int64_t row0 = (int64_t)blockIdx.x * (NT / TPR) + threadIdx.x / TPR;
  const Row<ELT, TPR, NCH> at(a.cols, row0 < a.rows);
  const int64_t row = at.live ? row0 : a.rows - 1;
  Chunk<ELT> s[NCH], r[NCH];
  float w[NCH][V];
  at.load((const uint8_t*)a.x + row * a.ld_x * EB, s);
  if (a.res != nullptr) at.load((const uint8_t*)a.res + row * a.ld_r * EB, r);
  if constexpr (!QUANT) at.load_w(a.w, a.w_f32, w);
  double ss = 0.0;
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    if (!at.some(i)) continue;
    if (a.res != nullptr) {
      float f[V];
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] = s[i].get(j) + r[i].get(j);
      s[i].pack(f);
      at.store((uint8_t*)a.sum + row * a.cols * EB, i, s[i]);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) ss = fma((double)s[i].get(j), (double)s[i].get(j), ss);
    s[i].hold();
  }
  if constexpr (QUANT) at.load_w(a.w, a.w_f32, w);
  ss = row_reduce<TPR, false>(ss, slots[0]);
  const double rstd = rsqrt64(fma(ss, a.per_col, (double)a.eps));
  if constexpr (!QUANT) {
    const float rs = (float)rstd;
    if (at.live && at.lane == 0) a.rstd[row] = rs;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      if (!at.some(i)) continue;
      float y[V];
      Chunk<ELT> o;
#pragma unroll
      for (int j = 0; j < V; ++j) y[j] = s[i].get(j) * rs * w[i][j];
      o.pack(y);
      at.store((uint8_t*)a.y + row * a.cols * EB, i, o);
    }
  } else {
    double top = 0.0;
    float wide = 0.0f;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      if (!at.some(i)) continue;
      if (at.full(i) || at.part(i)) {
        float f[V];
        s[i].unpack(f);
        quant_top<EXACT32, V>(f, w[i], top, wide);
      }
      s[i].hold();
    }
    top = row_reduce<TPR, true>(wide <= 1e20f ? top : __builtin_inf(), slots[1]);
    bool even = top < __builtin_inf();
    if (EXACT32 && !(top > 1e-30 && top < 1e30)) even = false;  // f32 products out of its range
    if (!even) {  // once more in 64 bits, with NaN seen (a row's threads take this together)
      top = 0.0;
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        if (!(at.full(i) || at.part(i))) continue;
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (j < at.left(i)) top = fmax(top, quant_abs((double)s[i].get(j) * (double)w[i][j]));
      }
      top = row_reduce<TPR, true>(top, slots[0]);
    }
    const Quant q(top, rstd, even);
    if (at.live && at.lane == 0) a.scales[row] = q.scale;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      if (!(at.full(i) || at.part(i))) continue;
      float f[V];
      uint32_t word[V / 4];
      s[i].unpack(f);
      quant_chunk<EXACT32, V>(f, w[i], q, word);
      store_codes<V>(a.q + row * a.cols + at.col(i), at.left(i), word);
    }
  }
}

// s of a chunk: x, or x + residual rounded to the type
template <int ELT> __device__ __forceinline__ void load_sum(const NormArgs& a, int64_t row, int64_t c, int left, Chunk<ELT>& s) {
  constexpr int EB = elt_bytes(ELT), V = Chunk<ELT>::V;
  s.load((const uint8_t*)a.x + (row * a.ld_x + c) * EB, left);
  if (a.res != nullptr) {
    Chunk<ELT> r;
    r.load((const uint8_t*)a.res + (row * a.ld_r + c) * EB, left);
    float f[V];
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = s.get(j) + r.get(j);
    s.pack(f);
  }
}

// rows past the register form: one workgroup per row, the row read again for its output
template <int ELT, bool QUANT>
__global__ __launch_bounds__(kLongThreads) void norm_long_kernel(NormArgs a) {
  constexpr int V = Chunk<ELT>::V, EB = elt_bytes(ELT);
  __shared__ double slots[2][kLongThreads / 64];
  const int64_t row = blockIdx.x;
  double ss = 0.0, top = 0.0;
  float wide = 0.0f;
  for (int64_t c = (int64_t)threadIdx.x * V; c < a.cols; c += kLongThreads * V) {
    const int left = a.cols - c < V ? (int)(a.cols - c) : V;
    Chunk<ELT> s;
    load_sum<ELT>(a, row, c, left, s);
#pragma unroll
    for (int j = 0; j < V; ++j) ss = fma((double)s.get(j), (double)s.get(j), ss);
    if constexpr (QUANT) {
      float w[V];
      load_weight<ELT, V>(a.w, a.w_f32, c, left, w);
      float f[V];
      s.unpack(f);
      quant_top<false, V>(f, w, top, wide);
    }
  }
  ss = row_reduce<kLongThreads, false>(ss, slots[0]);
  const double rstd = rsqrt64(fma(ss, a.per_col, (double)a.eps));
  bool even = true;
  if constexpr (QUANT) {
    top = row_reduce<kLongThreads, true>(wide <= 1e20f ? top : __builtin_inf(), slots[1]);
    even = top < __builtin_inf();
    if (!even) {
      top = 0.0;
      for (int64_t c = (int64_t)threadIdx.x * V; c < a.cols; c += kLongThreads * V) {
        const int left = a.cols - c < V ? (int)(a.cols - c) : V;
        Chunk<ELT> s;
        float w[V];
        load_sum<ELT>(a, row, c, left, s);
        load_weight<ELT, V>(a.w, a.w_f32, c, left, w);
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (j < left) top = fmax(top, quant_abs((double)s.get(j) * (double)w[j]));
      }
      top = row_reduce<kLongThreads, true>(top, slots[0]);
    }
  }
  const Quant q(top, rstd, even);
  if (threadIdx.x == 0) {
    if constexpr (QUANT) a.scales[row] = q.scale;
    else a.rstd[row] = (float)rstd;
  }
  // the sum is written here, after every read of x and the residual's first pass, chunk by chunk by
  // the thread that read it, so it may take the place of x or of the residual
  for (int64_t c = (int64_t)threadIdx.x * V; c < a.cols; c += kLongThreads * V) {
    const int left = a.cols - c < V ? (int)(a.cols - c) : V;
    Chunk<ELT> s;
    float w[V], f[V];
    load_sum<ELT>(a, row, c, left, s);
    load_weight<ELT, V>(a.w, a.w_f32, c, left, w);
    s.unpack(f);
    if (a.res != nullptr) s.store((uint8_t*)a.sum + (row * a.cols + c) * EB, left);
    if constexpr (QUANT) {
      uint32_t word[V / 4];
      quant_chunk<false, V>(f, w, q, word);
      store_codes<V>(a.q + row * a.cols + c, left, word);
    } else {
      const float rs = (float)rstd;
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] = f[j] * rs * w[j];
      store_vec<ELT, V>((uint8_t*)a.y + (row * a.cols + c) * EB, left, f);
    }
  }
}

// ---- backward --------------------------------------------------------------------------------
struct NormBwdArgs {
  const void* dy;
  const void* s;
  const void* dsum;  // or nullptr
  const void* w;     // or nullptr
  const float* rstd;
  void* dx;
  float* part;       // [workgroups][cols] partial dw, or nullptr
  int64_t rows, cols;
  double per_col;
  int w_f32;
};

// A workgroup walks the rows b, b + gridDim, ... (times the rows it holds at once): with dw each
// thread keeps the sums of its own columns in registers over all its rows, and the groups of a
// workgroup add theirs in LDS in group order, one partial row per workgroup.
// Waves a SIMD has to hold, by the registers that a row's three operands, weights and sums of dw take
// (without dw a few less than the compiler wants)
constexpr int bwd_waves(int tpr, int nch, bool dw) {
  if (tpr == 1024) return 4;
  return dw ? (nch == 1 ? 7 : nch == 2 ? 4 : nch == 3 ? 3 : 2) : (nch == 1 ? 7 : nch == 2 ? 5 : nch == 3 ? 4 : 3);
}

template <int ELT, int TPR, int NCH, bool DW>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR, bwd_waves(TPR, NCH, DW)) void norm_bwd_kernel(NormBwdArgs a) {
  constexpr int V = 16 / elt_bytes(ELT), EB = elt_bytes(ELT), NT = TPR < 256 ? 256 : TPR, RPB = NT / TPR;
  __shared__ double slots[2][NT / 64];
  __shared__ float acc[DW && RPB > 1 ? RPB * TPR * NCH * V : 1];
  const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
  float dw[NCH][V];
  if constexpr (DW) {
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) dw[i][j] = 0.0f;
  }
  int turn = 0;
  for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.rows; r0 += (int64_t)gridDim.x * RPB, turn ^= 1) {
    const Row<ELT, TPR, NCH> at(a.cols, r0 + group < a.rows);
    const int64_t row = at.live ? r0 + group : a.rows - 1, begin = row * a.cols * EB;
    const float rstd = at.live ? a.rstd[row] : 0.0f;
    Chunk<ELT> s[NCH], dy[NCH], ds[NCH];
    float w[NCH][V];
    at.load((const uint8_t*)a.s + begin, s);
    at.load((const uint8_t*)a.dy + begin, dy);
    if (a.dsum != nullptr) at.load((const uint8_t*)a.dsum + begin, ds);
    at.load_w(a.w, a.w_f32, w);
    double gs = 0.0;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      if (!at.some(i) || !(at.full(i) || at.part(i))) continue;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float sv = s[i].get(j), d = dy[i].get(j);
        if constexpr (DW) dw[i][j] += d * (sv * rstd);
        gs = fma((double)(d * w[i][j]), (double)sv, gs);
      }
      s[i].hold();
      dy[i].hold();
    }
    // two slots in turn: a wave may enter the next row's reduction while another still reads this one's
    gs = row_reduce<TPR, false>(gs, slots[turn]);
    const float k = (float)(gs * a.per_col * (double)rstd * (double)rstd);
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      if (!at.some(i)) continue;
      float d[V];
      Chunk<ELT> o;
#pragma unroll
      for (int j = 0; j < V; ++j) d[j] = rstd * (dy[i].get(j) * w[i][j] - s[i].get(j) * k);
      if (a.dsum != nullptr) {
#pragma unroll
        for (int j = 0; j < V; ++j) d[j] += ds[i].get(j);
      }
      o.pack(d);
      at.store((uint8_t*)a.dx + begin, i, o);
    }
  }
  if constexpr (DW) {
    float* out = a.part + (int64_t)blockIdx.x * a.cols;
    if constexpr (RPB > 1) {
#pragma unroll
      for (int i = 0; i < NCH; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) acc[(group * TPR * NCH + lane + TPR * i) * V + j] = dw[i][j];
      __syncthreads();
      for (int c = threadIdx.x; c < (int)a.cols; c += NT) {
        float t = acc[c];
        for (int r = 1; r < RPB; ++r) t += acc[r * TPR * NCH * V + c];
        out[c] = t;
      }
    } else {
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        const int64_t c = (int64_t)(lane + TPR * i) * V;
        const int left = c < a.cols ? (a.cols - c < V ? (int)(a.cols - c) : V) : 0;
        if (left > 0) store_vec<REELS_HIP_F32, V>(out + c, left, dw[i]);
      }
    }
  }
}

// rows past the register form: dx row by row, read twice
template <int ELT>
__global__ __launch_bounds__(kLongThreads) void norm_bwd_long_kernel(NormBwdArgs a) {
  constexpr int V = 16 / elt_bytes(ELT), EB = elt_bytes(ELT);
  __shared__ double slots[kLongThreads / 64];
  const int64_t row = blockIdx.x;
  const float rstd = a.rstd[row];
  auto load_g = [&](int64_t c, int left, float (&s)[V], float (&g)[V]) {
    float w[V];
    load_vec<ELT, V>((const uint8_t*)a.s + (row * a.cols + c) * EB, left, s);
    load_vec<ELT, V>((const uint8_t*)a.dy + (row * a.cols + c) * EB, left, g);
    load_weight<ELT, V>(a.w, a.w_f32, c, left, w);
#pragma unroll
    for (int j = 0; j < V; ++j) g[j] *= w[j];
  };
  double gs = 0.0;
  for (int64_t c = (int64_t)threadIdx.x * V; c < a.cols; c += kLongThreads * V) {
    const int left = a.cols - c < V ? (int)(a.cols - c) : V;
    float s[V], g[V];
    load_g(c, left, s, g);
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < left) gs = fma((double)g[j], (double)s[j], gs);
  }
  gs = row_reduce<kLongThreads, false>(gs, slots);
  const float k = (float)(gs * a.per_col * (double)rstd * (double)rstd);
  for (int64_t c = (int64_t)threadIdx.x * V; c < a.cols; c += kLongThreads * V) {
    const int left = a.cols - c < V ? (int)(a.cols - c) : V;
    float s[V], g[V], d[V];
    load_g(c, left, s, g);
#pragma unroll
    for (int j = 0; j < V; ++j) d[j] = rstd * (g[j] - s[j] * k);
    if (a.dsum != nullptr) {
      float t[V];
      load_vec<ELT, V>((const uint8_t*)a.dsum + (row * a.cols + c) * EB, left, t);
#pragma unroll
      for (int j = 0; j < V; ++j) d[j] += t[j];
    }
    store_vec<ELT, V>((uint8_t*)a.dx + (row * a.cols + c) * EB, left, d);
  }
}

// their dw: partial sums over the rows b, b + gridDim.y, ... of one column per thread
template <int ELT>
__global__ __launch_bounds__(256) void norm_dw_long_kernel(NormBwdArgs a) {
  constexpr int EB = elt_bytes(ELT);
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= a.cols) return;
  float t = 0.0f;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    float s[1], g[1];
    load_vec<ELT, 1>((const uint8_t*)a.s + (row * a.cols + c) * EB, 1, s);
    load_vec<ELT, 1>((const uint8_t*)a.dy + (row * a.cols + c) * EB, 1, g);
    t += g[0] * (s[0] * a.rstd[row]);
  }
  a.part[(int64_t)blockIdx.y * a.cols + c] = t;
}

// dw[c] = sum over the partial rows: 32 columns x 32 slices per workgroup, slice y adds the rows y,
// y + 32, ... and the slices follow in order
__global__ __launch_bounds__(1024) void norm_dw_kernel(const float* __restrict__ part, int n, int64_t cols,
                                                       float* __restrict__ dw) {
  __shared__ float acc[32][33];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + x;
  float t = 0.0f;
  if (c < cols) {
#pragma unroll 8
    for (int r = y; r < n; r += 32) t += part[(int64_t)r * cols + c];
  }
  acc[y][x] = t;
  __syncthreads();
  if (y == 0 && c < cols) {
#pragma unroll
    for (int i = 1; i < 32; ++i) t += acc[i][x];
    dw[c] = t;
  }
}

// ---- host ------------------------------------------------------------------------------------
struct Form { int tpr, nch; };  // tpr 0: the loop form
Form norm_form(int elt, int64_t cols) {
  const int64_t chunks = ceil_div(cols, 16 / elt_bytes(elt));
  for (int tpr : {16, 64, 256})
    if (chunks <= 4 * tpr) return {tpr, (int)ceil_div(chunks, tpr)};
  if (chunks <= 2048) return {512, (int)ceil_div(chunks, 512)};
  if (elt == REELS_HIP_F32 && chunks <= 4096) return {1024, (int)ceil_div(chunks, 1024)};  // half the values a chunk
  return {0, 0};
}

bool norm_fits(int64_t rows, Form f) {  // a group of threads for each row
  const int threads = f.tpr == 0 ? kLongThreads : f.tpr, wg = threads < 256 ? 256 : threads;
  return grid_fits(ceil_div(rows, wg / threads), wg);
}

template <int N> using Int = std::integral_constant<int, N>;
template <int ELT, typename F> void with_form(Form f, F&& g) {
  auto nch = [&](auto tpr) {
    switch (f.nch) {
      case 1: g(tpr, Int<1>{}); break;
      case 2: g(tpr, Int<2>{}); break;
      case 3: g(tpr, Int<3>{}); break;
      default: g(tpr, Int<4>{}); break;
    }
  };
  switch (f.tpr) {
    case 16: nch(Int<16>{}); break;
    case 64: nch(Int<64>{}); break;
    case 256: nch(Int<256>{}); break;
    case 512:
      if (f.nch == 3) g(Int<512>{}, Int<3>{});
      else g(Int<512>{}, Int<4>{});
      break;
    default:
      if constexpr (ELT == REELS_HIP_F32) {
        if (f.nch == 3) g(Int<1024>{}, Int<3>{});
        else g(Int<1024>{}, Int<4>{});
      }
      break;
  }
}

int norm_check(const char* fn, int dtype, int w_dtype, const void* w, int64_t rows, int64_t cols) {
  if (!known_elt(dtype) || (w != nullptr && w_dtype != dtype && w_dtype != REELS_HIP_F32))
    return fail(REELS_HIP_EDTYPE, std::string(fn) + ": dtype must be f32, bf16 or f16, and w_dtype the same or f32");
  if (rows < 0 || cols <= 0 || rows > ((int64_t)1 << 31) - 1 || cols > ((int64_t)1 << 31) - 1)
    return fail(REELS_HIP_EINVAL, std::string(fn) + ": rows >= 0 and cols > 0 below 2^31 required");
  return REELS_HIP_OK;
}

int norm_forward(const char* fn, const char* label, bool quant, NormArgs a, int dtype, int w_dtype, hipStream_t st) {
  clear_error();
  if (int rc = norm_check(fn, dtype, w_dtype, a.w, a.rows, a.cols)) return rc;
  if (!(a.eps >= 0.0f && a.eps <= 3.4e38f)) return fail(REELS_HIP_EINVAL, std::string(fn) + ": eps must be finite and not negative");
  if (a.ld_x < a.cols || (a.res != nullptr && a.ld_r < a.cols))
    return fail(REELS_HIP_EINVAL, std::string(fn) + ": row strides below cols");
  if (a.rows == 0) return REELS_HIP_OK;
  if (a.x == nullptr || (a.res != nullptr && a.sum == nullptr) || (quant ? a.q == nullptr || a.scales == nullptr : a.y == nullptr || a.rstd == nullptr))
    return fail(REELS_HIP_EINVAL, std::string(fn) + ": NULL operand");
  a.w_f32 = w_dtype == REELS_HIP_F32 && dtype != REELS_HIP_F32;
  a.per_col = 1.0 / (double)a.cols;
  const Form f = norm_form(dtype, a.cols);
  if (!norm_fits(a.rows, f)) return fail(REELS_HIP_EINVAL, std::string(fn) + ": too many rows for one launch");
  { TraceScope _ts(st, label);
    with_any_elt(dtype, [&](auto e) {
      constexpr int E = decltype(e)::value;
      if (f.tpr == 0) {
        if (quant) norm_long_kernel<E, true><<<(unsigned)a.rows, kLongThreads, 0, st>>>(a);
        else norm_long_kernel<E, false><<<(unsigned)a.rows, kLongThreads, 0, st>>>(a);
        return;
      }
      with_form<E>(f, [&](auto tpr, auto nch) {
        constexpr int T = decltype(tpr)::value, C = decltype(nch)::value, NT = T < 256 ? 256 : T;
        const unsigned grid = (unsigned)ceil_div(a.rows, NT / T);
        if (!quant) norm_kernel<E, T, C, 0><<<grid, NT, 0, st>>>(a);
        else if (E == REELS_HIP_F32 || a.w_f32) norm_kernel<E, T, C, 1><<<grid, NT, 0, st>>>(a);
        else if constexpr (E != REELS_HIP_F32) norm_kernel<E, T, C, 2><<<grid, NT, 0, st>>>(a);
      });
    }); }
  return check_launch(label);
}

// Workgroups of the backward with dw (each writes one partial row): as many as the GPU holds at once by
// their registers (1024 where 768 fit cost a second round: 32760 x 5120 380 -> 261 us), and at least two
// rows for each group of threads, so that the partial rows stay a small part of the traffic
int64_t norm_parts(int64_t rows, int elt, Form f) {
  const int64_t rpb = f.tpr == 0 ? 1 : (f.tpr < 256 ? 256 / f.tpr : 1);
  const int values = f.nch * 16 / elt_bytes(elt);  // of a thread
  const int64_t want = f.tpr == 0 ? 64 : f.tpr >= 512 ? 256 : values >= 24 ? 768 : elt == REELS_HIP_F32 || values >= 16 || f.tpr == 256 ? 1024 : 1792;
  const int64_t need = ceil_div(rows, 2 * rpb);
  return need < want ? need : want;
}

}  // namespace
}  // namespace reels

extern "C" int reels_hip_rms_norm(const void* x, int64_t ld_x, const void* residual, int64_t ld_r, const void* weight,
                                  int w_dtype, int dtype, int64_t rows, int64_t cols, float eps, void* sum, void* y,
                                  float* rstd, void* stream) {
  using namespace reels;
  return norm_forward("reels_hip_rms_norm", "norm_kernel", false,
                      NormArgs{x, residual, weight, sum, y, rstd, nullptr, nullptr, ld_x, ld_r, rows, cols, 0.0, eps, 0}, dtype,
                      w_dtype, (hipStream_t)stream);
}

extern "C" int reels_hip_rms_norm_i8(const void* x, int64_t ld_x, const void* residual, int64_t ld_r, const void* weight,
                                     int w_dtype, int dtype, int64_t rows, int64_t cols, float eps, void* sum, int8_t* q,
                                     float* scales, void* stream) {
  using namespace reels;
  return norm_forward("reels_hip_rms_norm_i8", "norm_kernel<int8>", true,
                      NormArgs{x, residual, weight, sum, nullptr, nullptr, q, scales, ld_x, ld_r, rows, cols, 0.0, eps, 0}, dtype,
                      w_dtype, (hipStream_t)stream);
}

extern "C" size_t reels_hip_rms_norm_workspace_bytes(int64_t rows, int64_t cols) {
  using namespace reels;
  if (rows < 0 || cols <= 0) return 0;
  // the most partial rows of any element type
  int64_t n = 1;
  for (int elt : {REELS_HIP_F32, REELS_HIP_BF16}) {
    const int64_t p = norm_parts(rows, elt, norm_form(elt, cols));
    n = p > n ? p : n;
  }
  return align_up((size_t)n * (size_t)cols * 4, 256);
}

extern "C" int reels_hip_rms_norm_bwd(const void* dy, const void* s, const void* dsum, const void* weight, int w_dtype,
                                      const float* rstd, int dtype, int64_t rows, int64_t cols, void* dx, float* dw,
                                      void* workspace, size_t ws_bytes, void* stream) {
  using namespace reels;
  clear_error();
  const char* fn = "reels_hip_rms_norm_bwd";
  const hipStream_t st = (hipStream_t)stream;
  if (int rc = norm_check(fn, dtype, w_dtype, weight, rows, cols)) return rc;
  if (dw != nullptr && (workspace == nullptr || ws_bytes < reels_hip_rms_norm_workspace_bytes(rows, cols)))
    return fail(REELS_HIP_EWORKSPACE, std::string(fn) + ": dw needs a workspace of reels_hip_rms_norm_workspace_bytes");
  if (rows > 0 && (dy == nullptr || s == nullptr || rstd == nullptr || dx == nullptr))
    return fail(REELS_HIP_EINVAL, std::string(fn) + ": NULL operand");
  if (rows == 0 && dw == nullptr) return REELS_HIP_OK;
  NormBwdArgs a{dy, s, dsum, weight, rstd, dx, (float*)workspace, rows, cols, 1.0 / (double)cols, w_dtype == REELS_HIP_F32 && dtype != REELS_HIP_F32};
  const Form f = norm_form(dtype, cols);
  if (((dw == nullptr || f.tpr == 0) && !norm_fits(rows, f)) || (dw != nullptr && !grid_fits(ceil_div(cols, 32), 1024)))
    return fail(REELS_HIP_EINVAL, std::string(fn) + ": too many rows or columns for one launch");
  const int64_t parts = rows == 0 ? 0 : norm_parts(rows, dtype, f);
  if (rows > 0) {
    TraceScope _ts(st, "norm_bwd_kernel");
    with_any_elt(dtype, [&](auto e) {
      constexpr int E = decltype(e)::value;
      if (f.tpr == 0) {
        norm_bwd_long_kernel<E><<<(unsigned)rows, kLongThreads, 0, st>>>(a);
        if (dw != nullptr) norm_dw_long_kernel<E><<<dim3((unsigned)ceil_div(cols, 256), (unsigned)parts), 256, 0, st>>>(a);
        return;
      }
      with_form<E>(f, [&](auto tpr, auto nch) {
        constexpr int T = decltype(tpr)::value, C = decltype(nch)::value, NT = T < 256 ? 256 : T;
        if (dw != nullptr) norm_bwd_kernel<E, T, C, true><<<(unsigned)parts, NT, 0, st>>>(a);
        else norm_bwd_kernel<E, T, C, false><<<(unsigned)ceil_div(rows, NT / T), NT, 0, st>>>(a);
      });
    });
  }
  if (int rc = check_launch("norm_bwd_kernel")) return rc;
  if (dw == nullptr) return REELS_HIP_OK;
  { TraceScope _ts(st, "norm_dw_kernel");
    norm_dw_kernel<<<(unsigned)ceil_div(cols, 32), 1024, 0, st>>>((const float*)workspace, (int)parts, cols, dw); }
  return check_launch("norm_dw_kernel");
}
