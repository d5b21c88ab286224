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
// All of it is bound by memory: each kernel reads its operands once and keeps the row in registers
// between the reduction and the output. A row belongs to a group of TPR threads that hold NCH
// 16-byte chunks each: TPR is the smallest of 16, 64, 256 and 1024 whose threads need at most four
// chunks, so short rows (one head) share a wave and long ones have many loads in flight; rows past
// 4096 chunks (32768 16-bit elements) run the loop form, which reads the row again from L2. Squares
// and products are summed in 64 bits (MI355X adds those at the rate of 32-bit ones), so rows of any
// magnitude that the type holds have the norm that they should.
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
  float eps;
  int w_f32;         // w holds f32 (else the row's type)
};

// sum (or maximum) over the TPR threads of a row's group; slot: per-block LDS, one per wave
template <int TPR, bool MAX> __device__ __forceinline__ double row_reduce(double v, double* slot) {
  constexpr int G = TPR < 64 ? TPR : 64;
  v = MAX ? group_max<G>(v) : group_sum<G>(v);
  if constexpr (TPR > 64) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) slot[wave] = v;
    __syncthreads();
    const int first = wave / (TPR / 64) * (TPR / 64);
    v = slot[first];
#pragma unroll
    for (int i = 1; i < TPR / 64; ++i) v = MAX ? fmax(v, slot[first + i]) : v + slot[first + i];
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

// the 127 steps of a row: |p| with every non-finite value as infinity, which the maximum keeps
__device__ __forceinline__ double quant_abs(double p) {
  const double a = fabs(p);
  return a <= 1.7976931348623157e308 ? a : __builtin_inf();
}
// round_ties_even(127 p / top): the product with the reciprocal is within 2^-50 of the quotient, so
// only values next to a border take the division
__device__ __forceinline__ int quant_code(double p, double top, double inv) {
  double t = p * inv, k = rint(t);
  if (fabs(t - k) > 0.4999999999) k = rint(127.0 * p / top);
  return (int)k;
}

template <int V> __device__ __forceinline__ void store_codes(int8_t* q, int left, const int (&c)[V]) {
  struct Pack { int8_t e[V]; };
  if (left >= V) {
    Pack p;
#pragma unroll
    for (int i = 0; i < V; ++i) p.e[i] = (int8_t)c[i];
    store_any(q, p);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < left) q[i] = (int8_t)c[i];
  }
}

template <int ELT, int TPR, int NCH, bool QUANT>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void norm_kernel(NormArgs a) {
  constexpr int V = 16 / elt_bytes(ELT), EB = elt_bytes(ELT), NT = TPR < 256 ? 256 : TPR;
  __shared__ double slots[2][NT / 64];
  const int lane = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * (NT / TPR) + threadIdx.x / TPR;
  const bool live = row < a.rows;  // a group past the end takes part in the barriers
  float s[NCH][V];
  double ss = 0.0;
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int64_t c = (int64_t)(lane + TPR * i) * V;
    const int left = live && c < a.cols ? (a.cols - c < V ? (int)(a.cols - c) : V) : 0;
    if (left <= 0) {
#pragma unroll
      for (int j = 0; j < V; ++j) s[i][j] = 0.0f;
      continue;
    }
    load_vec<ELT, V>((const uint8_t*)a.x + (row * a.ld_x + c) * EB, left, s[i]);
    if (a.res != nullptr) {
      float r[V];
      load_vec<ELT, V>((const uint8_t*)a.res + (row * a.ld_r + c) * EB, left, r);
#pragma unroll
      for (int j = 0; j < V; ++j) s[i][j] = Store<ELT>::get(Store<ELT>::put(s[i][j] + r[j]));
    }
  }
#pragma unroll
  for (int i = 0; i < NCH; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) ss = fma((double)s[i][j], (double)s[i][j], ss);
  ss = row_reduce<TPR, false>(ss, slots[0]);
  const double rstd = 1.0 / sqrt(ss / (double)a.cols + (double)a.eps);
  float w[NCH][V];
  double top = 0.0;
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int64_t c = (int64_t)(lane + TPR * i) * V;
    const int left = live && c < a.cols ? (a.cols - c < V ? (int)(a.cols - c) : V) : 0;
    if (left <= 0) continue;
    if (a.res != nullptr) store_vec<ELT, V>((uint8_t*)a.sum + (row * a.cols + c) * EB, left, s[i]);
    load_weight<ELT, V>(a.w, a.w_f32, c, left, w[i]);
    if constexpr (QUANT) {
#pragma unroll
      for (int j = 0; j < V; ++j) top = fmax(top, quant_abs((double)s[i][j] * (double)w[i][j]));
    } else {
      const float rs = (float)rstd;
      float y[V];
#pragma unroll
      for (int j = 0; j < V; ++j) y[j] = s[i][j] * rs * w[i][j];
      store_vec<ELT, V>((uint8_t*)a.y + (row * a.cols + c) * EB, left, y);
    }
  }
  if constexpr (QUANT) {
    top = row_reduce<TPR, true>(top, slots[1]);
    float scale = (float)(top * rstd / 127.0);
    const bool whole = __builtin_isfinite(scale);
    if (!whole) scale = __builtin_nanf("");
    if (top == 0.0 && whole) scale = 1.0f;
    if (live && lane == 0) a.scales[row] = scale;
    const bool zero = !whole || top == 0.0;
    const double inv = 127.0 / top;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int64_t c = (int64_t)(lane + TPR * i) * V;
      const int left = live && c < a.cols ? (a.cols - c < V ? (int)(a.cols - c) : V) : 0;
      if (left <= 0) continue;
      int code[V];
#pragma unroll
      for (int j = 0; j < V; ++j) code[j] = zero ? 0 : quant_code((double)s[i][j] * (double)w[i][j], top, inv);
      store_codes<V>(a.q + row * a.cols + c, left, code);
    }
  } else if (live && lane == 0) {
    a.rstd[row] = (float)rstd;
  }
}

// rows past the register form: one workgroup per row, the row read again for its output
template <int ELT, bool QUANT>
__global__ __launch_bounds__(kLongThreads) void norm_long_kernel(NormArgs a) {
  constexpr int V = 16 / elt_bytes(ELT), EB = elt_bytes(ELT);
  __shared__ double slots[2][kLongThreads / 64];
  const int64_t row = blockIdx.x;
  double ss = 0.0, top = 0.0;
  auto load_sum = [&](int64_t c, int left, float (&s)[V]) {
    load_vec<ELT, V>((const uint8_t*)a.x + (row * a.ld_x + c) * EB, left, s);
    if (a.res != nullptr) {
      float r[V];
      load_vec<ELT, V>((const uint8_t*)a.res + (row * a.ld_r + c) * EB, left, r);
#pragma unroll
      for (int j = 0; j < V; ++j) s[j] = Store<ELT>::get(Store<ELT>::put(s[j] + r[j]));
    }
  };
  for (int64_t c = (int64_t)threadIdx.x * V; c < a.cols; c += kLongThreads * V) {
    const int left = a.cols - c < V ? (int)(a.cols - c) : V;
    float s[V], w[V];
    load_sum(c, left, s);
#pragma unroll
    for (int j = 0; j < V; ++j) ss = fma((double)s[j], (double)s[j], ss);
    if constexpr (QUANT) {
      load_weight<ELT, V>(a.w, a.w_f32, c, left, w);
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (j < left) top = fmax(top, quant_abs((double)s[j] * (double)w[j]));
    }
  }
  ss = row_reduce<kLongThreads, false>(ss, slots[0]);
  const double rstd = 1.0 / sqrt(ss / (double)a.cols + (double)a.eps);
  float scale = 1.0f;
  bool zero = false;
  double inv = 0.0;
  if constexpr (QUANT) {
    top = row_reduce<kLongThreads, true>(top, slots[1]);
    scale = (float)(top * rstd / 127.0);
    const bool whole = __builtin_isfinite(scale);
    if (!whole) scale = __builtin_nanf("");
    if (top == 0.0 && whole) scale = 1.0f;
    zero = !whole || top == 0.0;
    inv = 127.0 / top;
    if (threadIdx.x == 0) a.scales[row] = scale;
  } else if (threadIdx.x == 0) {
    a.rstd[row] = (float)rstd;
  }
  // the sum is written here, after every read of x and the residual's first pass, chunk by chunk by
  // the thread that read it, so it may take the place of x or of the residual
  for (int64_t c = (int64_t)threadIdx.x * V; c < a.cols; c += kLongThreads * V) {
    const int left = a.cols - c < V ? (int)(a.cols - c) : V;
    float s[V], w[V];
    load_sum(c, left, s);
    load_weight<ELT, V>(a.w, a.w_f32, c, left, w);
    if (a.res != nullptr) store_vec<ELT, V>((uint8_t*)a.sum + (row * a.cols + c) * EB, left, s);
    if constexpr (QUANT) {
      int code[V];
#pragma unroll
      for (int j = 0; j < V; ++j) code[j] = zero ? 0 : quant_code((double)s[j] * (double)w[j], top, inv);
      store_codes<V>(a.q + row * a.cols + c, left, code);
    } else {
      const float rs = (float)rstd;
      float y[V];
#pragma unroll
      for (int j = 0; j < V; ++j) y[j] = s[j] * rs * w[j];
      store_vec<ELT, V>((uint8_t*)a.y + (row * a.cols + c) * EB, left, y);
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
  int w_f32;
};

// A workgroup walks the rows b, b + gridDim, ... (times the rows it holds at once): with dw each
// thread keeps the sums of its own columns in registers over all its rows, and the groups of a
// workgroup add theirs in LDS in group order, one partial row per workgroup.
template <int ELT, int TPR, int NCH, bool DW>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void norm_bwd_kernel(NormBwdArgs a) {
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
    const int64_t row = r0 + group;
    const bool live = row < a.rows;
    const float rstd = live ? a.rstd[row] : 0.0f;
    float s[NCH][V], g[NCH][V];
    double gs = 0.0;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int64_t c = (int64_t)(lane + TPR * i) * V;
      const int left = live && c < a.cols ? (a.cols - c < V ? (int)(a.cols - c) : V) : 0;
      if (left <= 0) {
#pragma unroll
        for (int j = 0; j < V; ++j) s[i][j] = g[i][j] = 0.0f;
        continue;
      }
      load_vec<ELT, V>((const uint8_t*)a.s + (row * a.cols + c) * EB, left, s[i]);
      load_vec<ELT, V>((const uint8_t*)a.dy + (row * a.cols + c) * EB, left, g[i]);
    }
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int64_t c = (int64_t)(lane + TPR * i) * V;
      const int left = live && c < a.cols ? (a.cols - c < V ? (int)(a.cols - c) : V) : 0;
      if (left <= 0) continue;
      float w[V];
      load_weight<ELT, V>(a.w, a.w_f32, c, left, w);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if constexpr (DW) dw[i][j] += g[i][j] * (s[i][j] * rstd);
        g[i][j] *= w[j];
        gs = fma((double)g[i][j], (double)s[i][j], gs);
      }
    }
    // two slots in turn: a wave may enter the next row's reduction while another still reads this one's
    gs = row_reduce<TPR, false>(gs, slots[turn]);
    const float k = (float)(gs / (double)a.cols * (double)rstd * (double)rstd);
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int64_t c = (int64_t)(lane + TPR * i) * V;
      const int left = live && c < a.cols ? (a.cols - c < V ? (int)(a.cols - c) : V) : 0;
      if (left <= 0) continue;
      float d[V];
#pragma unroll
      for (int j = 0; j < V; ++j) d[j] = rstd * (g[i][j] - s[i][j] * k);
      if (a.dsum != nullptr) {
        float t[V];
        load_vec<ELT, V>((const uint8_t*)a.dsum + (row * a.cols + c) * EB, left, t);
#pragma unroll
        for (int j = 0; j < V; ++j) d[j] += t[j];
      }
      store_vec<ELT, V>((uint8_t*)a.dx + (row * a.cols + c) * EB, left, d);
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
  const float k = (float)(gs / (double)a.cols * (double)rstd * (double)rstd);
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

// dw[c] = sum over the partial rows in order of 16 slices: 64 columns x 16 slices per workgroup
__global__ __launch_bounds__(1024) void norm_dw_kernel(const float* __restrict__ part, int n, int64_t cols,
                                                       float* __restrict__ dw) {
  __shared__ float acc[16][64];
  const int x = threadIdx.x & 63, y = threadIdx.x >> 6;
  const int64_t c = (int64_t)blockIdx.x * 64 + x;
  float t = 0.0f;
  if (c < cols)
    for (int r = y; r < n; r += 16) t += part[(int64_t)r * cols + c];
  acc[y][x] = t;
  __syncthreads();
  if (y == 0 && c < cols) {
#pragma unroll
    for (int i = 1; i < 16; ++i) t += acc[i][x];
    dw[c] = t;
  }
}

// ---- host ------------------------------------------------------------------------------------
struct Form { int tpr, nch; };  // tpr 0: the loop form
Form norm_form(int elt, int64_t cols) {
  const int64_t chunks = ceil_div(cols, 16 / elt_bytes(elt));
  for (int tpr : {16, 64, 256, 1024})
    if (chunks <= 4 * tpr) return {tpr, (int)ceil_div(chunks, tpr)};
  return {0, 0};
}

template <int N> using Int = std::integral_constant<int, N>;
template <typename F> void with_form(Form f, F&& g) {
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
    default: nch(Int<1024>{}); break;
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
  const Form f = norm_form(dtype, a.cols);
  { TraceScope _ts(st, label);
    with_any_elt(dtype, [&](auto e) {
      constexpr int E = decltype(e)::value;
      if (f.tpr == 0) {
        if (quant) norm_long_kernel<E, true><<<(unsigned)a.rows, kLongThreads, 0, st>>>(a);
        else norm_long_kernel<E, false><<<(unsigned)a.rows, kLongThreads, 0, st>>>(a);
        return;
      }
      with_form(f, [&](auto tpr, auto nch) {
        constexpr int T = decltype(tpr)::value, C = decltype(nch)::value, NT = T < 256 ? 256 : T;
        const unsigned grid = (unsigned)ceil_div(a.rows, NT / T);
        if (quant) norm_kernel<E, T, C, true><<<grid, NT, 0, st>>>(a);
        else norm_kernel<E, T, C, false><<<grid, NT, 0, st>>>(a);
      });
    }); }
  return check_launch(label);
}

// workgroups of the backward with dw (each writes one partial row): enough to fill the GPU
int64_t norm_parts(int64_t rows, Form f) {
  const int64_t rpb = f.tpr == 0 ? 1 : (f.tpr < 256 ? 256 / f.tpr : 1);
  const int64_t want = f.tpr == 0 ? 64 : (f.tpr <= 256 ? 1024 : 256), need = ceil_div(rows, rpb);
  return need < want ? need : want;
}

}  // namespace
}  // namespace reels

extern "C" int reels_hip_rms_norm(const void* x, int64_t ld_x, const void* residual, int64_t ld_r, const void* weight,
                                  int w_dtype, int dtype, int64_t rows, int64_t cols, float eps, void* sum, void* y,
                                  float* rstd, void* stream) {
  using namespace reels;
  return norm_forward("reels_hip_rms_norm", "norm_kernel", false,
                      NormArgs{x, residual, weight, sum, y, rstd, nullptr, nullptr, ld_x, ld_r, rows, cols, eps, 0}, dtype,
                      w_dtype, (hipStream_t)stream);
}

extern "C" int reels_hip_rms_norm_i8(const void* x, int64_t ld_x, const void* residual, int64_t ld_r, const void* weight,
                                     int w_dtype, int dtype, int64_t rows, int64_t cols, float eps, void* sum, int8_t* q,
                                     float* scales, void* stream) {
  using namespace reels;
  return norm_forward("reels_hip_rms_norm_i8", "norm_kernel<int8>", true,
                      NormArgs{x, residual, weight, sum, nullptr, nullptr, q, scales, ld_x, ld_r, rows, cols, eps, 0}, dtype,
                      w_dtype, (hipStream_t)stream);
}

extern "C" size_t reels_hip_rms_norm_workspace_bytes(int64_t rows, int64_t cols) {
  using namespace reels;
  if (rows < 0 || cols <= 0) return 0;
  // the most partial rows of any element type
  int64_t n = 1;
  for (int elt : {REELS_HIP_F32, REELS_HIP_BF16}) {
    const int64_t p = norm_parts(rows, norm_form(elt, cols));
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
  NormBwdArgs a{dy, s, dsum, weight, rstd, dx, (float*)workspace, rows, cols, w_dtype == REELS_HIP_F32 && dtype != REELS_HIP_F32};
  const Form f = norm_form(dtype, cols);
  const int64_t parts = rows == 0 ? 0 : norm_parts(rows, f);
  if (rows > 0) {
    TraceScope _ts(st, "norm_bwd_kernel");
    with_any_elt(dtype, [&](auto e) {
      constexpr int E = decltype(e)::value;
      if (f.tpr == 0) {
        norm_bwd_long_kernel<E><<<(unsigned)rows, kLongThreads, 0, st>>>(a);
        if (dw != nullptr) norm_dw_long_kernel<E><<<dim3((unsigned)ceil_div(cols, 256), (unsigned)parts), 256, 0, st>>>(a);
        return;
      }
      with_form(f, [&](auto tpr, auto nch) {
        constexpr int T = decltype(tpr)::value, C = decltype(nch)::value, NT = T < 256 ? 256 : T;
        if (dw != nullptr) norm_bwd_kernel<E, T, C, true><<<(unsigned)parts, NT, 0, st>>>(a);
        else norm_bwd_kernel<E, T, C, false><<<(unsigned)ceil_div(rows, NT / T), NT, 0, st>>>(a);
      });
    });
  }
  if (int rc = check_launch("norm_bwd_kernel")) return rc;
  if (dw == nullptr) return REELS_HIP_OK;
  { TraceScope _ts(st, "norm_dw_kernel");
    norm_dw_kernel<<<(unsigned)ceil_div(cols, 64), 1024, 0, st>>>((const float*)workspace, (int)parts, cols, dw); }
  return check_launch("norm_dw_kernel");
}
