// The norm between two sublayers of a transformer block whose output is modulated by the conditioning
// (the reference's modulation, src/layers/modulation.jl:2-11, layernorm of src/layers/linear.jl and rmsnorm),
// with the gated residual before it in the same pass. Forward; the backward is in modnorm_bwd.hip.
//
//   s = rnd(x + gate b)        (the product and the sum rounded to f32, then to the type; x + b without a gate)
//   n = (s - mean) rstd,  rstd = (mean_c (s - mean)^2 + eps)^(-1/2)      (mean = 0 for the root-mean-square norm)
//   y = rnd(n (1 + scale) + shift)
//   kept: s and b as 8-bit blocks for the backward;  4 bits: y's row as 4-bit blocks instead of y
//
// gate, scale and shift have one row for each group of rows (a sample's tokens, or a single token).
// Bound by memory: x and b are read once, s and y written once, the row stays in registers between the two
// reductions (the mean first, then the squares about it: with rows far from zero the difference of two large
// sums would lose the variance). Both are summed in 64 bits; the mean is kept as two f32 values, so that
// s - mean loses nothing where the mean is many times the spread. Rows in 4 bits are formed in 64 bits and
// rounded to f32 before their codes are taken, so a code does not depend on the order of f32 operations.
#include "modnorm.h"

namespace reels {
namespace {

struct ModArgs {
  const void *x, *branch, *gate, *scale, *shift;  // branch, gate, and scale with shift: or nullptr
  void *sum, *y;
  float* stats;            // [rows][3]: the mean in two parts, rstd
  int8_t *ks, *kb;         // kept codes of the sum and of the branch (nullptr: none)
  uint8_t *kss, *kbs;
  uint8_t *codes, *scales; // rows in 4 bits
  int64_t ld_x, ld_b, ld_gate, ld_scale, ld_shift, rows, cols, rpg;
  double per_col;
  float eps;
  int center, m_f32;
};

// the 8-bit codes of a thread's chunk of a row (all lanes take part; lanes past the row hold zeros)
template <int V>
__device__ __forceinline__ void keep_chunk(const float (&f)[V], int8_t* codes, uint8_t* scales, int64_t row, int col, int cols) {
  const uint32_t byte = mx_exponent<7>(mx_top<kMxBlock / V>(mx_top_of<V>(f)));
  if (col >= cols) return;
  uint32_t word[V / 4];
  mx8_codes<V>(f, byte, word);
  mx8_store<V>(codes + row * cols + col, cols - col, word);
  if (col % kMxBlock == 0) scales[row * ((cols + kMxBlock - 1) / kMxBlock) + col / kMxBlock] = (uint8_t)byte;
}

// MODE 0: y; 1: y and the kept rows; 2: y's rows in 4 bits
template <int ELT, int TPR, int NCH, int MODE>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void mod_kernel(ModArgs a) {
  constexpr int V = Chunk<ELT>::V, EB = elt_bytes(ELT), NT = TPR < 256 ? 256 : TPR;
  __shared__ double slots[2][NT / 64];
  // rows in 4 bits: neighbours share lines of scale bytes, so each XCD takes a run of rows
  unsigned wg = blockIdx.x;
  if constexpr (MODE == 2) {
    const unsigned n = gridDim.x, xcd = wg & 7;
    wg = xcd * (n >> 3) + (xcd < (n & 7) ? xcd : n & 7) + (wg >> 3);
  }
  const int64_t row0 = (int64_t)wg * (NT / TPR) + threadIdx.x / TPR;
  const Row<ELT, TPR, NCH> at(a.cols, row0 < a.rows);
  const int64_t row = at.live ? row0 : a.rows - 1;
  const int64_t group = (uint32_t)row / (uint32_t)a.rpg;
  Chunk<ELT> s[NCH], b[NCH];
  float m[NCH][V];
  at.load((const uint8_t*)a.x + row * a.ld_x * EB, s);
  if (a.branch != nullptr) {
    at.load((const uint8_t*)a.branch + row * a.ld_b * EB, b);
    if (a.gate != nullptr) load_mod(at, a.gate, a.ld_gate, a.m_f32, group, m);
  }
  double t = 0.0;
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    if (!at.some(i)) continue;
    if (a.branch != nullptr) {
      float f[V];
      {
#pragma clang fp contract(off)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float p = a.gate != nullptr ? m[i][j] * b[i].get(j) : b[i].get(j);
          f[j] = s[i].get(j) + p;
        }
      }
      // a lane without a chunk holds zeros in x and b; its gate is another's and may be infinite
      if (!at.full(i)) {
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] = at.live && j < at.left(i) ? f[j] : 0.0f;
      }
      s[i].pack(f);
      at.store((uint8_t*)a.sum + row * a.cols * EB, i, s[i]);
      if constexpr (MODE == 1) {
        if (a.kb != nullptr) {
          b[i].unpack(f);
          keep_chunk<V>(f, a.kb, a.kbs, row, at.live ? at.col(i) : at.cols, at.cols);
        }
      }
    }
    if constexpr (MODE == 1) {
      float f[V];
      s[i].unpack(f);
      keep_chunk<V>(f, a.ks, a.kss, row, at.live ? at.col(i) : at.cols, at.cols);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) t += (double)s[i].get(j);
    s[i].hold();
  }
  double mean = 0.0;
  if (a.center) mean = row_reduce<TPR, false>(t, slots[0]) * a.per_col;
  double ss = 0.0;
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    if (!at.some(i)) continue;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const double d = (double)s[i].get(j) - mean;
      if (at.full(i) || (at.part(i) && j < at.left(i))) ss = fma(d, d, ss);
    }
    s[i].hold();
  }
  ss = row_reduce<TPR, false>(ss, slots[1]);
  const double rstd = rsqrt64(fma(ss, a.per_col, (double)a.eps));
  const float hi = (float)mean, lo = (float)(mean - (double)hi), rs = (float)rstd;
  float h[NCH][V];
  if (a.scale != nullptr) {
    load_mod(at, a.scale, a.ld_scale, a.m_f32, group, m);
    load_mod(at, a.shift, a.ld_shift, a.m_f32, group, h);
  } else {
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) m[i][j] = h[i][j] = 0.0f;
  }
  if constexpr (MODE < 2) {
    if (at.live && at.lane == 0) {
      float* st = a.stats + row * 3;
      st[0] = hi;
      st[1] = lo;
      st[2] = rs;
    }
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      if (!at.some(i)) continue;
      float y[V];
      Chunk<ELT> o;
#pragma unroll
      for (int j = 0; j < V; ++j) y[j] = fmaf((s[i].get(j) - hi - lo) * rs, 1.0f + m[i][j], h[i][j]);
      o.pack(y);
      at.store((uint8_t*)a.y + row * a.cols * EB, i, o);
    }
  } else {
    const int tiles = (at.cols + 255) / 256;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      if (!at.some(i)) continue;
      float y[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const double n = ((double)s[i].get(j) - mean) * rstd;
        y[j] = (float)fma(n, 1.0 + (double)m[i][j], (double)h[i][j]);
        if (!at.full(i)) y[j] = j < at.left(i) ? y[j] : 0.0f;  // zeros up to the tile's end
      }
      const uint32_t byte = mx_exponent<2>(mx_top<kMxBlock / V>(mx_top_of<V>(y)));
      const int col = at.col(i);
      if (!at.live || col >= tiles * 256) continue;
      const uint32_t word = mx4_codes<V>(y, byte);
      uint8_t* p = a.codes + row * tiles * 128 + col / 2;
      if constexpr (V == 8) *reinterpret_cast<uint32_t*>(p) = word;
      else *reinterpret_cast<uint16_t*>(p) = (uint16_t)word;
      if (col % kMxBlock == 0) a.scales[mx4_scale_at(row, col / kMxBlock, tiles)] = (uint8_t)byte;
    }
  }
}

int mod_forward(const char* fn, const char* label, int mode, ModArgs a, int dtype, int m_dtype, hipStream_t st) {
  clear_error();
  if (int rc = mod_check(fn, dtype, m_dtype, a.rows, a.cols, a.rpg)) return rc;
  if (!(a.eps >= 0.0f && a.eps <= 3.4e38f)) return fail(REELS_HIP_EINVAL, std::string(fn) + ": eps must be finite and not negative");
  if (a.rows == 0) return REELS_HIP_OK;
  if ((a.scale == nullptr) != (a.shift == nullptr)) return fail(REELS_HIP_EINVAL, std::string(fn) + ": scale and shift go together");
  if (a.gate != nullptr && a.branch == nullptr) return fail(REELS_HIP_EINVAL, std::string(fn) + ": a gate needs a branch");
  if (a.ld_x < a.cols || (a.branch != nullptr && a.ld_b < a.cols))
    return fail(REELS_HIP_EINVAL, std::string(fn) + ": row strides below cols");
  if ((a.ks == nullptr) != (a.kss == nullptr) || (a.kb == nullptr) != (a.kbs == nullptr) || (a.kb != nullptr && (a.ks == nullptr || a.branch == nullptr)))
    return fail(REELS_HIP_EINVAL, std::string(fn) + ": kept codes and scales go together, the branch's with the sum's");
  if (a.x == nullptr || (a.branch != nullptr && a.sum == nullptr) ||
      (mode == 2 ? a.codes == nullptr || a.scales == nullptr : a.y == nullptr || a.stats == nullptr))
    return fail(REELS_HIP_EINVAL, std::string(fn) + ": NULL operand");
  if (mode == 2 && ((uintptr_t)a.codes & 3) != 0) return fail(REELS_HIP_EINVAL, std::string(fn) + ": codes must be 4-byte aligned");
  a.m_f32 = m_dtype == REELS_HIP_F32 && dtype != REELS_HIP_F32;
  a.per_col = 1.0 / (double)a.cols;
  const ModForm f = mod_form(dtype, a.cols);
  const int threads = f.tpr < 256 ? 256 : f.tpr;
  const int64_t grid = ceil_div(a.rows, threads / f.tpr);
  if (!grid_fits(grid, threads)) return fail(REELS_HIP_EINVAL, std::string(fn) + ": too many rows for one launch");
  { TraceScope _ts(st, label);
    with_any_elt(dtype, [&](auto e) {
      constexpr int E = decltype(e)::value;
      with_mod_form<E>(f, [&](auto tpr, auto nch) {
        constexpr int T = decltype(tpr)::value, C = decltype(nch)::value, NT = T < 256 ? 256 : T;
        if (mode == 2) mod_kernel<E, T, C, 2><<<(unsigned)grid, NT, 0, st>>>(a);
        else if (a.ks != nullptr) mod_kernel<E, T, C, 1><<<(unsigned)grid, NT, 0, st>>>(a);
        else mod_kernel<E, T, C, 0><<<(unsigned)grid, NT, 0, st>>>(a);
      });
    }); }
  return check_launch(label);
}

}  // namespace
}  // namespace reels

extern "C" int reels_hip_modulated_norm(const void* x, int64_t ld_x, const void* branch, int64_t ld_branch, const void* gate,
                                        int64_t ld_gate, const void* scale, int64_t ld_scale, const void* shift, int64_t ld_shift,
                                        int m_dtype, int dtype, int64_t rows, int64_t cols, int64_t rows_per_group, float eps,
                                        int center, void* sum, void* y, float* stats, int8_t* kept_sum, uint8_t* kept_sum_scales,
                                        int8_t* kept_branch, uint8_t* kept_branch_scales, void* stream) {
  using namespace reels;
  ModArgs a{};
  a.x = x; a.branch = branch; a.gate = gate; a.scale = scale; a.shift = shift;
  a.sum = sum; a.y = y; a.stats = stats;
  a.ks = kept_sum; a.kss = kept_sum_scales; a.kb = kept_branch; a.kbs = kept_branch_scales;
  a.ld_x = ld_x; a.ld_b = ld_branch; a.ld_gate = ld_gate; a.ld_scale = ld_scale; a.ld_shift = ld_shift;
  a.rows = rows; a.cols = cols; a.rpg = rows_per_group; a.eps = eps; a.center = center != 0;
  return mod_forward("reels_hip_modulated_norm", kept_sum ? "mod_kernel<kept>" : "mod_kernel", 0, a, dtype, m_dtype, (hipStream_t)stream);
}

extern "C" int reels_hip_modulated_norm_mx4(const void* x, int64_t ld_x, const void* branch, int64_t ld_branch, const void* gate,
                                            int64_t ld_gate, const void* scale, int64_t ld_scale, const void* shift,
                                            int64_t ld_shift, int m_dtype, int dtype, int64_t rows, int64_t cols,
                                            int64_t rows_per_group, float eps, int center, void* sum, uint8_t* codes,
                                            uint8_t* scales, void* stream) {
  using namespace reels;
  ModArgs a{};
  a.x = x; a.branch = branch; a.gate = gate; a.scale = scale; a.shift = shift;
  a.sum = sum; a.codes = codes; a.scales = scales;
  a.ld_x = ld_x; a.ld_b = ld_branch; a.ld_gate = ld_gate; a.ld_scale = ld_scale; a.ld_shift = ld_shift;
  a.rows = rows; a.cols = cols; a.rpg = rows_per_group; a.eps = eps; a.center = center != 0;
  return mod_forward("reels_hip_modulated_norm_mx4", "mod_kernel<4 bits>", 2, a, dtype, m_dtype, (hipStream_t)stream);
}
