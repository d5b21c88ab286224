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
// Bound by memory: x and b are read once, s and y written once, the row stays in registers in between. Sums
// are in 64 bits about the row's first element, which one pass over the row can take; the mean is kept as two
// f32 values, so that s - mean loses nothing where the mean is many times the spread. Rows in 4 bits are formed in 64 bits and
// rounded to f32 before their codes are taken, so a code does not depend on the order of f32 operations.
// 32760 x 5120 bf16 with branch, gate and f32 modulations: 245-257 us (5.2-5.5 TB/s; a copy of 1 GiB by 16 bytes a
// thread runs at 6.2, past the caches at 6.5), with both kept 335 (5.0 TB/s), to 4 bits 228-267 (4.1-4.8: 64-bit
// products and the blocks' maxima beside the loads). A modulation for each token, f32: 595 us (5.6 TB/s).
#include "modnorm.h"

#include <algorithm>

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
  float eps, far;
  int center, m_f32, over;  // over: the sum is written over x or the branch
};

// the 8-bit codes of a thread's chunk of a row (all lanes take part; lanes past the row hold zeros)
template <int V>
__device__ __forceinline__ void keep_chunk(const float (&f)[V], int8_t* codes, uint8_t* scales, int64_t row, int col, int cols) {
  const uint32_t byte = mx_exponent<7>(mx_top<kMxBlock / V>(mx_top_of<V>(f)));
  if (col >= cols) return;
  uint32_t word[V / 4];
  mx8_codes<V>(f, byte, word);
  // 32-bit offsets from scalar bases
  mx8_store<V>(codes + row * cols + (uint32_t)col, cols - col, word);
  if (col % kMxBlock == 0) (scales + row * ((cols + kMxBlock - 1) / kMxBlock))[(uint32_t)col / kMxBlock] = (uint8_t)byte;
}

// MODE 0: y; 1: y and the kept rows; 2: y's rows in 4 bits. A wave or workgroup walks `run` rows one after the
// other, the next row's x and b on their way meanwhile; the modulations stay in registers while the group is the
// same (as f32 they are half again what a row reads from memory).
template <int ELT, int TPR, int NCH, int NT, int KIND, int MODE>
__global__ __launch_bounds__(NT, NT == 512 ? (ELT == REELS_HIP_F32 ? 3 : 4) : 1) void mod_kernel(ModArgs a, uint32_t run) {
  constexpr int V = Chunk<ELT>::V, EB = elt_bytes(ELT);
  // f32 rows past 8192 elements leave no registers for the next row, which is asked for at a row's end
  constexpr bool AHEAD = !(NT == 1024 && ELT == REELS_HIP_F32);
  __shared__ double slots[2][16][2];
  const ModRow<ELT, TPR, NCH, KIND> at(a.cols);
  // rows in 32 bits, so that they and what follows from them stay in scalar registers (but for 16 lanes)
  const uint32_t begin = TPR == 0 ? blockIdx.x : TPR == 64 ? blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)
                                                          : blockIdx.x * 16 + (threadIdx.x >> 4);
  const uint32_t end = (uint32_t)a.rows, rpg = (uint32_t)a.rpg;
  if (begin >= end) return;
  // A row's operands on their way; raw: its first elements, which every thread needs. All loads are
  // unconditional, so that the waits for them need not count on the fewest: where there is no branch x takes
  // its place, past the last row the last one.
  typedef typename Store<ELT>::raw raw;
  struct Data { Chunk<ELT> x[NCH], b[NCH]; raw x0, b0; };
  const void* branch = a.branch != nullptr ? a.branch : a.x;
  const int64_t ld_b = a.branch != nullptr ? a.ld_b : a.ld_x;
  auto load = [&](uint32_t r, Data& d) {
    const int64_t row = r < end ? r : end - 1;
    at.load((const uint8_t*)a.x + row * a.ld_x * EB, d.x);
    at.load((const uint8_t*)branch + row * ld_b * EB, d.b);
    d.x0 = ((const raw*)a.x)[row * a.ld_x];
    d.b0 = ((const raw*)branch)[row * ld_b];
  };
  Data cur, next;
  load(begin, cur);
  float gate[NCH][V], up[NCH][V], shift[NCH][V], gate0 = 1.0f;
#pragma unroll
  for (int i = 0; i < NCH; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      gate[i][j] = 1.0f;
      up[i][j] = shift[i][j] = 0.0f;
    }
  uint32_t change = begin;
  int turn = 0;
  for (uint32_t r = begin; r < end; r += run, turn ^= 1) {
    const int64_t row = r;
    if (r >= change) {
      const uint32_t group = r / rpg;
      change = (group + 1) * rpg;
      if (a.gate != nullptr) {
        at.mods(a.gate, a.ld_gate, a.m_f32, group, gate);
        gate0 = a.m_f32 ? ((const float*)a.gate)[(int64_t)group * a.ld_gate] : Store<ELT>::get(((const raw*)a.gate)[(int64_t)group * a.ld_gate]);
      }
      if (a.scale != nullptr) {
        at.mods(a.scale, a.ld_scale, a.m_f32, group, up);
        at.mods(a.shift, a.ld_shift, a.m_f32, group, shift);
      }
      __builtin_amdgcn_s_waitcnt(0x0F70);  // here, and not at each row's use
    }
    if constexpr (AHEAD) load(r + run, next);
    // the sum, and its first element, which every thread forms for itself
    Chunk<ELT>(&s)[NCH] = cur.x;  // no branch: the row itself
    float s0 = Store<ELT>::get(cur.x0);
    at.trim(s);
    if (a.branch != nullptr) {
#pragma clang fp contract(off)
      at.trim(cur.b);
      s0 = Store<ELT>::get(Store<ELT>::put(s0 + gate0 * Store<ELT>::get(cur.b0)));
      // The sum over x or the branch: one thread is about to overwrite what all of the row's threads form s0 from,
      // so every wave has it before any stores.
      if (a.over) {
        asm volatile("" : "+v"(s0) : : "memory");
        if constexpr (TPR == 0) __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
      }
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        float f[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float p = gate[i][j] * cur.b[i].get(j);
          f[j] = s[i].get(j) + p;
        }
        s[i].pack(f);
        at.store((uint8_t*)a.sum + row * a.cols * EB, i, s[i]);
      }
      if constexpr (MODE == 1) {
        if (a.kb != nullptr) {
#pragma unroll
          for (int i = 0; i < NCH; ++i) {
            if (!at.some(i)) continue;
            float f[V];
            cur.b[i].unpack(f);
            keep_chunk<V>(f, a.kb, a.kbs, row, at.col(i), at.cols);
          }
        }
      }
    }
    if constexpr (MODE == 1) {
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        if (!at.some(i)) continue;
        float f[V];
        s[i].unpack(f);
        keep_chunk<V>(f, a.ks, a.kss, row, at.col(i), at.cols);
      }
    }
    // Sums of s - s0 and of its square in one pass. s0 is one of the row's elements, at most sqrt(cols)
    // times the spread from the mean, so the difference of the two sums loses at most log2(cols) bits of 53.
    const double pivot = a.center ? (double)s0 : 0.0;
    double sum = 0.0, sq = 0.0;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      if (at.all(i)) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const double d = (double)s[i].get(j) - pivot;
          sum += d;
          sq = fma(d, d, sq);
        }
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const double d = j < at.left(i) ? (double)s[i].get(j) - pivot : 0.0;
          sum += d;
          sq = fma(d, d, sq);
        }
      }
      s[i].hold();
    }
    row_sums<TPR>(sum, sq, slots[turn]);
    const double off = a.center ? sum * a.per_col : 0.0, mean = pivot + off;
    const double var = fmax(fma(-off, off, sq * a.per_col), 0.0) + (sum - sum);  // NaN stays
    const double rstd = rsqrt64(var + (double)a.eps);
    if constexpr (MODE < 2) {
      const float hi = (float)mean, lo = (float)(mean - (double)hi), rs = (float)rstd;
      const ModUnit n = mod_unit(hi, lo, rs, a.far);
      if (at.lane == 0) {
        float* st = a.stats + row * 3;
        st[0] = hi;
        st[1] = lo;
        st[2] = rs;
      }
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        float y[V];
        Chunk<ELT> o;
#pragma unroll
        for (int j = 0; j < V; ++j) y[j] = fmaf(fmaf(s[i].get(j) - n.hi, rs, n.k), 1.0f + up[i][j], shift[i][j]);
        o.pack(y);
        at.store((uint8_t*)a.y + row * a.cols * EB, i, o);
      }
    } else {
      const int tiles = (at.cols + 255) / 256;
      const double below = -mean * rstd;  // its rounding is 2^-53 of the mean over the spread
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        if (TPR != 16 && !at.some(i)) continue;
        float y[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          // the modulations stay in 32 bits between rows: as 64-bit values they take a workgroup's registers
          asm volatile("" : "+v"(up[i][j]), "+v"(shift[i][j]));
          y[j] = (float)fma(fma((double)s[i].get(j), rstd, below), 1.0 + (double)up[i][j], (double)shift[i][j]);
        }
        if (!at.all(i)) {  // zeros up to the tile's end
#pragma unroll
          for (int j = 0; j < V; ++j) y[j] = j < at.left(i) ? y[j] : 0.0f;
        }
        const uint32_t byte = mx_exponent<2>(mx_top<kMxBlock / V>(mx_top_of<V>(y)));
        const int col = at.col(i);
        if (col >= tiles * 256) continue;
        const uint32_t word = mx4_codes<V>(y, byte);
        uint8_t* p = a.codes + row * tiles * 128 + (uint32_t)col / 2;
        if constexpr (V == 8) *reinterpret_cast<uint32_t*>(p) = word;
        else *reinterpret_cast<uint16_t*>(p) = (uint16_t)word;
        if (col % kMxBlock == 0) (a.scales + (row >> 6) * tiles * 512)[(uint32_t)mx4_scale_at(row & 63, col / kMxBlock, tiles)] = (uint8_t)byte;
      }
    }
    if constexpr (MODE == 2 && TPR == 16 && NCH * V < 16) {  // the other half of the tile's 256 columns
      reinterpret_cast<uint32_t*>(a.codes + row * 128 + 64)[at.lane] = 0u;
      if (at.lane < 4) (a.scales + (row >> 6) * 512)[(uint32_t)mx4_scale_at(row & 63, 4 + at.lane, 1)] = 0;
    }
    if constexpr (AHEAD) cur = next;
    else load(r + run, cur);
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
  if (a.branch != nullptr && a.rows > 1 && ((a.sum == a.x && a.ld_x != a.cols) || (a.sum == a.branch && a.ld_b != a.cols)))
    return fail(REELS_HIP_EINVAL, std::string(fn) + ": sum may be x or branch only where their row stride is cols");
  a.m_f32 = m_dtype == REELS_HIP_F32 && dtype != REELS_HIP_F32;
  a.over = a.branch != nullptr && (a.sum == a.x || a.sum == a.branch);
  a.per_col = 1.0 / (double)a.cols;
  a.far = mod_far(a.cols);
  const ModForm f = mod_form(dtype, a.rows, a.cols);
  // Rows that follow each other in a wave or workgroup: as many as leave every one resident, one where
  // each row has its own modulations. Long rows take two workgroups a CU, where as many as fit queue for
  // memory: 32760 x 5120 bf16 256 us with two, 283 with three, and to 4 bits 232 and 239; 4096 wide 195 with two
  // and 206 with four. Shorter ones take all: 1536 wide 77 us with five, 81 with four, 113 with two.
  const int64_t per = mod_walkers(f), fit = 16 * 64 / f.threads;
  const int64_t resident = 256 * (f.tpr == 0 && a.cols > 2048 && f.threads >= 256 ? std::min<int64_t>(fit, 2) : fit) * per;
  const int64_t run = a.rpg == 1 || a.rows < resident ? a.rows : resident, grid = ceil_div(run, per);
  if (!grid_fits(grid, f.threads)) return fail(REELS_HIP_EINVAL, std::string(fn) + ": too many rows for one launch");
  { TraceScope _ts(st, label);
    with_any_elt(dtype, [&](auto e) {
      constexpr int E = decltype(e)::value;
      with_mod_form<E>(f, a.cols, [&](auto tpr, auto nch, auto nt, auto kind) {
        constexpr int T = decltype(tpr)::value, C = decltype(nch)::value, NT = decltype(nt)::value, Y = decltype(kind)::value;
        if (mode == 2) mod_kernel<E, T, C, NT, Y, 2><<<(unsigned)grid, f.threads, 0, st>>>(a, (uint32_t)run);
        else if (a.ks != nullptr) mod_kernel<E, T, C, NT, Y, 1><<<(unsigned)grid, f.threads, 0, st>>>(a, (uint32_t)run);
        else mod_kernel<E, T, C, NT, Y, 0><<<(unsigned)grid, f.threads, 0, st>>>(a, (uint32_t)run);
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
