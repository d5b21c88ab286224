// Backward of the modulated norm (modnorm.hip). With n = (s - mean) rstd and g = dy (1 + scale):
//
//   d = rstd (g - mean_c(g) - n mean_c(g n)) + dsum      (mean_c(g) = 0 for the root-mean-square norm)
//   dx = rnd(d), dbranch = rnd(d gate);  dgate = sum d b, dscale = sum dy n, dshift = sum dy   (f32)
//
// s and the branch come as they were stored, or from their 8-bit blocks, which are read in 33 bytes for 64.
// Bound by memory: dy, s, b and dsum are read once and dx, dbranch written once (32760 x 5120 bf16 400 us and 9
// for the sums' second launch, 4.9 TB/s; from 8 bits 334 in all, without the modulations' gradients 344, with a
// modulation for each token 967, 5.6 TB/s). Rows past 8192 elements, and f32 past 2048, are bound by registers as
// well: with the sums up to 54 of a lane's are spilled, the most in f32 from 8 bits (4000 x 13824 370 us, 2.7 TB/s).
//
// The sums over a group's rows stay in the registers of the threads that own the columns: a workgroup walks every
// parts-th row of one group and leaves one partial row of each sum, which a second launch adds in order (no
// atomics, so the results are bitwise reproducible). Groups of one row (a modulation for each token) write their
// gradients from the same pass.
//
// One source file per element type (modnorm_bwd_*.hip) instantiates launch_mod_bwd.
#pragma once
#include "modnorm.h"

namespace reels {

struct ModBwdArgs {
  const void *dy, *s, *dsum, *branch, *gate, *scale;  // dsum, branch, gate, scale: or nullptr
  const uint8_t *ss, *bs;                             // bytes of the blocks of s and branch
  const float* stats;
  void *dx, *db;                                      // db with a gate only
  float *dgate, *dscale, *dshift;                     // [groups][cols], or nullptr (dshift with dscale)
  float* part;                                        // [groups][parts][3][cols] where parts > 1
  int64_t ld_gate, ld_scale, rows, cols, rpg, run;    // run: rows that follow each other in a wave or workgroup
  double per_col;
  int center, m_f32, parts;
  float far;
};

template <int ELT> void launch_mod_bwd(const ModBwdArgs& a, ModForm f, bool kept, bool sums, int64_t grid, hipStream_t st);

}  // namespace reels
