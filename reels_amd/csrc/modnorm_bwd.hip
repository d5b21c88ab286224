// Host side of the modulated norm's backward (modnorm_bwd.h), and the pass that adds the partial sums.
#include "modnorm_bwd.h"

namespace reels {
namespace {

// sums of the partial rows: 32 columns x 32 slices per workgroup, slice y adds the rows y, y + 32, ... and
// the slices follow in order. part [groups][parts][3][cols]; grid (columns, 3, groups)
__global__ __launch_bounds__(1024) void mod_sum_kernel(const float* __restrict__ part, int parts, int64_t cols, float* __restrict__ dgate,
                                                       float* __restrict__ dscale, float* __restrict__ dshift) {
  __shared__ float acc[32][33];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5, which = blockIdx.y;
  float* out = which == 0 ? dgate : which == 1 ? dscale : dshift;
  if (out == nullptr) return;
  const int64_t c = (int64_t)blockIdx.x * 32 + x, group = blockIdx.z;
  float t = 0.0f;
  if (c < cols) {
#pragma unroll 4
    for (int r = y; r < parts; r += 32) t += part[((group * parts + r) * 3 + which) * cols + c];
  }
  acc[y][x] = t;
  __syncthreads();
  if (y == 0 && c < cols) {
#pragma unroll
    for (int i = 1; i < 32; ++i) t += acc[i][x];
    out[group * cols + c] = t;
  }
}


// Walkers (waves or workgroups) of a group's rows with the sums: together as many workgroups as the GPU holds
// at once by their registers (12 waves of a CU), and at least two rows for each. A workgroup's partial row of f32
// sums is written and read again, 24 bytes a column, which shows where it has few rows: 2 x 1560 x 1536 f16 14 MB
// beside 48 of the call's own, the second launch 4.3 of 19 us; twice the rows a partial row were level there and
// slower at 512 rows. {partial rows, rows that follow each other}
struct ModParts { int64_t parts, run; };
ModParts mod_parts(int64_t groups, int64_t rpg, ModForm f) {
  const int64_t walkers = mod_walkers(f), wgs = 256 * (12 * 64 / f.threads > 0 ? 12 * 64 / f.threads : 1);
  const int64_t share = ceil_div(wgs, groups) * walkers;
  int64_t run = ceil_div(rpg, share);
  if (run < 2) run = 2;
  const int64_t parts = ceil_div(rpg, run * walkers);
  return {parts, parts * walkers};
}

}  // namespace
}  // namespace reels

extern "C" size_t reels_hip_modulated_norm_workspace_bytes(int64_t rows, int64_t cols, int64_t rows_per_group) {
  using namespace reels;
  if (rows <= 0 || cols <= 0 || cols > kModCols || rows_per_group <= 1) return 0;
  const int64_t groups = ceil_div(rows, rows_per_group);
  int64_t n = 0;
  for (int elt : {REELS_HIP_F32, REELS_HIP_BF16}) {  // the most of any element type
    const int64_t p = mod_parts(groups, rows_per_group, mod_form(elt, rows, cols)).parts;
    n = p > n ? p : n;
  }
  return n <= 1 ? 0 : align_up((size_t)(groups * n) * 3 * (size_t)cols * 4, 256);
}

extern "C" int reels_hip_modulated_norm_bwd(const void* dy, const void* s, const uint8_t* s_scales, const void* dsum,
                                            const void* branch, const uint8_t* branch_scales, const void* gate, int64_t ld_gate,
                                            const void* scale, int64_t ld_scale, const float* stats, int m_dtype, int dtype,
                                            int64_t rows, int64_t cols, int64_t rows_per_group, int center, void* dx,
                                            void* dbranch, float* dgate, float* dscale, float* dshift, void* workspace,
                                            size_t ws_bytes, void* stream) {
  using namespace reels;
  clear_error();
  const char* fn = "reels_hip_modulated_norm_bwd";
  const hipStream_t st = (hipStream_t)stream;
  if (int rc = mod_check(fn, dtype, m_dtype, rows, cols, rows_per_group)) return rc;
  if (rows == 0) return REELS_HIP_OK;
  if ((gate == nullptr) != (dbranch == nullptr) || (dgate != nullptr && (gate == nullptr || branch == nullptr)))
    return fail(REELS_HIP_EINVAL, std::string(fn) + ": dbranch comes with a gate, dgate needs the branch too");
  if ((dscale == nullptr) != (dshift == nullptr) || (dscale != nullptr && scale == nullptr))
    return fail(REELS_HIP_EINVAL, std::string(fn) + ": dscale and dshift go together and need scale");
  if (dgate != nullptr && (s_scales == nullptr) != (branch_scales == nullptr))
    return fail(REELS_HIP_EINVAL, std::string(fn) + ": s and branch are both kept in 8 bits or neither");
  if (dy == nullptr || s == nullptr || stats == nullptr || dx == nullptr) return fail(REELS_HIP_EINVAL, std::string(fn) + ": NULL operand");
  const ModForm f = mod_form(dtype, rows, cols);
  const int64_t groups = rows / rows_per_group;
  const bool sums = rows_per_group > 1 && (dgate != nullptr || dscale != nullptr);
  const int64_t walkers = mod_walkers(f);
  const ModParts p = sums ? mod_parts(groups, rows_per_group, f) : ModParts{1, rows};  // without sums: a row each
  const int64_t parts = p.parts;
  if (parts > 1 && (workspace == nullptr || ws_bytes < reels_hip_modulated_norm_workspace_bytes(rows, cols, rows_per_group)))
    return fail(REELS_HIP_EWORKSPACE, std::string(fn) + ": workspace of reels_hip_modulated_norm_workspace_bytes required");
  const int64_t grid = sums ? groups * parts : ceil_div(p.run, walkers);
  if (!grid_fits(grid, f.threads)) return fail(REELS_HIP_EINVAL, std::string(fn) + ": too many rows for one launch");
  const ModBwdArgs a{dy, s, dsum, branch, gate, scale, s_scales, branch_scales, stats, dx, dbranch, dgate, dscale, dshift,
                     (float*)workspace, ld_gate, ld_scale, rows, cols, rows_per_group, p.run, 1.0 / (double)cols, center != 0,
                     m_dtype == REELS_HIP_F32 && dtype != REELS_HIP_F32, (int)parts, mod_far(cols)};
  { TraceScope _ts(st, "mod_bwd_kernel");
    with_any_elt(dtype, [&](auto e) { launch_mod_bwd<decltype(e)::value>(a, f, s_scales != nullptr, sums, grid, st); }); }
  if (int rc = check_launch("mod_bwd_kernel")) return rc;
  if (parts <= 1) return REELS_HIP_OK;
  { TraceScope _ts(st, "mod_sum_kernel");
    mod_sum_kernel<<<dim3((unsigned)ceil_div(cols, 32), 3, (unsigned)groups), 1024, 0, st>>>((const float*)workspace, (int)parts, cols,
                                                                                            dgate, dscale, dshift); }
  return check_launch("mod_sum_kernel");
}
