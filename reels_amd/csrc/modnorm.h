// What the forward and the backward of the modulated norm share.
#pragma once
#include "microscale.h"
#include "rows.h"

namespace reels {

struct ModForm { int tpr, nch; };

namespace {

// Threads of a row and its chunks a thread: a wave up to 256 chunks, 256 threads up to 1024, and 512 (f32:
// 1024 past 2048 chunks) up to 16384 elements, the longest row.
constexpr int64_t kModCols = 16384;
inline ModForm mod_form(int elt, int64_t cols) {
  const int64_t chunks = ceil_div(cols, 16 / elt_bytes(elt));
  for (int tpr : {64, 256, 512})
    if (chunks <= 4 * tpr) return {tpr, (int)ceil_div(chunks, tpr)};
  return {1024, (int)ceil_div(chunks, 1024)};
}
template <int ELT, typename F> void with_mod_form(ModForm f, F&& g) {
  auto some = [&](auto tpr) {
    if (f.nch == 2) g(tpr, Int<2>{});
    else if (f.nch == 3) g(tpr, Int<3>{});
    else g(tpr, Int<4>{});
  };
  switch (f.tpr) {
    case 64:
      if (f.nch == 1) g(Int<64>{}, Int<1>{});
      else some(Int<64>{});
      break;
    case 256: some(Int<256>{}); break;
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

// Modulations: [groups][cols] rows ld elements apart, f32 or the rows' type. A thread's values of a chunk
// that it has not are those of another one.
template <typename R, int N, int V>
__device__ __forceinline__ void load_mod(const R& at, const void* p, int64_t ld, int f32, int64_t group, float (&f)[N][V]) {
  at.load_w((const uint8_t*)p + group * ld * (f32 ? 4 : R::EB), f32, f);
}

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
