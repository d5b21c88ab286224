// Activations kept in 8 bits for the backward (microscale.h): a matrix to its blocks and back, the GELU that
// keeps its input on the way, and its pullback from the blocks (gelu_f and gelu_grad_f of common.h on the
// values that the blocks stand for).
//
// Bound by memory. A thread has 16 bytes of the matrix and 32 / V neighbours share a block, whose largest
// magnitude goes through their lanes; one pass over the data, every thread one chunk, streamed past the caches
// where nothing reads it soon. Rows whose length is no multiple of 32 end in a short block of their own.
// 32760 x 13824 bf16: the GELU that keeps its input 373 us (6.1 TB/s), the values back 228 (6.0), the pullback
// 415 (5.5).
#include "microscale.h"

namespace reels {
namespace {

constexpr int kT = 256;

// A thread's chunk: where it stands in the matrix and in the bytes of the blocks, how many elements of its row
// are left there (0: the thread has none), and the row's length. Threads are dealt to whole blocks, so that the
// lanes of a block are neighbours also where it is the short one at a row's end. FLAT: rows are whole blocks,
// so the matrix is one long row and nothing is divided by its length.
struct Spot { int64_t at, byte; int left, cols; };
template <int V, bool FLAT> __device__ __forceinline__ Spot spot(int64_t rows, int64_t cols, int blocks) {
  constexpr int L = kMxBlock / V;  // lanes of a block
  const int64_t t = (int64_t)blockIdx.x * kT + threadIdx.x, b = t / L;
  if constexpr (FLAT) return {t * V, b, t * V < rows * cols ? V : 0, V};
  const int64_t row = b / blocks;
  const int col = (int)(b - row * blocks) * kMxBlock + (int)(t % L) * V;
  return {row * cols + col, b, row < rows ? (int)cols - col : 0, (int)cols};
}

template <int ELT> __device__ __forceinline__ Chunk<ELT> stream_in(const void* p, int left) {
  Chunk<ELT> c;
  c.zero();
  if (left > 0) c.load(p, left);
  return c;
}

template <int ELT, bool FLAT, bool GELU>
__global__ __launch_bounds__(kT) void keep_kernel(const void* __restrict__ x, int64_t rows, int64_t cols, int blocks, void* __restrict__ y,
                                                  int8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  constexpr int V = Chunk<ELT>::V, EB = elt_bytes(ELT);
  const Spot p = spot<V, FLAT>(rows, cols, blocks);
  const Chunk<ELT> c = stream_in<ELT>((const uint8_t*)x + p.at * EB, p.left);
  float f[V];
  c.unpack(f);
  const uint32_t byte = mx_exponent<7>(mx_top<kMxBlock / V>(mx_top_of<V>(f)));
  if (p.left <= 0) return;
  uint32_t word[V / 4];
  mx8_codes<V>(f, byte, word);
  mx8_store<V>(codes + p.at, p.left, word);
  if (threadIdx.x % (kMxBlock / V) == 0) scales[p.byte] = (uint8_t)byte;
  if constexpr (GELU) {
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = gelu_f(f[j]);
    store_vec<ELT, V>((uint8_t*)y + p.at * EB, p.left, f);
  }
}

// BWD: dy gelu'(value); otherwise the values
template <int ELT, bool FLAT, bool BWD>
__global__ __launch_bounds__(kT) void restore_kernel(const int8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t rows,
                                                     int64_t cols, int blocks, const void* dy, void* out) {
  constexpr int V = Chunk<ELT>::V, EB = elt_bytes(ELT);
  const Spot p = spot<V, FLAT>(rows, cols, blocks);
  if (p.left <= 0) return;
  Codes<V> q;
  q.load(codes + p.at, p.left, p.cols);
  q.unit = mx8_unit(scales[p.byte]);
  float f[V];
#pragma unroll
  for (int j = 0; j < V; ++j) f[j] = q.get(j);
  if constexpr (BWD) {
    float d[V];
    load_vec<ELT, V>((const uint8_t*)dy + p.at * EB, p.left, d);
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = d[j] * gelu_grad_f(f[j]);
  } else if constexpr (ELT == REELS_HIP_F16) {
    // a block's largest values can round up to 65536, past the type's range
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = f[j] == f[j] ? __builtin_amdgcn_fmed3f(f[j], -65504.0f, 65504.0f) : f[j];
  }
  store_vec<ELT, V>((uint8_t*)out + p.at * EB, p.left, f);
}

struct Shape { int64_t rows, cols, grid; int blocks; bool flat; };
int shape_of(const std::string& fn, int dtype, int64_t rows, int64_t cols, Shape& s) {
  if (!known_elt(dtype)) return fail(REELS_HIP_EDTYPE, fn + "dtype must be f32, bf16 or f16");
  if (rows < 0 || cols <= 0 || cols > ((int64_t)1 << 30) || rows > ((int64_t)1 << 31) - 1)
    return fail(REELS_HIP_EINVAL, fn + "0 <= rows < 2^31 and 0 < cols <= 2^30 required");
  s.rows = rows;
  s.cols = cols;
  s.blocks = (int)ceil_div(cols, kMxBlock);
  s.flat = cols % kMxBlock == 0;
  s.grid = ceil_div(rows * s.blocks * (kMxBlock * elt_bytes(dtype) / 16), kT);
  if (!grid_fits(s.grid, kT)) return fail(REELS_HIP_EINVAL, fn + "too many elements for one launch");
  return REELS_HIP_OK;
}

int keep(const char* name, const char* label, const void* x, int dtype, int64_t rows, int64_t cols, void* y, int8_t* codes,
         uint8_t* scales, void* stream, bool gelu) {
  clear_error();
  const std::string fn = std::string(name) + ": ";
  Shape s;
  if (int rc = shape_of(fn, dtype, rows, cols, s)) return rc;
  if (rows == 0) return REELS_HIP_OK;
  if (x == nullptr || codes == nullptr || scales == nullptr || (gelu && y == nullptr)) return fail(REELS_HIP_EINVAL, fn + "NULL operand");
  const hipStream_t st = (hipStream_t)stream;
  { TraceScope _ts(st, label);
    with_any_elt(dtype, [&](auto e) {
      constexpr int E = decltype(e)::value;
      auto go = [&](auto flat) {
        constexpr bool F = decltype(flat)::value;
        if (gelu) keep_kernel<E, F, true><<<(unsigned)s.grid, kT, 0, st>>>(x, s.rows, s.cols, s.blocks, y, codes, scales);
        else keep_kernel<E, F, false><<<(unsigned)s.grid, kT, 0, st>>>(x, s.rows, s.cols, s.blocks, y, codes, scales);
      };
      if (s.flat) go(std::true_type{});
      else go(std::false_type{});
    }); }
  return check_launch(label);
}

int restore(const char* name, const char* label, const int8_t* codes, const uint8_t* scales, int dtype, int64_t rows, int64_t cols,
            const void* dy, void* out, void* stream, bool bwd) {
  clear_error();
  const std::string fn = std::string(name) + ": ";
  Shape s;
  if (int rc = shape_of(fn, dtype, rows, cols, s)) return rc;
  if (rows == 0) return REELS_HIP_OK;
  if (codes == nullptr || scales == nullptr || out == nullptr || (bwd && dy == nullptr)) return fail(REELS_HIP_EINVAL, fn + "NULL operand");
  const hipStream_t st = (hipStream_t)stream;
  { TraceScope _ts(st, label);
    with_any_elt(dtype, [&](auto e) {
      constexpr int E = decltype(e)::value;
      auto go = [&](auto flat) {
        constexpr bool F = decltype(flat)::value;
        if (bwd) restore_kernel<E, F, true><<<(unsigned)s.grid, kT, 0, st>>>(codes, scales, s.rows, s.cols, s.blocks, dy, out);
        else restore_kernel<E, F, false><<<(unsigned)s.grid, kT, 0, st>>>(codes, scales, s.rows, s.cols, s.blocks, dy, out);
      };
      if (s.flat) go(std::true_type{});
      else go(std::false_type{});
    }); }
  return check_launch(label);
}

}  // namespace
}  // namespace reels

extern "C" int reels_hip_act8_keep(const void* x, int dtype, int64_t rows, int64_t cols, int8_t* codes, uint8_t* scales, void* stream) {
  return reels::keep("reels_hip_act8_keep", "keep_kernel", x, dtype, rows, cols, nullptr, codes, scales, stream, false);
}
extern "C" int reels_hip_act8_gelu_tanh(const void* x, int dtype, int64_t rows, int64_t cols, void* y, int8_t* codes, uint8_t* scales,
                                        void* stream) {
  return reels::keep("reels_hip_act8_gelu_tanh", "keep_kernel<gelu>", x, dtype, rows, cols, y, codes, scales, stream, true);
}
extern "C" int reels_hip_act8_restore(const int8_t* codes, const uint8_t* scales, int dtype, int64_t rows, int64_t cols, void* x,
                                      void* stream) {
  return reels::restore("reels_hip_act8_restore", "restore_kernel", codes, scales, dtype, rows, cols, nullptr, x, stream, false);
}
extern "C" int reels_hip_act8_gelu_tanh_bwd(const int8_t* codes, const uint8_t* scales, const void* dy, int dtype, int64_t rows,
                                            int64_t cols, void* dx, void* stream) {
  return reels::restore("reels_hip_act8_gelu_tanh_bwd", "restore_kernel<gelu>", codes, scales, dtype, rows, cols, dy, dx, stream, true);
}
