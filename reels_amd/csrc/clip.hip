// Global norm of many gradient tensors and clipping by it (what the reference's training loop does
// with the adapters' gradients before the optimizer, src/training/wan_runner.jl:108-289).
//
//   norm = sqrt(sum over tensors of g^2);  out = rnd(g min(1, max_norm / (norm + 1e-6)))
//
// Bound by memory: the gradients are read for the norm and again for the scaled copy, which needs
// the finished norm. The tensors (their pointers, sizes and types) travel in kernel arguments to a
// table in the workspace, 96 at a time, so a call records into a graph and the host keeps nothing.
// The work is cut into pieces of 16384 elements, dealt to the workgroups in turn.
// Squares are summed in 64 bits, one partial per workgroup, and every workgroup of the second pass
// adds the partials in the same order: the result does not depend on the run.
#include "vec.h"

#include <algorithm>
#include <new>
#include <vector>

namespace reels {
namespace {

constexpr int kThreads = 256;
constexpr int64_t kPiece = 16384;
constexpr int kBlocks = 1024;   // workgroups of each pass: four per CU
constexpr int kBatch = 96;      // tensors per table launch (32 bytes each in 4 KiB of arguments)

struct Entry {
  const void* g;
  void* o;
  int64_t n;
  int64_t first;  // pieces before this tensor
};
// the type travels in the low bits of n's place: n < 2^61
struct Batch { Entry e[kBatch]; };

__global__ __launch_bounds__(128) void grad_table_kernel(Batch b, Entry* table, int count) {
  const int i = threadIdx.x;
  if (i < count) table[i] = b.e[i];
}

__device__ __forceinline__ int64_t entry_size(const Entry& e) { return e.n >> 2; }
__device__ __forceinline__ int entry_type(const Entry& e) { return (int)(e.n & 3); }

// Index of the tensor that holds a piece: in LDS, where a workgroup keeps the tensors' first pieces if
// they fit, else in the table
constexpr int kCached = 1024;
struct Finder {
  const Entry* table;
  int64_t* cache;
  int count;
  __device__ __forceinline__ Finder(const Entry* t, int n, int64_t* c) : table(t), cache(c), count(n) {
    if (n > kCached) return;
    for (int i = threadIdx.x; i < n; i += kThreads) c[i] = t[i].first;
    __syncthreads();
  }
  template <typename F> __device__ __forceinline__ int search(int64_t piece, F&& first) const {
    int lo = 0, hi = count - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (first(mid) <= piece) lo = mid;
      else hi = mid - 1;
    }
    return lo;
  }
  __device__ __forceinline__ int find(int64_t piece) const {
    const Entry* t = table;
    const int64_t* c = cache;
    return count <= kCached ? search(piece, [c](int i) { return c[i]; }) : search(piece, [t](int i) { return t[i].first; });
  }
};

__device__ __forceinline__ double block_sum(double v, double* slot) {
  v = group_reduce<64, false>(v);
  if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
  __syncthreads();
  v = slot[0];
#pragma unroll
  for (int i = 1; i < kThreads / 64; ++i) v += slot[i];
  return v;
}

// 16 bytes at a global address at any multiple of the element: the tensors' pointers come from memory,
// where the compiler cannot see that they are global and would take flat accesses. Nontemporal:
// each pass streams (524 MB read for the norm in 82 us, 129 without; scaled into another buffer in 191 us,
// 200 without)
typedef u32x4 __attribute__((aligned(2))) u32x4_any;
typedef __attribute__((address_space(1))) u32x4_any* global16;
__device__ __forceinline__ u32x4 load_global(const uint8_t* p) { return __builtin_nontemporal_load((global16)(uintptr_t)p); }
__device__ __forceinline__ void store_global(uint8_t* p, const u32x4& v) { __builtin_nontemporal_store((u32x4_any)v, (global16)(uintptr_t)p); }

// f(chunk, byte offset, how many exist) for this thread's chunks of a piece of n elements, eight loads in flight
template <int ELT, typename F> __device__ __forceinline__ void each_chunk(const uint8_t* g, int n, F&& f) {
  constexpr int V = Chunk<ELT>::V, U = 8, STEP = kThreads * 16;
  const int full = n / (kThreads * V);
  int it = 0, at = (int)threadIdx.x * 16;
  for (; it + U <= full; it += U, at += U * STEP) {
    Chunk<ELT> c[U];
#pragma unroll
    for (int u = 0; u < U; ++u) c[u].d = load_global(g + at + u * STEP);
#pragma unroll
    for (int u = 0; u < U; ++u) f(c[u], at + u * STEP, V);
  }
  for (; it < full; ++it, at += STEP) {
    Chunk<ELT> c;
    c.d = load_global(g + at);
    f(c, at, V);
  }
  const int left = n - at / elt_bytes(ELT);
  if (left <= 0) return;
  Chunk<ELT> c;
  c.load(g + at, left < V ? left : V);
  f(c, at, left < V ? left : V);
}

template <int ELT> __device__ __forceinline__ double piece_sum(const uint8_t* g, int n) {
  double t = 0.0;
  each_chunk<ELT>(g, n, [&](const Chunk<ELT>& c, int, int) {
#pragma unroll
    for (int j = 0; j < Chunk<ELT>::V; ++j) t = fma((double)c.get(j), (double)c.get(j), t);
  });
  return t;
}

// F: float, or double for a factor that f32 holds with fewer bits than 24 or not at all
template <int ELT, typename F> __device__ __forceinline__ void piece_scale(const uint8_t* g, uint8_t* o, int n, F factor) {
  constexpr int V = Chunk<ELT>::V;
  each_chunk<ELT>(g, n, [&](const Chunk<ELT>& c, int at, int left) {
    float f[V];
    Chunk<ELT> d;
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = (float)((F)c.get(j) * factor);
    d.pack(f);
    if (left == V) store_global(o + at, d.d);
    else d.store(o + at, left);
  });
}

template <typename F> __device__ __forceinline__ void with_type(int t, F&& f) {
  if (t == REELS_HIP_F32) f(std::integral_constant<int, REELS_HIP_F32>{});
  else if (t == REELS_HIP_F16) f(std::integral_constant<int, REELS_HIP_F16>{});
  else f(std::integral_constant<int, REELS_HIP_BF16>{});
}

// f(entry, element offset, elements) for every piece of this workgroup: neighbouring workgroups take
// neighbouring pieces (each its own run of pieces put all of them on the same memory channels at a
// time: 5% more). The second pass goes backwards, from what the first has read last.
template <bool BACK, typename F> __device__ __forceinline__ void each_piece(const Finder& at, int64_t pieces, F&& f) {
  const int64_t n = (pieces - blockIdx.x + gridDim.x - 1) / gridDim.x;
  for (int64_t i = 0; i < n; ++i) {
    const int64_t p = blockIdx.x + (BACK ? n - 1 - i : i) * gridDim.x;
    const Entry e = at.table[at.find(p)];
    const int64_t off = (p - e.first) * kPiece, left = entry_size(e) - off;
    f(e, off, left < kPiece ? left : kPiece);
  }
}

__global__ __launch_bounds__(kThreads) void grad_sum_kernel(const Entry* table, int count, int64_t pieces, double* part) {
  __shared__ double slot[kThreads / 64];
  __shared__ int64_t cache[kCached];
  const Finder at(table, count, cache);
  double t = 0.0;
  each_piece<false>(at, pieces, [&](const Entry& e, int64_t off, int64_t n) {
    with_type(entry_type(e), [&](auto ty) {
      constexpr int E = decltype(ty)::value;
      t += piece_sum<E>((const uint8_t*)e.g + off * elt_bytes(E), (int)n);
    });
  });
  t = block_sum(t, slot);
  if (threadIdx.x == 0) part[blockIdx.x] = t;
}

__device__ __forceinline__ double total_norm(const double* part, int n, double* slot) {
  double t = 0.0;
  for (int i = threadIdx.x; i < n; i += kThreads) t += part[i];
  return sqrt(block_sum(t, slot));
}

__global__ __launch_bounds__(kThreads) void grad_norm_kernel(const double* part, int n, float* norm) {
  __shared__ double slot[kThreads / 64];
  const double t = total_norm(part, n, slot);
  if (threadIdx.x == 0) *norm = (float)t;
}

__global__ __launch_bounds__(kThreads) void grad_scale_kernel(const Entry* table, int count, int64_t pieces,
                                                              const double* part, int n, float max_norm, float* norm) {
  __shared__ double slot[kThreads / 64];
  __shared__ int64_t cache[kCached];
  const Finder at(table, count, cache);
  const double t = total_norm(part, n, slot);
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)t;
  // gradients whose norm, as it is returned, is not finite are left as they are: a factor of 0 or NaN
  // would hide which of them it came from
  const double f = (double)max_norm / (t + 1e-6);
  const float factor = __builtin_isfinite((float)t) && f < 1.0 ? (float)f : 1.0f;
  const bool small = factor < 1.0f && f > 0.0 && f < 0x1p-126;
  each_piece<true>(at, pieces, [&](const Entry& e, int64_t off, int64_t m) {
    if (factor == 1.0f && e.g == e.o) return;  // in place and nothing to clip
    with_type(entry_type(e), [&](auto ty) {
      constexpr int E = decltype(ty)::value;
      const uint8_t* g = (const uint8_t*)e.g + off * elt_bytes(E);
      uint8_t* o = (uint8_t*)e.o + off * elt_bytes(E);
      if (small) piece_scale<E>(g, o, (int)m, f);
      else piece_scale<E>(g, o, (int)m, factor);
    });
  });
}

size_t table_bytes(int64_t count) { return align_up((size_t)count * sizeof(Entry), 256); }

// two ranges overlap, one of them an output, unless they are a tensor and its own output
bool outputs_overlap(const void* const* g, void* const* o, const int64_t* n, const int32_t* ty, int64_t count) {
  // outputs that follow each other in memory (pieces of one buffer), every gradient outside them: no sort
  uintptr_t lo = 0, hi = 0;
  bool rising = true;
  for (int64_t i = 0; i < count && rising; ++i) {
    if (n[i] == 0) continue;
    rising = (uintptr_t)o[i] >= hi;
    if (lo == 0) lo = (uintptr_t)o[i];
    hi = (uintptr_t)o[i] + (uintptr_t)n[i] * elt_bytes(ty[i]);
  }
  for (int64_t i = 0; i < count && rising; ++i)
    rising = n[i] == 0 || g[i] == o[i] || (uintptr_t)g[i] >= hi || (uintptr_t)g[i] + (uintptr_t)n[i] * elt_bytes(ty[i]) <= lo;
  if (rising) return false;
  struct Span { uintptr_t a, b; bool out; };
  std::vector<Span> v;
  v.reserve((size_t)count * 2);
  for (int64_t i = 0; i < count; ++i) {
    const uintptr_t bytes = (uintptr_t)n[i] * elt_bytes(ty[i]);
    if (bytes == 0) continue;
    v.push_back({(uintptr_t)o[i], (uintptr_t)o[i] + bytes, true});
    if (g[i] != o[i]) v.push_back({(uintptr_t)g[i], (uintptr_t)g[i] + bytes, false});
  }
  std::sort(v.begin(), v.end(), [](const Span& x, const Span& y) { return x.a < y.a; });
  uintptr_t end_any = 0, end_out = 0;
  for (const Span& s : v) {
    if (s.a < end_out || (s.out && s.a < end_any)) return true;
    end_any = std::max(end_any, s.b);
    if (s.out) end_out = std::max(end_out, s.b);
  }
  return false;
}

int clip_run(const char* name, const void* const* grads, void* const* outs, const int64_t* sizes, const int32_t* dtypes,
             int64_t count, bool clip, float max_norm, float* norm, void* workspace, size_t ws_bytes, hipStream_t st) {
  clear_error();
  const std::string fn = std::string(name) + ": ";
  if (count < 0 || count > ((int64_t)1 << 24)) return fail(REELS_HIP_EINVAL, fn + "0 to 2^24 tensors required");
  if (norm == nullptr || (count > 0 && (grads == nullptr || sizes == nullptr || dtypes == nullptr || (clip && outs == nullptr))))
    return fail(REELS_HIP_EINVAL, fn + "NULL operand");
  if (clip && !(max_norm >= 0.0f)) return fail(REELS_HIP_EINVAL, fn + "max_norm must not be negative or NaN");
  if (workspace == nullptr || ws_bytes < reels_hip_grad_workspace_bytes(count))
    return fail(REELS_HIP_EWORKSPACE, fn + "workspace of reels_hip_grad_workspace_bytes required");
  int64_t pieces = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (!known_elt(dtypes[i])) return fail(REELS_HIP_EDTYPE, fn + "dtypes must be f32, bf16 or f16");
    if (sizes[i] < 0 || sizes[i] > ((int64_t)1 << 48)) return fail(REELS_HIP_EINVAL, fn + "bad tensor size");
    if (sizes[i] > 0 && (grads[i] == nullptr || (clip && outs[i] == nullptr))) return fail(REELS_HIP_EINVAL, fn + "NULL tensor");
    pieces += ceil_div(sizes[i], kPiece);
  }
  if (clip && outputs_overlap(grads, outs, sizes, dtypes, count))
    return fail(REELS_HIP_EINVAL, fn + "an output overlaps another tensor (the same gradient twice?)");
  Entry* table = (Entry*)workspace;
  double* part = (double*)((uint8_t*)workspace + table_bytes(count));
  int64_t used = 0, first = 0;
  Batch b;
  int in = 0;
  auto flush = [&]() -> int {
    if (in == 0) return REELS_HIP_OK;
    { TraceScope _ts(st, "grad_table_kernel");
      grad_table_kernel<<<1, 128, 0, st>>>(b, table + used, in); }
    used += in;
    in = 0;
    return check_launch("grad_table_kernel");
  };
  for (int64_t i = 0; i < count; ++i) {
    if (sizes[i] == 0) continue;
    b.e[in++] = Entry{grads[i], clip ? outs[i] : nullptr, sizes[i] << 2 | dtypes[i], first};
    first += ceil_div(sizes[i], kPiece);
    if (in == kBatch)
      if (int rc = flush()) return rc;
  }
  if (int rc = flush()) return rc;
  const int grid = (int)(pieces < kBlocks ? (pieces > 0 ? pieces : 1) : kBlocks);
  { TraceScope _ts(st, "grad_sum_kernel");
    grad_sum_kernel<<<grid, kThreads, 0, st>>>(table, (int)used, pieces, part); }
  if (int rc = check_launch("grad_sum_kernel")) return rc;
  TraceScope _ts(st, clip ? "grad_scale_kernel" : "grad_norm_kernel");
  if (clip) grad_scale_kernel<<<grid, kThreads, 0, st>>>(table, (int)used, pieces, part, grid, max_norm, norm);
  else grad_norm_kernel<<<1, kThreads, 0, st>>>(part, grid, norm);
  return check_launch("grad_scale_kernel");
}

// nothing thrown crosses the C boundary (the overlap check allocates)
template <typename F> int guarded(const char* fn, F&& f) {
  try {
    return f();
  } catch (const std::bad_alloc&) {
    return fail(REELS_HIP_EINVAL, std::string(fn) + ": out of host memory");
  }
}

}  // namespace
}  // namespace reels

extern "C" size_t reels_hip_grad_workspace_bytes(int64_t count) {
  using namespace reels;
  if (count < 0 || count > ((int64_t)1 << 24)) return 0;
  return table_bytes(count) + kBlocks * sizeof(double);
}

extern "C" int reels_hip_grad_norm(const void* const* grads, const int64_t* sizes, const int32_t* dtypes, int64_t count,
                                   float* norm, void* workspace, size_t ws_bytes, void* stream) {
  using namespace reels;
  return guarded("reels_hip_grad_norm", [&] {
    return clip_run("reels_hip_grad_norm", grads, nullptr, sizes, dtypes, count, false, 0.0f, norm, workspace, ws_bytes,
                    (hipStream_t)stream);
  });
}

extern "C" int reels_hip_clip_gradients(const void* const* grads, void* const* outs, const int64_t* sizes,
                                        const int32_t* dtypes, int64_t count, float max_norm, float* norm,
                                        void* workspace, size_t ws_bytes, void* stream) {
  using namespace reels;
  return guarded("reels_hip_clip_gradients", [&] {
    return clip_run("reels_hip_clip_gradients", grads, outs, sizes, dtypes, count, true, max_norm, norm, workspace,
                    ws_bytes, (hipStream_t)stream);
  });
}
