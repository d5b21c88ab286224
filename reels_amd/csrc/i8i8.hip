// Product of int8 rows with an int8 weight, both with one scale per row (QuantizedMatrix), with bias,
// activation and residual in its epilogue:
//
//   y[m][n] = rnd( act( xs[m] ws[n] sum_k xq[m][k] wq[n][k] + bias[n] ) + residual[m][n] )
//
// The sums are whole numbers in 32 bits (K < 2^17 products of at most 2^14 stay below 2^31), so every
// form and split gives the same bits; the epilogue runs in f32 and rounds once.
#include "vec.h"

namespace reels {
namespace {

typedef __attribute__((__vector_size__(4 * sizeof(int)))) int i32v4;

struct ProductArgs {
  const int8_t* x;       // [M][K]
  const float* xs;       // [M]
  const int8_t* w;       // [N][K]
  const float* ws;       // [N]
  const void* bias;      // [N] or nullptr
  const void* res;       // [M][N] or nullptr
  void* y;               // [M][N]
  int64_t M, K, N;
  int gelu;
};

template <int ELT> __device__ __forceinline__ float finish_one(const ProductArgs& a, int64_t m, int64_t n, int acc) {
  float v = (float)acc * a.xs[m] * a.ws[n];
  float t[1];
  if (a.bias != nullptr) {
    load_vec<ELT, 1>((const uint8_t*)a.bias + n * elt_bytes(ELT), 1, t);
    v += t[0];
  }
  if (a.gelu) v = gelu_f(v);
  if (a.res != nullptr) {
    load_vec<ELT, 1>((const uint8_t*)a.res + (m * a.N + n) * elt_bytes(ELT), 1, t);
    v += t[0];
  }
  return v;
}

// 64 x 64 outputs per workgroup, a step of 64 codes through LDS, bytes past the edges as zeros
template <int ELT>
__global__ __launch_bounds__(256) void product_any_kernel(ProductArgs a) {
  __shared__ __attribute__((aligned(16))) int8_t sx[64][80], sw[64][80];
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, l16 = lane & 15, lq = lane >> 4;
  const int64_t m0 = (int64_t)blockIdx.y * 64, n0 = (int64_t)blockIdx.x * 64;
  i32v4 acc[4] = {};
  for (int64_t k0 = 0; k0 < a.K; k0 += 64) {
    for (int i = t; i < 64 * 64; i += 256) {
      const int r = i >> 6, c = i & 63;
      const int64_t k = k0 + c;
      sx[r][c] = m0 + r < a.M && k < a.K ? a.x[(m0 + r) * a.K + k] : (int8_t)0;
      sw[r][c] = n0 + r < a.N && k < a.K ? a.w[(n0 + r) * a.K + k] : (int8_t)0;
    }
    __syncthreads();
    const i32v4 wf = *reinterpret_cast<const i32v4*>(&sw[w * 16 + l16][lq * 16]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const i32v4 xf = *reinterpret_cast<const i32v4*>(&sx[j * 16 + l16][lq * 16]);
      acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf, xf, acc[j], 0, 0, 0);
    }
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int64_t m = m0 + j * 16 + l16, n = n0 + w * 16 + lq * 4 + v;
      if (m < a.M && n < a.N) {
        const float o[1] = {finish_one<ELT>(a, m, n, acc[j][v])};
        store_vec<ELT, 1>((uint8_t*)a.y + (m * a.N + n) * elt_bytes(ELT), 1, o);
      }
    }
}

}  // namespace
}  // namespace reels

extern "C" size_t reels_hip_i8i8_workspace_bytes(int64_t M, int64_t K, int64_t N) {
  if (M < 0 || K <= 0 || N <= 0) return 0;
  return 256;
}

extern "C" int reels_hip_i8i8_linear(const int8_t* x, const float* xs, const int8_t* w, const float* ws, const void* bias,
                                     const void* residual, int activation, int dtype, int64_t M, int64_t K, int64_t N,
                                     void* y, void* workspace, size_t ws_bytes, void* stream) {
  using namespace reels;
  clear_error();
  const std::string fn = "reels_hip_i8i8_linear: ";
  const hipStream_t st = (hipStream_t)stream;
  if (!known_elt(dtype)) return fail(REELS_HIP_EDTYPE, fn + "dtype must be f32, bf16 or f16");
  if (activation != REELS_HIP_ACT_NONE && activation != REELS_HIP_ACT_GELU_TANH) return fail(REELS_HIP_EINVAL, fn + "unknown activation");
  if (M < 0 || K <= 0 || N <= 0 || K >= (1 << 17) || M > ((int64_t)1 << 31) - 1 || N > ((int64_t)1 << 31) - 1)
    return fail(REELS_HIP_EINVAL, fn + "M >= 0, 0 < K < 131072 and N > 0 required");
  if (workspace == nullptr || ws_bytes < reels_hip_i8i8_workspace_bytes(M, K, N))
    return fail(REELS_HIP_EWORKSPACE, fn + "workspace of reels_hip_i8i8_workspace_bytes required");
  if (M == 0) return REELS_HIP_OK;
  if (x == nullptr || xs == nullptr || w == nullptr || ws == nullptr || y == nullptr) return fail(REELS_HIP_EINVAL, fn + "NULL operand");
  const ProductArgs a{x, xs, w, ws, bias, residual, y, M, K, N, activation == REELS_HIP_ACT_GELU_TANH};
  // grid.y holds 65535 tiles: more tokens run as consecutive launches
  for (int64_t m0 = 0; m0 < M; m0 += 65535 * 64) {
    ProductArgs c = a;
    c.M = M - m0 < 65535 * 64 ? M - m0 : 65535 * 64;
    c.x = a.x + m0 * K;
    c.xs = a.xs + m0;
    if (a.res) c.res = (const uint8_t*)a.res + m0 * N * elt_bytes(dtype);
    c.y = (uint8_t*)a.y + m0 * N * elt_bytes(dtype);
    TraceScope _ts(st, "product_any_kernel");
    with_any_elt(dtype, [&](auto e) {
      product_any_kernel<decltype(e)::value><<<dim3((unsigned)ceil_div(N, 64), (unsigned)ceil_div(c.M, 64)), 256, 0, st>>>(c);
    });
    if (int rc = check_launch("product_any_kernel")) return rc;
  }
  return REELS_HIP_OK;
}
