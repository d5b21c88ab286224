// Rotary positions with several axes (time, height, width), the reference's _rope!
// (src/layers/rope.jl:13-32), for the queries and the keys of one attention in one launch.
//
//   pair j of axis a (axis_pairs[a] pairs, the axes one after the other): angle = pos[token][a] *
//   theta^(-j / axis_pairs[a]);  (u, v) -> (u cos - v sin, u sin + v cos)
//   interleaved: pair p is elements 2p, 2p + 1; else p and p + P, P the number of pairs. Elements
//   past 2P are copied. The backward is the rotation by the negative angle (inverse).
//
// Bound by memory: one read and one write of q and k (32760 tokens of 80 heads of 128 in bf16: 225-252 us,
// 5.3-6.0 TB/s). A token's angles are shared by all its heads and by q and k, so a workgroup computes them
// once for its tokens into LDS. An angle is formed in turns in 64 bits (pos times the frequency over
// 2 pi) and only its fraction is taken to sine and cosine in 32 bits, so its reduction loses nothing: it
// is off by the roundings of the 64-bit frequency and product, at most (j + 2) 2^-52 of itself.
#include "vec.h"

#include <cmath>

namespace reels {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 256, kMaxAxes = 4;

struct RotaryArgs {
  const void* x[2];          // q, k
  void* y[2];
  const void* pos;           // [B or 1][S][axes] f32 or int32
  int64_t ld[2];             // token strides of q and k (elements); a batch is S of them
  int64_t pos_batch;         // tokens from one batch's positions to the next's (0: shared)
  int64_t tokens;            // B S
  int S, D, P, axes, tb;     // tb: tokens of a workgroup
  int heads[2];
  int pos_i32, inverse;
  int axis_end[kMaxAxes];    // pairs up to and with axis a
  double freq[kMaxPairs];    // turns per position of each pair
};

// Items of a head: interleaved V elements (V/2 pairs); else V pairs (their V lower and V upper
// elements) and after them V copied elements each. One item a thread and turn: four with their loads in
// flight before the angles take more registers and are slower (32760 x 80 heads 268 -> 293 us).
template <int ELT, int V, bool INTERLEAVED>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs a) {
  constexpr int EB = elt_bytes(ELT);
  extern __shared__ float2 turn[];  // [tb][P] cosine, sine
  const int64_t t0 = (int64_t)blockIdx.x * a.tb;
  const int nt = (int)(a.tokens - t0 < a.tb ? a.tokens - t0 : a.tb);
  for (int i = threadIdx.x; i < nt * a.P; i += kThreads) {
    const int tok = i / a.P, p = i - tok * a.P;
    int axis = 0;
    while (axis + 1 < a.axes && p >= a.axis_end[axis]) ++axis;
    const int64_t t = t0 + tok, b = t / a.S, s = t - b * a.S;
    const int64_t at = ((a.pos_batch ? b * a.pos_batch : 0) + s) * a.axes + axis;
    const double pos = a.pos_i32 ? (double)((const int32_t*)a.pos)[at] : (double)((const float*)a.pos)[at];
    const double r = pos * a.freq[p];
    float sn, cs;
    sincospif((float)(2.0 * (r - rint(r))), &sn, &cs);
    turn[i] = make_float2(cs, a.inverse ? -sn : sn);
  }
  __syncthreads();
  const int per_head = INTERLEAVED ? a.D / V : a.P / V + (a.D - 2 * a.P) / V;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    if (a.x[which] == nullptr) continue;
    const int H = a.heads[which], items = H * per_head;
    for (int i = threadIdx.x; i < nt * items; i += kThreads) {
      const int tok = i / items, rest = i - tok * items;
      const int head = rest / per_head, it = rest - head * per_head;
      const int64_t t = t0 + tok;
      const uint8_t* x = (const uint8_t*)a.x[which] + (t * a.ld[which] + (int64_t)head * a.D) * EB;
      uint8_t* y = (uint8_t*)a.y[which] + (t * H + head) * (int64_t)a.D * EB;
      const float2* cs = turn + tok * a.P;
      if constexpr (INTERLEAVED) {
        float e[V];
        load_vec<ELT, V>(x + it * V * EB, V, e);
#pragma unroll
        for (int j = 0; j < V; j += 2) {
          const int p = it * (V / 2) + j / 2;
          if (p < a.P) {
            const float2 c = cs[p];
            const float u = e[j], v = e[j + 1];
            e[j] = u * c.x - v * c.y;
            e[j + 1] = u * c.y + v * c.x;
          }
        }
        store_vec<ELT, V>(y + it * V * EB, V, e);
      } else {
        const int p = it * V;
        if (p < a.P) {
          float u[V], v[V];
          load_vec<ELT, V>(x + p * EB, V, u);
          load_vec<ELT, V>(x + (a.P + p) * EB, V, v);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float2 c = cs[p + j];
            const float uu = u[j], vv = v[j];
            u[j] = uu * c.x - vv * c.y;
            v[j] = uu * c.y + vv * c.x;
          }
          store_vec<ELT, V>(y + p * EB, V, u);
          store_vec<ELT, V>(y + (a.P + p) * EB, V, v);
        } else {
          float e[V];
          const int at = (a.P + p) * EB;
          load_vec<ELT, V>(x + at, V, e);
          store_vec<ELT, V>(y + at, V, e);
        }
      }
    }
  }
}

}  // namespace
}  // namespace reels

extern "C" int reels_hip_rotary(const void* q, int64_t ld_q, const void* k, int64_t ld_k, const void* pos, int pos_dtype,
                                int64_t pos_batches, int dtype, int64_t B, int64_t S, int64_t Hq, int64_t Hk, int64_t D,
                                const int32_t* axis_pairs, int axes, float theta, int interleaved, int inverse, void* yq,
                                void* yk, void* stream) {
  using namespace reels;
  clear_error();
  const hipStream_t st = (hipStream_t)stream;
  const std::string fn = "reels_hip_rotary: ";
  if (!known_elt(dtype)) return fail(REELS_HIP_EDTYPE, fn + "dtype must be f32, bf16 or f16");
  if (pos_dtype != REELS_HIP_F32 && pos_dtype != REELS_HIP_I32) return fail(REELS_HIP_EDTYPE, fn + "positions must be f32 or int32");
  if (B < 0 || S < 0 || Hq < 0 || Hk < 0 || D <= 0 || D % 2 != 0 || D > 2 * kMaxPairs)
    return fail(REELS_HIP_EINVAL, fn + "sizes must not be negative and D an even head dim up to 512");
  if (S > ((int64_t)1 << 30) || B > ((int64_t)1 << 30) || B * S > ((int64_t)1 << 31) - 1 || Hq * D > (1 << 24) || Hk * D > (1 << 24) ||
      Hq > (1 << 24) || Hk > (1 << 24))
    return fail(REELS_HIP_EINVAL, fn + "at most 2^31 - 1 tokens of at most 2^24 elements");
  if (axes < 1 || axes > kMaxAxes || axis_pairs == nullptr) return fail(REELS_HIP_EINVAL, fn + "1 to 4 axes required");
  if (!(theta > 0.0f && theta <= 3.4e38f)) return fail(REELS_HIP_EINVAL, fn + "theta must be finite and positive");
  if (pos_batches != 1 && pos_batches != B) return fail(REELS_HIP_EINVAL, fn + "positions of one batch or of every batch");
  RotaryArgs a{};
  int64_t P = 0;
  for (int x = 0; x < axes; ++x) {
    if (axis_pairs[x] < 0 || P + axis_pairs[x] > D / 2) return fail(REELS_HIP_EINVAL, fn + "the axes' pairs must not be negative nor exceed D / 2 together");
    // turns per position: theta^(-j / n) / (2 pi), the powers by repeated products of one root in 64 bits
    double f = 0.15915494309189533577;
    const double root = axis_pairs[x] > 0 ? std::pow((double)theta, -1.0 / axis_pairs[x]) : 1.0;
    for (int j = 0; j < axis_pairs[x]; ++j, f *= root) a.freq[P + j] = f;
    P += axis_pairs[x];
    a.axis_end[x] = (int)P;
  }
  if (B * S == 0 || (Hq == 0 && Hk == 0)) return REELS_HIP_OK;
  if (pos == nullptr || (Hq > 0 && (q == nullptr || yq == nullptr)) || (Hk > 0 && (k == nullptr || yk == nullptr)))
    return fail(REELS_HIP_EINVAL, fn + "NULL operand");
  if ((Hq > 0 && ld_q < Hq * D) || (Hk > 0 && ld_k < Hk * D)) return fail(REELS_HIP_EINVAL, fn + "token strides below the heads' elements");
  a.x[0] = Hq > 0 ? q : nullptr; a.x[1] = Hk > 0 ? k : nullptr;
  a.y[0] = yq; a.y[1] = yk;
  a.pos = pos; a.pos_i32 = pos_dtype == REELS_HIP_I32;
  a.ld[0] = ld_q; a.ld[1] = ld_k;
  a.pos_batch = pos_batches == 1 ? 0 : S;
  a.tokens = B * S;
  a.S = (int)S; a.D = (int)D; a.P = (int)P; a.axes = axes; a.inverse = inverse != 0;
  a.heads[0] = (int)Hq; a.heads[1] = (int)Hk;
  // tokens of a workgroup: about 32 KiB, so that the angles are a small part of its work, but no more
  // than leaves 2048 workgroups (1560 tokens of 6 KiB: 11.2 us in workgroups of five, 8.2 one by one)
  const int64_t token_bytes = (Hq + Hk) * D * elt_bytes(dtype);
  int64_t tb = 32768 / token_bytes;
  if (tb > a.tokens / 2048) tb = a.tokens / 2048;
  a.tb = (int)(tb < 1 ? 1 : tb > 16 ? 16 : tb);
  const unsigned grid = (unsigned)ceil_div(a.tokens, a.tb);
  if (!grid_fits(ceil_div(a.tokens, a.tb), kThreads)) return fail(REELS_HIP_EINVAL, fn + "too many tokens for one launch");
  const size_t lds = (size_t)a.tb * P * sizeof(float2);
  // the widest vector that divides the parts of a head
  int v = 16 / elt_bytes(dtype);
  while (v > 1 && (D % v != 0 || (!interleaved && P % v != 0))) v /= 2;
  { TraceScope _ts(st, "rotary_kernel");
    with_any_elt(dtype, [&](auto e) {
      constexpr int E = decltype(e)::value;
      auto run = [&](auto vv) {
        constexpr int V = decltype(vv)::value;
        if constexpr (V > 1) {
          if (interleaved) { rotary_kernel<E, V, true><<<grid, kThreads, lds, st>>>(a); return; }
        }
        rotary_kernel<E, V, false><<<grid, kThreads, lds, st>>>(a);
      };
      if constexpr (elt_bytes(E) == 2) {
        if (v == 8) { run(std::integral_constant<int, 8>{}); return; }
      }
      if (v == 4) run(std::integral_constant<int, 4>{});
      else if (v == 2) run(std::integral_constant<int, 2>{});
      else run(std::integral_constant<int, 1>{});
    }); }
  return check_launch("rotary_kernel");
}
