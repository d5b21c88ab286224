// The kernel of the modulated norm's backward (modnorm_bwd.h).
#include "modnorm_bwd.h"

namespace reels {
namespace {

// a thread's chunks of a row of s or the branch, as stored or in 8 bits
template <int ELT, int TPR, int NCH, bool KEPT> struct Held {
  static constexpr int V = Chunk<ELT>::V;
  Chunk<ELT> d[NCH];
  __device__ __forceinline__ void load(const Row<ELT, TPR, NCH>& at, const void* p, const uint8_t*, int64_t row) {
    at.load((const uint8_t*)p + row * at.cols * elt_bytes(ELT), d);
  }
  __device__ __forceinline__ float get(int i, int j) const { return d[i].get(j); }
};
template <int ELT, int TPR, int NCH> struct Held<ELT, TPR, NCH, true> {
  static constexpr int V = Chunk<ELT>::V;
  Codes<V> d[NCH];
  __device__ __forceinline__ void load(const Row<ELT, TPR, NCH>& at, const void* p, const uint8_t* scales, int64_t row) {
    const int8_t* q = (const int8_t*)p + row * at.cols;
    const uint8_t* sc = scales + row * ((at.cols + kMxBlock - 1) / kMxBlock);
    uint32_t byte[NCH];
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      d[i].zero();
      byte[i] = 0;
      if (at.some(i) && (at.full(i) || at.part(i))) {
        d[i].load(q + at.col(i), at.left(i), at.cols);
        byte[i] = sc[at.col(i) / kMxBlock];
      }
    }
#pragma unroll
    for (int i = 0; i < NCH; ++i) d[i].unit = mx8_unit(byte[i]);
  }
  __device__ __forceinline__ float get(int i, int j) const { return d[i].get(j); }
};

// SUMS: the gradients of the modulations are summed over a group's rows; otherwise (no such gradient, or
// groups of one row) a group of threads has one row
template <int ELT, int TPR, int NCH, bool KEPT, bool SUMS>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void mod_bwd_kernel(ModBwdArgs a) {
  constexpr int V = Chunk<ELT>::V, EB = elt_bytes(ELT), NT = TPR < 256 ? 256 : TPR, RPB = NT / TPR;
  __shared__ double slots[2][2][NT / 64];
  __shared__ float acc[SUMS && RPB > 1 ? RPB * TPR * NCH * V : 1];
  const int sub = threadIdx.x / TPR;
  const int64_t wg_group = SUMS ? blockIdx.x / (unsigned)a.parts : 0, wg_part = SUMS ? blockIdx.x % (unsigned)a.parts : blockIdx.x;
  const int64_t first = wg_group * a.rpg, end = SUMS ? a.rpg : a.rows, step = SUMS ? (int64_t)a.parts * RPB : (int64_t)gridDim.x * RPB;
  float tg[NCH][V], tc[NCH][V], th[NCH][V];
  if constexpr (SUMS) {
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) tg[i][j] = tc[i][j] = th[i][j] = 0.0f;
  }
  int turn = 0;
  for (int64_t r0 = wg_part * RPB; r0 < end; r0 += step, turn ^= 1) {
    const Row<ELT, TPR, NCH> at(a.cols, r0 + sub < end);
    const int64_t row = first + (at.live ? r0 + sub : end - 1), begin = row * a.cols * EB;
    const int64_t group = SUMS ? wg_group : (int64_t)((uint32_t)row / (uint32_t)a.rpg);
    const float hi = a.stats[row * 3], lo = a.stats[row * 3 + 1], rstd = a.stats[row * 3 + 2];
    Held<ELT, TPR, NCH, KEPT> s, b;
    Chunk<ELT> dy[NCH], ds[NCH];
    float m[NCH][V];
    s.load(at, a.s, a.ss, row);
    at.load((const uint8_t*)a.dy + begin, dy);
    if (a.dgate != nullptr) b.load(at, a.branch, a.bs, row);
    if (a.dsum != nullptr) at.load((const uint8_t*)a.dsum + begin, ds);
    if (a.scale != nullptr) {
      load_mod(at, a.scale, a.ld_scale, a.m_f32, group, m);
    } else {
#pragma unroll
      for (int i = 0; i < NCH; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) m[i][j] = 0.0f;
    }
    double g0 = 0.0, g1 = 0.0;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      if (!at.some(i)) continue;
      float n[V], d[V], p0 = 0.0f, p1 = 0.0f;
      const bool any = at.full(i) || at.part(i);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        d[j] = dy[i].get(j);
        n[j] = (s.get(i, j) - hi - lo) * rstd;
        const bool in = at.full(i) || j < at.left(i);
        if (!(any && in)) n[j] = 0.0f;
        if constexpr (SUMS) {
          th[i][j] += d[j];
          tc[i][j] = fmaf(d[j], n[j], tc[i][j]);
        }
        const float g = any && in ? d[j] * (1.0f + m[i][j]) : 0.0f;
        p0 += g;
        p1 = fmaf(g, n[j], p1);
      }
      if constexpr (!SUMS) {
        if (a.dscale != nullptr && any) {
          float up[V];
#pragma unroll
          for (int j = 0; j < V; ++j) up[j] = d[j] * n[j];
          store_vec<REELS_HIP_F32, V>(a.dscale + row * a.cols + at.col(i), at.left(i), up);
          store_vec<REELS_HIP_F32, V>(a.dshift + row * a.cols + at.col(i), at.left(i), d);
        }
      }
      g0 += (double)p0;
      g1 += (double)p1;
    }
    // two slots in turn: a wave may enter the next row's reduction while another still reads this one's
    if (a.center) g0 = row_reduce<TPR, false>(g0, slots[turn][0]);
    else g0 = 0.0;
    g1 = row_reduce<TPR, false>(g1, slots[turn][1]);
    const float m0 = (float)(g0 * a.per_col), m1 = (float)(g1 * a.per_col);
    float gate[NCH][V];
    if (a.gate != nullptr) load_mod(at, a.gate, a.ld_gate, a.m_f32, group, gate);
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      if (!at.some(i)) continue;
      const bool any = at.full(i) || at.part(i);
      float d[V];
      Chunk<ELT> o;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float n = (s.get(i, j) - hi - lo) * rstd;
        d[j] = rstd * (dy[i].get(j) * (1.0f + m[i][j]) - m0 - n * m1);
      }
      if (a.dsum != nullptr) {
#pragma unroll
        for (int j = 0; j < V; ++j) d[j] += ds[i].get(j);
      }
      o.pack(d);
      at.store((uint8_t*)a.dx + begin, i, o);
      if (a.dgate != nullptr && any) {
        float p[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          p[j] = d[j] * b.get(i, j);
          if constexpr (SUMS) tg[i][j] += at.full(i) || j < at.left(i) ? p[j] : 0.0f;
        }
        if constexpr (!SUMS) store_vec<REELS_HIP_F32, V>(a.dgate + row * a.cols + at.col(i), at.left(i), p);
      }
      if (a.gate != nullptr) {
#pragma unroll
        for (int j = 0; j < V; ++j) d[j] *= gate[i][j];
        o.pack(d);
        at.store((uint8_t*)a.db + begin, i, o);
      }
    }
  }
  if constexpr (SUMS) {
    const int lane = threadIdx.x % TPR;
    auto leave = [&](float (&v)[NCH][V], float* whole, int which) {
      if (whole == nullptr) return;
      float* out = a.parts == 1 ? whole + wg_group * a.cols : a.part + ((int64_t)blockIdx.x * 3 + which) * a.cols;
      if constexpr (RPB > 1) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) acc[(sub * TPR * NCH + lane + TPR * i) * V + j] = v[i][j];
        __syncthreads();
        for (int c = threadIdx.x; c < (int)a.cols; c += NT) {
          float t = acc[c];
#pragma unroll
          for (int r = 1; r < RPB; ++r) t += acc[r * TPR * NCH * V + c];
          out[c] = t;
        }
      } else {
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
          const int c = (lane + TPR * i) * V, left = (int)a.cols - c;
          if (left > 0) store_vec<REELS_HIP_F32, V>(out + c, left, v[i]);
        }
      }
    };
    leave(tg, a.dgate, 0);
    leave(tc, a.dscale, 1);
    leave(th, a.dshift, 2);
  }
}

}  // namespace

template <int ELT> void launch_mod_bwd(const ModBwdArgs& a, ModForm f, bool kept, bool sums, int64_t grid, hipStream_t st) {
  with_mod_form<ELT>(f, [&](auto tpr, auto nch) {
    constexpr int T = decltype(tpr)::value, C = decltype(nch)::value, NT = T < 256 ? 256 : T;
    if (kept) {
      if (sums) mod_bwd_kernel<ELT, T, C, true, true><<<(unsigned)grid, NT, 0, st>>>(a);
      else mod_bwd_kernel<ELT, T, C, true, false><<<(unsigned)grid, NT, 0, st>>>(a);
    } else {
      if (sums) mod_bwd_kernel<ELT, T, C, false, true><<<(unsigned)grid, NT, 0, st>>>(a);
      else mod_bwd_kernel<ELT, T, C, false, false><<<(unsigned)grid, NT, 0, st>>>(a);
    }
  });
}

}  // namespace reels
