// The kernel of the modulated norm's backward (modnorm_bwd.h).
#include "modnorm_bwd.h"

namespace reels {
namespace {

// a thread's chunks of a row of s or the branch, as stored or in 8 bits
template <int ELT, int TPR, int NCH, int KIND, bool KEPT> struct Held {
  Chunk<ELT> d[NCH];
  __device__ __forceinline__ void load(const ModRow<ELT, TPR, NCH, KIND>& at, const void* p, const uint8_t*, int64_t row) {
    at.load((const uint8_t*)p + row * at.cols * elt_bytes(ELT), d);
  }
  __device__ __forceinline__ void trim(const ModRow<ELT, TPR, NCH, KIND>& at) { at.trim(d); }
  __device__ __forceinline__ float get(int i, int j) const { return d[i].get(j); }
  __device__ __forceinline__ void hold() {
#pragma unroll
    for (int i = 0; i < NCH; ++i) d[i].hold();
  }
};
template <int ELT, int TPR, int NCH, int KIND> struct Held<ELT, TPR, NCH, KIND, true> {
  static constexpr int V = Chunk<ELT>::V;
  Codes<V> d[NCH];
  uint32_t byte[NCH];
  __device__ __forceinline__ void load(const ModRow<ELT, TPR, NCH, KIND>& at, const void* p, const uint8_t* scales, int64_t row) {
    const int8_t* q = (const int8_t*)p + row * at.cols;
    const uint8_t* sc = scales + row * ((at.cols + kMxBlock - 1) / kMxBlock);
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int l = at.left(i);
      if constexpr (KIND == kTiny) {
        d[i].zero();
        if (l > 0) d[i].load(q + at.col(i), l, at.cols);
      } else {
        d[i].load(q + (uint32_t)(KIND == kEven || l >= V ? at.col(i) : l > 0 ? at.cols - V : 0), V, V);
      }
      byte[i] = sc[(uint32_t)(KIND == kEven || l > 0 ? at.col(i) / kMxBlock : 0)];
    }
  }
  __device__ __forceinline__ void trim(const ModRow<ELT, TPR, NCH, KIND>& at) {
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      d[i].unit = mx8_unit(byte[i]);
      if (KIND == kTiny || at.all(i)) continue;
      const int l = at.left(i);
      if (l <= 0) d[i].zero();
      else if (l < V) d[i].shift_down(V - l);
    }
  }
  __device__ __forceinline__ float get(int i, int j) const { return d[i].get(j); }
  __device__ __forceinline__ void hold() {
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
      for (int j = 0; j < V / 4; ++j) asm volatile("" : "+v"(d[i].d[j]));
  }
};

// 16 lanes, a wave or a workgroup walk rows begin .. end of one group.
// SUMS: it leaves the sums of the modulations' gradients over them; otherwise (no such gradient, or groups
// of one row) rows of several groups may follow each other.
template <int ELT, int TPR, int NCH, int NT, int KIND, bool KEPT, bool SUMS>
__global__ __launch_bounds__(NT, NT == 512 ? 3 : 1) void mod_bwd_kernel(ModBwdArgs a) {
  constexpr int V = Chunk<ELT>::V, EB = elt_bytes(ELT), WALKERS = TPR == 0 ? 1 : 256 / (TPR == 0 ? 256 : TPR);
  __shared__ double slots[2][16][2];
  __shared__ float acc[SUMS && WALKERS > 1 ? WALKERS * TPR * NCH * V : 1];
  // A thread's gates wait in LDS until a row's end: with the sums they do not fit three waves' registers. Rows
  // past 8192 elements have one workgroup a CU, 128 registers and all of its LDS: 1 + scale is there, too.
  constexpr bool AWAY = (SUMS && NT == 512) || NT == 1024, UP_AWAY = NT == 1024;
  // The next row's s and dy are on their way while a row is worked on where the registers hold them (three waves
  // on a SIMD have 168 each), otherwise they are asked for at the row's end: 8000 x 13824 bf16 617 us with both
  // rows and the modulations in registers, 288 so; 4000 x 5120 f32 124 and 113, kept 137 and 100; 8000 x 5120
  // bf16 112 with the next row on its way, 115 without.
  constexpr bool AHEAD = NT < 512 || (NT == 512 && ELT != REELS_HIP_F32 && !(KEPT && KIND == kAny));
  __shared__ f32x4 gates[AWAY ? NCH * V / 4 : 1][AWAY ? NT : 1], ups[UP_AWAY ? NCH * V / 4 : 1][UP_AWAY ? NT : 1];
  const ModRow<ELT, TPR, NCH, KIND> at(a.cols);
  const int sub = TPR == 0 ? 0 : TPR == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : threadIdx.x >> 4;
  // rows in 32 bits, so that they and what follows from them stay in scalar registers (but for 16 lanes)
  const uint32_t wg_group = SUMS ? blockIdx.x / (uint32_t)a.parts : 0, part = SUMS ? blockIdx.x % (uint32_t)a.parts : blockIdx.x;
  const uint32_t rpg = (uint32_t)a.rpg, run = (uint32_t)a.run, last = (uint32_t)a.rows - 1;
  const uint32_t begin = wg_group * rpg + part * WALKERS + sub, end = SUMS ? (wg_group + 1) * rpg : last + 1;
  float tg[NCH][V], tc[NCH][V], th[NCH][V];
  if constexpr (SUMS) {
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) tg[i][j] = tc[i][j] = th[i][j] = 0.0f;
  }
  // a row's branch and dsum are on their way until they are needed after its sums (with these a row ahead, too,
  // 47 registers more than three waves on a SIMD have)
  struct Data {
    Held<ELT, TPR, NCH, KIND, KEPT> s;
    Chunk<ELT> dy[NCH];
    float hi, lo, rstd;
  };
  // all loads are unconditional, so that the waits for them need not count on the fewest: s and dy take the
  // place of a branch and a dsum that are not there, the last row that of one past it
  const void* branch = a.dgate != nullptr ? a.branch : a.s;
  const uint8_t* bs = a.dgate != nullptr ? a.bs : a.ss;
  const void* dsum = a.dsum != nullptr ? a.dsum : a.dy;
  auto load = [&](uint32_t r, Data& d) {
    const int64_t row = r < last ? r : last;
    d.s.load(at, a.s, a.ss, row);
    at.load((const uint8_t*)a.dy + row * a.cols * EB, d.dy);
    d.hi = a.stats[row * 3];
    d.lo = a.stats[row * 3 + 1];
    d.rstd = a.stats[row * 3 + 2];
  };
  Data cur, next;
  load(begin, cur);
  float up[NCH][V], gate[NCH][V];
#pragma unroll
  for (int i = 0; i < NCH; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) up[i][j] = gate[i][j] = 1.0f;
  auto put = [&](auto& lds, const float (&f)[NCH][V]) {
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
      for (int j = 0; j < V; j += 4) lds[(i * V + j) / 4][threadIdx.x] = f32x4{f[i][j], f[i][j + 1], f[i][j + 2], f[i][j + 3]};
  };
  auto take = [&](const auto& lds, int i, float (&f)[V]) {
#pragma unroll
    for (int j = 0; j < V; j += 4) {
      const f32x4 v = lds[(i * V + j) / 4][threadIdx.x];
#pragma unroll
      for (int q = 0; q < 4; ++q) f[j + q] = v[q];
    }
  };
  if constexpr (UP_AWAY) put(ups, up);
  uint32_t change = begin;
  int turn = 0;
  for (uint32_t r = begin; r < end; r += run, turn ^= 1) {
    const int64_t row = r, at0 = row * a.cols * EB;
    if (r >= change) {
      const uint32_t group = SUMS ? wg_group : r / rpg;
      change = (group + 1) * rpg;
      if (a.scale != nullptr) {
        at.mods(a.scale, a.ld_scale, a.m_f32, group, up);
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) up[i][j] += 1.0f;
        if constexpr (UP_AWAY) put(ups, up);
      }
      if (a.gate != nullptr) {
        at.mods(a.gate, a.ld_gate, a.m_f32, group, gate);
        if constexpr (AWAY) put(gates, gate);
      }
      __builtin_amdgcn_s_waitcnt(0x0F70);  // here, and not at each row's use
    }
    Held<ELT, TPR, NCH, KIND, KEPT> b;
    Chunk<ELT> ds[NCH];
    b.load(at, branch, bs, row);
    at.load((const uint8_t*)dsum + at0, ds);
    if constexpr (AHEAD) load(r + run, next);
    cur.s.trim(at);
    at.trim(cur.dy);
    const float rstd = cur.rstd;
    ModUnit of = mod_unit(cur.hi, cur.lo, rstd, a.far);
    // A workgroup's row: in a scalar register where the lanes' are scarce (8000 x 13824 bf16 268 us and 260). 512
    // threads without the sums have enough; there the compiler then takes more than four waves leave (32760 x 5120
    // 290 us and 360).
    if constexpr (NT == 1024 || (SUMS && NT == 512)) of.hi = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(of.hi)));
    double g0 = 0.0, g1 = 0.0;
    // dy is zero where the thread has no element, and so are its shares of the sums
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      float p0 = 0.0f, p1 = 0.0f, up1[V], u[V];
      if constexpr (UP_AWAY) take(ups, i, u);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = cur.dy[i].get(j), n = fmaf(cur.s.get(i, j) - of.hi, rstd, of.k), g = d * (UP_AWAY ? u[j] : up[i][j]);
        p0 += g;
        p1 = fmaf(g, n, p1);
        if constexpr (SUMS) {
          th[i][j] += d;
          tc[i][j] = fmaf(d, n, tc[i][j]);
        }
        up1[j] = d * n;
      }
      if constexpr (!SUMS) {
        if (a.dscale != nullptr) {
          float d[V];
          cur.dy[i].unpack(d);
          at.store(a.dscale + row * a.cols, i, up1);
          at.store(a.dshift + row * a.cols, i, d);
        }
      }
      g0 += (double)p0;
      g1 += (double)p1;
    }
    row_sums<TPR>(g0, g1, slots[turn]);
    b.trim(at);
    at.trim(ds);
    const float m0 = a.center ? (float)(g0 * a.per_col) : 0.0f, m1 = (float)(g1 * a.per_col);
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      float d[V], u[V];
      Chunk<ELT> o;
      if constexpr (UP_AWAY) take(ups, i, u);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float n = fmaf(cur.s.get(i, j) - of.hi, rstd, of.k);
        const float t = fmaf(-n, m1, fmaf(cur.dy[i].get(j), UP_AWAY ? u[j] : up[i][j], -m0));
        d[j] = a.dsum != nullptr ? fmaf(rstd, t, ds[i].get(j)) : rstd * t;
      }
      o.pack(d);
      at.store((uint8_t*)a.dx + at0, i, o);
      if (a.dgate != nullptr) {
        float p[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if constexpr (SUMS) tg[i][j] = fmaf(d[j], b.get(i, j), tg[i][j]);
          else p[j] = d[j] * b.get(i, j);
        }
        if constexpr (!SUMS) at.store(a.dgate + row * a.cols, i, p);
      }
      if (a.gate != nullptr) {
#pragma unroll
        for (int j = 0; j < V; ++j) d[j] *= AWAY ? gates[(i * V + j) / 4][threadIdx.x][j % 4] : gate[i][j];
        o.pack(d);
        at.store((uint8_t*)a.db + at0, i, o);
      }
    }
    if constexpr (AHEAD) cur = next;
    else load(r + run, cur);
  }
  if constexpr (SUMS) {
    auto leave = [&](float (&v)[NCH][V], float* whole, int which) {
      if (whole == nullptr) return;
      float* out = a.parts == 1 ? whole + (int64_t)wg_group * a.cols : a.part + ((int64_t)blockIdx.x * 3 + which) * a.cols;
      if constexpr (WALKERS > 1) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) acc[sub * TPR * NCH * V + at.col(i) + j] = v[i][j];
        __syncthreads();
        for (int c = threadIdx.x; c < (int)a.cols; c += 256) {
          float t = acc[c];
#pragma unroll
          for (int r = 1; r < WALKERS; ++r) t += acc[r * TPR * NCH * V + c];
          out[c] = t;
        }
      } else {
#pragma unroll
        for (int i = 0; i < NCH; ++i) at.store(out, i, v[i]);
      }
    };
    leave(tg, a.dgate, 0);
    leave(tc, a.dscale, 1);
    leave(th, a.dshift, 2);
  }
}

}  // namespace

template <int ELT> void launch_mod_bwd(const ModBwdArgs& a, ModForm f, bool kept, bool sums, int64_t grid, hipStream_t st) {
  with_mod_form<ELT>(f, a.cols, [&](auto tpr, auto nch, auto nt, auto kind) {
    constexpr int T = decltype(tpr)::value, C = decltype(nch)::value, NT = decltype(nt)::value, Y = decltype(kind)::value;
    if (kept) {
      if (sums) mod_bwd_kernel<ELT, T, C, NT, Y, true, true><<<(unsigned)grid, f.threads, 0, st>>>(a);
      else mod_bwd_kernel<ELT, T, C, NT, Y, true, false><<<(unsigned)grid, f.threads, 0, st>>>(a);
    } else {
      if (sums) mod_bwd_kernel<ELT, T, C, NT, Y, false, true><<<(unsigned)grid, f.threads, 0, st>>>(a);
      else mod_bwd_kernel<ELT, T, C, NT, Y, false, false><<<(unsigned)grid, f.threads, 0, st>>>(a);
    }
  });
}

}  // namespace reels
