// Product of int8 rows with an int8 weight, both with one scale per row (QuantizedMatrix), with bias,
// activation and residual in its epilogue:
//
//   y[m][n] = rnd( act( xs[m] ws[n] sum_k xq[m][k] wq[n][k] + bias[n] ) + residual[m][n] )
//
// The sums are whole numbers in 32 bits (K < 2^17 products of at most 2^14 stay below 2^31), so every
// form and split gives the same bits; the epilogue runs in f32 and rounds once.
#include "vec.h"

#include <atomic>

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

// gelu_tanh as x / (1 + exp(-2 k (x + 0.044715 x^3))), k = sqrt(2 / pi): 0.5 (1 + tanh z) is the logistic
// function of 2 z, which takes two operations for four and loses no digits where the result is small
// (32760 x 5120 -> 13824, where the epilogue's arithmetic counts: 1.98 ms with tanh)
__device__ __forceinline__ float gelu_logistic(float x) {
  const float c = -2.3022082f;  // -2 sqrt(2 / pi) log2(e)
  const float e = __builtin_amdgcn_exp2f(x * fmaf(c * 0.044715f, x * x, c));
  return x * __builtin_amdgcn_rcpf(1.0f + e);
}

// The f32 product of a sum and the row's scale stays in range below this scale (the sum is below 2^31).
// Rows past it (values of 1e30 and more) are scaled by 2^-64 on the way, which loses no bits: the
// weight's scale brings them back.
constexpr float kBigScale = 0x1p96f;
__device__ __forceinline__ float scaled_big(int acc, float xs, float ws, float bias) {
  return (float)acc * (xs * 0x1p-64f) * ws * 0x1p64f + bias;
}

// ---- tiled form --------------------------------------------------------------------------------
// 32 TJ x 32 TJ outputs per workgroup of TJ waves (TJ = 8: 256 x 256, TJ = 4: 128 x 128), a step of
// 128 codes, each wave 16 TJ tokens x 64 columns in 16 x 16 x 64 MFMAs. The operands travel from HBM
// to LDS directly (rows of 128 bytes, 16-byte chunks XOR-swizzled by the row), the activations in a
// ring of three stages and the weight in one of two: at the barrier that ends step kt every wave has
// read stage kt, so the weight copy of step kt + 2 goes into it right away, and the activation copy
// of step kt + 2 into the stage of step kt - 1 already during the first half of step kt. Per step a
// wave reads TJ + 4 fragments for 4 TJ MFMAs, twice. Rows past the edges read as zeros (the buffer's
// bounds). K and the rows' addresses are multiples of 4 here, which the copies need; others run on
// padded copies. Bound by the matrix cores at the power cap: 32760 x 13824 -> 5120 1.66-1.68 ms (2.75-2.79
// POP/s; the vendor's int8 product 2.49 on this size), with bias and residual 1.65-1.74, single launches
// 1.73-1.87; f32 output 1.73, with its residual 1.85.
template <int TJ> struct Tile {
  static constexpr int NW = TJ, NT = NW * 64, WN = NW / 2, BM = 32 * TJ, BN = 64 * WN, BK = 128;
  static constexpr int ACT = BM * BK, WB = BN * BK, LDS = 3 * ACT + 2 * WB;
};

// Zeros for the activations' bytes from `keep` on in a tile of 128-byte rows: where K is no multiple of
// 128 the last step's rows end in the next row's codes, and zeros on one side take them out of the sum
template <int ROWS, int NT> __device__ __forceinline__ void clear_tail(uint8_t* tile, int keep) {
  for (int i = threadIdx.x; i < ROWS * 8; i += NT) {
    const int row = i >> 3, c = i & 7, lo = keep - c * 16;  // lo: bytes of chunk c that stay
    if (lo >= 16) continue;
    i32v4* p = reinterpret_cast<i32v4*>(tile + row * 128 + ((c ^ (row & 7)) << 4));
    i32v4 v = *p;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int b = lo - 4 * q;
      v[q] = b >= 4 ? v[q] : b <= 0 ? 0 : v[q] & ((1 << (8 * b)) - 1);
    }
    *p = v;
  }
  __builtin_amdgcn_s_waitcnt(0xC07F);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Two waves on a SIMD are asked for by name: left alone the compiler holds the whole residual of an f32
// tile in registers at TJ = 4, one workgroup then has the CU to itself, and 6000 x 512 -> 768 in f32
// takes 17.3 us instead of 11.1.
template <int ELT, int TJ>
__global__ __launch_bounds__(Tile<TJ>::NT, 2) void product_tile_kernel(ProductArgs a, int tiles_n, int tiles_m) {
  using T = Tile<TJ>;
  constexpr int V = 16 / elt_bytes(ELT);
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const int t = threadIdx.x, lane = t & 63;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wm = w / T::WN, wn = w % T::WN, l16 = lane & 15, lq = lane >> 4;
  // consecutive tiles of one XCD share rows: groups of 4 tile rows, column by column
  const int nt = tiles_n * tiles_m, xcd = blockIdx.x & 7, idx = blockIdx.x >> 3;
  const int logical = xcd * (nt >> 3) + (xcd < (nt & 7) ? xcd : nt & 7) + idx;
  const int group = 4 * tiles_n, g = logical / group, first = g * 4;
  const int gm = tiles_m - first < 4 ? tiles_m - first : 4, within = logical - g * group;
  const int64_t m0 = (int64_t)(first + within % gm) * T::BM, n0 = (int64_t)(within / gm) * T::BN;
  const int K = (int)a.K, nk = (K + T::BK - 1) / T::BK, tail = K % T::BK;
  const int rows = (int)(a.M - m0 < T::BM ? a.M - m0 : T::BM), cols = (int)(a.N - n0 < T::BN ? a.N - n0 : T::BN);
  const i32x4 rx = buffer_rsrc(a.x + m0 * a.K, (uint32_t)rows * K), rw = buffer_rsrc(a.w + n0 * a.K, (uint32_t)cols * K);
  const i32x4 rnone = buffer_rsrc(a.x, 0u);  // zero records: a copy through it reads nothing
  uint32_t vo[4];  // copy i of wave w: tile rows 8 (4 w + i) + lane / 8, 16 bytes per lane
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = (w * 4 + i) * 8 + (lane >> 3);
    vo[i] = (uint32_t)(row * K + ((lane & 7) ^ (row & 7)) * 16);
  }
  auto abase = [&](int kt) { return smem + (kt % 3) * T::ACT; };
  auto wbase = [&](int kt) { return smem + 3 * T::ACT + (kt & 1) * T::WB; };
  auto issue_x = [&](const i32x4& r, int kt, int i) { dma16(r, vo[i], (uint32_t)kt * T::BK, abase(kt) + (w * 4 + i) * 1024); };
  auto issue_w = [&](const i32x4& r, int kt, int i) { dma16(r, vo[i], (uint32_t)kt * T::BK, wbase(kt) + (w * 4 + i) * 1024); };

  i32v4 acc[4][TJ] = {};
  const int swz = l16 & 7;
  auto read_w = [&](const uint8_t* s, int h, i32v4* f) {
    const int off = ((4 * h + lq) ^ swz) << 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = *reinterpret_cast<const i32v4*>(s + (wn * 64 + i * 16 + l16) * 128 + off);
  };
  auto read_x = [&](const uint8_t* s, int h, int j) {
    return *reinterpret_cast<const i32v4*>(s + (wm * 16 * TJ + j * 16 + l16) * 128 + (((4 * h + lq) ^ swz) << 4));
  };
  auto mfma4 = [&](const i32v4* f, const i32v4& xf, int j) {
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f[i], xf, acc[i][j], 0, 0, 0);
  };
  i32v4 w0[4], w1[4], x[TJ];
#pragma unroll
  for (int i = 0; i < 4; ++i) { issue_x(rx, 0, i); issue_w(rw, 0, i); }
  if (nk > 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i) { issue_x(rx, 1, i); issue_w(rw, 1, i); }
    __builtin_amdgcn_s_waitcnt(0x0F78);  // vmcnt(8): step 1 may stay in flight
  } else {
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  }
  __builtin_amdgcn_s_waitcnt(0xC07F);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  if (nk == 1 && tail != 0) clear_tail<T::BM, T::NT>(abase(0), tail);
  read_w(wbase(0), 0, w0);
#pragma unroll
  for (int j = 0; j < TJ; ++j) x[j] = read_x(abase(0), 0, j);
  // copies per step and kind: four, one per TJ / 4 groups of MFMAs. Step nk - 2 has no step to copy:
  // its copies read nothing (they write zeros into stages that no wave reads any more), so that every
  // step's waits count the same.
  auto kstep = [&](int kt, auto last) {
    constexpr bool LAST = decltype(last)::value;
    constexpr int PER = TJ / 4;
    const i32x4& cx = LAST ? rnone : rx;
    const i32x4& cw = LAST ? rnone : rw;
    // eight waves: w and w + 4 share a SIMD, and the younger one has the priority in the second half
    // of a step, so that both reach the barrier together
    if (TJ == 8 && w >= 4) __builtin_amdgcn_s_setprio(0);
    const uint8_t* sa = abase(kt);
    const uint8_t* sw = wbase(kt);
#pragma unroll
    for (int j = 0; j < TJ; ++j) {
      mfma4(w0, x[j], j);
      __builtin_amdgcn_sched_barrier(0);
      x[j] = read_x(sa, 1, j);
      if (j == 0) read_w(sw, 1, w1);
      if (j % PER == PER - 1) issue_x(cx, kt + 2, j / PER);
      __builtin_amdgcn_sched_barrier(0);
    }
    // the weight fragments have been read: all but the TJ - 1 activation reads after them, which the
    // LDS serves in order before the copies issued below land
    __builtin_amdgcn_s_waitcnt(0xC07F | (TJ - 1) << 8);
    __builtin_amdgcn_s_waitcnt(0x0F74);  // vmcnt(4): step kt + 1 has landed
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if constexpr (LAST) {
      if (tail != 0) clear_tail<T::BM, T::NT>(abase(kt + 1), tail);
    }
    if (TJ == 8 && w >= 4) __builtin_amdgcn_s_setprio(1);
    __builtin_amdgcn_sched_barrier(0);
    const uint8_t* san = abase(kt + 1);
    read_w(wbase(kt + 1), 0, w0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < TJ; ++j) {
      mfma4(w1, x[j], j);
      __builtin_amdgcn_sched_barrier(0);
      x[j] = read_x(san, 0, j);
      if (j % PER == PER - 1) issue_w(cw, kt + 2, j / PER);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  for (int kt = 0; kt + 2 < nk; ++kt) kstep(kt, std::false_type{});
  if (nk > 1) kstep(nk - 2, std::true_type{});
  if (TJ == 8 && w >= 4) __builtin_amdgcn_s_setprio(0);
  {
    const uint8_t* sa = abase(nk - 1);
    read_w(wbase(nk - 1), 1, w1);
#pragma unroll
    for (int j = 0; j < TJ; ++j) {
      mfma4(w0, x[j], j);
      x[j] = read_x(sa, 1, j);
    }
#pragma unroll
    for (int j = 0; j < TJ; ++j) mfma4(w1, x[j], j);
  }
  __builtin_amdgcn_s_waitcnt(0x0F70);  // the last copies have landed
  // Epilogue: f32 values of 64 tokens x 64 columns at a time in the wave's own 16 KiB of LDS (rows of
  // 256 bytes, 16-byte chunks XOR-swizzled), read back as rows: residual and stores in whole segments
  const int nb = wn * 64 + lq * 4;
  float sc[4][4], bs[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int left = cols - (nb + i * 16);
    load_vec<REELS_HIP_F32, 4>(a.ws + n0 + nb + i * 16, left < 0 ? 0 : left, sc[i]);
#pragma unroll
    for (int v = 0; v < 4; ++v) bs[i][v] = 0.0f;
    if (a.bias != nullptr) load_vec<ELT, 4>((const uint8_t*)a.bias + (n0 + nb + i * 16) * elt_bytes(ELT), left < 0 ? 0 : left, bs[i]);
  }
  __syncthreads();
  uint8_t* stage = smem + w * 16384;
  constexpr int LPR = 64 / V, RPI = 64 / LPR, ITS = 64 / RPI;  // lanes of a row, rows at once, turns
  const int c = (lane % LPR) * V, left = cols - (wn * 64 + c);
  const bool ahead = a.res != nullptr && a.M * a.N >= V;
#pragma unroll
  for (int h = 0; h < TJ / 4; ++h) {
    // the residual's whole chunks on their way while the values are formed; from its start where a lane
    // has none
    Chunk<ELT> res[ITS];
    if (ahead) {
#pragma unroll
      for (int it = 0; it < ITS; ++it) {
        const int mr = wm * 16 * TJ + h * 64 + it * RPI + lane / LPR;
        const int64_t at = mr < rows && left >= V ? (m0 + mr) * a.N + n0 + wn * 64 + c : 0;
        res[it].d = load_any<u32x4>((const typename Store<ELT>::raw*)((const uint8_t*)a.res + at * elt_bytes(ELT)));
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = j * 16 + l16, mr = wm * 16 * TJ + h * 64 + r;
      const float xs = mr < rows ? a.xs[m0 + mr] : 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f32x4 o;
#pragma unroll
        for (int v = 0; v < 4; ++v) o[v] = (float)acc[i][h * 4 + j][v] * xs * sc[i][v] + bs[i][v];
        if (fabsf(xs) >= kBigScale) {
#pragma unroll
          for (int v = 0; v < 4; ++v) o[v] = scaled_big(acc[i][h * 4 + j][v], xs, sc[i][v], bs[i][v]);
        }
        if (a.gelu) {
#pragma unroll
          for (int v = 0; v < 4; ++v) o[v] = gelu_logistic(o[v]);
        }
        *reinterpret_cast<f32x4*>(stage + r * 256 + (((i * 4 + lq) ^ (r & 15)) << 4)) = o;
      }
    }
    __builtin_amdgcn_s_waitcnt(0xC07F);
    asm volatile("" ::: "memory");
#pragma unroll
    for (int it = 0; it < ITS; ++it) {
      const int r = it * RPI + lane / LPR, mr = wm * 16 * TJ + h * 64 + r;
      if (mr >= rows || left <= 0) continue;
      float o[V];
#pragma unroll
      for (int q = 0; q < V / 4; ++q) {
        const f32x4 f = *reinterpret_cast<const f32x4*>(stage + r * 256 + (((c / 4 + q) ^ (r & 15)) << 4));
#pragma unroll
        for (int v = 0; v < 4; ++v) o[q * 4 + v] = f[v];
      }
      const int64_t at = (m0 + mr) * a.N + n0 + wn * 64 + c;
      if (a.res != nullptr) {
        if (left < V) res[it].load((const uint8_t*)a.res + at * elt_bytes(ELT), left);
#pragma unroll
        for (int v = 0; v < V; ++v) o[v] += res[it].get(v);
      }
      store_vec<ELT, V>((uint8_t*)a.y + at * elt_bytes(ELT), left, o);
    }
    __builtin_amdgcn_s_waitcnt(0xC07F);  // the rows have been read before the next half's are written
    asm volatile("" ::: "memory");
  }
}

// ---- small tiles -------------------------------------------------------------------------------
// 64 x 64 outputs per workgroup of eight waves, a step of 128 codes: for token counts whose larger
// tiles would leave most CUs idle. Waves w and w + 4 own the same 32 x 32 outputs and take the two
// halves of a step's codes (their whole-number sums are added in LDS at the end), so that each SIMD
// has a second wave under the first one's barrier, copy and LDS latencies. A ring of four 16 KiB
// stages, three steps in flight and one barrier per step; two workgroups fit a CU. Bound by LDS (768
// of about 1300 clocks of two workgroups' step). 333 x 5120 -> 5120: 28.4 us with the tiles of one
// weight tile spread over the XCDs, 18.7 us on one; four waves without the halves 14.5 us against
// 12.0 at 64 tokens; a ring of eight stages is slower everywhere (one workgroup per CU).
namespace small {
constexpr int BT = 64, BK = 128, STAGE = 2 * BT * BK, RING = 4, NT = 512;
}

// bias, activation and residual of four columns n.. (left of them exist) of token m, then one rounding
template <int ELT>
__device__ __forceinline__ void finish4(const ProductArgs& a, int64_t m, int64_t n, int left, const i32v4& acc, float xs,
                                        const float (&sc)[4], const float (&bs)[4]) {
  float o[4];
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    o[v] = (float)acc[v] * xs * sc[v] + bs[v];
    if (fabsf(xs) >= kBigScale) o[v] = scaled_big(acc[v], xs, sc[v], bs[v]);
    if (a.gelu) o[v] = gelu_logistic(o[v]);
  }
  const int64_t at = (m * a.N + n) * elt_bytes(ELT);
  if (a.res != nullptr) {
    float e[4];
    load_vec<ELT, 4>((const uint8_t*)a.res + at, left, e);
#pragma unroll
    for (int v = 0; v < 4; ++v) o[v] += e[v];
  }
  store_vec<ELT, 4>((uint8_t*)a.y + at, left, o);
}

template <int ELT>
__device__ __forceinline__ void load_columns(const ProductArgs& a, int64_t n, int left, float (&sc)[4], float (&bs)[4]) {
  load_vec<REELS_HIP_F32, 4>(a.ws + n, left, sc);
#pragma unroll
  for (int v = 0; v < 4; ++v) bs[v] = 0.0f;
  if (a.bias != nullptr) load_vec<ELT, 4>((const uint8_t*)a.bias + n * elt_bytes(ELT), left, bs);
}

template <int ELT>
__global__ __launch_bounds__(small::NT) void product_small_kernel(ProductArgs a, int tiles_m) {
  using namespace small;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[RING * STAGE];
  const int t = threadIdx.x, lane = t & 63;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int h = w >> 2, wm = (w >> 1) & 1, wn = w & 1, l16 = lane & 15, lq = lane >> 4;
  // the token tiles of one weight tile follow each other on one XCD: its codes come to that L2 once
  const int xcd = blockIdx.x & 7, nt = gridDim.x;
  const int logical = xcd * (nt >> 3) + (xcd < (nt & 7) ? xcd : nt & 7) + (blockIdx.x >> 3);
  const int64_t m0 = (int64_t)(logical % tiles_m) * BT, n0 = (int64_t)(logical / tiles_m) * BT;
  const int K = (int)a.K, nk = (K + BK - 1) / BK, tail = K % BK;
  const int rows = (int)(a.M - m0 < BT ? a.M - m0 : BT), cols = (int)(a.N - n0 < BT ? a.N - n0 : BT);
  const i32x4 rx = buffer_rsrc(a.x + m0 * a.K, (uint32_t)rows * K), rw = buffer_rsrc(a.w + n0 * a.K, (uint32_t)cols * K);
  const int crow = w * 8 + (lane >> 3);  // a wave copies rows 8 w .. 8 w + 7 of each tile
  const uint32_t vo = (uint32_t)(crow * K + ((lane & 7) ^ (crow & 7)) * 16);
  auto issue = [&](int kt) {  // past the end the copies read nothing, so that the waits count the same
    uint8_t* s = smem + (kt & (RING - 1)) * STAGE + w * 1024;
    const bool in = kt < nk;
    i32x4 cx = rx, cw = rw;
    cx[2] = in ? rx[2] : 0;
    cw[2] = in ? rw[2] : 0;
    dma16(cx, vo, (uint32_t)kt * BK, s);
    dma16(cw, vo, (uint32_t)kt * BK, s + BT * BK);
  };
#pragma unroll
  for (int kt = 0; kt < RING - 1; ++kt) issue(kt);
  i32v4 acc[2][2] = {};
  const int off = ((4 * h + lq) ^ (l16 & 7)) << 4;
  for (int kt = 0; kt < nk; ++kt) {
    __builtin_amdgcn_s_waitcnt(0x0F74);  // vmcnt(4): step kt has landed, the two after it may fly
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (kt == nk - 1 && tail != 0) clear_tail<BT, NT>(smem + (kt & (RING - 1)) * STAGE, tail);
    const uint8_t* s = smem + (kt & (RING - 1)) * STAGE + l16 * 128 + off;
    i32v4 xf[2], wf[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      xf[i] = *reinterpret_cast<const i32v4*>(s + (wm * 32 + i * 16) * 128);
      wf[i] = *reinterpret_cast<const i32v4*>(s + BT * BK + (wn * 32 + i * 16) * 128);
    }
    issue(kt + RING - 1);  // into the stage of step kt - 1, which every wave has read
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[i], xf[j], acc[i][j], 0, 0, 0);
    // the fragments are in registers before the next barrier lets their stage be overwritten
    __builtin_amdgcn_s_waitcnt(0xC07F);
  }
  __builtin_amdgcn_s_waitcnt(0x0F70);  // no copy outlives the loop
  __syncthreads();
  i32v4* part = reinterpret_cast<i32v4*>(smem) + (w & 3) * 256 + lane;
  if (h == 1) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) part[(i * 2 + j) * 64] = acc[i][j];
  }
  __syncthreads();
  if (h == 1) return;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int nb = wn * 32 + i * 16 + lq * 4, left = cols - nb;
    if (left <= 0) continue;
    float sc[4], bs[4];
    load_columns<ELT>(a, n0 + nb, left, sc, bs);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int mr = wm * 32 + j * 16 + l16;
      if (mr < rows) finish4<ELT>(a, m0 + mr, n0 + nb, left, acc[i][j] + part[(i * 2 + j) * 64], a.xs[m0 + mr], sc, bs);
    }
  }
}

// ---- few tokens --------------------------------------------------------------------------------
// Up to 16 tokens: 16 outputs per workgroup, its eight waves take lines of 128 codes in turn and read
// weight and activations straight into registers (each code of the weight is used once, so LDS would
// only add a trip), then add their whole-number sums in LDS. Any K and alignment. The weight's bytes would
// take 5.0 us at 5120 -> 5120 and 13.4 at 5120 -> 13824; measured are 8.8, 9.2, 10.0 and 11.5 us for 2, 4,
// 8 and 16 tokens -> 5120 (2.3-3.0 TB/s) and 23.5 us for 16 -> 13824 (3.0). Latency and balance make the
// difference: N / 16 workgroups are 320 on 256 CUs at 5120 outputs, and a wave's five lines there are
// two trips of loads, one after the other. With one token, four and sixteen waves are within 4% at 5120
// outputs, 2 to 14% slower at 13824.
constexpr int kFewTokens = 16, kFewWaves = 8, kFewUnroll = 4;

// 16 codes at p, the first `left` of which belong to its row of K, zeros for the others: a part of 16
// is the row's last 16 codes shifted down (a loop over bytes waits for each)
__device__ __forceinline__ i32v4 load_codes(const int8_t* p, int left, int K) {
  if (left >= 16) return load_any<i32v4>(p);
  i32v4 v = {0, 0, 0, 0};
  if (left <= 0) return v;
  if (K >= 16) {
    const unsigned __int128 u = load_any<unsigned __int128>(p + left - 16) >> (8 * (16 - left));
    return __builtin_bit_cast(i32v4, u);
  }
  for (int b = 0; b < left; ++b) {
    const int byte = (int)((uint32_t)(uint8_t)p[b] << (8 * (b % 4)));
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] |= b / 4 == q ? byte : 0;
  }
  return v;
}

template <int ELT>
__global__ __launch_bounds__(kFewWaves * 64) void product_few_kernel(ProductArgs a) {
  __shared__ i32v4 part[kFewWaves][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, l16 = lane & 15, lq = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16, K = a.K;
  const int8_t* wr = a.w + (n0 + l16 < a.N ? n0 + l16 : a.N - 1) * K + lq * 16;
  const int8_t* xr = a.x + (l16 < a.M ? l16 : a.M - 1) * K + lq * 16;
  i32v4 acc = {0, 0, 0, 0};
  const int lines = (int)(K / 128);
  int s = w;
  auto run = [&](auto count) {  // so many lines at once, all their loads in flight
    constexpr int C = 2 * decltype(count)::value;
    i32v4 wf[C], xf[C];
#pragma unroll
    for (int c = 0; c < C; ++c) wf[c] = load_any<i32v4>(wr + (s + c / 2 * kFewWaves) * 128 + (c & 1) * 64);
#pragma unroll
    for (int c = 0; c < C; ++c) xf[c] = load_any<i32v4>(xr + (s + c / 2 * kFewWaves) * 128 + (c & 1) * 64);
#pragma unroll
    for (int c = 0; c < C; ++c) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[c], xf[c], acc, 0, 0, 0);
    s += decltype(count)::value * kFewWaves;
  };
  while (s + (kFewUnroll - 1) * kFewWaves < lines) run(std::integral_constant<int, kFewUnroll>{});
  if (s + 2 * kFewWaves < lines) run(std::integral_constant<int, 3>{});
  else if (s + kFewWaves < lines) run(std::integral_constant<int, 2>{});
  else if (s < lines) run(std::integral_constant<int, 1>{});
  // what is left of K in pieces of 64, codes past it as zeros
  const int piece = (lines * 2 + w) * 64;
  if (w < 2 && piece < K)
    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(load_codes(wr + piece, (int)K - piece - lq * 16, (int)K),
                                                load_codes(xr + piece, (int)K - piece - lq * 16, (int)K), acc, 0, 0, 0);
  part[w][lane] = acc;
  __syncthreads();
  if (w > 0) return;
#pragma unroll
  for (int i = 1; i < kFewWaves; ++i) acc += part[i][lane];
  const int64_t m = l16, n = n0 + lq * 4;
  if (m >= a.M || n >= a.N) return;
  const int left = a.N - n < 4 ? (int)(a.N - n) : 4;
  float sc[4], bs[4];
  load_columns<ELT>(a, n, left, sc, bs);
  finish4<ELT>(a, m, n, left, acc, a.xs[m], sc, bs);
}

// ---- one token ---------------------------------------------------------------------------------
// A wave takes one output over the whole K: each lane multiplies 16 codes of every KiB with v_dot4,
// so the weight streams in whole lines and its rows spread evenly over the CUs, where the 16-row
// tiles above leave some CUs twice the work of others. Taken at K of 4096 and more, where it has
// several loads in flight: 1 x 13824 -> 5120 20.5 -> 13.9 us (5.1 TB/s), 5120 -> 13824 16.1 -> 13.5,
// 5120 -> 5120 8.6 -> 6.2; below it the two are level (1536 -> 8960 4.5 and 4.7 us). Two or four
// outputs a wave share the activations' loads and are slower at every one of these sizes.
constexpr int64_t kDotCodes = 4096;

template <int ELT>
__global__ __launch_bounds__(64) void product_dot_kernel(ProductArgs a) {
  const int64_t n = blockIdx.x;
  const int K = (int)a.K, lane = threadIdx.x;
  const int8_t* wr = a.w + n * a.K;
  int acc = 0;
  auto dot = [&](const i32v4& wf, const i32v4& xf) {
#pragma unroll
    for (int q = 0; q < 4; ++q) acc = __builtin_amdgcn_sdot4(wf[q], xf[q], acc, false);
  };
  constexpr int U = 4;
  int k = lane * 16;
  for (; k + (U - 1) * 1024 + 16 <= K; k += U * 1024) {
    i32v4 wf[U], xf[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      wf[u] = load_any<i32v4>(wr + k + u * 1024);
      xf[u] = load_any<i32v4>(a.x + k + u * 1024);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) dot(wf[u], xf[u]);
  }
  i32v4 wf[U], xf[U];  // fewer than U KiB are left, the last piece of a lane perhaps in part
#pragma unroll
  for (int u = 0; u < U; ++u) {
    wf[u] = load_codes(wr + k + u * 1024, K - k - u * 1024, K);
    xf[u] = load_codes(a.x + k + u * 1024, K - k - u * 1024, K);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) dot(wf[u], xf[u]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) acc += __shfl_xor(acc, o, 64);
  if (lane > 0) return;
  const i32v4 sum = {acc, 0, 0, 0};
  float sc[4], bs[4];
  load_columns<ELT>(a, n, 1, sc, bs);
  finish4<ELT>(a, 0, n, 1, sum, a.xs[0], sc, bs);
}

template <typename K> int launch_rows(K kernel, const char* label, int64_t grid, int threads, const ProductArgs& a, hipStream_t st) {
  if (!grid_fits(grid, threads)) return fail(REELS_HIP_EINVAL, "reels_hip_i8i8_linear: too many columns for one launch");
  { TraceScope _ts(st, label);
    kernel<<<(unsigned)grid, threads, 0, st>>>(a); }
  return check_launch(label);
}

int launch_small(const ProductArgs& a, int dtype, hipStream_t st) {
  const int64_t tn = ceil_div(a.N, small::BT), tm = ceil_div(a.M, small::BT);
  if (!grid_fits(tn * tm, small::NT)) return fail(REELS_HIP_EINVAL, "reels_hip_i8i8_linear: too many output tiles for one launch");
  { TraceScope _ts(st, "product_small_kernel");
    with_any_elt(dtype, [&](auto e) {
      product_small_kernel<decltype(e)::value><<<(unsigned)(tn * tm), small::NT, 0, st>>>(a, (int)tm);
    }); }
  return check_launch("product_small_kernel");
}

// rows of K codes at any address to rows of Kp (a multiple of 128), zeros past K; both operands in
// one launch (rows past r0 belong to the second), a wave per row
__global__ __launch_bounds__(256) void product_pad_kernel(const int8_t* __restrict__ x, int64_t r0, const int8_t* __restrict__ w,
                                                          int64_t r1, int K, int Kp, int8_t* __restrict__ px,
                                                          int8_t* __restrict__ pw) {
  for (int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < r0 + r1; i += (int64_t)gridDim.x * 4) {
    const bool second = i >= r0;
    const int64_t r = second ? i - r0 : i;
    const int8_t* src = (second ? w : x) + r * K;
    int8_t* dst = (second ? pw : px) + r * Kp;
    for (int c = (threadIdx.x & 63) * 16; c < Kp; c += 1024) *reinterpret_cast<i32v4*>(dst + c) = load_codes(src + c, K - c, K);
  }
}

template <int TJ> int launch_tiles(const ProductArgs& a, int dtype, hipStream_t st) {
  using T = Tile<TJ>;
  const int64_t tn = ceil_div(a.N, T::BN), tm = ceil_div(a.M, T::BM);
  if (!grid_fits(tn * tm, T::NT)) return fail(REELS_HIP_EINVAL, "reels_hip_i8i8_linear: too many output tiles for one launch");
  // the LDS size is an attribute of a kernel on a device: set once for each
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  hipError_t err = hipGetDevice(&dev);
  if (err == hipSuccess && (dev >= 64 || !(done.load(std::memory_order_relaxed) >> dev & 1))) {
    const void* ks[] = {(const void*)product_tile_kernel<REELS_HIP_BF16, TJ>, (const void*)product_tile_kernel<REELS_HIP_F16, TJ>,
                        (const void*)product_tile_kernel<REELS_HIP_F32, TJ>};
    for (const void* k : ks)
      if (err == hipSuccess) err = hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, T::LDS);
    if (err == hipSuccess && dev < 64) done.fetch_or((uint64_t)1 << dev, std::memory_order_relaxed);
  }
  if (err != hipSuccess)
    return fail(REELS_HIP_EHIP, std::string("product_tile: hipFuncSetAttribute: ") + hipGetErrorString(err));
  { TraceScope _ts(st, TJ == 8 ? "product_tile_kernel<256>" : "product_tile_kernel<128>");
    with_any_elt(dtype, [&](auto e) {
      product_tile_kernel<decltype(e)::value, TJ><<<(unsigned)(tn * tm), T::NT, T::LDS, st>>>(a, (int)tn, (int)tm);
    }); }
  return check_launch("product_tile_kernel");
}

// rows that the copies to LDS can take as they lie
bool whole_rows(const void* x, const void* w, int64_t K) { return K % 4 == 0 && ((uintptr_t)x & 3) == 0 && ((uintptr_t)w & 3) == 0; }

// The tiled form with the least estimated time, in microseconds. A workgroup's step of 128 codes
// takes about as long whatever the size: 64 x 64 tiles 0.27 us with one workgroup on a CU and 0.55
// with two, 128 x 128 tiles 0.75 and 1.15, 256 x 256 tiles (one per CU) 1.35; prologue and epilogue
// 4.5, 4 and 6 us. Measured with every form, 64 / 128 / 256 (us): 200 x 1536 -> 1536 5.6 / 12.7 /
// 20.9, 333 x 5120 -> 5120 18.7 / 31.8 / 50.9, 777 x 1024 -> 3001 12.7 / 11.5 / 18.5, 512 x 4096 ->
// 10240 47.8 / 38.9 / 48.3, 1560 x 1536 -> 8960 44.8 / 33.9 / 27.4, 2048 x 5120 -> 5120 119 / 70.0 /
// 53.7, 32760 x 5120 -> 5120 - / 928 / 670.
int tile_of(int64_t M, int64_t N, int64_t K) {
  const double steps = (double)ceil_div(K, 128);
  auto two = [](int64_t blocks, double one, double both) {  // two workgroups fit a CU
    const int64_t full = blocks / 512, rest = blocks % 512;
    return (double)full * both + (rest == 0 ? 0.0 : rest <= 256 ? one : both);
  };
  const double t64 = 4.5 + steps * two(ceil_div(M, 64) * ceil_div(N, 64), 0.27, 0.55);
  const double t128 = 4.0 + steps * two(ceil_div(M, 128) * ceil_div(N, 128), 0.75, 1.15);
  const double t256 = 6.0 + steps * 1.35 * (double)ceil_div(ceil_div(M, 256) * ceil_div(N, 256), 256);
  return t64 <= t128 && t64 <= t256 ? 64 : t128 <= t256 ? 128 : 256;
}

}  // namespace
}  // namespace reels

extern "C" size_t reels_hip_i8i8_workspace_bytes(int64_t M, int64_t K, int64_t N) {
  using namespace reels;
  if (M < 0 || K <= 0 || N <= 0 || M <= kFewTokens) return 0;
  return align_up((size_t)(M + N) * align_up((size_t)K, 128) + 256, 256);
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
  const bool copies = M > kFewTokens && !whole_rows(x, w, K);
  if (copies && (workspace == nullptr || ws_bytes < reels_hip_i8i8_workspace_bytes(M, K, N)))
    return fail(REELS_HIP_EWORKSPACE, fn + "workspace of reels_hip_i8i8_workspace_bytes required");
  if (M == 0) return REELS_HIP_OK;
  if (x == nullptr || xs == nullptr || w == nullptr || ws == nullptr || y == nullptr) return fail(REELS_HIP_EINVAL, fn + "NULL operand");
  const ProductArgs a{x, xs, w, ws, bias, residual, y, M, K, N, activation == REELS_HIP_ACT_GELU_TANH};
  if (M <= kFewTokens) {
    int rc = REELS_HIP_OK;
    with_any_elt(dtype, [&](auto e) {
      constexpr int E = decltype(e)::value;
      if (M == 1 && K >= kDotCodes) rc = launch_rows(product_dot_kernel<E>, "product_dot_kernel", N, 64, a, st);
      else rc = launch_rows(product_few_kernel<E>, "product_few_kernel", ceil_div(N, 16), kFewWaves * 64, a, st);
    });
    return rc;
  }
  ProductArgs c = a;
  if (copies) {
    const int Kp = (int)align_up((size_t)K, 128);
    int8_t* px = (int8_t*)align_up((size_t)workspace, 256);
    int8_t* pw = px + M * Kp;
    const int64_t blocks = ceil_div(M + N, 4);
    { TraceScope _ts(st, "product_pad_kernel");
      product_pad_kernel<<<(unsigned)(blocks < 8192 ? blocks : 8192), 256, 0, st>>>(x, M, w, N, (int)K, Kp, px, pw); }
    if (int rc = check_launch("product_pad_kernel")) return rc;
    c.x = px;
    c.w = pw;
    c.K = Kp;
  }
  const int tile = tile_of(M, N, c.K);
  return tile == 64 ? launch_small(c, dtype, st) : tile == 128 ? launch_tiles<4>(c, dtype, st) : launch_tiles<8>(c, dtype, st);
}
