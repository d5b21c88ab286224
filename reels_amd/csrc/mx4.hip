// Rows in microscaled 4 bits (microscale.h) and their product with a weight in the same form:
//
//   y[m][n] = rnd( act( sum_k x[m][k] w[n][k] + bias[n] ) + residual[m][n] )
//
// on the scaled matrix instructions of gfx950, which take 4-bit codes with one scale byte for 32 of them in each
// lane. The sums run in f32. The 32 x 32 x 64 form does 131072 operations in 32 clocks; the 16 x 16 x 128
// form of the same rate on paper reaches half of it here (registers alone, whole card: 6.6 and 4.4 PFLOP/s
// on varied codes, 9.8 and 5.2 on zeros; int8 2.4), so all but the few-token kernel use the first.
#include "microscale.h"

#include <atomic>

namespace reels {
namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef int v4i __attribute__((ext_vector_type(4)));

__device__ __forceinline__ v8i wide(const v4i& a) { return v8i{a[0], a[1], a[2], a[3], 0, 0, 0, 0}; }  // 4-bit operands use four registers

// ---- rows to 4 bits and back ---------------------------------------------------------------------
// 64 rows x 256 columns per workgroup, one tile of scale bytes: they are put together in LDS and leave in
// whole lines. A thread has 16 bytes of a row at a time, all its loads in flight. Bound by memory: 32760 x 13824
// bf16 242 us to 4 bits (4.7 TB/s), 200 back (5.7). Small matrices are bound by their few workgroups: 3001 x 1001 f32
// 188 of them on 256 CUs, 6.4 us and 6.6 back, where the bytes take 2.1.
template <int ELT> __global__ __launch_bounds__(256) void mx4_pack_kernel(const void* __restrict__ x, int64_t ld, int64_t rows, int64_t cols,
                                                                          int tiles, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  constexpr int V = Chunk<ELT>::V, EB = elt_bytes(ELT), LPR = 256 / V, RP = 256 / LPR, U = 8;
  __shared__ __attribute__((aligned(16))) uint8_t sc[512];
  const int kt = blockIdx.x % (unsigned)tiles;
  const int64_t tile = blockIdx.x / (unsigned)tiles, r0 = tile * 64 + threadIdx.x / LPR;
  const int64_t col = (int64_t)kt * 256 + (threadIdx.x % LPR) * V;
  const int left = cols - col < V ? (int)(cols - col) : V;
#pragma unroll
  for (int half = 0; half < 64 / (RP * U); ++half) {
    Chunk<ELT> c[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = r0 + (half * U + u) * RP;
      c[u].zero();
      if (row < rows && left > 0) c[u].load((const uint8_t*)x + (row * ld + col) * EB, left);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = r0 + (half * U + u) * RP;
      float f[V];
      c[u].unpack(f);
      const uint32_t byte = mx_exponent<2>(mx_top<kMxBlock / V>(mx_top_of<V>(f)));
      const uint32_t word = mx4_codes<V>(f, byte);
      const int in = (int)(row & 63), block = (threadIdx.x % LPR) * V / kMxBlock;
      if (threadIdx.x % (kMxBlock / V) == 0) sc[((block & 1) * 32 + (in & 31)) * 8 + (block >> 1) * 2 + (in >> 5)] = (uint8_t)byte;
      if (row >= rows) continue;
      uint8_t* p = codes + (row * tiles + kt) * 128 + (threadIdx.x % LPR) * V / 2;
      if constexpr (V == 8) *reinterpret_cast<uint32_t*>(p) = word;
      else *reinterpret_cast<uint16_t*>(p) = (uint16_t)word;
    }
  }
  __syncthreads();
  if (threadIdx.x < 128)
    reinterpret_cast<uint32_t*>(scales + (int64_t)blockIdx.x * 512)[threadIdx.x] = reinterpret_cast<const uint32_t*>(sc)[threadIdx.x];
}

template <int ELT> __global__ __launch_bounds__(256) void mx4_unpack_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                                            int64_t rows, int64_t cols, int tiles, void* __restrict__ y) {
  constexpr int EB = elt_bytes(ELT), V = 8, RP = 8, U = 8;
  typedef float f2 __attribute__((ext_vector_type(2)));
  const int kt = blockIdx.x % (unsigned)tiles;
  const int64_t r0 = (blockIdx.x / (unsigned)tiles) * 64 + threadIdx.x / 32;
  const int64_t col = (int64_t)kt * 256 + (threadIdx.x % 32) * V;
  const int left = cols - col < V ? (int)(cols - col) : V;
  if (left <= 0) return;
  uint32_t w[U], byte[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t row = r0 + u * RP;
    w[u] = byte[u] = 0u;
    if (row < rows) {
      w[u] = *reinterpret_cast<const uint32_t*>(codes + (row * tiles + kt) * 128 + (threadIdx.x % 32) * 4);
      byte[u] = scales[mx4_scale_at(row, (int)(col / kMxBlock), tiles)];
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t row = r0 + u * RP;
    if (row >= rows) continue;
    const float unit = mx4_unit(byte[u]);
    float f[V];
    const f2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], 1.0f, 1);
    const f2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], 1.0f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], 1.0f, 3);
    f[0] = a[0]; f[1] = a[1]; f[2] = b[0]; f[3] = b[1];
    f[4] = c[0]; f[5] = c[1]; f[6] = d[0]; f[7] = d[1];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      f[j] *= unit;
      // the largest values of a binary16 matrix can round up to 65536, past the type's range
      if (ELT == REELS_HIP_F16 && f[j] == f[j]) f[j] = __builtin_amdgcn_fmed3f(f[j], -65504.0f, 65504.0f);
    }
    store_vec<ELT, V>((uint8_t*)y + (row * cols + col) * EB, left, f);
  }
}

// ---- product -------------------------------------------------------------------------------------
constexpr int kFewTokens = 16;  // up to these a kernel of its own

struct Mx4Args {
  const uint8_t *x, *xs;  // codes [M][Kb], scale tiles
  const uint8_t *w, *ws;  // [N][Kb]
  const void* bias;       // [N] or nullptr
  const void* res;        // [M][N] or nullptr
  void* y;                // [M][N]
  int64_t M, N;
  int tiles, gelu;        // Kp / 256; Kb = 128 tiles
};

// gelu_tanh as a logistic function: x / (1 + exp(-2 k (x + 0.044715 x^3))), k = sqrt(2 / pi)
__device__ __forceinline__ float gelu_logistic(float x) {
  const float c = -2.3022082f;  // -2 sqrt(2 / pi) log2(e)
  const float e = __builtin_amdgcn_exp2f(x * fmaf(c * 0.044715f, x * x, c));
  return x * __builtin_amdgcn_rcpf(1.0f + e);
}

__device__ __forceinline__ f32x16 zeros16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.0f;
  return z;
}

// the product of two fragments; which byte of a lane's scale word belongs to them is part of the instruction
template <int SA, int SB> __device__ __forceinline__ f32x16 mfma(const v4i& a, const v4i& b, f32x16 c, uint32_t sa, uint32_t sb) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(a), wide(b), c, 4, 4, SA, (int)sa, SB, (int)sb);
}

// At the largest sizes bound by power: 32760 x 13824 -> 5120 takes 1070-1170 us (4.0-4.3 PFLOP/s) at 1.3-1.6 GHz, the
// products alone on operands in LDS 5.9 PFLOP/s; smaller ones by the first loads and the epilogue.
//
// 32 TJ x 32 TJ outputs per workgroup of TJ waves (TJ = 8: 256 x 256, TJ = 4: 128 x 128), each wave 16 TJ
// tokens x 64 columns, in steps of 128 codes (64 bytes of a row). The operands travel from HBM to LDS directly
// into a ring of four stages. While the products of step s run, the fragments of step s + 1 replace those that
// are used up; behind the first products of step s, when every wave has the last fragments of step s in
// registers, a barrier lets the copies of step s + 4 go into its stage, so a copy has three steps to arrive
// (a step of 256 codes in two stages gave it three quarters of one: 1176 us). Scale words, two steps' worth, go
// the same way in a ring of three. Rows past the edges read as zeros (the buffer's bounds, which count the
// scalar offset too and without a wrap), columns past K
// are zeros in the codes; copies past the last step read nothing, so that every step's waits count the same.
template <int TJ> struct Tile {
  static constexpr int NW = TJ, NT = NW * 64, WN = NW / 2, BM = 32 * TJ, BN = 64 * WN, BK = 64;
  static constexpr int ACT = BM * BK, WB = BN * BK, STAGE = ACT + WB, SCALES = NW * 512, LDS = 4 * STAGE + 3 * SCALES;
};

template <int ELT, int TJ>
__global__ __launch_bounds__(Tile<TJ>::NT, 2) void mx4_tile_kernel(Mx4Args a, int tiles_n, int tiles_m) {
  using T = Tile<TJ>;
  constexpr int V = 16 / elt_bytes(ELT), JT = TJ / 2, XT = TJ / 4;  // fragments of 32 tokens, tiles of 64
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const int t = threadIdx.x, lane = t & 63;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wm = w / T::WN, wn = w % T::WN, l32 = lane & 31, hi = lane >> 5;
  // consecutive tiles of one XCD share rows: groups of 4 tile rows, column by column
  const int nt = tiles_n * tiles_m, xcd = blockIdx.x & 7, idx = blockIdx.x >> 3;
  const int logical = xcd * (nt >> 3) + (xcd < (nt & 7) ? xcd : nt & 7) + idx;
  const int group = 4 * tiles_n, g = logical / group, first = g * 4;
  const int gm = tiles_m - first < 4 ? tiles_m - first : 4, within = logical - g * group;
  const int64_t m0 = (int64_t)(first + within % gm) * T::BM, n0 = (int64_t)(within / gm) * T::BN;
  const int Kb = a.tiles * 128, steps = a.tiles * 2;
  const int rows = (int)(a.M - m0 < T::BM ? a.M - m0 : T::BM), cols = (int)(a.N - n0 < T::BN ? a.N - n0 : T::BN);
  const i32x4 rx = buffer_rsrc(a.x + m0 * Kb, (uint32_t)rows * Kb), rw = buffer_rsrc(a.w + n0 * Kb, (uint32_t)cols * Kb);
  // Copy i of wave w: tile rows 16 (2 w + i) + lane / 4, 16 bytes per lane. Chunk c of a row of 64 bytes lies at
  // c ^ (row / 4 % 4): the 16 rows that a quarter of a fragment's lanes read lie in 64 different banks.
  const uint32_t vo = (uint32_t)((w * 32 + (lane >> 2)) * Kb + ((lane & 3) ^ (lane >> 4)) * 16);
  auto stage = [&](int s) { return smem + (s & 3) * T::STAGE; };
  auto issue = [&](int s, int q) {  // q: 0, 1 activations, 2, 3 weight
    i32x4 r = q < 2 ? rx : rw;
    r[2] = s < steps ? r[2] : 0;
    dma16(r, vo, (uint32_t)(s * T::BK + (q & 1) * 16 * Kb), stage(s) + (q < 2 ? 0 : T::ACT) + (w * 2 + (q & 1)) * 1024);
  };
  // scale words: wave w brings a tile of 64 rows' for two steps, lanes 0 .. 31. Tiles of rows past the last
  // read another's.
  const bool xs = w < T::NW / 2;
  const int64_t tile = xs ? m0 / 64 + w : n0 / 64 + w - T::NW / 2, last = ((xs ? a.M : a.N) + 63) / 64 - 1;
  const i32x4 rs = buffer_rsrc((xs ? a.xs : a.ws) + (tile < last ? tile : last) * a.tiles * 512, (uint32_t)a.tiles * 512);
  uint8_t* const ring = smem + 4 * T::STAGE;
  auto issue_scales = [&](int pair, int slot) {
    if (lane < 32) dma16(rs, (uint32_t)lane * 16, (uint32_t)pair * 512, ring + slot * T::SCALES + w * 512);
  };
  struct Scales { u32x2 x[XT], w; };
  auto read_scales = [&](int slot) {
    const uint8_t* p = ring + slot * T::SCALES + lane * 8;
    Scales s;
#pragma unroll
    for (int q = 0; q < XT; ++q) s.x[q] = *reinterpret_cast<const u32x2*>(p + (wm * XT + q) * 512);
    s.w = *reinterpret_cast<const u32x2*>(p + (T::NW / 2 + wn) * 512);
    return s;
  };

  f32x16 acc[2][JT];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < JT; ++j) acc[i][j] = zeros16();
  // where a lane's 16 bytes lie: chunk 2 ks + hi of its row, swizzled
  const int sel = (hi ^ (l32 >> 2 & 3)) << 4, xat = (wm * 16 * TJ + l32) * 64 + sel, wat = T::ACT + (wn * 64 + l32) * 64 + sel;
  // fragments of a step, 64 codes each: the weight's [ks][i], the activations' j = ks * JT + jt
  auto read_w = [&](const uint8_t* s, v4i (&f)[4]) {
#pragma unroll
    for (int q = 0; q < 4; ++q) f[q] = *reinterpret_cast<const v4i*>(s + (q & 1) * 2048 + (wat ^ ((q >> 1) << 5)));
  };
  auto read_x = [&](const uint8_t* s, int j) { return *reinterpret_cast<const v4i*>(s + (j % JT) * 2048 + (xat ^ ((j / JT) << 5))); };
  auto each = [&](auto&& f) {  // over the TJ activation fragments
    f(std::integral_constant<int, 0>{});
    f(std::integral_constant<int, 1>{});
    f(std::integral_constant<int, 2>{});
    f(std::integral_constant<int, 3>{});
    if constexpr (TJ == 8) {
      f(std::integral_constant<int, 4>{});
      f(std::integral_constant<int, 5>{});
      f(std::integral_constant<int, 6>{});
      f(std::integral_constant<int, 7>{});
    }
  };
  v4i w0[4], w1[4], x[TJ];
  // TJ = 4: the bias of the wave's columns, asked for here and used after the products
  typename Store<ELT>::raw bias = 0;
  if (TJ == 4 && a.bias != nullptr) {
    const int64_t n = n0 + wn * 64 + lane;
    bias = ((const typename Store<ELT>::raw*)a.bias)[n < a.N ? n : a.N - 1];
  }
  issue_scales(0, 0);
#pragma unroll
  for (int q = 0; q < 8; ++q) issue(q >> 2, q & 3);
  issue_scales(1, 1);
#pragma unroll
  for (int q = 8; q < 16; ++q) issue(q >> 2, q & 3);
  __builtin_amdgcn_s_waitcnt(0x0F7D);  // vmcnt(13): step 0 and its scale words have landed
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  Scales s0 = read_scales(0), s1;
  read_w(stage(0), w0);
#pragma unroll
  for (int j = 0; j < TJ; ++j) x[j] = read_x(stage(0), j);
  int slot = 0;  // of the pair's scale words
  // a step: its products on f, the next step's fragments into f1
  auto step = [&](int s, auto ec, v4i (&f)[4], v4i (&f1)[4]) {
    constexpr int e = decltype(ec)::value, B = TJ / 4 - 1;
    const uint8_t* sn = stage(s + 1);
    each([&](auto jc) {
      constexpr int j = decltype(jc)::value, ks = j / JT, jt = j % JT;
      acc[0][jt] = mfma<ks * 2, ks * 2 + (jt & 1)>(f[ks * 2], x[j], acc[0][jt], s0.w[e], s0.x[jt / 2][e]);
      acc[1][jt] = mfma<ks * 2 + 1, ks * 2 + (jt & 1)>(f[ks * 2 + 1], x[j], acc[1][jt], s0.w[e], s0.x[jt / 2][e]);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (j == B) {
        // This wave's fragments have arrived, and its copies of step s + 1 with their scale words: after them
        // two steps' copies and one of scale words were issued
        __builtin_amdgcn_s_waitcnt(0x0079);  // vmcnt(9) lgkmcnt(0)
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if constexpr (e == 0) issue_scales((s >> 1) + 2, slot == 0 ? 2 : slot - 1);
        else s1 = read_scales(slot == 2 ? 0 : slot + 1);
        read_w(sn, f1);
#pragma unroll
        for (int i = 0; i < j; ++i) x[i] = read_x(sn, i);
      }
      if constexpr (j >= B) {
        x[j] = read_x(sn, j);
        if constexpr (j - B < 4) issue(s + 4, j - B);
      }
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  for (int s = 0; s < steps; s += 2) {
    step(s, std::integral_constant<int, 0>{}, w0, w1);
    step(s + 1, std::integral_constant<int, 1>{}, w1, w0);
    s0 = s1;
    slot = slot == 2 ? 0 : slot + 1;
  }
  __builtin_amdgcn_s_waitcnt(0x0F70);  // no copy outlives the loop
  __syncthreads();
  if constexpr (TJ == 4) {
    // Outputs straight from the registers (777 x 1000 -> 3001 in f32, whose rows lie at odd offsets: 10.6 us,
    // by way of LDS 11.7): a lane has four columns each of its tokens; 16-bit types swap halves between lanes
    // l and l + 32, so that each has eight columns (16 bytes), two lanes 32 bytes of a row
    constexpr bool SWAP = V == 8;
    constexpr int PER = 16 / V;  // chunks of a lane's 16 values of a product
    const int64_t mrow = m0 + wm * 16 * TJ + l32, n1 = n0 + wn * 64;
    const int here = (int)(a.N - n1 < 64 ? a.N - n1 : 64);  // columns of the wave that exist, or none
    float* const biases = reinterpret_cast<float*>(smem) + w * 64;
    asm volatile("" : "+v"(bias));  // its conversion stays here, behind the wait for it
    biases[lane] = lane < here ? Store<ELT>::get(bias) : 0.0f;
    __builtin_amdgcn_s_waitcnt(0xC07F);
    asm volatile("" ::: "memory");
    auto column = [&](int i, int p) { return i * 32 + (SWAP ? p * 16 + hi * 8 : p * 8 + hi * 4); };
    auto leave = [&](auto all) {  // all: the wave's tokens and columns exist
      constexpr bool ALL = decltype(all)::value;
#pragma unroll
      for (int j = 0; j < JT; ++j) {
        const bool row = ALL || mrow + j * 32 < a.M;
        const int64_t at = (mrow + j * 32) * a.N + n1;
        Chunk<ELT> res[2][PER];
        if (a.res != nullptr) {
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int p = 0; p < PER; ++p) {
              // whole chunks without a branch, all in flight together: from the residual's start where a lane has
              // none (more than kFewTokens tokens: it has V elements)
              const int c = column(i, p);
              const int64_t from = ALL || (row && c + V <= here) ? at + c : 0;
              res[i][p].load((const uint8_t*)a.res + from * elt_bytes(ELT), V);
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int p = 0; p < PER; ++p) {
            const int c = column(i, p);
            float o[V];
#pragma unroll
            for (int q = 0; q < V / 4; ++q) {  // groups of four columns
              const int g4 = p * (V / 4) + q;
              const f32x4 b = *reinterpret_cast<const f32x4*>(biases + i * 32 + g4 * 8 + hi * 4);
#pragma unroll
              for (int v = 0; v < 4; ++v) o[q * 4 + v] = acc[i][j][g4 * 4 + v] + b[v];
            }
            if (a.gelu) {
#pragma unroll
              for (int v = 0; v < V; ++v) o[v] = gelu_logistic(o[v]);
            }
            if constexpr (SWAP) {
#pragma unroll
              for (int v = 0; v < 4; ++v) {
                const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(o[v]), __float_as_uint(o[4 + v]), false, false);
                o[v] = __uint_as_float(sw[0]);
                o[4 + v] = __uint_as_float(sw[1]);
              }
            }
            if (a.res != nullptr) {
              if (!ALL && row && c < here && c + V > here) res[i][p].load((const uint8_t*)a.res + (at + c) * elt_bytes(ELT), here - c);
#pragma unroll
              for (int v = 0; v < V; ++v) o[v] += res[i][p].get(v);
            }
            if (ALL || (row && c < here)) store_vec<ELT, V>((uint8_t*)a.y + (at + c) * elt_bytes(ELT), ALL ? V : here - c, o);
          }
      }
    };
    if (here == 64 && m0 + (wm + 1) * 16 * TJ <= a.M) leave(std::true_type{});
    else leave(std::false_type{});
    return;
  } else {
    uint8_t* out = smem + w * 16384;
    // Epilogue: f32 values of 64 tokens x 64 columns at a time in the wave's own 16 KiB of LDS (rows of
    // 256 bytes, 16-byte chunks XOR-swizzled), read back as rows: bias, residual and stores in whole segments
    constexpr int LPR = 64 / V, RPI = 64 / LPR, ITS = 64 / RPI;  // lanes of a row, rows at once, turns
    const int c = (lane % LPR) * V, left = cols - (wn * 64 + c);
    float bs[V];
#pragma unroll
    for (int v = 0; v < V; ++v) bs[v] = 0.0f;
    if (a.bias != nullptr && left > 0) load_vec<ELT, V>((const uint8_t*)a.bias + (n0 + wn * 64 + c) * elt_bytes(ELT), left, bs);
#pragma unroll
    for (int h = 0; h < TJ / 4; ++h) {
      // the residual's whole chunks on their way while the values are put in place; from its start where a
      // lane has none (more than kFewTokens tokens: it has V elements)
      Chunk<ELT> res[ITS];
      if (a.res != nullptr) {
#pragma unroll
        for (int it = 0; it < ITS; ++it) {
          const int mr = wm * 16 * TJ + h * 64 + it * RPI + lane / LPR;
          const int64_t at = mr < rows && left >= V ? (m0 + mr) * a.N + n0 + wn * 64 + c : 0;
          res[it].d = load_any<u32x4>((const typename Store<ELT>::raw*)((const uint8_t*)a.res + at * elt_bytes(ELT)));
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int r = j * 32 + l32;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            f32x4 o;
#pragma unroll
            for (int v = 0; v < 4; ++v) o[v] = acc[i][h * 2 + j][q * 4 + v];
            *reinterpret_cast<f32x4*>(out + r * 256 + (((i * 8 + q * 2 + hi) ^ (r & 15)) << 4)) = o;
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
          const f32x4 f = *reinterpret_cast<const f32x4*>(out + r * 256 + (((c / 4 + q) ^ (r & 15)) << 4));
#pragma unroll
          for (int v = 0; v < 4; ++v) o[q * 4 + v] = f[v] + bs[q * 4 + v];
        }
        if (a.gelu) {
#pragma unroll
          for (int v = 0; v < V; ++v) o[v] = gelu_logistic(o[v]);
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
}

// bias, activation and residual of four columns n.. (left of them exist) of token m, then one rounding
template <int ELT> __device__ __forceinline__ void finish4(const Mx4Args& a, int64_t m, int64_t n, int left, f32x4 o, const float (&bs)[4]) {
  float f[4];
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    f[v] = o[v] + bs[v];
    if (a.gelu) f[v] = gelu_logistic(f[v]);
  }
  const int64_t at = (m * a.N + n) * elt_bytes(ELT);
  if (a.res != nullptr) {
    float e[4];
    load_vec<ELT, 4>((const uint8_t*)a.res + at, left, e);
#pragma unroll
    for (int v = 0; v < 4; ++v) f[v] += e[v];
  }
  store_vec<ELT, 4>((uint8_t*)a.y + at, left, f);
}
template <int ELT> __device__ __forceinline__ void load_bias(const Mx4Args& a, int64_t n, int left, float (&bs)[4]) {
#pragma unroll
  for (int v = 0; v < 4; ++v) bs[v] = 0.0f;
  if (a.bias != nullptr) load_vec<ELT, 4>((const uint8_t*)a.bias + n * elt_bytes(ELT), left, bs);
}

// ---- small tiles ---------------------------------------------------------------------------------
// 64 x 64 outputs per workgroup of eight waves, a step of 256 codes: for token counts whose larger tiles
// would leave most CUs idle. Waves w and w + 4 own the same 32 x 32 outputs and take the two halves of a
// step's codes (their sums are added in LDS at the end). A ring of four stages, three steps in flight and one
// barrier per step; two workgroups fit a CU. The scale words come the same way, 512 bytes an operand and step,
// from waves 0 and 1; the others issue a copy that reads nothing, so that the waits count the same. 64 x 5120 -> 5120
// 9.1 us in a row of calls: 80 workgroups with 20 steps and a barrier each, so 176 CUs have nothing to do; the weight's
// bytes alone take 2.1. K is not divided among workgroups.
namespace small {
constexpr int BT = 64, BK = 128, STAGE = 2 * BT * BK + 2048, RING = 4, NT = 512, LDS = RING * STAGE + 1024;
}

template <int ELT> __global__ __launch_bounds__(small::NT) void mx4_small_kernel(Mx4Args a, int tiles_m) {
  using namespace small;
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const int t = threadIdx.x, lane = t & 63;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int h = w >> 2, wm = (w >> 1) & 1, wn = w & 1, l32 = lane & 31, hi = lane >> 5;
  // the token tiles of one weight tile follow each other on one XCD: its codes come to that L2 once
  const int xcd = blockIdx.x & 7, nt = gridDim.x;
  const int logical = xcd * (nt >> 3) + (xcd < (nt & 7) ? xcd : nt & 7) + (blockIdx.x >> 3);
  const int64_t tm = logical % tiles_m, tn = logical / tiles_m, m0 = tm * BT, n0 = tn * BT;
  const int Kb = a.tiles * 128, nk = a.tiles;
  const int rows = (int)(a.M - m0 < BT ? a.M - m0 : BT), cols = (int)(a.N - n0 < BT ? a.N - n0 : BT);
  const i32x4 rx = buffer_rsrc(a.x + m0 * Kb, (uint32_t)rows * Kb), rw = buffer_rsrc(a.w + n0 * Kb, (uint32_t)cols * Kb);
  const i32x4 rs = buffer_rsrc(w == 0 ? a.xs + tm * a.tiles * 512 : a.ws + tn * a.tiles * 512, w < 2 ? (uint32_t)a.tiles * 512 : 0u);
  const int crow = w * 8 + (lane >> 3);  // a wave copies rows 8 w .. 8 w + 7 of each tile
  const uint32_t vo = (uint32_t)(crow * Kb + ((lane & 7) ^ (crow >> 1 & 7)) * 16);
  auto issue = [&](int kt) {  // past the end the copies read nothing, so that the waits count the same
    uint8_t* s = smem + (kt & (RING - 1)) * STAGE;
    const bool in = kt < nk;
    i32x4 cx = rx, cw = rw, cs = rs;
    cx[2] = in ? rx[2] : 0;
    cw[2] = in ? rw[2] : 0;
    cs[2] = in ? rs[2] : 0;
    dma16(cx, vo, (uint32_t)kt * BK, s + w * 1024);
    dma16(cw, vo, (uint32_t)kt * BK, s + BT * BK + w * 1024);
    // lanes 32 .. 63 bring the next step's words, which nobody reads here
    dma16(cs, lane * 16, (uint32_t)kt * 512, w < 2 ? s + 2 * BT * BK + w * 1024 : smem + RING * STAGE);
  };
#pragma unroll
  for (int kt = 0; kt < RING - 1; ++kt) issue(kt);
  f32x16 acc = zeros16();
  const int off0 = ((4 * h + hi) ^ (l32 >> 1 & 7)) << 4, off1 = off0 ^ 32;
  for (int kt = 0; kt < nk; ++kt) {
    __builtin_amdgcn_s_waitcnt(0x0F76);  // vmcnt(6): step kt has landed, the two after it may fly
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    const uint8_t* s = smem + (kt & (RING - 1)) * STAGE;
    const uint8_t* px = s + (wm * 32 + l32) * 128;
    const uint8_t* pw = s + BT * BK + (wn * 32 + l32) * 128;
    const v4i x0 = *reinterpret_cast<const v4i*>(px + off0), w0 = *reinterpret_cast<const v4i*>(pw + off0);
    const v4i x1 = *reinterpret_cast<const v4i*>(px + off1), w1 = *reinterpret_cast<const v4i*>(pw + off1);
    // the word's bytes: [64 codes of this half][32 rows]
    const uint32_t sx = *reinterpret_cast<const uint32_t*>(s + 2 * BT * BK + lane * 8 + h * 4) >> (8 * wm);
    const uint32_t sw = *reinterpret_cast<const uint32_t*>(s + 2 * BT * BK + 1024 + lane * 8 + h * 4) >> (8 * wn);
    issue(kt + RING - 1);  // into the stage of step kt - 1, which every wave has read
    acc = mfma<0, 0>(w0, x0, acc, sw, sx);
    acc = mfma<2, 2>(w1, x1, acc, sw, sx);
    // the fragments are in registers before the next barrier lets their stage be overwritten
    __builtin_amdgcn_s_waitcnt(0xC07F);
  }
  __builtin_amdgcn_s_waitcnt(0x0F70);  // no copy outlives the loop
  __syncthreads();
  f32x4* part = reinterpret_cast<f32x4*>(smem) + (w & 3) * 256 + lane;
  if (h == 1) {
#pragma unroll
    for (int q = 0; q < 4; ++q) part[q * 64] = f32x4{acc[q * 4], acc[q * 4 + 1], acc[q * 4 + 2], acc[q * 4 + 3]};
  }
  __syncthreads();
  if (h == 1) return;
  const int mr = wm * 32 + l32;
  if (mr >= rows) return;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int nb = wn * 32 + q * 8 + hi * 4, left = cols - nb;
    if (left <= 0) continue;
    float bs[4];
    load_bias<ELT>(a, n0 + nb, left, bs);
    f32x4 o = part[q * 64];
#pragma unroll
    for (int v = 0; v < 4; ++v) o[v] += acc[q * 4 + v];
    finish4<ELT>(a, m0 + mr, n0 + nb, left, o, bs);
  }
}

// ---- few tokens ----------------------------------------------------------------------------------
// Up to 16 tokens: 16 outputs per workgroup, its waves take lines of 256 codes in turn and read codes and
// scale words straight into registers (each code of the weight is used once, so LDS would only add a trip),
// then add their sums in LDS in wave order. Lanes of tokens that are not there read nothing (an offset past the
// buffer's bounds). Bound by the weight's bytes and by latency: 1 x 5120 -> 13824 12 us (3.1 TB/s) between events,
// 9.8 a call in a row of calls.
constexpr int kFewWaves = 8;  // the most of a workgroup

template <int ELT> __global__ __launch_bounds__(kFewWaves * 64) void mx4_few_kernel(Mx4Args a) {
  __shared__ f32x4 part[kFewWaves][64];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, lq = lane >> 4;
  const int waves = (int)(blockDim.x >> 6);
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const int Kb = a.tiles * 128, rows = (int)(a.N - n0 < 16 ? a.N - n0 : 16);
  auto buffer = [](const uint8_t* p, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), (short)0, (int)bytes, 0x00020000);
  };
  const __amdgpu_buffer_rsrc_t rw = buffer(a.w + n0 * Kb, (uint32_t)rows * Kb), rx = buffer(a.x, (uint32_t)a.M * Kb);
  const __amdgpu_buffer_rsrc_t rws = buffer(a.ws + (n0 >> 6) * a.tiles * 512, (uint32_t)a.tiles * 512);
  const __amdgpu_buffer_rsrc_t rxs = buffer(a.xs, (uint32_t)a.tiles * 512);
  const uint32_t none = 0x80000000u, vw = (uint32_t)(l16 * Kb + lq * 16), vx = l16 < a.M ? vw : none;
  // a lane's blocks lq and 4 + lq of a line: the same byte of the two words
  const int nr = (int)(n0 & 63) + l16;  // n0 is a multiple of 16: all rows of one tile
  const uint32_t vws = (uint32_t)(((lq & 1) * 32 + (nr & 31)) * 8), vxs = l16 < a.M ? (uint32_t)(((lq & 1) * 32 + l16) * 8) : none;
  const int bw = 8 * ((lq >> 1) * 2 + (nr >> 5)), bx = 8 * ((lq >> 1) * 2);
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  int s = w;
  auto run = [&](auto count) {  // so many lines at once, all their loads in flight
    constexpr int C = decltype(count)::value;
    v4i wf[C][2], xf[C][2];
    u32x2 cw[C], cx[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int k = s + c * waves;
      wf[c][0] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rw, vw, k * 128, 0));
      wf[c][1] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rw, vw + 64, k * 128, 0));
      cw[c] = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rws, vws, k * 512, 0));
      xf[c][0] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rx, vx, k * 128, 0));
      xf[c][1] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rx, vx + 64, k * 128, 0));
      cx[c] = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rxs, vxs, k * 512, 0));
    }
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int q = 0; q < 2; ++q)
        acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(wf[c][q]), wide(xf[c][q]), acc, 4, 4, 0, (int)(cw[c][q] >> bw), 0,
                                                               (int)(cx[c][q] >> bx));
    s += C * waves;
  };
  while (s + 2 * waves < a.tiles) run(std::integral_constant<int, 3>{});
  if (s + waves < a.tiles) run(std::integral_constant<int, 2>{});
  else if (s < a.tiles) run(std::integral_constant<int, 1>{});
  part[w][lane] = acc;
  __syncthreads();
  if (w > 0) return;
  for (int i = 1; i < waves; ++i) {
    const f32x4 o = part[i][lane];
#pragma unroll
    for (int v = 0; v < 4; ++v) acc[v] += o[v];
  }
  const int64_t nb = n0 + lq * 4;
  if (l16 >= a.M || nb >= a.N) return;
  const int left = a.N - nb < 4 ? (int)(a.N - nb) : 4;
  float bs[4];
  load_bias<ELT>(a, nb, left, bs);
  finish4<ELT>(a, l16, nb, left, acc, bs);
}

// ---- host ----------------------------------------------------------------------------------------
// the LDS size is an attribute of a kernel on a device: set once for each
template <typename K> hipError_t lds_size(std::atomic<uint64_t>& done, int bytes, K&& kernels) {
  int dev = 0;
  hipError_t err = hipGetDevice(&dev);
  if (err == hipSuccess && (dev >= 64 || !(done.load(std::memory_order_relaxed) >> dev & 1))) {
    for (const void* k : kernels)
      if (err == hipSuccess) err = hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (err == hipSuccess && dev < 64) done.fetch_or((uint64_t)1 << dev, std::memory_order_relaxed);
  }
  return err;
}

int too_many() { return fail(REELS_HIP_EINVAL, "reels_hip_mx4_linear: too many outputs for one launch"); }
int lds_error(hipError_t err) {
  return fail(REELS_HIP_EHIP, std::string("reels_hip_mx4_linear: hipFuncSetAttribute: ") + hipGetErrorString(err));
}

template <int TJ> int launch_tiles(const Mx4Args& a, int dtype, hipStream_t st) {
  using T = Tile<TJ>;
  const int64_t tn = ceil_div(a.N, T::BN), tm = ceil_div(a.M, T::BM);
  if (!grid_fits(tn * tm, T::NT)) return too_many();
  static std::atomic<uint64_t> done{0};
  const void* ks[] = {(const void*)mx4_tile_kernel<REELS_HIP_BF16, TJ>, (const void*)mx4_tile_kernel<REELS_HIP_F16, TJ>,
                      (const void*)mx4_tile_kernel<REELS_HIP_F32, TJ>};
  if (hipError_t err = lds_size(done, T::LDS, ks); err != hipSuccess) return lds_error(err);
  { TraceScope _ts(st, TJ == 8 ? "mx4_tile_kernel<256>" : "mx4_tile_kernel<128>");
    with_any_elt(dtype, [&](auto e) {
      mx4_tile_kernel<decltype(e)::value, TJ><<<(unsigned)(tn * tm), T::NT, T::LDS, st>>>(a, (int)tn, (int)tm);
    }); }
  return check_launch("mx4_tile_kernel");
}

int launch_small(const Mx4Args& a, int dtype, hipStream_t st) {
  const int64_t tn = ceil_div(a.N, small::BT), tm = ceil_div(a.M, small::BT);
  if (!grid_fits(tn * tm, small::NT)) return too_many();
  static std::atomic<uint64_t> done{0};
  const void* ks[] = {(const void*)mx4_small_kernel<REELS_HIP_BF16>, (const void*)mx4_small_kernel<REELS_HIP_F16>,
                      (const void*)mx4_small_kernel<REELS_HIP_F32>};
  if (hipError_t err = lds_size(done, small::LDS, ks); err != hipSuccess) return lds_error(err);
  { TraceScope _ts(st, "mx4_small_kernel");
    with_any_elt(dtype, [&](auto e) {
      mx4_small_kernel<decltype(e)::value><<<(unsigned)(tn * tm), small::NT, small::LDS, st>>>(a, (int)tm);
    }); }
  return check_launch("mx4_small_kernel");
}

// The tiled form with the least estimated time, in microseconds: a workgroup's step of 256 codes takes 0.32 us
// in the 64 x 64 form with one workgroup on a CU and 0.61 with two, 0.48 and 1.1 in the 128 x 128 form, 1.5 in the
// 256 x 256 form (one on a CU); beginning and end 4.5, 5 and 6 us. Fitted to one round of tiles; over several the
// steps are slower and each round has an end of its own (32760 x 1536 -> 1536 is put at 33 us in the 256 form, 32760 x
// 13824 -> 5120 at 816), which moves the choice by 5% at most in what was measured. Every form, 64 / 128 / 256, us in a
// row of calls, the rule's own marked:
// 200 x 1536 -> 1536 7.8* / 7.7 / 13.5, 333 x 5120 -> 5120 14.1 / 13.7* / 31.1, 777 x 1024 -> 3001 9.9 / 7.9* / 12.8,
// 512 x 4096 -> 10240 28.1 / 21.3* / 28.4, 1560 x 1536 -> 8960 39.2 / 23.5 / 21.4*, 2048 x 5120 -> 5120 73.9 / 43.6 /
// 38.4*, 4096 x 5120 -> 5120 144 / 79* / 77, 8192 x 5120 -> 5120 277 / 144 / 125*, 32760 x 1536 -> 1536 145 / 62.0 / 63.0*,
// 32760 x 13824 -> 5120 - / 1517 / 1074*.
int tile_of(int64_t M, int64_t N, int64_t steps) {
  auto two = [](int64_t blocks, double one, double both) {  // two workgroups fit a CU
    const int64_t full = blocks / 512, rest = blocks % 512;
    return (double)full * both + (rest == 0 ? 0.0 : rest <= 256 ? one : both);
  };
  const double t64 = 4.5 + steps * two(ceil_div(M, 64) * ceil_div(N, 64), 0.32, 0.61);
  const double t128 = 5.0 + steps * two(ceil_div(M, 128) * ceil_div(N, 128), 0.48, 1.1);
  const double t256 = 6.0 + steps * 1.5 * (double)ceil_div(ceil_div(M, 256) * ceil_div(N, 256), 256);
  return t64 <= t128 && t64 <= t256 ? 64 : t128 <= t256 ? 128 : 256;
}

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

int rows_check(const std::string& fn, int dtype, int64_t rows, int64_t cols, const void* codes, const void* scales) {
  if (!known_elt(dtype)) return fail(REELS_HIP_EDTYPE, fn + "dtype must be f32, bf16 or f16");
  if (rows < 0 || cols <= 0 || cols >= (1 << 24) || rows > ((int64_t)1 << 31) - 1)
    return fail(REELS_HIP_EINVAL, fn + "0 <= rows < 2^31 and 0 < cols < 2^24 required");
  if (!aligned(codes, 16) || !aligned(scales, 16)) return fail(REELS_HIP_EINVAL, fn + "codes and scales must be 16-byte aligned");
  if (!grid_fits(ceil_div(rows, 64) * ceil_div(cols, 256), 256)) return fail(REELS_HIP_EINVAL, fn + "too many elements for one launch");
  return REELS_HIP_OK;
}

}  // namespace
}  // namespace reels

extern "C" size_t reels_hip_mx4_codes_bytes(int64_t rows, int64_t cols) {
  return rows <= 0 || cols <= 0 ? 0 : (size_t)rows * (size_t)reels::ceil_div(cols, 256) * 128;
}
extern "C" size_t reels_hip_mx4_scales_bytes(int64_t rows, int64_t cols) {
  return rows <= 0 || cols <= 0 ? 0 : (size_t)reels::ceil_div(rows, 64) * (size_t)reels::ceil_div(cols, 256) * 512;
}

extern "C" int reels_hip_mx4_pack(const void* x, int64_t ld_x, int dtype, int64_t rows, int64_t cols, uint8_t* codes, uint8_t* scales,
                                  void* stream) {
  using namespace reels;
  clear_error();
  const std::string fn = "reels_hip_mx4_pack: ";
  if (int rc = rows_check(fn, dtype, rows, cols, codes, scales)) return rc;
  if (ld_x < cols) return fail(REELS_HIP_EINVAL, fn + "row stride below cols");
  if (rows == 0) return REELS_HIP_OK;
  if (x == nullptr || codes == nullptr || scales == nullptr) return fail(REELS_HIP_EINVAL, fn + "NULL operand");
  const int tiles = (int)ceil_div(cols, 256);
  const hipStream_t st = (hipStream_t)stream;
  { TraceScope _ts(st, "mx4_pack_kernel");
    with_any_elt(dtype, [&](auto e) {
      mx4_pack_kernel<decltype(e)::value><<<(unsigned)(ceil_div(rows, 64) * tiles), 256, 0, st>>>(x, ld_x, rows, cols, tiles, codes, scales);
    }); }
  return check_launch("mx4_pack_kernel");
}

extern "C" int reels_hip_mx4_unpack(const uint8_t* codes, const uint8_t* scales, int dtype, int64_t rows, int64_t cols, void* y,
                                    void* stream) {
  using namespace reels;
  clear_error();
  const std::string fn = "reels_hip_mx4_unpack: ";
  if (int rc = rows_check(fn, dtype, rows, cols, codes, scales)) return rc;
  if (rows == 0) return REELS_HIP_OK;
  if (y == nullptr || codes == nullptr || scales == nullptr) return fail(REELS_HIP_EINVAL, fn + "NULL operand");
  const int tiles = (int)ceil_div(cols, 256);
  const hipStream_t st = (hipStream_t)stream;
  { TraceScope _ts(st, "mx4_unpack_kernel");
    with_any_elt(dtype, [&](auto e) {
      mx4_unpack_kernel<decltype(e)::value><<<(unsigned)(ceil_div(rows, 64) * tiles), 256, 0, st>>>(codes, scales, rows, cols, tiles, y);
    }); }
  return check_launch("mx4_unpack_kernel");
}

extern "C" int reels_hip_mx4_linear(const uint8_t* x, const uint8_t* x_scales, const uint8_t* w, const uint8_t* w_scales, const void* bias,
                                    const void* residual, int activation, int dtype, int64_t M, int64_t K, int64_t N, void* y,
                                    void* stream) {
  using namespace reels;
  clear_error();
  const std::string fn = "reels_hip_mx4_linear: ";
  const hipStream_t st = (hipStream_t)stream;
  if (activation != REELS_HIP_ACT_NONE && activation != REELS_HIP_ACT_GELU_TANH) return fail(REELS_HIP_EINVAL, fn + "unknown activation");
  if (int rc = rows_check(fn, dtype, M, K, x, x_scales)) return rc;
  if (int rc = rows_check(fn, dtype, N, K, w, w_scales)) return rc;
  if (N == 0) return fail(REELS_HIP_EINVAL, fn + "N must be positive");
  if (M == 0) return REELS_HIP_OK;
  if (x == nullptr || x_scales == nullptr || w == nullptr || w_scales == nullptr || y == nullptr) return fail(REELS_HIP_EINVAL, fn + "NULL operand");
  const Mx4Args a{x, x_scales, w, w_scales, bias, residual, y, M, N, (int)ceil_div(K, 256), activation == REELS_HIP_ACT_GELU_TANH};
  if (M <= kFewTokens) {
    const int64_t grid = ceil_div(N, 16);
    const int waves = a.tiles < kFewWaves ? a.tiles : kFewWaves;  // 4 to 16 are within 2% of each other where there are as many lines
    if (!grid_fits(grid, waves * 64)) return too_many();
    { TraceScope _ts(st, "mx4_few_kernel");
      with_any_elt(dtype, [&](auto e) { mx4_few_kernel<decltype(e)::value><<<(unsigned)grid, waves * 64, 0, st>>>(a); }); }
    return check_launch("mx4_few_kernel");
  }
  const int tile = tile_of(M, N, a.tiles);
  return tile == 64 ? launch_small(a, dtype, st) : tile == 128 ? launch_tiles<4>(a, dtype, st) : launch_tiles<8>(a, dtype, st);
}
