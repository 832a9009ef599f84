// Projections with 8-bit weights.
//
// A row t of K values is held as codes q in [-127, 127] and one scale s = max|t| / 127:
// q = 127 t / max|t| rounded to the nearest whole number, ties to even, exactly (not
// through a rounded quotient), so codes hang on the row alone and any program that
// rounds exactly gets the same ones.  A row of zeros has scale 0, a row with an
// infinity or NaN scale NaN and codes 0: its outputs are NaN.  Codes of a row take Kp
// bytes, K up to whole groups of 128, zeros behind.
//
// A product y[m][n] = s_m w_n sum_k q[m][k] c[n][k] is summed in whole numbers on the
// 8-bit matrix cores (K below 2^17, so 32 bits hold any sum of products): sums are exact and
// their order does not matter, however K is cut.
//
// A normalised row is coded as t = fp32(x gain) with the norm's factor in its scale: the
// factor is the whole row's, so it moves no code, and sums of squares in another order
// change none.  Factor and scale are taken in 64 bits and rounded once.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "sk_lds.h"

// Each operation rounds by itself (fused ones are written as such): all kernels give the same bits.
#pragma clang fp contract(off)

namespace sk {
namespace int8 {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));

constexpr int GROUP = 128;                        // codes of a row: whole groups of these

template <typename X> __device__ __forceinline__ float to_f(X v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<uint16_t>(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
template <typename X> __device__ __forceinline__ X from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ uint16_t from_f<uint16_t>(float v) {
  return __builtin_bit_cast(uint16_t, (__bf16)v);
}

// ------------------------------------------------------------ codes of a row

// 8 neighbouring values of a row from k on, 0 past K.  WHOLE: K is a multiple of 8, so
// that rows are aligned for pieces of 8.
template <typename X, bool WHOLE>
__device__ __forceinline__ void load8(const X* row, int k, int K, float (&t)[8]) {
  if constexpr (WHOLE) {                          // past K the last piece is loaded, and not taken
    const X* p = row + min(k, K - 8);
    if constexpr (sizeof(X) == 2) {
      const uint4 v = *reinterpret_cast<const uint4*>(p);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t x = k < K ? w[i] : 0u;
        t[2 * i] = __uint_as_float(x << 16);
        t[2 * i + 1] = __uint_as_float(x & 0xffff0000u);
      }
    } else {
      const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
      const float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = k < K ? x[i] : 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = k + i < K ? to_f<X>(row[k + i]) : 0.f;
  }
}
// x^2 of 8 values, and t times the gain (rounded to FP32: the definition's one rounding).
enum { PLAIN = 0, NORM = 1, GAIN = 2 };           // what becomes of a row first: nothing, a norm, a norm with a gain
template <bool WHOLE, int MODE>
__device__ __forceinline__ float weigh8(const float* gain, int k, int K, float (&t)[8]) {
  float squares = 0.f;
  if constexpr (MODE != PLAIN)
#pragma unroll
    for (int i = 0; i < 8; ++i) squares = fmaf(t[i], t[i], squares);
  if constexpr (MODE == GAIN) {
    float g[8];
    load8<float, WHOLE>(gain, k, K, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] *= g[i];
  }
  return squares;
}
// The largest |t| as bits: NaN above infinity above every number.
__device__ __forceinline__ uint32_t top8(const float (&t)[8], uint32_t top) {
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(t[i]) & 0x7fffffffu);
  return top;
}

// How a row with this largest |t| is coded.  Rows of less than 2^-60 or more than 2^100 are multiplied by a
// power of two first (exact but for values that are no code), so that nothing below over- or underflows.
struct Coder {
  float r, up, top;                               // 127 / (top up), up, top up
  float scale;                                    // top / 127
  float plain;                                    // top, NaN where it is no number
  __device__ explicit Coder(uint32_t bits) {
    const float t = __uint_as_float(bits);
    const bool bad = bits >= 0x7f800000u;
    up = t < 0x1p-60f ? 0x1p80f : t > 0x1p100f ? 0x1p-20f : 1.f;
    top = t * up;
    r = bad || bits == 0 ? 0.f : 127.f / top;
    plain = bad ? __uint_as_float(0x7fc00000u) : t;
    scale = plain / 127.f;
  }
  // fp32(top / 127 / sqrt(m)), m a mean of squares and eps: the GPU's own reciprocal root, within 2^-24, and one step of Newton's.
  __device__ __forceinline__ float normed(double m) const {
    double r = __builtin_amdgcn_rsq(m);
    r *= fma(-0.5 * m * r, r, 1.5);
    return (float)((double)plain * (1.0 / 127.0) * r);
  }
  // The nearest whole number of 127 t / top, t multiplied by up, exactly.  With the middle m = floor(t r) + 1/2 (floor
  // of the rounded product may be one off next to a whole number, where the other side of m decides alike), m top
  // is ph + pl exactly; 127 t - ph is rounded where it is far from 0, and exact where it matters: next to a
  // middle it is below 2^-13 top, a multiple of t's last place.
  __device__ __forceinline__ int exact(float t) const {
    const float l = floorf(t * r), m = l + 0.5f;
    const float ph = m * top, pl = fmaf(m, top, -ph), d = fmaf(127.f, t, -ph);
    const int c = (int)l;
    return c + (d > pl ? 1 : d < pl ? 0 : (c & 1));
  }
  // Values as the others want them.
  __device__ __forceinline__ void scale8(float (&t)[8]) const {
    if (up != 1.f)                                // the row's: all lanes alike
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] *= up;
  }
  // 8 codes; of a row that has none (r = 0: zeros, infinities, NaN) zeros.  The rounded product t r is off by at
  // most 127 * 2^-23 = 1.5e-5; adding 1.5 * 2^23 rounds it to a whole number, which the sum's lowest
  // byte holds.  Where one of a wave's is within 1e-4 of a middle, as quotients of BF16 values often are, they
  // are taken exactly (12,288 x 2048 in BF16: most waves).
  __device__ __forceinline__ uint2 code8(const float (&t)[8]) const {
    constexpr float MAGIC = 12582912.f;
    uint32_t q[8];
    float far = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float f = t[i] * r, s = f + MAGIC;
      q[i] = __float_as_uint(s);
      far = fmaxf(far, fabsf(f - (s - MAGIC)));
    }
    if (__any(far > 0.4999f)) {
#pragma unroll
      for (int i = 0; i < 8; ++i) q[i] = (uint32_t)exact(t[i]);
    }
    auto pack = [](uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
      return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400u), __builtin_amdgcn_perm(b, a, 0x0c0c0400u), 0x05040100u);
    };
    const uint32_t some = r != 0.f ? ~0u : 0u;
    return make_uint2(pack(q[0], q[1], q[2], q[3]) & some, pack(q[4], q[5], q[6], q[7]) & some);
  }
};

// Over a wave, in every lane: 16 neighbours by exchanges in registers, then the four groups.
template <int CTRL>
__device__ __forceinline__ int dpp(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, true); }
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  v = max(v, (uint32_t)dpp<0xb1>((int)v));        // quad_perm [1,0,3,2]
  v = max(v, (uint32_t)dpp<0x4e>((int)v));        // quad_perm [2,3,0,1]
  v = max(v, (uint32_t)dpp<0x141>((int)v));       // row_half_mirror
  v = max(v, (uint32_t)dpp<0x140>((int)v));       // row_mirror
  auto at = [&](int l) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); };
  return max(max(at(0), at(16)), max(at(32), at(48)));
}
__device__ __forceinline__ float wave_sum(float v) {
  v += __int_as_float(dpp<0xb1>(__float_as_int(v)));
  v += __int_as_float(dpp<0x4e>(__float_as_int(v)));
  v += __int_as_float(dpp<0x141>(__float_as_int(v)));
  v += __int_as_float(dpp<0x140>(__float_as_int(v)));
  auto at = [&](int l) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), l)); };
  return (at(0) + at(16)) + (at(32) + at(48));
}

// Sums of squares have one order whatever holds the row, so that a row's norm does not
// hang on the size of the call: 8 values one after the other, the 64 such sums of a block of 512 by
// wave_sum, the blocks one after the other.
constexpr int BLOCK = 512;
// The mean of a row's squares, in every lane of a whole wave.  Past FP32's range, or so far below it that squares lose bits which
// eps does not cover (up to 2^17 squares are each off by 2^-150), it is summed again in 64 bits from the row itself.
template <typename X>
__device__ __forceinline__ double mean_of(const X* x, const float* blocks, int K, double per, float eps) {
  float s = 0.f;
  for (int b = 0; b * BLOCK < K; ++b) s += blocks[b];
  double t = s;
  if (!(s <= 3.402823466e38f && (s >= 0x1p-100f || eps >= 0x1p-60f))) {
    t = 0.0;
    for (int k = threadIdx.x & 63; k < K; k += 64) {
      const double v = to_f<X>(x[k]);
      t = fma(v, v, t);
    }
    for (int o = 32; o; o >>= 1) t += __shfl_xor(t, o);
  }
  return t * per;
}

struct RowsArgs {
  const void* x; const float* gain; float eps;    // eps < 0: not normalised
  int R, K, Kp;
  int8_t* codes; float* scales;
  double per;                                     // 1 / K
};

// Codes of R rows: W waves per row, C chunks of 512 W values held in registers (C = 0:
// any K, read twice).  Bytes bound it: each value read once (the second read of C = 0
// comes from cache) and each code written once.  12,288 x 2048 in BF16: 15.4 us, 4.9 TB/s; 5,999 x 6144: 18.6 us,
// 6.0 TB/s; 32,816 x 1024 in FP32: 34 us, 4.9 TB/s.  A few hundred rows take 3 to 4 us, the time of a launch and
// of one load and one exchange after the other.
template <typename X, int W, int C, bool WHOLE, int MODE>
__global__ __launch_bounds__(256) void rows_kernel(RowsArgs a) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = blockIdx.x * (4 / W) + wave / W;
  static_assert(W == 1 || W == 4, "a row is a wave's or the workgroup's");
  if (W < 4 && row >= a.R) return;                // whole waves, and no barrier below
  const X* x = static_cast<const X*>(a.x) + (size_t)row * a.K;
  const int k0 = (wave % W * 64 + lane) * 8;
  constexpr int STEP = W * BLOCK, R = 4 / W;       // values per step, rows per workgroup
  __shared__ float blocks[R][C ? C * W : (1 << 17) / BLOCK];
  float* mine = blocks[wave / W];
  uint32_t top = 0;
  float t[C ? C : 1][8];
  auto take = [&](int k, float (&v)[8]) {
    float s = weigh8<WHOLE, MODE>(a.gain, k, a.K, v);
    top = top8(v, top);
    if constexpr (MODE != PLAIN) {
      s = wave_sum(s);
      if (lane == 0) mine[k / BLOCK] = s;
    }
  };
  if constexpr (C > 0) {
#pragma unroll
    for (int c = 0; c < C; ++c) load8<X, WHOLE>(x, k0 + c * STEP, a.K, t[c]);
#pragma unroll
    for (int c = 0; c < C; ++c) take(k0 + c * STEP, t[c]);
  } else {
    for (int k = k0; k - lane * 8 < a.K; k += STEP) {   // whole waves
      load8<X, WHOLE>(x, k, a.K, t[0]);
      take(k, t[0]);
    }
  }
  top = wave_max(top);
  if constexpr (W > 1) {
    __shared__ uint32_t tops[4];
    if (lane == 0) tops[wave] = top;
    __syncthreads();
    top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
  }
  const Coder coder(top);
  __builtin_amdgcn_wave_barrier();                // W = 1: the sums in `mine` are this wave's own
  if (wave % W == 0) {
    float s = coder.scale;
    if constexpr (MODE != PLAIN) s = coder.normed(mean_of(x, mine, a.K, a.per, a.eps) + (double)a.eps);
    if (lane == 0) a.scales[row] = s;
  }
  int8_t* q = a.codes + (size_t)row * a.Kp;
  if constexpr (C > 0) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int k = k0 + c * STEP;
      coder.scale8(t[c]);
      const uint2 v = coder.code8(t[c]);
      if (k < a.Kp) *reinterpret_cast<uint2*>(q + k) = v;
    }
  } else {
    for (int k = k0; k < a.Kp; k += STEP) {
      load8<X, WHOLE>(x, k, a.K, t[0]);
      weigh8<WHOLE, MODE>(a.gain, k, a.K, t[0]);
      coder.scale8(t[0]);
      *reinterpret_cast<uint2*>(q + k) = coder.code8(t[0]);
    }
  }
}

// ------------------------------------------------------------ products

struct LinearArgs {
  const int8_t* a; const float* as;               // codes [M][Kp] and scales of the activations' rows
  const int8_t* w; const float* ws;               // of the weights' [N] rows (SwiGLU: N gate rows, then N up rows)
  const float* bias;                              // [N] (SwiGLU: [2 N]) or null
  const void* res; void* out;                     // [M][N] of X; res may be null, or out itself
  int M, N, Kp;
  int mt, nt, gm;                                 // tiles along M and N, tiles along M per group
};

// g / (1 + e^-g) with the GPU's own powers of two and reciprocals (each within a step of the result).  For FP32 outputs
// t = -g log2(e) in two parts, 2^t_hi (1 + t_lo ln 2).  Below -87.3, where the reciprocal is denormal, it is 0 (silu is 1.03e-36 at
// most there; 1 / (1 + e^88.8) in FP32 is 0 as well).  For BF16 ones t alone: its rounding moves e^-g by
// |g| 2^-24, where the output's is 2^-8 (7,680 x 6144 outputs: 5 of 26 instructions each).
template <typename X>
__device__ __forceinline__ float silu(float g) {
  constexpr float L = 1.44269504088896341f, L2 = 1.92596299e-8f, LN2 = 0.693147181f;   // log2(e) = L + L2
  if constexpr (sizeof(X) == 2) return g * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-g * L));
  const float h = __builtin_amdgcn_fmed3f(g, -150.f, 150.f);   // past those e is 0 or infinite
  const float t = -h * L, lo = fmaf(-h, L2, fmaf(-h, L, -t));
  const float e = __builtin_amdgcn_exp2f(t) * fmaf(lo, LN2, 1.f);
  return g * __builtin_amdgcn_rcpf(1.f + e);
}
// A row's scale as two factors: what sums are multiplied by, and what columns' scales are.  Sums are below 2^31, so their
// products with 2^96 stay finite; what a larger scale (of values past 1e31) has beyond that, a power of two less, goes to the columns'.
struct RowScale {
  float s, t;
  __device__ __forceinline__ explicit RowScale(float x) : s(x > 0x1p96f ? 0x1p96f : x), t(x > 0x1p96f ? x * 0x1p-96f : 1.f) {}
};
// act of sums of row m (scale s) and column c (scale w, bias b; SwiGLU: and of its up column).
template <typename X, bool SWIGLU>
__device__ __forceinline__ float act_of(int acc, int up, RowScale s, float w, float w2, float b, float b2) {
  const float y = fmaf((float)acc * s.s, s.t * w, b);
  if constexpr (SWIGLU) return silu<X>(y) * fmaf((float)up * s.s, s.t * w2, b2);
  else return y;
}

// C (4 or 8) neighbouring outputs n .. n + C - 1 of row m before the residual.
template <typename X, int C>
__device__ __forceinline__ void emit(const LinearArgs& a, int m, int n, float (&y)[C]) {
  if (m >= a.M || n >= a.N) return;
  const size_t at = (size_t)m * a.N + n;
  X* o = static_cast<X*>(a.out) + at;
  const X* re = static_cast<const X*>(a.res) + at;
  if (a.N % C == 0) {                             // then n + C <= N, and rows are aligned for pieces of C
    if constexpr (sizeof(X) == 4) {
      if (a.res) {
#pragma unroll
        for (int i = 0; i < C / 4; ++i) {
          const float4 v = reinterpret_cast<const float4*>(re)[i];
          y[4 * i] += v.x; y[4 * i + 1] += v.y; y[4 * i + 2] += v.z; y[4 * i + 3] += v.w;
        }
      }
#pragma unroll
      for (int i = 0; i < C / 4; ++i)
        reinterpret_cast<float4*>(o)[i] = make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
    } else {
      typedef uint32_t Piece __attribute__((ext_vector_type(C / 2)));
      if (a.res) {
        const Piece v = *reinterpret_cast<const Piece*>(re);
#pragma unroll
        for (int i = 0; i < C / 2; ++i) {
          y[2 * i] += __uint_as_float(v[i] << 16);
          y[2 * i + 1] += __uint_as_float(v[i] & 0xffff0000u);
        }
      }
      Piece v;
#pragma unroll
      for (int i = 0; i < C / 2; ++i) v[i] = (uint32_t)from_f<X>(y[2 * i]) | (uint32_t)from_f<X>(y[2 * i + 1]) << 16;
      *reinterpret_cast<Piece*>(o) = v;
    }
  } else {
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (n + i < a.N) o[i] = from_f<X>(a.res ? y[i] + to_f<X>(re[i]) : y[i]);
  }
}

// Products of many rows, in tiles of BM x BN (SwiGLU: BN / 2 gate and the same BN / 2 up
// columns) by WM x WN waves.  A stage is 128 codes of every row of the tile, loaded straight
// to LDS: 8 lanes take a row's whole line, and the lane of slot c takes piece c ^ (row / 2 % 8),
// so that the rows of a matrix fragment lie in different banks.  S stages in a ring with one
// barrier each.  The matrix cores take the weights as their row operand, so a lane ends up
// with 4 neighbouring columns of one row.  Rows past M or N are clamped on load and not stored.
//
// The matrix cores alone reach 3.6 POP/s on random codes (4.9 on zeros: the clock follows the power).  7,680 rows of
// 2 x 6144 x 2048 (SwiGLU, BF16 out) take 201 us, 1.9 POP/s, 5,999 of 2048 x 6144 71 us with inputs in cache and 78 without, 2.1 and
// 1.9 POP/s: a tile's first stage, its epilogue (26 instructions per SwiGLU output) and its store have no products beside
// them, since LDS holds one 256 x 256 tile per CU.  Smaller tiles, two to a CU, overlap them, but load twice the
// bytes per product: 221 to 247 us in tiles of 128 x 128.
template <typename X, bool SWIGLU, int BM, int BN, int WM, int WN, int S>
__global__ __launch_bounds__(WM * WN * 64) void tiles_kernel(LinearArgs a) {
  constexpr int W = WM * WN, ROWS = BM + BN, LR = 8, PER = ROWS / LR / W;   // rows per load, loads per wave
  static_assert(ROWS % (LR * W) == 0 && BM % 16 == 0, "every wave loads alike");
  constexpr int TM = BM / WM / 32, TN = BN / WN / 32, RB = 128, STAGE = ROWS * RB;
  static_assert(!SWIGLU || TN % 2 == 0, "every wave holds gate and up of its columns");
  __shared__ __attribute__((aligned(1024))) char lds[S * STAGE];
  __shared__ __attribute__((aligned(16))) float row_s[BM], col_s[BN], col_b[BN];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i32 = lane & 31, hi = lane >> 5;

  // Tile of this workgroup: an XCD's workgroups (every eighth) take a run of tiles, in groups
  // of gm along M with M fastest, so that the tiles it works on at a time share panels in its L2.
  const int T = a.mt * a.nt, per = (T + 7) / 8;
  const int t = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per || t >= T) return;
  const int gsz = a.gm * a.nt, gi = t / gsz, gr = t - gi * gsz, gm = min(a.gm, a.mt - gi * a.gm);
  const int m0 = (gi * a.gm + gr % gm) * BM;
  constexpr int NC = SWIGLU ? BN / 2 : BN;
  const int n0 = gr / gm * NC;

  const int Kp = a.Kp, nst = Kp / RB;
  auto turn = [](int row) { return row >> 1 & 7; };
  const char* gb[PER];
  unsigned voff[PER];
#pragma unroll
  for (int c = 0; c < PER; ++c) {
    const int g = wave * PER + c;                 // rows LR g .. LR (g + 1) - 1 of the stage
    const char* base;
    int first, last;
    if (g < BM / LR) {
      base = reinterpret_cast<const char*>(a.a);
      first = m0 + g * LR;
      last = a.M - 1;
    } else {
      const int b = g * LR - BM;                 // row of the weights' part
      base = reinterpret_cast<const char*>(a.w);
      if (SWIGLU && b >= NC) base += (size_t)a.N * Kp;
      first = n0 + (SWIGLU && b >= NC ? b - NC : b);
      last = a.N - 1;
    }
    const int r0 = min(first, last);
    gb[c] = base + (size_t)r0 * Kp;
    const int lr = lane / 8, row = g * LR + lr;
    voff[c] = (unsigned)((min(first + lr, last) - r0) * Kp + ((lane & 7) ^ turn(row)) * 16);
  }
  auto issue = [&](int s, int c) {
    lds_load16(gb[c] + (size_t)s * RB, voff[c], lds + (s % S) * STAGE + (wave * PER + c) * 1024);
  };
  for (int i = tid; i < BM; i += W * 64) row_s[i] = a.as[min(m0 + i, a.M - 1)];
  for (int i = tid; i < BN; i += W * 64) {
    const int c = (SWIGLU && i >= NC ? a.N : 0) + min(n0 + (SWIGLU && i >= NC ? i - NC : i), a.N - 1);
    col_s[i] = a.ws[c];
    col_b[i] = a.bias ? a.bias[c] : 0.f;
  }
  const int wm = wave / WN, wn = wave % WN;
  // first row in the weights' part of column group j of this wave
  auto col = [&](int j) {
    if constexpr (SWIGLU) return j < TN / 2 ? (wn * (TN / 2) + j) * 32 : NC + (wn * (TN / 2) + j - TN / 2) * 32;
    else return (wn * TN + j) * 32;
  };
  v16i acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[i][j][v] = 0;
  // A stage's fragments come in four quarters of 32 codes, each a quarter ahead of its products, read
  // between the products of the one before.  While the last one's products run, the
  // stage's place in the ring is free for its next loads and the next stage's first quarter is on its way.
  v4i af[2][TM], bf[2][TN];
  auto piece = [&](int s, int q) { return lds + (s % S) * STAGE + i32 * RB + ((q * 2 + hi) ^ turn(i32)) * 16; };
  auto fetch = [&](const char* l, int set, int f) {   // fragment f of a quarter
    if (f < TN) bf[set][f] = *reinterpret_cast<const v4i*>(l + (BM + col(f)) * RB);
    else af[set][f - TN] = *reinterpret_cast<const v4i*>(l + (wm * TM + f - TN) * 32 * RB);
  };
  // Loads are spread over the products too: a wave that issues all of a stage's at once stands in line for
  // the memory pipe, and its matrix core idles.
  constexpr int P = TM * TN, L0 = (PER + 1) / 2;  // products of a quarter; loads in the stage's last quarter, the others in the next one's first
  auto multiply = [&](int set, const char* l, int load, int c0, int c1) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int i = p / TN, j = p % TN;
      acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(bf[set][j], af[set][i], acc[i][j], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int f = 0; f < TM + TN; ++f)
        if (f * P / (TM + TN) == p) fetch(l, set ^ 1, f);
      if (load >= 0) {
#pragma unroll
        for (int c = c0; c < c1; ++c)
          if ((2 * (c - c0) + 1) * P / (2 * (c1 - c0)) == p) issue(load, c);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // stages in flight behind the one that is waited for: at most S - 1 (first wait), then S - 2
  auto arrive = [&](int behind) {
    if (S > 3 && behind >= 3) stage_sync<(S > 3 ? 3 : 0) * PER>();
    else if (S > 2 && behind >= 2) stage_sync<(S > 2 ? 2 : 0) * PER>();
    else if (behind >= 1) stage_sync<PER>();
    else stage_sync<0>();
  };
  static_assert(S >= 2 && S <= 4, "arrive() counts up to three stages");
#pragma unroll
  for (int s = 0; s < S; ++s)
    if (s < nst) {
#pragma unroll
      for (int c = 0; c < PER; ++c) issue(s, c);
    }
  arrive(min(S, nst) - 1);
#pragma unroll
  for (int f = 0; f < TM + TN; ++f) fetch(piece(0, 0), 0, f);
  constexpr int Q = 4;                            // quarters of a stage
  for (int s = 0; s < nst; ++s) {
    // stage s - 1 + S goes on into the place of stage s - 1
    multiply(0, piece(s, 1), s && s - 1 + S < nst ? s - 1 + S : -1, L0, PER);
#pragma unroll
    for (int q = 1; q < Q - 1; ++q) multiply(q & 1, piece(s, q + 1), -1, 0, 0);
    if (s + 1 < nst) arrive(min(S - 2, nst - 2 - s));
    multiply(1, piece(s + 1, 0), s + S < nst ? s + S : -1, 0, L0);   // past the last stage: read and not used
  }
  // Lane: row m = lane % 32 of each 32 x 32 tile, columns 8 g + 4 (lane / 32) .. + 3 for g in 0 .. 3.  Through the
  // wave's own part of LDS, so that stores are of whole pieces of rows: as they lie they are
  // 8 or 16 bytes of 32 rows each (8192 x 8192 outputs in BF16: 75 us).
  constexpr int TO = SWIGLU ? TN / 2 : TN;        // tiles out
  constexpr int CJ = TO % 2 == 0 && W * 32 * 68 * 4 <= S * STAGE ? 2 : 1, CW = CJ * 32, LD = CW + 4;   // of them, and columns, at a time
  static_assert(W * 32 * LD * 4 <= S * STAGE, "the waves' parts lie in the ring");
  float* part = reinterpret_cast<float*>(lds) + wave * 32 * LD;
  __syncthreads();                                // the ring is read
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int r0 = (wm * TM + i) * 32;
    const RowScale sc(row_s[r0 + i32]);
#pragma unroll
    for (int j0 = 0; j0 < TO; j0 += CJ) {
#pragma unroll
      for (int j = j0; j < j0 + CJ; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int c = col(j) + g * 8 + hi * 4;
          const float4 w = *reinterpret_cast<const float4*>(col_s + c), b = *reinterpret_cast<const float4*>(col_b + c);
          float4 w2 = w, b2 = b;
          if constexpr (SWIGLU) {
            w2 = *reinterpret_cast<const float4*>(col_s + NC + c);
            b2 = *reinterpret_cast<const float4*>(col_b + NC + c);
          }
          const v16i &y = acc[i][j], &u = acc[i][SWIGLU ? j + TN / 2 : j];
          float4 o;
          o.x = act_of<X, SWIGLU>(y[4 * g], u[4 * g], sc, w.x, w2.x, b.x, b2.x);
          o.y = act_of<X, SWIGLU>(y[4 * g + 1], u[4 * g + 1], sc, w.y, w2.y, b.y, b2.y);
          o.z = act_of<X, SWIGLU>(y[4 * g + 2], u[4 * g + 2], sc, w.z, w2.z, b.z, b2.z);
          o.w = act_of<X, SWIGLU>(y[4 * g + 3], u[4 * g + 3], sc, w.w, w2.w, b.w, b2.w);
          *reinterpret_cast<float4*>(part + i32 * LD + (j - j0) * 32 + g * 8 + hi * 4) = o;
        }
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int e = 0; e < 32 * CW / 8 / 64; ++e) {
        const int r = (e * 64 + lane) / (CW / 8), c = (e * 64 + lane) % (CW / 8) * 8;
        const float4 lo = *reinterpret_cast<const float4*>(part + r * LD + c), up = *reinterpret_cast<const float4*>(part + r * LD + c + 4);
        float o[8] = {lo.x, lo.y, lo.z, lo.w, up.x, up.y, up.z, up.w};
        emit<X, 8>(a, m0 + r0 + r, n0 + col(j0) + c, o);
      }
      __builtin_amdgcn_wave_barrier();
    }
  }
}

// This wave's loads into LDS but the last N are in.
template <int N>
__device__ __forceinline__ void loads_but() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// Products of few rows: a workgroup has NT tiles of 16 weight rows (SwiGLU: half of them gate,
// half the same rows of up) and MT tiles of 16 activation rows, and its W waves take every W-th
// unit of 128 codes; their sums meet in LDS.  The weights' bytes bound it.  They go to LDS in whole lines,
// 8 lanes to a row, into a ring of D units that is the wave's own, so that no wave waits for another, and
// from there to registers as matrix fragments (a load in the order of a fragment's lanes, 16 rows next to each other,
// takes 3.5 times as long: 2048 x 6144, 128 workgroups, 4.5 us against 2.7 with the launch).  With two sets of inputs in turn 32 rows
// of 2 x 6144 x 2048 take 8.5 us, 3.0 TB/s of weights (7.2 in cache, 13.4 from memory; LDS holds one workgroup per CU, of 384), 32 rows
// of 2048 x 6144 5.0, 2 rows of 4096 x 2048 with their codes 5.4, 1 row of 2051 x 1024 4.6: the launch, the latency of a ring's first units and the sum over the waves, in turn.
//
// FUSED (up to 8 rows, a power of two times K at most 16,384): the workgroup codes the
// activations' rows itself, each into its own LDS, which saves the launch that writes them;
// the weights' first units are on their way meanwhile.
template <typename X, bool SWIGLU, bool FUSED, bool WHOLE, int MT, int NT, int W, int D>
__global__ __launch_bounds__(W * 64) void few_kernel(LinearArgs a, RowsArgs r) {
  static_assert(!SWIGLU || NT % 2 == 0, "gate and up of the same columns");
  static_assert(!FUSED || (MT == 1 && W == 8), "8 waves code up to 8 rows");
  constexpr int NC = (SWIGLU ? NT / 2 : NT) * 16, AT = FUSED ? 0 : MT, T = NT + AT;   // tiles that a unit loads
  constexpr int RING = W * D * T * 2048, VECS = MT * NT * 64;   // of four sums: [MT][NT][lane]
  static_assert(RING >= W * VECS * 16, "the waves' sums lie in the ring");
  __shared__ __attribute__((aligned(1024))) char ring[RING];
  __shared__ __attribute__((aligned(16))) char own[FUSED ? 8 * (2048 + 16) : 16];   // codes of rows, Kp + 16 apart
  __shared__ float row_scale[8];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i16 = lane & 15, q4 = lane >> 4;
  const int n0 = blockIdx.x * NC, m0 = blockIdx.y * (MT * 16);
  const int Kp = a.Kp, units = Kp / 128;
  const int mine = units > wave ? (units - wave + W - 1) / W : 0;

  // tile t, half h: 8 rows; the lane of slot c takes piece c ^ (row / 2 % 8) of its row, so that the 16 rows of a
  // fragment lie in different banks
  const char* gb[T];
  unsigned voff[T][2];
#pragma unroll
  for (int t = 0; t < T; ++t) {
    const bool act = t >= NT, is_up = SWIGLU && !act && t >= NT / 2;
    const int first = act ? m0 + (t - NT) * 16 : n0 + (is_up ? t - NT / 2 : t) * 16, last = act ? a.M - 1 : a.N - 1;
    const int r0 = min(first, last);
    gb[t] = reinterpret_cast<const char*>(act ? a.a : a.w) + ((size_t)(is_up ? a.N : 0) + r0) * Kp + wave * 128;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = h * 8 + (lane >> 3);
      voff[t][h] = (unsigned)((min(first + row, last) - r0) * Kp + ((lane & 7) ^ (row >> 1)) * 16);
    }
  }
  char* mine_at = ring + wave * (D * T * 2048);
  auto issue = [&](int d, int i) {
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h) lds_load16(gb[t] + (size_t)i * (W * 128), voff[t][h], mine_at + (d * T + t) * 2048 + h * 1024);
  };
#pragma unroll
  for (int d = 0; d < D; ++d)
    if (d < mine) issue(d, d);

  const int8_t* ap = nullptr;
  if constexpr (FUSED) {
    constexpr int C = 4;
    __shared__ uint32_t tops[8];
    __shared__ float blocks[8 * C];               // of a row: its waves' C
    const int rows2 = a.M > 4 ? 8 : a.M > 2 ? 4 : a.M;   // rows up to a power of two
    const int wpr = 8 / rows2, row = wave / wpr, step = wpr * BLOCK;
    const bool norm = r.eps >= 0.f;
    const float* gain = norm ? r.gain : nullptr;
    const int k0 = (wave % wpr * 64 + lane) * 8;
    float t[C][8];
    uint32_t top = 0;
    if (row < a.M) {
      const X* x = static_cast<const X*>(r.x) + (size_t)row * r.K;
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (c * step < r.K) load8<X, WHOLE>(x, k0 + c * step, r.K, t[c]);
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (c * step < r.K) {
          const int k = k0 + c * step;
          float s = norm ? weigh8<WHOLE, NORM>(nullptr, k, r.K, t[c]) : 0.f;
          if (gain) weigh8<WHOLE, GAIN>(gain, k, r.K, t[c]);
          top = top8(t[c], top);
          if (norm) {
            s = wave_sum(s);
            if (lane == 0) blocks[row * wpr * C + c * wpr + wave % wpr] = s;
          }
        }
    }
    top = wave_max(top);
    if (lane == 0) tops[wave] = top;
    __syncthreads();
    if (row < a.M) {
      for (int w = row * wpr; w < (row + 1) * wpr; ++w) top = max(top, tops[w]);
      const Coder coder(top);
      if (wave % wpr == 0) {
        float s = coder.scale;
        if (norm) s = coder.normed(mean_of(static_cast<const X*>(r.x) + (size_t)row * r.K, blocks + row * wpr * C, r.K, r.per, r.eps) + (double)r.eps);
        if (lane == 0) row_scale[row] = s;
      }
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int k = k0 + c * step;
        if (c * step < Kp) {
          coder.scale8(t[c]);
          const uint2 v = coder.code8(t[c]);
          if (k < Kp) *reinterpret_cast<uint2*>(own + (size_t)row * (Kp + 16) + k) = v;
        }
      }
    }
    __syncthreads();
    ap = reinterpret_cast<const int8_t*>(own) + min(i16, a.M - 1) * (Kp + 16) + wave * 128 + q4 * 16;
  }

  v4i acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = v4i{0, 0, 0, 0};
  constexpr int L = 2 * T;                        // loads of a unit
  static_assert((D == 2 || D == 3) && 2 * L < 64, "the waits below, and their counter");
  for (int i0 = 0; i0 < mine; i0 += D) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int i = i0 + d, behind = min(D - 1, mine - 1 - i);
      if (behind < 0) break;
      if (D > 2 && behind == 2) loads_but<(D > 2 ? 2 : 0) * L>();
      else if (behind == 1) loads_but<L>();
      else loads_but<0>();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const char* l = mine_at + d * T * 2048 + i16 * 128 + ((h * 4 + q4) ^ (i16 >> 1)) * 16;
        v4i bf[NT], af[MT];
#pragma unroll
        for (int j = 0; j < NT; ++j) bf[j] = *reinterpret_cast<const v4i*>(l + j * 2048);
#pragma unroll
        for (int m = 0; m < MT; ++m)
          af[m] = FUSED ? *reinterpret_cast<const v4i*>(ap + (size_t)i * (W * 128) + h * 64) : *reinterpret_cast<const v4i*>(l + (NT + m) * 2048);
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int m = 0; m < MT; ++m) acc[m][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bf[j], af[m], acc[m][j], 0, 0, 0);
      }
      if (i + D < mine) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the unit's place is read
        issue(d, i + D);
      }
    }
  }

  v4i* sum = reinterpret_cast<v4i*>(ring);
  __syncthreads();                                // the rings are read
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) sum[wave * VECS + (i * NT + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  auto add_waves = [&](int e) {
    v4i s = sum[e];
#pragma unroll
    for (int w = 1; w < W; ++w) s += sum[w * VECS + e];
    return s;
  };
  if constexpr (FUSED) a.as = row_scale;
  constexpr int OT = SWIGLU ? NT / 2 : NT;        // output tiles
  for (int e = tid; e < MT * OT * 64; e += W * 64) {
    const int l = e & 63, j = e / 64 % OT, i = e / 64 / OT;
    const v4i y = add_waves((i * NT + j) * 64 + l);
    const v4i up = SWIGLU ? add_waves((i * NT + j + NT / 2) * 64 + l) : y;
    const int m = m0 + i * 16 + (l & 15), n = n0 + j * 16 + (l >> 4) * 4;
    float out[4];
    const RowScale sc(a.as[min(m, a.M - 1)]);
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int c = min(n + v, a.N - 1);
      out[v] = act_of<X, SWIGLU>(y[v], up[v], sc, a.ws[c], SWIGLU ? a.ws[a.N + c] : 0.f, a.bias ? a.bias[c] : 0.f,
                                 SWIGLU && a.bias ? a.bias[a.N + c] : 0.f);
    }
    emit<X, 4>(a, m, n, out);
  }
}

}  // namespace int8
}  // namespace sk
