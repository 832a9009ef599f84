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
// change none.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "sk_lds.h"

// Each operation rounds by itself (fused ones are written as such): all kernels give the same bits.
#pragma clang fp contract(off)

namespace sk {
namespace int8 {

typedef int v4i __attribute__((ext_vector_type(4)));

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

// 8 neighbouring values of a row from k on, 0 past K.  `whole`: K is a multiple
// of 8 and rows are 16-byte aligned.
template <typename X>
__device__ __forceinline__ void load8(const X* row, int k, int K, bool whole, float (&t)[8]) {
  if (whole) {
    if (k >= K) {
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = 0.f;
    } else if constexpr (sizeof(X) == 2) {
      const uint4 v = *reinterpret_cast<const uint4*>(row + k);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        t[2 * i] = __uint_as_float(w[i] << 16);
        t[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    } else {
      const float4 a = *reinterpret_cast<const float4*>(row + k), b = *reinterpret_cast<const float4*>(row + k + 4);
      t[0] = a.x; t[1] = a.y; t[2] = a.z; t[3] = a.w;
      t[4] = b.x; t[5] = b.y; t[6] = b.z; t[7] = b.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = k + i < K ? to_f<X>(row[k + i]) : 0.f;
  }
}
// x^2 of 8 values, and t times the gain (rounded to FP32: the definition's one rounding).
__device__ __forceinline__ float weigh8(const float* gain, int k, int K, bool whole, float (&t)[8]) {
  float squares = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) squares = fmaf(t[i], t[i], squares);
  if (!gain) return squares;
  float g[8];
  load8<float>(gain, k, K, whole, g);
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] *= g[i];
  return squares;
}
// The largest |t| as bits: NaN above infinity above every number.
__device__ __forceinline__ uint32_t top8(const float (&t)[8], uint32_t top) {
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(t[i]) & 0x7fffffffu);
  return top;
}

// How a row with this largest |t| is coded.  Rows of less than 2^-60 are
// multiplied by 2^80 first (exact), so that 127 / top is a number.
struct Coder {
  float r, up, top;                               // 127 / (top up), up, top up
  float scale;                                    // top / 127
  __device__ explicit Coder(uint32_t bits) {
    const float t = __uint_as_float(bits);
    const bool bad = bits >= 0x7f800000u;
    up = t < 0x1p-60f ? 0x1p80f : 1.f;
    top = t * up;
    r = bad || bits == 0 ? 0.f : 127.f / top;
    scale = bad ? __uint_as_float(0x7fc00000u) : t / 127.f;
    if (bad) up = 0.f;                            // its values: 0 times r is no code either way
  }
  // The nearest whole number of 127 t / top.  The rounded product is off by at most
  // 127 * 2^-23 = 1.5e-5; within 1e-4 of a middle l + 1/2, 254 t and (2 l + 1) top (at most 33
  // bits each) are compared in 64 bits, exactly.
  __device__ __forceinline__ int code(float t) const {
    const float f = t * up * r, q = rintf(f), d = f - q;
    int c = (int)q;
    if (fabsf(d) > 0.4999f) {
      const int l = d > 0.f ? c : c - 1;
      const double a = 254.0 * (double)(t * up), b = (2.0 * l + 1.0) * (double)top;
      c = a > b ? l + 1 : a < b ? l : l + (l & 1);
    }
    return c;
  }
  // 8 codes; of a row that has none (r = 0: zeros, infinities, NaN) zeros.
  __device__ __forceinline__ uint2 code8(const float (&t)[8]) const {
    uint32_t w[2] = {0, 0};
    if (r != 0.f) {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i / 4] |= (uint32_t)(code(t[i]) & 0xff) << (8 * (i % 4));
    }
    return make_uint2(w[0], w[1]);
  }
};

// Over a wave, in every lane.
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o));
  return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// Sums of squares have one order whatever holds the row, so that a row's norm does not
// hang on the size of the call: 8 values one after the other, the 64 such sums of a block of 512 by
// wave_sum, the blocks one after the other.
constexpr int BLOCK = 512;
__device__ __forceinline__ float norm_of(const float* blocks, int K, float eps) {
  float s = 0.f;
  for (int b = 0; b * BLOCK < K; ++b) s += blocks[b];
  return 1.f / sqrtf(s / (float)K + eps);
}

struct RowsArgs {
  const void* x; const float* gain; float eps;    // eps < 0: not normalised
  int R, K, Kp;
  int8_t* codes; float* scales;
  int* zero; int n_zero;                          // words that the launch also sets to 0 (tickets of the product)
};

// Codes of R rows: W waves per row, C chunks of 512 W values held in registers (C = 0:
// any K, read twice).  Bytes bound it: each value read once (the second read of C = 0
// comes from cache) and each code written once.
template <typename X, int W, int C>
__global__ __launch_bounds__(256) void rows_kernel(RowsArgs a) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (blockIdx.x == 0)
    for (int i = tid; i < a.n_zero; i += 256) a.zero[i] = 0;
  const int row = blockIdx.x * (4 / W) + wave / W;
  if (W < 4 && row >= a.R) return;                // whole waves, and no barrier below for W = 1
  const bool whole = a.K % 8 == 0;
  const X* x = static_cast<const X*>(a.x) + (size_t)row * a.K;
  const int k0 = (wave % W * 64 + lane) * 8;
  const float* gain = a.eps >= 0.f ? a.gain : nullptr;
  constexpr int STEP = W * BLOCK, R = 4 / W;       // values per step, rows per workgroup
  __shared__ float blocks[R][C ? C * W : (1 << 17) / BLOCK];
  float* mine = blocks[wave / W];
  const bool norm = a.eps >= 0.f;
  uint32_t top = 0;
  float t[C ? C : 1][8];
  auto take = [&](int k, float (&v)[8]) {
    float s = weigh8(gain, k, a.K, whole, v);
    top = top8(v, top);
    if (norm) {
      s = wave_sum(s);
      if (lane == 0) mine[k / BLOCK] = s;
    }
  };
  if constexpr (C > 0) {
#pragma unroll
    for (int c = 0; c < C; ++c) load8<X>(x, k0 + c * STEP, a.K, whole, t[c]);
#pragma unroll
    for (int c = 0; c < C; ++c) take(k0 + c * STEP, t[c]);
  } else {
    for (int k = k0; k - lane * 8 < a.K; k += STEP) {   // whole waves
      load8<X>(x, k, a.K, whole, t[0]);
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
  if (wave % W == 0 && lane == 0) a.scales[row] = norm ? coder.scale * norm_of(mine, a.K, a.eps) : coder.scale;
  int8_t* q = a.codes + (size_t)row * a.Kp;
  if constexpr (C > 0) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int k = k0 + c * STEP;
      if (k < a.Kp) *reinterpret_cast<uint2*>(q + k) = coder.code8(t[c]);
    }
  } else {
    for (int k = k0; k < a.Kp; k += STEP) {
      load8<X>(x, k, a.K, whole, t[0]);
      weigh8(gain, k, a.K, whole, t[0]);
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
  int mt, nt, ksplit, gm;                         // tiles along M and N, cuts of K; tiles along M per group
  int* part; int* ticket;                         // ksplit > 1: sums of the cuts, arrivals per tile
};

__device__ __forceinline__ float silu(float g) { return g / (1.f + expf(-g)); }

// Four neighbouring outputs n .. n + 3 of row m from their sums.
template <typename X, bool SWIGLU>
__device__ __forceinline__ void finish4(const LinearArgs& a, int m, int n, v4i acc, v4i up) {
  if (m >= a.M || n >= a.N) return;
  const float s = a.as[m];
  const size_t at = (size_t)m * a.N + n;
  const bool four = (a.N & 3) == 0;               // then rows are 16-byte (BF16 8-byte) aligned, and n + 3 < N
  float y[4], r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = min(n + i, a.N - 1);
    y[i] = (float)acc[i] * s * a.ws[c];
    if (a.bias) y[i] += a.bias[c];
    if constexpr (SWIGLU) {
      float u = (float)up[i] * s * a.ws[a.N + c];
      if (a.bias) u += a.bias[a.N + c];
      y[i] = silu(y[i]) * u;
    }
  }
  X* o = static_cast<X*>(a.out) + at;
  const X* re = static_cast<const X*>(a.res) + at;
  if (four) {
    if constexpr (sizeof(X) == 4) {
      if (a.res) {
        const float4 v = *reinterpret_cast<const float4*>(re);
        y[0] += v.x; y[1] += v.y; y[2] += v.z; y[3] += v.w;
      }
      *reinterpret_cast<float4*>(o) = make_float4(y[0], y[1], y[2], y[3]);
    } else {
      if (a.res) {
        const uint2 v = *reinterpret_cast<const uint2*>(re);
        r[0] = __uint_as_float(v.x << 16); r[1] = __uint_as_float(v.x & 0xffff0000u);
        r[2] = __uint_as_float(v.y << 16); r[3] = __uint_as_float(v.y & 0xffff0000u);
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] += r[i];
      }
      *reinterpret_cast<uint2*>(o) = make_uint2((uint32_t)from_f<X>(y[0]) | (uint32_t)from_f<X>(y[1]) << 16,
                                                (uint32_t)from_f<X>(y[2]) | (uint32_t)from_f<X>(y[3]) << 16);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < a.N) o[i] = from_f<X>(a.res ? y[i] + to_f<X>(re[i]) : y[i]);
  }
}

// Products of many rows, in tiles of BM x BN (SwiGLU: BN / 2 gate and the same BN / 2 up
// columns) by WM x WN waves.  A stage is 128 codes of every row of the tile, loaded straight
// to LDS: 8 lanes take a row's whole line, and the lane of slot c takes piece c ^ (row % 8),
// so that the 16 rows of a matrix fragment lie in different banks.  S stages in a ring with one
// barrier each.  The matrix cores take the weights as their row operand, so a lane ends up
// with 4 neighbouring columns of one row.  Rows past M or N are clamped on load and not stored.
template <typename X, bool SWIGLU, int BM, int BN, int WM, int WN, int S>
__global__ __launch_bounds__(WM * WN * 64) void tiles_kernel(LinearArgs a) {
  constexpr int W = WM * WN, ROWS = BM + BN, PER = ROWS / 8 / W;   // loads of 8 rows, of them per wave
  static_assert(ROWS % (8 * W) == 0, "every wave loads alike");
  constexpr int TM = BM / WM / 16, TN = BN / WN / 16, STAGE = ROWS * 128;
  static_assert(!SWIGLU || TN % 2 == 0, "every wave holds gate and up of its columns");
  __shared__ __attribute__((aligned(1024))) char lds[S * STAGE];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i16 = lane & 15, q4 = lane >> 4;

  // Tile of this workgroup: an XCD's workgroups (every eighth) take a run of tiles, in groups
  // of gm along M with M fastest, so that the tiles it works on at a time share panels in its L2.
  const int T = a.mt * a.nt, per = (T + 7) / 8;
  const int t = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per || t >= T) return;
  const int gsz = a.gm * a.nt, gi = t / gsz, gr = t - gi * gsz, gm = min(a.gm, a.mt - gi * a.gm);
  const int m0 = (gi * a.gm + gr % gm) * BM;
  constexpr int NC = SWIGLU ? BN / 2 : BN;
  const int n0 = gr / gm * NC;

  const int Kp = a.Kp, nst = Kp / 128;
  const char* gb[PER];
  unsigned voff[PER];
#pragma unroll
  for (int c = 0; c < PER; ++c) {
    const int g = wave * PER + c;                 // rows 8 g .. 8 g + 7 of the stage
    const char* base;
    int first, last;
    if (g < BM / 8) {
      base = reinterpret_cast<const char*>(a.a);
      first = m0 + g * 8;
      last = a.M - 1;
    } else {
      const int b = g * 8 - BM;                   // row of the weights' part
      base = reinterpret_cast<const char*>(a.w);
      if (SWIGLU && b >= NC) base += (size_t)a.N * Kp;
      first = n0 + (SWIGLU && b >= NC ? b - NC : b);
      last = a.N - 1;
    }
    const int r0 = min(first, last);
    gb[c] = base + (size_t)r0 * Kp;
    voff[c] = (unsigned)((min(first + (lane >> 3), last) - r0) * Kp + (((lane & 7) ^ (lane >> 3)) * 16));
  }
  auto issue = [&](int s) {
    const char* l = lds + (s % S) * STAGE + wave * PER * 1024;
#pragma unroll
    for (int c = 0; c < PER; ++c) lds_load16(gb[c] + (size_t)s * 128, voff[c], l + c * 1024);
  };
  const int wm = wave / WN, wn = wave % WN;
  // first row in the weights' part of column group j of this wave
  auto col = [&](int j) {
    if constexpr (SWIGLU) return j < TN / 2 ? (wn * (TN / 2) + j) * 16 : NC + (wn * (TN / 2) + j - TN / 2) * 16;
    else return (wn * TN + j) * 16;
  };
  v4i acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = v4i{0, 0, 0, 0};
#pragma unroll
  for (int s = 0; s < S - 1; ++s)
    if (s < nst) issue(s);
  for (int s = 0; s < nst; ++s) {
    const int ahead = nst - 1 - s;
    if (ahead >= S - 2) stage_sync<PER * (S - 2)>();
    else if (S > 3 && ahead == 1) stage_sync<(S > 3 ? PER : 0)>();
    else stage_sync<0>();
    if (s + S - 1 < nst) issue(s + S - 1);
    const char* l = lds + (s % S) * STAGE + i16 * 128;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const char* lk = l + (((kb * 4 + q4) ^ (i16 & 7)) * 16);
      v4i af[TM], bf[TN];
#pragma unroll
      for (int i = 0; i < TM; ++i) af[i] = *reinterpret_cast<const v4i*>(lk + (wm * TM + i) * 2048);
#pragma unroll
      for (int j = 0; j < TN; ++j) bf[j] = *reinterpret_cast<const v4i*>(lk + (BM + col(j)) * 128);
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int i = 0; i < TM; ++i) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bf[j], af[i], acc[i][j], 0, 0, 0);
    }
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int m = m0 + (wm * TM + i) * 16 + i16;
#pragma unroll
    for (int j = 0; j < (SWIGLU ? TN / 2 : TN); ++j)
      finish4<X, SWIGLU>(a, m, n0 + col(j) + q4 * 4, acc[i][j], acc[i][SWIGLU ? j + TN / 2 : j]);
  }
}

// Products of few rows: a workgroup has NT tiles of 16 weight rows (SwiGLU: half of them gate,
// half the same rows of up) and MT tiles of 16 activation rows, and its W waves take every W-th
// unit of 128 codes; their sums meet in LDS.  The weights' bytes bound it: they go
// straight to registers as matrix fragments, D units ahead, and are read once for all
// rows.  K may be cut over ksplit workgroups; the last one to arrive adds the cuts up.
//
// FUSED (up to 8 rows, a power of two times K at most 16,384): the workgroup codes the
// activations' rows itself, each into its own LDS, which saves the launch that writes them;
// the weights' first units are on their way meanwhile.
template <typename X, bool SWIGLU, bool FUSED, int MT, int NT, int W>
__global__ __launch_bounds__(W * 64) void few_kernel(LinearArgs a, RowsArgs r) {
  static_assert(!SWIGLU || NT % 2 == 0, "gate and up of the same columns");
  static_assert(!FUSED || (MT == 1 && W == 8), "8 waves code up to 8 rows");
  constexpr int D = 2, NC = (SWIGLU ? NT / 2 : NT) * 16;
  extern __shared__ __attribute__((aligned(16))) char dyn[];   // FUSED: codes, rows Kp + 16 apart; then the waves' sums
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i16 = lane & 15, q4 = lane >> 4;
  const int tile = blockIdx.x / a.ksplit, ks = blockIdx.x - tile * a.ksplit;
  const int n0 = tile * NC, m0 = blockIdx.y * (MT * 16);
  const int Kp = a.Kp, units = Kp / 128;
  const int u0 = (int)((int64_t)units * ks / a.ksplit), nu = (int)((int64_t)units * (ks + 1) / a.ksplit) - u0;
  const int mine = nu > wave ? (nu - wave + W - 1) / W : 0;

  const int8_t* wp[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const bool is_up = SWIGLU && j >= NT / 2;
    const int n = min(n0 + (is_up ? j - NT / 2 : j) * 16 + i16, a.N - 1);
    wp[j] = a.w + ((size_t)(is_up ? a.N : 0) + n) * Kp + (size_t)(u0 + wave) * 128 + q4 * 16;
  }
  v4i b[D][NT][2];
  auto load_w = [&](int d, int i) {
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) b[d][j][h] = *reinterpret_cast<const v4i*>(wp[j] + (size_t)i * (W * 128) + h * 64);
  };
#pragma unroll
  for (int d = 0; d < D; ++d)
    if (d < mine) load_w(d, d);

  const int8_t* ap[MT];
  v4i af[D][MT][2];
  auto load_a = [&](int d, int i) {
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) af[d][j][h] = *reinterpret_cast<const v4i*>(ap[j] + (size_t)i * (W * 128) + h * 64);
  };
  __shared__ float row_scale[8];
  if constexpr (FUSED) {
    constexpr int C = 4;
    __shared__ uint32_t tops[8];
    __shared__ float blocks[8 * C];               // of a row: its waves' C
    const int rows2 = a.M > 4 ? 8 : a.M > 2 ? 4 : a.M;   // rows up to a power of two
    const int wpr = 8 / rows2, row = wave / wpr, step = wpr * BLOCK;
    const bool whole = r.K % 8 == 0, norm = r.eps >= 0.f;
    const float* gain = norm ? r.gain : nullptr;
    const int k0 = (wave % wpr * 64 + lane) * 8;
    float t[C][8];
    uint32_t top = 0;
    if (row < a.M) {
      const X* x = static_cast<const X*>(r.x) + (size_t)row * r.K;
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (c * step < r.K) load8<X>(x, k0 + c * step, r.K, whole, t[c]);
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (c * step < r.K) {
          float s = weigh8(gain, k0 + c * step, r.K, whole, t[c]);
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
      if (wave % wpr == 0 && lane == 0)
        row_scale[row] = norm ? coder.scale * norm_of(blocks + row * wpr * C, r.K, r.eps) : coder.scale;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int k = k0 + c * step;
        if (k < Kp) *reinterpret_cast<uint2*>(dyn + (size_t)row * (Kp + 16) + k) = coder.code8(t[c]);
      }
    }
    __syncthreads();
    ap[0] = reinterpret_cast<const int8_t*>(dyn) + min(i16, a.M - 1) * (Kp + 16) + wave * 128 + q4 * 16;
  } else {
#pragma unroll
    for (int j = 0; j < MT; ++j)
      ap[j] = a.a + (size_t)min(m0 + j * 16 + i16, a.M - 1) * Kp + (size_t)(u0 + wave) * 128 + q4 * 16;
#pragma unroll
    for (int d = 0; d < D; ++d)
      if (d < mine) load_a(d, d);
  }

  v4i acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = v4i{0, 0, 0, 0};
  for (int i0 = 0; i0 < mine; i0 += D) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      if (i0 + d >= mine) break;
      if constexpr (FUSED) load_a(d, i0 + d);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int i = 0; i < MT; ++i)
            acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(b[d][j][h], af[d][i][h], acc[i][j], 0, 0, 0);
      if (i0 + d + D < mine) {
        load_w(d, i0 + d + D);
        if constexpr (!FUSED) load_a(d, i0 + d + D);
      }
    }
  }

  constexpr int VECS = MT * NT * 64;              // of four sums: [MT][NT][lane]
  v4i* sum = reinterpret_cast<v4i*>(dyn);
  if constexpr (FUSED) __syncthreads();           // the codes are read
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
  const bool cut = !FUSED && a.ksplit > 1;
  const size_t all = (size_t)blockIdx.y * (gridDim.x / a.ksplit) + tile;
  v4i* part = reinterpret_cast<v4i*>(a.part) + all * a.ksplit * VECS;
  if (cut) {
    for (int e = tid; e < VECS; e += W * 64) part[(size_t)ks * VECS + e] = add_waves(e);
    __threadfence();
    __shared__ int arrived;
    __syncthreads();
    if (tid == 0) arrived = __hip_atomic_fetch_add(a.ticket + all, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (arrived != a.ksplit - 1) return;
    __threadfence();
  }
  auto total = [&](int e) {
    if (!cut) return add_waves(e);
    v4i s = part[e];
    for (int c = 1; c < a.ksplit; ++c) s += part[(size_t)c * VECS + e];
    return s;
  };
  if constexpr (FUSED) a.as = row_scale;
  constexpr int OT = SWIGLU ? NT / 2 : NT;        // output tiles
  for (int e = tid; e < MT * OT * 64; e += W * 64) {
    const int l = e & 63, j = e / 64 % OT, i = e / 64 / OT;
    const v4i y = total((i * NT + j) * 64 + l);
    const v4i up = SWIGLU ? total((i * NT + j + NT / 2) * 64 + l) : y;
    finish4<X, SWIGLU>(a, m0 + i * 16 + (l & 15), n0 + j * 16 + (l >> 4) * 4, y, up);
  }
}

}  // namespace int8
}  // namespace sk
