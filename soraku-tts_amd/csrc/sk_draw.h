// Sampling of many rows at once, every row with parameters of its own.
//
// A row's candidates are its finite and allowed values x (x = u + c (cond - u) with
// guidance), y = x / T in FP32, held to the finite range.  In the order of y, ties by the lower id
// first, the kept ones are always the first so many: top-k keeps those down to the k-th's
// value, top-p those up to and with the first whose sum of weights passes p times the
// whole, min-p those with a weight of at least that part of the first's.  The draw is the first kept one
// whose sum passes u times the sum of the kept.  So nothing needs the whole order, only the places
// where counts or sums of the largest values pass a bound:
//
// * a histogram of y (64 buckets per power of two of the weight) with counts and sums
//   tells the few buckets in which the bounds are passed;
// * their values alone are listed and sorted, and the bounds are found in the list by
//   bisection;
// * where those buckets hold more values than the list (thousands of equal logits), the bounds are
//   found digit by digit of the value, three passes over the row for each.
//
// Weights are 2^(t - ref), t = y log2(e) in 64 bits, ref the next whole number above the largest t.  A bucket lies within one
// power of two, and its values' weights are whole multiples of 2^-bits of that: their sums are exact in any order and in
// any number of parts.  The sum of all before a place in the order is that of the whole buckets before it, each rounded to the nearest
// 2^-bits of 2^ref, and that of its own bucket's values before it, rounded alike.  Every step below asks for this one number, wherever it
// gets the parts from, so bounds and draws agree with each other, and a row has the same bits however many workgroups share
// it.  Off by half a unit per bucket, 1,600 / 2: 2^-31 of the largest weight at 2^20 values, 2^-35 up to 2^16.  (Weights in
// units of the row's 2^ref lose a flat tail of light values, all of them rounded the same way, and sums cut to those
// units between workgroups disagree with sums of values.)  A row of which top-k leaves few is listed whole and its weights
// rounded to the row's units one by one, half a unit for each of at most 2,048.
//
// A row is small work with many steps that wait for each other, on few CUs: its latency bounds it.  16 rows of 2051 with
// guidance: 12 us; one row of 151,936: 11 us for the histograms and 19 for the rest; 64 of them in BF16 (19 MB): 23
// (VALU 87% busy, 59 instructions per value) and 30 us.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

// Each operation rounds by itself: guidance and quotients are defined so, and a t that enters a bucket
// and a weight is one number.
#pragma clang fp contract(off)

namespace sk {
namespace draw {

constexpr int NT = 1024;                          // threads of a workgroup
constexpr int PER_BIT = 64, FINE = 20 * PER_BIT;  // buckets per power of two of the weight, for the first 20 of them,
constexpr int STEP = 8, NB = FINE + 40 * PER_BIT / STEP;   // then an eighth as many, down to 2^-60 (2^20 weights of that are 2^-40)
constexpr double NEAR = 60.0;                     // a slice whose ref is further below the row's has nothing but weights of 0
constexpr int MOST_SLICES = 10;                   // workgroups per row
constexpr int CAP = 2048;                         // values of the list
constexpr int DIGITS = 2048;                      // of 11, 11 and 10 bits of a key
constexpr double LOG2E = 1.4426950408889634074, LN2 = 0.69314718055994530942;

struct Args {
  const void* logits; int64_t stride;             // rows of V (guidance: 2 R of them, cond and uncond in turn) so far apart
  const double* u;                                // [R]
  const float* temperature; const int* top_k; const float* top_p; const float* min_p;   // [R] or null: 1, none, none, none
  const float* cfg;                               // [R]: guidance, or null
  const uint32_t* allowed; int64_t allowed_stride;   // bits of the allowed ids, rows so far apart (0: one row for all), or null
  int R, V, bits;                                 // weights are multiples of 2^-bits
  int slices, slice;                              // workgroups per row, values of each
  int64_t* token; float* logprob; int* kept;      // [R]; logprob and kept may be null
  char* ws;                                       // slices > 1: RowSpace per row
};

// What the slices of a row leave for the second launch.
struct SliceInfo { double ref; unsigned long long best; int n; int wild; };

__device__ __forceinline__ uint32_t key_of(float y) {
  const uint32_t b = __float_as_uint(y + 0.f);    // -0 as 0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

template <typename X> __device__ __forceinline__ float to_f(X v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<uint16_t>(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }

// A row's parameters as they lie in memory: loaded before anything waits.
struct Given {
  float T, s, p, m;
  int k;
  double u;
  __device__ __forceinline__ Given(const Args& a, int r) {
    T = a.temperature ? a.temperature[r] : 1.f;
    s = a.cfg ? a.cfg[r] : 0.f;
    p = a.top_p ? a.top_p[r] : 0.f;
    m = a.min_p ? a.min_p[r] : 0.f;
    k = a.top_k ? a.top_k[r] : 0;
    u = a.u[r];
  }
  // Whether the row is listed down to its k-th value (or whole, where it has fewer than k).
  __device__ bool lists() const { return k > 0 && k <= CAP / 2; }
};

// One row's values as keys: larger values have larger keys, 0 is no candidate.  Keys of x, before the division, are enough
// wherever an order or a threshold is all that is asked: division by T > 0 keeps the order (but makes equals of some).
// WIDE: rows begin at multiples of 16 bytes and are whole pieces of 16, so that a load takes 4 or 8 values.
template <typename X, bool WIDE>
struct Row {
  static constexpr bool HELD = false;
  const X* cond; const X* uncond;
  const uint32_t* allowed;
  float s, T;
  double inv;                                     // 1 / T, or 0: divide
  bool whole;                                     // T = 1, or greedy: x itself
  int V;
  __device__ __forceinline__ Row(const Args& a, const Given& g, int r) {
    const X* l = static_cast<const X*>(a.logits);
    cond = l + (size_t)(a.cfg ? 2 * (size_t)r : r) * a.stride;
    uncond = a.cfg ? cond + a.stride : nullptr;
    allowed = a.allowed ? a.allowed + (size_t)r * a.allowed_stride : nullptr;
    s = g.s;
    T = g.T;
    inv = T > 0x1p-20f && T < 0x1p20f ? 1.0 / (double)T : 0.0;
    whole = __builtin_amdgcn_readfirstlane(T == 1.f || !(T > 0.f));   // one branch for a wave
    V = a.V;
  }
  // x / T rounded to FP32, held to the finite range.  By the reciprocal in 64 bits that is the same: its product is within
  // 2^-52 of the quotient, and a quotient of two 24-bit numbers is no middle of two FP32 numbers and lies at least
  // 2^-49 from any (x - T m is a multiple of the last place of a 49-bit product).  Results below the normal range
  // have fewer bits, so those are divided, and so is by temperatures that could make them of ordinary x.
  __device__ __forceinline__ float divided(float x) const {
    if (whole) return x;
    float y = (float)((double)x * inv);
    if (fabsf(y) < 0x1p-100f && x != 0.f) y = x / T;
    return __builtin_amdgcn_fmed3f(y, -3.402823466e38f, 3.402823466e38f);
  }
  // About the x of a y.
  __device__ __forceinline__ float near(double y) const { return (float)(whole ? y : y * (double)T); }
  // x of cond and uncond
  __device__ __forceinline__ float x_of(float x, float u) const { return u + s * (x - u); }
  static __device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.402823466e38f; }
  // the key of y
  __device__ __forceinline__ uint32_t key(int v) const {
    float x = to_f<X>(cond[v]);
    if (uncond) x = x_of(x, to_f<X>(uncond[v]));
    return finite(x) && (!allowed || (allowed[v >> 5] >> (v & 31) & 1u)) ? key_of(divided(x)) : 0u;
  }
  // f(id, x, whether it is a candidate) of values v0 .. v1, a thread's in the order of ids, 16 of them (8 of them one by one) on
  // their way at a time.  WIDE: v0 and v1 are at whole pieces.
  template <typename F>
  __device__ __forceinline__ void each(int v0, int v1, F f) const {
    if (uncond || allowed) each_as<true>(v0, v1, f);
    else each_as<false>(v0, v1, f);
  }
  template <bool MORE, typename F>
  __device__ __forceinline__ void each_as(int v0, int v1, F f) const {
    constexpr int P = WIDE ? 16 / (int)sizeof(X) : 1, U = WIDE ? 16 / P : 8;
    auto load = [](const X* p) {
      if constexpr (WIDE) return *reinterpret_cast<const uint4*>(p);
      else return to_f<X>(*p);
    };
    auto part = [](const auto& w, int j) {        // value j of a piece
      if constexpr (!WIDE) return w;
      else if constexpr (sizeof(X) == 4) return __uint_as_float(j == 0 ? w.x : j == 1 ? w.y : j == 2 ? w.z : w.w);
      else {
        const uint32_t pair = j < 2 ? w.x : j < 4 ? w.y : j < 6 ? w.z : w.w;
        return __uint_as_float(j & 1 ? pair & 0xffff0000u : pair << 16);
      }
    };
    using Piece = decltype(load(cond));
    for (int at = v0; at < v1; at += U * P * NT) {
      Piece c[U], u[MORE ? U : 1];
      uint32_t bits[MORE ? U : 1];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int l = min(at + (i * NT + (int)threadIdx.x) * P, v1 - P);
        c[i] = load(cond + l);
        if constexpr (MORE) {
          u[i] = uncond ? load(uncond + l) : c[i];
          bits[i] = allowed ? allowed[l >> 5] >> (l & 31) : ~0u;   // a piece's bits lie in one word
        }
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int v = at + (i * NT + (int)threadIdx.x) * P;
        if (v < v1) {
#pragma unroll
          for (int j = 0; j < P; ++j) {
            float x = part(c[i], j);
            if constexpr (MORE) {
              if (uncond) x = x_of(x, part(u[i], j));
              f(v + j, x, finite(x) && (bits[i] >> j & 1u));
            } else {
              f(v + j, x, finite(x));
            }
          }
        }
      }
    }
  }
};

// A row of up to 4 NT values, four of them in each thread's registers: read once (16 rows of 2051 with guidance and a mask: 12.4
// us in place of 15.0; 4,096 values without either 14.5 and 14.6; sixteen per thread 16,384 values 24 us, where reading them three
// times takes 19).  Its values' buckets are then found faster than the borders of ranges.
template <typename X>
struct Held : Row<X, false> {
  static constexpr bool HELD = true;
  static constexpr int N = 4;
  float x[N];                                     // NaN: no candidate
  __device__ __forceinline__ Held(const Args& a, const Given& g, int r) : Row<X, false>(a, g, r) {
    float c[N], u[N];
    uint32_t bits[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      c[i] = u[i] = 0.f;
      bits[i] = ~0u;
      if (i * NT < this->V) {                     // the workgroup's
        const int v = min(i * NT + (int)threadIdx.x, this->V - 1);
        c[i] = to_f<X>(this->cond[v]);
        if (this->uncond) u[i] = to_f<X>(this->uncond[v]);
        if (this->allowed) bits[i] = this->allowed[v >> 5] >> (v & 31);
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float y = this->uncond ? this->x_of(c[i], u[i]) : c[i];
      const bool on = this->finite(y) && (bits[i] & 1u) && i * NT + (int)threadIdx.x < this->V;
      x[i] = on ? y : __uint_as_float(0x7fc00000u);
    }
  }
  template <typename F>
  __device__ __forceinline__ void each(int, int, F f) const {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i * NT < this->V) f(i * NT + (int)threadIdx.x, x[i], x[i] == x[i]);
  }
};

__device__ __forceinline__ double log2_of(uint32_t key) { return (double)value_of(key) * LOG2E; }
// 2^-e, e = n + f: 2^-f by the exponential series in f ln 2 (|f ln 2| <= 0.347, terms to the 12th: 1e-16).
__device__ __forceinline__ double power(double e) {
  const double n = rint(e), z = (n - e) * LN2;
  double p = 1.0 / 479001600.0;
  p = fma(p, z, 1.0 / 39916800.0);
  p = fma(p, z, 1.0 / 3628800.0);
  p = fma(p, z, 1.0 / 362880.0);
  p = fma(p, z, 1.0 / 40320.0);
  p = fma(p, z, 1.0 / 5040.0);
  p = fma(p, z, 1.0 / 720.0);
  p = fma(p, z, 1.0 / 120.0);
  p = fma(p, z, 1.0 / 24.0);
  p = fma(p, z, 1.0 / 6.0);
  p = fma(p, z, 0.5);
  p = fma(p, z, 1.0);
  p = fma(p, z, 1.0);
  return ldexp(p, -(int)n);
}
// The weight of a value in units of 2^-bits of its step's power of two, rounded to nearest: 2^(-(b + 1/2) / 64) e^z of a value z
// above the middle of step b below a whole number.  The first from a table of 64, times 2^bits; the second by the exponential
// series (|z| < 0.006, terms to the 5th: 1e-16).  Below 1.001 2^bits.
__device__ __forceinline__ unsigned long long weight(double z, int b, const double* roots) {
  double p = fma(1.0 / 120.0, z, 1.0 / 24.0);
  p = fma(p, z, 1.0 / 6.0);
  p = fma(p, z, 0.5);
  p = fma(p, z, 1.0);
  p = fma(p, z, 1.0);
  const double x = fma(p, roots[b & (PER_BIT - 1)], 0x1p52);   // the sum's last bits are the whole number
  return (unsigned long long)__double_as_longlong(x) & 0xfffffffffffffull;
}
static_assert(PER_BIT == 64 && STEP == 8 && FINE % STEP == 0, "the shifts above and below");
constexpr int LAST = FINE + (NB - 1 - FINE) * STEP;   // the first step of the last bucket, which has all that is far below
// b < FINE ? b : FINE + (b - FINE) / STEP, b >= 0
__device__ __forceinline__ int bucket_of(int b) { return min(b, (FINE - FINE / STEP) + (b >> 3)); }
__device__ __forceinline__ int first_step(int bucket) { return max(bucket, FINE + (bucket - FINE) * STEP); }
// How many powers of two below the row's a bucket lies: all its steps within one, as 64 are, and 8 | 64.
__device__ __forceinline__ int powers_below(int bucket) { return first_step(bucket) >> 6; }
// A sum of a bucket's weights in the row's units, to nearest.
__device__ __forceinline__ unsigned long long in_row(unsigned long long sum, int bucket) {
  const int o = powers_below(bucket);
  return (sum + (1ull << o >> 1)) >> o;
}
// The largest sum of a bucket's weights that in_row keeps from passing x, x + 1 being at most in_row of them all.
__device__ __forceinline__ unsigned long long in_bucket(unsigned long long x, int bucket) {
  const int o = powers_below(bucket);
  return ((x + 1) << o) - (1ull << o >> 1) - 1;
}
// Where a row's values lie below its reference.  Steps of y are the same number for the same value wherever they are asked,
// larger for larger values, and counted down from 64 ref, ref a whole number, so counts from the refs of two slices are whole
// numbers apart.  FP32 does for that up to |y| of 4096 (steps within 0.05 of those of 64 bits).  Past it (a temperature of 1 /
// 1000, values of a mask's making) ref is the largest value itself, and its row is one workgroup's.
struct Scale {
  double ref, from, off;                          // in powers of two; e = (from - y) log2(e) + off
  float ref64, mid;                               // 64 ref - 1; what to take off a step for its middle, counted from `from` up
  bool wild;
  static __device__ __forceinline__ float steps(float y) { return floorf(y * (float)(LOG2E * PER_BIT)); }
  __device__ __forceinline__ explicit Scale(float of) {           // the workgroup's
    const uint32_t u = (uint32_t)__builtin_amdgcn_readfirstlane((int)__float_as_uint(of));
    const float y = __uint_as_float(u);
    wild = (u & 0x7fffffffu) >= 0x45800000u;      // 4096
    const float whole = floorf(steps(y) * (1.f / PER_BIT)) + 1.f;
    ref64 = whole * PER_BIT - 1.f;
    ref = wild ? (double)y * LOG2E : (double)whole;
    from = wild ? (double)y : 0.0;
    off = wild ? 0.0 : ref;
    mid = wild ? -.5f : ref64 + .5f;
  }
  // powers of two below ref
  __device__ __forceinline__ double e(float y) const { return fma(from - (double)y, LOG2E, off); }
  // whole steps below ref, at most LAST
  __device__ __forceinline__ float belowf(float y) const {
    if (wild) return (float)(int)fmin(e(y) * PER_BIT, (double)LAST);
    return __builtin_amdgcn_fmed3f(ref64 - steps(y), 0.f, (float)LAST);
  }
  __device__ __forceinline__ int bucket(float y) const { return bucket_of((int)belowf(y)); }
  // About the least y that is less than that many steps below.
  __device__ __forceinline__ double at_step(int step) const {
    return (double)(ref64 - (float)step + 1.f) * (LN2 / PER_BIT);
  }
  // The bucket of the least value that min-p keeps, give (-1) or take (1) rounding.
  __device__ __forceinline__ int least(float top, double m, double side) const {
    const double d = e(top) - log2(m) + side * 1e-3;
    return bucket_of((int)fmin(fmax(d * PER_BIT, 0.0), (double)LAST));
  }
  // The weight of a value that many steps below, in its bucket's units.  Nothing in it depends on ref (64 of which is what a
  // step's number and mid have in common): slices of a row give a value one weight.
  __device__ __forceinline__ unsigned long long weight_at(float y, float below, const double* roots) const {
    const double z = fma((double)(below - mid), LN2 / PER_BIT, (double)y - from);
    return draw::weight(z, (int)below, roots);
  }
  // A value's bucket, and its weight in the bucket's units: 0 in the last one.
  __device__ __forceinline__ unsigned long long weight(float y, int& bucket, const double* roots) const {
    const float d = belowf(y);
    bucket = bucket_of((int)d);
    return d < (float)LAST ? weight_at(y, d, roots) : 0;
  }
};

// The workgroup's shared memory.
struct Shared {
  double roots[PER_BIT];                          // 2^(bits - (i + 1/2) / 64)
  unsigned long long mass[NB + 1];                // of a bucket in its units, then of all before it in the row's
  alignas(16) unsigned long long list[2 * CAP];   // then their sums (digit by digit: histograms)
  unsigned count[NB + 1];
  unsigned long long wave64[16];
  unsigned wave32[16];
  unsigned listed;
  int flag, found;
  // ranges of buckets: first and last, the keys of x between them, where they begin in the list, what lies before them
  struct { int lo, hi, pos; uint32_t least, most; unsigned cp; unsigned long long mp; } range[4];
  int lo[4], hi[4], ranges, total;
  // digit by digit, within a bucket
  struct { unsigned prefix; unsigned cp; unsigned long long mp; unsigned cnt; unsigned long long mass; } at;
  __device__ __forceinline__ void fill_roots(int bits) {
    const int i = NT - 1 - threadIdx.x;
    if (i < PER_BIT) roots[i] = ldexp(power((i + 0.5) / PER_BIT), bits);
  }
};
static_assert(CAP * 16 >= (DIGITS + 1) * 12, "digits' histograms lie in the list's place");

// Exchanges between a wave's lanes in registers.
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned moved(unsigned v) { return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false); }
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned long long moved(unsigned long long v) {
  return (unsigned long long)moved<CTRL, ROWS>((unsigned)(v >> 32)) << 32 | moved<CTRL, ROWS>((unsigned)v);
}
// f of this lane's and all lower lanes' values, 0 being its neutral one: within rows of 16 lanes (shifted by 1, 2, 4, 8),
// then the last of a row into the next ones.
template <typename T, typename F>
__device__ __forceinline__ T wave_incl(T v, F f) {
  v = f(v, moved<0x111, 0xf>(v));
  v = f(v, moved<0x112, 0xf>(v));
  v = f(v, moved<0x114, 0xf>(v));
  v = f(v, moved<0x118, 0xf>(v));
  v = f(v, moved<0x142, 0xa>(v));                 // row_bcast15 into rows 1 and 3
  v = f(v, moved<0x143, 0xc>(v));                 // row_bcast31 into rows 2 and 3
  return v;
}
__device__ __forceinline__ unsigned at_lane(unsigned v, int l) { return (unsigned)__builtin_amdgcn_readlane((int)v, l); }
__device__ __forceinline__ unsigned long long at_lane(unsigned long long v, int l) {
  return (unsigned long long)at_lane((unsigned)(v >> 32), l) << 32 | at_lane((unsigned)v, l);
}
struct Plus { template <typename T> __device__ T operator()(T a, T b) const { return a + b; } };
struct Larger { template <typename T> __device__ T operator()(T a, T b) const { return a > b ? a : b; } };
template <typename T, typename F>
__device__ __forceinline__ T wave_all(T v, F f) { return at_lane(wave_incl(v, f), 63); }

// The largest of a and the sum of b over the workgroup, in every thread.
__device__ __forceinline__ void block_max_sum(unsigned long long& a, unsigned& b, Shared& s) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  a = wave_all(a, Larger{});
  b = wave_all(b, Plus{});
  __syncthreads();
  if (lane == 0) { s.wave64[wave] = a; s.wave32[wave] = b; }
  __syncthreads();
  a = wave_all(lane < 16 ? s.wave64[lane] : 0, Larger{});
  b = wave_all(lane < 16 ? s.wave32[lane] : 0, Plus{});
}
// The sum over the workgroup, in every thread.
__device__ __forceinline__ unsigned long long block_sum(unsigned long long v, Shared& s) {
  const int lane = threadIdx.x & 63;
  v = wave_all(v, Plus{});
  __syncthreads();
  if (lane == 0) s.wave64[threadIdx.x >> 6] = v;
  __syncthreads();
  return wave_all(lane < 16 ? s.wave64[lane] : 0, Plus{});
}
// Exclusive sums of count[0 .. n) and mass[0 .. n) in place, and the wholes at n; n at most 2 NT.  BUCKETS: masses are
// buckets' and become the row's.
template <bool BUCKETS>
__device__ __forceinline__ void block_scan(unsigned* count, unsigned long long* mass, int n, Shared& s) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, at = threadIdx.x * 2;
  const bool on0 = at < n, on1 = at + 1 < n;
  const unsigned c0 = on0 ? count[at] : 0, c1 = on1 ? count[at + 1] : 0;
  unsigned long long m0 = on0 ? mass[at] : 0, m1 = on1 ? mass[at + 1] : 0;
  if constexpr (BUCKETS) {
    m0 = in_row(m0, on0 ? at : 0);
    m1 = in_row(m1, on1 ? at + 1 : 0);
  }
  unsigned c = wave_incl(c0 + c1, Plus{});
  unsigned long long m = wave_incl(m0 + m1, Plus{});
  if (lane == 63) { s.wave32[wave] = c; s.wave64[wave] = m; }
  __syncthreads();
  // lane w: all of the waves before w + 1
  const unsigned wc = wave_incl(lane < 16 ? s.wave32[lane] : 0, Plus{});
  const unsigned long long wm = wave_incl(lane < 16 ? s.wave64[lane] : 0, Plus{});
  if (wave) { c += at_lane(wc, wave - 1); m += at_lane(wm, wave - 1); }
  c -= c0 + c1;
  m -= m0 + m1;
  if (on0) { count[at] = c; mass[at] = m; }
  if (on1) { count[at + 1] = c + c0; mass[at + 1] = m + m0; }
  if (threadIdx.x == 0) { count[n] = at_lane(wc, 15); mass[n] = at_lane(wm, 15); }
  __syncthreads();
}

// The largest key of x, the lowest id that has it, and how many candidates values v0 .. v1 hold.
template <typename R>
__device__ __forceinline__ void survey(const R& row, int v0, int v1, Shared& s, unsigned long long& best, int& n) {
  float most = -INFINITY;
  int id = 0;
  unsigned c = 0;
  row.each(v0, v1, [&](int v, float x, bool on) __attribute__((always_inline)) {
    c += on;
    if (on && x > most) { most = x; id = v; }     // ids come in order: the first of equal ones stays
  });
  best = c ? (unsigned long long)key_of(most) << 32 | (uint32_t)~id : 0ull;
  block_max_sum(best, c, s);
  n = (int)c;
}
// Counts and (with sums) sums of weights by bucket, in its units, of values v0 .. v1 in s.count and s.mass.
template <typename R>
__device__ __forceinline__ void histogram(const R& row, int v0, int v1, const Scale& at, bool sums, Shared& s) {
  for (int i = threadIdx.x; i < NB; i += NT) { s.count[i] = 0; s.mass[i] = 0; }
  __syncthreads();
  row.each(v0, v1, [&](int, float x, bool on) __attribute__((always_inline)) {
    const float y = row.divided(x), d = at.belowf(y);
    const int b = bucket_of((int)d);
    const unsigned long long w = sums ? at.weight_at(y, d, s.roots) : 0;
    if (on) {
      atomicAdd(&s.count[b], 1u);
      if (sums && d < (float)LAST) atomicAdd(&s.mass[b], w);
    }
  });
  __syncthreads();
}

// As the definitions read them, with n candidates.
struct Params {
  double p, m, u;                                 // p in (0, 1) or 0: none; m in (0, 1] or 0: none
  int k;                                          // 0: none
  bool greedy, list;                              // list: all that top-k leaves is listed, and no sums are asked of the histogram
  __device__ __forceinline__ Params(const Given& g, int n) {
    greedy = !(g.T > 0.f);
    list = g.lists();
    k = g.k > 0 && g.k < n ? g.k : 0;
    p = g.p > 0.f && g.p < 1.f ? (double)g.p : 0.0;
    m = g.m > 0.f && g.m <= 1.f ? (double)g.m : 0.0;
    u = g.u > 0.0 ? fmin(g.u, 1.0) : 0.0;         // NaN and less than 0: 0
  }
};
// Largest whole number not above part * all, and below all.
__device__ __forceinline__ unsigned long long part_of(double part, unsigned long long all) {
  const double t = part * (double)all;
  const unsigned long long x = t >= (double)all ? all : (unsigned long long)t;
  return x >= all ? (all ? all - 1 : 0) : x;
}
// The kept weights' threshold: 2^-(e - e0) >= m.
__device__ __forceinline__ bool heavy(uint32_t key, uint32_t top, double m) {
  return power(fmin(log2_of(top) - log2_of(key), 1000.0)) >= m;
}

// The buckets in which the row's bounds are passed, as ranges in s.range; s.total is the number of values
// that they hold.  The whole that top-p takes its part of, and the kept sum that the draw takes its part of, are
// known up to the bucket in which the bound before lies, so theirs may be several.  All threads:
// each looks at two buckets.
template <typename R>
__device__ __forceinline__ void plan(const R& row, const Params& q, const Scale& at, float top, Shared& s) {
  // the buckets b with a[b] <= x < a[b + 1] (sums of all before) for lo and hi
  auto find = [&](const auto* a, auto lo, auto hi, int& lo_b, int& hi_b, int i) {
    for (int b = threadIdx.x; b < NB; b += NT) {
      const auto x = a[b], y = a[b + 1];
      if (x <= lo && lo < y) s.lo[i] = b;
      if (x <= hi && hi < y) s.hi[i] = b;
    }
    __syncthreads();
    lo_b = s.lo[i];
    hi_b = s.hi[i];
  };
  constexpr int NONE = 1 << 20;
  int lo[4] = {NONE, NONE, NONE, NONE}, hi[4] = {NONE, NONE, NONE, NONE};   // of k, p, min-p, the draw
  unsigned long long w_lo = s.mass[NB], w_hi = w_lo;
  if (q.k) {
    find(s.count, (unsigned)(q.k - 1), (unsigned)(q.k - 1), lo[0], hi[0], 0);
    w_lo = s.mass[lo[0]]; w_hi = s.mass[lo[0] + 1];
  }
  if (q.list) {                                   // one range from the first bucket on
    lo[0] = 0;
    if (!q.k) hi[0] = NB - 1;
  } else {
    unsigned long long k_lo = w_lo, k_hi = w_hi;  // of the kept sum
    if (q.p > 0.0) {
      find(s.mass, part_of(q.p, w_lo), part_of(q.p, w_hi), lo[1], hi[1], 1);
      k_lo = s.mass[lo[1]]; k_hi = s.mass[hi[1] + 1];
    }
    if (q.m > 0.0) {
      lo[2] = at.least(top, q.m, -1.0); hi[2] = at.least(top, q.m, 1.0);
      k_lo = min(k_lo, s.mass[lo[2]]); k_hi = min(k_hi, s.mass[hi[2] + 1]);
    }
    find(s.mass, part_of(q.u, k_lo), part_of(q.u, k_hi), lo[3], hi[3], 3);
  }
  // by their first bucket
  auto order = [&](int i, int j) {
    if (lo[j] < lo[i]) {
      const int a = lo[i], b = hi[i];
      lo[i] = lo[j]; hi[i] = hi[j]; lo[j] = a; hi[j] = b;
    }
  };
  order(0, 1); order(2, 3); order(0, 2); order(1, 3); order(1, 2);
  if (threadIdx.x == 0) {
    unsigned total = 0;
    int r = 0, l = lo[0], h = hi[0];
    auto put = [&]() {
      const unsigned c = s.count[l];
      s.range[r].lo = l; s.range[r].hi = h;
      s.range[r].pos = (int)total;
      s.range[r].cp = c; s.range[r].mp = s.mass[l];
      total += s.count[h + 1] - c;
      ++r;
    };
#pragma unroll
    for (int i = 1; i < 4; ++i)
      if (lo[i] != NONE) {
        if (lo[i] <= h + 1) h = max(h, hi[i]);    // overlapping ones become one
        else { put(); l = lo[i]; h = hi[i]; }
      }
    put();
    s.ranges = r;
    s.total = (int)total;
    s.listed = 0;
  }
  __syncthreads();
  if constexpr (R::HELD) return;                  // gather looks at buckets
  // the keys of x that a range begins and ends with: the largest whose bucket is at least lo, the least whose
  // bucket is at most hi; a wave for each, which tries 64 keys at a time
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  if (wave < 2 * s.ranges) {
    const int i = wave / 2, border = __builtin_amdgcn_readfirstlane(wave & 1 ? s.range[i].hi + 1 : s.range[i].lo);
    // keys before `from` are on this side of the border, from `from + size` on they are not (border: the first
    // key whose bucket is before this one)
    uint32_t from = 0x00800000u, size = 0xff800000u - 0x00800000u;   // of the finite numbers
    auto past = [&](uint32_t key) { return at.bucket(row.divided(value_of(key))) < border; };
    if (border == 0) {
      from += size; size = 0;                     // none is
    } else if (border == NB) {
      size = 0;                                   // all are
    } else {
      // 64 keys where the border should be
      const float x = row.near(at.at_step(first_step(border)));
      const uint32_t k = min(max(key_of(x), from + 64), from + size - 64) - 32;
      const uint64_t is = __ballot(past(k + lane));
      if (is && !(is & 1)) {
        from = k + __builtin_ctzll(is);
        size = 0;
      }
    }
    while (size) {
      const uint32_t part = size / 64 + 1, end = from + size;   // lane l asks of key from + (l + 1) part - 1
      const uint64_t key = (uint64_t)from + (lane + 1) * (uint64_t)part - 1;
      const bool is = key >= end || past((uint32_t)key);   // 64 parts are more than size: one is past
      from += __builtin_ctzll(__ballot(is)) * part;
      size = min(part - 1, end - from);
    }
    if (lane == 0) {
      if (wave & 1) s.range[i].least = (uint32_t)from;
      else s.range[i].most = (uint32_t)from - 1;
    }
  }
  __syncthreads();
}

// Puts the values of v0 .. v1 that lie in the ranges into s.list, s.listed of them.
template <typename R>
__device__ __forceinline__ void gather(const R& row, const Scale& scale, int v0, int v1, Shared& s) {
  auto put = [&](int v, float y) __attribute__((always_inline)) {
    const unsigned at = atomicAdd(&s.listed, 1u);
    if (at < CAP) s.list[at] = (unsigned long long)key_of(y) << 32 | (uint32_t)~v;
  };
  if constexpr (R::HELD) {
    row.each(v0, v1, [&](int v, float x, bool on) __attribute__((always_inline)) {
      const float y = row.divided(x);
      const int b = scale.bucket(y);
      bool in = false;
      for (int i = 0; i < s.ranges; ++i) in |= b >= s.range[i].lo && b <= s.range[i].hi;
      if (in && on) put(v, y);
    });
    __syncthreads();
    return;
  }
  auto pass = [&](auto ranges) __attribute__((always_inline)) {
    constexpr int N = decltype(ranges)::value;
    float least[N], most[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const bool is = i < s.ranges;
      least[i] = is ? value_of(s.range[i].least) : INFINITY;
      most[i] = is ? value_of(s.range[i].most) : 0.f;
    }
    row.each(v0, v1, [&](int v, float x, bool on) __attribute__((always_inline)) {
      bool in = false;
#pragma unroll
      for (int i = 0; i < N; ++i) in |= x >= least[i] && x <= most[i];
      if (in && on) put(v, row.divided(x));
    });
  };
  if (s.ranges <= 2) pass(std::integral_constant<int, 2>{});   // most rows
  else pass(std::integral_constant<int, 4>{});
  __syncthreads();
}

// s.list[0 .. n), largest first; n at most CAP.  Up to NT values each finds its place by counting the
// larger ones, NT / P threads to a value (181 values: 2,000 clocks, by the network, whose steps are a barrier
// each, 17,600); more take the network.
__device__ __forceinline__ void sort_list(int n, Shared& s) {
  int P = 2;
  while (P < n) P <<= 1;
  if (P <= NT) {
    const int per = NT / P < 64 ? NT / P : 64, i = threadIdx.x / per, part = threadIdx.x % per;
    unsigned long long x = 0;
    unsigned place = 0;
    if (threadIdx.x == 0 && (n & 1)) s.list[n] = 0;
    __syncthreads();
    if (i < n) {
      const ulonglong2* pairs = reinterpret_cast<const ulonglong2*>(s.list);
      x = s.list[i];
#pragma unroll 8
      for (int j = part; j < (n + 1) / 2; j += per) {
        const ulonglong2 y = pairs[j];
        place += (y.x > x) + (y.y > x);
      }
    }
    for (int o = per / 2; o; o >>= 1) place += __shfl_xor(place, o);
    __syncthreads();
    if (i < n && part == 0) s.list[place] = x;
    __syncthreads();
    return;
  }
  for (int i = n + threadIdx.x; i < P; i += NT) s.list[i] = 0;
  __syncthreads();
  for (int k = 2; k <= P; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      for (int i = threadIdx.x; i < P; i += NT) {
        const int l = i ^ j;
        if (l > i) {
          const unsigned long long a = s.list[i], b = s.list[l];
          if ((i & k) == 0 ? b > a : a > b) { s.list[i] = b; s.list[l] = a; }
        }
      }
      __syncthreads();
    }
}

__device__ __forceinline__ void answer(const Args& a, int r, int token, double logprob, int kept) {
  a.token[r] = token;
  if (a.logprob) a.logprob[r] = kept == 1 ? 0.f : (float)logprob;   // the only one is the whole: exactly 0
  if (a.kept) a.kept[r] = kept;
}
// ln of the drawn one's part of the kept sum, which may be all that the sum holds of it.
__device__ __forceinline__ double part_log(uint32_t key, const Scale& at, unsigned long long kept, int bits) {
  return fmin((bits - at.e(value_of(key))) * LN2 - log((double)kept), 0.0);
}

// The row's answer from the sorted list of its ranges.
__device__ __forceinline__ void finish_list(const Args& a, int r, const Params& q, const Scale& scale, uint32_t top, int n, Shared& s) {
  const int total = s.total, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  unsigned long long* sum_at = s.list + CAP;
  // sums up to and with each, `per` neighbours to a thread: of the row's units if all that is kept is listed, of each bucket's own
  // if not (differences within a bucket are all that is taken of them)
  const int per = (total + NT - 1) / NT;
  {
    unsigned long long v[CAP / NT], mine = 0;
#pragma unroll
    for (int i = 0; i < CAP / NT; ++i) {
      const int at = tid * per + i;
      v[i] = 0;
      if (i < per && at < total) {
        const uint32_t key = (uint32_t)(s.list[at] >> 32);
        int b;
        v[i] = scale.weight(value_of(key), b, s.roots);
        if (q.list) v[i] = in_row(v[i], b);
      }
      mine += v[i];
    }
    const unsigned long long incl = wave_incl(mine, Plus{});
    if (lane == 63) s.wave64[wave] = incl;
    __syncthreads();
    unsigned long long x = incl - mine;
    for (int w = 0; w < wave; ++w) x += s.wave64[w];
#pragma unroll
    for (int i = 0; i < CAP / NT; ++i) {
      const int at = tid * per + i;
      x += v[i];
      if (i < per && at < total) sum_at[at] = x;
    }
  }
  __syncthreads();
  if (wave) return;
  // one wave from here on
  auto end_of = [&](int i) { return i + 1 < s.ranges ? s.range[i + 1].pos : total; };
  // sum of all up to and with list entry i of range g
  auto upto = [&](int g, int i) {
    if (q.list) return sum_at[i];
    const int b = scale.bucket(value_of((uint32_t)(s.list[i] >> 32)));
    const int p = s.range[g].pos + (int)(s.count[b] - s.range[g].cp);   // where the bucket begins
    return s.mass[b] + in_row(sum_at[i] - (p ? sum_at[p - 1] : 0), b);
  };
  // first entry of range g for which `past` holds (it holds from some entry on), or its end; 64 at a time
  auto first = [&](int g, auto past) {
    int from = s.range[g].pos, size = end_of(g) - from;
    while (size) {
      const int part = size / 64 + 1, at = from + (lane + 1) * part - 1, end = from + size;
      from += __builtin_ctzll(__ballot(at >= end || past(at))) * part;   // 64 parts are more than size: one is past
      size = min(part - 1, end - from);
    }
    return from;
  };
  // (values, sum) of all before entry i of range g
  auto before = [&](int g, int i, unsigned& c, unsigned long long& w) {
    c = s.range[g].cp + (unsigned)(i - s.range[g].pos);
    w = i > s.range[g].pos ? upto(g, i - 1) : s.range[g].mp;
  };
  auto range_of_count = [&](unsigned c) {         // the range that holds the c-th of all (from 0)
    int g = 0;
    while (g + 1 < s.ranges && s.range[g + 1].cp <= c) ++g;
    return g;
  };
  auto range_of_mass = [&](unsigned long long T) {
    int g = 0;
    while (g + 1 < s.ranges && s.range[g + 1].mp <= T) ++g;
    return g;
  };
  unsigned kept = (unsigned)n;
  unsigned long long sum = q.list ? sum_at[total - 1] : s.mass[NB];
  if (q.k) {
    const int g = range_of_count(q.k - 1), at = s.range[g].pos + (int)(q.k - 1 - s.range[g].cp);
    const uint32_t cut = (uint32_t)(s.list[at] >> 32);
    before(g, first(g, [&](int i) { return (uint32_t)(s.list[i] >> 32) < cut; }), kept, sum);
  }
  if (q.p > 0.0) {
    const unsigned long long T = part_of(q.p, sum);
    const int g = range_of_mass(T);
    const int i = min(first(g, [&](int i) { return upto(g, i) > T; }), end_of(g) - 1);
    unsigned c;
    unsigned long long w;
    before(g, i + 1, c, w);
    if (c < kept) { kept = c; sum = w; }
  }
  if (q.m > 0.0) {
    // its range holds the bucket of the bound
    const int b = scale.least(value_of(top), q.m, -1.0);
    int g = 0;
    while (g + 1 < s.ranges && s.range[g + 1].lo <= b) ++g;
    unsigned c;
    unsigned long long w;
    before(g, first(g, [&](int i) { return !heavy((uint32_t)(s.list[i] >> 32), top, q.m); }), c, w);
    if (c < kept) { kept = c; sum = w; }
  }
  const unsigned long long T = part_of(q.u, sum);
  const int g = range_of_mass(T);
  const int i = min(first(g, [&](int i) { return upto(g, i) > T; }), end_of(g) - 1);
  if (lane == 0) answer(a, r, (int)~(uint32_t)s.list[i], part_log((uint32_t)(s.list[i] >> 32), scale, sum, a.bits), (int)kept);
}

// Digit by digit among the values of one bucket: the value at which their count, largest first (by_count), or the sum of their weights
// in the bucket's units passes T, less than the whole, in s.at: its key, the count and sum of all above it, and its own.
template <typename X, bool WIDE>
__device__ __forceinline__ void descend(const Row<X, WIDE>& row, const Scale& scale, int bucket, bool by_count, unsigned long long T, Shared& s) {
  unsigned long long* mass = s.list;              // [DIGITS + 1], then counts
  unsigned* count = reinterpret_cast<unsigned*>(s.list + DIGITS + 1);
  uint32_t prefix = 0, mask = 0;
  unsigned cp = 0;
  unsigned long long mp = 0;
  for (int level = 0; level < 3; ++level) {
    const int shift = level == 0 ? 21 : level == 1 ? 10 : 0, digits = level < 2 ? 2048 : 1024;
    for (int i = threadIdx.x; i <= DIGITS; i += NT) { mass[i] = 0; count[i] = 0; }
    __syncthreads();
    for (int v0 = 0; v0 < row.V; v0 += NT) {      // whole waves
      const int v = v0 + threadIdx.x;
      const uint32_t k = v < row.V ? row.key(v) : 0;
      int b = -1;
      unsigned long long w = 0;
      if (k && (k & mask) == prefix) w = scale.weight(value_of(k), b, s.roots);
      const bool on = b == bucket;
      const int d = digits - 1 - (int)(k >> shift & (digits - 1));
      // where a wave's values all have one digit, as equal logits do, one lane adds for all
      const unsigned long long who = __ballot(on);
      if (!who) continue;
      const int d0 = __builtin_amdgcn_readlane(d, __builtin_ctzll(who));
      if (__ballot(on && d == d0) == who) {
        w = wave_all(on ? w : 0ull, Plus{});
        if ((threadIdx.x & 63) == 0) {
          atomicAdd(&count[d0], (unsigned)__popcll(who));
          atomicAdd(&mass[d0], w);
        }
      } else if (on) {
        atomicAdd(&count[d], 1u);
        atomicAdd(&mass[d], w);
      }
    }
    __syncthreads();
    block_scan<false>(count, mass, digits, s);
    if (threadIdx.x == 0) {
      int lo = 0, hi = digits - 1;
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (by_count ? cp + count[mid + 1] > T : mp + mass[mid + 1] > T) hi = mid;
        else lo = mid + 1;
      }
      s.at.prefix = prefix | (uint32_t)(digits - 1 - lo) << shift;
      s.at.cp = cp + count[lo]; s.at.mp = mp + mass[lo];
      s.at.cnt = count[lo + 1] - count[lo]; s.at.mass = mass[lo + 1] - mass[lo];
    }
    __syncthreads();
    prefix = s.at.prefix;
    mask |= (uint32_t)(digits - 1) << shift;
    cp = s.at.cp;
    mp = s.at.mp;
    __syncthreads();
  }
}

// The row's answer where the list does not hold its ranges: the bucket of each bound from the histogram's sums, then its value.
template <typename X, bool WIDE>
__device__ __forceinline__ void finish_digits(const Args& a, int r, const Row<X, WIDE>& row, const Params& q, const Scale& scale, uint32_t top,
                              int n, Shared& s) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (q.list) {                                   // the histogram has no sums yet
    histogram(row, 0, a.V, scale, true, s);
    block_scan<true>(s.count, s.mass, NB, s);
  }
  // the bucket b with of[b] <= x < of[b + 1], x less than the whole
  auto bucket = [&](const auto* of, auto x) {
    int lo = 0, hi = NB - 1;
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (of[mid + 1] > x) hi = mid;
      else lo = mid + 1;
    }
    return lo;
  };
  unsigned kept = (unsigned)n;
  unsigned long long sum = s.mass[NB];
  // all down to the value of the c-th of all (from 0) are kept
  auto keep_to = [&](unsigned c) {
    const int b = bucket(s.count, c);
    descend(row, scale, b, true, c - s.count[b], s);
    kept = s.count[b] + s.at.cp + s.at.cnt;
    sum = s.mass[b] + in_row(s.at.mp + s.at.mass, b);
  };
  // the value at which the sum of all passes T, in s.at, and how many of its equal ones are before the one that does
  auto pass = [&](unsigned long long T, int& b, unsigned long long& w) {
    b = bucket(s.mass, T);
    const unsigned long long most = in_bucket(T - s.mass[b], b);
    descend(row, scale, b, false, most, s);
    w = s.at.mass / s.at.cnt;                     // equal values have one weight, and not 0 where sums pass anything
    return (unsigned)((most - s.at.mp) / w);
  };
  int b;
  unsigned long long w;
  if (q.k) keep_to(q.k - 1);
  if (q.p > 0.0) {
    const unsigned nth = pass(part_of(q.p, sum), b, w), c = s.count[b] + s.at.cp + nth + 1;
    if (c < kept) { kept = c; sum = s.mass[b] + in_row(s.at.mp + (nth + 1) * w, b); }
  }
  if (q.m > 0.0) {
    unsigned long long c = 0;
    for (int v = tid; v < row.V; v += NT) {
      const uint32_t k = row.key(v);
      c += k && heavy(k, top, q.m);
    }
    c = block_sum(c, s);
    if (c < kept) keep_to((unsigned)c - 1);       // equal values are alike: these and no others
  }
  const unsigned nth = pass(part_of(q.u, sum), b, w);
  const uint32_t key = s.at.prefix;
  // each wave counts the equal ones of its run of ids, then the one that has it looks again
  const int run = (row.V + NT / 64 - 1) / (NT / 64), v0 = wave * run, v1 = min(v0 + run, row.V);
  unsigned c = 0;
  for (int v = v0 + lane; v - lane < v1; v += 64) c += (unsigned)__popcll(__ballot(v < v1 && row.key(v) == key));
  __syncthreads();
  if (lane == 0) s.wave32[wave] = c;
  __syncthreads();
  unsigned ahead = 0;
  for (int i = 0; i < wave; ++i) ahead += s.wave32[i];
  if (nth >= ahead && nth < ahead + c) {          // one wave
    for (int v = v0 + lane; v - lane < v1; v += 64) {
      const bool is = v < v1 && row.key(v) == key;
      const unsigned long long who = __ballot(is);
      const unsigned mine = ahead + (unsigned)__popcll(who & ((1ull << lane) - 1));
      if (is && mine == nth) answer(a, r, v, part_log(key, scale, sum, a.bits), (int)kept);
      ahead += (unsigned)__popcll(who);
    }
  }
}

// A row that needs no sums: greedy, or without candidates.
__device__ __forceinline__ bool finish_early(const Args& a, int r, const Params& q, unsigned long long best, int n) {
  if (n && !q.greedy) return false;
  if (threadIdx.x == 0) answer(a, r, n ? (int)~(uint32_t)best : -1, n ? 0.0 : -INFINITY, n ? 1 : 0);
  return true;
}

// A whole row in one workgroup.
template <typename R>
__device__ __forceinline__ void whole_row(const Args& a, int r, const Given& given, const R& row, Shared& s) {
  s.fill_roots(a.bits);
  unsigned long long best;
  int n;
  survey(row, 0, a.V, s, best, n);
  const Params q(given, n);
  if (finish_early(a, r, q, best, n)) return;
  const uint32_t top = key_of(row.divided(value_of((uint32_t)(best >> 32))));
  const Scale scale(value_of(top));
  histogram(row, 0, a.V, scale, !q.list, s);
  block_scan<true>(s.count, s.mass, NB, s);
  plan(row, q, scale, value_of(top), s);
  if (s.total > CAP) {
    finish_digits(a, r, row, q, scale, top, n, s);
    return;
  }
  gather(row, scale, 0, a.V, s);
  sort_list(s.total, s);
  finish_list(a, r, q, scale, top, n, s);
}
template <typename X>
__global__ __launch_bounds__(NT) void held_kernel(Args a) {
  __shared__ Shared s;
  const int r = blockIdx.x;
  const Given given(a, r);
  const Held<X> row(a, given, r);
  whole_row(a, r, given, row, s);
}
template <typename X, bool WIDE>
__global__ __launch_bounds__(NT) void row_kernel(Args a) {
  __shared__ Shared s;
  const int r = blockIdx.x;
  const Given given(a, r);
  const Row<X, WIDE> row(a, given, r);
  whole_row(a, r, given, row, s);
}

// A row over several workgroups, in two launches.  The first leaves each slice's histogram,
// counted from the slice's own ref; the second adds them up (every workgroup for itself: that needs no
// arrival to wait for), lists its slice's values of the ranges, and the last one to arrive finishes.
struct RowSpace {
  SliceInfo* info;                                // [slices]
  unsigned long long* mass; unsigned* count;      // [slices][NB]
  unsigned long long* list;                       // [CAP]
  unsigned* listed; unsigned* arrived;
  static __host__ __device__ size_t bytes(int slices) {
    return (slices * (sizeof(SliceInfo) + NB * 12) + CAP * 8 + 8 + 255) / 256 * 256;
  }
  __device__ __forceinline__ RowSpace(const Args& a, int r) {
    char* p = a.ws + r * bytes(a.slices);
    info = reinterpret_cast<SliceInfo*>(p); p += a.slices * sizeof(SliceInfo);
    mass = reinterpret_cast<unsigned long long*>(p); p += (size_t)a.slices * NB * 8;
    list = reinterpret_cast<unsigned long long*>(p); p += CAP * 8;
    count = reinterpret_cast<unsigned*>(p); p += (size_t)a.slices * NB * 4;
    listed = reinterpret_cast<unsigned*>(p);
    arrived = listed + 1;
  }
};

template <typename X, bool WIDE>
__global__ __launch_bounds__(NT) void slice_kernel(Args a) {
  __shared__ Shared s;
  s.fill_roots(a.bits);
  const int r = blockIdx.y, g = blockIdx.x;
  const Given given(a, r);
  const Row<X, WIDE> row(a, given, r);
  const RowSpace w(a, r);
  const int v0 = g * a.slice, v1 = min(v0 + a.slice, a.V);
  unsigned long long best;
  int n;
  survey(row, v0, v1, s, best, n);
  const Scale scale(n ? row.divided(value_of((uint32_t)(best >> 32))) : 0.f);
  if (threadIdx.x == 0) {
    w.info[g] = {scale.ref, best, n, scale.wild};
    if (g == 0) { *w.listed = 0; *w.arrived = 0; }
  }
  if (n == 0 || !(row.T > 0.f) || scale.wild) return;   // nothing of it is read
  histogram(row, v0, v1, scale, !given.lists(), s);
  for (int i = threadIdx.x; i < NB; i += NT) {
    w.count[g * NB + i] = s.count[i];
    w.mass[g * NB + i] = s.mass[i];
  }
}

template <typename X, bool WIDE>
__global__ __launch_bounds__(NT) void pick_kernel(Args a) {
  __shared__ Shared s;
  s.fill_roots(a.bits);
  const int r = blockIdx.y, g = blockIdx.x;
  const Given given(a, r);
  const Row<X, WIDE> row(a, given, r);
  const RowSpace w(a, r);
  // a lane for each slice
  const int lane = threadIdx.x & 63;
  SliceInfo info{0.0, 0ull, 0, 0};
  if (lane < a.slices) info = w.info[lane];
  const unsigned long long best = wave_all(info.best, Larger{});
  const int n = (int)wave_all((unsigned)info.n, Plus{});
  const Params q(given, n);
  if (n == 0 || q.greedy) {
    if (g == 0) finish_early(a, r, q, best, n);
    return;
  }
  const uint32_t top = key_of(row.divided(value_of((uint32_t)(best >> 32))));
  const Scale scale(value_of(top));
  const double up = scale.ref - info.ref;         // a whole number, or of no use
  const bool near = info.n && up < NEAR;
  const int lower = near ? (int)up : -1;
  // One workgroup does all if the row's values, or those of a slice near the largest, are such that there is no histogram.
  const bool alone = scale.wild || __any(near && info.wild);
  if (alone && g) return;
  if (alone) {
    histogram(row, 0, a.V, scale, !q.list, s);
  } else {
    // A slice's ref is `by` powers of two lower, so its steps lie 64 by further below the row's: a fine bucket has one of
    // the slice's fine ones, a wide one has one of its wide ones, or eight of its last fine ones, in the same units.  All loads
    // are on their way at once: they come from other XCDs' stores, 1 us away.
    constexpr int U = (NB + NT - 1) / NT;         // buckets of a thread
    const bool sums = !q.list;
    unsigned x[MOST_SLICES][U];
    unsigned long long y[MOST_SLICES][U];
#pragma unroll
    for (int i = 0; i < MOST_SLICES; ++i)
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int b = j * NT + threadIdx.x, by = __builtin_amdgcn_readlane(lower, i);   // -1 past the slices too
        const int d = b < FINE ? b - by * PER_BIT : b - by * (PER_BIT / STEP);
        x[i][j] = 0;
        y[i][j] = 0;
        if (by >= 0 && b < NB - 1 && d >= (b < FINE ? 0 : FINE)) {   // the row's last bucket has the rest
          x[i][j] = w.count[i * NB + d];
          if (sums) y[i][j] = w.mass[i * NB + d];
        }
      }
    // a wave for each slice's last fine ones, the first of them on their way too
    static_assert(MOST_SLICES <= NT / 64, "a wave for each");
    constexpr int AHEAD = 3;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), by = __builtin_amdgcn_readlane(lower, wave);
    const int d0 = max(FINE - by * PER_BIT, 0) + lane;   // none where by is -1 or 0
    unsigned xf[AHEAD];
    unsigned long long yf[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int d = d0 + j * 64;
      xf[j] = d < FINE ? w.count[wave * NB + d] : 0;
      yf[j] = sums && d < FINE ? w.mass[wave * NB + d] : 0;
    }
    for (int i = threadIdx.x; i < NB; i += NT) { s.count[i] = 0; s.mass[i] = 0; }
    __syncthreads();
    auto put = [&](int d, unsigned c, unsigned long long m) __attribute__((always_inline)) {
      const int to = bucket_of(d + by * PER_BIT);
      if (to < NB - 1 && c) {
        atomicAdd(&s.count[to], c);
        if (sums) atomicAdd(&s.mass[to], m);
      }
    };
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) put(d0 + j * 64, xf[j], yf[j]);
    for (int d = d0 + AHEAD * 64; d < FINE; d += 64) put(d, w.count[wave * NB + d], sums ? w.mass[wave * NB + d] : 0);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int b = j * NT + threadIdx.x;
      unsigned c = 0;
      unsigned long long m = 0;
#pragma unroll
      for (int i = 0; i < MOST_SLICES; ++i) {
        c += x[i][j];
        m += y[i][j];
      }
      if (b < NB) { s.count[b] += c; s.mass[b] += m; }
    }
    __syncthreads();
  }
  block_scan<true>(s.count, s.mass, NB, s);
  if (threadIdx.x == 0) s.count[NB] = n;
  __syncthreads();
  plan(row, q, scale, value_of(top), s);
  if (s.total > CAP) {
    if (g == 0) finish_digits(a, r, row, q, scale, top, n, s);
    return;
  }
  // The list passes between workgroups of one launch, on whatever XCD they run: its stores and loads are of device
  // scope, which pass the L2s by, and done before the arrival is counted.  (Plain stores and a fence write
  // back the whole L2 for every workgroup.)
  gather(row, scale, alone ? 0 : g * a.slice, alone ? a.V : min((g + 1) * a.slice, a.V), s);
  if (threadIdx.x == 0) s.found = (int)atomicAdd(w.listed, s.listed);
  __syncthreads();
  for (int i = threadIdx.x; i < (int)s.listed && s.found + i < CAP; i += NT)   // (never past it but where the logits change meanwhile)
    __hip_atomic_store(w.list + s.found + i, s.list[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0)
    s.flag = alone || (int)__hip_atomic_fetch_add(w.arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.slices - 1;
  __syncthreads();
  if (!s.flag) return;
  for (int i = threadIdx.x; i < s.total; i += NT) s.list[i] = __hip_atomic_load(w.list + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  sort_list(s.total, s);
  finish_list(a, r, q, scale, top, n, s);
}

}  // namespace draw
}  // namespace sk
