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
// * a histogram of y (32 buckets per power of two of the weight) with counts and sums
//   tells the few buckets in which the bounds are passed;
// * their values alone are listed and sorted, and the bounds are found in the list by
//   bisection;
// * where those buckets hold more values than the list (thousands of equal logits), the bounds are
//   found digit by digit of the value, three passes over the row for each.
//
// Weights are 2^(t - ref), t = y log2(e) in 64 bits, ref the next whole number above the largest t, as
// whole multiples of 2^-bits: their sums are exact in any order, so results repeat bit for bit
// and do not hang on how a row is cut.  They differ from sums in floating point of 64 bits by
// parts of 1e-11 of the largest weight.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

// Each operation rounds by itself: guidance and quotients are defined so, and a t that enters a bucket
// and a weight is one number.
#pragma clang fp contract(off)

namespace sk {
namespace draw {

constexpr int NT = 1024;                          // threads of a workgroup
constexpr int NB = 1536;                          // buckets: e = ref - t below 48
constexpr int PER_BIT = 32;                       // buckets per power of two
constexpr int CAP = 4096;                         // values of the list
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
struct SliceInfo { double ref; unsigned long long best; int n; int pad; };

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

// One row's values as keys: larger values have larger keys, 0 is no candidate.
template <typename X>
struct Row {
  const X* cond; const X* uncond;
  const uint32_t* allowed;
  float s, T;
  int V;
  __device__ Row(const Args& a, int r) {
    const X* l = static_cast<const X*>(a.logits);
    cond = l + (size_t)(a.cfg ? 2 * (size_t)r : r) * a.stride;
    uncond = a.cfg ? cond + a.stride : nullptr;
    allowed = a.allowed ? a.allowed + (size_t)r * a.allowed_stride : nullptr;
    s = a.cfg ? a.cfg[r] : 0.f;
    T = a.temperature ? a.temperature[r] : 1.f;
    V = a.V;
  }
  __device__ __forceinline__ uint32_t key(int v) const {
    float x = to_f<X>(cond[v]);
    if (uncond) {
      const float u = to_f<X>(uncond[v]);
      x = u + s * (x - u);
    }
    const bool ok = fabsf(x) <= 3.402823466e38f && (!allowed || (allowed[v >> 5] >> (v & 31) & 1u));
    if (T > 0.f) x = fminf(fmaxf(x / T, -3.402823466e38f), 3.402823466e38f);
    return ok ? key_of(x) : 0u;
  }
};

// e = ref - t of a key, and its weight 2^-e in units of 2^-bits, rounded to nearest: e = n + f,
// 2^-f by the exponential series in f ln 2 (|f ln 2| <= 0.347, terms to the 12th: 1e-16).
__device__ __forceinline__ double log2_of(uint32_t key) { return (double)value_of(key) * LOG2E; }
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
// e at most bits + 2, past which a weight is 0
__device__ __forceinline__ unsigned long long weight(double e, int bits) {
  if (!(e <= bits + 2)) return 0;
  const double x = ldexp(power(e), bits) + 0x1p52;   // the sum's last bits are the whole number
  return (unsigned long long)__double_as_longlong(x) & 0xfffffffffffffull;
}
// The bucket of t: whole numbers are compared, so that t has the same one whichever ref it is counted from.
__device__ __forceinline__ int bucket(double ref, double t) {
  const double d = ref * PER_BIT - floor(t * PER_BIT) - 1.0;
  return d >= NB - 1 ? NB - 1 : d > 0.0 ? (int)d : 0;
}
// A value's weight: 0 in the last bucket, which has all that is far below.
__device__ __forceinline__ unsigned long long weight_of(double ref, double t, int b, int bits) {
  return b < NB - 1 ? weight(ref - t, bits) : 0;
}

// The workgroup's shared memory.
struct Shared {
  unsigned long long mass[NB + 1];                // of a bucket, then of all before it
  unsigned long long list[CAP], sum[CAP];
  unsigned count[NB + 1];
  unsigned long long wave64[16];
  unsigned wave32[16];
  unsigned listed;
  int flag;
  struct { int lo, hi, pos; unsigned cp; unsigned long long mp; } range[4];
  int lo[4], hi[4], ranges, total;
  // digit by digit
  struct { unsigned prefix; unsigned cp; unsigned long long mp; unsigned cnt; unsigned long long mass; } at;
};
static_assert(sizeof(unsigned long long) * CAP * 2 >= DIGITS * 12, "digits' histograms lie in the list's place");

template <typename T, typename F>
__device__ __forceinline__ T wave_all(T v, F f) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v = f(v, (T)__shfl_xor(v, o));
  return v;
}
__device__ __forceinline__ unsigned long long wave_incl(unsigned long long v, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const unsigned long long x = __shfl_up(v, o);
    if (lane >= o) v += x;
  }
  return v;
}

// Largest of a value over the workgroup, in every thread.
__device__ __forceinline__ unsigned long long block_max(unsigned long long v, Shared& s) {
  v = wave_all(v, [](unsigned long long a, unsigned long long b) { return a > b ? a : b; });
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s.wave64[threadIdx.x >> 6] = v;
  __syncthreads();
  v = s.wave64[0];
  for (int w = 1; w < NT / 64; ++w) v = s.wave64[w] > v ? s.wave64[w] : v;
  return v;
}
__device__ __forceinline__ unsigned block_sum(unsigned v, Shared& s) {
  v = wave_all(v, [](unsigned a, unsigned b) { return a + b; });
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s.wave32[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
  for (int w = 0; w < NT / 64; ++w) v += s.wave32[w];
  return v;
}
// Exclusive sums of a[0 .. n) in place and the whole at a[n]; n at most 4 NT.
template <typename T>
__device__ __forceinline__ void block_scan(T* a, int n, Shared& s) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int per = (n + NT - 1) / NT, at = tid * per;
  T v[4], mine = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = i < per && at + i < n ? a[at + i] : T(0);
    mine += v[i];
  }
  const unsigned long long incl = wave_incl(mine, lane);
  __syncthreads();
  if (lane == 63) s.wave64[wave] = incl;
  __syncthreads();
  unsigned long long base = 0, all = 0;
  for (int w = 0; w < NT / 64; ++w) {
    if (w < wave) base += s.wave64[w];
    all += s.wave64[w];
  }
  T x = (T)(base + incl) - mine;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i < per && at + i < n) a[at + i] = x;
    x += v[i];
  }
  if (tid == 0) a[n] = (T)all;
  __syncthreads();
}

// The largest key, the lowest id that has it, and how many candidates values v0 .. v1 hold.
template <typename X>
__device__ void survey(const Row<X>& row, int v0, int v1, Shared& s, unsigned long long& best, int& n) {
  unsigned long long b = 0;
  unsigned c = 0;
  for (int v = v0 + threadIdx.x; v < v1; v += NT) {
    const uint32_t k = row.key(v);
    const unsigned long long x = (unsigned long long)k << 32 | (uint32_t)~v;
    if (k) { ++c; b = x > b ? x : b; }
  }
  best = block_max(b, s);
  n = (int)block_sum(c, s);
}
__device__ __forceinline__ double ref_of(unsigned long long best) { return floor(log2_of((uint32_t)(best >> 32))) + 1.0; }

// Counts and sums by bucket of values v0 .. v1 in s.count and s.mass.
template <typename X>
__device__ void histogram(const Row<X>& row, int v0, int v1, double ref, int bits, Shared& s) {
  for (int i = threadIdx.x; i < NB; i += NT) { s.count[i] = 0; s.mass[i] = 0; }
  __syncthreads();
  for (int v = v0 + threadIdx.x; v < v1; v += NT) {
    const uint32_t k = row.key(v);
    if (!k) continue;
    const double t = log2_of(k);
    const int b = bucket(ref, t);
    atomicAdd(&s.count[b], 1u);
    if (b < NB - 1) atomicAdd(&s.mass[b], weight(ref - t, bits));
  }
  __syncthreads();
}

// The parameters of a row as the definitions read them.
struct Params {
  double p, m, u;                                 // p in (0, 1) or 0: none; m in (0, 1] or 0: none
  int k;                                          // 0: none
  bool greedy;
  __device__ Params(const Args& a, int r, int n) {
    const float T = a.temperature ? a.temperature[r] : 1.f;
    greedy = !(T > 0.f);
    k = a.top_k ? a.top_k[r] : 0;
    if (k <= 0 || k >= n) k = 0;
    const float tp = a.top_p ? a.top_p[r] : 0.f, mp = a.min_p ? a.min_p[r] : 0.f;
    p = tp > 0.f && tp < 1.f ? (double)tp : 0.0;
    m = mp > 0.f && mp <= 1.f ? (double)mp : 0.0;
    u = a.u[r];
    u = u > 0.0 ? fmin(u, 1.0) : 0.0;             // NaN and less than 0: 0
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

// The t down to which weights are kept, give (1) or take (-1) rounding.
__device__ __forceinline__ double least_t(double m, double top, double side) {
  return fmin(top + log2(m) + side * (1e-6 + fabs(top) * 0x1p-50), top);
}

// Bucket b with mass[b] <= T < mass[b + 1] (sums of all before).
__device__ int find_mass(const Shared& s, unsigned long long T) {
  int lo = 0, hi = NB - 1;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (s.mass[mid + 1] > T) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}
// Bucket b with count[b] <= c < count[b + 1].
__device__ int find_count(const Shared& s, unsigned c) {
  int lo = 0, hi = NB - 1;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (s.count[mid + 1] > c) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// One thread: the buckets in which the row's bounds are passed, as ranges in s.range; s.total is
// the number of values that they hold.  The whole that top-p takes its part of, and the kept sum that the draw
// takes its part of, are known up to the bucket in which the bound before lies, so theirs may be several.
__device__ void plan(const Params& q, double ref, double top, Shared& s) {
  int (&lo)[4] = s.lo, (&hi)[4] = s.hi, n = 0;    // in shared memory: indexed as the run goes
  unsigned long long w_lo = s.mass[NB], w_hi = s.mass[NB];
  if (q.k) {
    const int b = find_count(s, q.k - 1);
    lo[n] = hi[n] = b; ++n;
    w_lo = s.mass[b]; w_hi = s.mass[b + 1];
  }
  unsigned long long k_lo = w_lo, k_hi = w_hi;    // of the kept sum
  if (q.p > 0.0) {
    lo[n] = find_mass(s, part_of(q.p, w_lo));
    hi[n] = find_mass(s, part_of(q.p, w_hi));
    k_lo = s.mass[lo[n]]; k_hi = s.mass[hi[n] + 1];
    ++n;
  }
  if (q.m > 0.0) {
    lo[n] = bucket(ref, least_t(q.m, top, 1.0)); hi[n] = bucket(ref, least_t(q.m, top, -1.0));
    k_lo = min(k_lo, s.mass[lo[n]]); k_hi = min(k_hi, s.mass[hi[n] + 1]);
    ++n;
  }
  lo[n] = find_mass(s, part_of(q.u, k_lo));
  hi[n] = find_mass(s, part_of(q.u, k_hi));
  ++n;
  for (int i = 1; i < n; ++i)                     // by their first bucket
    for (int j = i; j > 0 && lo[j] < lo[j - 1]; --j) {
      const int a = lo[j], b = hi[j];
      lo[j] = lo[j - 1]; hi[j] = hi[j - 1]; lo[j - 1] = a; hi[j - 1] = b;
    }
  int r = 0;
  for (int i = 1; i < n; ++i) {                   // overlapping ones become one
    if (lo[i] <= hi[r] + 1) hi[r] = max(hi[r], hi[i]);
    else { ++r; lo[r] = lo[i]; hi[r] = hi[i]; }
  }
  unsigned total = 0;
  for (int i = 0; i <= r; ++i) {
    s.range[i].lo = lo[i]; s.range[i].hi = hi[i];
    s.range[i].pos = (int)total;
    s.range[i].cp = s.count[lo[i]]; s.range[i].mp = s.mass[lo[i]];
    total += s.count[hi[i] + 1] - s.count[lo[i]];
  }
  s.ranges = r + 1;
  s.total = (int)total;
}

// Adds the values of v0 .. v1 that lie in the ranges to a list.
template <typename X>
__device__ void gather(const Row<X>& row, int v0, int v1, double ref, const Shared& s, unsigned long long* list, unsigned* listed) {
  const int nr = s.ranges;
  for (int v = v0 + threadIdx.x; v < v1; v += NT) {
    const uint32_t k = row.key(v);
    if (!k) continue;
    const int b = bucket(ref, log2_of(k));
    bool in = false;
    for (int i = 0; i < nr; ++i) in |= b >= s.range[i].lo && b <= s.range[i].hi;
    if (in) {
      const unsigned at = atomicAdd(listed, 1u);
      if (at < CAP) list[at] = (unsigned long long)k << 32 | (uint32_t)~v;
    }
  }
}

// s.list[0 .. n), largest first; n at most CAP.
__device__ void sort_list(int n, Shared& s) {
  int P = 2;
  while (P < n) P <<= 1;
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

__device__ void answer(const Args& a, int r, int token, double logprob, int kept) {
  a.token[r] = token;
  if (a.logprob) a.logprob[r] = (float)logprob;
  if (a.kept) a.kept[r] = kept;
}
// ln of the drawn one's part of the kept sum.
__device__ __forceinline__ double part_log(uint32_t key, double ref, unsigned long long kept, int bits) {
  return (log2_of(key) - ref + bits) * LN2 - log((double)kept);
}

// The row's answer from the sorted list of its ranges.
__device__ void finish_list(const Args& a, int r, const Params& q, double ref, unsigned long long best, int n, Shared& s) {
  const int total = s.total;
  for (int i = threadIdx.x; i < total; i += NT) {
    const double t = log2_of((uint32_t)(s.list[i] >> 32));
    s.sum[i] = weight_of(ref, t, bucket(ref, t), a.bits);
  }
  __syncthreads();
  // sums up to and with each: four to a thread
  {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    unsigned long long v[CAP / NT], mine = 0;
#pragma unroll
    for (int i = 0; i < CAP / NT; ++i) {
      const int at = tid * (CAP / NT) + i;
      v[i] = at < total ? s.sum[at] : 0;
      mine += v[i];
    }
    const unsigned long long incl = wave_incl(mine, lane);
    __syncthreads();
    if (lane == 63) s.wave64[wave] = incl;
    __syncthreads();
    unsigned long long x = incl - mine;
    for (int w = 0; w < wave; ++w) x += s.wave64[w];
#pragma unroll
    for (int i = 0; i < CAP / NT; ++i) {
      const int at = tid * (CAP / NT) + i;
      x += v[i];
      if (at < total) s.sum[at] = x;
    }
  }
  __syncthreads();
  if (threadIdx.x) return;
  const uint32_t top = (uint32_t)(best >> 32);
  auto end_of = [&](int i) { return i + 1 < s.ranges ? s.range[i + 1].pos : total; };
  // sum of all up to and with list entry i of range g
  auto upto = [&](int g, int i) {
    const int p = s.range[g].pos;
    return s.range[g].mp + s.sum[i] - (p ? s.sum[p - 1] : 0);
  };
  // first entry of range g for which `past` holds (it holds from some entry on), or its end
  auto first = [&](int g, auto past) {
    int lo = s.range[g].pos, hi = end_of(g);
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (past(mid)) hi = mid;
      else lo = mid + 1;
    }
    return lo;
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
  unsigned long long sum = s.mass[NB];
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
    const int b = bucket(ref, least_t(q.m, log2_of(top), 1.0));
    int g = 0;
    while (g + 1 < s.ranges && s.range[g + 1].lo <= b) ++g;
    unsigned c;
    unsigned long long w;
    before(g, first(g, [&](int i) { return !heavy((uint32_t)(s.list[i] >> 32), top, q.m); }), c, w);
    if (c < kept) { kept = c; sum = w; }
  }
  const unsigned long long T = part_of(q.u, sum);
  const int g = range_of_mass(T);
  int i = min(first(g, [&](int i) { return upto(g, i) > T; }), end_of(g) - 1);
  const uint32_t key = (uint32_t)(s.list[i] >> 32);
  answer(a, r, (int)~(uint32_t)s.list[i], part_log(key, ref, sum, a.bits), (int)kept);
}

// Digit by digit: the value at which the count of the largest (by_count) or their sum passes T, in
// s.at: its key, the count and sum of all above it, and its own.
template <typename X>
__device__ void descend(const Row<X>& row, double ref, int bits, bool by_count, unsigned long long T, Shared& s) {
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
      const bool on = k && (k & mask) == prefix;
      const int d = digits - 1 - (int)(k >> shift & (digits - 1));
      unsigned long long w = 0;
      if (on) {
        const double t = log2_of(k);
        w = weight_of(ref, t, bucket(ref, t), bits);
      }
      // where a wave's values all have one digit, as equal logits do, one lane adds for all
      const unsigned long long who = __ballot(on);
      if (!who) continue;
      const int d0 = __builtin_amdgcn_readlane(d, __builtin_ctzll(who));
      if (__ballot(on && d == d0) == who) {
        w = wave_all(w, [](unsigned long long x, unsigned long long y) { return x + y; });
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
    block_scan(mass, digits, s);
    block_scan(count, digits, s);
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

// The row's answer where the list does not hold its ranges.
template <typename X>
__device__ void finish_digits(const Args& a, int r, const Row<X>& row, const Params& q, double ref, unsigned long long best,
                              int n, Shared& s) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  unsigned kept = (unsigned)n;
  unsigned long long sum = s.mass[NB];
  if (q.k) {
    descend(row, ref, a.bits, true, q.k - 1, s);
    kept = s.at.cp + s.at.cnt;
    sum = s.at.mp + s.at.mass;
  }
  if (q.p > 0.0) {
    const unsigned long long T = part_of(q.p, sum);
    __syncthreads();
    descend(row, ref, a.bits, false, T, s);
    // of the equal values so many that the sum passes T
    const unsigned long long w = s.at.cnt ? s.at.mass / s.at.cnt : 0;
    unsigned c = w ? (unsigned)min((T - s.at.mp) / w + 1, (unsigned long long)s.at.cnt) : s.at.cnt;
    if (s.at.cp + c < kept) { kept = s.at.cp + c; sum = s.at.mp + c * w; }
  }
  if (q.m > 0.0) {
    unsigned c = 0;
    unsigned long long w = 0;
    for (int v = tid; v < row.V; v += NT) {
      const uint32_t k = row.key(v);
      if (k && heavy(k, (uint32_t)(best >> 32), q.m)) {
        const double t = log2_of(k);
        ++c;
        w += weight_of(ref, t, bucket(ref, t), a.bits);
      }
    }
    c = block_sum(c, s);
    w = wave_all(w, [](unsigned long long x, unsigned long long y) { return x + y; });
    __syncthreads();
    if (lane == 0) s.wave64[wave] = w;
    __syncthreads();
    w = 0;
    for (int i = 0; i < NT / 64; ++i) w += s.wave64[i];
    if (c < kept) { kept = c; sum = w; }
  }
  const unsigned long long T = part_of(q.u, sum);
  __syncthreads();
  descend(row, ref, a.bits, false, T, s);
  const uint32_t key = s.at.prefix;
  const unsigned long long w = s.at.cnt ? s.at.mass / s.at.cnt : 0;
  const unsigned long long nth = w ? (T - s.at.mp) / w : 0;   // from 0, among the equal ones by id
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
      if (is && mine == nth) answer(a, r, v, part_log(key, ref, sum, a.bits), (int)kept);
      ahead += (unsigned)__popcll(who);
    }
  }
}

// A row that needs no sums: greedy, or without candidates.
__device__ bool finish_early(const Args& a, int r, const Params& q, unsigned long long best, int n) {
  if (n && !q.greedy) return false;
  if (threadIdx.x == 0) answer(a, r, n ? (int)~(uint32_t)best : -1, n ? 0.0 : -INFINITY, n ? 1 : 0);
  return true;
}

// A whole row in one workgroup.
template <typename X>
__global__ __launch_bounds__(NT) void row_kernel(Args a) {
  __shared__ Shared s;
  const int r = blockIdx.x;
  const Row<X> row(a, r);
  unsigned long long best;
  int n;
  survey(row, 0, a.V, s, best, n);
  const Params q(a, r, n);
  if (finish_early(a, r, q, best, n)) return;
  const double ref = ref_of(best);
  histogram(row, 0, a.V, ref, a.bits, s);
  block_scan(s.mass, NB, s);
  block_scan(s.count, NB, s);
  if (threadIdx.x == 0) {
    plan(q, ref, log2_of((uint32_t)(best >> 32)), s);
    s.listed = 0;
  }
  __syncthreads();
  if (s.total > CAP) {
    finish_digits(a, r, row, q, ref, best, n, s);
    return;
  }
  gather(row, 0, a.V, ref, s, s.list, &s.listed);
  __syncthreads();
  sort_list(s.total, s);
  finish_list(a, r, q, ref, best, n, s);
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
  __device__ RowSpace(const Args& a, int r) {
    char* p = a.ws + r * bytes(a.slices);
    info = reinterpret_cast<SliceInfo*>(p); p += a.slices * sizeof(SliceInfo);
    mass = reinterpret_cast<unsigned long long*>(p); p += (size_t)a.slices * NB * 8;
    list = reinterpret_cast<unsigned long long*>(p); p += CAP * 8;
    count = reinterpret_cast<unsigned*>(p); p += (size_t)a.slices * NB * 4;
    listed = reinterpret_cast<unsigned*>(p);
    arrived = listed + 1;
  }
};

template <typename X>
__global__ __launch_bounds__(NT) void slice_kernel(Args a) {
  __shared__ Shared s;
  const int r = blockIdx.y, g = blockIdx.x;
  const Row<X> row(a, r);
  const RowSpace w(a, r);
  const int v0 = g * a.slice, v1 = min(v0 + a.slice, a.V);
  unsigned long long best;
  int n;
  survey(row, v0, v1, s, best, n);
  const double ref = n ? ref_of(best) : 0.0;
  if (threadIdx.x == 0) {
    w.info[g] = {ref, best, n, 0};
    if (g == 0) { *w.listed = 0; *w.arrived = 0; }
  }
  if (n == 0 || !(row.T > 0.f)) return;           // nothing of it is read
  histogram(row, v0, v1, ref, a.bits, s);
  for (int i = threadIdx.x; i < NB; i += NT) {
    w.count[(size_t)g * NB + i] = s.count[i];
    w.mass[(size_t)g * NB + i] = s.mass[i];
  }
}

template <typename X>
__global__ __launch_bounds__(NT) void pick_kernel(Args a) {
  __shared__ Shared s;
  const int r = blockIdx.y, g = blockIdx.x;
  const Row<X> row(a, r);
  const RowSpace w(a, r);
  unsigned long long best = 0;
  int n = 0;
  for (int i = 0; i < a.slices; ++i) {
    const SliceInfo f = w.info[i];
    best = f.best > best ? f.best : best;
    n += f.n;
  }
  const Params q(a, r, n);
  if (n == 0 || q.greedy) {
    if (g == 0) finish_early(a, r, q, best, n);
    return;
  }
  const double ref = ref_of(best), top = log2_of((uint32_t)(best >> 32));
  // Past 2^40 the slices' refs need not be whole numbers apart: one workgroup takes the row.
  const bool alone = !(fabs(ref) < 0x1p40);
  if (alone && g) return;
  if (alone) {
    histogram(row, 0, a.V, ref, a.bits, s);
  } else {
    for (int b = threadIdx.x; b < NB; b += NT) {
      unsigned c = 0;
      unsigned long long m = 0;
      for (int i = 0; i < a.slices; ++i) {
        const SliceInfo f = w.info[i];
        const double up = ref - f.ref;            // a whole number
        if (!f.n || up >= NB / PER_BIT) continue;
        const int at = b - (int)up * PER_BIT;
        if (at >= 0 && b < NB - 1) {
          c += w.count[(size_t)i * NB + at];
          m += w.mass[(size_t)i * NB + at] >> (int)up;
        }
      }
      s.count[b] = c;
      s.mass[b] = m;
    }
    __syncthreads();
  }
  block_scan(s.mass, NB, s);
  block_scan(s.count, NB, s);
  if (threadIdx.x == 0) {
    s.count[NB] = n;                              // the last bucket has the rest
    plan(q, ref, top, s);
  }
  __syncthreads();
  if (s.total > CAP) {
    if (g == 0) finish_digits(a, r, row, q, ref, best, n, s);
    return;
  }
  gather(row, alone ? 0 : g * a.slice, alone ? a.V : min((g + 1) * a.slice, a.V), ref, s, w.list, w.listed);
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0)
    s.flag = alone || (int)__hip_atomic_fetch_add(w.arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.slices - 1;
  __syncthreads();
  if (!s.flag) return;
  __threadfence();
  for (int i = threadIdx.x; i < s.total; i += NT) s.list[i] = w.list[i];
  sort_list(s.total, s);
  finish_list(a, r, q, ref, best, n, s);
}

}  // namespace draw
}  // namespace sk
