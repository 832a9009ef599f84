// The attention half of a trunk layer over a cache in pages.
//
// K and V lie in a pool of pages [n_pages][Hkv][page][hd] (the engine's cache
// is one page of max_ctx tokens per row); sequence s has the pages table[s][0 ..
// width), slot j of it in page j / page.  Its n new tokens of a call are the
// packed rows starts[s] .. starts[s + 1] of q, and lens[s] is its length with
// them, so token i has slot lens[s] - n + i.  Query heads h G .. h G + G - 1 share key
// head h.  A page is a multiple of 16 tokens: 16 keys of one tile lie in one
// page, one look into the table serves a tile, and a tile is loaded whole (its
// slots past the length are memory of the pool).
//
// starts, lens and table are device memory that the host does not look at, so the
// kernels hold them in range: starts to [0, T] and not falling, lens to [0,
// width * page], and an entry outside the pool reads page 0 with its keys counted as
// NaN, so that rows that see it come out as NaN.  A sequence whose length is past its table has
// no place for all of its tokens: none is stored, and all of its pages count as outside the pool.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "sk_lds.h"

namespace sk {
namespace paged {

typedef float v4f __attribute__((ext_vector_type(4)));

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
constexpr int TILE = 16;                          // keys of a tile

struct Cache {
  void* k; void* v;                               // [n_pages][Hkv][page][hd]
  const int* table; int64_t stride; int width;    // [S][width] at rows of stride entries
  const int* starts; const int* lens;             // [S + 1], [S]
  int T, S, Hq, Hkv, G, n_pages, page;
  uint32_t page_mul; int page_shift;              // j / page = j * page_mul >> page_shift for 0 <= j < 2^31
};

// ------------------------------------------------------------ small helpers
template <int CTRL>
__device__ __forceinline__ float dpp_f(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
// Sum over 2, 4, 8 or 16 neighbouring lanes, in every one of them.
template <int N>
__device__ __forceinline__ float group_sum(float v) {
  v += dpp_f<0xb1>(v);                            // quad_perm [1,0,3,2]
  if constexpr (N >= 4) v += dpp_f<0x4e>(v);      // quad_perm [2,3,0,1]
  if constexpr (N >= 8) v += dpp_f<0x141>(v);     // row_half_mirror
  if constexpr (N >= 16) v += dpp_f<0x140>(v);    // row_mirror
  return v;
}
// Over lanes l, l ^ 16, l ^ 32 and l ^ 48 (the four that share a row or key of a
// matrix tile), in every one of them: two exchanges in registers.
template <typename F>
__device__ __forceinline__ float fold4(float v, F f) {
  const int x = __float_as_int(v);
  const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  const int y = __float_as_int(f(__int_as_float(a[0]), __int_as_float(a[1])));
  const auto b = __builtin_amdgcn_permlane32_swap(y, y, false, false);
  return f(__int_as_float(b[0]), __int_as_float(b[1]));
}
template <typename F>
__device__ __forceinline__ float fold2(float v, F f) {   // lanes l and l ^ 32
  const int x = __float_as_int(v);
  const auto a = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return f(__int_as_float(a[0]), __int_as_float(a[1]));
}
__device__ __forceinline__ float sum2(float v) { return fold2(v, [](float a, float b) { return a + b; }); }
__device__ __forceinline__ float max2(float v) { return fold2(v, [](float a, float b) { return fmaxf(a, b); }); }
__device__ __forceinline__ float sum4(float v) { return fold4(v, [](float a, float b) { return a + b; }); }
__device__ __forceinline__ float max4(float v) { return fold4(v, [](float a, float b) { return fmaxf(a, b); }); }

__device__ __forceinline__ uint16_t to_bf16(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }   // to nearest even

// N consecutive elements as loaded; get(i) widens one.
template <typename T, int N>
struct Piece {
  uint32_t w[(N * sizeof(T) + 3) / 4];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (N * sizeof(T) > 16) {
#pragma unroll
      for (int i = 0; i < N * (int)sizeof(T) / 16; ++i) {
        const uint4 v = reinterpret_cast<const uint4*>(p)[i];
        w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
      }
    } else if constexpr (N * sizeof(T) == 16) {
      const uint4 v = *reinterpret_cast<const uint4*>(p);
      w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else if constexpr (N * sizeof(T) == 8) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      w[0] = v.x; w[1] = v.y;
    } else if constexpr (N * sizeof(T) == 4) {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
      w[0] = *reinterpret_cast<const uint16_t*>(p);
    }
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
    else return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (auto& x : w) x = 0;
  }
  // infinities and NaN to 0; whether there were any
  __device__ __forceinline__ bool tame() {
    bool b = false;
#pragma unroll
    for (uint32_t& x : w) {
      const bool hi = (x & 0x7f800000u) == 0x7f800000u, lo = sizeof(T) == 2 && (x & 0x7f80u) == 0x7f80u;
      b |= hi || lo;
      if (hi) x = sizeof(T) == 4 ? 0u : x & 0xffffu;
      if (lo) x &= 0xffff0000u;
    }
    return b;
  }
};
template <typename T>
__device__ __forceinline__ void store4(T* p, float a, float b, float c, float d) {
  if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
  else *reinterpret_cast<uint2*>(p) = make_uint2(to_bf16(a) | (uint32_t)to_bf16(b) << 16, to_bf16(c) | (uint32_t)to_bf16(d) << 16);
}

// First row and number of sequence s's new tokens.
__device__ __forceinline__ void seq_rows(const Cache& c, int s, int& first, int& n) {
  first = min(max(c.starts[s], 0), c.T);
  n = min(max(c.starts[s + 1], first), c.T) - first;
}
__device__ __forceinline__ int page_of(const Cache& c, int j) {
  return (int)(__umulhi((uint32_t)j, c.page_mul) >> (c.page_shift - 32));
}
__device__ __forceinline__ int seq_len(const Cache& c, int s) { return min(max(c.lens[s], 0), c.width * c.page); }
__device__ __forceinline__ bool too_long(const Cache& c, int s) { return c.lens[s] > c.width * c.page; }

// The sequence that row m belongs to (wave-uniform; S if none): the last one that starts at or before it.
__device__ __forceinline__ int seq_of_row(const Cache& c, int m) {
  int count = 0;
  for (int s0 = 0; s0 < c.S; s0 += 64) {
    const int s = s0 + (threadIdx.x & 63);
    count += __popcll(__ballot(s < c.S && c.starts[min(s, c.S)] <= m));
  }
  if (count == 0) return c.S;
  return m < c.starts[count] ? count - 1 : c.S;
}

// Inclusive sum over a wave's lanes.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);    // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);    // row_shr:2
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);    // row_shr:4
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);    // row_shr:8
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);   // row_bcast:15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);   // row_bcast:31 into rows 2 and 3
  return v;
}

// Tile x of all sequences' tiles of R (token, head of the group) rows: its sequence, its number
// there, the sequence's first row, new tokens and the slot of the first (slot), and the pool's pages that count
// (none for a length past the table, whose tokens take the last slots, all of them seen); false past the last.
// Every lane brings one sequence's numbers, in one trip to memory.
struct TileAt {
  int seq, tile, first, n, p0, n_pages;
  __device__ __forceinline__ int slot(const Cache& c, int tok) const { return min(p0 + tok, c.width * c.page - 1); }
};
__device__ __forceinline__ bool find_tile(const Cache& c, int R, int x, TileAt& at) {
  const int lane = threadIdx.x & 63;
  int base = 0;
  for (int s0 = 0; s0 < c.S; s0 += 64) {
    const int s = min(s0 + lane, c.S - 1);
    int first, n;
    seq_rows(c, s, first, n);
    const bool over = too_long(c, s);
    const int p0 = over ? max(c.width * c.page - n, 0) : seq_len(c, s) - n;
    const int t = s0 + lane < c.S ? (n * c.G + R - 1) / R : 0, sum = wave_scan(t);
    const uint64_t past = __ballot(base + sum > x), none = __ballot(over);
    if (past) {
      const int l = __builtin_ctzll(past);
      at.seq = s0 + l;
      at.tile = x - base - (__builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(t, l));
      at.first = __builtin_amdgcn_readlane(first, l);
      at.n = __builtin_amdgcn_readlane(n, l);
      at.p0 = __builtin_amdgcn_readlane(p0, l);
      at.n_pages = none >> l & 1 ? 0 : c.n_pages;
      return true;
    }
    base += __builtin_amdgcn_readlane(sum, 63);
  }
  return false;
}

// ------------------------------------------------------------ append
// Token m: q and k of every head normalised over the head (RMSNorm with a gain,
// if there are gains), then rotated: pair (i, i + hd / 2) by the angle position
// * inv_freq[i]; q to its row, k and v to the token's slot, whose account of
// attention weight starts at 0.  One workgroup per token, hd / 8 lanes per
// head with four pairs each, so that every load and store is 16 bytes (8 of BF16).
//
// The angle is formed and brought into [-pi, pi] in 64 bits (in 32 a product
// of 2^17 is off by 2^-7), then cos(r + e) = cos r - e sin r with r its nearest FP32
// and e the rest; one lane per pair, shared through LDS.
//
// Bound by bytes: 5,760 tokens of 16 + 2 x 8 heads of 128, FP32 into BF16 with accounts, 165 MB in
// 28.8 us (5.7 TB/s, part of it from the last-level cache).  32 tokens take 3.8 us, three trips to
// memory (starts, the table, the store) beside the angle.
template <typename XT, typename KT, int HD>
__global__ __launch_bounds__(256) void append_kernel(Cache c, const XT* qkv, const float* q_gain, const float* k_gain,
                                                     const float* inv_freq, const int* positions, float eps,
                                                     float* mass, XT* q_out) {
  constexpr int LPH = HD / 8, NG = 256 / LPH, HALF = HD / 2;
  __shared__ float2 cs[HALF];
  const int m = blockIdx.x, tid = threadIdx.x, g = tid / LPH, i = (tid % LPH) * 4;
  const int H = c.Hq + 2 * c.Hkv;
  const XT* row = qkv + (size_t)m * H * HD + i;
  Piece<XT, 4> a, b;
  if (g < H) { a.load(row + (size_t)g * HD); b.load(row + (size_t)g * HD + HALF); }
  if (tid < HALF) {
    constexpr double TWO_PI = 6.283185307179586476925286766559;
    const double t = (double)positions[m] * (double)inv_freq[tid];
    const double w = t - rint(t / TWO_PI) * TWO_PI;
    const float r = (float)w, e = (float)(w - (double)r), co = cosf(r), si = sinf(r);
    cs[tid] = make_float2(fmaf(-e, si, co), fmaf(e, co, si));
  }
  const int s = seq_of_row(c, m);
  if (s >= c.S) return;                           // behind the last sequence (the whole workgroup)
  int first, n;
  seq_rows(c, s, first, n);
  const int slot = seq_len(c, s) - n + (m - first);
  int at = -1;                                    // the slot's page, if it has one
  const int pg = page_of(c, max(slot, 0));
  if (slot >= 0 && m - first < n) at = c.table[s * c.stride + pg];
  const bool live = at >= 0 && at < c.n_pages && !too_long(c, s);
  const size_t base = live ? (size_t)at * c.Hkv * c.page + (slot - pg * c.page) : 0;   // in rows of hd, for head 0
  __syncthreads();
  float2 t4[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) t4[u] = cs[i + u];
  for (int h = g; h < H; h += NG) {
    if (h != g) { a.load(row + (size_t)h * HD); b.load(row + (size_t)h * HD + HALF); }
    float y1[4], y2[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) { y1[u] = a.get(u); y2[u] = b.get(u); }
    if (h < c.Hq + c.Hkv) {
      const float* gain = h < c.Hq ? q_gain : k_gain;
      if (gain) {
        float ss = 0.f;
#pragma unroll
        for (int u = 0; u < 4; ++u) ss = fmaf(y1[u], y1[u], fmaf(y2[u], y2[u], ss));
        const float inv = 1.0f / sqrtf(group_sum<LPH>(ss) / (float)HD + eps);
        const float4 g1 = *reinterpret_cast<const float4*>(gain + i), g2 = *reinterpret_cast<const float4*>(gain + i + HALF);
        y1[0] = g1.x * (y1[0] * inv); y1[1] = g1.y * (y1[1] * inv); y1[2] = g1.z * (y1[2] * inv); y1[3] = g1.w * (y1[3] * inv);
        y2[0] = g2.x * (y2[0] * inv); y2[1] = g2.y * (y2[1] * inv); y2[2] = g2.z * (y2[2] * inv); y2[3] = g2.w * (y2[3] * inv);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float p = y1[u], q = y2[u];
        y1[u] = p * t4[u].x - q * t4[u].y;
        y2[u] = q * t4[u].x + p * t4[u].y;
      }
    }
    if (h < c.Hq) {
      XT* d = q_out + ((size_t)m * c.Hq + h) * HD + i;
      store4(d, y1[0], y1[1], y1[2], y1[3]);
      store4(d + HALF, y2[0], y2[1], y2[2], y2[3]);
    } else if (live) {
      const bool isk = h < c.Hq + c.Hkv;
      const size_t r = base + (size_t)(h - c.Hq - (isk ? 0 : c.Hkv)) * c.page;
      KT* d = static_cast<KT*>(isk ? c.k : c.v) + r * HD + i;
      store4(d, y1[0], y1[1], y1[2], y1[3]);
      store4(d + HALF, y2[0], y2[1], y2[2], y2[3]);
      if (isk && mass && i == 0) mass[r] = 0.f;
    }
  }
}

// ------------------------------------------------------------ attention
// Rows are (token, head of the group) pairs, token by token: row f of a sequence
// is token f / G, head f % G, so any group size fills the matrix tiles.  Row
// at slot p sees key j when j <= p and, with a window, j > p - window or j < sinks.
//   s_j = scale q . k_j;  m = max s_j;  l = sum exp(s_j - m);  out = sum exp(s_j - m) v_j / l
//   lse = m + ln l
// in one pass with a running m (of the raw q . k_j, scale > 0), l and out; a key
// range cut over workgroups leaves (out, m, l) per cut, joined by combine_kernel.
// A row that sees nothing gives 0 and -infinity.
struct AttendArgs {
  Cache c;
  const void* q; void* out; float* lse;           // [T][Hq][hd], [T][Hq] (may be null)
  float scale2;                                   // scale * log2 e: exp(s - m) = 2^(scale2 (qk - max qk))
  int window, sinks;                              // window 0: all keys
  int cut;                                        // tiles of keys per cut; cuts of a row: blockIdx.z
  int last;                                       // the last row tile of the launch: the others follow down from it
  float* part; float* ml;                         // [cuts][T * Hq][hd], [cuts][T * Hq][2]: sums of V, (maximum times scale2, sum)
  int* count;                                     // [T * Hq]: a row's cuts to join (0: none), negative if it sees nothing
};
constexpr float LOWEST = -3e38f;                  // a maximum of nothing: finite, so that -infinity less it is -infinity

// The tiles that the rows of slots p_lo .. p_hi walk: 0 .. n - 1, first those of the sinks, then the window's.
struct Walk {
  int n, sink, skip;
  __device__ __forceinline__ int tile(int t) const { return t < sink ? t : t + skip; }
};
__device__ __forceinline__ Walk walk_of(int p_lo, int p_hi, int window, int sinks) {
  Walk w;
  const int lo = window > 0 && p_lo >= window ? (p_lo - window + 1) / TILE : 0;
  w.sink = min(sinks / TILE + (sinks % TILE != 0), lo);
  w.skip = lo - w.sink;
  w.n = p_hi < 0 ? 0 : p_hi / TILE + 1 - w.skip;
  return w;
}
__device__ __forceinline__ bool sees(int p, int j, int window, int sinks) {
  return j <= p && (window == 0 || j > p - window || j < sinks);
}
// whether every row of slots p_lo .. p_hi sees every key j0 .. j1
__device__ __forceinline__ bool all_see(int j0, int j1, int p_lo, int p_hi, int window, int sinks) {
  return j1 <= p_lo && (window == 0 || j0 > p_hi - window || j1 < sinks);
}

// The factor from sums that refer to the maximum m to ones for m2.  Weights refer to m scale2 as rounded, so that
// is what counts here too: fused, the product would be off from it by half a step of an exponent that may be large.
__device__ __forceinline__ float rescale_of(float m, float scale2, float m2) {
#pragma clang fp contract(off)
  const float was = m * scale2;
  return __builtin_amdgcn_exp2f(was - m2);
}

__device__ __forceinline__ int cuts_of(const AttendArgs& a, const Walk& w, bool none) {
  const int ns = w.n <= a.cut ? 0 : (w.n + a.cut - 1) / a.cut;
  return none ? -ns : ns;
}

// Offsets (in elements, for head 0 dims) of a run of tiles: lane i holds that of
// the wave's i-th tile from a walk position on; one division and table entry per lane, for 64 tiles.
struct TileOffsets {
  uint32_t lo, hi;
  uint64_t bad;                                   // lanes whose page is not in the pool
  // tiles t0, t0 + step ..; as pairs: t0, t0 + 1, t0 + step, t0 + step + 1 ..
  __device__ __forceinline__ void load(const Cache& c, int n_pages, const int* table, const Walk& w, int t0, int step,
                                       int end, int h, int hd, bool pairs = false) {
    const int l = threadIdx.x & 63, t = min(t0 + (pairs ? (l >> 1) * step + (l & 1) : l * step), end - 1);
    const int j = w.tile(t) * TILE, pg = page_of(c, j);
    const int e = table[pg];
    const bool ok = e >= 0 && e < n_pages;
    const size_t off = (((size_t)(ok ? e : 0) * c.Hkv + h) * c.page + (j - pg * c.page)) * hd;
    lo = (uint32_t)off;
    hi = (uint32_t)(off >> 32);
    bad = __ballot(!ok);
  }
  __device__ __forceinline__ size_t at(int i) const {
    return (size_t)(uint32_t)__builtin_amdgcn_readlane(lo, i) | (size_t)(uint32_t)__builtin_amdgcn_readlane(hi, i) << 32;
  }
};

template <typename KT, int HD>
struct Dims {
  static constexpr int KW = (16 / (int)sizeof(KT)) < HD / 4 ? 16 / (int)sizeof(KT) : HD / 4;   // dims per K load
  static constexpr int NK = HD / (4 * KW);                                                     // K loads per tile
  static constexpr int NDT = HD / 16;                                                          // 16-dim output tiles
  static constexpr int VW = (16 / (int)sizeof(KT)) < NDT ? 16 / (int)sizeof(KT) : NDT;         // dims per V load
  static constexpr int NV = NDT / VW;                                                          // V loads per key row
  static constexpr int LDO = HD + 4;                                                           // merge row stride
};

// V of a key that a row does not see must not reach it, but a matrix product
// takes 0 times infinity or NaN for NaN.  So where a tile is seen by some rows only, the
// loops take such elements of V as 0, and this adds them afterwards, element by element, to the
// rows that do see them, in the output (or the cut's part) already stored: rare, and slow.
// Rows f_lo .. f_hi of the sequence by one wave; tiles begin .. end for which tamed(t); stat(f):
// the row's maximum (times scale2) and the factor of its sums.
template <typename QT, typename KT, int HD, typename Tamed, typename Stat>
__device__ __forceinline__ void add_wild(const AttendArgs& a, int h, const int* table, int first, int p0, int f_lo,
                                         int f_hi, const Walk& w, int begin, int end, float* part, Tamed tamed,
                                         Stat stat) {
  constexpr int E = HD >= 64 ? HD / 64 : 1;
  const Cache& c = a.c;
  const int lane = threadIdx.x & 63, d = min(lane, HD / E - 1) * E;
  const bool live = lane * E < HD;
  for (int t = begin; t < end; ++t) {
    const int k0 = w.tile(t) * TILE, e = table[k0 / c.page];
    if (!tamed(t) || e < 0 || e >= c.n_pages) continue;
    for (int key = k0; key < k0 + TILE; ++key) {
      const size_t at = (((size_t)e * c.Hkv + h) * c.page + key % c.page) * HD + d;
      Piece<KT, E> v;
      v.load(static_cast<const KT*>(c.v) + at);
      Piece<KT, E> x = v;
      const bool odd = x.tame() && live;
      if (!__any(odd)) continue;
      Piece<KT, E> k;
      k.load(static_cast<const KT*>(c.k) + at);
      for (int f = f_lo; f < f_hi; ++f) {
        const int tok = f / c.G;
        if (!sees(p0 + tok, key, a.window, a.sinks)) continue;
        const size_t row = (size_t)(first + tok) * c.Hq + h * c.G + (f - tok * c.G);
        Piece<QT, E> q;
        q.load(static_cast<const QT*>(a.q) + row * HD + d);
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) s = live ? fmaf(q.get(i), k.get(i), s) : 0.f;
#pragma unroll
        for (int i = 1; i < 64; i *= 2) s += __shfl_xor(s, i, 64);
        const float2 st = stat(f);
        const float p = __builtin_amdgcn_exp2f(fmaf(s, a.scale2, -st.x)) * st.y;
#pragma unroll
        for (int i = 0; i < E; ++i)
          if (odd && x.get(i) != v.get(i)) {      // the elements that were taken as 0
            if (part) {
              part[row * HD + d + i] += p * v.get(i);
            } else if constexpr (sizeof(QT) == 4) {
              static_cast<QT*>(a.out)[row * HD + d + i] += p * v.get(i);
            } else {
              QT* y = static_cast<QT*>(a.out) + row * HD + d + i;
              *y = to_bf16(__uint_as_float((uint32_t)*y << 16) + p * v.get(i));
            }
          }
      }
    }
  }
}

// The end of a workgroup whose WK waves shared R rows' keys: each wave's sums of V are in po [WK][R][HD
// + 4], maxima (of the raw products) and sums in pm, pl [WK][R].  Joins them, stores rows (or the cut's part)
// and adds what V's infinities and NaN left out.
template <typename QT, typename KT, int HD, int R, int WK>
__device__ __forceinline__ void meet_rows(const AttendArgs& a, const float* po, float* pm, const float* pl, float2* stats,
                                          bool wild, int h, int cut, const int* table, int first, int p0, int f0, int rows,
                                          int p_lo, int p_hi, const Walk& w, int end) {
  constexpr int LDO = HD + 4;
  const Cache& c = a.c;
  const int tid = threadIdx.x;
  __syncthreads();
  const bool alone = w.n <= a.cut;                // no other cut: the answer itself
  if (tid < R) {
    float mx = -INFINITY, l = 0.f, f[WK];
#pragma unroll
    for (int u = 0; u < WK; ++u) mx = fmaxf(mx, pm[u * R + tid]);
    const float m2 = mx == -INFINITY ? LOWEST : mx * a.scale2;
#pragma unroll
    for (int u = 0; u < WK; ++u) {
      f[u] = rescale_of(pm[u * R + tid], a.scale2, m2);
      l = fmaf(f[u], pl[u * R + tid], l);
    }
    const int row = f0 + tid, tok = row / c.G;
    const bool none = p0 + tok < 0;               // no key is seen
#pragma unroll
    for (int u = 0; u < WK; ++u) pm[u * R + tid] = alone ? none ? 0.f : f[u] / l : f[u];
    stats[tid] = make_float2(m2, alone ? 1.f / l : 1.f);
    if (row < rows) {
      const size_t at = (size_t)(first + tok) * c.Hq + h * c.G + (row - tok * c.G);
      if (cut == 0 && a.count) a.count[at] = cuts_of(a, w, none);
      if (!alone) {
        float* d = a.ml + ((size_t)cut * c.T * c.Hq + at) * 2;
        d[0] = m2;
        d[1] = l;
      } else if (a.lse) {
        a.lse[at] = none ? -INFINITY : (m2 + log2f(l)) * LN2;
      }
    }
  }
  __syncthreads();
  constexpr int NF = HD / 4;
  for (int it = tid; it < R * NF; it += WK * 64) {
    const int r = it / NF, d = (it - r * NF) * 4, row = f0 + r, tok = row / c.G;
    if (row >= rows) break;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int u = 0; u < WK; ++u) {
      const float wt = pm[u * R + r];
      const float4 x = *reinterpret_cast<const float4*>(po + (u * R + r) * LDO + d);
      y.x = fmaf(wt, x.x, y.x); y.y = fmaf(wt, x.y, y.y); y.z = fmaf(wt, x.z, y.z); y.w = fmaf(wt, x.w, y.w);
    }
    const size_t at = (size_t)(first + tok) * c.Hq + h * c.G + (row - tok * c.G);
    if (alone) store4(static_cast<QT*>(a.out) + at * HD + d, y.x, y.y, y.z, y.w);
    else *reinterpret_cast<float4*>(a.part + ((size_t)cut * c.T * c.Hq + at) * HD + d) = y;
  }
  if (__syncthreads_or(wild) && tid < 64)
    add_wild<QT, KT, HD>(a, h, table, first, p0, f0, min(f0 + R, rows), w, cut * a.cut, end,
                         alone ? nullptr : a.part + (size_t)cut * c.T * c.Hq * HD,
                         [&](int t) { const int k0 = w.tile(t) * TILE;
                                      return !all_see(k0, k0 + TILE - 1, p_lo, p_hi, a.window, a.sinks); },
                         [&](int f) { return stats[f - f0]; });
}

// The workgroup holds NT matrix tiles of 16 rows; its WK waves take key tiles in
// turn, each with its own running maximum, and meet in LDS at the end.  No LDS and no barrier in the loop:
//   S^T = K Q^T on the FP32 matrix cores: lane l holds row l % 16's products with
//     keys 4 (l / 16) + v, v < 4; a row's maximum is 4 values and two exchanges;
//   O^T += V^T P^T takes those values as they are: step v multiplies keys 4 q + v, q = 0 .. 3.
// K and V come straight from the pages, 16 bytes per lane; K of the next tile loads under this one's softmax and V.
// Two rows of 240 and 481 tokens, FP32, 8 cuts: 6.7 us, latency.  Prompts of 194 and 387: 22 us (34 TFLOP/s):
// what a CU draws of K and V, and the ends of uneven walks.  2,047 tokens over 8,000:
// 980 us, 119 TFLOP/s of the 151 that a large FP32 product reaches here.  Products of BF16 parts, three of K, Q, P
// and V each, took 870 us there, but 88 for 69 with a prompt of 1,000 tokens and 125 for 93 with a window.
template <typename QT, typename KT, int HD, int NT, int WK>
__global__ __launch_bounds__(WK * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void attend_rows_kernel(AttendArgs a) {
  using D = Dims<KT, HD>;
  constexpr int KW = D::KW, NK = D::NK, NDT = D::NDT, VW = D::VW, NV = D::NV, LDO = D::LDO, R = NT * 16;
  __shared__ __attribute__((aligned(16))) float po[WK * R * LDO];
  __shared__ float pm[WK * R], pl[WK * R];
  __shared__ float2 stats[R];
  const Cache& c = a.c;
  const int h = blockIdx.x, cut = blockIdx.z;
  TileAt tile;
  if (!find_tile(c, R, a.last - (int)blockIdx.y, tile)) return;   // the longest walks first
  const int seq = tile.seq, first = tile.first, n = tile.n, p0 = tile.p0, rows = n * c.G, f0 = tile.tile * R;
  const int p_lo = tile.slot(c, f0 / c.G), p_hi = tile.slot(c, (min(f0 + R, rows) - 1) / c.G);
  const Walk w = walk_of(p_lo, p_hi, a.window, a.sinks);
  const int end = min(w.n, (cut + 1) * a.cut);
  if (cut > 0 && cut * a.cut >= w.n) return;      // the first cut also answers for rows that see nothing
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i16 = lane & 15, q4 = lane >> 4;
  const int* table = c.table + seq * c.stride;
  const KT* kp = static_cast<const KT*>(c.k);
  const KT* vp = static_cast<const KT*>(c.v);

  int qp[NT];                                     // the slot of this lane's rows (rows past the last repeat it)
  float qf[NT][NK * KW];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int f = min(f0 + j * 16 + i16, rows - 1), tok = f / c.G;
    qp[j] = tile.slot(c, tok);
    const QT* qr = static_cast<const QT*>(a.q) + ((size_t)(first + tok) * c.Hq + h * c.G + (f - tok * c.G)) * HD;
#pragma unroll
    for (int t = 0; t < NK; ++t) {
      Piece<QT, KW> x;
      x.load(qr + t * 4 * KW + KW * q4);
#pragma unroll
      for (int e = 0; e < KW; ++e) qf[j][t * KW + e] = x.get(e);
    }
  }
  Piece<KT, KW> kf[NK];
  Piece<KT, VW> vf[4][NV];
  auto load_k = [&](size_t off) {
    const KT* p = kp + off + i16 * HD + KW * q4;
#pragma unroll
    for (int t = 0; t < NK; ++t) kf[t].load(p + t * 4 * KW);
  };
  auto load_v = [&](size_t off) {
    const KT* p = vp + off + 4 * q4 * HD + VW * i16;
#pragma unroll
    for (int v = 0; v < 4; ++v)
#pragma unroll
      for (int t = 0; t < NV; ++t) vf[v][t].load(p + v * HD + t * 16 * VW);
  };
  v4f o[NT][NDT];
  float mr[NT], lr[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    mr[j] = -INFINITY;
    lr[j] = 0.f;
#pragma unroll
    for (int t = 0; t < NDT; ++t) o[j][t] = v4f{0.f, 0.f, 0.f, 0.f};
  }

  TileOffsets offs;
  const int t_first = cut * a.cut + wave;
  bool wild = false;                              // infinities or NaN in V beside a mask
  if (t_first < end) {
    offs.load(c, tile.n_pages, table, w, t_first, WK, end, h, HD);
    load_k(offs.at(0));
  }
  int i = 0;                                      // the tile's lane in offs
  for (int t = t_first; t < end; t += WK) {
    const size_t off = offs.at(i);
    const bool bad = offs.bad >> i & 1;
    load_v(off);
    v4f s[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) s[j] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < NK; ++u)
#pragma unroll
      for (int e = 0; e < KW; ++e) {
        const float k = kf[u].get(e);
#pragma unroll
        for (int j = 0; j < NT; ++j) s[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(k, qf[j][u * KW + e], s[j], 0, 0, 0);
      }
    if (++i == 64 && t + WK < end) {
      i = 0;
      offs.load(c, tile.n_pages, table, w, t + WK, WK, end, h, HD);
    }
    load_k(offs.at(min(i, 63)));                  // the last tile again after the last: a load without a branch
    const int k0 = w.tile(t) * TILE;
    const bool whole = !bad && all_see(k0, k0 + TILE - 1, p_lo, p_hi, a.window, a.sinks);
    if (!whole) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const int key = k0 + 4 * q4 + v;
          if (bad) s[j][v] = NAN;
          if (!sees(qp[j], key, a.window, a.sinks)) s[j][v] = -INFINITY;
        }
      bool odd = false;
#pragma unroll
      for (int v = 0; v < 4; ++v)
#pragma unroll
        for (int u = 0; u < NV; ++u) odd |= vf[v][u].tame();
      if (__any(odd)) wild = true;
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      float mx = fmaxf(fmaxf(s[j][0], s[j][1]), fmaxf(s[j][2], s[j][3]));
      mx = max4(mx);
      const float mn = fmaxf(mr[j], mx);
      const float m2 = mn == -INFINITY ? 0.f : mn * a.scale2;
      const float sc = mr[j] == mn ? 1.f : rescale_of(mr[j], a.scale2, m2);
      float sum = 0.f;
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        s[j][v] = __builtin_amdgcn_exp2f(fmaf(s[j][v], a.scale2, -m2));
        sum += s[j][v];
      }
      lr[j] = lr[j] * sc + sum;                   // this lane's keys; a row's four lanes add up at the end
      mr[j] = mn;
      if (__any(sc != 1.f)) {
#pragma unroll
        for (int u = 0; u < NDT; ++u) o[j][u] *= sc;
      }
    }
#pragma unroll
    for (int v = 0; v < 4; ++v)
#pragma unroll
      for (int u = 0; u < NV; ++u)
#pragma unroll
        for (int e = 0; e < VW; ++e) {
          const float x = vf[v][u].get(e);
#pragma unroll
          for (int j = 0; j < NT; ++j)
            o[j][u * VW + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(x, s[j][v], o[j][u * VW + e], 0, 0, 0);
        }
  }
  // the waves meet: their rows of O and (max, sum), then a weight for each
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const float l = sum4(lr[j]);
    const int at = wave * R + j * 16 + i16;
    if (q4 == 0) { pm[at] = mr[j]; pl[at] = l; }
    float* row = po + at * LDO;
#pragma unroll
    for (int u = 0; u < NV; ++u)
#pragma unroll
      for (int v = 0; v < 4; ++v)
#pragma unroll
        for (int e = 0; e < VW; ++e) row[16 * VW * u + VW * (4 * q4 + v) + e] = o[j][u * VW + e][v];
  }
  meet_rows<QT, KT, HD, R, WK>(a, po, pm, pl, stats, wild, h, cut, table, first, p0, f0, rows, p_lo, p_hi, w, end);
}

// ------------------------------------------------------------ many rows, BF16 cache
// The same sums for chunks, on the BF16 matrix cores (32 x 32 x 16: half the
// instructions of 16 x 16 x 32 for the same products, and VALU work beside them runs under
// them).  A workgroup's 4 waves own 32 rows each and share steps of 64 keys in LDS, two
// slots each for K and V, loaded ahead straight from the pages.
//   S^T = K Q^T: K in fragments, Q in registers; lane l holds row l % 32's products with keys
//     8 i + 4 (l / 32) + r (i, r < 4) of each 32;
//   O^T += V^T P^T: eight of those values are P's fragment for 16 keys as they are.  V
//     lies in LDS row by row; the transposing LDS read gives a lane 4 keys of one dim.
// FP32 activations: Q and P as three BF16 parts of 8 bits that add up to the FP32 value
// exactly, three products each, so results are those of FP32 products (NP = 3).  BF16
// activations: P keeps 16 bits, two parts (off by 2^-16 of a weight at most, 256 times less than the output's own
// rounding; one part, off by 2^-8, adds as much again to it: 0.0023 of the output against 0.0017, for 269 us
// in place of 353 to 372 below).
//
// 2,047 BF16 tokens over 16,384, 16 heads on 8 of 128, with the join of its two cuts: 353 to 372 us by the
// card, 1,040 to 1,098 TFLOP/s of the three products per pair (a large BF16 product reaches 1,200 here).  The matrix cores
// are busy 68% of the time, the VALU (exponentials, maxima, parts) 60%.  LDS does not bound it (no bank conflicts).
// 4,500 FP32 tokens with a window of 1,024: 171 us, 725 TFLOP/s of the three-part products, matrix cores 52%
// busy: no registers are left to run a step's scores ahead.
constexpr int KEYS = 64;                          // keys of a step

template <int HD>
struct TileLds {
  static constexpr int K = KEYS * HD * 2;         // bytes of a slot
  // V row `key` holds its 32 bytes number x at x ^ turn(key), so that what half a wave's
  // transposing read takes, 4 keys x 64 bytes for 32 dims or 8 x 32 for 16 (turn16), lies in different banks
  static __device__ __forceinline__ int turn(int key) { return HD == 128 ? 2 * (key & 3) : HD == 64 ? key & 2 : 0; }
  static __device__ __forceinline__ int turn16(int key) { return HD == 128 ? key & 7 : HD == 64 ? key >> 1 & 3 : key >> 2 & 1; }
};

typedef float v16f __attribute__((ext_vector_type(16)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));

// Eight FP32 values as NP BF16 fragments: cut to 8 bits, what is left cut again; the
// third takes the rest exactly.  With two, the second is the rest rounded to nearest: off by 2^-16 of the value at most.
template <int NP>
__device__ __forceinline__ void parts8(const float* x, bf8* out) {
  static_assert(NP == 2 || NP == 3, "parts of 8 bits");
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = x[i];
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    if constexpr (NP == 2) {
      if (p == 1) {
#pragma unroll
        for (int i = 0; i < 8; ++i) out[1][i] = (__bf16)r[i];
        return;
      }
    }
    uint4 w;
    uint32_t* u = &w.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = __builtin_amdgcn_perm(__float_as_uint(r[2 * i + 1]), __float_as_uint(r[2 * i]), 0x07060302);
    out[p] = __builtin_bit_cast(bf8, w);
    if (p + 1 < NP) {
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] -= __uint_as_float(__float_as_uint(r[i]) & 0xffff0000u);
    }
  }
}

template <typename QT, int HD>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void attend_tiles_kernel(AttendArgs a) {
  constexpr int NP = sizeof(QT) == 4 ? 3 : 1, PP = NP == 3 ? 3 : 2, KS = HD / 32, R = 128;   // parts of Q, of P
  constexpr int GROUP = TILE * HD * 2;            // bytes of 16 keys
  using L = TileLds<HD>;
  __shared__ __attribute__((aligned(1024))) char lds[4 * L::K];   // two slots of K, two of V
  const Cache& c = a.c;
  const int h = blockIdx.x, cut = blockIdx.z;
  TileAt tile;
  // the last tiles of a sequence walk furthest: they start first
  if (!find_tile(c, R, a.last - (int)blockIdx.y, tile)) return;
  const int seq = tile.seq, first = tile.first, n = tile.n, p0 = tile.p0, rows = n * c.G, f0 = tile.tile * R;
  const int p_lo = tile.slot(c, f0 / c.G), p_hi = tile.slot(c, (min(f0 + R, rows) - 1) / c.G);
  const Walk w = walk_of(p_lo, p_hi, a.window, a.sinks);
  const int begin = cut * a.cut, end = min(w.n, begin + a.cut);
  if (cut > 0 && begin >= w.n) return;            // the first cut also answers for rows that see nothing
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i16 = lane & 15, q4 = lane >> 4, i32 = lane & 31, half = lane >> 5;
  const int* table = c.table + seq * c.stride;

  int qp;                                         // the slot of this lane's row (rows past the last repeat it)
  bf8 qf[NP][2 * KS];
  {
    const int f = min(f0 + wave * 32 + i32, rows - 1), tok = f / c.G;
    qp = tile.slot(c, tok);
    const QT* qr = static_cast<const QT*>(a.q) + ((size_t)(first + tok) * c.Hq + h * c.G + (f - tok * c.G)) * HD;
#pragma unroll
    for (int k = 0; k < 2 * KS; ++k) {
      Piece<QT, 8> x;
      x.load(qr + k * 16 + half * 8);
      if constexpr (NP == 1) {
        qf[0][k] = __builtin_bit_cast(bf8, x);
      } else {
        float y[8];
        bf8 part[NP];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = x.get(e);
        parts8<NP>(y, part);
#pragma unroll
        for (int p = 0; p < NP; ++p) qf[p][k] = part[p];
      }
    }
  }

  // wave u loads the u-th 16 keys of a step: K as blocks of 16 keys x 32 dims (16 bytes per
  // lane, keys first), V as rows, KS loads of 1 KB each
  const unsigned koff = (i16 * HD + q4 * 8) * 2;
  const int vrow = lane / (HD / 8);
  const unsigned voff = (vrow * HD + (lane % (HD / 8) ^ 2 * L::turn(vrow)) * 8) * 2;
  // this lane's bytes of K's fragment for a 32 x 16 block, and of 32 dims (the u-th) of V: vbase + (64 u ^ vturn)
  const unsigned kbase = (i32 >> 4) * KS * 1024 + (half * 16 + i16) * 16;
  const int vkey = 4 * half + (i16 >> 2);
  const unsigned vbase = vkey * HD * 2 + (i16 & 3) * 8, vturn = ((q4 & 1) ^ L::turn(vkey)) * 32;
  // AHEAD: K runs a step ahead of V, and while the weights of one step form, the matrix
  // cores have the next one's scores to work on (registers for both scores: not
  // beside the three parts of 128 dims)
  constexpr bool AHEAD = NP * HD <= 256;
  TileOffsets offs;
  int at = 0;                                     // the next step's first lane in offs
  size_t v_off = 0;                               // where V of the step after lies
  auto place = [&](int t) -> int {                // the step whose first tile is t; gives which of its tiles have no page
    if (at == 64) at = 0;
    if (at == 0) offs.load(c, tile.n_pages, table, w, t, 1, end, h, HD);
    v_off = offs.at(at + wave) * 2;
    const int none = offs.bad >> at & 15;
    at += 4;
    return none;
  };
  auto load_k = [&](int t) {
    const char* st = lds + ((t - begin) / 4 % 2) * L::K + wave * GROUP;
    const char* kb = static_cast<const char*>(c.k) + v_off;
#pragma unroll
    for (int k = 0; k < KS; ++k) lds_load16(kb + k * 64, koff, st + k * 1024);
  };
  auto load_v = [&](int t, size_t off) {
    const char* st = lds + 2 * L::K + ((t - begin) / 4 % 2) * L::K + wave * GROUP;
    const char* vb = static_cast<const char*>(c.v) + off;
#pragma unroll
    for (int k = 0; k < KS; ++k) lds_load16(vb + k * 1024, voff, st + k * 1024);
  };
  v16f o[KS], s[2];
  float m2 = LOWEST, lr = 0.f;                    // the maximum that sums refer to (times scale2), the sum
#pragma unroll
  for (int u = 0; u < KS; ++u)
#pragma unroll
    for (int v = 0; v < 16; ++v) o[u][v] = 0.f;
  // scores against 32 keys (i / KP) of a step, KU times 16 dims at a time: the fragments, the products
  constexpr int KU = AHEAD ? KS : KS / 2, KP = 2 * KS / KU;
  auto read_k = [&](int t, int i, bf8 (&kf)[KU]) {
    const char* st = lds + ((t - begin) / 4 % 2) * L::K + kbase + i / KP * 2 * GROUP;
#pragma unroll
    for (int k = 0; k < KU; ++k) kf[k] = *reinterpret_cast<const bf8*>(st + (i % KP * KU + k) * 512);
  };
  auto scores = [&](int i, const bf8 (&kf)[KU], v16f (&x)[2]) {
    if (i % KP == 0) {
#pragma unroll
      for (int v = 0; v < 16; ++v) x[i / KP][v] = 0.f;
    }
#pragma unroll
    for (int k = 0; k < KU; ++k)
#pragma unroll
      for (int p = NP - 1; p >= 0; --p)
        x[i / KP] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[k], qf[p][i % KP * KU + k], x[i / KP], 0, 0, 0);
  };
  // V of 16 keys (q / VP): VU times 32 dims at a time
  constexpr int VU = AHEAD ? KS : KS / 2, VP = KS / VU;
  auto read_v = [&](const char* vst, int q, bf8 (&vf)[VU]) {
#pragma unroll
    for (int u = 0; u < VU; ++u) {
      typedef __attribute__((address_space(3))) s4 lds4;
      const char* vr = vst + (vbase + ((q % VP * VU + u) * 64 ^ vturn)) + q / VP * GROUP;
      const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)vr);
      const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(vr + GROUP / 2));
      vf[u] = __builtin_bit_cast(bf8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  };
  bool wild = false;                              // infinities or NaN in V beside a mask
  int bad = 0, bad1 = 0;                          // tiles without a page of this step, the next
  // the step at t: V of it and K (of the next one with AHEAD, whose scores of this one are in s) are loaded
  auto step = [&](int t, auto more) {
    constexpr bool MORE = decltype(more)::value;
    int bad2 = 0;
    stage_sync<0>();                              // they are in, and every wave is done with the slots loaded next
    bf8 kf[2][KU];
    if constexpr (!AHEAD) {
      if (t + 4 < end) {
        bad2 = place(t + 4);
        load_k(t + 4);
        load_v(t + 4, v_off);
      }
      read_k(t, 0, kf[0]);
#pragma unroll
      for (int i = 0; i < 2 * KP; ++i) {
        if (i + 1 < 2 * KP) read_k(t, i + 1, kf[(i + 1) % 2]);
        __builtin_amdgcn_sched_barrier(0);
        scores(i, kf[i % 2], s);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else if constexpr (MORE) {
      load_v(t + 4, v_off);
      if (t + 8 < end) {
        bad2 = place(t + 8);
        load_k(t + 8);
      }
      read_k(t + 4, 0, kf[0]);
    }
    char* vst = lds + 2 * L::K + ((t - begin) / 4 % 2) * L::K;
    const int k_first = w.tile(t) * TILE, k_last = w.tile(min(t + 3, end - 1)) * TILE + TILE - 1;
    if (bad || t + 4 > end || !all_see(k_first, k_last, p_lo, p_hi, a.window, a.sinks)) {
      bool odd = false;                           // each wave tames the V that it loaded
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        auto* x = reinterpret_cast<Piece<uint16_t, 8>*>(vst + wave * GROUP + k * 1024 + lane * 16);
        Piece<uint16_t, 8> y = *x;
        odd |= y.tame();
        *x = y;
      }
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int k0 = w.tile(min(t + g, end - 1)) * TILE + 4 * half;
#pragma unroll
        for (int v = 0; v < 8; ++v) {
          if (bad >> g & 1) s[g / 2][g % 2 * 8 + v] = NAN;
          if (t + g >= end || !sees(qp, k0 + v / 4 * 8 + v % 4, a.window, a.sinks)) s[g / 2][g % 2 * 8 + v] = -INFINITY;
        }
      }
      wild |= __builtin_amdgcn_readfirstlane(__syncthreads_or(odd)) != 0;
    }
    // a row's sums refer to a maximum of earlier steps until one is past it by 2^8: weights are
    // at most that, and O is rarely rescaled
    float sc = s[0][0];
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int v = 0; v < 16; ++v) sc = fmaxf(sc, s[g][v]);
    sc = max2(sc);
    sc *= a.scale2;
    const bool grown = __any(sc > m2 + 8.f);
    if (grown) {
      const float x = fmaxf(m2, sc);
      sc = m2 == x ? 1.f : __builtin_amdgcn_exp2f(m2 - x);
      lr *= sc;
      m2 = x;
    }
    // the matrix cores' part of a step goes first where two waves of a SIMD are apart (2,047
    // tokens over 16,384, BF16: 287 -> 262 us; no change with three parts)
    if constexpr (AHEAD) __builtin_amdgcn_s_setprio(1);
    v16f s2[2];
    bf8 pf[4][PP], vf[2][VU];                     // weights of the four sets of 16 keys
    auto weights = [&](int g) {
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        y[e] = __builtin_amdgcn_exp2f(fmaf(s[g / 2][g % 2 * 8 + e], a.scale2, -m2));
        lr += y[e];                               // this lane's keys; a row's two lanes add up at the end
      }
      parts8<PP>(y, pf[g]);
      // formed here, under the products beside it
#pragma unroll
      for (int p = 0; p < PP; ++p) asm volatile("" : "+v"(pf[g][p]));
      asm volatile("" : "+v"(lr));
    };
    auto values = [&](int q) {
#pragma unroll
      for (int u = 0; u < VU; ++u)
#pragma unroll
        for (int p = PP - 1; p >= 0; --p)
          o[q % VP * VU + u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[q % 2][u], pf[q / VP][p], o[q % VP * VU + u], 0, 0, 0);
    };
    auto rescale = [&]() {
      if (!grown) return;
#pragma unroll
      for (int u = 0; u < KS; ++u) o[u] *= sc;
    };
    // sets of products with the LDS reads of the next ahead of each and the weights spread under them
    if constexpr (AHEAD) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {               // 0, 1: scores of the next step's first 32 keys; 2 - 5: values; 6, 7: the other scores
        constexpr int NEXT_K[8] = {1, -1, -1, -1, -1, 2, 3, -1}, NEXT_V[8] = {-1, 0, 1, 2, 3, -1, -1, -1};
        if constexpr (MORE) {
          if (NEXT_K[i] >= 0) read_k(t + 4, NEXT_K[i], kf[NEXT_K[i] % 2]);
        }
        if (NEXT_V[i] >= 0) read_v(vst, NEXT_V[i], vf[NEXT_V[i] % 2]);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (MORE) {
          if (i < 2) scores(i, kf[i % 2], s2);
          if (i > 5) scores(i - 4, kf[i % 2], s2);
        }
        if (i == 2) rescale();
        if (i >= 2 && i < 6) values(i - 2);
        if (i < 4) weights(i);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
#pragma unroll
      for (int i = 0; i <= 4 * VP; ++i) {
        if (i < 4 * VP) read_v(vst, i, vf[i % 2]);
        __builtin_amdgcn_sched_barrier(0);
        if (i == 1) rescale();
        if (i > 0) values(i - 1);
        if (i % VP == 0 && i < 4 * VP) weights(i / VP);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if constexpr (MORE) {
      s[0] = s2[0];
      s[1] = s2[1];
    }
    if constexpr (AHEAD) __builtin_amdgcn_s_setprio(0);
    bad = AHEAD ? bad1 : bad2;
    bad1 = bad2;
  };
  if (begin < end) {
    bad = place(begin);
    load_k(begin);
    load_v(begin, v_off);
  }
  if constexpr (!AHEAD) {
    for (int t = begin; t < end; t += 4) step(t, std::false_type{});
  } else if (begin < end) {
    if (begin + 4 < end) {
      bad1 = place(begin + 4);
      load_k(begin + 4);
    }
    stage_sync<0>();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      bf8 kf[KU];
      read_k(begin, i, kf);
      scores(i, kf, s);
    }
    int t = begin;
    for (; t + 4 < end; t += 4) step(t, std::true_type{});
    step(t, std::false_type{});
  }

  const bool alone = w.n <= a.cut;                // no other cut: the answer itself
  const int f = f0 + wave * 32 + i32, tok = f / c.G;
  const float l = sum2(lr);
  if (f < rows) {
    const size_t row = (size_t)(first + tok) * c.Hq + h * c.G + (f - tok * c.G);
    const bool none = qp < 0;                     // no key is seen
    const float y = alone ? none ? 0.f : 1.f / l : 1.f;
    if (half == 0) {
      if (cut == 0 && a.count) a.count[row] = cuts_of(a, w, none);
      if (!alone) {
        float* d = a.ml + ((size_t)cut * c.T * c.Hq + row) * 2;
        d[0] = m2;
        d[1] = l;
      } else if (a.lse) {
        a.lse[row] = none ? -INFINITY : (m2 + log2f(l)) * LN2;
      }
    }
#pragma unroll
    for (int u = 0; u < KS; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = 32 * u + 8 * i + 4 * half;
        if (alone) store4(static_cast<QT*>(a.out) + row * HD + d, y * o[u][4 * i], y * o[u][4 * i + 1], y * o[u][4 * i + 2], y * o[u][4 * i + 3]);
        else *reinterpret_cast<float4*>(a.part + ((size_t)cut * c.T * c.Hq + row) * HD + d) =
            make_float4(o[u][4 * i], o[u][4 * i + 1], o[u][4 * i + 2], o[u][4 * i + 3]);
      }
  }
  if (wild) {
    __threadfence_block();                        // the stores above, by other lanes
    TileAt again;                                 // few registers are held for this through the loop
    find_tile(c, R, a.last - (int)blockIdx.y, again);
    const int t2 = again.tile * R, f_lo = t2 + wave * 32, f_hi = min(t2 + R, again.n * c.G);
    const int q_lo = again.slot(c, t2 / c.G), q_hi = again.slot(c, (f_hi - 1) / c.G);
    const Walk v = walk_of(q_lo, q_hi, a.window, a.sinks);
    const int b2 = blockIdx.z * a.cut, e2 = min(v.n, b2 + a.cut);
    const int* tab = c.table + again.seq * c.stride;
    add_wild<QT, uint16_t, HD>(
        a, h, tab, again.first, again.p0, f_lo, min(f_lo + 32, f_hi), v, b2, e2,
        v.n <= a.cut ? nullptr : a.part + (size_t)blockIdx.z * c.T * c.Hq * HD,
        [&](int t) {
          const int t0 = b2 + (t - b2) / 4 * 4, t3 = min(t0 + 3, e2 - 1);
          bool none = t0 + 4 > e2;                // as the loop above judged the step
          for (int u = t0; u <= t3; ++u) {
            const int e = tab[page_of(c, v.tile(u) * TILE)];
            none |= e < 0 || e >= c.n_pages;
          }
          return none || !all_see(v.tile(t0) * TILE, v.tile(t3) * TILE + TILE - 1, q_lo, q_hi, a.window, a.sinks);
        },
        [&](int g) {
          return make_float2(__shfl(m2, g - f_lo, 64), v.n <= a.cut ? 1.f / __shfl(l, g - f_lo, 64) : 1.f);
        });
  }
}

// ------------------------------------------------------------ few rows, BF16 cache
// Single tokens and short chunks, where the bytes of K and V decide.  As in the row kernel a
// workgroup's WK waves share NT tiles of 16 rows and take keys in turn, 32 at a
// time, with no barrier in the loop, but on the BF16 matrix cores (16 x 16 x 32, parts as above): FP32 products
// take 1,024 cycles of a SIMD per 4 KB of the cache, these 64 to 192 (with BF16 activations P keeps 16
// bits, two parts: it costs nothing here).  K goes from the pages to registers as fragments, V to
// two slots of LDS of the wave's own, both a step ahead.
// 32 rows of 328 to 657 tokens, FP32 on BF16: 17 us for 65 MB, one workgroup per CU at what it draws (10.7 at
// the 6.1 TB/s of a pure read); two rows of 30,720 and 61,441 in 16 cuts: 66 us, 5.7 TB/s.
template <typename QT, int HD, int NT, int WK>
__global__ __launch_bounds__(WK * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void attend_few_kernel(AttendArgs a) {
  constexpr int NP = sizeof(QT) == 4 ? 3 : 1, PP = NP == 3 ? 3 : 2;   // parts of Q, of P
  constexpr int KS = HD / 32, NDT = HD / 16, R = NT * 16, LDO = HD + 4;
  constexpr int GROUP = TILE * HD * 2;            // bytes of 16 keys
  using L = TileLds<HD>;
  constexpr int SLOTS = WK * 4 * GROUP, MEET = WK * R * LDO * 4;
  __shared__ __attribute__((aligned(1024))) char lds[SLOTS > MEET ? SLOTS : MEET];
  __shared__ float pm[WK * R], pl[WK * R];
  __shared__ float2 stats[R];
  const Cache& c = a.c;
  const int h = blockIdx.x, cut = blockIdx.z;
  TileAt tile;
  if (!find_tile(c, R, a.last - (int)blockIdx.y, tile)) return;   // the longest walks first
  const int seq = tile.seq, first = tile.first, n = tile.n, p0 = tile.p0, rows = n * c.G, f0 = tile.tile * R;
  const int p_lo = tile.slot(c, f0 / c.G), p_hi = tile.slot(c, (min(f0 + R, rows) - 1) / c.G);
  const Walk w = walk_of(p_lo, p_hi, a.window, a.sinks);
  const int end = min(w.n, (cut + 1) * a.cut);
  if (cut > 0 && cut * a.cut >= w.n) return;      // the first cut also answers for rows that see nothing
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i16 = lane & 15, q4 = lane >> 4;
  const int* table = c.table + seq * c.stride;

  const int t_first = cut * a.cut + 2 * wave;     // the wave's tiles: two of every 2 WK
  TileOffsets offs;
  if (t_first < end) offs.load(c, tile.n_pages, table, w, t_first, 2 * WK, end, h, HD, true);
  const unsigned koff = i16 * HD + q4 * 8;        // elements
  const int vrow = lane / (HD / 8);
  const unsigned voff = (vrow * HD + (lane % (HD / 8) ^ 2 * L::turn16(vrow)) * 8) * 2;
  const int vkey = 4 * q4 + (i16 >> 2);
  const unsigned vbase = vkey * HD * 2 + (i16 & 3) * 8, vturn = L::turn16(vkey) * 32;
  char* vlds = lds + wave * 4 * GROUP;
  auto load = [&](int i, int slot, bf8 (&kf)[2][KS]) {   // tiles i, i + 1 of offs
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const size_t off = offs.at(i + g);
      const char* vb = static_cast<const char*>(c.v) + off * 2;
#pragma unroll
      for (int k = 0; k < KS; ++k)
        lds_load16(vb + k * 1024, HD == 128 && k % 2 ? voff ^ 128 : voff, vlds + (2 * slot + g) * GROUP + k * 1024);
      const uint16_t* kr = static_cast<const uint16_t*>(c.k) + off + koff;
#pragma unroll
      for (int k = 0; k < KS; ++k) kf[g][k] = *reinterpret_cast<const bf8*>(kr + k * 32);
    }
  };
  int qp[NT];                                     // the slot of this lane's rows (rows past the last repeat it)
  bf8 qf[NT][NP][KS];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int f = min(f0 + j * 16 + i16, rows - 1), tok = f / c.G;
    qp[j] = tile.slot(c, tok);
    const QT* qr = static_cast<const QT*>(a.q) + ((size_t)(first + tok) * c.Hq + h * c.G + (f - tok * c.G)) * HD;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      Piece<QT, 8> x;
      x.load(qr + k * 32 + q4 * 8);
      if constexpr (NP == 1) {
        qf[j][0][k] = __builtin_bit_cast(bf8, x);
      } else {
        float y[8];
        bf8 part[NP];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = x.get(e);
        parts8<NP>(y, part);
#pragma unroll
        for (int p = 0; p < NP; ++p) qf[j][p][k] = part[p];
      }
    }
  }
  v4f o[NT][NDT];
  float mr[NT], lr[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    mr[j] = -INFINITY;
    lr[j] = 0.f;
#pragma unroll
    for (int t = 0; t < NDT; ++t) o[j][t] = v4f{0.f, 0.f, 0.f, 0.f};
  }
  bool wild = false;                              // infinities or NaN in V beside a mask
  int i = 0;                                      // the step's first lane in offs
  // the step of tiles t and t + 1: kf and slot hold it; the next goes to the others
  auto step = [&](int t, int slot, bf8 (&kf)[2][KS], bf8 (&other)[2][KS]) {
    const int bad = offs.bad >> i & 3;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
    for (int g = 0; g < 2; ++g)                   // here, not behind the next step's loads, which the compiler counts too
#pragma unroll
      for (int k = 0; k < KS; ++k) asm volatile("" : "+v"(kf[g][k]));
    i += 2;
    if (t + 2 * WK < end) {
      if (i == 64) {
        i = 0;
        offs.load(c, tile.n_pages, table, w, t + 2 * WK, 2 * WK, end, h, HD, true);
      }
      load(i, slot ^ 1, other);
    }
    v4f s[NT][2];
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int j = 0; j < NT; ++j) s[j][g] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int p = NP - 1; p >= 0; --p)
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
          for (int j = 0; j < NT; ++j) s[j][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[g][k], qf[j][p][k], s[j][g], 0, 0, 0);
    char* vst = vlds + 2 * slot * GROUP;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int k0 = w.tile(min(t + g, end - 1)) * TILE;
      if (!(bad >> g & 1) && t + g < end && all_see(k0, k0 + TILE - 1, p_lo, p_hi, a.window, a.sinks)) continue;
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          if (bad >> g & 1) s[j][g][v] = NAN;
          if (t + g >= end || !sees(qp[j], k0 + 4 * q4 + v, a.window, a.sinks)) s[j][g][v] = -INFINITY;
        }
      bool odd = false;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        auto* x = reinterpret_cast<Piece<uint16_t, 8>*>(vst + g * GROUP + k * 1024 + lane * 16);
        Piece<uint16_t, 8> y = *x;
        odd |= y.tame();
        *x = y;
      }
      __builtin_amdgcn_wave_barrier();            // this wave's own LDS, read below by other lanes of it
      if (__any(odd)) wild = true;
    }
    bf8 pf[NT][PP];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      float mx = s[j][0][0];
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int v = 0; v < 4; ++v) mx = fmaxf(mx, s[j][g][v]);
      const float mn = fmaxf(mr[j], max4(mx)), m2 = mn == -INFINITY ? 0.f : mn * a.scale2;
      const float sc = mr[j] == mn ? 1.f : rescale_of(mr[j], a.scale2, m2);
      float y[8], sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        y[e] = __builtin_amdgcn_exp2f(fmaf(s[j][e / 4][e % 4], a.scale2, -m2));
        sum += y[e];
      }
      parts8<PP>(y, pf[j]);
      lr[j] = lr[j] * sc + sum;                   // this lane's keys; a row's four lanes add up at the end
      mr[j] = mn;
      if (__any(sc != 1.f)) {
#pragma unroll
        for (int u = 0; u < NDT; ++u) o[j][u] *= sc;
      }
    }
#pragma unroll
    for (int u = 0; u < NDT; ++u) {
      typedef __attribute__((address_space(3))) s4 lds4;
      const char* vr = vst + (vbase + (u * 32 ^ vturn));
      const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)vr);
      const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(vr + GROUP));
      const bf8 vf = __builtin_bit_cast(bf8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
      for (int p = PP - 1; p >= 0; --p)
#pragma unroll
        for (int j = 0; j < NT; ++j) o[j][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[j][p], o[j][u], 0, 0, 0);
    }
    // the next step's loads into this slot come after these reads
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  };
  bf8 ka[2][KS], kb[2][KS];
  if (t_first < end) load(0, 0, ka);
  for (int t = t_first; t < end; t += 4 * WK) {
    step(t, 0, ka, kb);
    if (t + 2 * WK < end) step(t + 2 * WK, 1, kb, ka);
  }
  // the waves meet: their rows of O and (max, sum)
  __syncthreads();                                // V's slots become rows of O
  float* po = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const float l = sum4(lr[j]);
    const int at = wave * R + j * 16 + i16;
    if (q4 == 0) { pm[at] = mr[j]; pl[at] = l; }
#pragma unroll
    for (int u = 0; u < NDT; ++u)
      *reinterpret_cast<float4*>(po + at * LDO + 16 * u + 4 * q4) = make_float4(o[j][u][0], o[j][u][1], o[j][u][2], o[j][u][3]);
  }
  meet_rows<QT, uint16_t, HD, R, WK>(a, po, pm, pl, stats, wild, h, cut, table, first, p0, f0, rows, p_lo, p_hi, w, end);
}

// Joins the cuts of rows that have several (at most 64); WPR waves per row (token, query head),
// half a wave per cut and 16 bytes per lane, the parts of a wave's cuts loading together.
// What the kernel before left in `count` spares the way to the row's sequence (2,047
// tokens: 25 -> 17 us).
template <typename QT, int HD, int WPR>
__global__ __launch_bounds__(256) void combine_kernel(AttendArgs a, int cuts) {
  constexpr int NL = HD / 4, PER = 64 / NL < 2 ? 1 : 2, U = 4;   // lanes of a part, cuts of a wave at a time, loads under way
  __shared__ float4 meet[WPR > 1 ? WPR * NL : 1];
  const Cache& c = a.c;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), sub = wave % WPR;
  const int at = blockIdx.x * (4 / WPR) + wave / WPR;
  if (at >= c.T * c.Hq) return;                   // WPR 4: one row per workgroup, so all of it
  const size_t step = (size_t)c.T * c.Hq;
  const int m = at / c.Hq, count = a.count[at], from = c.starts[0], to = c.starts[c.S];
  const float2 own = *reinterpret_cast<const float2*>(a.ml + (min(lane, cuts - 1) * step + at) * 2);
  if (m < from || m >= to || count == 0) return;  // no sequence's row, or one whose only cut's workgroup wrote the answer
  const bool none = count < 0;
  const int ns = min(none ? -count : count, cuts);
  const float2 ml = lane < ns ? own : make_float2(LOWEST, 0.f);
  float m2 = ml.x;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) m2 = fmaxf(m2, __shfl_xor(m2, d, 64));
  const float wt = __builtin_amdgcn_exp2f(ml.x - m2);   // of cut number `lane`
  float l = lane < ns ? wt * ml.y : 0.f;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) l += __shfl_xor(l, d, 64);
  const int half = lane / NL, dim = lane % NL;    // lanes past PER parts (short heads) repeat the last one's work
  const int mine = min(half, PER - 1);
  const float* p = a.part + (size_t)at * HD + dim * 4;
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = sub * PER * U; s0 < ns; s0 += WPR * PER * U) {
    float4 x[U];
    float f[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = s0 + u * PER + mine;
      x[u] = *reinterpret_cast<const float4*>(p + min(s, ns - 1) * step * HD);
      f[u] = __shfl(wt, min(s, ns - 1), 64);
      if (s >= ns) { f[u] = 0.f; x[u] = make_float4(0.f, 0.f, 0.f, 0.f); }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      y.x = fmaf(f[u], x[u].x, y.x); y.y = fmaf(f[u], x[u].y, y.y); y.z = fmaf(f[u], x[u].z, y.z); y.w = fmaf(f[u], x[u].w, y.w);
    }
  }
  if constexpr (PER == 2) {
    const float4 z = make_float4(__shfl_xor(y.x, NL, 64), __shfl_xor(y.y, NL, 64), __shfl_xor(y.z, NL, 64), __shfl_xor(y.w, NL, 64));
    y.x += z.x; y.y += z.y; y.z += z.z; y.w += z.w;
  }
  if constexpr (WPR > 1) {
    if (half == 0) meet[sub * NL + dim] = y;
    __syncthreads();
    if (sub > 0) return;
#pragma unroll
    for (int u = 1; u < WPR; ++u) {
      const float4 z = meet[u * NL + dim];
      y.x += z.x; y.y += z.y; y.z += z.z; y.w += z.w;
    }
  }
  const float r = none ? 0.f : 1.f / l;
  if (half == 0) store4(static_cast<QT*>(a.out) + (size_t)at * HD + dim * 4, none ? 0.f : r * y.x, none ? 0.f : r * y.y, none ? 0.f : r * y.z, none ? 0.f : r * y.w);
  if (a.lse && lane == 0) a.lse[at] = none ? -INFINITY : (m2 + log2f(l)) * LN2;
}

// ------------------------------------------------------------ accounts of attention weight
// mass[j] += sum over the rows of key head h that see j of exp(s_j - lse): with
// the statistics known every weight is one exponential, and a workgroup that holds
// its keys and walks the rows adds up without atomics, in one order.
//   S = Q K^T: lane l holds rows 4 (l / 16) + v against key l % 16; the sum over rows stays in the lane.
// A wave holds NK2 tiles of 16 keys in registers; four waves per workgroup.  On the FP32 matrix cores: for single
// tokens over FP32 caches, where the bytes of K decide, and for heads of 16.
struct MassArgs {
  Cache c;
  const void* q; const float* lse; float* mass;   // [n_pages][Hkv][page]
  float scale;
  int window, sinks;
  int cut, cuts;                                  // rows per cut, cuts of a sequence's rows
  float* part;                                    // [S][cuts][Hkv][width * page] of sequences with several
};
// The rows (token, head of the group) of a sequence that can see one of `keys` slots from k0 on.
__device__ __forceinline__ void mass_rows(const MassArgs& a, int n, int p0, int k0, int keys, int& f_lo, int& f_hi) {
  const int G = a.c.G;
  f_lo = min(max(0, k0 - p0), n) * G;
  f_hi = n * G;
  if (a.window > 0 && k0 >= a.sinks)
    f_hi = (int)max((int64_t)0, min((int64_t)n, (int64_t)k0 + keys - 1 + a.window - p0)) * G;
}

template <typename QT, typename KT, int HD, int NK2>
__global__ __launch_bounds__(256) void mass_kernel(MassArgs a) {
  using D = Dims<KT, HD>;
  constexpr int KW = D::KW, NK = D::NK;
  const Cache& c = a.c;
  const int h = blockIdx.x, seq = blockIdx.z;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i16 = lane & 15, q4 = lane >> 4;
  int first, n;
  seq_rows(c, seq, first, n);
  const int len = seq_len(c, seq), p0 = len - n;
  const int k0 = (blockIdx.y * 4 + wave) * NK2 * TILE;
  if (n == 0 || k0 >= len || too_long(c, seq)) return;
  const int* table = c.table + seq * c.stride;
  const KT* kp = static_cast<const KT*>(c.k);
  float kf[NK2][NK * KW], sum[NK2];
  size_t at[NK2];
  bool bad[NK2];
#pragma unroll
  for (int j = 0; j < NK2; ++j) {
    const int key0 = min(k0 + j * TILE, (len - 1) / TILE * TILE), e = table[key0 / c.page];
    bad[j] = e < 0 || e >= c.n_pages;
    at[j] = ((size_t)(bad[j] ? 0 : e) * c.Hkv + h) * c.page + key0 % c.page + i16;
    sum[j] = 0.f;
#pragma unroll
    for (int t = 0; t < NK; ++t) {
      Piece<KT, KW> x;
      x.load(kp + at[j] * HD + t * 4 * KW + KW * q4);
#pragma unroll
      for (int e2 = 0; e2 < KW; ++e2) kf[j][t * KW + e2] = x.get(e2);
    }
  }
  int f_lo, f_hi;
  mass_rows(a, n, p0, k0, NK2 * TILE, f_lo, f_hi);
  for (int f0 = f_lo; f0 < f_hi; f0 += 16) {
    const int f = min(f0 + i16, n * c.G - 1), tok = f / c.G;
    const QT* qr = static_cast<const QT*>(a.q) + ((size_t)(first + tok) * c.Hq + h * c.G + (f - tok * c.G)) * HD;
    Piece<QT, KW> x[NK];
#pragma unroll
    for (int t = 0; t < NK; ++t) x[t].load(qr + t * 4 * KW + KW * q4);
    float ls[4];
    int p[4];
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int fv = f0 + 4 * q4 + v, tv = min(fv, n * c.G - 1) / c.G;
      p[v] = fv < n * c.G ? p0 + tv : -1;
      ls[v] = a.lse[(size_t)(first + tv) * c.Hq + h * c.G + (min(fv, n * c.G - 1) - tv * c.G)];
    }
    v4f s[NK2];
#pragma unroll
    for (int j = 0; j < NK2; ++j) s[j] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < NK; ++t)
#pragma unroll
      for (int e = 0; e < KW; ++e) {
        const float xq = x[t].get(e);
#pragma unroll
        for (int j = 0; j < NK2; ++j) s[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(xq, kf[j][t * KW + e], s[j], 0, 0, 0);
      }
#pragma unroll
    for (int j = 0; j < NK2; ++j)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const float y = __builtin_amdgcn_exp2f(fmaf(s[j][v], a.scale, -ls[v]) * LOG2E);
        sum[j] += sees(p[v], k0 + j * TILE + i16, a.window, a.sinks) ? y : 0.f;
      }
  }
#pragma unroll
  for (int j = 0; j < NK2; ++j) {
    const float y = sum4(sum[j]);
    if (q4 == 0 && k0 + j * TILE + i16 < len && !bad[j]) a.mass[at[j]] += y;
  }
}

// On the BF16 matrix cores.  Each wave holds 64 keys as fragments in registers (32 of an FP32 cache,
// in three parts), and the workgroup's keys meet the rows in LDS, N at a time: FP32 ones are cut into
// their three BF16 parts there, once for all waves, the next ones loading meanwhile in registers; two slots, one
// barrier per stage.  Parts of both sides: all nine products, so that none is lost (the six of the largest parts take
// 142 us in place of 183 for prompts of 900 and 1,800 over 1,800 and 3,600 FP32 tokens, and leave out up to 2^-21 of a
// product, always towards 0).
//   N = 32 (many rows): S = Q K^T by 32 x 32 x 16; lane l holds rows 8 i + 4 (l / 32) + r (i, r < 4) against key l % 32.
//   N = 16 (few rows, where the bytes of K decide: 64 bytes of 16 keys per load): 16 x 16 x 32; rows
//     4 (l / 16) + r against key l % 16.
// Many rows on few keys are cut over workgroups, whose sums mass_join_kernel adds in order.
//
// 32 rows of 2,400 to 4,800 tokens, FP32 on BF16: 52 us, 244 MB at 4.7 TB/s.  Prompts of 900 and 1,800 over
// 1,800 and 3,600: 92 + 5 us, 810 TFLOP/s of the three-part products, matrix cores 48% busy beside one exponential
// per weight and the parts (three waves per SIMD spill: 109; cuts for fewer than twelve workgroups per CU: 132 to 140).
template <typename QT, typename KT, int HD, int N>
__global__ __launch_bounds__(256) void mass_tiles_kernel(MassArgs a) {
  constexpr int NP = sizeof(QT) == 4 ? 3 : 1, KD = 512 / N, KS = HD / KD;   // dims of a fragment, fragments of a row tile
  constexpr int KP = sizeof(KT) == 4 ? 3 : 1, NJ = (KP == 1 ? 64 : 32) / N, KEYS = NJ * N, NV = N * N / 64, NF = (KS + 3) / 4;            // key tiles of a wave, values per lane, fragments per wave
  using acc = std::conditional_t<N == 32, v16f, v4f>;
  __shared__ __attribute__((aligned(1024))) char frag[2][KS * NP * 1024];
  __shared__ __attribute__((aligned(16))) float lse[2][N];
  __shared__ __attribute__((aligned(16))) int slot[2][N];
  const Cache& c = a.c;
  const int h = blockIdx.x, seq = blockIdx.z / a.cuts, cut = blockIdx.z - seq * a.cuts;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int in = lane % N, part = lane / N;       // row or key of a fragment, its piece of 8 dims
  int first, n;
  seq_rows(c, seq, first, n);
  const int len = seq_len(c, seq), p0 = len - n, rows = n * c.G;
  const int b0 = blockIdx.y * 4 * KEYS, k0 = b0 + wave * KEYS;   // first keys of the workgroup, of the wave
  if (n == 0 || b0 >= len || too_long(c, seq)) return;
  int f_lo, f_end;
  mass_rows(a, n, p0, b0, 4 * KEYS, f_lo, f_end);
  const bool alone = f_end - f_lo <= a.cut;       // one cut: added to the accounts here
  f_lo += cut * a.cut;
  if (f_lo >= f_end) return;
  const int f_hi = min(f_end, f_lo + a.cut);
  const int* table = c.table + seq * c.stride;
  // this lane's account: key k0 + lane
  const int key = min(k0 + lane, len - 1), pg = page_of(c, key), page = table[pg];
  const bool live = lane < KEYS && k0 + lane < len && page >= 0 && page < c.n_pages;
  float* account = alone ? a.mass + ((size_t)(live ? page : 0) * c.Hkv + h) * c.page + (key - pg * c.page)
                         : a.part + (((size_t)seq * a.cuts + cut) * c.Hkv + h) * ((size_t)c.width * c.page) + key;
  const float before = alone && live ? *account : 0.f;
  bf8 kf[NJ][KP][KS];
#pragma unroll
  for (int j = 0; j < NJ; ++j) {                  // lanes past the length read its last 16 keys
    const int t = min((k0 + j * N + in) / TILE * TILE, (len - 1) / TILE * TILE), g = page_of(c, t), e = table[g];
    const KT* kr = static_cast<const KT*>(c.k) +
                   (((size_t)(e >= 0 && e < c.n_pages ? e : 0) * c.Hkv + h) * c.page + (t - g * c.page) + in % TILE) * HD + part * 8;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      if constexpr (KP == 1) {
        kf[j][0][k] = *reinterpret_cast<const bf8*>(kr + k * KD);
      } else {
        Piece<KT, 8> x;
        float y[8];
        bf8 parts[KP];
        x.load(kr + k * KD);
#pragma unroll
        for (int e2 = 0; e2 < 8; ++e2) y[e2] = x.get(e2);
        parts8<KP>(y, parts);
#pragma unroll
        for (int p = 0; p < KP; ++p) kf[j][p][k] = parts[p];
      }
    }
  }

  // this lane's rows by (token, head), carried along: a stage is N / G tokens and N % G heads further
  const int dt = N / c.G, dg = N - dt * c.G;
  struct Row {
    int f, tok, g;
  };
  auto row_at = [&](int f) { const int tok = f / c.G; return Row{f, tok, f - tok * c.G}; };
  auto advance = [&](Row& r) {
    r.f += N;
    r.tok += dt;
    r.g += dg;
    if (r.g >= c.G) { r.g -= c.G; ++r.tok; }
  };
  auto place = [&](const Row& r) -> size_t {      // rows past the last read the first
    return r.f < rows ? (size_t)(first + r.tok) * c.Hq + h * c.G + r.g : (size_t)first * c.Hq + h * c.G;
  };
  Row mine = row_at(f_lo + in);                   // threads of the first row's N lanes also bring lse and slot
  Piece<QT, 8> next[NF];
  float lse_next = 0.f;
  int slot_next = -1;
  auto load = [&]() {
    const size_t at = place(mine);
    const QT* q = static_cast<const QT*>(a.q) + at * HD + part * 8;
#pragma unroll
    for (int i = 0; i < NF; ++i) next[i].load(q + min(wave * NF + i, KS - 1) * KD);
    if (tid < N) {
      slot_next = mine.f < f_hi ? p0 + mine.tok : -1;   // -1: sees nothing
      lse_next = a.lse[at];
    }
    advance(mine);
  };
  float sum[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) sum[j] = 0.f;
  load();
  int b = 0;
  for (int f0 = f_lo; f0 < f_hi; f0 += N, b ^= 1) {
#pragma unroll
    for (int i = 0; i < NF; ++i) {
      if (wave * NF + i >= KS) break;
      char* d = frag[b] + (wave * NF + i) * NP * 1024 + lane * 16;
      if constexpr (NP == 1) {
        *reinterpret_cast<Piece<QT, 8>*>(d) = next[i];
      } else {
        float y[8];
        bf8 parts[NP];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = next[i].get(e);
        parts8<NP>(y, parts);
#pragma unroll
        for (int p = 0; p < NP; ++p) *reinterpret_cast<bf8*>(d + p * 1024) = parts[p];
      }
    }
    if (tid < N) {
      lse[b][tid] = lse_next;
      slot[b][tid] = slot_next;
    }
    __syncthreads();                              // also: every wave is done with this slot's stage before last
    if (f0 + N < f_hi) load();
    acc s[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int v = 0; v < NV; ++v) s[j][v] = 0.f;
    constexpr int ALL = KS * NP, C = ALL % 4 == 0 ? 4 : ALL % 3 == 0 ? 3 : ALL % 2 == 0 ? 2 : 1;   // fragments read ahead of the products
    static_assert(ALL % C == 0, "whole sets of fragments");
    bf8 qf[2][C];
    auto read = [&](int i) {
#pragma unroll
      for (int u = 0; u < C; ++u) qf[i % 2][u] = *reinterpret_cast<const bf8*>(frag[b] + (i * C + u) * 1024 + lane * 16);
    };
    read(0);
#pragma unroll
    for (int i = 0; i < ALL / C; ++i) {
      if (i + 1 < ALL / C) read(i + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int u = 0; u < C; ++u)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int p = KP - 1; p >= 0; --p) {
            const bf8 kk = kf[j][p][(i * C + u) / NP];
            if constexpr (N == 32) s[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(qf[i % 2][u], kk, s[j], 0, 0, 0);
            else s[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(qf[i % 2][u], kk, s[j], 0, 0, 0);
          }
      __builtin_amdgcn_sched_barrier(0);
    }
    const int p_lo = slot[b][0], p_hi = slot[b][N - 1];
    const bool whole = __builtin_amdgcn_readfirstlane(p_hi >= 0 && all_see(k0, k0 + KEYS - 1, p_lo, p_hi, a.window, a.sinks));
#pragma unroll
    for (int i = 0; i < NV / 4; ++i) {
      const int r0 = 8 * i + 4 * part;
      const float4 l4 = *reinterpret_cast<const float4*>(&lse[b][r0]);
      const float ls[4] = {l4.x, l4.y, l4.z, l4.w};
      if (whole) {
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) sum[j] += __builtin_amdgcn_exp2f(fmaf(s[j][4 * i + r], a.scale, -ls[r]) * LOG2E);
      } else {
        const int4 p4 = *reinterpret_cast<const int4*>(&slot[b][r0]);
        const int ps[4] = {p4.x, p4.y, p4.z, p4.w};
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float y = __builtin_amdgcn_exp2f(fmaf(s[j][4 * i + r], a.scale, -ls[r]) * LOG2E);
            sum[j] += sees(ps[r], k0 + j * N + in, a.window, a.sinks) ? y : 0.f;
          }
      }
    }
  }
  float y = 0.f;                                  // key k0 + lane
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const float t = N == 32 ? sum2(sum[j]) : sum4(sum[j]);
    y = part == j ? t : y;
  }
  if (live) *account = before + y;
}

// Adds the cuts' sums of keys whose rows took several; one thread per key.
__global__ __launch_bounds__(256) void mass_join_kernel(MassArgs a, int keys) {
  const Cache& c = a.c;
  const int h = blockIdx.x, seq = blockIdx.z, key = blockIdx.y * 256 + threadIdx.x;
  int first, n, f_lo, f_hi;
  seq_rows(c, seq, first, n);
  const int len = seq_len(c, seq);
  if (n == 0 || key >= len || too_long(c, seq)) return;
  mass_rows(a, n, len - n, key / keys * keys, keys, f_lo, f_hi);
  if (f_hi - f_lo <= a.cut) return;
  const int pg = page_of(c, key), page = c.table[seq * c.stride + pg];
  if (page < 0 || page >= c.n_pages) return;
  const size_t step = (size_t)c.Hkv * c.width * c.page;
  const float* p = a.part + (size_t)seq * a.cuts * step + (size_t)h * c.width * c.page + key;
  const int cuts = min((f_hi - f_lo + a.cut - 1) / a.cut, a.cuts);
  float y = 0.f;
  for (int i = 0; i < cuts; ++i) y += p[i * step];
  a.mass[((size_t)page * c.Hkv + h) * c.page + (key - pg * c.page)] += y;
}

// ------------------------------------------------------------ eviction
// Which slots of key head h of a sequence stay: n = min(len, keep) of them, the
// first `sinks`, the last `recent`, and of the others those of most attention
// weight, ties to the lowest slot.  A slot's rank is a 32-bit whole number that orders as the
// weights do (NaN above all, a sure slot above that, none for slots past the length), so the
// n-th largest is found bit by bit with one count each.
//
// One workgroup per (sequence, head).  Wave w owns a run of slots, lane by lane; a lane's first NV
// ranks stay in registers, the next NLDS in LDS, what is past those is read again for each
// look (61,440 slots: 54 us, 94 read again).
// A histogram of the ranks' upper 12 bits leaves the few in the cut's bin; those go to a
// list in LDS (where they fit), and two bits at a time, three counts by ballot, give the cut; it
// ends early where a bound has exactly n ranks at or above it.  256 heads of up to 4,800 slots: 14 us;
// 16 of up to 61,440: 55, one workgroup's latencies (table, accounts, histogram, places) on 16 of 256 CUs.
__device__ __forceinline__ uint32_t rank_of(float x) {
  if (x != x) return 0xfffffffeu;
  const uint32_t b = __float_as_uint(x + 0.f);    // -0 counts as 0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

template <int NV, int NLDS>
__global__ __launch_bounds__(1024) void choose_kernel(Cache c, const float* mass, int keep, int sinks, int recent,
                                                      int* new_lens, int* kept) {
  constexpr int BINS = 4096;
  __shared__ uint32_t list[BINS];                 // bins, then the ranks of one
  __shared__ uint32_t rest[NLDS > 0 ? NLDS * 1024 : 1];
  __shared__ int red[2][3][16], eq_of[16], found[4];
  const int h = blockIdx.x, seq = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int len = seq_len(c, seq), n = min(len, keep);
  const int per = (len + 1023) / 1024;            // slots per lane
  const int j0 = wave * per * 64 + lane;
  const int* table = c.table + seq * c.stride;
  int* out = kept + ((size_t)seq * c.Hkv + h) * keep;
  if (tid == 0 && h == 0) new_lens[seq] = n;
  for (int d = n + tid; d < keep; d += 1024) out[d] = -1;
  if (n == 0) return;
  auto rank_at = [&](float x, int j) -> uint32_t {
    return j >= len ? 0u : j < sinks || j >= len - recent ? 0xffffffffu : rank_of(x);
  };
  auto page_at = [&](int j) { return table[page_of(c, min(j, len - 1))]; };
  auto mass_at = [&](int j, int e) -> float {     // NaN where there is no page
    const bool ok = e >= 0 && e < c.n_pages;
    const int jc = min(j, len - 1);
    const float x = mass[((size_t)(ok ? e : 0) * c.Hkv + h) * c.page + (jc - page_of(c, jc) * c.page)];
    return ok ? x : NAN;
  };
  constexpr int SET = 8;                          // slots of a lane whose table entries, then accounts, load together
  auto load = [&](int i0, uint32_t (&x)[SET]) {
    int e[SET];
#pragma unroll
    for (int i = 0; i < SET; ++i) e[i] = page_at(j0 + (i0 + i) * 64);
    float m[SET];
#pragma unroll
    for (int i = 0; i < SET; ++i) m[i] = mass_at(j0 + (i0 + i) * 64, e[i]);
#pragma unroll
    for (int i = 0; i < SET; ++i) x[i] = i0 + i < per ? rank_at(m[i], j0 + (i0 + i) * 64) : 0u;
  };
  uint32_t r[NV / SET][SET];
#pragma unroll
  for (int i0 = 0; i0 < NV; i0 += SET) {
    asm volatile("" ::: "memory");                // one set under way at a time (more spill)
    if (i0 < per) load(i0, r[i0 / SET]);
  }
  for (int i0 = NV; i0 < min(per, NV + NLDS); i0 += SET) {
    uint32_t x[SET];
    load(i0, x);
#pragma unroll
    for (int i = 0; i < SET; ++i) rest[(i0 - NV + i) * 1024 + tid] = x[i];
  }
  // f(rank, i) for this lane's slots
  auto each = [&](auto f) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (i < per) f(r[i / SET][i % SET], i);
    for (int i0 = NV; i0 < per; i0 += SET) {
      uint32_t x[SET];
      if (i0 < NV + NLDS) {
#pragma unroll
        for (int i = 0; i < SET; ++i) x[i] = rest[(i0 - NV + i) * 1024 + tid];
      } else {
        load(i0, x);
      }
#pragma unroll
      for (int i = 0; i < SET; ++i)
        if (i0 + i < per) f(x[i], i0 + i);
    }
  };
  // the bin of the n-th largest rank, from the top: rank >> 20, turned round
  for (int i = tid; i < BINS; i += 1024) list[i] = 0;
  __syncthreads();
  each([&](uint32_t y, int) {
    const int bin = BINS - 1 - (int)(y >> 20), one = __builtin_amdgcn_readfirstlane(bin);
    if (__all(bin == one)) {                      // sure ones and ties: 64 at once
      if (lane == 0) atomicAdd(&list[one], 64u);
    } else {
      atomicAdd(&list[bin], 1u);
    }
  });
  __syncthreads();
  int own[4], sum = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) sum += own[i] = (int)list[4 * tid + i];
  int upto = sum;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int o = __shfl_up(upto, d, 64);
    if (lane >= d) upto += o;
  }
  if (lane == 63) eq_of[wave] = upto;
  __syncthreads();
  for (int u = 0; u < wave; ++u) upto += eq_of[u];
  int before = upto - sum;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (before < n && n <= before + own[i]) { found[0] = 4 * tid + i; found[1] = before; found[2] = own[i]; found[3] = 0; }
    before += own[i];
  }
  __syncthreads();
  // ranks >= cut + 2^20: hi; in the bin: inside
  uint32_t cut = (uint32_t)(BINS - 1 - found[0]) << 20;
  const int hi = found[1], inside = found[2];
  bool exact = hi + inside == n;                  // n ranks are above the cut
  if (exact) --cut;                               // not 0: the live ranks are above it, and at least n
  const bool listed = inside <= BINS;
  if (!exact && listed) {                         // any order: they are only counted
    each([&](uint32_t y, int) {
      const bool in = y - cut < 1u << 20;
      const uint64_t who = __ballot(in);
      if (!who) return;
      int at = 0;
      if (lane == 0) at = atomicAdd(&found[3], __popcll(who));
      at = __builtin_amdgcn_readfirstlane(at) + __popcll(who & ((1ull << lane) - 1));
      if (in) list[at] = y;
    });
    __syncthreads();
  }
  const uint32_t base = cut;
  auto in_bin = [&](auto f) {                     // f(rank) for whole waves, 0 in the place of others
    if (listed) {
      for (int i = wave * 64; i < inside; i += 1024) f(i + lane < inside ? list[i + lane] : 0u);
    } else {
      each([&](uint32_t y, int) { f(y - base < 1u << 20 ? y : 0u); });
    }
  };
  for (int bit = 18; bit >= 0 && !exact; bit -= 2) {
    const uint32_t x = 1u << bit;
    int k1 = 0, k2 = 0, k3 = 0;
    in_bin([&](uint32_t y) {
      k1 += __popcll(__ballot(y >= cut + x));
      k2 += __popcll(__ballot(y >= cut + 2 * x));
      k3 += __popcll(__ballot(y >= cut + 3 * x));
    });
    int(*rd)[16] = red[bit >> 1 & 1];
    if (lane == 0) { rd[0][wave] = k1; rd[1][wave] = k2; rd[2][wave] = k3; }
    __syncthreads();
    int all[3];
#pragma unroll
    for (int u = 0; u < 3; ++u) {
      int v = rd[u][lane & 15];
      v += __builtin_amdgcn_update_dpp(0, v, 0xb1, 0xf, 0xf, true);
      v += __builtin_amdgcn_update_dpp(0, v, 0x4e, 0xf, 0xf, true);
      v += __builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, true);
      v += __builtin_amdgcn_update_dpp(0, v, 0x140, 0xf, 0xf, true);
      all[u] = hi + __builtin_amdgcn_readfirstlane(v);
    }
    const int at = all[2] >= n ? 3 : all[1] >= n ? 2 : all[0] >= n ? 1 : 0;
    cut += at * x;
    if (at > 0 && all[at - 1] == n) {
      --cut;
      exact = true;
    }
  }
  int more = 0, same = 0;
  each([&](uint32_t y, int) { more += __popcll(__ballot(y > cut)); same += __popcll(__ballot(y == cut)); });
  __syncthreads();
  if (lane == 0) { red[0][0][wave] = more; eq_of[wave] = same; }
  __syncthreads();
  int above = 0, pos = 0, ties = 0;               // slots above the cut in all; above it and on it before this wave
#pragma unroll
  for (int u = 0; u < 16; ++u) {
    above += red[0][0][u];
    if (u < wave) { pos += red[0][0][u]; ties += eq_of[u]; }
  }
  const int room = n - above;                     // of those on it, the first ones stay
  each([&](uint32_t y, int i) {
    const uint64_t gt = __ballot(y > cut), eq = __ballot(y == cut), below = (1ull << lane) - 1;
    if (!(gt | eq)) return;
    const int gb = __popcll(gt & below), eb = ties + __popcll(eq & below);
    if (y > cut || (y == cut && eb < room)) out[pos + gb + min(eb, room)] = j0 + i * 64;
    pos += __popcll(gt);
    ties += __popcll(eq);
  });
}

// K, V and weight of the slots that stay, in their order, to the pages of `to`
// [S][to_width]; a slot on a page outside the pool becomes NaN, one for such a
// page is dropped.  Rows as 16-byte pieces, SLOTS slots of a head per workgroup.
// Bound by bytes: 629 MB of BF16 rows (2,400 slots of 32 x 8 heads) in 134 us, 4.7 TB/s of the 5.1 that a large
// copy reaches here; 252 MB of FP32 in 58, 4.3.
template <int PIECES, int SLOTS>
__global__ __launch_bounds__(256) void move_kernel(Cache c, float* mass, const int* kept, int keep, const int* to,
                                                   int64_t to_stride) {
  constexpr int RPW = 256 / PIECES, U = SLOTS / RPW;   // rows at a time, times
  static_assert(SLOTS % RPW == 0, "whole rows");
  const int h = blockIdx.y, seq = blockIdx.z, piece = threadIdx.x % PIECES, r0 = threadIdx.x / PIECES;
  const int n = min(seq_len(c, seq), keep), d0 = blockIdx.x * SLOTS + r0;
  if (blockIdx.x * SLOTS >= n) return;
  const int* out = kept + ((size_t)seq * c.Hkv + h) * keep;
  uint4 k[U], v[U];
  float w[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int d = d0 + u * RPW, j = out[min(d, n - 1)], pg = page_of(c, j), e = c.table[seq * c.stride + pg];
    const bool ok = e >= 0 && e < c.n_pages;
    const size_t row = ((size_t)(ok ? e : 0) * c.Hkv + h) * c.page + (j - pg * c.page);
    k[u] = static_cast<const uint4*>(c.k)[row * PIECES + piece];
    v[u] = static_cast<const uint4*>(c.v)[row * PIECES + piece];
    w[u] = mass[row];
    if (!ok) {
      k[u] = v[u] = make_uint4(~0u, ~0u, ~0u, ~0u);
      w[u] = NAN;
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int d = d0 + u * RPW;
    if (d >= n) break;
    const int pg = page_of(c, d), e = to[seq * to_stride + pg];
    if (e < 0 || e >= c.n_pages) continue;
    const size_t row = ((size_t)e * c.Hkv + h) * c.page + (d - pg * c.page);
    static_cast<uint4*>(c.k)[row * PIECES + piece] = k[u];
    static_cast<uint4*>(c.v)[row * PIECES + piece] = v[u];
    if (piece == 0) mass[row] = w[u];
  }
}

}  // namespace paged
}  // namespace sk
