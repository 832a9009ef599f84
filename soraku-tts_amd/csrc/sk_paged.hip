// Operator API: the attention half of a trunk layer over a cache in pages
// (append, attention, accounts of attention weight, eviction), on a caller
// stream.  The layer's arithmetic is that of the reference's trunk
// (modeling_qwen3.py:237-262); pages, window and eviction have no counterpart there.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <numeric>

#include "sk_error.h"
#include "sk_paged.h"
#include "soraku_mi355x.h"

using namespace sk;
using namespace sk::paged;

namespace {

constexpr int MOST = 65535;                       // of a grid's y and z

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// What every entry point asks of its sizes.
int check_sizes(int32_t T, int32_t S, int32_t Hq, int32_t Hkv, int32_t hd, int32_t page, int32_t n_pages, int32_t width,
                int64_t stride) {
  // a row or tile finds its sequence by a pass over all S: more of them belong in several calls
  SK_CHECK(T >= 0 && T < 1 << 24 && S > 0 && S <= MOST, SK_EINVAL, "T must be in [0, 2^24) and S in [1, %d]", MOST);
  SK_CHECK(Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && Hq <= 4096, SK_EINVAL,
           "Hq must be a positive multiple of Hkv, at most 4096");
  SK_CHECK(hd == 16 || hd == 32 || hd == 64 || hd == 128, SK_EINVAL, "hd must be a power of two in [16, 128]");
  SK_CHECK(page > 0 && page % TILE == 0, SK_EINVAL, "page must be a positive multiple of %d", TILE);
  SK_CHECK(n_pages > 0 && width > 0 && stride >= width, SK_EINVAL,
           "n_pages and width must be positive, and the table's rows at least width entries apart");
  SK_CHECK((int64_t)page * width <= INT32_MAX / 2, SK_EINVAL, "width * page must be at most 2^30 tokens");
  SK_CHECK((int64_t)T * Hq <= INT32_MAX / 2, SK_EINVAL, "T * Hq must be at most 2^30");
  return SK_OK;
}
int check_types(int32_t xdtype, int32_t kvdtype) {
  SK_CHECK((xdtype == SK_F32 && (kvdtype == SK_F32 || kvdtype == SK_BF16)) || (xdtype == SK_BF16 && kvdtype == SK_BF16),
           SK_EINVAL, "types must be float32 on either cache, or bfloat16 on a bfloat16 cache");
  return SK_OK;
}
int check_window(float scale, int32_t window, int32_t sinks) {
  SK_CHECK(scale > 0.f && scale <= 1e30f, SK_EINVAL, "scale must be positive and at most 1e30");
  SK_CHECK(window >= 0 && sinks >= 0, SK_EINVAL, "window and sinks must not be negative");
  return SK_OK;
}

Cache cache_of(int32_t T, int32_t S, int32_t Hq, int32_t Hkv, int32_t page, int32_t n_pages, int32_t width,
               int64_t stride, const int32_t* starts, const int32_t* lens, const int32_t* table, const void* k,
               const void* v) {
  int bits = 4;                                   // 2^bits >= page
  while ((int64_t)1 << bits < page) ++bits;
  const uint32_t mul = (uint32_t)((((uint64_t)1 << (31 + bits)) + page - 1) / page);
  return {const_cast<void*>(k), const_cast<void*>(v), table, stride, width, starts, lens, T, S, Hq, Hkv, Hq / Hkv,
          n_pages, page, mul, 31 + bits};
}

template <int N> using Int = std::integral_constant<int, N>;
template <typename F>
void with_hd(int hd, F&& f) {
  switch (hd) {
    case 16: f(Int<16>{}); break;
    case 32: f(Int<32>{}); break;
    case 64: f(Int<64>{}); break;
    default: f(Int<128>{}); break;
  }
}
// f(a value of the activations' type, one of the cache's)
template <typename F>
void with_types(int32_t xdtype, int32_t kvdtype, F&& f) {
  if (xdtype == SK_BF16) f(uint16_t{}, uint16_t{});
  else if (kvdtype == SK_BF16) f(float{}, uint16_t{});
  else f(float{}, float{});
}

// How an attention call is cut up: R rows per workgroup (of 64-key steps on the
// BF16 matrix cores: `tiles`; else WK waves that share the keys), `cut` tiles of keys per cut.
struct Plan {
  bool tiles;
  int R, WK, blocks, cut, cuts;
};
Plan plan_attention(int T, int S, int Hq, int Hkv, int hd, int xdtype, int kvdtype, int page, int width, int window,
                    int sinks) {
  Plan p;
  const int G = Hq / Hkv;
  const int64_t rows = (int64_t)T * G / S;        // of a sequence, on average
  const bool bf16 = kvdtype == SK_BF16 && hd >= 32;
  // tiles of n G rows: at most R - gcd(G, R) of a sequence's last one are empty
  auto blocks = [&](int R) { return ((int64_t)T * G + (int64_t)std::min(S, T) * (R - std::gcd(G, R))) / R; };
  const int64_t keys = window > 0 ? std::min((int64_t)page * width, (int64_t)window + sinks) : (int64_t)page * width;
  // Up to 1,024 keys, and where tiles of 16 rows still fit on the GPU at once, those start and end sooner
  // (FP32 on BF16, 16 heads on 8: a prompt of 33 tokens 8 us against 12, of 200 10 against 17 + 4; eight
  // of 200, past that bound: 22 by tiles of 128 rows).
  const bool small = keys <= 1024 && blocks(16) * Hkv <= 512;
  p.tiles = bf16 && rows > 32 && !small;
  // 32 rows where the registers hold them (not as three parts of 128 dims) and every CU has a workgroup, two on
  // the FP32 matrix cores, whose long walks then even out (prompts of 194 and 387: 22 us, 28 by tiles of 32 on 304
  // workgroups; of 2,047: 189 by 32 on 1,024, 199 by 16; 30 x 16 BF16 tokens of up to 2,000: 36 by 32, 43 by 16)
  const bool pairs = rows > 16 && (xdtype == kvdtype || hd < 128) && blocks(32) * Hkv >= (bf16 ? 256 : 512);
  p.R = p.tiles ? 128 : pairs ? 32 : 16;
  p.blocks = (int)blocks(p.R);
  int64_t most = (int64_t)page * width / TILE;    // tiles that a row tile can walk
  if (window > 0)
    most = std::min(most, ((int64_t)window + p.R / G + 2) / TILE + 2 + ((int64_t)sinks + TILE - 1) / TILE);
  const int64_t base = std::max<int64_t>((int64_t)p.blocks * Hkv, 1);
  // A CU draws some 40 GB/s, so keys are cut until every CU has a workgroup (two of the tile kernel's), down to
  // one round of a workgroup's waves: a pair of FP32 rows over 481 tokens takes 17 us uncut, with 8 waves or
  // not, 7 + 4 in 8 cuts.  Past that a cut only adds its parts and a launch (32 BF16 rows of up to 657: 17 us
  // uncut, 18 + 4 in two), and below six rounds it saves less than the launch (FP32 on BF16, 128 tokens: 9 us
  // uncut, 16 + 4 in two).  8 waves where each still has 8 tiles (a pair over 61,441: 74 us in 32 cuts by 4
  // waves, 66 in 16 by 8).
  const int64_t round = p.tiles || !bf16 ? 4 : 8;
  const int64_t most_cuts = std::min<int64_t>({(p.tiles ? 512 : 256) / base, most / round, 64});
  const int64_t cuts = most < 6 * round ? 1 : std::max<int64_t>(1, most_cuts);
  p.cut = (int)((most + cuts - 1) / cuts + 3) / 4 * 4;   // whole steps of 64 keys
  p.cuts = (int)((most + p.cut - 1) / p.cut);
  p.WK = p.R == 16 && base * p.cuts <= 256 && p.cut >= 64 ? 8 : 4;
  return p;
}

// Keys per workgroup of a call for accounts, and its rows per cut.
struct MassPlan {
  bool tiles, few;
  int keys, cut, cuts;
  int64_t blocks;
};
constexpr int NK2 = 2;                            // key tiles per wave of mass_kernel
MassPlan plan_mass(int T, int S, int Hq, int Hkv, int hd, int kvdtype, int page, int width) {
  MassPlan p;
  const int64_t rows = (int64_t)T * (Hq / Hkv);
  p.few = rows <= 16ll * S;
  p.tiles = hd >= 32 && (kvdtype == SK_BF16 || !p.few);   // few FP32 rows: FP32 products are enough beside K's bytes
  p.keys = !p.tiles ? 4 * NK2 * TILE : kvdtype == SK_BF16 ? 4 * 64 : 4 * 32;
  p.blocks = ((int64_t)page * width + p.keys - 1) / p.keys;
  const int64_t base = p.blocks * Hkv * S;
  const int64_t cuts = p.tiles && !p.few ? std::max<int64_t>(1, std::min<int64_t>(12 * 256 / base, rows / 256)) : 1;
  p.cut = (int)std::max<int64_t>(32, ((rows + cuts - 1) / cuts + 31) / 32 * 32);
  p.cuts = (int)std::max<int64_t>(1, (rows + p.cut - 1) / p.cut);
  return p;
}
int check_mass(const MassPlan& p, int S) {
  SK_CHECK(p.blocks <= MOST && (int64_t)S * p.cuts <= MOST, SK_EINVAL, "width * page must be at most %lld for accounts",
           (long long)MOST * p.keys);
  return SK_OK;
}
int64_t workspace_of(const MassPlan& p, int S, int Hkv, int page, int width) {
  return p.cuts > 1 ? (int64_t)p.cuts * S * Hkv * page * width * 4 : 0;
}
int64_t workspace_of(const Plan& p, int T, int Hq, int hd) {
  return p.cuts > 1 ? ((int64_t)p.cuts * (hd + 2) + 1) * T * Hq * 4 : 0;
}

}  // namespace

extern "C" {

int sk_op_paged_append(void* stream, int32_t T, int32_t S, int32_t Hq, int32_t Hkv, int32_t hd, int32_t page,
                       int32_t n_pages, int32_t width, int64_t table_stride, int32_t xdtype, int32_t kvdtype, float eps,
                       const void* qkv, const float* q_gain, const float* k_gain, const float* inv_freq,
                       const int32_t* positions, const int32_t* starts, const int32_t* lens, const int32_t* table,
                       void* k_pages, void* v_pages, float* mass, void* q_out) {
  if (int rc = check_sizes(T, S, Hq, Hkv, hd, page, n_pages, width, table_stride)) return rc;
  if (int rc = check_types(xdtype, kvdtype)) return rc;
  SK_CHECK(eps >= 0.f && isfinite(eps), SK_EINVAL, "eps must be finite and not negative");
  if (T == 0) return SK_OK;
  SK_CHECK(qkv && inv_freq && positions && starts && lens && table && k_pages && v_pages && q_out, SK_EINVAL,
           "NULL operand");
  SK_CHECK(!q_gain == !k_gain, SK_EINVAL, "gains of q and k come together");
  SK_CHECK(q_out != qkv, SK_EINVAL, "q_out must not be qkv");
  SK_CHECK(aligned16(qkv) && aligned16(q_gain) && aligned16(k_gain) && aligned16(k_pages) && aligned16(v_pages) &&
               aligned16(q_out),
           SK_EINVAL, "operands must be 16-byte aligned");
  const Cache c = cache_of(T, S, Hq, Hkv, page, n_pages, width, table_stride, starts, lens, table, k_pages, v_pages);
  with_hd(hd, [&](auto d) {
    with_types(xdtype, kvdtype, [&](auto x, auto k) {
      using X = decltype(x);
      using K = decltype(k);
      hipLaunchKernelGGL((append_kernel<X, K, decltype(d)::value>), dim3(T), dim3(256), 0, (hipStream_t)stream, c,
                         (const X*)qkv, q_gain, k_gain, inv_freq, positions, eps, mass, (X*)q_out);
    });
  });
  SK_HIP(hipGetLastError());
  return SK_OK;
}

int sk_op_paged_attention_workspace(int32_t T, int32_t S, int32_t Hq, int32_t Hkv, int32_t hd, int32_t page,
                                    int32_t width, int32_t xdtype, int32_t kvdtype, int32_t window, int32_t sinks,
                                    int64_t* bytes) {
  if (int rc = check_sizes(T, S, Hq, Hkv, hd, page, 1, width, width)) return rc;
  if (int rc = check_types(xdtype, kvdtype)) return rc;
  if (int rc = check_window(1.f, window, sinks)) return rc;
  SK_CHECK(bytes, SK_EINVAL, "NULL operand");
  *bytes = workspace_of(plan_attention(T, S, Hq, Hkv, hd, xdtype, kvdtype, page, width, window, sinks), T, Hq, hd);
  return SK_OK;
}

int sk_op_paged_attention(void* stream, int32_t T, int32_t S, int32_t Hq, int32_t Hkv, int32_t hd, int32_t page,
                          int32_t n_pages, int32_t width, int64_t table_stride, int32_t xdtype, int32_t kvdtype,
                          float scale, int32_t window, int32_t sinks, const void* q, const void* k_pages,
                          const void* v_pages, const int32_t* table, const int32_t* starts, const int32_t* lens,
                          void* out, float* lse, void* workspace, int64_t workspace_bytes) {
  if (int rc = check_sizes(T, S, Hq, Hkv, hd, page, n_pages, width, table_stride)) return rc;
  if (int rc = check_types(xdtype, kvdtype)) return rc;
  if (int rc = check_window(scale, window, sinks)) return rc;
  if (T == 0) return SK_OK;
  SK_CHECK(q && k_pages && v_pages && table && starts && lens && out, SK_EINVAL, "NULL operand");
  SK_CHECK(aligned16(q) && aligned16(k_pages) && aligned16(v_pages) && aligned16(out) && aligned16(workspace), SK_EINVAL,
           "operands must be 16-byte aligned");
  SK_CHECK(out != q, SK_EINVAL, "out must not be q");
  const Plan p = plan_attention(T, S, Hq, Hkv, hd, xdtype, kvdtype, page, width, window, sinks);
  SK_CHECK(p.cuts == 1 || (workspace && workspace_bytes >= workspace_of(p, T, Hq, hd)), SK_EINVAL,
           "the workspace must hold %lld bytes", (long long)workspace_of(p, T, Hq, hd));
  AttendArgs a;
  a.c = cache_of(T, S, Hq, Hkv, page, n_pages, width, table_stride, starts, lens, table, k_pages, v_pages);
  a.q = q; a.out = out; a.lse = lse;
  a.scale2 = scale * LOG2E;
  a.window = window; a.sinks = sinks;
  a.cut = p.cut;
  const bool cut = p.cuts > 1;
  a.part = cut ? (float*)workspace : nullptr;
  a.ml = cut ? a.part + (size_t)p.cuts * T * Hq * hd : nullptr;
  a.count = cut ? (int*)(a.ml + (size_t)p.cuts * T * Hq * 2) : nullptr;
  const hipStream_t st = (hipStream_t)stream;
  hipError_t err = hipSuccess;
  with_hd(hd, [&](auto d) {
    with_types(xdtype, kvdtype, [&](auto x, auto k) {
      using X = decltype(x);
      using K = decltype(k);
      constexpr int HD = decltype(d)::value;
      // the kernels that share keys, with 16 NT rows and WK waves
      auto share = [&](dim3 grid, auto nt, auto wk) {
        constexpr int NT = decltype(nt)::value, WK = decltype(wk)::value;
        if constexpr (HD >= 32 && sizeof(K) == 2) {
          if constexpr (NT == 1 || sizeof(X) * HD <= 256)
            hipLaunchKernelGGL((attend_few_kernel<X, HD, NT, WK>), grid, dim3(64 * WK), 0, st, a);
        } else {
          hipLaunchKernelGGL((attend_rows_kernel<X, K, HD, NT, WK>), grid, dim3(64 * WK), 0, st, a);
        }
      };
      // as many row tiles per launch as a grid takes
      for (a.last = p.blocks - 1; a.last >= 0 && err == hipSuccess; a.last -= MOST) {
        const dim3 grid(Hkv, std::min(a.last + 1, MOST), p.cuts);
        if (p.tiles) {
          if constexpr (HD >= 32 && sizeof(K) == 2)
            hipLaunchKernelGGL((attend_tiles_kernel<X, HD>), grid, dim3(256), 0, st, a);
        } else if (p.R == 32) {
          share(grid, Int<2>{}, Int<4>{});
        } else {
          if (p.WK == 8) share(grid, Int<1>{}, Int<8>{});
          else share(grid, Int<1>{}, Int<4>{});
        }
        err = hipGetLastError();
      }
      if (p.cuts == 1 || err != hipSuccess) return;
      // 4 waves per row where there are few rows with many cuts to go through
      if (p.cuts > 16) hipLaunchKernelGGL((combine_kernel<X, HD, 4>), dim3(T * Hq), dim3(256), 0, st, a, p.cuts);
      else hipLaunchKernelGGL((combine_kernel<X, HD, 1>), dim3((T * Hq + 3) / 4), dim3(256), 0, st, a, p.cuts);
      err = hipGetLastError();
    });
  });
  SK_HIP(err);
  return SK_OK;
}

int sk_op_paged_attention_mass_workspace(int32_t T, int32_t S, int32_t Hq, int32_t Hkv, int32_t hd, int32_t page,
                                         int32_t width, int32_t xdtype, int32_t kvdtype, int64_t* bytes) {
  if (int rc = check_sizes(T, S, Hq, Hkv, hd, page, 1, width, width)) return rc;
  if (int rc = check_types(xdtype, kvdtype)) return rc;
  SK_CHECK(bytes, SK_EINVAL, "NULL operand");
  const MassPlan p = plan_mass(T, S, Hq, Hkv, hd, kvdtype, page, width);
  if (int rc = check_mass(p, S)) return rc;
  *bytes = workspace_of(p, S, Hkv, page, width);
  return SK_OK;
}

int sk_op_paged_attention_mass(void* stream, int32_t T, int32_t S, int32_t Hq, int32_t Hkv, int32_t hd, int32_t page,
                               int32_t n_pages, int32_t width, int64_t table_stride, int32_t xdtype, int32_t kvdtype,
                               float scale, int32_t window, int32_t sinks, const void* q, const float* lse,
                               const void* k_pages, const int32_t* table, const int32_t* starts, const int32_t* lens,
                               float* mass, void* workspace, int64_t workspace_bytes) {
  if (int rc = check_sizes(T, S, Hq, Hkv, hd, page, n_pages, width, table_stride)) return rc;
  if (int rc = check_types(xdtype, kvdtype)) return rc;
  if (int rc = check_window(scale, window, sinks)) return rc;
  if (T == 0) return SK_OK;
  SK_CHECK(q && lse && k_pages && table && starts && lens && mass, SK_EINVAL, "NULL operand");
  SK_CHECK(aligned16(q) && aligned16(k_pages) && aligned16(workspace), SK_EINVAL, "operands must be 16-byte aligned");
  const MassPlan p = plan_mass(T, S, Hq, Hkv, hd, kvdtype, page, width);
  if (int rc = check_mass(p, S)) return rc;
  const int64_t need = workspace_of(p, S, Hkv, page, width);
  SK_CHECK(p.cuts == 1 || (workspace && workspace_bytes >= need), SK_EINVAL, "the workspace must hold %lld bytes",
           (long long)need);
  MassArgs a;
  a.c = cache_of(T, S, Hq, Hkv, page, n_pages, width, table_stride, starts, lens, table, k_pages, nullptr);
  a.q = q; a.lse = lse; a.mass = mass;
  a.scale = scale; a.window = window; a.sinks = sinks;
  a.cut = p.cut; a.cuts = p.cuts;
  a.part = (float*)workspace;
  const hipStream_t st = (hipStream_t)stream;
  hipError_t err = hipSuccess;
  with_hd(hd, [&](auto d) {
    with_types(xdtype, kvdtype, [&](auto x, auto k) {
      using X = decltype(x);
      using K = decltype(k);
      constexpr int HD = decltype(d)::value;
      const dim3 grid(Hkv, (unsigned)p.blocks, S * p.cuts);
      if constexpr (HD >= 32) {
        if (p.tiles && !p.few)
          hipLaunchKernelGGL((mass_tiles_kernel<X, K, HD, 32>), grid, dim3(256), 0, st, a);
        else if constexpr (sizeof(K) == 2)
          hipLaunchKernelGGL((mass_tiles_kernel<X, K, HD, 16>), grid, dim3(256), 0, st, a);
        else
          hipLaunchKernelGGL((mass_kernel<X, K, HD, NK2>), grid, dim3(256), 0, st, a);
      } else {
        hipLaunchKernelGGL((mass_kernel<X, K, HD, NK2>), grid, dim3(256), 0, st, a);
      }
      err = hipGetLastError();
    });
  });
  SK_HIP(err);
  if (p.cuts > 1) {
    hipLaunchKernelGGL(mass_join_kernel, dim3(Hkv, (unsigned)(((int64_t)page * width + 255) / 256), S), dim3(256), 0, st, a,
                       p.keys);
    SK_HIP(hipGetLastError());
  }
  return SK_OK;
}

int sk_op_paged_evict(void* stream, int32_t S, int32_t Hkv, int32_t hd, int32_t page, int32_t n_pages, int32_t width,
                      int64_t table_stride, int32_t kvdtype, int32_t keep, int32_t sinks, int32_t recent, void* k_pages,
                      void* v_pages, float* mass, const int32_t* table, const int32_t* lens, const int32_t* to,
                      int64_t to_stride, int32_t to_width, int32_t* new_lens, int32_t* kept) {
  if (int rc = check_sizes(0, S, Hkv, Hkv, hd, page, n_pages, width, table_stride)) return rc;
  if (int rc = check_types(SK_F32, kvdtype)) return rc;
  SK_CHECK(keep > 0 && sinks >= 0 && recent >= 0 && (int64_t)sinks + recent <= keep, SK_EINVAL,
           "keep must be positive, sinks and recent not negative, and their sum at most keep");
  SK_CHECK(to_width > 0 && to_stride >= to_width && (int64_t)to_width * page >= keep, SK_EINVAL,
           "the new table must have pages for keep tokens");
  SK_CHECK((int64_t)S * Hkv * keep <= INT32_MAX, SK_EINVAL, "S * Hkv * keep must be below 2^31");
  SK_CHECK(k_pages && v_pages && mass && table && lens && to && new_lens && kept, SK_EINVAL, "NULL operand");
  SK_CHECK(table != to, SK_EINVAL, "the new table must have pages of its own");
  SK_CHECK(lens != new_lens, SK_EINVAL, "new_lens must not be lens");
  SK_CHECK(aligned16(k_pages) && aligned16(v_pages), SK_EINVAL, "operands must be 16-byte aligned");
  const Cache c = cache_of(0, S, Hkv, Hkv, page, n_pages, width, table_stride, nullptr, lens, table, k_pages, v_pages);
  const hipStream_t st = (hipStream_t)stream;
  auto choose = [&](auto nv, auto nlds) {
    hipLaunchKernelGGL((choose_kernel<decltype(nv)::value, decltype(nlds)::value>), dim3(Hkv, S), dim3(1024), 0, st, c,
                       mass, keep, sinks, recent, new_lens, kept);
  };
  const int64_t cap = (int64_t)page * width;
  if (cap <= 8 * 1024) choose(Int<8>{}, Int<0>{});
  else if (cap <= 32 * 1024) choose(Int<32>{}, Int<0>{});
  else choose(Int<32>{}, Int<32>{});
  SK_HIP(hipGetLastError());
  const int pieces = hd * (kvdtype == SK_BF16 ? 2 : 4) / 16;
  auto move = [&](auto np) {
    constexpr int P = decltype(np)::value, SLOTS = 256 / P * 4;
    hipLaunchKernelGGL((move_kernel<P, SLOTS>), dim3((keep + SLOTS - 1) / SLOTS, Hkv, S), dim3(256), 0, st, c, mass,
                       (const int*)kept, keep, to, to_stride);
  };
  switch (pieces) {
    case 2: move(Int<2>{}); break;
    case 4: move(Int<4>{}); break;
    case 8: move(Int<8>{}); break;
    case 16: move(Int<16>{}); break;
    default: move(Int<32>{}); break;
  }
  SK_HIP(hipGetLastError());
  return SK_OK;
}

}  // extern "C"
