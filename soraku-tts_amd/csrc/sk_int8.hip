// Operator API: projections with 8-bit weights, on a caller stream.  The reference
// keeps its weights in FP32 or BF16 (soraku_inference/model.py:100-145); the projections are those of its trunk and
// depth head (modeling_qwen3.py:81-84, model.py:82-98).
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "sk_error.h"
#include "sk_int8.h"
#include "soraku_mi355x.h"

using namespace sk;
using namespace sk::int8;

namespace {

constexpr int MOST_K = (1 << 17) - 128;           // 127 * 128 * K stays below 2^31

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
int padded(int K) { return (K + GROUP - 1) / GROUP * GROUP; }

int check_type(int32_t xdtype) {
  SK_CHECK(xdtype == SK_F32 || xdtype == SK_BF16, SK_EINVAL, "xdtype must be SK_F32 or SK_BF16");
  return SK_OK;
}
int check_linear(int32_t M, int32_t N, int32_t K, int32_t xdtype, int32_t act) {
  SK_CHECK(M >= 0 && M < 1 << 24, SK_EINVAL, "M must be in [0, 2^24)");
  SK_CHECK(N > 0 && N <= 1 << 20, SK_EINVAL, "N must be in [1, 2^20]");
  SK_CHECK(K > 0 && K <= MOST_K, SK_EINVAL, "K must be in [1, %d]", MOST_K);
  SK_CHECK(act == SK_ACT_NONE || act == SK_ACT_SWIGLU, SK_EINVAL, "act must be SK_ACT_NONE or SK_ACT_SWIGLU");
  return check_type(xdtype);
}

// A wave per row where rows are short and many (12,288 of 2,048), four where not, so that 32 rows spread
// over as many CUs; up to 8,192 values stay in registers.
template <typename X, int MODE>
void launch_rows_as(const RowsArgs& a, hipStream_t st) {
  auto go = [&](auto kernel, int per) { hipLaunchKernelGGL(kernel, dim3((a.R + per - 1) / per), dim3(256), 0, st, a); };
  if (a.K % 8 != 0) go(rows_kernel<X, 4, 0, false, MODE>, 1);
  else if (a.Kp <= 2048 && a.R >= 1024) {
    if (a.Kp <= 512) go(rows_kernel<X, 1, 1, true, MODE>, 4);
    else if (a.Kp <= 1024) go(rows_kernel<X, 1, 2, true, MODE>, 4);
    else go(rows_kernel<X, 1, 4, true, MODE>, 4);
  } else {
    if (a.Kp <= 2048) go(rows_kernel<X, 4, 1, true, MODE>, 1);
    else if (a.Kp <= 4096) go(rows_kernel<X, 4, 2, true, MODE>, 1);
    else if (a.Kp <= 8192) go(rows_kernel<X, 4, 4, true, MODE>, 1);
    else go(rows_kernel<X, 4, 0, true, MODE>, 1);
  }
}
template <typename X>
void launch_rows(const RowsArgs& a, hipStream_t st) {
  if (a.eps < 0.f) launch_rows_as<X, PLAIN>(a, st);
  else if (a.gain) launch_rows_as<X, GAIN>(a, st);
  else launch_rows_as<X, NORM>(a, st);
}

// How a product is computed: by few_kernel, whose workgroups take few rows and columns and may code the rows
// themselves, or in tiles.
struct Plan {
  bool fused, few;
  int kind, bm, bn;                               // of FEW or TILES; rows and columns (SwiGLU: gate and up together) of a workgroup
};
// Estimated us of few_kernel when a CU has r workgroups, which each load u units of `tiles` tiles of 16 rows: 2.1 + 0.9
// (r - 1) + 0.0265 r u tiles, a CU's 75 GB/s (16 to 256 rows of six projections: within 15%, but 30 to 40% less than SwiGLU products
// of 25 MB, which come from HBM).  E.g. 32 rows of 2048 x 6144: 16 rows by 16 columns 4.6 us, 32 by 32 6.8, in tiles
// of 64 x 64 15.4; 128 rows: 32 by 32 7.1, 64 by 32 9.4, 64 x 64 15.2; 256 rows of 4096 x 2048: 64 by 32 9.6, 64 x 64 7.6.
struct Few { int mt, nt; };
constexpr Few FEW[] = {{1, 1}, {2, 1}, {1, 2}, {2, 2}, {4, 2}};   // SwiGLU: from the third on
// Estimated us of a launch of tiles when a CU has r of them, of u stages: fix + r round + u lat + (r - 1) u thr, fitted
// to 207 times of launches one after the other with inputs in cache (33 to 7,680 rows, the trunks' projections and odd ones; rms error 7 to
// 24%, and 28% too little for the long one below).  It is there to choose, and the tile chosen is on average within 6% of the fastest (SwiGLU
// 3%).  Measured with inputs in cache, then from memory: 7,680 rows of 2 x 6144 x 2048: 256 x 256 199 and 201 us, 128 x 128 221 and
// 247; 5,999 of 2048 x 6144 (51 estimated): 192 x 256 71 and 78, 256 x 256 77 and 83, 128 x 128 91 and 107; 774 of 4096 x 1024 (128 x
// 128 taken, 9.5 estimated): 64 x 128 9.1 and 11.4, 128 x 128 10.0 and 12.7, 256 x 256 16.1 and 18.9; 64 of 2048 x 6144: 64 x 64 15.2 and
// 17.7, 64 x 128 21.5 and 45.
struct Tile { int bm, bn, waves; float fix, round, lat, thr, fix2, round2, lat2, thr2; };   // 2: SwiGLU
constexpr Tile TILES[] = {{256, 256, 16, 0.f, 7.19f, 1.10f, 2.28f, 0.f, 8.47f, 1.15f, 1.87f},
                          {192, 256, 8, 0.f, 7.00f, .92f, 1.53f, 0.f, 7.23f, 1.00f, 1.40f},
                          {128, 128, 4, .98f, 4.06f, .56f, .37f, 2.16f, 1.92f, .62f, .49f},
                          {64, 128, 4, 2.07f, 1.73f, .41f, .26f, 2.27f, .75f, .44f, .31f},
                          {64, 64, 4, 1.93f, 1.35f, .26f, .18f, 2.31f, 1.04f, .42f, .19f}};
// Up to 8 rows the workgroups code the rows themselves where each wave then has at most 2,048 values (2 rows x 4096 x
// 2048: 5.6 us, with a launch for the codes 7 in two).
Plan plan_linear(int M, int N, int K, bool swiglu) {
  const int rows2 = M > 4 ? 8 : M > 2 ? 4 : M;
  Plan p{};
  if (M <= 8 && rows2 * K <= 16384) {
    p.few = p.fused = true;
    p.bm = 16;
    p.bn = swiglu ? 32 : 16;
    return p;
  }
  const float u = (float)(padded(K) / 128);
  float best = 1e30f;
  auto take = [&](bool few, int kind, int bm, int bn, auto us) {
    const int nc = swiglu ? bn / 2 : bn;
    const int64_t groups = (int64_t)((M + bm - 1) / bm) * ((N + nc - 1) / nc);
    const float t = us((float)((groups + 255) / 256));
    if (t < best) { best = t; p = Plan{false, few, kind, bm, bn}; }
  };
  for (int i = swiglu ? 2 : 0; i < (int)(sizeof(FEW) / sizeof(Few)) && M <= 1024; ++i) {
    const Few f = FEW[i];
    take(true, i, f.mt * 16, f.nt * 16, [&](float r) { return 2.1f + .9f * (r - 1) + .0265f * r * u * (f.mt + f.nt); });
  }
  for (int i = 0; i < (int)(sizeof(TILES) / sizeof(Tile)); ++i) {
    const Tile& t = TILES[i];
    take(false, i, t.bm, t.bn, [&](float r) {
      return swiglu ? t.fix2 + r * t.round2 + u * (t.lat2 + (r - 1) * t.thr2) : t.fix + r * t.round + u * (t.lat + (r - 1) * t.thr);
    });
  }
  return p;
}
int cols_of(const Plan& p, bool swiglu) { return swiglu ? p.bn / 2 : p.bn; }
// Workspace: the activations' codes, then their scales.
int64_t codes_of(int M, int K) { return ((int64_t)M * padded(K) + 255) / 256 * 256; }
int64_t space_of(const Plan& p, int M, int K) { return p.fused || M == 0 ? 0 : codes_of(M, K) + (int64_t)M * 4; }

template <typename X, bool SWIGLU>
void launch_few(const Plan& p, const LinearArgs& a, const RowsArgs& r, hipStream_t st) {
  auto go = [&](auto kernel, int waves) { hipLaunchKernelGGL(kernel, dim3(a.nt, a.mt), dim3(waves * 64), 0, st, a, r); };
  constexpr int NT = SWIGLU ? 2 : 1;
  if (p.fused) {
    if (r.K % 8 == 0) go(few_kernel<X, SWIGLU, true, true, 1, NT, 8, 3>, 8);
    else go(few_kernel<X, SWIGLU, true, false, 1, NT, 8, 3>, 8);
    return;
  }
  switch (p.kind) {
    case 0: if constexpr (!SWIGLU) go(few_kernel<X, SWIGLU, false, true, 1, 1, 8, 2>, 8); break;
    case 1: if constexpr (!SWIGLU) go(few_kernel<X, SWIGLU, false, true, 2, 1, 8, 2>, 8); break;
    case 2: go(few_kernel<X, SWIGLU, false, true, 1, 2, 8, 2>, 8); break;
    case 3: go(few_kernel<X, SWIGLU, false, true, 2, 2, 8, 2>, 8); break;
    default: go(few_kernel<X, SWIGLU, false, true, 4, 2, 4, 2>, 4); break;
  }
}
template <typename X, bool SWIGLU>
void launch_tiles(const Plan& p, const LinearArgs& a, hipStream_t st) {
  auto go = [&](auto kernel, int waves) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)((a.mt * a.nt + 7) / 8 * 8)), dim3(waves * 64), 0, st, a);
  };
  switch (p.kind) {
    case 0: go(tiles_kernel<X, SWIGLU, 256, 256, 4, 4, 2>, 16); break;
    case 1: go(tiles_kernel<X, SWIGLU, 192, 256, 2, 4, 2>, 8); break;
    case 2: go(tiles_kernel<X, SWIGLU, 128, 128, 2, 2, 2>, 4); break;
    case 3: go(tiles_kernel<X, SWIGLU, 64, 128, 2, 2, 2>, 4); break;
    default:
      if constexpr (SWIGLU) go(tiles_kernel<X, SWIGLU, 64, 64, 2, 1, 3>, 2);
      else go(tiles_kernel<X, SWIGLU, 64, 64, 2, 2, 4>, 4);
      break;
  }
}

template <typename X>
int run_linear(hipStream_t st, const Plan& p, const LinearArgs& a, const RowsArgs& r, bool swiglu) {
  if (!p.fused) {
    launch_rows<X>(r, st);
    SK_HIP(hipGetLastError());
  }
  if (p.few) swiglu ? launch_few<X, true>(p, a, r, st) : launch_few<X, false>(p, a, r, st);
  else swiglu ? launch_tiles<X, true>(p, a, st) : launch_tiles<X, false>(p, a, st);
  SK_HIP(hipGetLastError());
  return SK_OK;
}

}  // namespace

extern "C" {

int sk_op_int8_rows(void* stream, int32_t R, int32_t K, int32_t xdtype, const void* x, int8_t* codes, float* scales) {
  SK_CHECK(R >= 0 && R < 1 << 24, SK_EINVAL, "R must be in [0, 2^24)");
  SK_CHECK(K > 0 && K <= MOST_K, SK_EINVAL, "K must be in [1, %d]", MOST_K);
  if (int rc = check_type(xdtype)) return rc;
  if (R == 0) return SK_OK;
  SK_CHECK(x && codes && scales, SK_EINVAL, "NULL operand");
  SK_CHECK(aligned16(x) && aligned16(codes), SK_EINVAL, "operands must be 16-byte aligned");
  const RowsArgs a{x, nullptr, -1.f, R, K, padded(K), codes, scales, 1.0 / K};
  if (xdtype == SK_BF16) launch_rows<uint16_t>(a, (hipStream_t)stream);
  else launch_rows<float>(a, (hipStream_t)stream);
  SK_HIP(hipGetLastError());
  return SK_OK;
}

int sk_op_int8_linear_workspace(int32_t M, int32_t N, int32_t K, int32_t xdtype, int32_t act, int64_t* bytes) {
  if (int rc = check_linear(M, N, K, xdtype, act)) return rc;
  SK_CHECK(bytes, SK_EINVAL, "NULL operand");
  *bytes = space_of(plan_linear(M, N, K, act == SK_ACT_SWIGLU), M, K);
  return SK_OK;
}

int sk_op_int8_linear(void* stream, int32_t M, int32_t N, int32_t K, int32_t xdtype, int32_t act, float eps,
                      const void* x, const float* gain, const int8_t* codes, const float* scales, const float* bias,
                      const void* residual, void* out, void* workspace, int64_t workspace_bytes) {
  if (int rc = check_linear(M, N, K, xdtype, act)) return rc;
  SK_CHECK(isfinite(eps), SK_EINVAL, "eps must be finite");
  SK_CHECK(eps >= 0.f || !gain, SK_EINVAL, "a gain needs eps >= 0");
  if (M == 0) return SK_OK;
  SK_CHECK(x && codes && scales && out, SK_EINVAL, "NULL operand");
  SK_CHECK(aligned16(x) && aligned16(gain) && aligned16(codes) && aligned16(residual) && aligned16(out) &&
               aligned16(workspace),
           SK_EINVAL, "operands must be 16-byte aligned");
  SK_CHECK(out != x, SK_EINVAL, "out must not be x");
  const bool swiglu = act == SK_ACT_SWIGLU;
  const Plan p = plan_linear(M, N, K, swiglu);
  const int64_t need = space_of(p, M, K);
  SK_CHECK(need == 0 || (workspace && workspace_bytes >= need), SK_EINVAL, "the workspace must hold %lld bytes",
           (long long)need);
  char* ws = static_cast<char*>(workspace);
  const int nc = cols_of(p, swiglu);
  LinearArgs a{};
  a.a = p.fused ? nullptr : (int8_t*)ws;
  a.as = p.fused ? nullptr : (float*)(ws + codes_of(M, K));
  a.w = codes; a.ws = scales; a.bias = bias; a.res = residual; a.out = out;
  a.M = M; a.N = N; a.Kp = padded(K);
  a.mt = (M + p.bm - 1) / p.bm; a.nt = (N + nc - 1) / nc; a.gm = 8;
  SK_CHECK(p.few || ((int64_t)a.mt * a.nt + 7) * TILES[p.kind].waves * 64 < (int64_t)1 << 32, SK_EINVAL,
           "M * N is too large: several calls are needed");   // a launch has less than 2^32 threads
  const RowsArgs r{x, gain, eps, M, K, padded(K), const_cast<int8_t*>(a.a), const_cast<float*>(a.as), 1.0 / K};
  return xdtype == SK_BF16 ? run_linear<uint16_t>((hipStream_t)stream, p, a, r, swiglu)
                           : run_linear<float>((hipStream_t)stream, p, a, r, swiglu);
}

}  // extern "C"
