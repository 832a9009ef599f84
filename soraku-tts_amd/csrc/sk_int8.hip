// Operator API: projections with 8-bit weights, on a caller stream.  The reference
// keeps its weights in FP32 or BF16 (soraku_inference/model.py:100-145); the projections are those of its trunk and
// depth head (modeling_qwen3.py:81-84, model.py:82-98).
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

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

template <typename X, int W>
void launch_rows_w(const RowsArgs& a, hipStream_t st) {
  const dim3 grid((a.R + 4 / W - 1) / (4 / W));
  switch ((a.Kp + W * 512 - 1) / (W * 512)) {
    case 1: hipLaunchKernelGGL((rows_kernel<X, W, 1>), grid, dim3(256), 0, st, a); break;
    case 2: hipLaunchKernelGGL((rows_kernel<X, W, 2>), grid, dim3(256), 0, st, a); break;
    case 3:
    case 4: hipLaunchKernelGGL((rows_kernel<X, W, 4>), grid, dim3(256), 0, st, a); break;
    default: hipLaunchKernelGGL((rows_kernel<X, W, 0>), grid, dim3(256), 0, st, a); break;
  }
}
template <typename X>
void launch_rows(const RowsArgs& a, hipStream_t st) {
  if (a.Kp <= 2048 && a.R >= 1024) launch_rows_w<X, 1>(a, st);
  else launch_rows_w<X, 4>(a, st);
}

// How a product is computed.
struct Plan {
  bool fused, few;
  int bm, bn, ksplit;                             // tile (few: 16 MT x 16 NT), cuts of K
};
Plan plan_linear(int M, int N, int K, bool swiglu) {
  const int rows2 = M > 4 ? 8 : M > 2 ? 4 : M;
  Plan p{};
  p.ksplit = 1;
  p.few = M <= 64;
  p.fused = M <= 8 && rows2 * K <= 16384;
  if (p.few) {
    p.bm = M <= 16 ? 16 : M <= 32 ? 32 : 64;
    p.bn = swiglu ? 32 : 16;
  } else {
    p.bm = p.bn = 128;
  }
  return p;
}
int cols_of(const Plan& p, bool swiglu) { return swiglu ? p.bn / 2 : p.bn; }
int64_t tiles_of(const Plan& p, int M, int N, bool swiglu) {
  const int nc = cols_of(p, swiglu);
  return (int64_t)((M + p.bm - 1) / p.bm) * ((N + nc - 1) / nc);
}
// Workspace: the activations' codes, their scales, then tickets and sums of the cuts.
struct Space { int64_t scales, tickets, parts, bytes; };
Space space_of(const Plan& p, int M, int N, int K, bool swiglu) {
  auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
  Space s{};
  if (p.fused || M == 0) return s;
  const int64_t tiles = tiles_of(p, M, N, swiglu);
  s.scales = up((int64_t)M * padded(K));
  s.tickets = s.scales + up((int64_t)M * 4);
  s.parts = s.tickets + (p.ksplit > 1 ? up(tiles * 4) : 0);
  s.bytes = s.parts + (p.ksplit > 1 ? tiles * p.ksplit * p.bm * p.bn * 4 : 0);
  return s;
}

template <typename X, bool SWIGLU>
void launch_few(const Plan& p, LinearArgs a, const RowsArgs& r, hipStream_t st) {
  const dim3 grid(a.nt * a.ksplit, a.mt);
  constexpr int NT = SWIGLU ? 2 : 1;
  auto go = [&](auto kernel, int W, int MT, bool fused) {
    const size_t codes = fused ? (size_t)a.M * (a.Kp + 16) : 0;
    hipLaunchKernelGGL(kernel, grid, dim3(W * 64), std::max<size_t>(codes, (size_t)W * MT * NT * 1024), st, a, r);
  };
  if (p.fused) go(few_kernel<X, SWIGLU, true, 1, NT, 8>, 8, 1, true);
  else if (p.bm == 16) go(few_kernel<X, SWIGLU, false, 1, NT, 8>, 8, 1, false);
  else if (p.bm == 32) go(few_kernel<X, SWIGLU, false, 2, NT, 8>, 8, 2, false);
  else go(few_kernel<X, SWIGLU, false, 4, NT, 4>, 4, 4, false);
}
template <typename X, bool SWIGLU>
void launch_tiles(const Plan&, const LinearArgs& a, hipStream_t st) {
  const int tiles = a.mt * a.nt;
  hipLaunchKernelGGL((tiles_kernel<X, SWIGLU, 128, 128, 2, 2, 3>), dim3((tiles + 7) / 8 * 8), dim3(256), 0, st, a);
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
  const RowsArgs a{x, nullptr, -1.f, R, K, padded(K), codes, scales, nullptr, 0};
  if (xdtype == SK_BF16) launch_rows<uint16_t>(a, (hipStream_t)stream);
  else launch_rows<float>(a, (hipStream_t)stream);
  SK_HIP(hipGetLastError());
  return SK_OK;
}

int sk_op_int8_linear_workspace(int32_t M, int32_t N, int32_t K, int32_t xdtype, int32_t act, int64_t* bytes) {
  if (int rc = check_linear(M, N, K, xdtype, act)) return rc;
  SK_CHECK(bytes, SK_EINVAL, "NULL operand");
  const bool swiglu = act == SK_ACT_SWIGLU;
  *bytes = space_of(plan_linear(M, N, K, swiglu), M, N, K, swiglu).bytes;
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
  const Space s = space_of(p, M, N, K, swiglu);
  SK_CHECK(s.bytes == 0 || (workspace && workspace_bytes >= s.bytes), SK_EINVAL, "the workspace must hold %lld bytes",
           (long long)s.bytes);
  char* ws = static_cast<char*>(workspace);
  const int nc = cols_of(p, swiglu);
  LinearArgs a{};
  a.a = p.fused ? nullptr : (int8_t*)ws;
  a.as = p.fused ? nullptr : (float*)(ws + s.scales);
  a.w = codes; a.ws = scales; a.bias = bias; a.res = residual; a.out = out;
  a.M = M; a.N = N; a.Kp = padded(K);
  a.mt = (M + p.bm - 1) / p.bm; a.nt = (N + nc - 1) / nc; a.ksplit = p.ksplit; a.gm = 8;
  if (p.ksplit > 1) { a.ticket = (int*)(ws + s.tickets); a.part = (int*)(ws + s.parts); }
  const RowsArgs r{x, gain, eps, M, K, padded(K), const_cast<int8_t*>(a.a), const_cast<float*>(a.as), a.ticket,
                   p.ksplit > 1 ? a.mt * a.nt : 0};
  return xdtype == SK_BF16 ? run_linear<uint16_t>((hipStream_t)stream, p, a, r, swiglu)
                           : run_linear<float>((hipStream_t)stream, p, a, r, swiglu);
}

}  // extern "C"
