// Operator API: sampling of many rows, each with its own parameters, on a caller stream
// (the reference's _sample_logits, soraku_inference/model.py:686-708, takes one).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "sk_draw.h"
#include "sk_error.h"
#include "soraku_mi355x.h"

using namespace sk;
using namespace sk::draw;

namespace {

constexpr int MOST_ROWS = 65535, MOST_V = 1 << 20;

int check_sizes(int32_t R, int32_t V, int32_t dtype) {
  SK_CHECK(R >= 0 && R <= MOST_ROWS, SK_EINVAL, "R must be in [0, %d]", MOST_ROWS);
  SK_CHECK(V > 0 && V <= MOST_V, SK_EINVAL, "V must be in [1, 2^20]");
  SK_CHECK(dtype == SK_F32 || dtype == SK_BF16, SK_EINVAL, "dtype must be SK_F32 or SK_BF16");
  return SK_OK;
}
// Workgroups per row: one of the GPU's 256 CUs each, as few rows allow, but no more than ten, whose histograms every
// one of them adds up. Calls one after the other over changing logits, FP32: a row of 151,936 88 us whole, 44 in 3, 29 in 8, 27 in
// 10; 64 of them 62 us in 2, 48 in 4, 69 in 5 (BF16 60, 42 and 61); 256 114 us whole, 136 in 2. Short rows stay whole, as
// a second launch costs more: 12,000 values 17.5 us whole, 20 to 21 in 2 to 10; 16,384 19.6 and 20.5 to 22; 32,000 27.5 and 22.
int slices_of(int R, int V) { return V <= 16384 ? 1 : std::max(1, std::min(MOST_SLICES, 256 / std::max(R, 1))); }
// Sums of V weights of up to 2^bits stay below 2^63.
int bits_of(int V) {
  int b = 0;
  while ((1 << b) < V) ++b;
  return std::min(46, 62 - b);
}

template <typename X, bool WIDE>
int run(const Args& a, hipStream_t st) {
  if (a.slices == 1) {
    if (a.V <= Held<X>::N * NT) hipLaunchKernelGGL((held_kernel<X>), dim3(a.R), dim3(NT), 0, st, a);
    else hipLaunchKernelGGL((row_kernel<X, WIDE>), dim3(a.R), dim3(NT), 0, st, a);
    SK_HIP(hipGetLastError());
    return SK_OK;
  }
  const dim3 grid(a.slices, a.R);
  hipLaunchKernelGGL((slice_kernel<X, WIDE>), grid, dim3(NT), 0, st, a);
  SK_HIP(hipGetLastError());
  hipLaunchKernelGGL((pick_kernel<X, WIDE>), grid, dim3(NT), 0, st, a);
  SK_HIP(hipGetLastError());
  return SK_OK;
}

}  // namespace

extern "C" {

int sk_op_sample_rows_workspace(int32_t R, int32_t V, int32_t dtype, int64_t* bytes) {
  if (int rc = check_sizes(R, V, dtype)) return rc;
  SK_CHECK(bytes, SK_EINVAL, "NULL operand");
  const int n = slices_of(R, V);
  *bytes = n > 1 ? (int64_t)R * RowSpace::bytes(n) : 0;
  return SK_OK;
}

int sk_op_sample_rows(void* stream, int32_t R, int32_t V, int32_t dtype, const void* logits, int64_t stride, const double* u,
                      const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                      const float* cfg_scale, const uint32_t* allowed, int64_t allowed_stride, int64_t* token, float* logprob,
                      int32_t* kept, void* workspace, int64_t workspace_bytes) {
  if (int rc = check_sizes(R, V, dtype)) return rc;
  SK_CHECK(stride >= V, SK_EINVAL, "rows of logits must be at least V apart");
  SK_CHECK(!allowed || allowed_stride == 0 || allowed_stride >= (V + 31) / 32, SK_EINVAL,
           "rows of allowed must be at least V / 32 words apart, or 0 for one row");
  if (R == 0) return SK_OK;
  SK_CHECK(logits && u && token, SK_EINVAL, "NULL operand");
  SK_CHECK(((uintptr_t)workspace & 15) == 0, SK_EINVAL, "the workspace must be 16-byte aligned");
  Args a{logits, stride, u, temperature, top_k, top_p, min_p, cfg_scale, allowed, allowed_stride, R, V, bits_of(V),
         slices_of(R, V), 0, token, logprob, kept, (char*)workspace};
  // whole pieces of 16 bytes to a slice
  a.slice = ((V + a.slices - 1) / a.slices + 7) / 8 * 8;
  const int64_t need = a.slices > 1 ? (int64_t)R * RowSpace::bytes(a.slices) : 0;
  SK_CHECK(need == 0 || (workspace && workspace_bytes >= need), SK_EINVAL, "the workspace must hold %lld bytes", (long long)need);
  const int64_t size = dtype == SK_BF16 ? 2 : 4;
  const bool wide = (uintptr_t)logits % 16 == 0 && stride * size % 16 == 0 && V * size % 16 == 0;
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == SK_BF16) return wide ? run<uint16_t, true>(a, st) : run<uint16_t, false>(a, st);
  return wide ? run<float, true>(a, st) : run<float, false>(a, st);
}

}  // extern "C"
