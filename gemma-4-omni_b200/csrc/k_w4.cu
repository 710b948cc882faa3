// Matrix-vector products with 4-bit weights and group scales:
//   out[m][o] = sum_g s[o][g] sum_{k in g} (n[o][k] - 8) x[m][k] * xs[m][k / gx]
// A warp an output feature: it reads the feature's codes once, a word (8 codes) a
// lane and step, for all rows of x.
#include <cuda_fp8.h>

#include "../../include/listener_b200.h"
#include "common.cuh"

namespace lb {
namespace {

constexpr int kWarps = 8;
constexpr int kRows = 8;  // rows of x a pass over the weights

__device__ __forceinline__ float x_as_float(const void* p, int dtype, long long i) {
  if (dtype == LB_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  if (dtype == LB_F16) return __half2float(static_cast<const __half*>(p)[i]);
  if (dtype == LB_I8) return static_cast<float>(static_cast<const int8_t*>(p)[i]);
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<const uint8_t*>(p)[i], __NV_E4M3)));
}

__global__ void __launch_bounds__(kWarps * 32) w4_kernel(const void* x, long long x_ld, int x_dtype,
                                                         const float* x_scale, int x_group, int m,
                                                         const uint32_t* codes, const __half* w_scale, int group,
                                                         int out_features, int k, void* out, long long ld_out,
                                                         int out_dtype) {
  const int o = blockIdx.x * kWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (o >= out_features) return;
  const long long words = k / 8;
  const int gx = x_group ? x_group : k;
  for (int m0 = 0; m0 < m; m0 += kRows) {
    float acc[kRows] = {};
    for (int w = lane; w < words; w += 32) {
      const uint32_t c = codes[o * words + w];
      const float s = __half2float(w_scale[static_cast<long long>(o) * (k / group) + w * 8 / group]);
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        if (m0 + r >= m) break;
        const float f = x_scale ? s * x_scale[static_cast<long long>(m0 + r) * (k / gx) + w * 8 / gx] : s;
        float part = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          part = fmaf(static_cast<float>(static_cast<int>((c >> (4 * j)) & 15u) - 8),
                      x_as_float(x, x_dtype, (m0 + r) * x_ld + w * 8 + j), part);
        acc[r] = fmaf(part, f, acc[r]);
      }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const float v = warp_sum(acc[r]);
      if (lane != 0 || m0 + r >= m) continue;
      const long long at = (m0 + r) * ld_out + o;
      if (out_dtype == LB_F32) static_cast<float*>(out)[at] = v;
      else if (out_dtype == LB_BF16) static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(v);
      else static_cast<__half*>(out)[at] = __float2half_rn(v);
    }
  }
}

}  // namespace
}  // namespace lb

extern "C" int lb_op_w4_matvec(const void* x, int64_t x_ld, int x_dtype, const float* x_scale, int x_group, int m,
                               const void* codes, const void* w_scale, int group, int out_features, int k,
                               void* out, int64_t ld_out, int out_dtype, void* stream) {
  using namespace lb;
  if (!x || !codes || !w_scale || !out || m < 1 || out_features < 1 || k < 1 || x_ld < k || ld_out < out_features)
    return LB_ERR_INVALID_ARGUMENT;
  if ((group != 32 && group != 64 && group != 128) || k % group != 0 || reinterpret_cast<uintptr_t>(codes) % 16 != 0)
    return LB_ERR_INVALID_ARGUMENT;
  const bool eight = x_dtype == LB_E4M3 || x_dtype == LB_I8;
  if ((!eight && x_dtype != LB_BF16 && x_dtype != LB_F16) || eight != (x_scale != nullptr))
    return LB_ERR_INVALID_ARGUMENT;
  if (x_group < 0 || (x_group && (!eight || x_group % 128 != 0 || k % x_group != 0))) return LB_ERR_INVALID_ARGUMENT;
  if (out_dtype != LB_F32 && out_dtype != LB_BF16 && out_dtype != LB_F16) return LB_ERR_INVALID_ARGUMENT;
  w4_kernel<<<(out_features + kWarps - 1) / kWarps, kWarps * 32, 0, static_cast<cudaStream_t>(stream)>>>(
      x, x_ld, x_dtype, x_scale, x_group, m, static_cast<const uint32_t*>(codes), static_cast<const __half*>(w_scale),
      group, out_features, k, out, ld_out, out_dtype);
  return cudaGetLastError() == cudaSuccess ? LB_OK : LB_ERR_CUDA;
}
