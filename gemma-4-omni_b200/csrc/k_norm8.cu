// RMS norm with the residual's addition and an 8-bit output with scales.
//
//   h = x + r;  y = h * rsqrt(mean(h^2) + eps) * w;  s_g = max_g |y| / top;
//   code = round(y / s_g)  (top 448 for e4m3, 127 for int8; g a row or `group` columns)
//
// A CTA a row; the row's h stays in shared memory between its three uses.
#include <cuda_fp8.h>

#include "../../include/listener_b200.h"
#include "common.cuh"

namespace lb {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float load_as_float(const void* p, int dtype, long long i) {
  if (dtype == LB_F32) return static_cast<const float*>(p)[i];
  if (dtype == LB_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_from_float(void* p, int dtype, long long i, float v) {
  if (dtype == LB_F32) static_cast<float*>(p)[i] = v;
  else if (dtype == LB_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

// max that keeps a NaN of either side
__device__ __forceinline__ float max_nan(float a, float b) { return (a > b || isnan(a)) ? a : b; }

__device__ __forceinline__ float warp_max_nan(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

__global__ void __launch_bounds__(kThreads) rms_norm8_kernel(const void* x, long long x_ld, const void* res,
                                                             long long r_ld, int dtype, const void* w, int w_dtype,
                                                             int dim, float eps, int group, int e4m3, uint8_t* codes,
                                                             float* scales, void* hidden) {
  extern __shared__ float row_smem[];
  __shared__ float part[kThreads / 32];
  const long long row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  float sum = 0.0f;
  for (int i = tid; i < dim; i += kThreads) {
    float h = load_as_float(x, dtype, row * x_ld + i);
    if (res) h += load_as_float(res, dtype, row * r_ld + i);
    if (hidden) store_from_float(hidden, dtype, row * dim + i, h);
    row_smem[i] = h;
    sum = fmaf(h, h, sum);
  }
  sum = warp_sum(sum);
  if (lane == 0) part[warp] = sum;
  __syncthreads();
  sum = 0.0f;
  for (int i = 0; i < kThreads / 32; ++i) sum += part[i];
  const float r = rsqrtf(sum / static_cast<float>(dim) + eps);
  for (int i = tid; i < dim; i += kThreads) row_smem[i] = row_smem[i] * r * load_as_float(w, w_dtype, i);
  __syncthreads();
  const int width = group ? group : dim, n_groups = dim / width;
  const float top = e4m3 ? 448.0f : 127.0f;
  for (int g = group ? warp : 0; g < n_groups; g += group ? kThreads / 32 : 1) {
    // a warp a group; for one scale a row every warp finds the row's maximum
    float m = 0.0f;
    for (int i = lane; i < width; i += 32) m = max_nan(m, fabsf(row_smem[g * width + i]));
    const float s = warp_max_nan(m) / top;
    if (lane == 0 && (group || warp == 0)) scales[row * n_groups + g] = s;
    for (int i = group ? lane : tid; i < width; i += group ? 32 : kThreads) {
      const float q = s > 0.0f ? row_smem[g * width + i] / s : 0.0f;
      uint8_t c;
      if (e4m3) c = __nv_cvt_float_to_fp8(q, __NV_SATFINITE, __NV_E4M3);
      else c = static_cast<uint8_t>(static_cast<int8_t>(__float2int_rn(fminf(fmaxf(q, -127.0f), 127.0f))));
      codes[row * dim + g * width + i] = c;
    }
  }
}

}  // namespace
}  // namespace lb

extern "C" int lb_op_rms_norm8(const void* x, int64_t x_ld, const void* residual, int64_t residual_ld, int dtype,
                               const void* weight, int weight_dtype, int rows, int dim, float eps, int group,
                               int out_dtype, void* codes, float* scales, void* hidden, void* stream) {
  using namespace lb;
  if (!x || !weight || !codes || !scales || rows < 1 || dim < 1 || dim > 16384 || x_ld < dim ||
      (residual && residual_ld < dim) || group < 0 || (group && dim % group != 0))
    return LB_ERR_INVALID_ARGUMENT;
  if ((dtype != LB_F32 && dtype != LB_BF16 && dtype != LB_F16) || (weight_dtype != LB_F32 && weight_dtype != dtype) ||
      (out_dtype != LB_E4M3 && out_dtype != LB_I8))
    return LB_ERR_INVALID_ARGUMENT;
  const size_t smem = sizeof(float) * dim;
  if (smem > 40 * 1024 && cudaFuncSetAttribute(rms_norm8_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               16384 * static_cast<int>(sizeof(float))) != cudaSuccess)
    return LB_ERR_CUDA;
  rms_norm8_kernel<<<rows, kThreads, smem, static_cast<cudaStream_t>(stream)>>>(
      x, x_ld, residual, residual_ld, dtype, weight, weight_dtype, dim, eps, group, out_dtype == LB_E4M3,
      static_cast<uint8_t*>(codes), scales, hidden);
  return cudaGetLastError() == cudaSuccess ? LB_OK : LB_ERR_CUDA;
}
