// RMS norm with the residual's addition and an 8-bit output with scales.
//
//   h = x + r;  y = h * rsqrt(mean(h^2) + eps) * w;  s_g = max_g |y| / top;
//   code = round(y / s_g)  (top 448 for e4m3, 127 for int8; g a row or `group` columns)
//
// The bytes bound it: 7 an element in 16 bits (x, r, the stored h, the code).  So a row is
// read once and stays in registers between its three uses, T threads a row with
// C pieces of 8 columns each.  With many rows C is 2 to 4: 16384 x 2048 bf16 with a scale for
// 128 columns takes 45 to 47 us with 128 threads a row (5.1 TB/s, 79 % of the copy rate; when measured against
// one another, 46.6 us against 56.9 with a warp a row, whose 8 pieces a lane leave 16 warps an SM,
// 50.1 with 64 and 49.4 with 256 threads).  What is left is instructions: 72 % of the issue slots (int8 codes: 2 us more).
// With few rows a piece a thread, since then the latency of one row is all there is (2 x 1536: 2.1 us
// inside a graph).  Rows that are not
// 16-byte aligned, odd widths and groups that are no power of two of pieces take the plain kernel at the end
// (16384 x 2047: 140 us, groups of 41 in 2050: 200 us).
#include <cuda_fp8.h>

#include "../../include/listener_b200.h"
#include "common.cuh"

namespace lb {
namespace {

struct NormArgs {
  const void *x, *res, *w;
  long long x_ld, r_ld;
  int w_f32, rows, dim, group, e4m3;
  float eps, inv_dim, inv_top;
  uint8_t* codes;
  float* scales;
  void* hidden;
};

template <typename T>
__device__ __forceinline__ float load_as_float(const T* p) {
  if constexpr (__is_same(T, float)) return *p;
  else if constexpr (__is_same(T, __half)) return __half2float(*p);
  else return __bfloat162float(*p);
}
template <typename T>
__device__ __forceinline__ void store_from_float(T* p, float v) {
  if constexpr (__is_same(T, float)) *p = v;
  else if constexpr (__is_same(T, __half)) *p = __float2half_rn(v);
  else *p = __float2bfloat16_rn(v);
}

// 8 columns
template <typename T>
struct Piece {
  uint4 raw[sizeof(T) == 4 ? 2 : 1];
};
template <typename T>
__device__ __forceinline__ Piece<T> load_piece(const T* p) {
  Piece<T> v;
  v.raw[0] = reinterpret_cast<const uint4*>(p)[0];
  if constexpr (sizeof(T) == 4) v.raw[1] = reinterpret_cast<const uint4*>(p)[1];
  return v;
}
template <typename T>
__device__ __forceinline__ void widen(const Piece<T>& v, float (&f)[8]) {
  const T* e = reinterpret_cast<const T*>(v.raw);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (__is_same(T, float)) f[i] = e[i];
    else if constexpr (__is_same(T, __half)) f[i] = __half2float(e[i]);
    else f[i] = __bfloat162float(e[i]);
  }
}
template <typename T>
__device__ __forceinline__ void store_piece(T* p, const float (&f)[8]) {
  Piece<T> v;
  T* e = reinterpret_cast<T*>(v.raw);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (__is_same(T, float)) e[i] = f[i];
    else if constexpr (__is_same(T, __half)) e[i] = __float2half_rn(f[i]);
    else e[i] = __float2bfloat16_rn(f[i]);
  }
  reinterpret_cast<uint4*>(p)[0] = v.raw[0];
  if constexpr (sizeof(T) == 4) reinterpret_cast<uint4*>(p)[1] = v.raw[1];
}

// |y| as bits: their order is that of the values, with NaN above all
__device__ __forceinline__ uint32_t size_of(float y) { return __float_as_uint(y) & 0x7fffffffu; }

__device__ __forceinline__ uint8_t code_of(float q, bool e4m3) {
  if (e4m3) return __nv_cvt_float_to_fp8(q, __NV_SATFINITE, __NV_E4M3);
  return static_cast<uint8_t>(static_cast<int8_t>(__float2int_rn(fminf(fmaxf(q, -127.0f), 127.0f))));
}

// y / s with inv close to 1 / s: the product, then what it leaves of y (one fused multiply-add, exact) divided
// the same way (Markstein's correction of a quotient, 1990).  Ties of the codes are those of the quotient.
__device__ __forceinline__ float quotient(float y, float s, float inv) {
  const float q = y * inv;
  return fmaf(fmaf(-q, s, y), inv, q);
}
__device__ __forceinline__ float near_inverse(float s) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(s));
  return y;
}

// The codes of 8 columns whose group's scale is s: round(y / s).  Far from 1 both take a power of two
// first, so that nothing leaves the range of normal numbers.
__device__ __forceinline__ uint2 codes_of(float (&y)[8], float s, bool e4m3) {
  if (!(s > 0.0f && s < INFINITY)) return make_uint2(0, 0);  // all zero, or a value that is not finite: the scale says so
  if (s < 0x1p-90f || s > 0x1p90f) {
    const float k = s < 1.0f ? 0x1p80f : 0x1p-80f;
    s *= k;
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] *= k;
  }
  const float inv = near_inverse(s);
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = quotient(y[i], s, inv);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (e4m3) {
      w[i] = __nv_cvt_float2_to_fp8x2(make_float2(y[2 * i], y[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
    } else {  // a sum with 1.5 * 2^23 rounds to the nearest even and leaves the code in its low byte
      const uint32_t lo = __float_as_uint(fminf(fmaxf(y[2 * i], -127.0f), 127.0f) + 12582912.0f);
      const uint32_t hi = __float_as_uint(fminf(fmaxf(y[2 * i + 1], -127.0f), 127.0f) + 12582912.0f);
      w[i] = __byte_perm(lo, hi, 0x0040);
    }
  }
  return make_uint2(__byte_perm(w[0], w[1], 0x5410), __byte_perm(w[2], w[3], 0x5410));
}

template <typename T, int kT, int C>
__global__ void __launch_bounds__(kT < 256 ? 256 : kT) norm_rows_kernel(const NormArgs a) {
  constexpr int kBlock = kT < 256 ? 256 : kT, kRowsBlock = kBlock / kT, kWarpsRow = kT / 32;
  __shared__ float part[kBlock / 32];
  const int in_row = threadIdx.x % kT, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long row = static_cast<long long>(blockIdx.x) * kRowsBlock + threadIdx.x / kT;
  const bool live = row < a.rows;
  const int pieces = a.dim / 8;
  const T* x = static_cast<const T*>(a.x) + row * a.x_ld;
  const T* res = static_cast<const T*>(a.res) + row * a.r_ld;
  float h[C][8];
  Piece<T> px[C], pr[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int i = in_row + c * kT;
    if (live && i < pieces) {
      px[c] = load_piece<T>(x + i * 8);
      if (a.res) pr[c] = load_piece<T>(res + i * 8);
    }
  }
  float sum = 0.0f;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int i = in_row + c * kT;
#pragma unroll
    for (int e = 0; e < 8; ++e) h[c][e] = 0.0f;
    if (live && i < pieces) {
      widen<T>(px[c], h[c]);
      if (a.res) {
        float r[8];
        widen<T>(pr[c], r);
#pragma unroll
        for (int e = 0; e < 8; ++e) h[c][e] += r[e];
      }
      if (a.hidden) store_piece<T>(static_cast<T*>(a.hidden) + row * a.dim + i * 8, h[c]);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = fmaf(h[c][e], h[c][e], sum);
    }
  }
  sum = warp_sum(sum);
  if constexpr (kWarpsRow > 1) {
    if (lane == 0) part[warp] = sum;
    __syncthreads();
    sum = 0.0f;
#pragma unroll
    for (int k = 0; k < kWarpsRow; ++k) sum += part[warp / kWarpsRow * kWarpsRow + k];
  }
  const float r = rsqrtf(fmaf(sum, a.inv_dim, a.eps));
  uint32_t m[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int i = in_row + c * kT;
    m[c] = 0u;
    if (live && i < pieces) {
      float w[8];
      if (a.w_f32) widen<float>(load_piece<float>(static_cast<const float*>(a.w) + i * 8), w);
      else widen<T>(load_piece<T>(static_cast<const T*>(a.w) + i * 8), w);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        h[c][e] = h[c][e] * r * w[e];
        m[c] = max(m[c], size_of(h[c][e]));
      }
    }
  }
  if (a.group) {
    // a group's pieces are neighbouring lanes
    const int width = a.group / 8, width_log = 31 - __clz(width);
    for (int o = 1; o < width; o <<= 1) {
#pragma unroll
      for (int c = 0; c < C; ++c) m[c] = max(m[c], __shfl_xor_sync(0xffffffffu, m[c], o));
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int i = in_row + c * kT;
      if (live && i < pieces) {
        const float s = __uint_as_float(m[c]) * a.inv_top;
        if ((i & (width - 1)) == 0) a.scales[row * (pieces >> width_log) + (i >> width_log)] = s;
        *reinterpret_cast<uint2*>(a.codes + row * a.dim + i * 8) = codes_of(h[c], s, a.e4m3);
      }
    }
    return;
  }
  uint32_t most = 0u;
#pragma unroll
  for (int c = 0; c < C; ++c) most = max(most, m[c]);
  most = __reduce_max_sync(0xffffffffu, most);
  if constexpr (kWarpsRow > 1) {
    __syncthreads();  // the sums have been read
    if (lane == 0) part[warp] = __uint_as_float(most);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kWarpsRow; ++k) most = max(most, __float_as_uint(part[warp / kWarpsRow * kWarpsRow + k]));
  }
  const float s = __uint_as_float(most) * a.inv_top;
  if (live && in_row == 0) a.scales[row] = s;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int i = in_row + c * kT;
    if (live && i < pieces) *reinterpret_cast<uint2*>(a.codes + row * a.dim + i * 8) = codes_of(h[c], s, a.e4m3);
  }
}

// Any width, alignment and group: kT threads a row (a warp where rows are narrow and many), the row in
// shared memory, a value a load.
template <typename T, int kT>
__global__ void __launch_bounds__(256) norm_any_kernel(const NormArgs a) {
  constexpr int kRowsBlock = 256 / kT;
  extern __shared__ float row_smem[];
  __shared__ float part[8];
  const int in_row = threadIdx.x % kT, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, dim = a.dim;
  const long long row = static_cast<long long>(blockIdx.x) * kRowsBlock + threadIdx.x / kT;
  if (kT == 32 && row >= a.rows) return;  // (one row a CTA: every row is there)
  float* held = row_smem + threadIdx.x / kT * dim;
  const T* x = static_cast<const T*>(a.x) + row * a.x_ld;
  const T* res = a.res ? static_cast<const T*>(a.res) + row * a.r_ld : nullptr;
  T* hidden = a.hidden ? static_cast<T*>(a.hidden) + row * dim : nullptr;
  float sum = 0.0f;
#pragma unroll 4
  for (int i = in_row; i < dim; i += kT) {
    float h = load_as_float<T>(x + i);
    if (res) h += load_as_float<T>(res + i);
    if (hidden) store_from_float<T>(hidden + i, h);
    held[i] = h;
    sum = fmaf(h, h, sum);
  }
  sum = warp_sum(sum);
  if constexpr (kT > 32) {
    if (lane == 0) part[warp] = sum;
    __syncthreads();
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += part[i];
    __syncthreads();  // the sums have been read
  }
  const float r = rsqrtf(fmaf(sum, a.inv_dim, a.eps));
  uint32_t most = 0;
#pragma unroll 4
  for (int i = in_row; i < dim; i += kT) {  // (a thread's own values)
    const float y = held[i] * r * (a.w_f32 ? static_cast<const float*>(a.w)[i] : load_as_float<T>(static_cast<const T*>(a.w) + i));
    held[i] = y;
    most = max(most, size_of(y));
  }
  const auto write = [&](int from, int width, uint32_t m, int first, int step) {
    const float s = __uint_as_float(m) * a.inv_top;
    const bool plain = s > 0x1p-90f && s < 0x1p90f, some = s > 0.0f && s < INFINITY;
    const float inv = plain ? near_inverse(s) : 0.0f;
#pragma unroll 4
    for (int i = first; i < width; i += step) {
      const float y = held[from + i];
      a.codes[row * dim + from + i] = plain ? code_of(quotient(y, s, inv), a.e4m3) : some ? code_of(y / s, a.e4m3) : uint8_t(0);
    }
    return s;
  };
  if (a.group == 0) {
    most = __reduce_max_sync(0xffffffffu, most);
    if constexpr (kT > 32) {
      if (lane == 0) part[warp] = __uint_as_float(most);
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(part[i]));
    }
    const float s = write(0, dim, most, in_row, kT);
    if (in_row == 0) a.scales[row] = s;
    return;
  }
  if constexpr (kT > 32) __syncthreads();
  else __syncwarp();
  const int n_groups = dim / a.group;
  for (int g = in_row / 32; g < n_groups; g += kT / 32) {  // a warp a group
    uint32_t m = 0;
    for (int i = lane; i < a.group; i += 32) m = max(m, size_of(held[g * a.group + i]));
    const float s = write(g * a.group, a.group, __reduce_max_sync(0xffffffffu, m), lane, 32);
    if (lane == 0) a.scales[row * n_groups + g] = s;
  }
}
template <typename T>
cudaError_t launch_any(const NormArgs& a, cudaStream_t s) {
  if (a.rows >= 148 * 8 && a.dim <= 1024) {
    norm_any_kernel<T, 32><<<(a.rows + 7) / 8, 256, 8 * sizeof(float) * a.dim, s>>>(a);
    return cudaGetLastError();
  }
  const size_t smem = sizeof(float) * a.dim;
  if (smem > 40 * 1024) {
    static std::atomic<unsigned long long> done{0};
    const cudaError_t e = ensure_smem(done, reinterpret_cast<const void*>(norm_any_kernel<T, 256>),
                                      16384 * static_cast<int>(sizeof(float)));
    if (e != cudaSuccess) return e;
  }
  norm_any_kernel<T, 256><<<a.rows, 256, smem, s>>>(a);
  return cudaGetLastError();
}

template <typename T, int kT, int C>
cudaError_t launch(const NormArgs& a, cudaStream_t s) {
  constexpr int kBlock = kT < 256 ? 256 : kT, kRowsBlock = kBlock / kT;
  norm_rows_kernel<T, kT, C><<<(a.rows + kRowsBlock - 1) / kRowsBlock, kBlock, 0, s>>>(a);
  return cudaGetLastError();
}
template <typename T>
cudaError_t launch(const NormArgs& a, cudaStream_t s) {
  const int pieces = a.dim / 8;
  if (a.rows < 148 * 8) {  // fewer than a warp a row would fill the SMs with: a piece a thread
    if (pieces <= 256) return launch<T, 256, 1>(a, s);
    return pieces <= 1024 ? launch<T, 1024, 1>(a, s) : launch<T, 1024, 2>(a, s);
  }
  if (pieces <= 32) return launch<T, 32, 1>(a, s);
  if (pieces <= 64) return launch<T, 32, 2>(a, s);
  if (pieces <= 128) return launch<T, 32, 4>(a, s);
  if (pieces <= 256) return launch<T, 128, 2>(a, s);
  if (pieces <= 512) return launch<T, 128, 4>(a, s);
  return pieces <= 1024 ? launch<T, 256, 4>(a, s) : launch<T, 512, 4>(a, s);
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
  const NormArgs a{x, residual, weight, x_ld, residual_ld, weight_dtype == LB_F32, rows, dim, group,
                   out_dtype == LB_E4M3, eps, 1.0f / static_cast<float>(dim), out_dtype == LB_E4M3 ? 1.0f / 448.0f : 1.0f / 127.0f,
                   static_cast<uint8_t*>(codes), scales, hidden};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t size = dtype == LB_F32 ? 4 : 2;
  const auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  const int width = group / 8;  // a group's pieces
  const bool vec = dim % 8 == 0 && aligned(x) && aligned(residual) && aligned(weight) && aligned(hidden) &&
                   reinterpret_cast<uintptr_t>(codes) % 8 == 0 && x_ld * size % 16 == 0 && residual_ld * size % 16 == 0 &&
                   (group == 0 || (group % 8 == 0 && width <= 32 && (width & (width - 1)) == 0));
  cudaError_t e;
  if (vec) e = dtype == LB_F32 ? launch<float>(a, s) : dtype == LB_BF16 ? launch<__nv_bfloat16>(a, s) : launch<__half>(a, s);
  else
    e = dtype == LB_F32 ? launch_any<float>(a, s)
                        : dtype == LB_BF16 ? launch_any<__nv_bfloat16>(a, s) : launch_any<__half>(a, s);
  return e == cudaSuccess ? LB_OK : LB_ERR_CUDA;
}
