// Attention over the paged 8-bit cache.
//
//   x_j = cap(scale * sk[page(j)] * q . kc_j),  p_j = exp(x_j - max),  j <= position, j > position - window
//   out = sum_j p_j sv[page(j)] vc_j / sum_j p_j,  lse = max + log sum_j p_j
//
// A warp a (token, head): each lane holds dim / 32 columns and the running maximum
// and sum pass over the keys once.
#include "../../include/listener_b200.h"
#include "common.cuh"

namespace lb {
namespace {

struct AttendArgs {
  const void* q;
  long long q_token_stride, q_head_stride;
  int n_tokens, n_rows, heads, kv_heads;
  const int8_t *k_codes, *v_codes;
  const float *k_scale, *v_scale;
  int n_pages, page_tokens, max_pages;
  const int *row_tables, *kv_len, *cu_tokens;
  float scale, softcap;
  int window;
  void* out;
  float* lse;
  int* status;
};

template <typename T>
__device__ __forceinline__ float to_f(T v) {
  if constexpr (sizeof(T) == 2 && __is_same(T, __half)) return __half2float(v);
  else return __bfloat162float(v);
}

template <typename T, int D>
__global__ void __launch_bounds__(128) attend_kernel(AttendArgs a) {
  constexpr int E = D / 32;
  const long long item = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (item >= static_cast<long long>(a.n_tokens) * a.heads) return;
  const int t = static_cast<int>(item / a.heads), h = static_cast<int>(item - static_cast<long long>(t) * a.heads);
  const int hk = h / (a.heads / a.kv_heads), P = a.page_tokens;
  int lo = 0, hi = a.n_rows - 1;  // last row that begins at or before the token
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.cu_tokens[mid] <= t) lo = mid; else hi = mid - 1;
  }
  const int begin = a.cu_tokens[lo], end = a.cu_tokens[lo + 1];
  int stop = 0, start = 0;
  if (t >= begin && t < end) {
    const long long room = static_cast<long long>(a.max_pages) * P;
    const int len = static_cast<int>(min(static_cast<long long>(a.kv_len[lo]), room));
    stop = min(len, a.kv_len[lo] - (end - begin) + (t - begin) + 1);
    if (a.window) start = max(0, a.kv_len[lo] - (end - begin) + (t - begin) + 1 - a.window);
  }
  const T* q = static_cast<const T*>(a.q) + t * a.q_token_stride + h * a.q_head_stride + lane * E;
  float qv[E], acc[E] = {};
#pragma unroll
  for (int i = 0; i < E; ++i) qv[i] = to_f<T>(q[i]);
  float m = -INFINITY, total = 0.0f;
  for (int j = start; j < stop; ++j) {
    const int page = a.row_tables[static_cast<long long>(lo) * a.max_pages + j / P];
    if (page < 0 || page >= a.n_pages) {
      if (a.status && lane == 0) atomicOr(a.status, static_cast<int>(LB_DEV_BAD_PAGE));
      continue;
    }
    const long long ph = static_cast<long long>(page) * a.kv_heads + hk;
    const long long at = (ph * P + j % P) * D + lane * E;
    float x = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) x = fmaf(qv[i], static_cast<float>(a.k_codes[at + i]), x);
    x = warp_sum(x) * a.k_scale[ph] * a.scale;
    if (a.softcap > 0.0f) x = a.softcap * tanhf(x / a.softcap);
    const float m1 = fmaxf(m, x), f = expf(m - m1), p = expf(x - m1), pv = p * a.v_scale[ph];
    total = total * f + p;
#pragma unroll
    for (int i = 0; i < E; ++i) acc[i] = fmaf(pv, static_cast<float>(a.v_codes[at + i]), acc[i] * f);
    m = m1;
  }
  T* out = static_cast<T*>(a.out) + item * D + lane * E;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const float y = total != 0.0f ? acc[i] / total : 0.0f;
    if constexpr (__is_same(T, __half)) out[i] = __float2half_rn(y);
    else out[i] = __float2bfloat16_rn(y);
  }
  if (a.lse && lane == 0) a.lse[item] = total != 0.0f ? m + logf(total) : -INFINITY;
}

template <typename T>
cudaError_t launch(const AttendArgs& a, int dim, cudaStream_t s) {
  const unsigned ctas = static_cast<unsigned>((static_cast<long long>(a.n_tokens) * a.heads + 3) / 4);
  if (dim == 64) attend_kernel<T, 64><<<ctas, 128, 0, s>>>(a);
  else if (dim == 128) attend_kernel<T, 128><<<ctas, 128, 0, s>>>(a);
  else attend_kernel<T, 256><<<ctas, 128, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace
}  // namespace lb

extern "C" int lb_op_kv8_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, int q_dtype,
                                   int n_tokens, int n_rows, int heads, int kv_heads, int dim,
                                   const int8_t* k_codes, const int8_t* v_codes, const float* k_scale,
                                   const float* v_scale, int n_pages, int page_tokens, const int32_t* row_tables,
                                   int max_pages, const int32_t* kv_len, const int32_t* cu_tokens, float scale,
                                   int window, float softcap, void* out, float* lse, int32_t* status,
                                   void* stream) {
  using namespace lb;
  if (!q || !k_codes || !v_codes || !k_scale || !v_scale || !row_tables || !kv_len || !cu_tokens || !out ||
      n_tokens < 1 || n_rows < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || n_pages < 1 ||
      max_pages < 1 || window < 0 || !(softcap >= 0.0f))
    return LB_ERR_INVALID_ARGUMENT;
  if ((q_dtype != LB_BF16 && q_dtype != LB_F16) || (dim != 64 && dim != 128 && dim != 256) || page_tokens < 16 ||
      page_tokens > 256 || page_tokens % 16 != 0 || static_cast<long long>(max_pages) * page_tokens > 0x7fffffffll)
    return LB_ERR_INVALID_ARGUMENT;
  if (static_cast<long long>(n_tokens) * heads > 0x7fffffffll) return LB_ERR_CAPACITY;
  const auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  if (!aligned(k_codes) || !aligned(v_codes)) return LB_ERR_INVALID_ARGUMENT;
  AttendArgs a{q, q_token_stride, q_head_stride, n_tokens, n_rows, heads, kv_heads, k_codes, v_codes, k_scale, v_scale,
               n_pages, page_tokens, max_pages, row_tables, kv_len, cu_tokens, scale, softcap, window, out, lse, status};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = q_dtype == LB_BF16 ? launch<__nv_bfloat16>(a, dim, s) : launch<__half>(a, dim, s);
  return e == cudaSuccess ? LB_OK : LB_ERR_CUDA;
}
