// New keys and values written into the 8-bit cache.
//
// A group is the run of batch tokens that follow one another in one page, first at
// offset o.  For each kv head and side:
//   s1 = max(s0, max |x| / 127)  (s0 the page's scale, 0 when the page begins here)
//   codes before o: c -> rint(c * s0 / s1) where the scale grew; new: rint(x / s1)
// so value = code * scale holds for the whole page with one scale, and a page is
// only touched where its scale grows.
//
// A warp a (group, head, side): the maximum and the codes need no exchange
// beyond it, and the groups of a tick (one or two tokens) keep a warp busy each.  The
// warps look for the first tokens of groups in windows of the batch, so nothing
// but the slots has to be known: a token begins a group unless the token before
// it in the batch has the slot before it in the same page.
#include "../../include/listener_b200.h"
#include "common.cuh"

namespace lb {
namespace {

constexpr int kWarps = 8;

struct AppendArgs {
  const void* src[2];
  long long token_stride[2], head_stride[2];
  int8_t* codes[2];
  float* scale[2];
  const long long* slots;
  int n_tokens, kv_heads, dim, n_pages, page_tokens, window;
  int* status;
};

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// 8 elements; VEC: 16-byte loads (the row starts are 16-byte aligned)
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  if constexpr (VEC) {
    alignas(16) T raw[8];
    const int4* s = reinterpret_cast<const int4*>(p);
    int4* d = reinterpret_cast<int4*>(raw);
#pragma unroll
    for (int i = 0; i < static_cast<int>(8 * sizeof(T) / 16); ++i) d[i] = s[i];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_float<T>(raw[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_float<T>(p[i]);
  }
}

// rint(x / s) within +-127; NaN (0 / 0 or a NaN x) -> 0
__device__ __forceinline__ int code_of(float x, float s) {
  const float q = __fdiv_rn(x, s);
  return isnan(q) ? 0 : __float2int_rn(fminf(fmaxf(q, -127.0f), 127.0f));
}

__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d) {
  return (a & 0xff) | (b & 0xff) << 8 | (c & 0xff) << 16 | static_cast<uint32_t>(d) << 24;
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kWarps * 32) append_kernel(AppendArgs a) {
  const int lane = threadIdx.x & 31;
  const long long item = static_cast<long long>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int per_window = 2 * a.kv_heads;
  const long long win = item / per_window;
  const int which = static_cast<int>(item - win * per_window);
  const int side = which & 1, head = which >> 1;
  const long long t0 = win * a.window;
  if (t0 >= a.n_tokens) return;
  const int P = a.page_tokens, D = a.dim, chunks = D / 8;

  bool first = false;
  if (lane < a.window && t0 + lane < a.n_tokens) {
    const long long s = a.slots[t0 + lane];
    first = s >= 0 && (s % P == 0 || t0 + lane == 0 || a.slots[t0 + lane - 1] + 1 != s);
  }
  const T* src = static_cast<const T*>(side ? a.src[1] : a.src[0]) + head * (side ? a.head_stride[1] : a.head_stride[0]);
  const long long ts = side ? a.token_stride[1] : a.token_stride[0];
  for (unsigned todo = __ballot_sync(0xffffffffu, first); todo; todo &= todo - 1) {
    const long long t = t0 + __ffs(todo) - 1;
    const long long slot = a.slots[t], page = slot / P;
    const int off = static_cast<int>(slot - page * P);
    if (page >= a.n_pages) {
      if (lane == 0 && a.status) atomicOr(a.status, static_cast<int>(LB_DEV_BAD_PAGE));
      continue;
    }
    int run = 1;
    while (true) {
      const int j = run + lane;
      const bool next = off + j < P && t + j < a.n_tokens && a.slots[t + j] == slot + j;
      const unsigned all = __ballot_sync(0xffffffffu, next);
      if (all != 0xffffffffu) {
        run += __ffs(~all) - 1;
        break;
      }
      run += 32;
    }
    const T* from = src + t * ts;
    float most = 0.0f;
    bool odd = false;  // an infinite value or a NaN
    for (int c = lane; c < run * chunks; c += 32) {
      const int j = c / chunks;
      float v[8];
      load8<T, VEC>(from + j * ts + (c - j * chunks) * 8, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float m = fabsf(v[i]);
        if (m < INFINITY) most = fmaxf(most, m);
        else odd = true;
      }
    }
    most = warp_max(most);
    if (odd && a.status) atomicOr(a.status, static_cast<int>(LB_DEV_NONFINITE));
    float* scale = (side ? a.scale[1] : a.scale[0]) + page * a.kv_heads + head;
    const float s0 = off > 0 ? *scale : 0.0f;
    const float s1 = fmaxf(s0, __fdiv_rn(most, 127.0f));
    int8_t* base = (side ? a.codes[1] : a.codes[0]) + (page * a.kv_heads + head) * static_cast<long long>(P) * D;
    if (s1 != s0) {
      for (int c = lane; c < off * (D / 16); c += 32) {
        int4* at = reinterpret_cast<int4*>(base) + c;
        int4 raw = *at;
        uint32_t w[4] = {static_cast<uint32_t>(raw.x), static_cast<uint32_t>(raw.y), static_cast<uint32_t>(raw.z),
                         static_cast<uint32_t>(raw.w)};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          int q[4];
#pragma unroll
          for (int b = 0; b < 4; ++b) q[b] = code_of(static_cast<float>(static_cast<int8_t>(w[i] >> (8 * b))) * s0, s1);
          w[i] = pack4(q[0], q[1], q[2], q[3]);
        }
        *at = make_int4(w[0], w[1], w[2], w[3]);
      }
    }
    for (int c = lane; c < run * chunks; c += 32) {
      const int j = c / chunks, d = (c - j * chunks) * 8;
      float v[8];
      load8<T, VEC>(from + j * ts + d, v);
      int q[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) q[i] = code_of(v[i], s1);
      *reinterpret_cast<uint2*>(base + static_cast<long long>(off + j) * D + d) =
          make_uint2(pack4(q[0], q[1], q[2], q[3]), pack4(q[4], q[5], q[6], q[7]));
    }
    __syncwarp();  // every lane has read the scale
    if (lane == 0) *scale = s1;
  }
}

template <typename T>
cudaError_t launch(const AppendArgs& a, bool vec, cudaStream_t s) {
  const long long windows = (static_cast<long long>(a.n_tokens) + a.window - 1) / a.window;
  const long long ctas = (windows * 2 * a.kv_heads + kWarps - 1) / kWarps;
  if (vec) append_kernel<T, true><<<static_cast<unsigned>(ctas), kWarps * 32, 0, s>>>(a);
  else append_kernel<T, false><<<static_cast<unsigned>(ctas), kWarps * 32, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace
}  // namespace lb

extern "C" int lb_op_kv8_append(const void* k, int64_t k_token_stride, int64_t k_head_stride, const void* v,
                                int64_t v_token_stride, int64_t v_head_stride, int dtype, int n_tokens,
                                int kv_heads, int dim, const int64_t* slots, int8_t* k_codes, int8_t* v_codes,
                                float* k_scale, float* v_scale, int n_pages, int page_tokens, int32_t* status,
                                void* stream) {
  using namespace lb;
  if (!k || !v || !slots || !k_codes || !v_codes || !k_scale || !v_scale || n_tokens < 1 || kv_heads < 1 ||
      n_pages < 1 || dim < 16 || dim > 512 || dim % 16 != 0 || page_tokens < 16 || page_tokens > 256 ||
      page_tokens % 16 != 0)
    return LB_ERR_INVALID_ARGUMENT;
  if (dtype != LB_F32 && dtype != LB_BF16 && dtype != LB_F16) return LB_ERR_INVALID_ARGUMENT;
  const auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  if (!aligned(k_codes) || !aligned(v_codes)) return LB_ERR_INVALID_ARGUMENT;
  const int64_t size = dtype == LB_F32 ? 4 : 2;
  const bool vec = aligned(k) && aligned(v) && k_token_stride * size % 16 == 0 && k_head_stride * size % 16 == 0 &&
                   v_token_stride * size % 16 == 0 && v_head_stride * size % 16 == 0;
  // as many tokens a window as leave a warp for each of the SMs' schedulers
  int window = 32;
  while (window > 1 && static_cast<long long>(n_tokens) * kv_heads * 2 / window < 148 * 8) window /= 2;
  AppendArgs a{{k, v}, {k_token_stride, v_token_stride}, {k_head_stride, v_head_stride}, {k_codes, v_codes},
               {k_scale, v_scale}, reinterpret_cast<const long long*>(slots), n_tokens, kv_heads, dim, n_pages,
               page_tokens, window, status};
  if ((static_cast<long long>(n_tokens) + window - 1) / window * 2 * kv_heads / kWarps >= 0x7fffffffll)
    return LB_ERR_CAPACITY;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == LB_F32 ? launch<float>(a, vec, s)
                        : dtype == LB_BF16 ? launch<__nv_bfloat16>(a, vec, s) : launch<__half>(a, vec, s);
  return e == cudaSuccess ? LB_OK : LB_ERR_CUDA;
}
