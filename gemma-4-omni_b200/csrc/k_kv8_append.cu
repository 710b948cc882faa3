// New keys and values written into the 8-bit cache.
//
// A group is the run of batch tokens that follow one another in one page, first at
// offset o.  For each kv head and side:
//   s1 = max(s0, max |x| / 127)  (s0 the page's scale, 0 when the page begins here)
//   codes before o: c -> rint(c * s0 / s1) where the scale grew; new: rint(x / s1)
// so value = code * scale holds for the whole page with one scale, and a page is
// only touched where its scale grows.
//
// The floor of a prompt's append is its bytes (the tokens read once, their codes written): 16 prompts of
// 22 thousand tokens with 8 heads of 128 in 16 bits take 46 us against 20.5 at the copy rate, bound by
// the instructions of the rounding (80 % of the issue slots), in f32 8 us more, and 8 us more where the scale of every
// page grows, whose older codes take a division each.  The floor of a
// tick's is a launch: 3.6 us inside a graph for 128 sessions.  A CTA of 128 threads a (group, head,
// side): with a warp a group the prompt took 69 us, its values filling the registers of 16 warps an SM.  The
// CTAs look for the first tokens of groups in windows of the batch, so nothing
// but the slots has to be known: a token begins a group unless the token before
// it in the batch has the slot before it in the same page.  Where the last token before it that is not skipped is of
// the same page all the same, two groups would read and write that page at once: the later one is refused.  A
// group of up to 512 pieces of 8 values stays in registers between its maximum and its codes; larger ones are read again.
#include <cstring>

#include "../../include/listener_b200.h"
#include "common.cuh"

namespace lb {
namespace {

constexpr int kThreads = 128;

struct AppendArgs {
  const void* src[2];
  long long token_stride[2], head_stride[2];
  int8_t* codes[2];
  float* scale[2];
  const long long* slots;
  int n_tokens, kv_heads, dim, n_pages, page_tokens, window;
  int piece_log;  // log2 of a token's pieces of 8 values, -1 where that is no power of two
  int* status;
};

// slot / P for slot >= 0: in 32 bits where it fits (a 64-bit division costs as much as 8 values' codes)
__device__ __forceinline__ long long page_of(long long slot, int P) {
  return slot >> 32 ? slot / P : static_cast<long long>(static_cast<uint32_t>(slot) / static_cast<uint32_t>(P));
}

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// rint(x / s) within +-127; NaN (0 / 0 or a NaN x) -> 0
__device__ __forceinline__ int code_of(float x, float s) {
  const float q = __fdiv_rn(x, s);
  return isnan(q) ? 0 : __float2int_rn(fminf(fmaxf(q, -127.0f), 127.0f));
}

// Codes of 8 finite values by `inv`, the rounded 1 / s: x * inv is within 2.4e-5 of x / s, and the bits of
// `near` tell where that could change the nearest whole number (with 16-bit values x / s often lies
// exactly halfway, so those are few but not rare: some 0.5 %).  The sum with 1.5 * 2^23 rounds to the
// nearest even and leaves the code in its low byte.
__device__ __forceinline__ uint2 codes8(const float (&v)[8], float inv, uint32_t& near) {
  uint32_t b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float q = v[i] * inv, r = q + 12582912.0f;
    near = near << 1 | (fabsf(q - (r - 12582912.0f)) > 0.49996f);  // value i ends in bit 7 - i
    b[i] = __float_as_uint(r);
  }
  return make_uint2(__byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410),
                    __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410));
}

// 8 elements as they come
template <typename T>
struct Piece {
  uint4 raw[sizeof(T) == 4 ? 2 : 1];
};
template <typename T, bool VEC>
__device__ __forceinline__ Piece<T> load_piece(const T* p) {
  Piece<T> v;
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(v) / 16); ++i) v.raw[i] = reinterpret_cast<const uint4*>(p)[i];
  } else {
    T* e = reinterpret_cast<T*>(v.raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = p[i];
  }
  return v;
}
template <typename T>
__device__ __forceinline__ void widen(const Piece<T>& v, float (&f)[8]) {
  const T* e = reinterpret_cast<const T*>(v.raw);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = to_float<T>(e[i]);
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads, 8) append_kernel(const AppendArgs a) {
  constexpr int kHeld = 4;  // pieces a thread keeps
  __shared__ uint32_t tops[kThreads / 32];
  __shared__ float mosts[kThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per_window = 2 * a.kv_heads;
  const int win = blockIdx.x / per_window, which = blockIdx.x - win * per_window;
  const int side = which & 1, head = which >> 1;
  const long long t0 = static_cast<long long>(win) * a.window;
  const int P = a.page_tokens, D = a.dim, chunks = D / 8;

  // the slots of 64 tokens: bit i of `follows` is set where token t0 + i goes on in the page of the one before it
  const auto slot_at = [&](long long i) { return i >= 0 && i < a.n_tokens ? a.slots[i] : -1ll; };
  const long long before = lane == 0 ? slot_at(t0 - 1) : 0;
  const long long slot0 = slot_at(t0 + lane), slot1 = slot_at(t0 + 32 + lane);
  long long prev0 = __shfl_up_sync(0xffffffffu, slot0, 1), prev1 = __shfl_up_sync(0xffffffffu, slot1, 1);
  const long long edge = __shfl_sync(0xffffffffu, slot0, 31);
  if (lane == 0) {
    prev0 = t0 > 0 ? before : -2;
    prev1 = edge;
  }
  const long long page0 = slot0 >= 0 ? page_of(slot0, P) : -1;
  const unsigned on0 = __ballot_sync(0xffffffffu, slot0 > 0 && slot0 == prev0 + 1 && page0 * P != slot0);
  const unsigned on1 = __ballot_sync(0xffffffffu, slot1 > 0 && slot1 == prev1 + 1 && page_of(slot1, P) * P != slot1);
  const unsigned long long follows = on0 | static_cast<unsigned long long>(on1) << 32;
  const bool first = lane < a.window && slot0 >= 0 && !(on0 >> lane & 1u);
  // first tokens after one that is skipped or of the same page
  const unsigned look = __ballot_sync(0xffffffffu, first && t0 + lane > 0 && (prev0 < 0 || (prev0 >= page0 * P && prev0 - page0 * P < P)));
  const T* src = static_cast<const T*>(side ? a.src[1] : a.src[0]) + head * (side ? a.head_stride[1] : a.head_stride[0]);
  const long long ts = side ? a.token_stride[1] : a.token_stride[0];
  // every warp finds the same groups
  for (unsigned todo = __ballot_sync(0xffffffffu, first); todo; todo &= todo - 1) {
    const int at = __ffs(todo) - 1;
    const long long t = t0 + at;
    const long long slot = __shfl_sync(0xffffffffu, slot0, at), page = __shfl_sync(0xffffffffu, page0, at);
    const int off = static_cast<int>(slot - page * P);
    if (page >= a.n_pages) {
      if (tid == 0 && a.status) atomicOr(a.status, static_cast<int>(LB_DEV_BAD_PAGE));
      continue;
    }
    if (look >> at & 1u) {  // the last token before it that is not skipped
      bool split = false;
#pragma unroll 1
      for (long long j = t - 1; j >= 0; j -= 32) {
        const long long s = slot_at(j - lane);
        const unsigned there = __ballot_sync(0xffffffffu, s >= 0);
        if (there) {
          const long long last = __shfl_sync(0xffffffffu, s, __ffs(there) - 1);
          split = last >= page * P && last - page * P < P;
          break;
        }
      }
      if (split) {
        if (tid == 0 && a.status) atomicOr(a.status, static_cast<int>(LB_DEV_SPLIT_PAGE));
        continue;
      }
    }
    int run = __ffsll(static_cast<long long>(~(follows >> at >> 1)));  // the token and those that follow
    while (at + run >= 64 && off + run < P) {  // past the 64 tokens (pages of more than 32)
      const int j = run + lane;
      const unsigned all = __ballot_sync(0xffffffffu, off + j < P && slot_at(t + j) == slot + j);
      run += all == 0xffffffffu ? 32 : __ffs(~all) - 1;
      if (all != 0xffffffffu) break;
    }
    float* scale = (side ? a.scale[1] : a.scale[0]) + page * a.kv_heads + head;
    const float s0 = off > 0 ? *scale : 0.0f;
    const T* from = src + t * ts;
    const int pieces = run * chunks;
    const bool held = a.piece_log >= 0 && pieces <= kThreads * kHeld;
    Piece<T> raw[kHeld];
    uint32_t top = 0;
    const auto look = [&](const Piece<T>& v) {  // the largest absolute value, by its bits
      const uint32_t* w = reinterpret_cast<const uint32_t*>(v.raw);
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(v) / 4); ++i) {
        if constexpr (sizeof(T) == 4) top = max(top, w[i] & 0x7fffffffu);
        else top = __vmaxu2(top, w[i] & 0x7fff7fffu);
      }
    };
    if (held) {
#pragma unroll
      for (int k = 0; k < kHeld; ++k) {
        const int c = tid + kThreads * k, j = c >> a.piece_log;
        if (c < pieces) raw[k] = load_piece<T, VEC>(from + j * ts + (c - (j << a.piece_log)) * 8);
      }
#pragma unroll
      for (int k = 0; k < kHeld; ++k)
        if (tid + kThreads * k < pieces) look(raw[k]);
    } else {
#pragma unroll 4
      for (int c = tid; c < pieces; c += kThreads) {
        const int j = c / chunks;
        look(load_piece<T, VEC>(from + j * ts + (c - j * chunks) * 8));
      }
    }
    if constexpr (sizeof(T) == 2) top = max(top & 0xffffu, top >> 16);
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) tops[warp] = top;
    __syncthreads();
    top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
    float most;
    if constexpr (sizeof(T) == 4) {
      most = __uint_as_float(top);
    } else {
      const uint16_t bits = static_cast<uint16_t>(top);
      T v;
      memcpy(&v, &bits, 2);
      most = to_float<T>(v);
    }
    const bool odd = !(most < INFINITY);  // there is an infinite value or a NaN: the largest of the others
    if (odd) {
      most = 0.0f;
#pragma unroll 1
      for (int c = tid; c < pieces * 8; c += kThreads) {
        const float f = fabsf(to_float<T>(from[c / D * ts + c % D]));
        if (f < INFINITY) most = fmaxf(most, f);
      }
      most = warp_max(most);
      if (lane == 0) mosts[warp] = most;
      __syncthreads();
      most = fmaxf(fmaxf(mosts[0], mosts[1]), fmaxf(mosts[2], mosts[3]));
      if (tid == 0 && a.status) atomicOr(a.status, static_cast<int>(LB_DEV_NONFINITE));
    }
    const float s1 = fmaxf(s0, __fdiv_rn(most, 127.0f));
    int8_t* base = (side ? a.codes[1] : a.codes[0]) + (page * a.kv_heads + head) * static_cast<long long>(P) * D;
    if (s1 != s0) {
      for (int c = tid; c < off * (D / 16); c += kThreads) {
        int4* at = reinterpret_cast<int4*>(base) + c;
        const int4 old = *at;
        uint32_t w[4] = {static_cast<uint32_t>(old.x), static_cast<uint32_t>(old.y), static_cast<uint32_t>(old.z),
                         static_cast<uint32_t>(old.w)};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t made = 0;
#pragma unroll 1
          for (int b = 0; b < 32; b += 8)
            made |= static_cast<uint32_t>(code_of(static_cast<float>(static_cast<int8_t>(w[i] >> b)) * s0, s1) & 0xff) << b;
          w[i] = made;
        }
        *at = make_int4(w[0], w[1], w[2], w[3]);
      }
    }
    const float inv = __fdiv_rn(1.0f, s1);
    const bool plain = !odd && inv < INFINITY;  // else (a zero or tiny scale, values that are not finite): one by one
    int8_t* to = base + static_cast<long long>(off) * D;  // the page's tokens are neighbours
    const auto exact = [&](int c, int i) {  // value i of piece c, by the division
      to[c * 8 + i] = static_cast<int8_t>(code_of(to_float<T>(from[c / chunks * ts + c % chunks * 8 + i]), s1));
    };
    if (plain && held) {
      uint32_t near = 0;
#pragma unroll
      for (int k = 0; k < kHeld; ++k) {
        const int c = tid + kThreads * k;
        if (c < pieces) {
          float f[8];
          widen<T>(raw[k], f);
          *reinterpret_cast<uint2*>(to + c * 8) = codes8(f, inv, near);
        } else {
          near <<= 8;
        }
      }
#pragma unroll 1
      for (; near; near &= near - 1) {
        const int bit = 8 * kHeld - __ffs(near);  // the value's number among the thread's
        exact(tid + kThreads * (bit >> 3), bit & 7);
      }
    } else {
#pragma unroll 1
      for (int c = tid; c < pieces; c += kThreads) {
        uint32_t near = plain ? 0u : 0xffu;
        if (plain) {
          const int j = c / chunks;
          float f[8];
          widen<T>(load_piece<T, VEC>(from + j * ts + (c - j * chunks) * 8), f);
          *reinterpret_cast<uint2*>(to + c * 8) = codes8(f, inv, near);
        }
#pragma unroll 1
        for (; near; near &= near - 1) exact(c, 8 - __ffs(near));
      }
    }
    __syncthreads();  // every thread has read the scale and the warps' maxima
    if (tid == 0) *scale = s1;
  }
}

template <typename T>
cudaError_t launch(const AppendArgs& a, bool vec, cudaStream_t s) {
  const long long windows = (static_cast<long long>(a.n_tokens) + a.window - 1) / a.window;
  const long long ctas = windows * 2 * a.kv_heads;
  if (vec) append_kernel<T, true><<<static_cast<unsigned>(ctas), kThreads, 0, s>>>(a);
  else append_kernel<T, false><<<static_cast<unsigned>(ctas), kThreads, 0, s>>>(a);
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
  // as many tokens a window as leave eight CTAs for each SM
  int window = 32;
  while (window > 1 && static_cast<long long>(n_tokens) * kv_heads * 2 / window < 148 * 8) window /= 2;
  AppendArgs a{{k, v}, {k_token_stride, v_token_stride}, {k_head_stride, v_head_stride}, {k_codes, v_codes},
               {k_scale, v_scale}, reinterpret_cast<const long long*>(slots), n_tokens, kv_heads, dim, n_pages,
               page_tokens, window, (dim / 8 & (dim / 8 - 1)) == 0 ? 31 - __builtin_clz(dim / 8) : -1, status};
  if ((static_cast<long long>(n_tokens) + window - 1) / window * 2 * kv_heads >= 0x7fffffffll)
    return LB_ERR_CAPACITY;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == LB_F32 ? launch<float>(a, vec, s)
                        : dtype == LB_BF16 ? launch<__nv_bfloat16>(a, vec, s) : launch<__half>(a, vec, s);
  return e == cudaSuccess ? LB_OK : LB_ERR_CUDA;
}
