// Norms of queries and keys for each head, with the position rotation in the same pass:
//   y = x / sqrt(mean(x^2) + eps) * w        (over the dim values of one head)
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t),   t = position * frequency_i
// for the first `rotary` values of a head, paired as halves (i, i + rotary / 2) or neighbours (2 i, 2 i + 1).
//
// Angles: a frequency is a fraction of a turn, rounded to 2^-64, and its product with the position modulo 2^64 is the fraction of a
// turn that is left, exactly.  So an angle is off by at most 2^-65 turns times the position (4e-10 at 2^31, 2e-7 at 2^40, 2e-4 at
// 2^50) and 2^-32 turns (1.5e-9), as the upper half of its bits goes on to the sines.  sin and cos of what is left of a quadrant
// (at most pi / 4) are their Taylor series up to x^9 and x^10 (first terms left out: 2e-9 and 2e-10).
//
// The pass is bound by its bytes: a value is read once, kept in registers through sum, norm and
// rotation (all in 32 bits) and rounded once.  A warp takes a token, turns its angles into sines
// once and walks over the token's heads; a head of dim values takes dim / 8 lanes, each with four neighbours
// and the four that they are paired with.  Where tokens are few, a token's heads are dealt out to several warps.
//
// 16384 tokens of 32 + 8 heads of 128 in bf16 (336 MB) take 58 us, 5.8 TB/s, 88 % of the copy rate, with four steps under way in
// each of 32 warps an SM (two: 66 us; one: 78).  The usual heads have kernels of their own, without branches for the other pairs,
// parts and norms (a third fewer instructions; with the branches 75 us).  What is left is waiting for loads (6.5 of 13 cycles
// between a warp's instructions).  8 + 1 heads of 256 (151 MB) take 36 us, 4.2 TB/s: these kernels hold 16 or, at 256, 68 bytes of
// registers in local memory.  Values of 32 bits, a quarter rotated in neighbours, 3001 tokens of 16 + 4 heads of 64 (31 MB): 11.5
// us, 2.7 TB/s, some 20 warps an SM with two loads ahead each. The kernel for any size takes 81 us for 8192 tokens of 8 + 1 heads
// of 512 (1.9 TB/s).  Two tokens of 9 heads of 256 take 2.8 us among others in a graph, nearly all of it the launch.
#include "../../include/listener_b200.h"
#include "common.cuh"
#include "rows.h"

namespace lb {
namespace {

constexpr int kWarps = 4;     // of a CTA
constexpr int kMaxDim = 1024;

struct HeadsSide {
  const void* x;
  void* out;
  const void* weight;  // or null
  long long token, head, out_token, out_head;  // strides
  int heads;
};
struct HeadsArgs {
  HeadsSide q, k;
  const void* positions;
  const unsigned long long* turns;
  int n_tokens, dim, rotary, neighbours, positions64, weight_f32, norm, slices;
  float eps;
};

template <typename T>
__device__ __forceinline__ float as_float(T v) {
  if constexpr (__is_same(T, float)) return v;
  else if constexpr (__is_same(T, __half)) return __half2float(v);
  else return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T from_float(float v) {
  if constexpr (__is_same(T, float)) return v;
  else if constexpr (__is_same(T, __half)) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}
__device__ __forceinline__ void sin_cos(unsigned long long turns, float& s, float& c) {
  const unsigned h = static_cast<unsigned>(turns >> 32);       // 2^-32 turns
  const unsigned quadrant = (h + (1u << 29)) >> 30;            // (wraps to 0 with the turn)
  const int left = static_cast<int>(h - (quadrant << 30));     // at most an eighth of a turn either way
  const float x = static_cast<float>(left) * 1.4629180792671596e-9f;  // 2 pi / 2^32
  const float z = x * x;
  const float sx = fmaf(x * z, fmaf(z, fmaf(z, fmaf(z, 1.0f / 362880.0f, -1.0f / 5040.0f), 1.0f / 120.0f), -1.0f / 6.0f), x);
  const float cx = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -1.0f / 3628800.0f, 1.0f / 40320.0f), -1.0f / 720.0f), 1.0f / 24.0f), -0.5f), 1.0f);
  const bool swap = quadrant & 1u;
  s = swap ? cx : sx;
  c = swap ? sx : cx;
  if (quadrant & 2u) s = -s;
  if ((quadrant + 1u) & 2u) c = -c;
}
__device__ __forceinline__ unsigned long long position_of(const HeadsArgs& a, int token) {
  return a.positions64 ? static_cast<unsigned long long>(static_cast<const long long*>(a.positions)[token])
                       : static_cast<unsigned long long>(static_cast<long long>(static_cast<const int*>(a.positions)[token]));
}
// four neighbouring weights
template <typename T>
__device__ __forceinline__ void weights4(const HeadsArgs& a, const HeadsSide& s, int i, float (&w)[4]) {
  if (!s.weight) {
    w[0] = w[1] = w[2] = w[3] = 1.0f;
  } else if (a.weight_f32) {
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = static_cast<const float*>(s.weight)[i + j];
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = as_float(static_cast<const T*>(s.weight)[i + j]);
  }
}
template <typename T>
__device__ __forceinline__ float weight_at(const HeadsArgs& a, const HeadsSide& s, int i) {
  if (!s.weight) return 1.0f;
  return a.weight_f32 ? static_cast<const float*>(s.weight)[i] : as_float(static_cast<const T*>(s.weight)[i]);
}

// two 32-bit values an instruction
typedef unsigned long long pair_t;
__device__ __forceinline__ pair_t pair_of(float a, float b) {
  pair_t p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
  return p;
}
__device__ __forceinline__ void unpair(pair_t p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
__device__ __forceinline__ pair_t fma2(pair_t a, pair_t b, pair_t c) {
  pair_t p;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(p) : "l"(a), "l"(b), "l"(c));
  return p;
}
__device__ __forceinline__ pair_t mul2(pair_t a, pair_t b) {
  pair_t p;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(p) : "l"(a), "l"(b));
  return p;
}
template <typename T>
__device__ __forceinline__ void load4(const T* at, uint32_t (&r)[sizeof(T)]) {  // (a register a pair of 16-bit values, or a value)
  if constexpr (sizeof(T) == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(at);
    r[0] = v.x, r[1] = v.y, r[2] = v.z, r[3] = v.w;
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(at);
    r[0] = v.x, r[1] = v.y;
  }
}
template <typename T>
__device__ __forceinline__ void widen4(const uint32_t (&r)[sizeof(T)], pair_t (&v)[2]) {
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    if constexpr (sizeof(T) == 4) {
      v[p] = pair_of(__uint_as_float(r[2 * p]), __uint_as_float(r[2 * p + 1]));
    } else if constexpr (__is_same(T, __half)) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r[p]));
      v[p] = pair_of(f.x, f.y);
    } else {
      v[p] = pair_of(__uint_as_float(r[p] << 16), __uint_as_float(r[p] & 0xffff0000u));
    }
  }
}
template <typename T>
__device__ __forceinline__ void store4(T* at, const pair_t (&v)[2]) {
  float a, b, c, d;
  unpair(v[0], a, b);
  unpair(v[1], c, d);
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(at) = make_float4(a, b, c, d);
  } else if constexpr (__is_same(T, __half)) {
    const __half2 x = __floats2half2_rn(a, b), y = __floats2half2_rn(c, d);
    *reinterpret_cast<uint2*>(at) = make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
  } else {
    const __nv_bfloat162 x = __floats2bfloat162_rn(a, b), y = __floats2bfloat162_rn(c, d);
    *reinterpret_cast<uint2*>(at) = make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
  }
}

// The heads [first, last) of a side that this group of lanes takes, in steps of a warp's heads.  A lane's eight values are two
// pairs at ea and two at eb; rotated ones become v * own + other * cross, with the weights in the factors (of the token and lane, for all its
// heads) and 1 / rms behind them.
// kPlain: the usual heads (of 8 * LANES values, all rotated in halves, with norms), without branches.
template <typename T, int LANES, bool kPlain>
__device__ __forceinline__ void walk(const HeadsArgs& a, const HeadsSide& side, int token, int first, int last, int ea, int eb,
                                     bool there_, bool turned_, const float (&sn)[4], const float (&cs)[4]) {
  const bool there = kPlain || there_, turned = kPlain || turned_, neighbours = !kPlain && a.neighbours, norm = kPlain || a.norm;
  constexpr int kStep = 32 / LANES, kAhead = kPlain && sizeof(T) == 2 ? 4 : 2;
  pair_t own[2][2], cross[2][2];  // [at ea, at eb][pair]
  {
    float w[2][4] = {};
    if (there) {
      weights4<T>(a, side, ea, w[0]);
      weights4<T>(a, side, eb, w[1]);
    }
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      if (neighbours) {  // of a pair (v0, v1): v0 c - v1 s, v1 c + v0 s
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float c = cs[2 * e + p], s = sn[2 * e + p];
          own[e][p] = pair_of(w[e][2 * p] * c, w[e][2 * p + 1] * c);
          cross[e][p] = pair_of(-w[e][2 * p + 1] * s, w[e][2 * p] * s);
        }
      } else {
        own[0][p] = pair_of(w[0][2 * p] * cs[2 * p], w[0][2 * p + 1] * cs[2 * p + 1]);
        own[1][p] = pair_of(w[1][2 * p] * cs[2 * p], w[1][2 * p + 1] * cs[2 * p + 1]);
        cross[0][p] = pair_of(-w[1][2 * p] * sn[2 * p], -w[1][2 * p + 1] * sn[2 * p + 1]);
        cross[1][p] = pair_of(w[0][2 * p] * sn[2 * p], w[0][2 * p + 1] * sn[2 * p + 1]);
      }
    }
  }
  const int group = (threadIdx.x & 31) / LANES;
  const T* x = static_cast<const T*>(side.x) + token * side.token + (first + group) * side.head;
  T* out = static_cast<T*>(side.out) + token * side.out_token + (first + group) * side.out_head;
  const long long x_step = kStep * side.head, out_step = kStep * side.out_head;
  const float inv_dim = 1.0f / static_cast<float>(a.dim);
  for (int h0 = first + group; h0 - group < last; h0 += kStep * kAhead) {  // (the warp's groups together)
    uint32_t ra[kAhead][sizeof(T)], rb[kAhead][sizeof(T)];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (there && h0 + u * kStep < last) {
        load4<T>(x + ea, ra[u]);
        load4<T>(x + eb, rb[u]);
      } else {
#pragma unroll
        for (int j = 0; j < static_cast<int>(sizeof(T)); ++j) ra[u][j] = rb[u][j] = 0;
      }
      x += x_step;
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      pair_t v[2][2];
      widen4<T>(ra[u], v[0]);
      widen4<T>(rb[u], v[1]);
      float inv = 1.0f;
      if (norm) {
        const pair_t two = fma2(v[0][0], v[0][0], fma2(v[0][1], v[0][1], fma2(v[1][0], v[1][0], mul2(v[1][1], v[1][1]))));
        float lo, hi;
        unpair(two, lo, hi);
        float sum = lo + hi;
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        inv = rsqrtf(fmaf(sum, inv_dim, a.eps));
      }
      const pair_t inv2 = pair_of(inv, inv);
      pair_t y[2][2];
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          pair_t other = v[1 - e][p];
          if (neighbours) {
            float lo, hi;
            unpair(v[e][p], lo, hi);
            other = pair_of(hi, lo);
          }
          y[e][p] = mul2(v[e][p], own[e][p]);
          if (turned) y[e][p] = fma2(other, cross[e][p], y[e][p]);
          y[e][p] = mul2(y[e][p], inv2);
        }
      if (there && h0 + u * kStep < last) {
        store4<T>(out + ea, y[0]);
        store4<T>(out + eb, y[1]);
      }
      out += out_step;
    }
  }
}

// LANES: lanes of a head, at least dim / 8
template <typename T, int LANES, bool kPlain>
__global__ void __launch_bounds__(kWarps * 32, kPlain && sizeof(T) == 2 ? 8 : 4) heads_kernel(const HeadsArgs a) {
  const long long warp = static_cast<long long>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (warp >= static_cast<long long>(a.n_tokens) * a.slices) return;
  const int token = static_cast<int>(warp / a.slices), slice = static_cast<int>(warp - static_cast<long long>(token) * a.slices);
  constexpr int kStep = 32 / LANES;
  const int l = threadIdx.x & (LANES - 1);
  const bool there = kPlain || 8 * l < a.dim, turned = kPlain || 8 * l < a.rotary;
  int ea = 8 * l, eb = 8 * l + 4;
  if (kPlain || (!a.neighbours && turned)) {
    ea = 4 * l;
    eb = 4 * l + (kPlain ? 4 * LANES : a.rotary / 2);
  }
  float sn[4] = {0.0f, 0.0f, 0.0f, 0.0f}, cs[4] = {1.0f, 1.0f, 1.0f, 1.0f};
  if (turned) {
    const unsigned long long p = position_of(a, token);
#pragma unroll
    for (int j = 0; j < 4; ++j) sin_cos(p * a.turns[4 * l + j], sn[j], cs[j]);
  }
  // the token's heads in one line, q's before k's, in steps of a warp's heads; this warp's part of it
  const int q_steps = (a.q.heads + kStep - 1) / kStep, k_steps = (a.k.heads + kStep - 1) / kStep;
  const int from = static_cast<int>(static_cast<long long>(q_steps + k_steps) * slice / a.slices);
  const int to = static_cast<int>(static_cast<long long>(q_steps + k_steps) * (slice + 1) / a.slices);
  if (from < q_steps)
    walk<T, LANES, kPlain>(a, a.q, token, from * kStep, min(min(to, q_steps) * kStep, a.q.heads), ea, eb, there, turned, sn, cs);
  if (to > q_steps)
    walk<T, LANES, kPlain>(a, a.k, token, (max(from, q_steps) - q_steps) * kStep, min((to - q_steps) * kStep, a.k.heads), ea, eb, there,
                   turned, sn, cs);
}

// Any even dim and rotary, any alignment: a warp a head, read twice, value by value.
template <typename T>
__global__ void __launch_bounds__(kWarps * 32) heads_any_kernel(const HeadsArgs a) {
  const long long warp = static_cast<long long>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int all = a.q.heads + a.k.heads;
  if (warp >= static_cast<long long>(a.n_tokens) * all) return;
  const int token = static_cast<int>(warp / all), lane = threadIdx.x & 31;
  int h = static_cast<int>(warp - static_cast<long long>(token) * all);
  const bool is_k = h >= a.q.heads;
  const HeadsSide& side = is_k ? a.k : a.q;
  if (is_k) h -= a.q.heads;
  const T* x = static_cast<const T*>(side.x) + token * side.token + h * side.head;
  T* out = static_cast<T*>(side.out) + token * side.out_token + h * side.out_head;
  float inv = 1.0f;
  if (a.norm) {
    float sum = 0.0f;
    for (int i = lane; i < a.dim; i += 32) {
      const float v = as_float(x[i]);
      sum = fmaf(v, v, sum);
    }
    inv = __frsqrt_rn(fmaf(warp_sum(sum), 1.0f / static_cast<float>(a.dim), a.eps));
  }
  const unsigned long long p = position_of(a, token);
  const int half = a.rotary / 2;
  // a lane reads both values of a pair before it writes them, so that out may be x
  for (int i = lane; i < half; i += 32) {
    const int ia = a.neighbours ? 2 * i : i, ib = a.neighbours ? 2 * i + 1 : i + half;
    float s, c, va = as_float(x[ia]), vb = as_float(x[ib]);
    sin_cos(p * a.turns[i], s, c);
    if (a.norm) {
      va *= inv * weight_at<T>(a, side, ia);
      vb *= inv * weight_at<T>(a, side, ib);
    }
    out[ia] = from_float<T>(fmaf(va, c, -vb * s));
    out[ib] = from_float<T>(fmaf(vb, c, va * s));
  }
  for (int i = a.rotary + lane; i < a.dim; i += 32) {
    const float v = as_float(x[i]);
    out[i] = from_float<T>(a.norm ? v * (inv * weight_at<T>(a, side, i)) : v);
  }
}

bool aligned(const HeadsSide& s, int n_tokens, int unit, int size) {
  if (s.heads == 0) return true;
  const uintptr_t bytes = static_cast<uintptr_t>(unit) * size;
  const auto whole = [&](long long stride, int n) { return n == 1 || stride % unit == 0; };
  return reinterpret_cast<uintptr_t>(s.x) % bytes == 0 && reinterpret_cast<uintptr_t>(s.out) % bytes == 0 &&
         whole(s.token, n_tokens) && whole(s.out_token, n_tokens) && whole(s.head, s.heads) && whole(s.out_head, s.heads);
}

// An output may be its own input, with the same strides; no other two share memory.
bool apart(const HeadsArgs& a, int64_t size) {
  const auto rows = [&](const void* at, long long token, long long head, int heads) {
    return Rows{at, token * size, head * size, a.n_tokens, heads, a.dim * size};
  };
  const Rows in[2] = {rows(a.q.x, a.q.token, a.q.head, a.q.heads), rows(a.k.x, a.k.token, a.k.head, a.k.heads)};
  const Rows out[2] = {rows(a.q.out, a.q.out_token, a.q.out_head, a.q.heads), rows(a.k.out, a.k.out_token, a.k.out_head, a.k.heads)};
  for (int i = 0; i < 2; ++i) {
    const bool own = in[i].at == out[i].at && (a.n_tokens == 1 || in[i].token == out[i].token) && (in[i].heads == 1 || in[i].head == out[i].head);
    if ((!own && rows_meet(out[i], in[i])) || rows_meet(out[i], in[1 - i])) return false;
  }
  return !rows_meet(out[0], out[1]);
}

template <typename T>
cudaError_t launch(HeadsArgs a, cudaStream_t s) {
  const bool fast = a.dim % 8 == 0 && a.dim <= 256 && a.rotary % 8 == 0 && aligned(a.q, a.n_tokens, 4, sizeof(T)) &&
                    aligned(a.k, a.n_tokens, 4, sizeof(T));
  if (!fast) {
    const long long warps = static_cast<long long>(a.n_tokens) * (a.q.heads + a.k.heads);
    heads_any_kernel<T><<<static_cast<unsigned>((warps + kWarps - 1) / kWarps), kWarps * 32, 0, s>>>(a);
    return cudaGetLastError();
  }
  const int lanes = a.dim <= 64 ? 8 : a.dim <= 128 ? 16 : 32, step = 32 / lanes;
  const int steps = (a.q.heads + step - 1) / step + (a.k.heads + step - 1) / step;
  // as many warps as the GPU holds at 16 an SM, if the heads go that far
  const long long want = (148ll * 16 + a.n_tokens - 1) / a.n_tokens;
  a.slices = static_cast<int>(want < steps ? want : steps);
  const long long warps = static_cast<long long>(a.n_tokens) * a.slices;
  const unsigned grid = static_cast<unsigned>((warps + kWarps - 1) / kWarps);
  const bool plain = a.dim == 8 * lanes && a.rotary == a.dim && !a.neighbours && a.norm;
  const auto kernel = lanes == 8    ? (plain ? heads_kernel<T, 8, true> : heads_kernel<T, 8, false>)
                      : lanes == 16 ? (plain ? heads_kernel<T, 16, true> : heads_kernel<T, 16, false>)
                                    : (plain ? heads_kernel<T, 32, true> : heads_kernel<T, 32, false>);
  kernel<<<grid, kWarps * 32, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace
}  // namespace lb

extern "C" int lb_op_head_norm_rotary(const void* q, int64_t q_token_stride, int64_t q_head_stride, int heads, const void* k,
                                      int64_t k_token_stride, int64_t k_head_stride, int kv_heads, int dtype, int n_tokens,
                                      int dim, const void* positions, int positions64, const uint64_t* turns, int rotary,
                                      int neighbours, const void* q_weight, const void* k_weight, int weight_dtype, int norm,
                                      float eps, void* q_out, int64_t q_out_token_stride, int64_t q_out_head_stride,
                                      void* k_out, int64_t k_out_token_stride, int64_t k_out_head_stride, void* stream) {
  using namespace lb;
  if (!q || !q_out || n_tokens < 1 || heads < 1 || kv_heads < 0 || (kv_heads > 0 && (!k || !k_out))) return LB_ERR_INVALID_ARGUMENT;
  if (dim < 2 || dim > kMaxDim || dim % 2 != 0 || rotary < 0 || rotary > dim || rotary % 2 != 0 || !(eps >= 0.0f))
    return LB_ERR_INVALID_ARGUMENT;
  if (!positions || (rotary > 0 && !turns)) return LB_ERR_INVALID_ARGUMENT;
  if (dtype != LB_F32 && dtype != LB_BF16 && dtype != LB_F16) return LB_ERR_INVALID_ARGUMENT;
  if (weight_dtype != LB_F32 && weight_dtype != dtype) return LB_ERR_INVALID_ARGUMENT;
  if (heads > 65536 || kv_heads > 65536 || static_cast<long long>(n_tokens) * (heads + kv_heads) > (1ll << 32))
    return LB_ERR_CAPACITY;
  HeadsArgs a{};
  a.q = {q, q_out, q_weight, q_token_stride, q_head_stride, q_out_token_stride, q_out_head_stride, heads};
  a.k = {k, k_out, k_weight, k_token_stride, k_head_stride, k_out_token_stride, k_out_head_stride, kv_heads};
  a.positions = positions;
  a.turns = reinterpret_cast<const unsigned long long*>(turns);
  a.n_tokens = n_tokens;
  a.dim = dim;
  a.rotary = rotary;
  a.neighbours = neighbours != 0;
  a.positions64 = positions64 != 0;
  a.weight_f32 = weight_dtype == LB_F32;
  a.norm = norm != 0;
  a.eps = eps;
  if (!apart(a, dtype == LB_F32 ? 4 : 2)) return LB_ERR_INVALID_ARGUMENT;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == LB_F32 ? launch<float>(a, s) : dtype == LB_BF16 ? launch<__nv_bfloat16>(a, s) : launch<__half>(a, s);
  return e == cudaSuccess ? LB_OK : LB_ERR_CUDA;
}
