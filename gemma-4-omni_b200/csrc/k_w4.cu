// Matrix-vector products with 4-bit weights and group scales:
//   out[m][o] = sum_g s[o][g] sum_{k in g} (n[o][k] - 8) x[m][k] * xs[m][k / gx]
//
// With a few rows of x the codes' bytes bound the product, so the kernel is built
// around their stream: each warp has its own ring of cp.async stages (32 outputs x
// 128 k, 2 KB of codes and the groups' scales) that runs on from one tile of outputs
// to the next, and no barrier of the block in the main loop.  x lies in shared memory
// (16 bits, loaded once a CTA).  The codes become the A fragments of mma.sync in
// registers by the published conversion under an exponent (Kim, Henry, Fahim and Awadalla,
// 2022): a word of 8 codes masks into four pairs (k, k + 4) by shifts and one logic operation
// each, as 1024 + n (fp16) or 128 + n (bf16), from which one subtraction leaves n - 8
// exactly; x is stored in the pairs' order, so neither side is shuffled.  8-bit x is exact in fp16.  A group's sum is held in 32 bits and takes its
// scale there.  mma.sync runs at 0.5 m16n8k16 a cycle and SM, and the stream of 16 rows needs 0.36, so the
// tensor pipe is not what binds (27 % busy): instructions are, some 450 a stage and warp, nearly half of them on
// the half-rate integer pipe (50 % busy; the widening alone is 11 for 8 codes in bf16, 9 in fp16).  16 x 2048 x
// 131072 in groups of 64 takes 61.5 us, 2.4 TB/s (fp16 3 us less, one row 9 us less).  Whole tiles are dealt out,
// so the last pass leaves SMs idle: of that product's 148 CTAs 40 make one pass where 108 make two; 16 x 1536 x
// 12288 has 96 CTAs.
//
// More rows than 16 (8 where k is above some 4600) read and widen the whole matrix again for every 16: 128, 512 and 2048
// rows of 1536 x 12288 take 47, 117 and 426 us, the last against 46 for its operations.
//
// K is split among the warps of a CTA (and summed in shared memory) as far as one wave of CTAs goes: 2 x
// 1536 x 6144 takes 6.8 us inside a graph.  Larger products run 16 warps an SM that walk over the tiles (8
// warps, each CTA loading x for itself: 115 us for the product above).
#include <cuda_fp8.h>

#include "../../include/listener_b200.h"
#include "common.cuh"

namespace lb {
namespace {

constexpr int kTileO = 32;          // outputs of a stage
constexpr int kBlockK = 128;        // k of a stage
constexpr int kCodeBytes = kTileO * kBlockK / 2;
constexpr int kScaleBytes = kTileO * 4 * 2;  // at most four groups
constexpr int kStageBytes = kCodeBytes + kScaleBytes;
constexpr int kXPad = 64;           // bytes between rows of x: eight lanes' pieces in different banks
constexpr int kMaxSmem = 220 * 1024;

struct W4Args {
  const void* x;
  long long x_ld, ld_out;
  const float* x_scale;
  int x_dtype, x_group, m, group, out_features, k, out_dtype, splits, stages, tiles, m_tiles;
  const uint8_t* codes;
  const __half* w_scale;
  void* out;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void cp_async_wait_pending(int n) {  // at most n groups still under way
  if (n >= 6) asm volatile("cp.async.wait_group 6;" ::: "memory");
  else if (n == 5) asm volatile("cp.async.wait_group 5;" ::: "memory");
  else if (n == 4) asm volatile("cp.async.wait_group 4;" ::: "memory");
  else if (n == 3) asm volatile("cp.async.wait_group 3;" ::: "memory");
  else if (n == 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
  else if (n == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
  else asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// kFirst: a sum begins (c is only written)
template <bool kBf16, bool kFirst>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
#define LB_MMA(type, c0)                                                                                        \
  "mma.sync.aligned.m16n8k16.row.col.f32." type "." type ".f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, " c0 ";"
#define LB_IN "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1)
  if constexpr (kFirst) {
    if constexpr (kBf16)
      asm volatile(LB_MMA("bf16", "{%10,%10,%10,%10}") : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : LB_IN, "f"(0.0f));
    else
      asm volatile(LB_MMA("f16", "{%10,%10,%10,%10}") : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : LB_IN, "f"(0.0f));
  } else {
    if constexpr (kBf16)
      asm volatile(LB_MMA("bf16", "{%0,%1,%2,%3}") : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : LB_IN);
    else
      asm volatile(LB_MMA("f16", "{%0,%1,%2,%3}") : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : LB_IN);
  }
#undef LB_IN
#undef LB_MMA
}

template <typename H>
__device__ __forceinline__ uint32_t bits_of(H v) { return *reinterpret_cast<const uint32_t*>(&v); }
__device__ __forceinline__ __half2 half2_of(uint32_t v) { return *reinterpret_cast<const __half2*>(&v); }
__device__ __forceinline__ __nv_bfloat162 bf162_of(uint32_t v) { return *reinterpret_cast<const __nv_bfloat162*>(&v); }

// 8 codes -> the pairs (0, 4), (1, 5), (2, 6), (3, 7), less 8
template <bool kBf16>
__device__ __forceinline__ void widen8(uint32_t w, uint32_t (&p)[4]) {
  if constexpr (kBf16) {
    const __nv_bfloat162 bias = __floats2bfloat162_rn(136.0f, 136.0f);
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = bits_of(__hsub2(bf162_of(((w >> (4 * i)) & 0x000f000fu) | 0x43004300u), bias));
  } else {
    const __half2 bias = __floats2half2_rn(1032.0f, 1032.0f);
    const __half2 sixteenth = __floats2half2_rn(0.0625f, 0.0625f), high = __floats2half2_rn(-72.0f, -72.0f);
    const uint32_t u = w >> 8;
    p[0] = bits_of(__hsub2(half2_of((w & 0x000f000fu) | 0x64006400u), bias));
    p[1] = bits_of(__hfma2(half2_of((w & 0x00f000f0u) | 0x64006400u), sixteenth, high));  // 1024 + 16 n
    p[2] = bits_of(__hsub2(half2_of((u & 0x000f000fu) | 0x64006400u), bias));
    p[3] = bits_of(__hfma2(half2_of((u & 0x00f000f0u) | 0x64006400u), sixteenth, high));
  }
}

// 8 consecutive x of a row as 16 bits, in the order 0 4 1 5 2 6 3 7
__device__ __forceinline__ uint4 load_x8(const W4Args& a, int row, int k) {
  uint16_t v[8];
  const long long at = row * a.x_ld + k;
  if (a.x_dtype == LB_BF16 || a.x_dtype == LB_F16) {
    const uint16_t* p = static_cast<const uint16_t*>(a.x) + at;
    if (reinterpret_cast<uintptr_t>(p) % 16 == 0) {
      const uint4 w = *reinterpret_cast<const uint4*>(p);
      return make_uint4(__byte_perm(w.x, w.z, 0x5410), __byte_perm(w.x, w.z, 0x7632), __byte_perm(w.y, w.w, 0x5410),
                        __byte_perm(w.y, w.w, 0x7632));
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = p[i];
  } else {
    const uint8_t* p = static_cast<const uint8_t*>(a.x) + at;
    uint8_t raw[8];
    if (reinterpret_cast<uintptr_t>(p) % 8 == 0) {
      *reinterpret_cast<uint2*>(raw) = *reinterpret_cast<const uint2*>(p);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) raw[i] = p[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      v[i] = a.x_dtype == LB_I8 ? __half_as_ushort(__int2half_rn(static_cast<int8_t>(raw[i])))
                                : __half_raw(__nv_cvt_fp8_to_halfraw(raw[i], __NV_E4M3)).x;
  }
  return make_uint4(v[0] | static_cast<uint32_t>(v[4]) << 16, v[1] | static_cast<uint32_t>(v[5]) << 16,
                    v[2] | static_cast<uint32_t>(v[6]) << 16, v[3] | static_cast<uint32_t>(v[7]) << 16);
}

// kXShared: x lies in shared memory; otherwise (k too large for it) every fragment is read from x itself.
template <bool kBf16, int NT, bool kXShared, int kWarps, int kGroup>
__global__ void __launch_bounds__(kWarps * 32) w4_kernel(const W4Args a) {
  extern __shared__ __align__(128) unsigned char w4_smem[];
  constexpr int kThreads = kWarps * 32, kPerBlock = kBlockK / kGroup;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int blocks = (a.k + kBlockK - 1) / kBlockK, groups = a.k / kGroup;
  const int x_row = blocks * kBlockK * 2 + kXPad;
  unsigned char* x_s = w4_smem;                                                // [8 NT][x_row]
  unsigned char* ring = x_s + (kXShared ? 8 * NT * x_row : 0) + warp * a.stages * kStageBytes;
  float* sums = reinterpret_cast<float*>(w4_smem + (kXShared ? 8 * NT * x_row : 0));  // the rings, between tiles
  const int m0 = (blockIdx.x % a.m_tiles) * (8 * NT), m_live = min(8 * NT, a.m - m0);

  // ---- this warp's tiles of outputs and blocks of k
  const int rows = kWarps / a.splits, split = warp % a.splits;
  const int per = (blocks + a.splits - 1) / a.splits;
  const int b0 = min(blocks, split * per), nb = min(blocks, b0 + per) - b0;
  const int first = (blockIdx.x / a.m_tiles) * rows + warp / a.splits;  // + rows * gridDim for each pass
  const int step = static_cast<int>(gridDim.x / a.m_tiles) * rows;
  const int passes = (a.tiles - (static_cast<int>(blockIdx.x) / a.m_tiles) * rows + step - 1) / step;  // of the CTA
  const int mine = first < a.tiles ? (a.tiles - first + step - 1) / step : 0;
  const int n_units = mine * nb;
  const uint32_t ring_at = smem_u32(ring);

  // scales travel by registers, one unit behind the codes (they have no 16-byte rows)
  uint32_t pend[2] = {0, 0};
  int pend_slot = -1;
  const auto flush_scales = [&]() {
    if (pend_slot >= 0) *reinterpret_cast<uint2*>(ring + pend_slot * kStageBytes + kCodeBytes + lane * 8) = make_uint2(pend[0], pend[1]);
    pend_slot = -1;
  };
  int iss_tile = first, iss_b = 0, iss_slot = 0, issued = 0;
  const uint8_t* from = nullptr;      // this lane's 16 bytes of the unit's first row group
  const uint16_t* scale_from = nullptr;
  unsigned rows_there = 0;            // bit i: row 8 i + lane / 4 of the tile exists; bit 4: row `lane` does
  const uint32_t lane_dst = (lane >> 2) * 64;
  const auto aim = [&]() {            // at the first unit of iss_tile
    const int o0 = iss_tile * kTileO;
    from = a.codes + static_cast<long long>(o0 + (lane >> 2)) * (a.k / 2) + b0 * (kBlockK / 2) + 16 * (lane & 3);
    scale_from = reinterpret_cast<const uint16_t*>(a.w_scale) + static_cast<long long>(o0 + lane) * groups + b0 * kPerBlock;
    rows_there = o0 + lane < a.out_features ? 16u : 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) rows_there |= o0 + 8 * i + (lane >> 2) < a.out_features ? 1u << i : 0u;
  };
  if (n_units > 0) aim();
  const auto issue = [&]() {
    flush_scales();
    if (issued < n_units) {
      const int k0 = (b0 + iss_b) * kBlockK;
      const uint32_t dst = ring_at + iss_slot * kStageBytes + lane_dst;
      const bool k_there = k0 + 32 * (lane & 3) < a.k;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (k_there && (rows_there >> i & 1u))
          cp_async16(dst + i * 512 + (((lane & 3) ^ (((lane >> 2) >> 1) & 3)) << 4), from + static_cast<long long>(i) * 4 * a.k);
      uint32_t s[4] = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < kPerBlock; ++i)
        if ((rows_there & 16u) && (k0 / kGroup + i) < groups) s[i] = scale_from[i];
      pend[0] = s[0] | s[1] << 16;
      pend[1] = s[2] | s[3] << 16;
      pend_slot = iss_slot;
      ++issued;
      from += kBlockK / 2;
      scale_from += kPerBlock;
      if (++iss_b == nb) {
        iss_b = 0;
        iss_tile += step;
        if (issued < n_units) aim();
      }
      if (++iss_slot == a.stages) iss_slot = 0;
    }
    cp_async_commit();
  };
  for (int i = 0; i < a.stages - 1; ++i) issue();

  if constexpr (kXShared) {
    for (int i = tid; i < 8 * NT * blocks * (kBlockK / 8); i += kThreads) {
      const int r = i / (blocks * (kBlockK / 8)), k = (i - r * (blocks * (kBlockK / 8))) * 8;
      *reinterpret_cast<uint4*>(x_s + r * x_row + k * 2) =
          r < m_live && k < a.k ? load_x8(a, m0 + r, k) : make_uint4(0, 0, 0, 0);
    }
    __syncthreads();
  }

  // a lane's words of a stage: the same place in each of the rows g, g + 8, g + 16, g + 24
  int word_at[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) word_at[j] = g * 64 + ((j ^ ((g >> 1) & 3)) << 4) + 4 * t;
  const unsigned char* x_lane = x_s + g * x_row + b0 * (kBlockK * 2) + t * 16;
  int slot = 0;
  for (int pass = 0; pass < passes; ++pass) {
    float acc[2][NT][4] = {};
    if (pass < mine) {
      for (int b = 0; b < nb; ++b) {
        cp_async_wait_pending(a.stages - 2);
        __syncwarp();  // the stage is there for every lane, and every lane has left the one before
        issue();
        const unsigned char* st = ring + slot * kStageBytes;
        if (++slot == a.stages) slot = 0;
        const int k0 = (b0 + b) * kBlockK;
        float part[2][NT][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint4 xb[NT];
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if constexpr (kXShared) {
              xb[n] = *reinterpret_cast<const uint4*>(x_lane + 8 * n * x_row + b * (kBlockK * 2) + j * 64);
            } else {
              const int k = k0 + 32 * j + 8 * t;
              xb[n] = 8 * n + g < m_live && k < a.k ? load_x8(a, m0 + 8 * n + g, k) : make_uint4(0, 0, 0, 0);
            }
          }
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) {
            uint32_t lo[4], hi[4];
            widen8<kBf16>(*reinterpret_cast<const uint32_t*>(st + word_at[j] + mt * 1024), lo);
            widen8<kBf16>(*reinterpret_cast<const uint32_t*>(st + word_at[j] + mt * 1024 + 512), hi);
            const uint32_t a0[4] = {lo[0], hi[0], lo[1], hi[1]}, a1[4] = {lo[2], hi[2], lo[3], hi[3]};
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              if ((32 * j) % kGroup == 0) mma_16816<kBf16, true>(part[mt][n], a0, xb[n].x, xb[n].y);
              else mma_16816<kBf16, false>(part[mt][n], a0, xb[n].x, xb[n].y);
              mma_16816<kBf16, false>(part[mt][n], a1, xb[n].z, xb[n].w);
            }
          }
          if ((32 * (j + 1)) % kGroup == 0) {  // a group ends: its sum takes its scale (and x's, of a group of 128 or more)
            const __half* sc = reinterpret_cast<const __half*>(st + kCodeBytes) + 32 * (j + 1) / kGroup - 1;
            float xs[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) xs[n][0] = xs[n][1] = 1.0f;
            if (a.x_group) {
#pragma unroll
              for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const int row = 8 * n + 2 * t + e;
                  if (row < m_live) xs[n][e] = a.x_scale[static_cast<long long>(m0 + row) * (a.k / a.x_group) + k0 / a.x_group];
                }
#pragma unroll
              for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                  for (int e = 0; e < 4; ++e) part[mt][n][e] *= xs[n][e & 1];
            }
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
              const float s0 = __half2float(sc[(16 * mt + g) * 4]), s1 = __half2float(sc[(16 * mt + g + 8) * 4]);
#pragma unroll
              for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[mt][n][e] = fmaf(part[mt][n][e], e < 2 ? s0 : s1, acc[mt][n][e]);
            }
          }
        }
      }
    }
    // ---- the tile: lane (g, t) holds outputs 16 mt + g (+ 8) of rows 8 n + 2 t (+ 1)
    const int tile = first + pass * step;
    const auto store = [&](int o, int row, float v) {
      if (o >= a.out_features || row >= m_live) return;
      if (a.x_scale && !a.x_group) v *= a.x_scale[m0 + row];
      const long long at = (m0 + row) * a.ld_out + o;
      if (a.out_dtype == LB_F32) static_cast<float*>(a.out)[at] = v;
      else if (a.out_dtype == LB_BF16) static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(v);
      else static_cast<__half*>(a.out)[at] = __float2half_rn(v);
    };
    if (a.splits == 1) {
      if (pass < mine) {
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              store(tile * kTileO + 16 * mt + g + (e >> 1) * 8, 8 * n + 2 * t + (e & 1), acc[mt][n][e]);
      }
    } else {
      // one pass a CTA (the host sees to it), so the rings are idle
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      __syncthreads();
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            sums[(warp * 8 * NT + 8 * n + 2 * t + (e & 1)) * (kTileO + 1) + 16 * mt + g + (e >> 1) * 8] = acc[mt][n][e];
      __syncthreads();
      for (int i = tid; i < rows * m_live * kTileO; i += kThreads) {
        const int o = i % kTileO, row = i / kTileO % m_live, tr = i / (kTileO * m_live);
        float v = 0.0f;
        for (int s = 0; s < a.splits; ++s) v += sums[((tr * a.splits + s) * 8 * NT + row) * (kTileO + 1) + o];
        const int tile_r = (blockIdx.x / a.m_tiles) * rows + tr + pass * step;
        if (tile_r < a.tiles) store(tile_r * kTileO + o, row, v);
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

template <bool kBf16, int NT, bool kXShared, int kWarps, int kGroup>
cudaError_t launch(const W4Args& a, int grid, size_t smem, cudaStream_t s) {
  const auto kernel = w4_kernel<kBf16, NT, kXShared, kWarps, kGroup>;
  if (smem > 48 * 1024) {
    static std::atomic<unsigned long long> done{0};
    const cudaError_t e = ensure_smem(done, reinterpret_cast<const void*>(kernel), kMaxSmem);
    if (e != cudaSuccess) return e;
  }
  kernel<<<grid, kWarps * 32, smem, s>>>(a);
  return cudaGetLastError();
}
template <bool kBf16, int NT, bool kXShared, int kWarps>
cudaError_t launch(const W4Args& a, int grid, size_t smem, cudaStream_t s) {
  if (a.group == 32) return launch<kBf16, NT, kXShared, kWarps, 32>(a, grid, smem, s);
  if (a.group == 64) return launch<kBf16, NT, kXShared, kWarps, 64>(a, grid, smem, s);
  return launch<kBf16, NT, kXShared, kWarps, 128>(a, grid, smem, s);
}
template <bool kBf16, int NT>
cudaError_t launch(const W4Args& a, int warps, bool shared, int grid, size_t smem, cudaStream_t s) {
  if (!shared) return launch<kBf16, NT, false, 8>(a, grid, smem, s);
  return warps == 8 ? launch<kBf16, NT, true, 8>(a, grid, smem, s) : launch<kBf16, NT, true, 16>(a, grid, smem, s);
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
  if (static_cast<long long>(out_features) + kTileO > 0x7fffffffll || m > (1 << 24)) return LB_ERR_CAPACITY;

  const int blocks = (k + kBlockK - 1) / kBlockK, tiles = (out_features + kTileO - 1) / kTileO;
  const size_t x_row = static_cast<size_t>(blocks) * kBlockK * 2 + kXPad;
  constexpr size_t kLimit = kMaxSmem, kRing8 = 8 * kStageBytes, kRing16 = 16 * kStageBytes;  // of one stage
  // 16 rows of x a pass where they fit beside rings of four stages, else 8, else x stays where it is
  int nt = m > 8 ? 2 : 1;
  if (8 * nt * x_row + 4 * kRing8 > kLimit) nt = 1;
  const bool shared = 8 * nt * x_row + 4 * kRing8 <= kLimit;
  if (!shared) nt = m > 8 ? 2 : 1;
  const int m_tiles = (m + 8 * nt - 1) / (8 * nt);
  const size_t x_bytes = shared ? 8 * nt * x_row : 0;
  // Small products: CTAs of 8 warps, two an SM, with K split among a CTA's warps as far as one wave of
  // CTAs goes.  Large ones: 16 warps an SM (each SM loads x once) that walk over the tiles.
  const bool two = x_bytes + 4 * kRing8 <= kLimit / 2;
  const long long wave = 148ll * (two ? 2 : 1);
  int warps = 8, splits = 1;
  const auto ctas = [&](int w, int sp) { return static_cast<long long>((tiles + w / sp - 1) / (w / sp)) * m_tiles; };
  while (splits < 8 && splits < blocks && ctas(8, 2 * splits) <= wave) splits *= 2;
  if (ctas(8, splits) > wave && shared && x_bytes + 4 * kRing16 <= kLimit) {
    warps = 16;
    while (splits < 16 && splits < blocks && ctas(16, 2 * splits) <= 148) splits *= 2;
  }
  const size_t ring = warps == 8 ? kRing8 : kRing16, room = (warps == 8 && two ? kLimit / 2 : kLimit) - x_bytes;
  const int stages = room / ring > 8 ? 8 : static_cast<int>(room / ring);
  const size_t smem = x_bytes + stages * ring;
  // a split tile's CTA makes one pass (its sums take the rings' place)
  const long long all = (tiles + warps / splits - 1) / (warps / splits), fit = wave / (warps == 16 && two ? 2 : 1) / m_tiles;
  const long long grid = splits > 1 || all <= fit ? all : fit > 0 ? fit : 1;
  if (grid * m_tiles > 0x7fffffffll) return LB_ERR_CAPACITY;
  const W4Args a{x, x_ld, ld_out, x_scale, x_dtype, x_group, m, group, out_features, k, out_dtype, splits, stages, tiles, m_tiles,
                 static_cast<const uint8_t*>(codes), static_cast<const __half*>(w_scale), out};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int n = static_cast<int>(grid * m_tiles);
  cudaError_t e;
  if (x_dtype == LB_BF16)
    e = nt == 1 ? launch<true, 1>(a, warps, shared, n, smem, s) : launch<true, 2>(a, warps, shared, n, smem, s);
  else
    e = nt == 1 ? launch<false, 1>(a, warps, shared, n, smem, s) : launch<false, 2>(a, warps, shared, n, smem, s);
  return e == cudaSuccess ? LB_OK : LB_ERR_CUDA;
}
