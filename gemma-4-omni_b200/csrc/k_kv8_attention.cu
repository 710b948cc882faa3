// Attention over the paged 8-bit cache.
//
//   x_j = cap(scale * sk[page(j)] * q . kc_j),  p_j = exp(x_j - max),  j <= position, j > position - window
//   out = sum_j p_j sv[page(j)] vc_j / sum_j p_j,  lse = max + log sum_j p_j
//
// A task is 16 query rows of one (row, kv head): the tokens of the row times the
// query heads that share the kv head, so the cache is read once for all of them.
// Its keys are walked in tiles of 64, and all tasks' tiles in one line are dealt out
// evenly to as many CTAs as the SMs hold: rows of any lengths, many or one, keep
// every SM busy.  A CTA finds its share from prefix sums over the rows' lengths
// (on the device: the lengths may change under a captured graph).  Where a task is
// cut between CTAs, each leaves an unnormalised partial sum with its maximum in the
// workspace, and combine_kernel adds them up in the order of the keys, so results
// do not depend on which CTA finishes first.
//
// Inside a CTA each of four warps owns a quarter of the keys and its own ring of
// cp.async stages (16 keys of K and V), so the main loop has no block barrier.  The
// codes go from shared memory to mma.sync fragments without a layout pass: both
// products leave the order of the summed index free, so a lane takes the 16-byte
// pieces that it can load without bank conflicts (K: 32 columns of one key; V: 16
// columns of four keys) and q and the outputs are permuted to match.  Codes widen
// to fp16 exactly (byte permute into 1024 + u, minus 1152).  q is exact in fp16: fp16 as it
// is, bf16 times a power of two a row that brings the row's maximum to 2^14.  p is
// rounded to fp16 (2^-11, the one rounding between the scores and the sum); maximum,
// sums and outputs are held in 32 bits.  The V scale rides on the outputs: they are
// held in units of the current page's scale and change units with the rescaling
// that the running maximum asks for anyway.
#include "../../include/listener_b200.h"
#include "common.cuh"

namespace lb {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kRows = 16;       // query rows of a task (the m of the mma)
constexpr int kGroup = 16;      // keys of a stage
constexpr int kTile = kWarps * kGroup;
constexpr int kMinTiles = 2;    // a CTA takes at least this many tiles
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// the running maximum moves only when a score passes it by this much (log2):
// p stays below 2^8, far inside fp16, and most groups skip the rescaling
constexpr float kSlack = 8.0f;

struct AttendArgs {
  const void* q;
  long long q_token_stride, q_head_stride;
  int n_tokens, n_rows, heads, kv_heads;
  const int8_t *k_codes, *v_codes;
  const float *k_scale, *v_scale;
  int n_pages, page_tokens, max_pages;
  const int *row_tables, *kv_len, *cu_tokens;
  float scale, softcap;
  int window, q_vec;
  void* out;
  float* lse;
  int* status;
  float* parts;  // [2 * grid][16 * dim + 32]: outputs, maxima, sums of a cut task's parts
  int4* cuts;    // [grid]: (row, kv head, query tile, last CTA) of the task cut at the CTA's end; row -1: none
};

template <int D>
struct Shape {
  static constexpr int kHalf = D < 128 ? D : 128;       // columns a lane's K pieces cover together
  static constexpr int kHalves = D / kHalf;
  static constexpr int kSteps = kHalf / 16;             // mma k-steps a half
  static constexpr int kWords = kHalf / 16;             // 4-code words of K a lane and half: dims t * kHalf / 4 ...
  static constexpr int kCols = kHalf / 8;               // V columns a lane owns in a half
  static constexpr int kSide = kGroup * D;              // bytes of K (or V) of a stage
  static constexpr int kStages = D == 256 ? 3 : 4;
  static constexpr int kRing = kWarps * kStages * 2 * kSide;
  static constexpr bool kQShared = D == 256;            // q fragments in shared memory: 64 registers otherwise
  static constexpr int kQBytes = kQShared ? kHalves * kSteps * 512 : 0;
  static constexpr int kSmem = kRing + kQBytes;
  static constexpr int kCtas = D == 256 ? 2 : 3;        // an SM
  static constexpr int kPart = kRows * D + 2 * kRows;   // floats of a part
};

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// two biased codes (c + 128, with 0x64 above them: 1024 + c + 128) -> two fp16 codes
__device__ __forceinline__ uint32_t unbias(uint32_t h) {
  const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&h), __floats2half2_rn(1152.0f, 1152.0f));
  return *reinterpret_cast<const uint32_t*>(&v);
}
// 4 codes -> (c0, c1), (c2, c3)
__device__ __forceinline__ void widen4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  w ^= 0x80808080u;
  lo = unbias(__byte_perm(w, 0x64646464u, 0x4140));
  hi = unbias(__byte_perm(w, 0x64646464u, 0x4342));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t h;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(h) : "f"(hi), "f"(lo));
  return h;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 16-byte piece `col` of key `row` in a stage: the low bits are exchanged so
// that eight lanes' pieces of one access lie in different banks
template <int D>
__device__ __forceinline__ int piece(int row, int col) {
  if constexpr (D == 64) return row * 4 + (col ^ ((row >> 1) & 3));
  else return row * (D / 16) + (col ^ (row & 7));
}

template <typename T>
__device__ __forceinline__ float to_f(T v) {
  if constexpr (__is_same(T, __half)) return __half2float(v);
  else return __bfloat162float(v);
}

// What a row of the batch asks for.
struct Row {
  int begin, count, len, low, tiles, q_tiles;
};
__device__ __forceinline__ Row row_of(const AttendArgs& a, int r) {
  Row w{0, 0, 0, 0, 0, 0};
  if (r >= a.n_rows) return w;
  w.begin = min(max(a.cu_tokens[r], 0), a.n_tokens);
  w.count = min(max(a.cu_tokens[r + 1], w.begin), a.n_tokens) - w.begin;
  w.len = a.kv_len[r];
  if (w.count == 0) return w;
  const int room = a.max_pages * a.page_tokens;
  const int stop = min(max(w.len, 0), room);
  if (a.window) w.low = max(0, min(w.len - w.count + 1 - a.window, stop)) & ~(kGroup - 1);
  w.tiles = max(1, (stop - w.low + kTile - 1) / kTile);
  w.q_tiles = (w.count * (a.heads / a.kv_heads) + kRows - 1) / kRows;
  return w;
}
__device__ __forceinline__ long long row_work(const AttendArgs& a, const Row& w) {
  return static_cast<long long>(w.tiles) * w.q_tiles * a.kv_heads;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, Shape<D>::kCtas) attend_kernel(AttendArgs a) {
  using S = Shape<D>;
  extern __shared__ __align__(128) unsigned char attend_smem[];
  __shared__ long long pre[kThreads + 1];
  __shared__ float merge_m[kWarps][kRows], merge_l[kWarps][kRows];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int G = a.heads / a.kv_heads, P = a.page_tokens;

  // ---- this CTA's share of the line of tiles
  const int each = (a.n_rows + kThreads - 1) / kThreads;
  long long mine = 0;
  for (int r = tid * each; r < min(a.n_rows, (tid + 1) * each); ++r) mine += row_work(a, row_of(a, r));
  long long sum = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += y;
  }
  __shared__ long long warp_sum_[kWarps];
  if (lane == 31) warp_sum_[warp] = sum;
  __syncthreads();
  for (int w = 0; w < warp; ++w) sum += warp_sum_[w];
  pre[tid + 1] = sum;
  if (tid == 0) pre[0] = 0;
  __syncthreads();
  const long long W = pre[kThreads];
  const long long n_ctas = min(static_cast<long long>(gridDim.x), (W + kMinTiles - 1) / kMinTiles);
  // tokens of no row
  {
    const int last = min(max(a.cu_tokens[a.n_rows], 0), a.n_tokens);
    const int first = min(max(a.cu_tokens[0], 0), a.n_tokens);
    const long long pieces = static_cast<long long>(a.heads) * D / 8;
    for (long long i = static_cast<long long>(blockIdx.x) * kThreads + tid; i < a.n_tokens * pieces;
         i += static_cast<long long>(gridDim.x) * kThreads) {
      if (first == 0 && last == a.n_tokens) break;
      const long long tok = i / pieces;
      if (tok >= first && tok < last) continue;
      reinterpret_cast<int4*>(a.out)[i] = make_int4(0, 0, 0, 0);
      if (a.lse && i % (D / 8) == 0) a.lse[i / (D / 8)] = -INFINITY;
    }
  }
  const long long b = blockIdx.x;
  if (tid == 0) a.cuts[b] = make_int4(-1, 0, 0, 0);
  if (b >= n_ctas) return;
  long long x = W * b / n_ctas;
  const long long x_end = W * (b + 1) / n_ctas;
  if (x >= x_end) return;

  // the row that holds tile x: the thread chunk, then the row inside it
  int chunk = 0;
  {
    int lo = 0, hi = kThreads - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (pre[mid] <= x) lo = mid; else hi = mid - 1;
    }
    chunk = lo;
  }
  int win = chunk * each;          // rows [win, win + 32) are held by the lanes
  long long base = pre[chunk];     // tiles before row `win`
  Row held = row_of(a, win + lane);
  long long upto = row_work(a, held);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += y;
  }

  const uint32_t ring = smem_u32(attend_smem) + warp * (S::kStages * 2 * S::kSide);
  const unsigned char* ring_p = attend_smem + warp * (S::kStages * 2 * S::kSide);
  uint4* q_shared = reinterpret_cast<uint4*>(attend_smem + S::kRing);

  while (x < x_end) {
    // ---- the task
    unsigned after = __ballot_sync(0xffffffffu, base + upto > x);
    while (after == 0) {
      base += __shfl_sync(0xffffffffu, upto, 31);
      win += 32;
      held = row_of(a, win + lane);
      upto = row_work(a, held);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
      }
      after = __ballot_sync(0xffffffffu, base + upto > x);
    }
    const int at = __ffs(after) - 1, row = win + at;
    Row w;
    w.begin = __shfl_sync(0xffffffffu, held.begin, at);
    w.count = __shfl_sync(0xffffffffu, held.count, at);
    w.len = __shfl_sync(0xffffffffu, held.len, at);
    w.low = __shfl_sync(0xffffffffu, held.low, at);
    w.tiles = __shfl_sync(0xffffffffu, held.tiles, at);
    w.q_tiles = __shfl_sync(0xffffffffu, held.q_tiles, at);
    const long long y = x - (base + __shfl_sync(0xffffffffu, upto, at) - row_work(a, w));
    const int task = static_cast<int>(y / w.tiles), tile0 = static_cast<int>(y - static_cast<long long>(task) * w.tiles);
    const int hk = task / w.q_tiles, qt = task - hk * w.q_tiles;
    const int tile1 = static_cast<int>(min(static_cast<long long>(w.tiles), tile0 + (x_end - x)));
    const bool from_start = tile0 == 0, to_end = tile1 == w.tiles;
    x += tile1 - tile0;

    // rows of this task: query row i is token i / G, head hk * G + i % G
    const int rows = min(kRows, w.count * G - qt * kRows);
    const int r0 = qt * kRows + g, r1 = r0 + 8;
    const int pos0 = w.len - w.count + r0 / G, pos1 = w.len - w.count + r1 / G;
    const int pos_low = w.len - w.count + qt * kRows / G, pos_high = w.len - w.count + (qt * kRows + rows - 1) / G;
    const int stop = min(min(max(w.len, 0), a.max_pages * P), pos_high + 1);
    const int start = a.window ? max(w.low, pos_low + 1 - a.window) : 0;

    // this warp's groups, as indices of 16 keys from key 0
    const int per = ((tile1 - tile0) * kTile / kGroup + kWarps - 1) / kWarps;
    const int g_first = w.low / kGroup + tile0 * (kTile / kGroup);
    int ga = max(g_first + warp * per, start / kGroup);
    const int gb = min(g_first + min((warp + 1) * per, (tile1 - tile0) * (kTile / kGroup)), (stop + kGroup - 1) / kGroup);
    const int* table = a.row_tables + static_cast<long long>(row) * a.max_pages;

    // page and scales of 32 groups, a lane each
    int batch = ga;
    long long my_base = -1;
    float my_ks = 0.0f, my_vs = 0.0f;
    auto fetch_batch = [&](int from) {
      const int gi = from + lane;
      my_base = -1;
      my_ks = my_vs = 0.0f;
      if (gi < gb) {
        const int c = gi * kGroup / P;
        const int page = table[c];
        if (page >= 0 && page < a.n_pages) {
          const long long ph = static_cast<long long>(page) * a.kv_heads + hk;
          my_base = (ph * P + (gi * kGroup - c * P)) * D;
          my_ks = a.k_scale[ph];
          my_vs = a.v_scale[ph];
        } else if (a.status) {
          atomicOr(a.status, static_cast<int>(LB_DEV_BAD_PAGE));
        }
      }
    };
    if (ga < gb) fetch_batch(batch);
    // the batch that loads run ahead into
    int ahead = batch;
    long long ahead_base = my_base;
    auto issue = [&](int gi) {  // stage of group gi
      if (gi < gb) {
        if (gi - ahead >= 32) {
          ahead += 32;
          const int c = (ahead + lane) * kGroup / P;
          ahead_base = -1;
          if (ahead + lane < gb) {
            const int page = table[c];
            if (page >= 0 && page < a.n_pages)
              ahead_base = ((static_cast<long long>(page) * a.kv_heads + hk) * P + ((ahead + lane) * kGroup - c * P)) * D;
          }
        }
        const long long from = __shfl_sync(0xffffffffu, ahead_base, gi - ahead);
        if (from >= 0) {
          const uint32_t dst = ring + ((gi - ga) % S::kStages) * (2 * S::kSide);
#pragma unroll
          for (int i = 0; i < D / 32; ++i) {
            const int c = lane + 32 * i, kr = c / (D / 16), kc = c % (D / 16);
            const uint32_t o = piece<D>(kr, kc) * 16;
            cp_async16(dst + o, a.k_codes + from + c * 16);
            cp_async16(dst + S::kSide + o, a.v_codes + from + c * 16);
          }
        }
      }
      cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < S::kStages - 1; ++i) issue(ga + i);

    // ---- q fragments: lane (g, t) takes rows g and g + 8, columns half * 128 + t * kHalf / 4 + [0, kHalf / 4)
    uint32_t qf[S::kQShared ? 1 : S::kHalves * S::kSteps][4];
    float fac[2];
    {
      float top[2] = {0.0f, 0.0f};
      uint32_t raw[2][S::kHalves * S::kHalf / 8];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = e ? r1 : r0;
        const bool live = r - qt * kRows < rows;
        const T* src = static_cast<const T*>(a.q) + (w.begin + (live ? r / G : 0)) * a.q_token_stride +
                       (hk * G + (live ? r % G : 0)) * a.q_head_stride + t * (S::kHalf / 4);
#pragma unroll
        for (int h = 0; h < S::kHalves; ++h) {
          uint32_t* d = raw[e] + h * (S::kHalf / 8);
          if (a.q_vec) {
#pragma unroll
            for (int i = 0; i < S::kHalf / 32; ++i)
              *reinterpret_cast<int4*>(d + 4 * i) = live ? *reinterpret_cast<const int4*>(src + h * 128 + 8 * i)
                                                         : make_int4(0, 0, 0, 0);
          } else {
            const uint16_t* s16 = reinterpret_cast<const uint16_t*>(src + h * 128);
#pragma unroll
            for (int i = 0; i < S::kHalf / 8; ++i)
              d[i] = live ? s16[2 * i] | static_cast<uint32_t>(s16[2 * i + 1]) << 16 : 0u;
          }
        }
        if constexpr (!__is_same(T, __half)) {
#pragma unroll
          for (int i = 0; i < S::kHalves * S::kHalf / 8; ++i) {
            top[e] = fmaxf(top[e], fabsf(__uint_as_float(raw[e][i] << 16)));
            top[e] = fmaxf(top[e], fabsf(__uint_as_float(raw[e][i] & 0xffff0000u)));
          }
          top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 1));
          top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 2));
          // exponent that brings the row's maximum to [2^14, 2^15)
          const int ex = top[e] > 0.0f && top[e] < INFINITY ? 14 - ilogbf(top[e]) : 0;
#pragma unroll
          for (int i = 0; i < S::kHalves * S::kHalf / 8; ++i)
            raw[e][i] = pack_f16(ldexpf(__uint_as_float(raw[e][i] << 16), ex),
                                 ldexpf(__uint_as_float(raw[e][i] & 0xffff0000u), ex));
          fac[e] = ldexpf(a.softcap > 0.0f ? a.scale / a.softcap : a.scale * kLog2e, -ex);
        } else {
          fac[e] = a.softcap > 0.0f ? a.scale / a.softcap : a.scale * kLog2e;
        }
      }
      // step s of a half: columns 4 s + (0, 1) are k = 2t, 2t + 1 and 4 s + (2, 3) are k = 2t + 8, 2t + 9
      if constexpr (S::kQShared) {
        if (warp == 0) {
#pragma unroll
          for (int s = 0; s < S::kHalves * S::kSteps; ++s)
            q_shared[s * 32 + lane] = make_uint4(raw[0][2 * s], raw[1][2 * s], raw[0][2 * s + 1], raw[1][2 * s + 1]);
        }
        __syncthreads();
      } else {
#pragma unroll
        for (int s = 0; s < S::kHalves * S::kSteps; ++s) {
          qf[s][0] = raw[0][2 * s];
          qf[s][1] = raw[1][2 * s];
          qf[s][2] = raw[0][2 * s + 1];
          qf[s][3] = raw[1][2 * s + 1];
        }
      }
    }

    // ---- the keys
    float o[S::kHalves][S::kCols][4];
#pragma unroll
    for (int h = 0; h < S::kHalves; ++h)
#pragma unroll
      for (int i = 0; i < S::kCols; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[h][i][e] = 0.0f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f, unit = 1.0f;
    for (int gi = ga; gi < gb; ++gi) {
      cp_async_wait<S::kStages - 2>();
      __syncwarp();  // every lane's pieces of the stage are there, and every lane has left the one before
      issue(gi + S::kStages - 1);
      if (gi - batch >= 32) {
        batch += 32;
        fetch_batch(batch);
      }
      const bool there = __shfl_sync(0xffffffffu, my_base, gi - batch) >= 0;
      const float ks = __shfl_sync(0xffffffffu, my_ks, gi - batch);
      const float vs = __shfl_sync(0xffffffffu, my_vs, gi - batch);
      if (!there) continue;
      const unsigned char* kp = ring_p + ((gi - ga) % S::kStages) * (2 * S::kSide);
      const unsigned char* vp = kp + S::kSide;

      // scores of 16 keys: two n-tiles of 8, lane (g, t) supplies key 8 j + g
      float c[2][2][4] = {};  // [n-tile][even / odd step]: independent chains
#pragma unroll
      for (int h = 0; h < S::kHalves; ++h) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint32_t kw[S::kWords];
          if constexpr (D == 64) {
            *reinterpret_cast<uint4*>(kw) = *reinterpret_cast<const uint4*>(kp + piece<D>(8 * j + g, t) * 16);
          } else {
#pragma unroll
            for (int i = 0; i < 2; ++i)
              *reinterpret_cast<uint4*>(kw + 4 * i) =
                  *reinterpret_cast<const uint4*>(kp + piece<D>(8 * j + g, 8 * h + 2 * t + i) * 16);
          }
#pragma unroll
          for (int s = 0; s < S::kSteps; ++s) {
            uint32_t b0, b1;
            widen4(kw[s], b0, b1);
            if constexpr (S::kQShared) {
              const uint4 q4 = q_shared[(h * S::kSteps + s) * 32 + lane];
              mma_f16(c[j][s & 1], q4.x, q4.y, q4.z, q4.w, b0, b1);
            } else {
              const uint32_t* q4 = qf[h * S::kSteps + s];
              mma_f16(c[j][s & 1], q4[0], q4[1], q4[2], q4[3], b0, b1);
            }
          }
        }
      }
      // lane (g, t): rows g (v[.][0..1]) and g + 8 (v[.][2..3]), keys 8 j + 2 t + (0, 1)
      float v[2][4];
      const float f0 = ks * fac[0], f1 = ks * fac[1];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[j][e] = (c[j][0][e] + c[j][1][e]) * (e < 2 ? f0 : f1);
      if (a.softcap > 0.0f) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)  // tanh(u) = 1 - 2 / (1 + e^2u)
            v[j][e] = a.softcap * kLog2e * (1.0f - __fdividef(2.0f, 1.0f + exp2_fast(v[j][e] * (2.0f * kLog2e))));
      }
      const int key = gi * kGroup + 2 * t;
      if (gi * kGroup + kGroup > min(pos_low + 1, stop) || (a.window && gi * kGroup <= pos_high - a.window)) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int k = key + 8 * j + (e & 1), pos = e < 2 ? pos0 : pos1;
            if (k > pos || k >= stop || (a.window && k <= pos - a.window)) v[j][e] = -INFINITY;
          }
      }
      float t0 = fmaxf(fmaxf(v[0][0], v[0][1]), fmaxf(v[1][0], v[1][1]));
      float t1 = fmaxf(fmaxf(v[0][2], v[0][3]), fmaxf(v[1][2], v[1][3]));
#pragma unroll
      for (int s = 1; s < 4; s <<= 1) {
        t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, s));
        t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, s));
      }
      float s0 = 1.0f, s1 = 1.0f;
      if (t0 > m0 + kSlack || m0 == -INFINITY) {
        s0 = m0 == -INFINITY ? 0.0f : exp2_fast(m0 - t0);
        m0 = t0;
      }
      if (t1 > m1 + kSlack || m1 == -INFINITY) {
        s1 = m1 == -INFINITY ? 0.0f : exp2_fast(m1 - t1);
        m1 = t1;
      }
      // a page whose values are all zero adds nothing and keeps the unit
      float p_unit = 1.0f;
      if (vs != unit && vs != 0.0f) {
        p_unit = __fdividef(unit, vs);
        if (fabsf(p_unit) > 1e30f) p_unit = copysignf(1e30f, p_unit);
        unit = vs;
      }
      if (__any_sync(0xffffffffu, s0 != 1.0f || s1 != 1.0f) || p_unit != 1.0f) {
        l0 *= s0;
        l1 *= s1;
        const float u0 = s0 * p_unit, u1 = s1 * p_unit;
#pragma unroll
        for (int h = 0; h < S::kHalves; ++h)
#pragma unroll
          for (int i = 0; i < S::kCols; ++i) {
            o[h][i][0] *= u0;
            o[h][i][1] *= u0;
            o[h][i][2] *= u1;
            o[h][i][3] *= u1;
          }
      }
      const float n0 = m0 == -INFINITY ? 0.0f : m0, n1 = m1 == -INFINITY ? 0.0f : m1;
      uint32_t pa[4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float a0 = exp2_fast(v[j][0] - n0), a1 = exp2_fast(v[j][1] - n0);
        const float b0 = exp2_fast(v[j][2] - n1), b1 = exp2_fast(v[j][3] - n1);
        l0 += a0 + a1;
        l1 += b0 + b1;
        pa[2 * j] = pack_f16(a0, a1);
        pa[2 * j + 1] = pack_f16(b0, b1);
      }
      if (vs == 0.0f) continue;
      // outputs: lane (g, t) supplies keys 2t, 2t + 1, 2t + 8, 2t + 9 and the columns half * 128 + kCols g + i of n-tile i
#pragma unroll
      for (int h = 0; h < S::kHalves; ++h) {
        uint32_t vw[4][S::kCols / 4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int kr = 2 * t + (k & 1) + (k >> 1) * 8;
          if constexpr (D == 64) {
            *reinterpret_cast<uint2*>(vw[k]) =
                *reinterpret_cast<const uint2*>(vp + piece<D>(kr, g >> 1) * 16 + (g & 1) * 8);
          } else {
            *reinterpret_cast<uint4*>(vw[k]) = *reinterpret_cast<const uint4*>(vp + piece<D>(kr, 8 * h + g) * 16);
          }
        }
#pragma unroll
        for (int q = 0; q < S::kCols / 4; ++q) {
          uint32_t b[2][4];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t x0 = vw[2 * e][q] ^ 0x80808080u, x1 = vw[2 * e + 1][q] ^ 0x80808080u;
            const uint32_t lo = __byte_perm(x0, x1, 0x5140), hi = __byte_perm(x0, x1, 0x7362);
            b[e][0] = unbias(__byte_perm(lo, 0x64646464u, 0x4140));
            b[e][1] = unbias(__byte_perm(lo, 0x64646464u, 0x4342));
            b[e][2] = unbias(__byte_perm(hi, 0x64646464u, 0x4140));
            b[e][3] = unbias(__byte_perm(hi, 0x64646464u, 0x4342));
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
            mma_f16(o[h][4 * q + i], pa[0], pa[1], pa[2], pa[3], b[0][i], b[1][i]);
        }
      }
    }
    cp_async_wait<0>();
    l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 2);

    // ---- the four warps' parts, joined in shared memory (the rings are idle now)
    if (t == 0) {
      merge_m[warp][g] = m0;
      merge_m[warp][g + 8] = m1;
      merge_l[warp][g] = l0;
      merge_l[warp][g + 8] = l1;
    }
    __syncthreads();
    float* joined = reinterpret_cast<float*>(attend_smem);  // [warp][16][D], columns as lanes hold them
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = g + 8 * e;
      if (r < rows) {
        float top = merge_m[0][r];
#pragma unroll
        for (int k = 1; k < kWarps; ++k) top = fmaxf(top, merge_m[k][r]);
        const float f = top == -INFINITY ? 0.0f : exp2_fast((e ? m1 : m0) - top) * unit;
        // a lane's columns of a half are neighbours: kCols (2t) + i and kCols (2t + 1) + i
        float* d = joined + (warp * kRows + r) * D + t * 2 * S::kCols;
#pragma unroll
        for (int h = 0; h < S::kHalves; ++h)
#pragma unroll
          for (int c2 = 0; c2 < 2; ++c2)
#pragma unroll
            for (int i = 0; i < S::kCols; i += 4)
              *reinterpret_cast<float4*>(d + h * 128 + c2 * S::kCols + i) =
                  make_float4(o[h][i][2 * e + c2] * f, o[h][i + 1][2 * e + c2] * f, o[h][i + 2][2 * e + c2] * f,
                              o[h][i + 3][2 * e + c2] * f);
      }
    }
    __syncthreads();
    const bool whole = from_start && to_end;
    float* part = a.parts + (2 * b + (from_start ? 1 : 0)) * S::kPart;
    for (int i = tid; i < rows * (D / 4); i += kThreads) {
      const int r = i / (D / 4), d = (i - r * (D / 4)) * 4;
      float top = merge_m[0][r], l = 0.0f;
#pragma unroll
      for (int k = 1; k < kWarps; ++k) top = fmaxf(top, merge_m[k][r]);
      float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int k = 0; k < kWarps; ++k) {
        if (merge_m[k][r] > -INFINITY || merge_l[k][r] != 0.0f) {
          l += merge_l[k][r] * exp2_fast(merge_m[k][r] - top);
          const float4 z = *reinterpret_cast<const float4*>(joined + (k * kRows + r) * D + d);
          y.x += z.x;
          y.y += z.y;
          y.z += z.z;
          y.w += z.w;
        }
      }
      if (whole) {
        const float inv = l != 0.0f ? 1.0f / l : 0.0f;
        const int qr = qt * kRows + r;
        const long long to = (static_cast<long long>(w.begin + qr / G) * a.heads + hk * G + qr % G);
        T* dst = static_cast<T*>(a.out) + to * D + d;
        uint2 packed;
        if constexpr (__is_same(T, __half)) {
          packed = make_uint2(pack_f16(y.x * inv, y.y * inv), pack_f16(y.z * inv, y.w * inv));
        } else {
          packed = make_uint2(act_bits2(y.x * inv, y.y * inv, false), act_bits2(y.z * inv, y.w * inv, false));
        }
        *reinterpret_cast<uint2*>(dst) = packed;
        if (a.lse && d == 0) a.lse[to] = l != 0.0f ? (top + log2f(l)) * kLn2 : -INFINITY;
      } else {
        *reinterpret_cast<float4*>(part + r * D + d) = y;
        if (d == 0) {
          part[kRows * D + r] = top;
          part[kRows * D + kRows + r] = l;
        }
      }
    }
    if (from_start && !to_end && tid == 0) {
      // the last CTA of the task: the one whose share holds its last tile
      const long long last = x + (w.tiles - tile1) - 1;
      a.cuts[b] = make_int4(row, hk, qt, static_cast<int>(((last + 1) * n_ctas - 1) / W));
    }
    __syncthreads();  // the rings and the merge arrays are free again
  }
}

// Joins the parts of the task that is cut at the end of CTA blockIdx.x: query row
// blockIdx.y.  Lanes over columns, the warps' groups over parts, then the groups' sums in order.
template <typename T, int D>
__global__ void __launch_bounds__(256) combine_kernel(AttendArgs a) {
  using S = Shape<D>;
  constexpr int kLanes = D / 4, kParts = 256 / kLanes;
  __shared__ float4 sum_o[kParts][kLanes];
  __shared__ float sum_l[kParts], sum_m[kParts];
  const int4 cut = a.cuts[blockIdx.x];
  if (cut.x < 0) return;
  const int G = a.heads / a.kv_heads, r = blockIdx.y, qr = cut.z * kRows + r;
  const Row w = row_of(a, cut.x);
  if (qr >= w.count * G) return;
  const int lane = threadIdx.x % kLanes, grp = threadIdx.x / kLanes;
  const int first = blockIdx.x, n = cut.w - first + 1;
  float m = -INFINITY, l = 0.0f;
  float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int i = grp; i < n; i += kParts) {
    const float* part = a.parts + (2ll * (first + i) + (i == 0 ? 1 : 0)) * S::kPart;
    const float pm = part[kRows * D + r], pl = part[kRows * D + kRows + r];
    const float4 z = *reinterpret_cast<const float4*>(part + r * D + lane * 4);
    if (pm == -INFINITY && pl == 0.0f) continue;
    const float top = fmaxf(m, pm);
    const float f = m == -INFINITY ? 0.0f : exp2_fast(m - top), pf = exp2_fast(pm - top);
    l = l * f + pl * pf;
    y = make_float4(y.x * f + z.x * pf, y.y * f + z.y * pf, y.z * f + z.z * pf, y.w * f + z.w * pf);
    m = top;
  }
  sum_o[grp][lane] = y;
  if (lane == 0) {
    sum_m[grp] = m;
    sum_l[grp] = l;
  }
  __syncthreads();
  if (grp != 0) return;
  float top = -INFINITY;
  for (int k = 0; k < kParts; ++k) top = fmaxf(top, sum_m[k]);
  l = 0.0f;
  y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int k = 0; k < kParts; ++k) {
    if (sum_m[k] == -INFINITY && sum_l[k] == 0.0f) continue;
    const float f = exp2_fast(sum_m[k] - top);
    const float4 z = sum_o[k][lane];
    l += sum_l[k] * f;
    y = make_float4(y.x + z.x * f, y.y + z.y * f, y.z + z.z * f, y.w + z.w * f);
  }
  const float inv = l != 0.0f ? 1.0f / l : 0.0f;
  const long long to = static_cast<long long>(w.begin + qr / G) * a.heads + cut.y * G + qr % G;
  T* dst = static_cast<T*>(a.out) + to * D + lane * 4;
  if constexpr (__is_same(T, __half))
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_f16(y.x * inv, y.y * inv), pack_f16(y.z * inv, y.w * inv));
  else
    *reinterpret_cast<uint2*>(dst) =
        make_uint2(act_bits2(y.x * inv, y.y * inv, false), act_bits2(y.z * inv, y.w * inv, false));
  if (a.lse && lane == 0) a.lse[to] = l != 0.0f ? (top + log2f(l)) * kLn2 : -INFINITY;
}

int grid_of(int dim) { return 148 * (dim == 256 ? Shape<256>::kCtas : Shape<64>::kCtas); }

template <typename T, int D>
cudaError_t launch(const AttendArgs& a, cudaStream_t s) {
  using S = Shape<D>;
  cudaError_t e = cudaFuncSetAttribute(attend_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
  if (e != cudaSuccess) return e;
  const int grid = grid_of(D);
  attend_kernel<T, D><<<grid, kThreads, S::kSmem, s>>>(a);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  combine_kernel<T, D><<<dim3(grid, kRows), 256, 0, s>>>(a);
  return cudaGetLastError();
}
template <typename T>
cudaError_t launch(const AttendArgs& a, int dim, cudaStream_t s) {
  if (dim == 64) return launch<T, 64>(a, s);
  if (dim == 128) return launch<T, 128>(a, s);
  return launch<T, 256>(a, s);
}

bool bad_dim(int dim) { return dim != 64 && dim != 128 && dim != 256; }

}  // namespace
}  // namespace lb

extern "C" int64_t lb_kv8_attention_workspace(int dim) {
  if (lb::bad_dim(dim)) return LB_ERR_INVALID_ARGUMENT;
  const int64_t grid = lb::grid_of(dim);
  return grid * (2 * (lb::kRows * dim + 2 * lb::kRows) * 4 + 16);
}

extern "C" int lb_op_kv8_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, int q_dtype,
                                   int n_tokens, int n_rows, int heads, int kv_heads, int dim,
                                   const int8_t* k_codes, const int8_t* v_codes, const float* k_scale,
                                   const float* v_scale, int n_pages, int page_tokens, const int32_t* row_tables,
                                   int max_pages, const int32_t* kv_len, const int32_t* cu_tokens, float scale,
                                   int window, float softcap, void* out, float* lse, int32_t* status,
                                   void* workspace, void* stream) {
  using namespace lb;
  if (!q || !k_codes || !v_codes || !k_scale || !v_scale || !row_tables || !kv_len || !cu_tokens || !out ||
      !workspace || n_tokens < 1 || n_rows < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || n_pages < 1 ||
      max_pages < 1 || window < 0 || !(softcap >= 0.0f))
    return LB_ERR_INVALID_ARGUMENT;
  if ((q_dtype != LB_BF16 && q_dtype != LB_F16) || bad_dim(dim) || page_tokens < 16 || page_tokens > 256 ||
      page_tokens % 16 != 0 || static_cast<long long>(max_pages) * page_tokens > 0x7fffffffll - 64)
    return LB_ERR_INVALID_ARGUMENT;
  if (static_cast<long long>(n_tokens) * heads > 0x7fffffffll) return LB_ERR_CAPACITY;
  const auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  if (!aligned(k_codes) || !aligned(v_codes) || !aligned(out) || !aligned(workspace)) return LB_ERR_INVALID_ARGUMENT;
  const int q_vec = aligned(q) && q_token_stride % 8 == 0 && q_head_stride % 8 == 0;
  const int64_t grid = grid_of(dim);
  int4* cuts = static_cast<int4*>(workspace);
  AttendArgs a{q, q_token_stride, q_head_stride, n_tokens, n_rows, heads, kv_heads, k_codes, v_codes, k_scale, v_scale,
               n_pages, page_tokens, max_pages, row_tables, kv_len, cu_tokens, scale, softcap, window, q_vec, out, lse,
               status, reinterpret_cast<float*>(cuts + grid), cuts};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = q_dtype == LB_BF16 ? launch<__nv_bfloat16>(a, dim, s) : launch<__half>(a, dim, s);
  return e == cudaSuccess ? LB_OK : LB_ERR_CUDA;
}
