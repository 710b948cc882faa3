// Attention over the paged 8-bit cache.
//
//   x_j = cap(scale * sk[page(j)] * q . kc_j),  p_j = exp(x_j - max),  j <= position, j > position - window
//   out = sum_j p_j sv[page(j)] vc_j / sum_j p_j,  lse = max + log sum_j p_j
//
// Both products run on the tensor cores in whole numbers, on the codes as they lie in the
// cache (tcgen05 kind::i8): no code is ever widened.  q and p are split into signed
// 8-bit digits instead, which become neighbouring columns of one MMA:
//   q * 2^e = 65536 q2 + 256 q1 + q0   (e brings the row's maximum to 2^21: 22 bits and a sign)
//   p * sv / max sv * 63 * 2^16 = 65536 p2 + 256 p1 + p0   (per tile, relative to the tile's largest
//                                            score: an error of 2^-23 of the tile's largest term)
//   S^T[key, (digit, query)] = K . Q^T,   O^T[column, (digit, query)] = V^T . P^T
// The products are exact in 32-bit integers, and the digits' sums are joined in 32-bit
// floating point.  The fixed point of p is one of 128 keys: a tile's outputs leave
// the tensor memory each time and are added up in registers with the tile's factor.
//
// A task is R query rows of one (row, kv head): the tokens of the row times the
// query heads that share the kv head, so the cache is read once for all of them.
// Its keys are walked in tiles of 128, and all tasks' tiles in one line are dealt out
// evenly to one CTA per SM: rows of any lengths, many or one, keep every SM busy.
// A CTA finds its share from prefix sums over the rows' lengths (on the device: the
// lengths may change under a captured graph).  Where a task is cut between
// CTAs, each leaves an unnormalised part with its reference maximum in the workspace, and
// combine_kernel adds the parts up in the order of the keys, so results do not
// depend on which CTA finishes first.
//
// Warp roles: 0 loads (TMA boxes of 64 keys, or of the largest power of two that divides a
// page: an issued box costs the warp about 120 cycles whatever its size), 1 issues the MMAs of
// the scores, 14 those of the outputs (a thread that waits on a barrier before each tile's MMAs
// loses some 500 cycles to it, so the two do not share one), 2-5 and 6-9 turn the scores of
// even and of odd tiles into digits of p (a thread a key: tensor memory's lanes), each
// with a running sum of its own, 10-13 add up the outputs (a thread a column).
// Scores, digits and outputs have two buffers each, so neighbouring tiles overlap; the
// ring of K and V tiles takes the rest of the shared memory.
#include "../../include/listener_b200.h"
#include "common.cuh"
#include "kernels.h"

namespace lb {
namespace {

constexpr int kThreads = 480;
constexpr int kTile = 128;   // keys of a tile: the lanes of the tensor memory
constexpr int kBoxes = 8;    // most TMA boxes of a tile (pages are multiples of 16)
constexpr int kSms = 148;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kFixed = 4128768.0f;  // 63 * 2^16, below 2^22: rounded by one addition
// The reference maximum of a query is its first tile's and moves only when a tile's passes
// it by 2^60: sums of 2^60 * 2^31 terms are far inside the floating range.
constexpr float kSlack = 60.0f;

struct AttendArgs {
  const void* q;
  long long q_token_stride, q_head_stride;
  int n_tokens, n_rows, heads, kv_heads;
  const float *k_scale, *v_scale;
  int n_pages, page_tokens, max_pages;
  const int *row_tables, *kv_len, *cu_tokens;
  float scale, softcap;
  int window, q_vec;
  int box;  // keys of a TMA box: 16, 32 or 64, a divisor of page_tokens
  void* out;
  float* lse;
  int* status;
  float* parts;  // [2 * grid][R * dim + 2 R]: outputs, maxima, sums of a cut task's parts
  int4* cuts;    // [grid]: (row, kv head, query tile, last CTA) of the task cut at the CTA's end; row -1: none
};

template <int D, int R>
struct Shape {
  static constexpr int kHalves = D / 128 > 0 ? D / 128 : 1;
  static constexpr int kRow = D < 128 ? D : 128;            // bytes of a shared-memory row: the swizzle's span
  static constexpr int kHalfBytes = kTile * kRow;
  static constexpr int kSide = kTile * D;                   // K (or V) of a tile
  static constexpr int kN1 = R == 8 ? 32 : 3 * R;           // score columns: three digits (8 rows: and 8 of padding)
  static constexpr int kN2 = kN1;                           // output columns: three digits
  static constexpr int kS = (kN1 + 31) / 32 * 32;           // tensor-memory columns of a score buffer
  static constexpr int kOutBuffers = 2 * kS + 2 * kHalves * kN2 <= 512 ? 2 : 1;
  static constexpr int kColumns = 2 * kS + kOutBuffers * kHalves * kN2;
  static constexpr int kAlloc = kColumns <= 128 ? 128 : kColumns <= 256 ? 256 : 512;
  static constexpr int kQBytes = kHalves * kN1 * kRow;
  static constexpr int kPBytes = kN2 * kTile;
  static constexpr int kFixedBytes = (kQBytes + 1023) / 1024 * 1024 + 2 * kPBytes + 1024;
  static constexpr int kStages = (225 * 1024 - 8192 - kFixedBytes) / (2 * kSide) < 8
                                     ? (225 * 1024 - 8192 - kFixedBytes) / (2 * kSide) : 8;
  static constexpr int kSmem = kFixedBytes + kStages * 2 * kSide;
  static constexpr int kPart = R * D + 2 * R;
};

// ------------------------------------------------------------------ helpers
// D(tmem, s32) (+)= A(smem) * B(smem)^T, signed 8-bit operands
__device__ __forceinline__ void umma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
      "r"(accumulate)
      : "memory");
}
// s32 accumulators, s8 A and B; a_mn: A's rows are its contiguous dimension
__host__ __device__ constexpr uint32_t idesc_i8(int m, int n, bool a_mn) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (a_mn ? 1u << 15 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}
// Shared-memory matrix descriptor of rows of kRow bytes swizzled over their own span
// (128 or 64 bytes), eight rows a group.  The leading offset is 0: along the
// contiguous dimension a tile has one span (128-byte rows), or (64-byte rows, V^T with
// 64 columns) lanes 64-127 repeat lanes 0-63 and are not read.
template <int kRow>
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr) {
  return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | static_cast<uint64_t>((8 * kRow) >> 4) << 32 |
         static_cast<uint64_t>(1u) << 46 | static_cast<uint64_t>(kRow == 128 ? 2u : 4u) << 61;
}
template <int kRow>
__device__ __forceinline__ uint32_t swizzled(uint32_t off) {
  return off ^ (((off >> 7) & (kRow == 128 ? 7u : 3u)) << 4);
}

// three loads of C columns each and their wait in one statement: the
// registers are not valid, and must not be touched, before the wait
template <int C>
__device__ __forceinline__ void tmem_ld3(uint32_t a0, uint32_t a1, uint32_t a2, int (&x)[C], int (&y)[C], int (&z)[C]);
#define LB_R8(v) "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
#define LB_R16(v) LB_R8(v), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
template <>
__device__ __forceinline__ void tmem_ld3<8>(uint32_t a0, uint32_t a1, uint32_t a2, int (&x)[8], int (&y)[8], int (&z)[8]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%24];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%8,%9,%10,%11,%12,%13,%14,%15}, [%25];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%16,%17,%18,%19,%20,%21,%22,%23}, [%26];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : LB_R8(x), LB_R8(y), LB_R8(z)
      : "r"(a0), "r"(a1), "r"(a2)
      : "memory");
}
template <>
__device__ __forceinline__ void tmem_ld3<16>(uint32_t a0, uint32_t a1, uint32_t a2, int (&x)[16], int (&y)[16],
                                             int (&z)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%48];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%49];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47}, [%50];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : LB_R16(x), LB_R16(y), LB_R16(z)
      : "r"(a0), "r"(a1), "r"(a2)
      : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) { return (a > b || isnan(a)) ? a : b; }
// the largest of the warp's values, a NaN if there is one
__device__ __forceinline__ float warp_top(float x) {
  float y;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ float to_f(uint16_t bits) {
  if constexpr (__is_same(T, __half)) return __half2float(__ushort_as_half(bits));
  else return __uint_as_float(static_cast<uint32_t>(bits) << 16);
}
template <typename T>
__device__ __forceinline__ uint16_t to_bits(float v) {
  if constexpr (__is_same(T, __half)) return __half_as_ushort(__float2half_rn(v));
  else return __bfloat16_as_ushort(__float2bfloat16_rn(v));
}

// ------------------------------------------------------------------ the line of tasks
// What a row of the batch asks for.
struct Row {
  int begin, count, len, low, tiles, q_tiles;
};
template <int R>
__device__ __forceinline__ Row row_of(const AttendArgs& a, int r) {
  Row w{0, 0, 0, 0, 0, 0};
  if (r >= a.n_rows) return w;
  w.begin = min(max(a.cu_tokens[r], 0), a.n_tokens);
  w.count = min(max(a.cu_tokens[r + 1], w.begin), a.n_tokens) - w.begin;
  w.len = a.kv_len[r];
  if (w.count == 0) return w;
  const int stop = min(max(w.len, 0), a.max_pages * a.page_tokens);
  if (a.window) w.low = max(0, min(w.len - w.count + 1 - a.window, stop)) & ~(a.box - 1);
  w.tiles = max(1, (stop - w.low + kTile - 1) / kTile);
  w.q_tiles = (w.count * (a.heads / a.kv_heads) + R - 1) / R;
  return w;
}
__device__ __forceinline__ long long row_work(const AttendArgs& a, const Row& w) {
  return static_cast<long long>(w.tiles) * w.q_tiles * a.kv_heads;
}
__device__ __forceinline__ long long warp_prefix(long long v) {  // inclusive
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  return v;
}

// A CTA's part of a task.
struct Task {
  Row w;
  int row, hk, qt, rows, tile0, tile1;
  int pos_low, pos_high;  // positions of its first and last token
  int start, stop;        // keys that any of its tokens sees
  long long next;         // the line's tile after it
  __device__ __forceinline__ bool from_start() const { return tile0 == 0; }
  __device__ __forceinline__ bool to_end() const { return tile1 == w.tiles; }
};

// Walks the tasks of a CTA's share [x, x_end) of the line; a warp at a time, every role for itself.
template <int R>
struct Walk {
  long long x, x_end, base, upto;
  int win;
  Row held;
  __device__ __forceinline__ void begin(const AttendArgs& a, const long long* pre, int each, long long from, long long to) {
    x = from;
    x_end = to;
    int lo = 0, hi = kThreads - 1;
    while (lo < hi) {  // the chunk of rows that holds tile x
      const int mid = (lo + hi + 1) >> 1;
      if (pre[mid] <= x) lo = mid; else hi = mid - 1;
    }
    win = lo * each;
    base = pre[lo];
    held = row_of<R>(a, win + (threadIdx.x & 31));
    upto = warp_prefix(row_work(a, held));
  }
  __device__ __forceinline__ bool next(const AttendArgs& a, Task& t) {
    if (x >= x_end) return false;
    unsigned after = __ballot_sync(0xffffffffu, base + upto > x);
    while (after == 0) {
      base += __shfl_sync(0xffffffffu, upto, 31);
      win += 32;
      held = row_of<R>(a, win + (threadIdx.x & 31));
      upto = warp_prefix(row_work(a, held));
      after = __ballot_sync(0xffffffffu, base + upto > x);
    }
    const int at = __ffs(after) - 1;
    t.row = win + at;
    t.w.begin = __shfl_sync(0xffffffffu, held.begin, at);
    t.w.count = __shfl_sync(0xffffffffu, held.count, at);
    t.w.len = __shfl_sync(0xffffffffu, held.len, at);
    t.w.low = __shfl_sync(0xffffffffu, held.low, at);
    t.w.tiles = __shfl_sync(0xffffffffu, held.tiles, at);
    t.w.q_tiles = __shfl_sync(0xffffffffu, held.q_tiles, at);
    const long long y = x - (base + __shfl_sync(0xffffffffu, upto, at) - row_work(a, t.w));
    const int task = static_cast<int>(y / t.w.tiles);
    t.tile0 = static_cast<int>(y - static_cast<long long>(task) * t.w.tiles);
    t.hk = task / t.w.q_tiles;
    t.qt = task - t.hk * t.w.q_tiles;
    t.tile1 = static_cast<int>(min(static_cast<long long>(t.w.tiles), t.tile0 + (x_end - x)));
    x += t.tile1 - t.tile0;
    t.next = x;
    const int G = a.heads / a.kv_heads;
    t.rows = min(R, t.w.count * G - t.qt * R);
    t.pos_low = t.w.len - t.w.count + t.qt * R / G;
    t.pos_high = t.w.len - t.w.count + (t.qt * R + t.rows - 1) / G;
    t.stop = min(min(max(t.w.len, 0), a.max_pages * a.page_tokens), t.pos_high + 1);
    t.start = a.window ? max(t.w.low, t.pos_low + 1 - a.window) : 0;
    return true;
  }
};

// ------------------------------------------------------------------ the kernel
template <typename T, int D, int R>
__global__ void __launch_bounds__(kThreads, 1) attend_kernel(const AttendArgs a, const __grid_constant__ CUtensorMap k_map,
                                                             const __grid_constant__ CUtensorMap v_map) {
  using S = Shape<D, R>;
  extern __shared__ unsigned char attend_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(attend_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* ring = smem;                                  // [stage][K, V][half][128 keys][kRow]
  unsigned char* q_digits = ring + S::kStages * 2 * S::kSide;  // [half][digit * R + query][kRow]
  unsigned char* p_digits = q_digits + (S::kQBytes + 1023) / 1024 * 1024;  // [buffer][digit * R + query][128 keys]
  __shared__ uint64_t full[S::kStages], empty[S::kStages], s_full[2], s_empty[2], p_full[2], p_empty[2], o_full[2], o_empty[2];
  __shared__ uint64_t q_full, q_empty, f_full[4], tops[2], l_full, l_empty;
  __shared__ uint32_t tmem_slot;
  __shared__ long long pre[kThreads + 1];
  __shared__ long long warp_total[kThreads / 32];
  __shared__ float g_ks[S::kStages][kBoxes], g_vs[S::kStages][kBoxes], g_top[S::kStages];
  __shared__ unsigned g_there[S::kStages];
  __shared__ __align__(16) float fac_s[R];       // a query: its factor to log2 scores, and the keys that it sees
  __shared__ int last_s[R], first_s[R];
  __shared__ __align__(16) float tops_s[2][4][R];  // a tile's largest scores, by warp
  __shared__ __align__(16) float top_s[8][R], beta_s[8][R];
  __shared__ float mx_ring[4][R], v_ring[4];     // a tile's largest scores and largest V scale
  __shared__ __align__(16) float out_f[4][R];
  __shared__ float l_part[8][R], m_ref[2][R];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = a.heads / a.kv_heads, P = a.page_tokens;

  // ---- set-up, and this CTA's share of the line of tiles
  if (tid == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&s_full[b], 1);
      mbar_init(&s_empty[b], 4);
      mbar_init(&p_full[b], 4);
      mbar_init(&p_empty[b], 1);
      mbar_init(&o_full[b], 1);
      mbar_init(&o_empty[b], 4);
      mbar_init(&tops[b], 4);
    }
    for (int b = 0; b < 4; ++b) mbar_init(&f_full[b], 1);
    mbar_init(&q_full, 8);
    mbar_init(&q_empty, 1);
    mbar_init(&l_full, 8);
    mbar_init(&l_empty, 4);
    fence_barrier_init();
    a.cuts[blockIdx.x] = make_int4(-1, 0, 0, 0);
  }
  const int each = (a.n_rows + kThreads - 1) / kThreads;
  long long mine = 0;
  for (int r = tid * each; r < min(a.n_rows, (tid + 1) * each); ++r) mine += row_work(a, row_of<R>(a, r));
  long long sum = warp_prefix(mine);
  if (lane == 31) warp_total[warp] = sum;
  __syncthreads();
  for (int w = 0; w < warp; ++w) sum += warp_total[w];
  pre[tid + 1] = sum;
  if (tid == 0) pre[0] = 0;
  if constexpr (R == 8) {  // rows of padding: zero once
    for (int i = tid; i < S::kHalves * 8 * S::kRow / 4; i += kThreads) {
      const int h = i / (8 * S::kRow / 4), o = i - h * (8 * S::kRow / 4);
      reinterpret_cast<uint32_t*>(q_digits + h * S::kN1 * S::kRow + 24 * S::kRow)[o] = 0u;
    }
    fence_proxy_async_smem();
  }
  // tokens of no row
  {
    const int first = min(max(a.cu_tokens[0], 0), a.n_tokens);
    const int last = min(max(a.cu_tokens[a.n_rows], 0), a.n_tokens);
    const long long pieces = static_cast<long long>(a.heads) * D / 8;
    if (first != 0 || last != a.n_tokens)
      for (long long i = static_cast<long long>(blockIdx.x) * kThreads + tid; i < a.n_tokens * pieces;
           i += static_cast<long long>(gridDim.x) * kThreads) {
        const long long tok = i / pieces;
        if (tok >= first && tok < last) continue;
        reinterpret_cast<int4*>(a.out)[i] = make_int4(0, 0, 0, 0);
        if (a.lse && i % (D / 8) == 0) a.lse[i / (D / 8)] = -INFINITY;
      }
  }
  __syncthreads();
  const long long W = pre[kThreads];
  const long long n_ctas = min(static_cast<long long>(gridDim.x), W);
  const long long b = blockIdx.x;
  if (b >= n_ctas) return;
  Walk<R> walk;
  walk.begin(a, pre, each, W * b / n_ctas, W * (b + 1) / n_ctas);
  if (warp == 1) {
    tmem_alloc(&tmem_slot, S::kAlloc);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const uint32_t tmem_o = tmem + 2 * S::kS;
  bool ok = true;
  Task t;

  if (warp == 0) {
    // ---------------------------------------------------------------- loads
    int i = 0;  // tiles so far
    const uint64_t once = l2_policy_evict_first();
    const int nb = kTile / a.box, batch = 32 / nb;  // boxes of a tile, tiles of a batch
    const int own_tile = lane / nb, k = lane - own_tile * nb;
    while (ok && walk.next(a, t)) {
      const int* table = a.row_tables + static_cast<long long>(t.row) * a.max_pages;
      // the boxes of some tiles at a time, a lane each: where they lie and their scales
      for (int tile = t.tile0; ok && tile < t.tile1; tile += batch) {
        const int key = t.w.low + tile * kTile + lane * a.box;
        int where = -1;
        float ks = 0.0f, vs = 0.0f;
        if (key < t.stop && key + a.box > t.start && tile + own_tile < t.tile1) {
          const int c = key / P, page = table[c];
          if (page >= 0 && page < a.n_pages) {
            const int ph = page * a.kv_heads + t.hk;
            where = ph * P + (key - c * P);
            ks = a.k_scale[ph];
            vs = a.v_scale[ph];
          } else if (a.status) {
            atomicOr(a.status, static_cast<int>(LB_DEV_BAD_PAGE));
          }
        }
        const unsigned there = __ballot_sync(0xffffffffu, where >= 0);
        float v_top = fabsf(vs);
        for (int o = 1; o < nb; o <<= 1) v_top = max_nan(v_top, __shfl_xor_sync(0xffffffffu, v_top, o));
        for (int j = 0; j < batch && tile + j < t.tile1; ++j, ++i) {
          const int s = i % S::kStages;
          if (i >= S::kStages) ok = mbar_wait(&empty[s], ((i / S::kStages) - 1) & 1, a.status);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          const bool own = own_tile == j;
          const unsigned mask = (there >> (j * nb)) & ((1u << nb) - 1u);
          if (own) {
            g_ks[s][k] = ks;
            g_vs[s][k] = vs;
            if (k == 0) {
              g_there[s] = mask;
              g_top[s] = v_top;
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive_expect_tx(&full[s], __popc(mask) * (2 * a.box * D));
          __syncwarp();
          if (own && where >= 0) {
            unsigned char* kd = ring + s * 2 * S::kSide + k * a.box * S::kRow;
#pragma unroll
            for (int h = 0; h < S::kHalves; ++h) {
              tma_load_2d(kd + h * S::kHalfBytes, &k_map, &full[s], h * 128, where, once);
              tma_load_2d(kd + S::kSide + h * S::kHalfBytes, &v_map, &full[s], h * 128, where, once);
            }
          }
          __syncwarp();
        }
      }
    }
    // loads that nobody waited for (after a wait that ran out) end before the CTA does
    if (!ok)
      for (int k = max(0, i - S::kStages); k < i; ++k) mbar_wait(&full[k % S::kStages], (k / S::kStages) & 1, a.status);
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMAs of the scores: one thread
    constexpr uint32_t id = idesc_i8(128, S::kN1, false);
    int i = 0, task = 0;
    while (ok && walk.next(a, t)) {
      if (lane == 0) {
        const uint32_t q = smem_u32(q_digits);
        ok = mbar_wait(&q_full, task & 1, a.status);
        for (int tile = t.tile0; ok && tile < t.tile1; ++tile, ++i) {
          const int s = i % S::kStages, buf = i & 1;
          if (i >= 2) ok = mbar_wait(&s_empty[buf], ((i >> 1) - 1) & 1, a.status);
          if (!ok || !(ok = mbar_wait(&full[s], (i / S::kStages) & 1, a.status))) break;
          tc_fence_after();
          const uint32_t k = smem_u32(ring + s * 2 * S::kSide);
#pragma unroll
          for (int h = 0; h < S::kHalves; ++h)
#pragma unroll
            for (int n = 0; n < S::kRow / 32; ++n)
              umma_i8(tmem + buf * S::kS, smem_desc<S::kRow>(k + h * S::kHalfBytes + n * 32),
                      smem_desc<S::kRow>(q + h * S::kN1 * S::kRow + n * 32), id, h > 0 || n > 0);
          umma_commit(&s_full[buf]);
        }
        if (ok) umma_commit(&q_empty);
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      ++task;
    }
  } else if (warp == 14) {
    // ---------------------------------------------------------------- MMAs of the outputs: one thread
    constexpr uint32_t id = idesc_i8(128, S::kN2, true);
    constexpr int B = S::kOutBuffers;
    int i = 0;
    while (ok && walk.next(a, t)) {
      if (lane == 0) {
        for (int tile = t.tile0; ok && tile < t.tile1; ++tile, ++i) {
          const int s = i % S::kStages, buf = i & 1, ob = i % B;
          if (i >= B) ok = mbar_wait(&o_empty[ob], (i / B - 1) & 1, a.status);
          if (ok) ok = mbar_wait(&full[s], (i / S::kStages) & 1, a.status);
          if (!ok || !(ok = mbar_wait(&p_full[buf], (i >> 1) & 1, a.status))) break;
          tc_fence_after();
          const uint32_t v = smem_u32(ring + s * 2 * S::kSide + S::kSide), p = smem_u32(p_digits + buf * S::kPBytes);
#pragma unroll
          for (int h = 0; h < S::kHalves; ++h)
#pragma unroll
            for (int n = 0; n < kTile / 32; ++n)
              umma_i8(tmem_o + (ob * S::kHalves + h) * S::kN2,
                      smem_desc<S::kRow>(v + h * S::kHalfBytes + n * 32 * S::kRow), smem_desc<128>(p + n * 32), id, n > 0);
          umma_commit(&o_full[ob]);
          umma_commit(&p_empty[buf]);
          umma_commit(&empty[s]);
        }
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
    }
  } else if (warp < 10) {
    // ---------------------------------------------------------------- scores -> digits of p
    const int side = (warp - 2) >> 2, wq = (warp - 2) & 3, sub = warp & 3, key_row = sub * 32 + lane;
    const uint32_t scores = tmem + side * S::kS + (static_cast<uint32_t>(sub * 32) << 16);
    unsigned char* p = p_digits + side * S::kPBytes;
    constexpr int C = R < 16 ? R : 16;
    int i = 0, task = 0;
    while (ok && walk.next(a, t)) {
      // ---- the task's q, in digits: kPer threads a query, four columns at a time
      if (task > 0) ok = __all_sync(0xffffffffu, mbar_wait(&q_empty, (task - 1) & 1, a.status));
      if (!ok) break;
      constexpr int kPer = 256 / R < D / 4 ? 256 / R : D / 4, kE = D / kPer;
      const int qi = (tid - 64) / kPer, d0 = (tid - 64) % kPer * kE;
      if (qi < R) {  // whole warps: kPer divides 32, R * kPer is a multiple of 32
        const int qr = t.qt * R + qi;
        const bool live = qi < t.rows;
        const int tok = live ? qr / G : 0;
        const uint16_t* src = static_cast<const uint16_t*>(a.q) + (t.w.begin + tok) * a.q_token_stride +
                              (t.hk * G + (live ? qr - tok * G : 0)) * a.q_head_stride + d0;
        const auto four = [&](int e, float (&v)[4]) {
          uint16_t raw[4];
          if (a.q_vec) {
            const uint2 w = *reinterpret_cast<const uint2*>(src + e);
            raw[0] = static_cast<uint16_t>(w.x);
            raw[1] = static_cast<uint16_t>(w.x >> 16);
            raw[2] = static_cast<uint16_t>(w.y);
            raw[3] = static_cast<uint16_t>(w.y >> 16);
          } else {
#pragma unroll
            for (int c = 0; c < 4; ++c) raw[c] = src[e + c];
          }
#pragma unroll
          for (int c = 0; c < 4; ++c) v[c] = to_f<T>(raw[c]);
        };
        float top = 0.0f;
#pragma unroll 2
        for (int e = 0; e < kE; e += 4) {
          float v[4];
          four(e, v);
#pragma unroll
          for (int c = 0; c < 4; ++c) top = max_nan(top, fabsf(v[c]));
        }
#pragma unroll
        for (int o = 1; o < kPer; o <<= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
        const bool use = live && top < INFINITY;  // no NaN either
        // 2^ex brings the maximum to [2^21, 2^22); in two factors, each inside the floating range
        const int ex = use && top > 0.0f ? 21 + 127 - max(1, __float_as_int(top) >> 23) : 0;
        const int e1 = ex / 2, e2 = ex - e1;
        const float up1 = __int_as_float((127 + e1) << 23), up2 = __int_as_float((127 + e2) << 23);
        if (d0 == 0) {
          const float down = __int_as_float((127 - e1) << 23) * (a.softcap > 0.0f ? a.scale / a.softcap : a.scale * kLog2e);
          fac_s[qi] = top < INFINITY ? down * __int_as_float((127 - e2) << 23) : NAN;
          const int pos = t.w.len - t.w.count + qr / G;
          last_s[qi] = live ? min(pos, t.stop - 1) : t.stop - 1;
          first_s[qi] = live && a.window ? pos - a.window + 1 : 0;
        }
#pragma unroll 1
        for (int e = 0; e < kE; e += 4) {
          float f[4];
          four(e, f);
          uint32_t w0 = 0, w1 = 0, w2 = 0;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int v = use ? __float2int_rn(f[c] * up1 * up2) : 0;
            const uint32_t digits = (v + 0x8080) ^ 0x8080;  // bytes 0, 1, 2 (see the digits of p below)
            w0 |= ((digits >> 16) & 0xff) << (8 * c);
            w1 |= ((digits >> 8) & 0xff) << (8 * c);
            w2 |= (digits & 0xff) << (8 * c);
          }
          const int d = d0 + e, h = d / 128, col = d - h * 128;
          unsigned char* q = q_digits + h * S::kN1 * S::kRow;
          *reinterpret_cast<uint32_t*>(q + swizzled<S::kRow>(qi * S::kRow + col)) = w0;
          *reinterpret_cast<uint32_t*>(q + swizzled<S::kRow>((R + qi) * S::kRow + col)) = w1;
          *reinterpret_cast<uint32_t*>(q + swizzled<S::kRow>((2 * R + qi) * S::kRow + col)) = w2;
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full);
      ok = __all_sync(0xffffffffu, mbar_wait(&q_full, task & 1, a.status));  // what the other warps know of the queries

      float l[R];
#pragma unroll
      for (int q = 0; q < R; ++q) l[q] = 0.0f;
      float ref = -INFINITY;  // lane q: the reference maximum of query q (the four warps keep the same)
      for (int tile = t.tile0; ok && tile < t.tile1; ++tile, ++i) {
        if ((i & 1) != side) continue;
        const int s = i % S::kStages, phase = (i >> 1) & 1;
        ok = mbar_wait(&full[s], (i / S::kStages) & 1, a.status);
        if (ok) ok = mbar_wait(&s_full[side], phase, a.status);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        const int grp = key_row / a.box;
        const float ks = g_ks[s][grp], vs = g_vs[s][grp], v_top = g_top[s];
        const bool there = (g_there[s] >> grp) & 1u;
        float x[R];
#pragma unroll
        for (int c0 = 0; c0 < R; c0 += C) {
          int d2[C], d1[C], dd[C];
          tmem_ld3<C>(scores + c0, scores + R + c0, scores + 2 * R + c0, d2, d1, dd);
#pragma unroll
          for (int c = 0; c < C; ++c)
            x[c0 + c] = fmaf(__int2float_rn(d2[c]), 65536.0f, __int2float_rn(d1[c] * 256 + dd[c])) * (ks * fac_s[c0 + c]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_empty[side]);
        if (a.softcap > 0.0f) {
#pragma unroll
          for (int q = 0; q < R; ++q)  // tanh(u) = 1 - 2 / (1 + e^2u)
            x[q] = a.softcap * kLog2e * (1.0f - __fdividef(2.0f, 1.0f + exp2_fast(x[q] * (2.0f * kLog2e))));
        }
        const int key0 = t.w.low + tile * kTile, key = key0 + key_row;
        if (key0 + kTile > min(t.pos_low + 1, t.stop) || (a.window && key0 <= t.pos_high - a.window) ||
            __any_sync(0xffffffffu, !there)) {
#pragma unroll
          for (int q = 0; q < R; ++q)
            if (!there || key > last_s[q] || key < first_s[q]) x[q] = -INFINITY;
        }
        // the tile's largest score of each query: warp, then the four warps
        float mx = -INFINITY;
#pragma unroll
        for (int q = 0; q < R; ++q) {
          const float m = warp_top(x[q]);
          if (lane == q) mx = m;
        }
        if (lane < R) tops_s[side][wq][lane] = mx;
        __syncwarp();
        if (lane == 0) mbar_arrive(&tops[side]);
        ok = mbar_wait(&tops[side], phase, a.status);
        if (ok && i >= 2) ok = mbar_wait(&p_empty[side], phase ^ 1, a.status);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        float alpha = 1.0f;
        if (lane < R) {
          mx = max_nan(max_nan(tops_s[side][0][lane], tops_s[side][1][lane]),
                       max_nan(tops_s[side][2][lane], tops_s[side][3][lane]));
          if (ref == -INFINITY) {
            ref = mx;
          } else if (mx > ref + kSlack) {
            alpha = exp2_fast(ref - mx);
            ref = mx;
          }
          top_s[warp - 2][lane] = mx == -INFINITY ? 0.0f : mx;
          beta_s[warp - 2][lane] = mx == -INFINITY ? 0.0f : exp2_fast(mx - ref);
          if (wq == 0) mx_ring[i & 3][lane] = mx;
        }
        if (wq == 0 && lane == 0) v_ring[i & 3] = v_top;
        const bool moved = __any_sync(0xffffffffu, alpha != 1.0f);
        __syncwarp();
        if (wq == 0 && lane == 0) mbar_arrive(&f_full[i & 3]);
        if (moved) {
#pragma unroll
          for (int q = 0; q < R; ++q) l[q] *= __shfl_sync(0xffffffffu, alpha, q);
        }
        const float to_fixed = v_top > 0.0f ? __fdividef(vs, v_top) * kFixed : 0.0f;
#pragma unroll
        for (int q = 0; q < R; ++q) {
          const float e = exp2_fast(x[q] - top_s[warp - 2][q]);
          l[q] = fmaf(e, beta_s[warp - 2][q], l[q]);
          // v = rint(e * to_fixed) by a sum with 1.5 * 2^23.  With 128 added to each of the two lower
          // digits' places, the bytes of v are its signed digits, the lower two with the sign bit turned over.
          const uint32_t v = __float_as_uint(fmaf(e, to_fixed, 12582912.0f)) - 0x4B400000u;
          const uint32_t digits = (v + 0x8080u) ^ 0x8080u;
          p[swizzled<128>(q * kTile + key_row)] = static_cast<unsigned char>(digits >> 16);
          p[swizzled<128>((R + q) * kTile + key_row)] = static_cast<unsigned char>(digits >> 8);
          p[swizzled<128>((2 * R + q) * kTile + key_row)] = static_cast<unsigned char>(digits);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[side]);
      }
      // ---- the task's sums
      if (ok && task > 0) ok = mbar_wait(&l_empty, (task - 1) & 1, a.status);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
#pragma unroll
      for (int q = 0; q < R; ++q) {
        const float v = warp_sum(l[q]);
        if (lane == q) l_part[warp - 2][q] = v;
      }
      if (wq == 0 && lane < R) m_ref[side][lane] = ref;
      __syncwarp();
      if (lane == 0) mbar_arrive(&l_full);
      ++task;
    }
  } else {
    // ---------------------------------------------------------------- outputs
    const int sub = warp & 3, col = sub * 32 + lane;
    const uint32_t lane_at = static_cast<uint32_t>(sub * 32) << 16;
    constexpr int C = R < 16 ? R : 16;
    float* factor = out_f[sub];
    int i = 0, task = 0;
    while (ok && walk.next(a, t)) {
      float o[S::kHalves][R];
#pragma unroll
      for (int h = 0; h < S::kHalves; ++h)
#pragma unroll
        for (int q = 0; q < R; ++q) o[h][q] = 0.0f;
      float ref = -INFINITY;  // lane q: the reference maximum of query q
      for (int tile = t.tile0; ok && tile < t.tile1; ++tile, ++i) {
        const int buf = i % S::kOutBuffers;
        ok = __all_sync(0xffffffffu, mbar_wait(&f_full[i & 3], (i >> 2) & 1, a.status));
        if (!ok) break;
        float alpha = 1.0f;
        if (lane < R) {
          const float mx = mx_ring[i & 3][lane];
          if (ref == -INFINITY) {
            ref = mx;
          } else if (mx > ref + kSlack) {
            alpha = exp2_fast(ref - mx);
            ref = mx;
          }
          factor[lane] = mx == -INFINITY ? 0.0f : exp2_fast(mx - ref) * v_ring[i & 3] * (1.0f / kFixed);
        }
        __syncwarp();
        if (__any_sync(0xffffffffu, alpha != 1.0f)) {
#pragma unroll
          for (int q = 0; q < R; ++q) {
            const float f = __shfl_sync(0xffffffffu, alpha, q);
#pragma unroll
            for (int h = 0; h < S::kHalves; ++h) o[h][q] *= f;
          }
        }
        ok = __all_sync(0xffffffffu, mbar_wait(&o_full[buf], (i / S::kOutBuffers) & 1, a.status));
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int h = 0; h < S::kHalves; ++h)
#pragma unroll
          for (int c0 = 0; c0 < R; c0 += C) {
            int d2[C], d1[C], d0[C];
            const uint32_t at = tmem_o + (buf * S::kHalves + h) * S::kN2 + lane_at + c0;
            tmem_ld3<C>(at, at + R, at + 2 * R, d2, d1, d0);
#pragma unroll
            for (int c = 0; c < C; ++c)
              o[h][c0 + c] = fmaf(fmaf(__int2float_rn(d2[c]), 65536.0f, __int2float_rn(d1[c] * 256 + d0[c])),
                                  factor[c0 + c], o[h][c0 + c]);
          }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_empty[buf]);
      }
      if (ok) ok = mbar_wait(&l_full, task & 1, a.status);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      // lane q: the query's sum, its inverse, where it goes
      float l = 0.0f;
      long long to = 0;
      if (lane < t.rows) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float part = l_part[4 * k][lane] + l_part[4 * k + 1][lane] + l_part[4 * k + 2][lane] + l_part[4 * k + 3][lane];
          if (part != 0.0f) l += part * exp2_fast(m_ref[k][lane] - ref);
        }
        const int qr = t.qt * R + lane;
        to = static_cast<long long>(t.w.begin + qr / G) * a.heads + t.hk * G + qr % G;
      }
      const bool whole = t.from_start() && t.to_end();
      float* part = a.parts + (2 * b + (t.from_start() ? 1 : 0)) * S::kPart;
      if (lane < t.rows && sub == 0) {
        if (!whole) {
          part[R * D + lane] = ref;
          part[R * D + R + lane] = l;
        } else if (a.lse) {
          a.lse[to] = l != 0.0f ? (ref + log2f(l)) * kLn2 : -INFINITY;
        }
      }
      const float inv = whole ? (l != 0.0f ? 1.0f / l : 0.0f) : 1.0f;
#pragma unroll
      for (int q = 0; q < R; ++q) {
        if (q >= t.rows) break;
        const float f = __shfl_sync(0xffffffffu, inv, q);
        const long long at = __shfl_sync(0xffffffffu, to, q);
        if (col < D) {
#pragma unroll
          for (int h = 0; h < S::kHalves; ++h) {
            if (whole) static_cast<uint16_t*>(a.out)[at * D + h * 128 + col] = to_bits<T>(o[h][q] * f);
            else part[q * D + h * 128 + col] = o[h][q];
          }
        }
      }
      if (t.from_start() && !t.to_end() && sub == 0 && lane == 0) {
        // the last CTA of the task: the one whose share holds its last tile
        const long long last = t.next + (t.w.tiles - t.tile1) - 1;
        a.cuts[b] = make_int4(t.row, t.hk, t.qt, static_cast<int>(((last + 1) * n_ctas - 1) / W));
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&l_empty);
      ++task;
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, S::kAlloc);
  }
}

// Joins the parts of the task that is cut at the end of CTA blockIdx.x: query row
// blockIdx.y.  Lanes over columns, the groups of lanes over parts, then the groups' sums in order.
template <typename T, int D, int R>
__global__ void __launch_bounds__(256) combine_kernel(const AttendArgs a) {
  using S = Shape<D, R>;
  constexpr int kLanes = D / 4, kParts = 256 / kLanes;
  __shared__ float4 sum_o[kParts][kLanes];
  __shared__ float sum_l[kParts], sum_m[kParts];
  pdl_wait();
  const int4 cut = a.cuts[blockIdx.x];
  if (cut.x < 0) return;
  const int G = a.heads / a.kv_heads, r = blockIdx.y, qr = cut.z * R + r;
  const Row w = row_of<R>(a, cut.x);
  if (qr >= w.count * G) return;
  const int lane = threadIdx.x % kLanes, grp = threadIdx.x / kLanes;
  const int first = blockIdx.x, n = cut.w - first + 1;
  float m = -INFINITY, l = 0.0f;
  float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int i = grp; i < n; i += kParts) {
    const float* part = a.parts + (2ll * (first + i) + (i == 0 ? 1 : 0)) * S::kPart;
    const float pm = part[R * D + r], pl = part[R * D + R + r];
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
  uint16_t* dst = static_cast<uint16_t*>(a.out) + to * D + lane * 4;
  *reinterpret_cast<uint2*>(dst) =
      make_uint2(to_bits<T>(y.x * inv) | static_cast<uint32_t>(to_bits<T>(y.y * inv)) << 16,
                 to_bits<T>(y.z * inv) | static_cast<uint32_t>(to_bits<T>(y.w * inv)) << 16);
  if (a.lse && lane == 0) a.lse[to] = l != 0.0f ? (top + log2f(l)) * kLn2 : -INFINITY;
}

// Query rows of a task: as few as hold the rows of most requests, so that the tensor
// memory's columns and the threads' work are not spent on padding.
int rows_of(int max_new, int group) {
  const long long rows = static_cast<long long>(max_new) * group;
  return rows <= 8 ? 8 : rows <= 16 ? 16 : 32;
}

template <typename T, int D, int R>
cudaError_t launch(const AttendArgs& a, const CUtensorMap& k_map, const CUtensorMap& v_map, cudaStream_t s) {
  using S = Shape<D, R>;
  static std::atomic<unsigned long long> done{0};
  cudaError_t e = ensure_smem(done, reinterpret_cast<const void*>(attend_kernel<T, D, R>), S::kSmem);
  if (e != cudaSuccess) return e;
  attend_kernel<T, D, R><<<kSms, kThreads, S::kSmem, s>>>(a, k_map, v_map);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  return launch_kernel(true, combine_kernel<T, D, R>, dim3(kSms, R), dim3(256), 0, s, a);
}
template <typename T, int D>
cudaError_t launch(const AttendArgs& a, int rows, const CUtensorMap& k_map, const CUtensorMap& v_map, cudaStream_t s) {
  if (rows == 8) return launch<T, D, 8>(a, k_map, v_map, s);
  if (rows == 16) return launch<T, D, 16>(a, k_map, v_map, s);
  return launch<T, D, 32>(a, k_map, v_map, s);
}
template <typename T>
cudaError_t launch(const AttendArgs& a, int dim, int rows, const CUtensorMap& k_map, const CUtensorMap& v_map,
                   cudaStream_t s) {
  if (dim == 64) return launch<T, 64>(a, rows, k_map, v_map, s);
  if (dim == 128) return launch<T, 128>(a, rows, k_map, v_map, s);
  return launch<T, 256>(a, rows, k_map, v_map, s);
}

bool bad_dim(int dim) { return dim != 64 && dim != 128 && dim != 256; }

}  // namespace
}  // namespace lb

extern "C" int64_t lb_kv8_attention_workspace(int dim, int heads, int kv_heads, int max_new) {
  if (lb::bad_dim(dim) || kv_heads < 1 || heads < 1 || heads % kv_heads != 0 || max_new < 1) return LB_ERR_INVALID_ARGUMENT;
  const int64_t rows = lb::rows_of(max_new, heads / kv_heads);
  return lb::kSms * (2 * (rows * dim + 2 * rows) * 4 + 16);
}

extern "C" int lb_op_kv8_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, int q_dtype,
                                   int n_tokens, int n_rows, int heads, int kv_heads, int dim,
                                   const int8_t* k_codes, const int8_t* v_codes, const float* k_scale,
                                   const float* v_scale, int n_pages, int page_tokens, const int32_t* row_tables,
                                   int max_pages, const int32_t* kv_len, const int32_t* cu_tokens, int max_new,
                                   float scale, int window, float softcap, void* out, float* lse, int32_t* status,
                                   void* workspace, void* stream) {
  using namespace lb;
  if (!q || !k_codes || !v_codes || !k_scale || !v_scale || !row_tables || !kv_len || !cu_tokens || !out ||
      !workspace || n_tokens < 1 || n_rows < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || n_pages < 1 ||
      max_pages < 1 || max_new < 1 || window < 0 || !(softcap >= 0.0f))
    return LB_ERR_INVALID_ARGUMENT;
  if ((q_dtype != LB_BF16 && q_dtype != LB_F16) || bad_dim(dim) || page_tokens < 16 || page_tokens > 256 ||
      page_tokens % 16 != 0 || static_cast<long long>(max_pages) * page_tokens > 0x7fffffffll - 2 * kTile)
    return LB_ERR_INVALID_ARGUMENT;
  // rows of the cache are TMA coordinates, and a row's query rows are counted in 32 bits
  if (static_cast<long long>(n_tokens) * heads > 0x7fffffffll ||
      static_cast<long long>(n_pages) * kv_heads > 0x7fffffffll / page_tokens)
    return LB_ERR_CAPACITY;
  const auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  if (!aligned(k_codes) || !aligned(v_codes) || !aligned(out) || !aligned(workspace)) return LB_ERR_INVALID_ARGUMENT;
  const int q_vec = aligned(q) && q_token_stride % 8 == 0 && q_head_stride % 8 == 0;
  const int box = page_tokens % 64 == 0 ? 64 : page_tokens % 32 == 0 ? 32 : 16;
  int4* cuts = static_cast<int4*>(workspace);
  AttendArgs a{q, q_token_stride, q_head_stride, n_tokens, n_rows, heads, kv_heads, k_scale, v_scale, n_pages,
               page_tokens, max_pages, row_tables, kv_len, cu_tokens, scale, softcap, window, q_vec, box, out, lse, status,
               reinterpret_cast<float*>(cuts + kSms), cuts};
  const uint64_t cache_rows = static_cast<uint64_t>(n_pages) * kv_heads * page_tokens;
  const uint32_t span = dim < 128 ? dim : 128;
  CUtensorMap k_map, v_map;
  if (make_tensor_map_u8(&k_map, k_codes, dim, cache_rows, span, box) != 0 ||
      make_tensor_map_u8(&v_map, v_codes, dim, cache_rows, span, box) != 0)
    return LB_ERR_CUDA;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int rows = rows_of(max_new, heads / kv_heads);
  const cudaError_t e = q_dtype == LB_BF16 ? launch<__nv_bfloat16>(a, dim, rows, k_map, v_map, s)
                                           : launch<__half>(a, dim, rows, k_map, v_map, s);
  return e == cudaSuccess ? LB_OK : LB_ERR_CUDA;
}
