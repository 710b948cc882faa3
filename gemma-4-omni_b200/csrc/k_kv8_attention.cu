// Attention over the paged 8-bit cache.
//
//   x_j = cap(scale * sk[page(j)] * q . kc_j),  p_j = exp(x_j - max),  j <= position, j > position - window
//   out = sum_j p_j sv[page(j)] vc_j / sum_j p_j,  lse = max + log sum_j p_j
//
// Both products run on the tensor cores in whole numbers, on the codes as they lie in the
// cache (tcgen05 kind::i8): no code is ever widened.  q and p are split into signed
// 8-bit digits instead, which become neighbouring columns of one MMA:
//   q * 2^e = 2^24 q3 + 65536 q2 + 256 q1 + q0   (e brings the row's maximum to 2^29: 30 bits and a sign, so that
//                  16-bit values keep all their bits down to 2^-19 (fp16) or 2^-22 (bf16) of the largest)
//   p * sv * c = 65536 p2 + 256 p1 + p0   (c, of each tile and query, brings the largest p * sv among the
//                  keys that the query sees to 63 * 2^16: an error of 2^-23 of that largest p * sv a key)
//   S^T[key, (digit, query)] = K . Q^T,   O^T[column, (digit, query)] = V^T . P^T
// c takes the largest p * sv, not the largest p times the largest sv: the pages of a tile may have scales far
// apart, and the key with the weight the smallest.  Pages that a query does not see do not count for it.
// The products are exact in 32-bit integers, and the digits' sums are joined in 32-bit
// floating point (up to 2^45 before they take the scale of K, so that one stays in range below 2^80).  The
// fixed point of p is one of 128 keys: a tile's outputs leave the tensor memory each time and are added up in
// registers with the tile's factor.
//
// A task is R query rows of one (row, kv head): the tokens of the row times the
// query heads that share the kv head, so the cache is read once for all of them.
// Its keys are walked in tiles of 128, and all tasks' tiles in one line (a few more for a task's
// set-up: without them the CTAs with the short rows took up to 1.5 times as long as the rest) are dealt
// out evenly to one CTA per SM: rows of any lengths, many or one, keep every SM busy.
// A CTA finds its share from prefix sums over the rows' lengths (on the device: the
// lengths may change under a captured graph).  Where a task is cut between
// CTAs, each leaves an unnormalised part with its reference maximum in the workspace, and
// combine_kernel adds the parts up in the order of the keys, so results do not
// depend on which CTA finishes first.
//
// Warp roles: 0 loads (TMA boxes of 64 keys, or of the largest power of two that divides a page; the page
// tables of the batch of tiles after the next and the scales of the next are under way meanwhile), 1
// issues the MMAs of the scores, 2 those of the outputs (a thread that waits on a barrier before
// each tile's MMAs loses some 500 cycles to it, so the two do not share one), 3 splits the next task's
// q into digits while the present one runs, 4-7 and 8-11 turn scores into digits of p (a thread a key: tensor
// memory's lanes), 12-15 add up the outputs (a thread a column).  K and V lie in one ring of units
// of 128 keys, K freed by its scores, V by its outputs.
//
// Six roles in sixteen warps share one instruction cache, and its misses bound the kernel before anything else
// did: loops are kept rolled, a score warpgroup takes 8 queries at a time (16 unrolled took 6.9 thousand
// cycles a tile, 8 take 2.5), waits are a few instructions.  Measured: 64 answers over 0.5 million keys with 8 kv
// heads of 128 in 207 to 215 us (1.02 GB at 4.8 TB/s, 75 % of the copy rate; bound by the load warp and the rows'
// raggedness), ticks of 1024 sessions with a window of 1024 keys and 16 query rows of 256 columns in 131 us (3.5
// TB/s; bound by the score warps' chain), one answer over 16384 keys in 22 us (the chain of set-up, one
// tile and the join), chunks of 128 to 512 tokens with a soft cap in 900 us (101 TFLOP/s; bound by the score warps'
// instructions, some 27 a query and key).  Four score warpgroups instead of two were slower (answers 289 us).
#include "../../include/listener_b200.h"
#include "common.cuh"
#include "kernels.h"

namespace lb {
namespace {

constexpr int kThreads = 512;
constexpr int kTile = 128;   // keys of a tile: the lanes of the tensor memory
constexpr int kBoxes = 8;    // most TMA boxes of a tile (pages are multiples of 16)
constexpr int kQueries = 8;    // queries of a score warpgroup's turn
constexpr int kScorers = 2;    // score warpgroups
constexpr int kFirstScorer = 4, kFirstOutput = 12;  // warps
constexpr int kRing = 8;       // tiles whose largest scores are kept: more than the digits' and outputs' buffers together
constexpr int kTasks = 8;      // tasks that the loading warp may be ahead
constexpr int kInfo = 16;      // tiles whose scales are kept: more than the ring's units reach ahead
constexpr int kTaskCost = 6;   // a task's set-up in tiles, as the line counts it (measured: 2 and 8 are slower for one case each)
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
  int box, box_log;  // keys of a TMA box: 16, 32 or 64, a divisor of page_tokens
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
  static constexpr int kN1 = 4 * R;                         // score columns: four digits
  static constexpr int kN2 = R == 8 ? 32 : 3 * R;           // output columns: three digits (8 rows: and 8 that nobody reads)
  static constexpr int kS = (kN1 + 31) / 32 * 32;           // tensor-memory columns of a score buffer
  static constexpr int kBuffers = 4 * kS + 2 * kHalves * kN2 <= 512 ? 4 : 2;  // of scores and of digits of p
  static constexpr int kColumns = kBuffers * kS + 2 * kHalves * kN2;
  static_assert(kColumns <= 512, "tensor memory");
  static constexpr int kAlloc = kColumns <= 128 ? 128 : kColumns <= 256 ? 256 : 512;
  static constexpr int kQBytes = (kHalves * kN1 * kRow + 1023) / 1024 * 1024;
  static constexpr int kPBytes = kN2 * kTile;
  static constexpr int kFixedBytes = 2 * kQBytes + kBuffers * kPBytes + 1024;
  static constexpr int kRoom = (219 * 1024 - kFixedBytes) / kSide;  // (up to 8 KB are declared beside it)
  static constexpr int kUnits = kRoom < kInfo ? kRoom : kInfo;  // (a tile's scales outlive its units)
  static constexpr int kSmem = kFixedBytes + kUnits * kSide;
  static constexpr int kTurns = R / kQueries;             // of the score warpgroups, a tile
  static constexpr int kEvery = kScorers / kTurns;        // a warpgroup takes its turn in every so many tiles
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

// three (or four) loads of C columns each and their wait in one statement: the
// registers are not valid, and must not be touched, before the wait
template <int C>
__device__ __forceinline__ void tmem_ld3(uint32_t a0, uint32_t a1, uint32_t a2, int (&x)[C], int (&y)[C], int (&z)[C]);
#define LB_R8(v) "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
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
__device__ __forceinline__ void tmem_ld4(uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, int (&x)[8], int (&y)[8],
                                         int (&z)[8], int (&w)[8]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%32];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%8,%9,%10,%11,%12,%13,%14,%15}, [%33];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%16,%17,%18,%19,%20,%21,%22,%23}, [%34];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%24,%25,%26,%27,%28,%29,%30,%31}, [%35];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : LB_R8(x), LB_R8(y), LB_R8(z), LB_R8(w)
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3)
      : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
struct Scores {
  float v[kQueries];
};
// cap * tanh(s / cap), inv = 1 / cap, for a warp together.  Near zero (u = s / cap, w = u * u below kSmall) s times the
// series of tanh(u) / u, whose first term left out is below 2^-26; elsewhere 1 - 2 / (1 + e^2u).  An error of some
// 2^-20 of the result for every cap.  The second form is not in line: most scores are small beside their cap.
constexpr float kSmall = 0.0625f;
__device__ __forceinline__ float tanh_series(float w) {
  return fmaf(w, fmaf(w, fmaf(w, fmaf(w, 62.0f / 2835.0f, -17.0f / 315.0f), 2.0f / 15.0f), -1.0f / 3.0f), 1.0f);
}
__device__ __noinline__ Scores capped_far(Scores s, float cap, float inv) {
#pragma unroll
  for (int q = 0; q < kQueries; ++q) {
    const float u = s.v[q] * inv, w = u * u;
    s.v[q] = w < kSmall ? s.v[q] * tanh_series(w) : cap - __fdividef(2.0f, 1.0f + exp2_fast(u * (2.0f * kLog2e))) * cap;
  }
  return s;
}
__device__ __forceinline__ Scores capped(Scores s, float cap, float inv) {
  float w[kQueries];
  bool near = true;
#pragma unroll
  for (int q = 0; q < kQueries; ++q) {
    w[q] = s.v[q] * inv;
    w[q] *= w[q];
    near = near && w[q] < kSmall;
  }
  if (!__all_sync(0xffffffffu, near)) return capped_far(s, cap, inv);
#pragma unroll
  for (int q = 0; q < kQueries; ++q) s.v[q] *= tanh_series(w[q]);
  return s;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Waits for a phase.  Bounded by the number of polls: try_wait sleeps in hardware, for up to the 20 us
// that it is given, so the limit is at most 2.6 s.  Kept short, because all roles
// together are bound by the instructions they issue.
constexpr int kPolls = 1 << 17;
__device__ __forceinline__ bool wait_one(uint64_t* bar, uint32_t parity) {
  const uint32_t at = smem_u32(bar);
#pragma unroll 1
  for (int n = 0; n < kPolls; ++n) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(at), "r"(parity), "r"(20000u)
        : "memory");
    if (done) return true;
  }
  return false;
}
// by a whole warp: the same answer for every lane
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, wait_one(bar, parity));
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
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
  int pos0;  // position of its first token
};
template <int R>
__device__ __forceinline__ Row row_of(const AttendArgs& a, int r) {
  Row w{0, 0, 0, 0, 0, 0, 0};
  if (r >= a.n_rows) return w;
  w.begin = min(max(a.cu_tokens[r], 0), a.n_tokens);
  w.count = min(max(a.cu_tokens[r + 1], w.begin), a.n_tokens) - w.begin;
  w.len = a.kv_len[r];
  w.pos0 = w.len - (max(a.cu_tokens[r + 1], w.begin) - w.begin);  // (also where q ends before the row does)
  if (w.count == 0) return w;
  const int stop = min(max(w.len, 0), a.max_pages * a.page_tokens);
  if (a.window) {
    const long long low = min(static_cast<long long>(w.pos0) + 1 - a.window, static_cast<long long>(stop));
    w.low = static_cast<int>(max(0ll, low)) & ~(a.box - 1);
  }
  w.tiles = max(1, (stop - w.low + kTile - 1) / kTile);
  w.q_tiles = (w.count * (a.heads / a.kv_heads) + R - 1) / R;
  return w;
}
// in the line's units
__device__ __forceinline__ long long row_work(const AttendArgs& a, const Row& w) {
  return static_cast<long long>(w.tiles + kTaskCost) * w.q_tiles * a.kv_heads;
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

// A CTA's part of a task, as the loading warp hands it to the others (n 0: there are no more).
struct Task {
  int n;                    // tiles
  int tile0, low;           // its first tile; key 0 of tile 0
  int rows, hk, qt, begin;  // query rows; kv head, query tile; the batch row's first token
  int pos_low, pos_high;    // positions of its first and last token
  int start, stop;          // keys that any of its tokens sees
  int row, q_tiles;
  int from_start, to_end;   // whether the task's first and last tiles are among these
  int last_cta;             // of a task that goes on after them: the CTA that has its last tile
};

// Walks the tasks of a CTA's share [x, x_end) of the line (a warp together).
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
  __device__ __noinline__ bool next(const AttendArgs& a, long long line, long long n_ctas, Task& t) {
    Row w;
    do {  // (the share may end, or begin, in a task's set-up: a part without tiles is passed over)
      if (x >= x_end) {
        t.n = 0;
        return false;
      }
      unsigned after = __ballot_sync(0xffffffffu, base + upto > x);
#pragma unroll 1
      while (after == 0) {
        base += __shfl_sync(0xffffffffu, upto, 31);
        win += 32;
        if (win >= a.n_rows) {  // (only where the lengths changed under the call: its outputs are lost, but it ends)
          t.n = 0;
          return false;
        }
        held = row_of<R>(a, win + (threadIdx.x & 31));
        upto = warp_prefix(row_work(a, held));
        after = __ballot_sync(0xffffffffu, base + upto > x);
      }
      const int at = __ffs(after) - 1;
      t.row = win + at;
      w.begin = __shfl_sync(0xffffffffu, held.begin, at);
      w.count = __shfl_sync(0xffffffffu, held.count, at);
      w.len = __shfl_sync(0xffffffffu, held.len, at);
      w.low = __shfl_sync(0xffffffffu, held.low, at);
      w.tiles = __shfl_sync(0xffffffffu, held.tiles, at);
      w.q_tiles = __shfl_sync(0xffffffffu, held.q_tiles, at);
      w.pos0 = __shfl_sync(0xffffffffu, held.pos0, at);
      const int length = w.tiles + kTaskCost;
      const long long y = x - (base + __shfl_sync(0xffffffffu, upto, at) - row_work(a, w));
      const int task = static_cast<int>(y / length);
      const int from = static_cast<int>(y - static_cast<long long>(task) * length);
      const int to = static_cast<int>(min(static_cast<long long>(length), from + (x_end - x)));
      t.hk = task / w.q_tiles;
      t.qt = task - t.hk * w.q_tiles;
      t.tile0 = max(0, from - kTaskCost);
      t.n = max(0, to - kTaskCost) - t.tile0;
      x += to - from;
      // the CTA whose share holds the task's last tile
      t.last_cta = static_cast<int>(min(((x + (length - to)) * n_ctas - 1) / line, n_ctas - 1));
    } while (t.n == 0);
    t.from_start = t.tile0 == 0;
    t.to_end = t.tile0 + t.n == w.tiles;
    const int G = a.heads / a.kv_heads;
    t.low = w.low;
    t.begin = w.begin;
    t.q_tiles = w.q_tiles;
    t.rows = min(R, w.count * G - t.qt * R);
    t.pos_low = w.pos0 + t.qt * R / G;
    t.pos_high = w.pos0 + (t.qt * R + t.rows - 1) / G;
    t.stop = min(min(max(w.len, 0), a.max_pages * a.page_tokens), t.pos_high + 1);
    t.start = a.window ? static_cast<int>(max(static_cast<long long>(w.low), static_cast<long long>(t.pos_low) + 1 - a.window)) : 0;
    return true;
  }
};

// ------------------------------------------------------------------ the kernel
// kHalves: boxes of 16 keys, so that a score warp's two halves have a scale of V each.  kCapped: scores have a soft cap.
// Kernels of their own, for the loops' instructions: with both in every kernel windowed ticks took 162 us instead of
// 149, answers 235 instead of 215 (in graphs).
template <typename T, int D, int R, bool kHalves, bool kCapped>
__global__ void __launch_bounds__(kThreads, 1) attend_kernel(const AttendArgs a, const __grid_constant__ CUtensorMap k_map,
                                                             const __grid_constant__ CUtensorMap v_map) {
  using S = Shape<D, R>;
  extern __shared__ unsigned char attend_raw[];
  // 1024-byte aligned (an offset, not a cast of the address: the accesses stay shared-memory ones)
  unsigned char* smem = attend_raw + ((1024 - (smem_u32(attend_raw) & 1023)) & 1023);
  unsigned char* ring = smem;                                  // [unit][half][128 keys][kRow]
  unsigned char* q_digits = ring + S::kUnits * S::kSide;       // [buffer][half][digit * R + query][kRow]
  unsigned char* p_digits = q_digits + 2 * S::kQBytes;         // [buffer][digit * R + query][128 keys]
  __shared__ uint64_t full[S::kUnits], empty[S::kUnits], o_full[2], o_empty[2];
  __shared__ uint64_t s_full[S::kBuffers], s_empty[S::kBuffers], p_full[S::kBuffers], p_empty[S::kBuffers];
  __shared__ uint64_t q_full[2], q_empty[2], tops[kScorers], l_full, l_empty;
  __shared__ uint64_t task_full[kTasks], task_empty[kTasks];
  __shared__ Task tasks[kTasks];
  __shared__ uint32_t tmem_slot;
  __shared__ long long warp_total[kThreads / 32], line_length;
  // the prefix sums, which only the loading warp reads, and before it announces a task: p comes after that
  static_assert((kThreads + 1) * sizeof(long long) <= S::kBuffers * S::kPBytes, "room");
  long long* pre = reinterpret_cast<long long*>(p_digits);
  // by box: the scales of K, those of V over the tile's unit (a power of two; kept over kFixed); bits of the boxes
  // that are there, and from bit 8 on of those whose scale of V is not finite
  __shared__ float g_ks[kInfo][kBoxes], g_vs[kInfo][kBoxes], g_unit[kInfo];
  __shared__ unsigned g_there[kInfo];
  __shared__ __align__(16) float fac_s[2][R];    // a query: its factor to log2 scores, and the keys that it sees
  __shared__ int last_s[2][R], first_s[2][R];
  __shared__ __align__(16) float2 tops_s[kScorers][2][4][kQueries];  // a turn's largest scores by warp, and p * sv over theirs
  __shared__ __align__(16) float top_s[4 * kScorers][kQueries], beta_s[4 * kScorers][kQueries];
  __shared__ __align__(16) float factor_s[4 * kScorers][kQueries], up_s[4 * kScorers][kQueries];
  __shared__ float mx_ring[kRing][R], down_ring[kRing][R];  // a tile's largest scores, and 1 / c
  __shared__ __align__(16) float out_f[4][R];
  __shared__ float l_part[4 * kScorers][kQueries], m_ref[kScorers][kQueries];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = a.heads / a.kv_heads, P = a.page_tokens;

  // ---- set-up, and this CTA's share of the line of tiles
  if (warp == 1) {
    tmem_alloc(&tmem_slot, S::kAlloc);
    tmem_relinquish();
  }
  if (tid == 0) {
    for (int s = 0; s < S::kUnits; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < S::kBuffers; ++b) {
      mbar_init(&s_full[b], 2);  // the MMAs, and the thread that saw the tile's scales
      mbar_init(&s_empty[b], 4 * S::kTurns);
      mbar_init(&p_full[b], 4 * S::kTurns);
      mbar_init(&p_empty[b], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&o_full[b], 2);  // the MMAs, and the thread that saw the tile's largest scores
      mbar_init(&o_empty[b], 4);
      mbar_init(&q_full[b], 1);
      mbar_init(&q_empty[b], 1 + 4 * kScorers);
    }
    for (int b = 0; b < kScorers; ++b) mbar_init(&tops[b], 4);
    for (int b = 0; b < kTasks; ++b) {
      mbar_init(&task_full[b], 1);
      mbar_init(&task_empty[b], 3 + 4 * kScorers + 4);
    }
    mbar_init(&l_full, 4 * kScorers);
    mbar_init(&l_empty, 4);
    fence_barrier_init();
    a.cuts[blockIdx.x] = make_int4(-1, 0, 0, 0);
    tma_prefetch_desc(&k_map);
    tma_prefetch_desc(&v_map);
  }
  const int first_token = min(max(a.cu_tokens[0], 0), a.n_tokens);
  const int last_token = min(max(a.cu_tokens[a.n_rows], 0), a.n_tokens);
  const int each = (a.n_rows + kThreads - 1) / kThreads;
  long long mine = 0;
#pragma unroll 2
  for (int r = tid * each; r < min(a.n_rows, (tid + 1) * each); ++r) {
    const Row w = row_of<R>(a, r);
    mine += row_work(a, w);
    // keys past the row's table are not seen: said once
    if (blockIdx.x == 0 && w.count > 0 && w.len > a.max_pages * P && a.status) atomicOr(a.status, static_cast<int>(LB_DEV_BAD_PAGE));
  }
  long long sum = warp_prefix(mine);
  if (lane == 31) warp_total[warp] = sum;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
#pragma unroll 1
  for (int w = 0; w < warp; ++w) sum += warp_total[w];
  pre[tid + 1] = sum;
  if (tid == 0) pre[0] = 0;
  if (tid == kThreads - 1) line_length = sum;
  // tokens of no row
  if (first_token != 0 || last_token != a.n_tokens) {
    const long long pieces = static_cast<long long>(a.heads) * D / 8;
    for (long long i = static_cast<long long>(blockIdx.x) * kThreads + tid; i < a.n_tokens * pieces;
         i += static_cast<long long>(gridDim.x) * kThreads) {
      const long long tok = i / pieces;
      if (tok >= first_token && tok < last_token) continue;
      reinterpret_cast<int4*>(a.out)[i] = make_int4(0, 0, 0, 0);
      if (a.lse && i % (D / 8) == 0) a.lse[i / (D / 8)] = -INFINITY;
    }
  }
  __syncthreads();
  const uint32_t tmem = tmem_slot;
  const uint32_t tmem_o = tmem + S::kBuffers * S::kS;
  const long long W = line_length;
  const long long n_ctas = min(static_cast<long long>(gridDim.x), W);
  const long long b = blockIdx.x;
  bool ok = b < n_ctas;
  // The next task, for the warps that do not load: false when there is none, or the wait ran out.
  int task = 0;
  const auto next = [&]() {
    ok = wait_warp(&task_full[task % kTasks], (task / kTasks) & 1);
    return ok && tasks[task % kTasks].n > 0;
  };
  const auto done = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(&task_empty[task % kTasks]);
    ++task;
  };

  if (warp == 0) {
    // ---------------------------------------------------------------- loads
    int i = 0, last = 0;  // tiles so far; tile i has the units 2 i (K) and 2 i + 1 (V); units issued
    int s = 0;  // the next unit, and the phase of the ring's turn before
    uint32_t turn = 1;
    const uint64_t once = l2_policy_evict_first();
    uint64_t again;
    asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(again));
    const int nb = kTile / a.box;                            // boxes of a tile
    const int own_tile = lane / nb, k = lane - own_tile * nb;  // a lane's box among those of a batch of tiles
    const int batch = nb == 2 ? 8 : 32 / nb;
    Walk<R> walk;
    if (ok) walk.begin(a, pre, each, W * b / n_ctas, W * (b + 1) / n_ctas);
    int known = 0;  // tasks made known
    // Three batches are in hand, so that no load is waited for: the tables of the third, the scales of the second
    // and the boxes of the first are under way together.  n 0: there are no more tasks.
    struct Batch {
      int task, tile, n;
    };
    const auto following = [&](const Batch& c) {
      Batch d{c.task, c.tile + batch, c.n};
      if (c.task >= 0 && (c.n == 0 || d.tile < c.n)) return d;
      d.task = c.task + 1;
      d.tile = 0;
      if (d.task == known) {
        Task t;
        walk.next(a, W, n_ctas, t);
        if (known >= kTasks) ok = wait_warp(&task_empty[known % kTasks], (known / kTasks - 1) & 1) && ok;
        if (!ok) t.n = 0;
        if (ok && lane == 0) {
          tasks[known % kTasks] = t;
          mbar_arrive(&task_full[known % kTasks]);
        }
        __syncwarp();
        ++known;
        d.n = t.n;
      }
      return d;
    };
    const auto box_key = [&](const Batch& c) {  // the first key of this lane's box, -1 where it has none
      const Task& t = tasks[c.task % kTasks];
      if (own_tile >= batch || c.tile + own_tile >= c.n) return -1;
      const int key = t.low + (t.tile0 + c.tile) * kTile + lane * a.box;
      return key < t.stop && key + a.box > t.start ? key : -1;
    };
    const auto page_at = [&](const Batch& c) {
      const int key = box_key(c);
      if (key < 0) return -1;
      const int page = a.row_tables[static_cast<long long>(tasks[c.task % kTasks].row) * a.max_pages + key / P];
      if (page >= 0 && page < a.n_pages) return page;
      if (a.status) atomicOr(a.status, static_cast<int>(LB_DEV_BAD_PAGE));
      return -1;
    };
    struct Where {
      int at;  // row of the cache, -1: not there
      float ks, vs;
    };
    const auto scales_at = [&](const Batch& c, int page) {
      Where w{-1, 0.0f, 0.0f};
      if (page >= 0) {
        const int ph = page * a.kv_heads + tasks[c.task % kTasks].hk;
        w.at = ph * P + box_key(c) % P;
        w.ks = a.k_scale[ph];
        w.vs = a.v_scale[ph];
      }
      return w;
    };
    Batch b0{-1, 0, 0}, b1;
    int page1 = -1;
    Where w0{-1, 0.0f, 0.0f};
    if (ok) {
      b0 = following(b0);
      const int page0 = page_at(b0);
      b1 = following(b0);
      page1 = page_at(b1);
      w0 = scales_at(b0, page0);
    }
#pragma unroll 1
    while (ok && b0.n > 0) {
      const Batch b2 = following(b1);
      const int page2 = page_at(b2);
      const Where w1 = scales_at(b1, page1);
      const int tiles = min(batch, b0.n - b0.tile);
      const uint64_t policy = tasks[b0.task % kTasks].q_tiles > 1 ? again : once;  // other query tiles read the same keys
      const unsigned there = __ballot_sync(0xffffffffu, w0.at >= 0);
      // the tile's unit: its largest finite scale of V, less the fraction (its inverse is a normal number)
      int v_unit = __float_as_int(w0.vs) & 0x7f800000;
      if (v_unit == 0x7f800000) v_unit = 0;
#pragma unroll 1
      for (int o = 1; o < nb; o <<= 1) v_unit = max(v_unit, __shfl_xor_sync(0xffffffffu, v_unit, o));
      v_unit = min(max(v_unit, 0x00800000), 0x7e800000);
      float v_own = w0.vs * __int_as_float(0x7f000000 - v_unit);
      const bool v_bad = !(fabsf(v_own) < INFINITY);
      if (v_bad) v_own = 0.0f;  // (a key that does not count has digits of 0 all the same)
      const unsigned bad = __ballot_sync(0xffffffffu, v_bad), all = (1u << nb) - 1u;
      const unsigned boxes = own_tile < batch ? (there >> (own_tile * nb) & all) | (bad >> (own_tile * nb) & all) << 8 : 0u;
#pragma unroll 1
      for (int j = 0; ok && j < tiles; ++j, ++i) {
        const int info = i % kInfo;
        const bool own = own_tile == j;
        const unsigned mask = (there >> (j * nb)) & ((1u << nb) - 1u);
#pragma unroll
        for (int side = 0; side < 2; ++side) {
          if (ok && last >= S::kUnits) ok = wait_warp(&empty[s], turn);
          if (!ok) break;
          if (side == 0 && own) {
            g_ks[info][k] = w0.ks;
            g_vs[info][k] = v_own;
            if (k == 0) {
              g_there[info] = boxes;
              g_unit[info] = __int_as_float(v_unit) * (1.0f / kFixed);
            }
          }
          __syncwarp();
          if (lane == 0) {
            mbar_arrive_expect_tx(&full[s], __popc(mask) * (a.box * D));
          }
          __syncwarp();
          if (own && w0.at >= 0) {
            unsigned char* d = ring + s * S::kSide + k * a.box * S::kRow;
#pragma unroll
            for (int h = 0; h < S::kHalves; ++h)
              tma_load_2d(d + h * S::kHalfBytes, side ? &v_map : &k_map, &full[s], h * 128, w0.at, policy);
          }
          ++last;
          if (++s == S::kUnits) {
            s = 0;
            turn ^= 1;
          }
        }
      }
      b0 = b1;
      w0 = w1;
      b1 = b2;
      page1 = page2;
    }
    // loads that nobody waited for (after a wait that ran out) end before the CTA does
    if (!ok && lane == 0)
#pragma unroll 1
      for (int u = max(0, last - S::kUnits); u < last; ++u) wait_one(&full[u % S::kUnits], (u / S::kUnits) & 1);
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMAs of the scores: one thread
    constexpr uint32_t id = idesc_i8(128, S::kN1, false);
    int i = 0, s = 0;  // s: the tile's unit
    uint32_t turn = 0;
    while (ok && next()) {
      const int n_tiles = tasks[task % kTasks].n;
      if (lane == 0) {
        const uint32_t q = smem_u32(q_digits + (task & 1) * S::kQBytes);
        ok = wait_one(&q_full[task & 1], (task >> 1) & 1);
#pragma unroll 1
        for (int tile = 0; ok && tile < n_tiles; ++tile, ++i) {
          const int buf = i % S::kBuffers;
          // (scores that are there say that their digits' buffer is free as well)
          if (i >= S::kBuffers)
            ok = wait_one(&s_empty[buf], (i / S::kBuffers - 1) & 1) &&
                 wait_one(&p_empty[buf], (i / S::kBuffers - 1) & 1);
          if (!ok || !(ok = wait_one(&full[s], turn))) break;
          tc_fence_after();
          uint64_t k = smem_desc<S::kRow>(smem_u32(ring + s * S::kSide)), qd = smem_desc<S::kRow>(q);
#pragma unroll 1
          for (int n = 0; n < D / 32; ++n) {  // 32 columns a step; every 128 the next half
            umma_i8(tmem + buf * S::kS, k, qd, id, n > 0);
            const bool next = S::kHalves > 1 && n % 4 == 3;
            k += (next ? S::kHalfBytes - 96 : 32) >> 4;
            qd += (next ? S::kN1 * S::kRow - 96 : 32) >> 4;
          }
          umma_commit(&s_full[buf]);
          mbar_arrive(&s_full[buf]);
          umma_commit(&empty[s]);
          if ((s += 2) >= S::kUnits) {
            s -= S::kUnits;
            turn ^= 1;
          }
        }
        if (ok) umma_commit(&q_empty[task & 1]);
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      done();
    }
  } else if (warp == 2) {
    // ---------------------------------------------------------------- MMAs of the outputs: one thread
    constexpr uint32_t id = idesc_i8(128, S::kN2, true);
    int i = 0, s = 1;
    uint32_t turn = 0;
    while (ok && next()) {
      const int n_tiles = tasks[task % kTasks].n;
      if (lane == 0) {
#pragma unroll 1
        for (int tile = 0; ok && tile < n_tiles; ++tile, ++i) {
          const int buf = i % S::kBuffers, ob = i & 1;
          if (i >= 2) ok = wait_one(&o_empty[ob], ((i >> 1) - 1) & 1);
          if (ok) ok = wait_one(&full[s], turn);
          if (!ok || !(ok = wait_one(&p_full[buf], (i / S::kBuffers) & 1))) break;
          tc_fence_after();
          uint64_t v = smem_desc<S::kRow>(smem_u32(ring + s * S::kSide));
          const uint64_t p = smem_desc<128>(smem_u32(p_digits + buf * S::kPBytes));
#pragma unroll 1
          for (int n = 0; n < 4 * S::kHalves; ++n, v += 32 * S::kRow >> 4)  // 32 keys a step; the halves are neighbours
            umma_i8(tmem_o + (ob * S::kHalves + n / 4) * S::kN2, v, p + (n % 4) * 2, id, n % 4 > 0);
          umma_commit(&o_full[ob]);
          mbar_arrive(&o_full[ob]);
          umma_commit(&p_empty[buf]);
          umma_commit(&empty[s]);
          if ((s += 2) >= S::kUnits) {
            s -= S::kUnits;
            turn ^= 1;
          }
        }
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      done();
    }
  } else if (warp == 3) {
    // ---------------------------------------------------------------- q -> digits, a task ahead
    constexpr int kE = D / 32;  // columns a lane
    struct alignas(16) Columns {
      uint16_t v[kE];
    };
    while (ok && next()) {
      const Task t = tasks[task % kTasks];
      const int buf = task & 1;
      if (task >= 2) ok = wait_warp(&q_empty[buf], ((task >> 1) - 1) & 1);
      if (!ok) break;
      unsigned char* digits = q_digits + buf * S::kQBytes + (lane * kE / 128) * (S::kN1 * S::kRow);
      const int col = lane * kE % 128;
      int tok = t.qt * R / G, head = t.qt * R - tok * G;  // of the next row to load
      const auto load = [&](int q) {
        Columns c{};
        if (q < t.rows) {
          const uint16_t* src = static_cast<const uint16_t*>(a.q) + (t.begin + tok) * a.q_token_stride +
                                (t.hk * G + head) * a.q_head_stride + lane * kE;
          if (!a.q_vec) {
#pragma unroll
            for (int e = 0; e < kE; ++e) c.v[e] = src[e];
          } else if constexpr (kE == 8) {
            *reinterpret_cast<uint4*>(c.v) = *reinterpret_cast<const uint4*>(src);
          } else if constexpr (kE == 4) {
            *reinterpret_cast<uint2*>(c.v) = *reinterpret_cast<const uint2*>(src);
          } else {
            *reinterpret_cast<uint32_t*>(c.v) = *reinterpret_cast<const uint32_t*>(src);
          }
        }
        if (++head == G) {
          head = 0;
          ++tok;
        }
        return c;
      };
      int pos = t.pos_low, left = G - head;  // of the row in hand, and rows of its token still to come
      Columns r0 = load(0), r1 = load(1), r2 = load(2);  // three rows' loads are under way
#pragma unroll 1
      for (int qi = 0; qi < R; ++qi) {
        const Columns raw = r0;
        r0 = r1;
        r1 = r2;
        r2 = load(qi + 3);
        uint32_t size = 0;  // absolute values by their bits: a NaN is above all
#pragma unroll
        for (int e = 0; e < kE; ++e) size = max(size, __float_as_uint(to_f<T>(raw.v[e])) & 0x7fffffffu);
        const float top = __uint_as_float(__reduce_max_sync(0xffffffffu, size));
        const bool fine = top < INFINITY;
        // 2^ex brings the maximum to [2^29, 2^30); in two factors, each inside the floating range
        const int ex = fine && top > 0.0f ? 29 + 127 - max(1, __float_as_int(top) >> 23) : 0;
        const int e1 = ex / 2, e2 = ex - e1;
        const float up1 = copysignf(__int_as_float((127 + e1) << 23), a.scale), up2 = __int_as_float((127 + e2) << 23);
        if (lane == 0) {
          // positive (a negative scale turns the digits over) and not zero, so that masked scores stay at -inf
          const float down = __int_as_float((127 - e1) << 23) * (fabsf(a.scale) * kLog2e) *
                             __int_as_float((127 - e2) << 23);
          fac_s[buf][qi] = !fine ? NAN : down < 0x1p-126f ? 0x1p-126f : down;
          last_s[buf][qi] = min(qi < t.rows ? pos : 0x7fffffff, t.stop - 1);
          first_s[buf][qi] = qi < t.rows && a.window ? pos - a.window + 1 : 0;
        }
        if (--left == 0) {
          left = G;
          ++pos;
        }
        uint32_t w[4][kE / 4 > 0 ? kE / 4 : 1] = {};
#pragma unroll
        for (int e = 0; e < kE; ++e) {
          const int v = fine ? __float2int_rn(to_f<T>(raw.v[e]) * up1 * up2) : 0;
          const uint32_t d = (v + 0x808080) ^ 0x808080;  // its bytes (see the digits of p below)
#pragma unroll
          for (int c = 0; c < 4; ++c) w[c][e / 4] |= ((d >> (24 - 8 * c)) & 0xffu) << (8 * (e & 3));
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          unsigned char* to = digits + swizzled<S::kRow>((c * R + qi) * S::kRow + col);
          if constexpr (kE == 8) *reinterpret_cast<uint2*>(to) = make_uint2(w[c][0], w[c][1]);
          else if constexpr (kE == 4) *reinterpret_cast<uint32_t*>(to) = w[c][0];
          else *reinterpret_cast<uint16_t*>(to) = static_cast<uint16_t>(w[c][0]);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[buf]);
      done();
    }
  } else if (warp < kFirstOutput) {
    // ---------------------------------------------------------------- scores -> digits of p
    // A turn is 8 queries of a tile: with 8 query rows the two warpgroups take a tile each in turn, with
    // 16 half of a tile's queries each.
    const int side = (warp - kFirstScorer) >> 2, wq = warp & 3, key_row = wq * 32 + lane;
    const uint32_t lane_at = static_cast<uint32_t>(wq * 32) << 16;
    constexpr int C = kQueries;
    const int c0 = side % S::kTurns * C;  // the warpgroup's first query
    float* own_top = top_s[warp - kFirstScorer];
    float* own_beta = beta_s[warp - kFirstScorer];
    float* own_fac = factor_s[warp - kFirstScorer];
    float* own_up = up_s[warp - kFirstScorer];
    const unsigned all_boxes = (1u << (kTile >> a.box_log)) - 1u;
    const float cap = fminf(a.softcap * kLog2e, 0x1p127f), cap_inv = fminf(kLn2 / a.softcap, 0x1p127f);  // of log2 scores
    int i = 0, turn = 0;
    while (ok && next()) {
      const Task& t = tasks[task % kTasks];
      const int n_tiles = t.n, first_key = t.low + t.tile0 * kTile;
      const int plain_stop = min(t.pos_low + 1, t.stop), plain_start = a.window ? t.pos_high - a.window + 1 : 0;  // keys all queries see
      const int qb = task & 1;
      ok = wait_warp(&q_full[qb], (task >> 1) & 1);  // what is known of the queries
      float l[C];
#pragma unroll
      for (int q = 0; q < C; ++q) l[q] = 0.0f;
      float ref = -INFINITY;  // lane q: the reference maximum of query q (the four warps keep the same)
      // (a capped score has its factor already)
      const float fac = kCapped ? 1.0f : fac_s[qb][c0 + lane % C];
      const float fac_up = fac * (1.0f + 0x1p-22f), fac_down = fac * (1.0f - 0x1p-22f);
      if (lane < C) own_fac[lane] = fac;
      __syncwarp();
#pragma unroll 1
      for (int tile = 0; ok && tile < n_tiles; ++tile, ++i) {
        if (i % S::kEvery != side / S::kTurns) continue;
        const int buf = i % S::kBuffers, phase = (i / S::kBuffers) & 1, info = i % kInfo;
        ok = wait_warp(&s_full[buf], phase);
        if (!ok) break;
        tc_fence_after();
        const int grp = key_row >> a.box_log;
        const float ks = g_ks[info][grp], vs = g_vs[info][grp], unit = g_unit[info];
        const float v0 = fabsf(g_vs[info][wq * 32 >> a.box_log]), v1 = fabsf(g_vs[info][(wq * 32 + 16) >> a.box_log]);  // of the warp's halves
        const unsigned boxes = g_there[info];
        const bool there = (boxes >> grp) & 1u;
        const int key0 = first_key + tile * kTile, key = key0 + key_row;
        const bool masked = key0 + kTile > plain_stop || key0 < plain_start || boxes != all_boxes;
        unsigned char* p = p_digits + buf * S::kPBytes;
        Scores x;
        {
          int d3[C], d2[C], d1[C], d0[C];
          const uint32_t at = tmem + buf * S::kS + lane_at + c0;
          tmem_ld4(at, at + R, at + 2 * R, at + 3 * R, d3, d2, d1, d0);
#pragma unroll
          for (int c = 0; c < C; ++c)  // (a digit's sum is below 2^22)
            x.v[c] = fmaf(__int2float_rn(d3[c] * 256 + d2[c]), 65536.0f, __int2float_rn(d1[c] * 256 + d0[c])) * ks;
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_empty[buf]);
        if constexpr (kCapped) {
#pragma unroll
          for (int q = 0; q < C; ++q) x.v[q] *= fac_s[qb][c0 + q];
          x = capped(x, cap, cap_inv);
        }
        if (masked) {
#pragma unroll
          for (int q = 0; q < C; ++q)
            if (!there || key > last_s[qb][c0 + q] || key < first_s[qb][c0 + q]) x.v[q] = -INFINITY;
            else if (boxes >> 8 >> grp & 1u) x.v[q] = NAN;  // a scale of V that is no number: so is the query's output
        }
        // the turn's largest score of each query, still without its (positive) factor: warp, then the four warps
        float mx = -INFINITY, my = -INFINITY;
        if constexpr (kHalves) {
#pragma unroll
          for (int q = 0; q < C; ++q) {
            const float m0 = warp_top(lane < 16 ? x.v[q] : -INFINITY), m1 = warp_top(lane < 16 ? -INFINITY : x.v[q]);
            if (lane == q) {
              mx = m0;
              my = m1;
            }
          }
        } else {
#pragma unroll
          for (int q = 0; q < C; ++q) {
            const float m = warp_top(x.v[q]);
            if (lane == q) mx = m;
          }
        }
        if (lane < C) {
          // rounded up, so that no exponential below passes 1 however large the scores are (-inf, no key, also stays
          // where the factor is NaN)
          mx = mx == -INFINITY ? mx : fmaxf(mx * fac_up, mx * fac_down);
          float pv = v0;
          if constexpr (kHalves) {
            my = my == -INFINITY ? my : fmaxf(my * fac_up, my * fac_down);
            const float most = max_nan(mx, my);
            pv = fmaxf(exp2_fast(mx - most) * v0, exp2_fast(my - most) * v1);
            mx = most;
          }
          tops_s[side][turn & 1][wq][lane] = make_float2(mx, pv);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&tops[side]);
        ok = wait_warp(&tops[side], turn & 1);
        if (!ok) break;
        float alpha = 1.0f;
        if (lane < C) {
          const float2* tw = &tops_s[side][turn & 1][0][lane];
          const float2 t0 = tw[0], t1 = tw[C], t2 = tw[2 * C], t3 = tw[3 * C];
          mx = max_nan(max_nan(t0.x, t1.x), max_nan(t2.x, t3.x));
          // the largest p * sv (a maximum drops the NaN of no key at all, and a NaN score is a NaN in mx)
          const float pv = fmaxf(fmaxf(exp2_fast(t0.x - mx) * t0.y, exp2_fast(t1.x - mx) * t1.y),
                                 fmaxf(exp2_fast(t2.x - mx) * t2.y, exp2_fast(t3.x - mx) * t3.y));
          if (ref == -INFINITY) {
            ref = mx;
          } else if (mx > ref + kSlack) {
            alpha = exp2_fast(ref - mx);
            ref = mx;
          }
          own_top[lane] = mx == -INFINITY ? 0.0f : mx;
          own_beta[lane] = mx == -INFINITY ? 0.0f : exp2_fast(mx - ref);
          // Over the unit, so powers of two are exact: pages that the query does not see change no bit.  Not below
          // 2^-100 of it, where c * sv would not stay finite.
          const float top_pv = fmaxf(pv, 0x1p-100f);
          own_up[lane] = rcp_fast(top_pv) * kFixed;
          if (wq == 0) {
            mx_ring[i % kRing][c0 + lane] = mx;
            down_ring[i % kRing][c0 + lane] = top_pv * unit;
          }
        }
        const bool moved = __any_sync(0xffffffffu, alpha != 1.0f);
        __syncwarp();
        if (moved) {
#pragma unroll
          for (int q = 0; q < C; ++q) l[q] *= __shfl_sync(0xffffffffu, alpha, q);
        }
#pragma unroll
        for (int q = 0; q < C; ++q) {
          const float e = exp2_fast(fmaf(x.v[q], own_fac[q], -own_top[q]));
          l[q] = fmaf(e, own_beta[q], l[q]);
          // v = rint(e * sv * c) by a sum with 1.5 * 2^23.  With 128 added to each of the two lower
          // digits' places, the bytes of v are its signed digits, the lower two with the sign bit turned over.
          const uint32_t v = __float_as_uint(fmaf(e, vs * own_up[q], 12582912.0f)) - 0x4B400000u;
          const uint32_t digits = (v + 0x8080u) ^ 0x8080u;
          unsigned char* to = p + swizzled<128>(q * kTile + key_row) + c0 * kTile;  // (c0 is a multiple of 8 rows)
          to[0] = static_cast<unsigned char>(digits >> 16);
          to[R * kTile] = static_cast<unsigned char>(digits >> 8);
          to[2 * R * kTile] = static_cast<unsigned char>(digits);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[buf]);
        ++turn;
      }
      // ---- the task's sums
      if (ok && task > 0) ok = wait_warp(&l_empty, (task - 1) & 1);
      if (!ok) break;
      // eight sums over the warp at once: a half of them, by a bit of the lane, goes on at each step
#pragma unroll
      for (int o = 16; o >= 4; o >>= 1) {
        const bool high = lane & o;
#pragma unroll
        for (int q = 0; q < o / 4; ++q) {
          const float give = high ? l[q] : l[q + o / 4], keep = high ? l[q + o / 4] : l[q];
          l[q] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
      }
      float sum_q = l[0] + __shfl_xor_sync(0xffffffffu, l[0], 2);
      sum_q += __shfl_xor_sync(0xffffffffu, sum_q, 1);
      // a query that saw no key has no sum, though its own values be NaN
      if (__shfl_sync(0xffffffffu, ref, lane / 4) == -INFINITY) sum_q = 0.0f;
      if ((lane & 3) == 0) l_part[warp - kFirstScorer][lane / 4] = sum_q;
      if (wq == 0 && lane < C) m_ref[side][lane] = ref;
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&q_empty[qb]);
        mbar_arrive(&l_full);
      }
      done();
    }
  } else {
    // ---------------------------------------------------------------- outputs
    const int sub = warp & 3, col = sub * 32 + lane;
    const uint32_t lane_at = static_cast<uint32_t>(sub * 32) << 16;
    constexpr int C = kQueries;
    float* factor = out_f[sub];
    int i = 0;
    while (ok && next()) {
      const Task& t = tasks[task % kTasks];
      const int n_tiles = t.n;
      float o[S::kHalves][R];
#pragma unroll
      for (int h = 0; h < S::kHalves; ++h)
#pragma unroll
        for (int q = 0; q < R; ++q) o[h][q] = 0.0f;
      float ref = -INFINITY;  // lane q: the reference maximum of query q
#pragma unroll 1
      for (int tile = 0; ok && tile < n_tiles; ++tile, ++i) {
        const int buf = i & 1;
        ok = wait_warp(&o_full[buf], (i >> 1) & 1);
        if (!ok) break;
        tc_fence_after();
        float alpha = 1.0f;
        if (lane < R) {
          const float mx = mx_ring[i % kRing][lane];
          if (ref == -INFINITY) {
            ref = mx;
          } else if (mx > ref + kSlack) {
            alpha = exp2_fast(ref - mx);
            ref = mx;
          }
          factor[lane] = mx == -INFINITY ? 0.0f : exp2_fast(mx - ref) * down_ring[i % kRing][lane];
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
      if (ok) ok = wait_warp(&l_full, task & 1);
      if (!ok) break;
      // lane q: the query's sum, its inverse, where it goes
      float l = 0.0f;
      int to = 0;  // (the entry refuses more than 2^31 rows)
      if (lane < t.rows) {
#pragma unroll
        for (int k = 0; k < S::kEvery; ++k) {  // the query's warpgroups
          const int w = lane / C + k * S::kTurns, q = lane % C;
          const float part = l_part[4 * w][q] + l_part[4 * w + 1][q] + l_part[4 * w + 2][q] + l_part[4 * w + 3][q];
          if (part != 0.0f) l += part * exp2_fast(m_ref[w][q] - ref);
        }
        const int qr = t.qt * R + lane;
        to = (t.begin + qr / G) * a.heads + t.hk * G + qr % G;
      }
      const int rows = t.rows;
      const bool whole = t.from_start && t.to_end;
      float* part = a.parts + (2 * b + (t.from_start ? 1 : 0)) * S::kPart;
      if (lane < rows && sub == 0) {
        if (!whole) {
          part[R * D + lane] = ref;
          part[R * D + R + lane] = l;
        } else if (a.lse) {
          a.lse[to] = l != 0.0f ? (ref + log2f(l)) * kLn2 : -INFINITY;
        }
      }
      if (whole) {
        const float inv = l != 0.0f ? 1.0f / l : 0.0f;
        uint16_t* out = static_cast<uint16_t*>(a.out) + col;
#pragma unroll
        for (int q = 0; q < R; ++q) {
          const float f = __shfl_sync(0xffffffffu, inv, q);
          uint16_t* d = out + static_cast<long long>(__shfl_sync(0xffffffffu, to, q)) * D;
          if (q < rows && col < D) {
#pragma unroll
            for (int h = 0; h < S::kHalves; ++h) d[h * 128] = to_bits<T>(o[h][q] * f);
          }
        }
      } else if (col < D) {
        float* d = part + col;
#pragma unroll
        for (int q = 0; q < R; ++q) {
          if (q < rows) {
#pragma unroll
            for (int h = 0; h < S::kHalves; ++h) d[q * D + h * 128] = o[h][q];
          }
        }
      }
      if (t.from_start && !t.to_end && sub == 0 && lane == 0) a.cuts[b] = make_int4(t.row, t.hk, t.qt, t.last_cta);
      __syncwarp();
      if (lane == 0) mbar_arrive(&l_empty);
      done();
    }
  }
  if (!ok && b < n_ctas && a.status) atomicOr(a.status, static_cast<int>(kStatusWaitTimeout));
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, S::kAlloc);
  }
}

// Joins the parts of the task that is cut at the end of CTA blockIdx.x: query row
// blockIdx.y.  First the parts' weights, a thread each, then groups of lanes (over columns) over the
// parts, then the groups' sums in order.
template <typename T, int D, int R>
__global__ void __launch_bounds__(512) combine_kernel(const AttendArgs a) {
  using S = Shape<D, R>;
  constexpr int kLanes = D / 4, kParts = 512 / kLanes;
  __shared__ float4 sum_o[kParts][kLanes];
  __shared__ float weight[kSms];
  __shared__ float top_w[8], sum_w[8];
  pdl_wait();
  const int4 cut = a.cuts[blockIdx.x];
  if (cut.x < 0) return;
  const int G = a.heads / a.kv_heads, r = blockIdx.y, qr = cut.z * R + r, tid = threadIdx.x;
  const Row w = row_of<R>(a, cut.x);
  if (qr >= w.count * G) return;
  const int first = blockIdx.x, n = cut.w - first + 1;  // at most kSms parts
  const auto part = [&](int i) { return a.parts + (2ll * (first + i) + (i == 0 ? 1 : 0)) * S::kPart; };
  // a thread a part: its maximum and sum, then its weight
  float m = -INFINITY, l = 0.0f;
  if (tid < n) {
    m = part(tid)[R * D + r];
    l = part(tid)[R * D + R + r];
  }
  float top = warp_max(m);
  if ((tid & 31) == 0 && tid < 256) top_w[tid >> 5] = top;
  __syncthreads();
  top = top_w[0];
#pragma unroll
  for (int k = 1; k < (kSms + 31) / 32; ++k) top = fmaxf(top, top_w[k]);
  const float f = tid < n && !(m == -INFINITY && l == 0.0f) ? exp2_fast(m - top) : 0.0f;
  if (tid < n) weight[tid] = f;
  l = warp_sum(f != 0.0f ? l * f : 0.0f);
  if ((tid & 31) == 0 && tid < 256) sum_w[tid >> 5] = l;
  __syncthreads();
  l = 0.0f;
#pragma unroll
  for (int k = 0; k < (kSms + 31) / 32; ++k) l += sum_w[k];
  const int lane = tid % kLanes, grp = tid / kLanes;
  float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int i = grp; i < n; i += kParts) {
    const float4 z = *reinterpret_cast<const float4*>(part(i) + r * D + lane * 4);
    const float c = weight[i];
    if (c != 0.0f) y = make_float4(fmaf(z.x, c, y.x), fmaf(z.y, c, y.y), fmaf(z.z, c, y.z), fmaf(z.w, c, y.w));
  }
  sum_o[grp][lane] = y;
  __syncthreads();
  if (grp != 0) return;
  y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
  for (int k = 0; k < kParts; ++k) {
    const float4 z = sum_o[k][lane];
    y = make_float4(y.x + z.x, y.y + z.y, y.z + z.z, y.w + z.w);
  }
  const float inv = l != 0.0f ? 1.0f / l : 0.0f;
  const long long to = static_cast<long long>(w.begin + qr / G) * a.heads + cut.y * G + qr % G;
  uint16_t* dst = static_cast<uint16_t*>(a.out) + to * D + lane * 4;
  *reinterpret_cast<uint2*>(dst) =
      make_uint2(to_bits<T>(y.x * inv) | static_cast<uint32_t>(to_bits<T>(y.y * inv)) << 16,
                 to_bits<T>(y.z * inv) | static_cast<uint32_t>(to_bits<T>(y.w * inv)) << 16);
  if (a.lse && lane == 0) a.lse[to] = l != 0.0f ? (top + log2f(l)) * kLn2 : -INFINITY;
}

// Query rows of a task: as few as hold the rows of most requests, so that the tensor memory's columns
// and the threads' work are not spent on padding; at most what two score warpgroups' turns hold.
int rows_of(int max_new, int group) { return static_cast<long long>(max_new) * group <= 8 ? 8 : 16; }

template <typename T, int D, int R, bool kHalves, bool kCapped>
cudaError_t launch(const AttendArgs& a, const CUtensorMap& k_map, const CUtensorMap& v_map, cudaStream_t s) {
  using S = Shape<D, R>;
  const auto kernel = attend_kernel<T, D, R, kHalves, kCapped>;
  static std::atomic<unsigned long long> done{0};
  cudaError_t e = ensure_smem(done, reinterpret_cast<const void*>(kernel), S::kSmem);
  if (e != cudaSuccess) return e;
  kernel<<<kSms, kThreads, S::kSmem, s>>>(a, k_map, v_map);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  return launch_kernel(true, combine_kernel<T, D, R>, dim3(kSms, R), dim3(512), 0, s, a);
}
template <typename T, int D, int R, bool kHalves>
cudaError_t launch(const AttendArgs& a, const CUtensorMap& k_map, const CUtensorMap& v_map, cudaStream_t s) {
  if (a.softcap > 0.0f) return launch<T, D, R, kHalves, true>(a, k_map, v_map, s);
  return launch<T, D, R, kHalves, false>(a, k_map, v_map, s);
}
template <typename T, int D, int R>
cudaError_t launch(const AttendArgs& a, const CUtensorMap& k_map, const CUtensorMap& v_map, cudaStream_t s) {
  return a.box == 16 ? launch<T, D, R, true>(a, k_map, v_map, s) : launch<T, D, R, false>(a, k_map, v_map, s);
}
template <typename T, int D>
cudaError_t launch(const AttendArgs& a, int rows, const CUtensorMap& k_map, const CUtensorMap& v_map, cudaStream_t s) {
  if (rows == 8) return launch<T, D, 8>(a, k_map, v_map, s);
  return launch<T, D, 16>(a, k_map, v_map, s);
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
      max_pages < 1 || max_new < 1 || window < 0 || !(softcap >= 0.0f && softcap < INFINITY))
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
               page_tokens, max_pages, row_tables, kv_len, cu_tokens, scale, softcap, window, q_vec, box, 31 - __builtin_clz(box), out, lse, status,
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
