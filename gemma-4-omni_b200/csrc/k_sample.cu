// The next token from the logits x of a row: temperature T, top-k, top-p and min-p, with a given random number u.
//
//   m_i = rint(2^45 exp((x_i - max x) / T))          a token's mass, a whole number
//   top-k: the first k by (x down, index up)
//   top-p: of those, each whose predecessors' masses sum to less than ceil(p * their total)
//   min-p: m_i >= ceil(p_min * 2^45)
//   token: the first by index with (sum of the kept masses up to it) > floor(u * their total)
//
// Masses are whole numbers, so that sums of them are the same in any order: no result depends on
// which thread comes first.  They are computed in 64-bit floating point (to some 2^-49): a row has 10^5 borders between tokens,
// and u falls between two roundings of one of them the more rarely the finer they are.  2^45 * 2^18 tokens stay below 2^63.
//
// The logits are read once.  A cluster of CTAs takes a row, each CTA holds its part of it in shared
// memory, each warp a part of that.  Nothing is sorted but the few hundred tokens around a cut: counts, and for top-p masses, by
// bins of the distance to the maximum (shared-memory atomics on whole numbers; a mass in three limbs of 16 bits), added up
// over the cluster, say in which bin a cut lies.  If at most 512 tokens lie in and above it, as with the usual settings, one CTA
// gathers and sorts them and finishes alone.  Otherwise the bin's tokens are sorted, or divided again where they are many; one
// value that they all have is cut by index.  What a cut leaves, each warp moves together in place, in the order of the indexes,
// so that every later pass goes over that alone: for top-p the sum of all masses and a look at a few distances come first, and
// only what lies above the distance behind the cut is divided into bins.
//
// Measured (calls in one graph, logits out of L2): one row of 131072 with top-k 64 and top-p 13.1 us, a chain of loads, four
// barriers of the cluster and 128 tokens that are ranked; 250 rows of 131072 in 32 bits by a share of 0.9 (9 thousand tokens kept a
// row) 260 us, 0.5 TB/s, with top-k 50 too 122, unfiltered 102, greedy 58 (2.3 TB/s); 1000 rows of 32003 by min-p 68 us.  Beyond
// 131072 tokens a CTA holds twice as many and an SM one CTA instead of two: 125 rows of 262144 in bf16 by that share 401 us (250 of
// 131072: 275), one row as above 17.2.  Bound by instructions and barriers: some 45 instructions a token for its mass and the sums
// (11 of them in 64 bits), as many again for the loads, the moves and the bins, and 16 warps that wait for one another. Sorting or
// ranking fewer tokens in one CTA holds up the other seven of a row: 512 sorted took 12 thousand cycles, 128 ranked take 3.
#include <cfloat>
#include <cooperative_groups.h>

#include "../../include/listener_b200.h"
#include "common.cuh"

namespace cg = cooperative_groups;

namespace lb {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBins = kThreads;
constexpr int kGroups = 8, kGroupBins = kBins / kGroups;  // of bins
constexpr int kList = kThreads;       // tokens that are sorted
constexpr int kFew = 128;             // of them, that are ranked instead (a sort takes as long as some 100)
constexpr int kMaxCluster = 8;
constexpr int kMaxVocab = 1 << 18;
constexpr int kMaxPart = kMaxVocab / kMaxCluster;  // tokens of a CTA
constexpr int kTop = 45;              // log2 of the largest mass
constexpr int kPowers = 128;
constexpr float kMaxHeat = 1e30f;     // so that 47 octaves stay inside the 32-bit numbers
constexpr unsigned long long kNone = ~0ull;
// Distances to the maximum, in units of T, between which a share's cut is looked for first.  Where it lies nearer or farther the bins
// start at the maximum or reach 32 units down; the result is the same, more tokens are put into bins.
constexpr int kZones = 4;
__host__ __device__ constexpr float zone_end(int z) { return z == 0 ? 4.0f : z == 1 ? 8.0f : z == 2 ? 11.0f : 14.0f; }

typedef unsigned long long u64;

struct SampleArgs {
  const void* logits;
  long long row_stride;
  const void* uniform;
  const float *temperature, *top_p, *min_p;  // by row, or null: the values below
  const int* top_k;
  float temperature1, top_p1, min_p1;
  int top_k1, rows, vocab, part, uniform64;
  long long* tokens;
  float* logprobs;
};

struct Result {  // of one division into bins
  u64 above;         // weight before the bin
  int bin, count, before;  // tokens in it and before it
};

struct Zone {  // of distances that hold a share's cut
  u64 limit;
  float lo, hi, top, low;  // top: the logits above are nearer than lo; low: those from it down are farther than hi
};

struct alignas(16) Shared {
  double power[kPowers];        // 2^(j / kPowers)
  union {
    alignas(16) unsigned hist[4][kBins];    // counts; masses in limbs of 16 bits
    u64 mass[kList];            // while tokens are sorted
  };
  u64 list[kList];
  u64 scan[kWarps], scan2[kWarps];
  unsigned zone[kWarps][kZones];
  // written by the other CTAs
  float top[kMaxCluster];
  u64 group_mass[2][kGroups][kMaxCluster];
  unsigned group_count[2][kGroups][kMaxCluster];
  Result result;
  Zone chosen;
  unsigned warp_count[kWarps];
  unsigned low[kMaxCluster], high[kMaxCluster];
  unsigned tie_count[kMaxCluster];
  u64 part_mass[kMaxCluster], zone_sum[kZones][kMaxCluster], above_mass[kMaxCluster];
  u64 above_count[kMaxCluster];
  int cut_index;
  float cut_value;
  double scale, reach, floor_reach;  // of the row: log2(e) / T; how far below the top the masses end, and min_p reaches
  unsigned listed;
  int at;
};

static_assert(sizeof(Shared) % 16 == 0, "the logits after it are stored 16 bytes at a time");

// (the struct, the logits, their indexes; by its symbol in every function, so that the accesses are known to be to shared memory)
extern __shared__ __align__(16) unsigned char sample_smem[];
#define LB_S (*reinterpret_cast<Shared*>(sample_smem))

template <typename T>
__device__ __forceinline__ float logit(T v) {  // a NaN is never drawn
  float f;
  if constexpr (__is_same(T, float)) f = v;
  else if constexpr (__is_same(T, __half)) f = __half2float(v);
  else f = __bfloat162float(v);
  return f == f ? f : -INFINITY;
}
// whole numbers in the order of the values (both zeros are one value)
__device__ __forceinline__ unsigned ordered(float x) {
  const unsigned b = __float_as_uint(x + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(unsigned u) {
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}

// 2^y by a table of 2^(j / 128) and a Taylor series in f, |f| <= 2^-8 (first term left out below 2^-49 of the result).
struct Masses {
  double top, scale;  // the maximum, log2(e) / T
  float top_f, least; // least: so far down that its mass, and all below it, is 0
  // the mass in the low 52 bits; above them, always the same, the exponent of 2^52 (which the sum with it left there)
  __device__ __forceinline__ u64 bits(float x) const {
    const double y = (static_cast<double>(fmaxf(x, least)) - top) * scale;
    const double magic = 52776558133248.0;  // 1.5 * 2^45: the sum's last bit is 2^-7
    const double t = y + magic;
    const int n = __double2loint(t);        // 128 y, rounded
    const double f = y - (t - magic);
    constexpr double kLn2 = 0.69314718055994530942;
    const double p = fma(f, fma(f, fma(f, fma(f, kLn2 * kLn2 * kLn2 * kLn2 / 24.0, kLn2 * kLn2 * kLn2 / 6.0), kLn2 * kLn2 / 2.0), kLn2), 1.0);
    const double w = LB_S.power[n & (kPowers - 1)];
    // (the exponent goes up by whole powers of two)
    const double v = p * __hiloint2double(__double2hiint(w) + ((n & ~(kPowers - 1)) << (20 - 7)) + (kTop << 20), __double2loint(w));
    return static_cast<u64>(__double_as_longlong(v + 4503599627370496.0));  // rint: below 2^51
  }
  __device__ __forceinline__ u64 operator()(float x) const { return bits(x) & 0xfffffffffffffull; }
};
constexpr u64 kExponent = 0x433ull << 52;  // of 2^52
// 2^(j / 128)
__device__ const double powers[kPowers] = {
    1.0, 1.0054299011128027, 1.0108892860517005, 1.016378314910953, 1.0218971486541166, 1.0274459491187637,
    1.0330248790212284, 1.0386341019613787, 1.0442737824274138, 1.0499440858006872, 1.0556451783605572, 1.061377227289262,
    1.0671404006768237, 1.0729348675259756, 1.0787607977571199, 1.0846183622133092, 1.0905077326652577, 1.0964290818163769,
    1.102382583307841, 1.1083684117236787, 1.1143867425958924, 1.1204377524096067, 1.1265216186082418, 1.1326385195987192,
    1.1387886347566916, 1.1449721444318042, 1.1511892299529827, 1.1574400736337511, 1.1637248587775775, 1.1700437696832502,
    1.1763969916502812, 1.182784710984341, 1.189207115002721, 1.1956643920398273, 1.202156731452703, 1.2086843236265816,
    1.215247359980469, 1.2218460329727576, 1.22848053610687, 1.2351510639369334, 1.241857812073484, 1.2486009771892048,
    1.255380757024691, 1.2621973503942507, 1.2690509571917332, 1.275941778396392, 1.2828700160787783, 1.2898358734066657,
    1.2968395546510096, 1.3038812651919358, 1.3109612115247644, 1.318079601266064, 1.3252366431597413, 1.3324325470831615,
    1.339667524053303, 1.3469417862329458, 1.3542555469368927, 1.3616090206382248, 1.3690024229745905, 1.3764359707545302,
    1.383909881963832, 1.3914243757719262, 1.3989796725383112, 1.4065759938190154, 1.4142135623730951, 1.4218926021691656,
    1.42961333839197, 1.4373759974489824, 1.4451808069770467, 1.4530279958490526, 1.460917794180647, 1.4688504333369818,
    1.4768261459394993, 1.4848451658727524, 1.4929077282912648, 1.5010140696264256, 1.5091644275934228, 1.5173590411982147,
    1.5255981507445384, 1.533881997840956, 1.5422108254079407, 1.550584877685, 1.559004400237837, 1.567469639965553,
    1.5759808451078865, 1.5845382652524937, 1.593142151342267, 1.6017927556826934, 1.6104903319492543, 1.6192351351948637,
    1.6280274218573478, 1.6368674497669644, 1.645755478153965, 1.6546917676561943, 1.6636765803267364, 1.6727101796415966,
    1.681792830507429, 1.6909247992693053, 1.7001063537185235, 1.709337763100463, 1.718619298122478, 1.7279512309618377,
    1.7373338352737062, 1.746767386199169, 1.7562521603732995, 1.7657884359332727, 1.7753764925265212, 1.785016611318935,
    1.7947090750031072, 1.804454167806624, 1.8142521755003989, 1.8241033854070534, 1.8340080864093424, 1.843966568958626,
    1.8539791250833855, 1.864046048397789, 1.8741676341103, 1.8843441790323345, 1.8945759815869656, 1.9048633418176741,
    1.9152065613971474, 1.925605943636125, 1.9360617934922943, 1.9465744175792332, 1.9571441241754002, 1.9677712232331759,
    1.978456026387951, 1.9891988469672663,
};

__device__ __forceinline__ u64 warp_inclusive(u64 v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  return v;
}
__device__ __forceinline__ u64 warp_sum64(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// by the whole CTA; total: of all threads
__device__ __forceinline__ u64 block_inclusive(u64 v, u64* scan, u64& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  v = warp_inclusive(v);
  __syncthreads();
  if (lane == 31) scan[warp] = v;
  __syncthreads();
  u64 sums = lane < kWarps ? scan[lane] : 0;
#pragma unroll
  for (int o = 1; o < kWarps; o <<= 1) {
    const u64 y = __shfl_up_sync(0xffffffffu, sums, o);
    if (lane >= o) sums += y;
  }
  total = __shfl_sync(0xffffffffu, sums, kWarps - 1);
  const u64 before = __shfl_sync(0xffffffffu, sums, (warp + 31) & 31);
  return warp ? v + before : v;
}
// the sum alone
__device__ __forceinline__ u64 block_sum(u64 v, u64* scan) {
  const int lane = threadIdx.x & 31;
  v = warp_sum64(v);
  __syncthreads();
  if (lane == 0) scan[threadIdx.x >> 5] = v;
  __syncthreads();
  return warp_sum64(lane < kWarps ? scan[lane] : 0);
}
// over the CTAs of the cluster, one value each (by a warp): the sum, and of those before `rank`
__device__ __forceinline__ u64 slot_sum(const u64* slot, int ctas, int rank, u64& before) {
  const int lane = threadIdx.x & 31;
  const u64 v = lane < ctas ? slot[lane] : 0;
  u64 all = v, low = lane < rank ? v : 0;
#pragma unroll
  for (int o = kMaxCluster / 2; o > 0; o >>= 1) {
    all += __shfl_xor_sync(0xffffffffu, all, o);
    low += __shfl_xor_sync(0xffffffffu, low, o);
  }
  before = __shfl_sync(0xffffffffu, low, 0);
  return __shfl_sync(0xffffffffu, all, 0);
}
// 512 values, one a thread, rising
__device__ __forceinline__ u64 block_sort(u64 v, u64* room) {
  const int t = threadIdx.x;
#pragma unroll 1
  for (int size = 2; size <= kList; size <<= 1) {
#pragma unroll 1
    for (int step = size >> 1; step > 0; step >>= 1) {
      u64 other;
      if (step >= 32) {
        __syncthreads();
        room[t] = v;
        __syncthreads();
        other = room[t ^ step];
      } else {
        other = __shfl_xor_sync(0xffffffffu, v, step);
      }
      const bool low = ((t & step) == 0) == ((t & size) == 0);
      v = low ? (v < other ? v : other) : (v < other ? other : v);
    }
  }
  return v;
}

__device__ __forceinline__ u64 share_of(double p, u64 total) {  // ceil(p * total), at least 1
  const double x = ceil(p * static_cast<double>(total));
  return x >= 1.0 ? static_cast<u64>(x) : 1;
}
__device__ __forceinline__ u64 target_of(double u, u64 total) {  // floor(u * total), below the total
  const double x = floor(u * static_cast<double>(total));
  const u64 t = x > 0.0 ? static_cast<u64>(x) : 0;
  return t < total ? t : total - 1;
}

// What all threads of a row's CTAs know.
struct Row {
  int row, first, k;         // first: the index of this CTA's first token
  int pad, part;             // floats before its logits in shared memory; tokens of a CTA
  double u, top_p;
  u64 min_mass;
  float floor;               // below it no token has min_mass
  float heat, inv_heat;
  Masses mass;
  // Several passes have to put a token into the same bin, so nothing here may be contracted in one place and not in another.
  __device__ __forceinline__ float distance(float v) const { return __fmul_rn(__fsub_rn(mass.top_f, v), inv_heat); }
  __device__ __forceinline__ float* logits() const { return reinterpret_cast<float*>(sample_smem + sizeof(Shared)) + pad; }
  __device__ __forceinline__ uint16_t* indexes() const {
    return reinterpret_cast<uint16_t*>(sample_smem + sizeof(Shared) + (part + 8) * sizeof(float));
  }
};

// A warp's tokens that are left: at first all of its part of the CTA's tokens.
struct Left {
  int base, n;
  bool moved;  // they have been moved together, and their indexes (less base) stand beside them
  // body(logit, index in the CTA) for each, in order, lanes taking neighbours
  template <typename Body>
  __device__ __forceinline__ void each(const Row& r, Body body) const {
    const float* x = r.logits() + base;
    const int lane = threadIdx.x & 31;
    if (moved) {
      const uint16_t* at = r.indexes() + base;
#pragma unroll 1
      for (int j = lane; j < n; j += 32) body(x[j], base + at[j]);
    } else {
#pragma unroll 4
      for (int j = lane; j < n; j += 32) body(x[j], base + j);
    }
  }
  // moves those together that pred(logit, index in the CTA) picks
  template <typename Pred>
  __device__ __forceinline__ void keep(const Row& r, Pred pred) {
    float* x = r.logits() + base;
    uint16_t* at = r.indexes() + base;
    const int lane = threadIdx.x & 31;
    const unsigned before = (1u << lane) - 1;
    int kept = 0;
    if (moved) {
#pragma unroll 1
      for (int j0 = 0; j0 < n; j0 += 32) {
        const int j = j0 + lane;
        const float v = j < n ? x[j] : 0.0f;
        const int i = j < n ? at[j] : 0;
        const bool take = j < n && pred(v, base + i);
        const unsigned who = __ballot_sync(0xffffffffu, take);  // (everyone has read before anyone writes)
        if (take) {
          const int to = kept + __popc(who & before);
          x[to] = v;
          at[to] = static_cast<uint16_t>(i);
        }
        kept += __popc(who);
        __syncwarp();
      }
    } else {
      constexpr int kLooks = 4;
#pragma unroll 1
      for (int j0 = 0; j0 < n; j0 += 32 * kLooks) {
        float v[kLooks];
        unsigned who[kLooks];
#pragma unroll
        for (int q = 0; q < kLooks; ++q) {
          const int j = j0 + 32 * q + lane;
          v[q] = j < n ? x[j] : 0.0f;
          who[q] = __ballot_sync(0xffffffffu, j < n && pred(v[q], base + j));
        }
#pragma unroll
        for (int q = 0; q < kLooks; ++q) {
          if (who[q] == 0) continue;
          if (who[q] >> lane & 1u) {
            const int to = kept + __popc(who[q] & before);
            x[to] = v[q];
            at[to] = static_cast<uint16_t>(j0 + 32 * q + lane);
          }
          kept += __popc(who[q]);
        }
        __syncwarp();
      }
    }
    n = kept;
    moved = true;
  }
};

__device__ __forceinline__ void emit(const SampleArgs& a, const Row& r, int token, u64 mass, u64 total) {
  a.tokens[r.row] = token;
  if (a.logprobs) a.logprobs[r.row] = static_cast<float>(log(static_cast<double>(mass) / static_cast<double>(total)));
}

// One CTA has in s.list all tokens that can be drawn (n, in any order): the rest of the work.  k: of them the first k
// count; limit: the mass up to which top-p keeps, 0 where it is to be taken from their own sum.
__device__ __forceinline__ void finish_list(const SampleArgs& a, const Row& r, int n, int k, u64 limit) {
  Shared& s = LB_S;
  const int t = threadIdx.x;
  if (n <= kFew) {  // each token finds what comes before it, by value and then by index
    const u64 key = t < n ? s.list[t] : kNone;
    u64 m = t < n ? r.mass(from_ordered(~static_cast<unsigned>(key >> 32))) : 0, before = 0;
    if (t < n) s.mass[t] = m;
    __syncthreads();
    int rank = 0;
    if (t < n)
#pragma unroll 4
      for (int j = 0; j < n; ++j) {
        const bool first = s.list[j] < key;
        rank += first;
        before += first ? s.mass[j] : 0;
      }
    if (rank >= k) m = 0;
    if (r.top_p < 1.0) {
      if (limit == 0) limit = share_of(r.top_p, block_sum(m, s.scan));
      if (before >= limit) m = 0;
    }
    if (m < r.min_mass) m = 0;
    const u64 total = block_sum(m, s.scan), target = target_of(r.u, total);  // (everyone has read the masses)
    if (t < n) s.mass[t] = m;
    __syncthreads();
    if (m) {
      u64 to = 0;
#pragma unroll 4
      for (int j = 0; j < n; ++j) to += static_cast<unsigned>(s.list[j]) < static_cast<unsigned>(key) ? s.mass[j] : 0;
      if (to <= target && target < to + m) emit(a, r, static_cast<int>(static_cast<unsigned>(key)), m, total);
    }
    return;
  }
  const u64 key = block_sort(t < n ? s.list[t] : kNone, s.mass);
  const float x = from_ordered(~static_cast<unsigned>(key >> 32));
  const int index = static_cast<int>(static_cast<unsigned>(key));
  u64 m = t < n && t < k ? r.mass(x) : 0, total;
  const u64 upto = block_inclusive(m, s.scan, total);
  if (r.top_p < 1.0) {
    if (limit == 0) limit = share_of(r.top_p, total);
    if (upto - m >= limit) m = 0;
  }
  if (m < r.min_mass) m = 0;
  __syncthreads();  // (the sort's room is free)
  s.mass[t] = m;
  const u64 by_index = block_sort(m ? static_cast<u64>(index) << 32 | t : kNone, s.list);
  const u64 mine = by_index == kNone ? 0 : s.mass[by_index & (kList - 1)];
  const u64 to = block_inclusive(mine, s.scan, total);
  const u64 target = target_of(r.u, total);
  if (mine && target >= to - mine && target < to) emit(a, r, static_cast<int>(by_index >> 32), mine, total);
}

// Cuts what is left to the first k tokens (kMass false), or to the first whose masses reach a share of the sum (true), in the
// order (value down, index up).  Returns true where the leading CTA has all that can be drawn in its list, as finish_list takes it.
struct Listed {
  int n, k;
  u64 limit;
};
template <bool kMass>
__device__ __forceinline__ bool select(const Row& r, cg::cluster_group& cluster, Left& left, Listed& listed) {
  Shared& s = LB_S;
  const int t = threadIdx.x, rank = cluster.block_rank(), ctas = cluster.num_blocks(), lane = t & 31, warp = t >> 5;
  u64 limit = kMass ? 0 : r.k, above = 0;
  int before = 0;
  unsigned lo = 0, hi = 0;
  int shift = 0;
  // the first division: distances from zone_lo on
  float zone_lo = 0.0f, zone_top = INFINITY, zone_bins = 16.0f;
  if constexpr (kMass) {
    // the sum of all masses, and what comes of it up to some distances in 2^24 units, each token's part rounded down
    u64 sum = 0;
    unsigned zone[kZones];
#pragma unroll
    for (int z = 0; z < kZones; ++z) zone[z] = 0;
    float end[kZones];
#pragma unroll
    for (int z = 0; z < kZones; ++z) end[z] = __fsub_rn(r.mass.top_f, __fmul_rn(zone_end(z), r.heat));
    left.each(r, [&](float x, int) {
      const u64 m = r.mass.bits(x);
      sum += m;
      const unsigned about = static_cast<unsigned>(m >> 24) & ((1u << 28) - 1);
#pragma unroll
      for (int z = 0; z < kZones; ++z) zone[z] += x > end[z] ? about : 0u;
    });
    sum -= static_cast<u64>(lane < left.n ? (left.n - lane + 31) / 32 : 0) * kExponent;
#pragma unroll
    for (int z = 0; z < kZones; ++z) {  // (2^12 tokens a warp, each at most 2^21)
      const u64 all = warp_sum64(zone[z]);
      if (lane == 0) s.zone[warp][z] = static_cast<unsigned>(all >> 3);
    }
    u64 total = block_sum(sum, s.scan), none;  // (a barrier for the zones too)
    if (t < ctas) {
      *cluster.map_shared_rank(&s.part_mass[rank], t) = total;
#pragma unroll
      for (int z = 0; z < kZones; ++z) {
        u64 v = 0;
        for (int w = 0; w < kWarps; ++w) v += s.zone[w][z];
        *cluster.map_shared_rank(&s.zone_sum[z][rank], t) = v;
      }
    }
    cluster.sync();
    if (warp == 0) {  // (one warp for all: sixteen would take the others' issue slots)
      limit = share_of(r.top_p, slot_sum(s.part_mass, ctas, 0, none));
      // The sums are in units of 2^27, each short of its true value by less than 2^16 of them: a unit for each of 2^18 tokens and each
      // warp.
      const u64 want = limit >> 27;
      Zone z0{limit, 0.0f, INFINITY, INFINITY, r.mass.least};
#pragma unroll
      for (int z = kZones - 1; z >= 0; --z) {
        const u64 v = slot_sum(s.zone_sum[z], ctas, 0, none);
        if (v > want) {
          z0.hi = zone_end(z);
          z0.low = end[z];
        }
        if (z0.lo == 0.0f && v + (1u << 16) < want) {
          z0.lo = zone_end(z);
          z0.top = end[z];
        }
      }
      if (lane == 0) s.chosen = z0;
    }
    __syncthreads();
    limit = s.chosen.limit;
    zone_lo = s.chosen.lo;
    zone_top = s.chosen.top;
    const float zone_hi = s.chosen.hi, low = s.chosen.low;
    zone_bins = zone_hi < INFINITY ? kBins / (zone_hi - zone_lo) : 16.0f;
    left.keep(r, [&](float x, int) { return x > low; });
  }
  for (int level = 0; level < 6; ++level) {  // (each division leaves one value, or 512 times fewer: six are never reached)
    const int turn = level & 1;
    // ---- tokens and masses by bins
    for (int i = t; i < (kMass ? 4 : 1) * kBins; i += kThreads) (&s.hist[0][0])[i] = 0;
    if (t == 0) s.listed = 0;
    __syncthreads();
    // In bins from the zone's beginning; infinite (of -infinity, and where a product overflows, far below any mass): in none.
    const auto place_of = [&](float x) { return __fmul_rn(__fsub_rn(r.distance(x), zone_lo), zone_bins); };
    const auto bin_of = [&](float x) -> int {  // -1: below, -2: above
      if (level == 0) {
        const float place = place_of(x);
        return place >= INFINITY ? -1 : x > zone_top ? -2 : max(0, min(kBins - 1, __float2int_rz(place)));
      }
      const unsigned o = ordered(x);
      return o < lo ? -1 : o > hi ? -2 : static_cast<int>((hi - o) >> shift);
    };
    u64 over = 0;  // of the tokens above the zone
    unsigned over_count = 0;
    left.each(r, [&](float x, int) {
      const int b = bin_of(x);
      if (b >= 0) atomicAdd(&s.hist[0][b], 1u);
      if constexpr (kMass) {
        if (b == -1) return;
        if (b == -2 && level > 0) return;
        const u64 m = r.mass(x);
        if (b >= 0) {
          const unsigned m0 = m & 0xffff, m1 = (m >> 16) & 0xffff, m2 = static_cast<unsigned>(m >> 32);
          if (m0) atomicAdd(&s.hist[1][b], m0);
          if (m1) atomicAdd(&s.hist[2][b], m1);
          if (m2) atomicAdd(&s.hist[3][b], m2);
        } else {
          over += m;
          ++over_count;
        }
      }
    });
    if (kMass && level == 0) {
      over = block_sum(over, s.scan);
      const u64 count = block_sum(over_count, s.scan2);
      if (t < ctas) {
        *cluster.map_shared_rank(&s.above_mass[rank], t) = over;
        *cluster.map_shared_rank(&s.above_count[rank], t) = count;
      }
    }
    __syncthreads();
    // ---- sums of groups of bins go to every CTA
    u64 mass_here = 0;
    {
      const unsigned c = __reduce_add_sync(0xffffffffu, s.hist[0][t]);
      if constexpr (kMass) mass_here = s.hist[1][t] + (static_cast<u64>(s.hist[2][t]) << 16) + (static_cast<u64>(s.hist[3][t]) << 32);
      const u64 m = kMass ? warp_sum64(mass_here) : 0;
      if (lane == 0) {
        s.warp_count[warp] = c;
        s.scan[warp] = m;
      }
    }
    __syncthreads();
    if constexpr (kMass) reinterpret_cast<u64*>(&s.hist[2][0])[t] = mass_here;  // (the limbs have been read: whole masses take their place)
    if (t < kGroups * ctas) {
      constexpr int kEach = kWarps / kGroups;
      const int g = t % kGroups, to = t / kGroups;
      unsigned c = 0;
      u64 m = 0;
#pragma unroll
      for (int w = 0; w < kEach; ++w) {
        c += s.warp_count[g * kEach + w];
        m += s.scan[g * kEach + w];
      }
      *cluster.map_shared_rank(&s.group_count[turn][g][rank], to) = c;
      if constexpr (kMass) *cluster.map_shared_rank(&s.group_mass[turn][g][rank], to) = m;
    }
    cluster.sync();
    // ---- the group that holds the cut, then its bins over the cluster: every CTA finds the bin for itself
    if (warp == 0) {
      if (kMass && level == 0) {
        u64 none;
        above = slot_sum(s.above_mass, ctas, 0, none);
        before = static_cast<int>(slot_sum(s.above_count, ctas, 0, none));
      }
      // a lane has a group and every fourth CTA
      const int g = lane % kGroups;
      unsigned c = 0;
      u64 m = 0;
#pragma unroll
      for (int q = 0; q < kMaxCluster; q += 32 / kGroups) {
        const int from = q + lane / kGroups;
        if (from < ctas) {
          c += s.group_count[turn][g][from];
          if constexpr (kMass) m += s.group_mass[turn][g][from];
        }
      }
#pragma unroll
      for (int o = kGroups; o < 32; o <<= 1) {
        c += __shfl_xor_sync(0xffffffffu, c, o);
        if constexpr (kMass) m += __shfl_xor_sync(0xffffffffu, m, o);
      }
      unsigned upto_c = c;
      u64 upto_m = m;
#pragma unroll
      for (int o = 1; o < kGroups; o <<= 1) {
        const unsigned y = __shfl_up_sync(0xffffffffu, upto_c, o, kGroups);
        const u64 z = kMass ? __shfl_up_sync(0xffffffffu, upto_m, o, kGroups) : 0;
        if (g >= o) {
          upto_c += y;
          upto_m += z;
        }
      }
      const u64 to = above + (kMass ? upto_m : upto_c), mine = kMass ? m : c;
      const unsigned who = __ballot_sync(0xffffffffu, lane < kGroups && to - mine < limit && limit <= to);
      const int group = who ? __ffs(who) - 1 : 0;
      const u64 base = __shfl_sync(0xffffffffu, to - mine, group);
      const unsigned seen = before + __shfl_sync(0xffffffffu, upto_c - c, group);
      if (who == 0 && lane == 0) s.result = {0, -1, 0, 0};
      // two bins a lane
      static_assert(kGroupBins == 64, "two bins a lane");
      u64 w[2] = {0, 0};
      unsigned n[2] = {0, 0};
#pragma unroll
      for (int q0 = 0; q0 < kMaxCluster; q0 += 4) {  // four CTAs' bins are under way at once
        uint2 c[4];
        ulonglong2 m[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if (q0 + q < ctas) {
            const unsigned* p = cluster.map_shared_rank(&s.hist[0][0], q0 + q);
            c[q] = reinterpret_cast<const uint2*>(p + group * kGroupBins)[lane];
            if constexpr (kMass) m[q] = reinterpret_cast<const ulonglong2*>(p + 2 * kBins + 2 * group * kGroupBins)[lane];
          }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if (q0 + q < ctas) {
            n[0] += c[q].x;
            n[1] += c[q].y;
            if constexpr (kMass) {
              w[0] += m[q].x;
              w[1] += m[q].y;
            }
          }
        }
      }
      if constexpr (!kMass) {
        w[0] = n[0];
        w[1] = n[1];
      }
      u64 upto = base + warp_inclusive(w[0] + w[1]);
      unsigned upto_n = n[0] + n[1];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned y = __shfl_up_sync(0xffffffffu, upto_n, o);
        if (lane >= o) upto_n += y;
      }
      upto -= w[1];
      if (who && upto - w[0] < limit && limit <= upto)
        s.result = {upto - w[0], group * kGroupBins + 2 * lane, static_cast<int>(n[0]), static_cast<int>(seen + upto_n - n[1] - n[0])};
      if (who && upto < limit && limit <= upto + w[1])
        s.result = {upto, group * kGroupBins + 2 * lane + 1, static_cast<int>(n[1]), static_cast<int>(seen + upto_n - n[1])};
    }
    __syncthreads();
    const Result found = s.result;
    if (found.bin < 0) return false;  // (counts: no more than k tokens, all are kept)
    above = found.above;
    before = found.before;
    const bool all = found.before + found.count <= kList;  // everything down to the cut fits the list
    // the tokens of the bin and above: at level 0 by the product that the bin is the whole part of
    const float edge = found.bin == kBins - 1 ? INFINITY : static_cast<float>(found.bin + 1);
    const auto down_to = [&](float x) {
      if (level == 0) return place_of(x) < edge;
      const int b = bin_of(x);
      return b == -2 || (b >= 0 && b <= found.bin);
    };
    if (all || found.count <= kList) {
      Shared& lead = *cluster.map_shared_rank(&s, 0);
      if (level == 0) left.keep(r, [&](float x, int) { return place_of(x) < edge; });
      else left.keep(r, [&](float x, int) { return down_to(x); });
      const float* x = r.logits() + left.base;
      const uint16_t* at = r.indexes() + left.base;
      int mine = 0;
      if (all) mine = left.n;
      else left.each(r, [&](float v, int) { mine += bin_of(v) == found.bin; });
      if (!all) mine = __reduce_add_sync(0xffffffffu, mine);
      if (mine > 0) {
        unsigned to = 0;
        if (lane == 0) to = atomicAdd(&lead.listed, mine);
        to = __shfl_sync(0xffffffffu, to, 0);
        for (int j0 = 0; j0 < left.n; j0 += 32) {
          const int j = j0 + lane;
          const bool take = j < left.n && (all || bin_of(x[j]) == found.bin);
          const unsigned who = __ballot_sync(0xffffffffu, take);
          const unsigned place = to + __popc(who & ((1u << lane) - 1));
          if (take && place < kList) lead.list[place] = static_cast<u64>(~ordered(x[j])) << 32 | static_cast<unsigned>(r.first + left.base + at[j]);
          to += __popc(who);
        }
      }
      cluster.sync();
      if (all) {
        listed = {found.before + found.count, kMass ? kList : r.k, limit * kMass};
        return true;
      }
      if (rank == 0) {
        u64 key = t < found.count ? s.list[t] : kNone, w, to;
        if (found.count <= kFew) {  // each finds what comes before it
          w = t < found.count ? (kMass ? r.mass(from_ordered(~static_cast<unsigned>(key >> 32))) : 1) : 0;
          if (t < found.count) s.mass[t] = w;
          __syncthreads();
          to = above + w;
          if (t < found.count)
#pragma unroll 4
            for (int j = 0; j < found.count; ++j) to += s.list[j] < key ? s.mass[j] : 0;
        } else {
          key = block_sort(key, s.mass);
          w = t < found.count ? (kMass ? r.mass(from_ordered(~static_cast<unsigned>(key >> 32))) : 1) : 0;
          u64 total;
          to = above + block_inclusive(w, s.scan, total);
        }
        if (to - w < limit && limit <= to) {
          for (int c = 0; c < ctas; ++c) {
            *cluster.map_shared_rank(&s.cut_value, c) = from_ordered(~static_cast<unsigned>(key >> 32));
            *cluster.map_shared_rank(&s.cut_index, c) = static_cast<int>(static_cast<unsigned>(key));
          }
        }
      }
      cluster.sync();
    } else {
      // ---- too many: the bin's values are the next division's range
      bool single;
      if (level == 0) {
        left.keep(r, [&](float x, int) { return down_to(x); });
        unsigned least = 0xffffffffu, most = 0;
        left.each(r, [&](float x, int) {
          if (bin_of(x) == found.bin) {
            least = min(least, ordered(x));
            most = max(most, ordered(x));
          }
        });
        least = __reduce_min_sync(0xffffffffu, least);
        most = __reduce_max_sync(0xffffffffu, most);
        __syncthreads();
        if (lane == 0) s.scan[warp] = static_cast<u64>(most) << 32 | least;
        __syncthreads();
        if (t < ctas) {
          for (int w = 0; w < kWarps; ++w) {
            least = min(least, static_cast<unsigned>(s.scan[w]));
            most = max(most, static_cast<unsigned>(s.scan[w] >> 32));
          }
          *cluster.map_shared_rank(&s.low[rank], t) = least;
          *cluster.map_shared_rank(&s.high[rank], t) = most;
        }
        cluster.sync();
        lo = s.low[0];
        hi = s.high[0];
        for (int c = 1; c < ctas; ++c) {
          lo = min(lo, s.low[c]);
          hi = max(hi, s.high[c]);
        }
        single = lo == hi;
      } else {
        cluster.sync();  // (the bins have been read everywhere)
        single = shift == 0;
        hi -= static_cast<unsigned>(found.bin) << shift;
        lo = hi - lo >= 1u << shift ? hi - ((1u << shift) - 1) : lo;
      }
      if (!single) {
        for (shift = 0; (hi - lo) >> shift >= kBins;) ++shift;
        continue;
      }
      // ---- one value: so many of its tokens, the lowest indexes first
      const float value = from_ordered(lo);
      const u64 w = kMass ? r.mass(value) : 1;
      const unsigned want = static_cast<unsigned>((limit - above + w - 1) / w);
      unsigned ties = 0;
      left.each(r, [&](float x, int) { ties += x == value; });
      ties = __reduce_add_sync(0xffffffffu, ties);
      u64 cta_ties;
      const u64 upto = block_inclusive(lane == 31 ? ties : 0, s.scan, cta_ties);
      if (t < ctas) *cluster.map_shared_rank(&s.tie_count[rank], t) = static_cast<unsigned>(cta_ties);
      cluster.sync();
      unsigned seen = 0;
      for (int c = 0; c < rank; ++c) seen += s.tie_count[c];
      seen += __shfl_sync(0xffffffffu, static_cast<unsigned>(upto), 31) - ties;  // before this warp
      if (seen < want && want <= seen + ties) {
        const float* x = r.logits() + left.base;
        for (int j0 = 0; j0 < left.n; j0 += 32) {
          const int j = j0 + lane;
          const bool tie = j < left.n && x[j] == value;
          const unsigned who = __ballot_sync(0xffffffffu, tie);
          if (tie && seen + __popc(who & ((2u << lane) - 1)) == want) {
            const int at = r.first + left.base + (left.moved ? r.indexes()[left.base + j] : j);
            for (int c = 0; c < ctas; ++c) {
              *cluster.map_shared_rank(&s.cut_value, c) = value;
              *cluster.map_shared_rank(&s.cut_index, c) = at;
            }
          }
          seen += __popc(who);
        }
      }
      cluster.sync();
    }
    const float cut = s.cut_value;
    const int cut_index = s.cut_index;
    left.keep(r, [&](float x, int i) { return x > cut || (x == cut && r.first + i <= cut_index); });
    return false;
  }
  return false;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const SampleArgs a) {
  Shared& s = LB_S;
  cg::cluster_group cluster = cg::this_cluster();
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int rank = cluster.block_rank(), ctas = cluster.num_blocks();
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // (this CTA has begun)
  Row r;
  r.row = blockIdx.x / ctas;
  r.first = min(a.vocab, rank * a.part);
  r.part = a.part;
  const int n = min(a.vocab, r.first + a.part) - r.first;

  // ---- this CTA's logits as floats; the aligned part by 16 bytes
  constexpr int kVec = 16 / sizeof(T);
  const T* src = static_cast<const T*>(a.logits) + r.row * a.row_stride + r.first;
  const int head = min(n, static_cast<int>((16 - reinterpret_cast<uintptr_t>(src) % 16) % 16 / sizeof(T)));
  const int vecs = (n - head) / kVec, pad = (kVec - head) % kVec;
  r.pad = pad;
  float* x = r.logits();
  float top = -INFINITY;
  const uint4* body = reinterpret_cast<const uint4*>(src + head);
  constexpr int kAhead = sizeof(T) == 4 ? 8 : 4;
  for (int v0 = t; v0 < vecs; v0 += kThreads * kAhead) {
    uint4 raw[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (v0 + j * kThreads < vecs) raw[j] = __ldcs(body + v0 + j * kThreads);
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int v = v0 + j * kThreads;
      if (v >= vecs) break;
      const T* part = reinterpret_cast<const T*>(&raw[j]);
#pragma unroll
      for (int e = 0; e < kVec; e += 4) {
        const float4 f = make_float4(logit(part[e]), logit(part[e + 1]), logit(part[e + 2]), logit(part[e + 3]));
        top = fmaxf(top, fmaxf(fmaxf(f.x, f.y), fmaxf(f.z, f.w)));
        *reinterpret_cast<float4*>(x + head + v * kVec + e) = f;
      }
    }
  }
  const int rest = n - head - vecs * kVec;
  if (t < head + rest) {
    const int i = t < head ? t : head + vecs * kVec + (t - head);
    x[i] = logit(src[i]);
    top = fmaxf(top, x[i]);
  }
  if (t < kPowers) s.power[t] = powers[t];

  // ---- the row's settings and its maximum
  const float heat = fminf(a.temperature ? a.temperature[r.row] : a.temperature1, kMaxHeat);  // (NaN: the limit)
  const float p = a.top_p ? a.top_p[r.row] : a.top_p1, least = a.min_p ? a.min_p[r.row] : a.min_p1;
  r.k = a.top_k ? a.top_k[r.row] : a.top_k1;
  if (r.k <= 0 || r.k > a.vocab) r.k = a.vocab;
  r.top_p = p < 1.0f ? static_cast<double>(p) : 1.0;
  r.min_mass = least > 0.0f ? static_cast<u64>(ceil(static_cast<double>(fminf(least, 1.0f)) * static_cast<double>(1ull << kTop))) : 0;
  r.u = a.uniform64 ? static_cast<const double*>(a.uniform)[r.row] : static_cast<double>(static_cast<const float*>(a.uniform)[r.row]);
  if (t == 32) {
    s.scale = 1.4426950408889634074 / static_cast<double>(heat);
    s.reach = 47.0 * 0.69314718055994530942 * (1.0 + 1e-9) * static_cast<double>(heat);
    s.floor_reach = r.min_mass ? (kTop + 0.01 - log2(static_cast<double>(r.min_mass))) / s.scale : 0.0;  // (a hundredth of an octave to spare)
  }
  const bool greedy = !(heat > 0.0f) || (a.temperature && a.temperature[r.row] != a.temperature[r.row]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) s.scan[warp] = __float_as_uint(top);
  __syncthreads();
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // all have, before one writes to another
  if (t < ctas) {
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, __uint_as_float(static_cast<unsigned>(s.scan[w])));
    *cluster.map_shared_rank(&s.top[rank], t) = top;
  }
  cluster.sync();
  top = s.top[0];
  for (int c = 1; c < ctas; ++c) top = fmaxf(top, s.top[c]);
  if (top == -INFINITY) {  // nothing to draw from
    if (rank == 0 && t == 0) {
      a.tokens[r.row] = -1;
      if (a.logprobs) a.logprobs[r.row] = -INFINITY;
    }
    return;
  }
  if (greedy) {  // the lowest index of the maximum
    unsigned at = 0xffffffffu;
    for (int i = t; i < n; i += kThreads)
      if (x[i] == top) at = min(at, static_cast<unsigned>(r.first + i));
    at = __reduce_min_sync(0xffffffffu, at);
    __syncthreads();
    if (lane == 0) s.scan[warp] = at;
    __syncthreads();
    if (t == 0) {
      for (int w = 0; w < kWarps; ++w) at = min(at, static_cast<unsigned>(s.scan[w]));
      *cluster.map_shared_rank(&s.low[rank], 0) = at;
    }
    cluster.sync();
    if (rank == 0 && t == 0) {
      for (int c = 0; c < ctas; ++c) at = min(at, s.low[c]);
      a.tokens[r.row] = at;
      if (a.logprobs) a.logprobs[r.row] = 0.0f;
    }
    return;
  }
  // Infinities share the draw alone: they become 0, the rest nothing.  Where the numbers end within the masses' reach of the maximum (a row
  // that a mask filled with the lowest number) nothing finite would be left for those without a mass, -infinity
  // among them: such a row is moved up by its maximum, which is exact for numbers within a factor of two.
  const bool infinite = top == INFINITY, low = top == -FLT_MAX || static_cast<double>(top) - s.reach < -static_cast<double>(FLT_MAX);
  if (infinite || low) {
    for (int i = t; i < n; i += kThreads) x[i] = low ? x[i] - top : x[i] == INFINITY ? 0.0f : -INFINITY;
    top = 0.0f;
    __syncthreads();
  }
  r.heat = heat;
  r.inv_heat = fminf(1.0f / heat, 1e30f);
  r.mass = {static_cast<double>(top), s.scale, top, 0.0f};
  // Where the next number below the top has no mass any more, no larger scale is needed: exponents stay above -150.
  const int bits = __float_as_int(top);
  const float below = top == 0.0f ? __int_as_float(0x80000001u) : __int_as_float(bits + (bits < 0 ? 1 : -1));
  const double next = static_cast<double>(top) - static_cast<double>(below);
  if (r.mass.scale * next > 47.0) r.mass.scale = 47.0 / next;
  r.mass.least = __double2float_rd(static_cast<double>(top) - (s.reach > next ? s.reach : next));  // 2^-47 of the top's mass is 0
  r.floor = r.min_mass ? __double2float_rd(static_cast<double>(top) - s.floor_reach) : -INFINITY;
  const int seg = ((a.part + kWarps - 1) / kWarps + 31) / 32 * 32;
  Left left{min(n, warp * seg), min(n, (warp + 1) * seg) - min(n, warp * seg), false};
  Listed listed{kList, r.k, 0};
  bool done = false;
  if (a.vocab <= kList) {  // (one CTA; what cannot be drawn sorts behind the rest and has no mass)
    const bool there = t < n && x[t] > -INFINITY;
    s.list[t] = there ? static_cast<u64>(~ordered(x[t])) << 32 | static_cast<unsigned>(t) : kNone;
    done = true;
  }
  if (!done && r.k < a.vocab) done = select<false>(r, cluster, left, listed);
  if (!done && r.top_p < 1.0) done = select<true>(r, cluster, left, listed);
  if (done) {
    if (rank == 0) finish_list(a, r, listed.n, listed.k, listed.limit);
    return;
  }

  // ---- the kept masses in the order of the indexes: by warps, by CTAs, and the warp with the target once more
  const auto mass_of = [&](float v) -> u64 {
    if (v < r.floor) return 0;
    const u64 m = r.mass(v);
    return m >= r.min_mass ? m : 0;
  };
  u64 mine = 0, cta_mass;
  if (r.min_mass) {
    left.each(r, [&](float v, int) { mine += mass_of(v); });
  } else {
    left.each(r, [&](float v, int) { mine += r.mass.bits(v); });
    mine -= static_cast<u64>(lane < left.n ? (left.n - lane + 31) / 32 : 0) * kExponent;
  }
  mine = warp_sum64(mine);
  u64 upto = __shfl_sync(0xffffffffu, block_inclusive(lane == 31 ? mine : 0, s.scan, cta_mass), 31);
  if (t < ctas) *cluster.map_shared_rank(&s.part_mass[rank], t) = cta_mass;
  cluster.sync();
  u64 base;
  const u64 total = slot_sum(s.part_mass, ctas, rank, base);
  const u64 target = target_of(r.u, total);
  if (target < base || target >= base + cta_mass) return;
  if (base + upto - mine <= target && target < base + upto) {  // this warp's tokens, which all warps share now
    if (lane == 0) {
      s.at = warp;
      s.list[0] = base + upto - mine;
      s.list[1] = static_cast<u64>(left.base) << 32 | static_cast<unsigned>(left.n) << 1 | (left.moved ? 1u : 0u);
    }
  }
  __syncthreads();
  base = s.list[0];
  const u64 where = s.list[1];
  const int share = static_cast<int>(static_cast<unsigned>(where) >> 1), from_base = static_cast<int>(where >> 32);
  const bool moved = where & 1;
  const int sub = (share + kWarps * 32 - 1) / (kWarps * 32) * 32, from = min(share, warp * sub), to = min(share, from + sub);
  mine = 0;
  for (int j = from + lane; j < to; j += 32) mine += mass_of(x[from_base + j]);
  mine = warp_sum64(mine);
  upto = base + __shfl_sync(0xffffffffu, block_inclusive(lane == 31 ? mine : 0, s.scan, cta_mass), 31);
  if (upto - mine <= target && target < upto) {
    u64 sum_before = upto - mine;
    for (int j0 = from; j0 < to; j0 += 32) {
      const int j = j0 + lane;
      const u64 m = j < to ? mass_of(x[from_base + j]) : 0;
      const u64 sum = sum_before + warp_inclusive(m);
      if (m && sum - m <= target && target < sum)
        emit(a, r, r.first + from_base + (moved ? r.indexes()[from_base + j] : j), m, total);
      sum_before = __shfl_sync(0xffffffffu, sum, 31);
    }
  }
}

// two CTAs an SM at 16384 tokens: 228 KB, of which each takes one besides
static_assert(sizeof(Shared) + (16384 + 8) * 6 <= 113 * 1024, "room");

template <typename T>
cudaError_t launch(SampleArgs a, int ctas, cudaStream_t s) {
  const auto kernel = sample_kernel<T>;
  static std::atomic<unsigned long long> done{0};
  cudaError_t e = ensure_smem(done, reinterpret_cast<const void*>(kernel), static_cast<int>(sizeof(Shared)) + (kMaxPart + 8) * 6);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = static_cast<unsigned>(a.rows) * ctas;
  cfg.blockDim = kThreads;
  cfg.dynamicSmemBytes = sizeof(Shared) + (a.part + 8) * (sizeof(float) + sizeof(uint16_t));
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {static_cast<unsigned>(ctas), 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kernel, a);
  return e == cudaSuccess ? cudaGetLastError() : e;
}

}  // namespace
}  // namespace lb

extern "C" int lb_op_sample(const void* logits, int64_t row_stride, int dtype, int rows, int vocab, const void* uniform,
                            int uniform64, const float* temperature, float temperature1, const int32_t* top_k, int top_k1,
                            const float* top_p, float top_p1, const float* min_p, float min_p1, int64_t* tokens,
                            float* logprobs, void* stream) {
  using namespace lb;
  if (!logits || !uniform || !tokens || rows < 1 || vocab < 1 || row_stride < vocab) return LB_ERR_INVALID_ARGUMENT;
  if (dtype != LB_F32 && dtype != LB_BF16 && dtype != LB_F16) return LB_ERR_INVALID_ARGUMENT;
  if (!temperature && !(temperature1 >= 0.0f && temperature1 <= kMaxHeat)) return LB_ERR_INVALID_ARGUMENT;
  if ((!top_p && !(top_p1 >= 0.0f)) || (!min_p && !(min_p1 >= 0.0f && min_p1 <= 1.0f))) return LB_ERR_INVALID_ARGUMENT;
  if (vocab > kMaxVocab || rows > (1 << 24)) return LB_ERR_CAPACITY;
  // 16384 tokens a CTA, 32768 beyond 131072
  int ctas = 1;
  while (ctas < kMaxCluster && (vocab + ctas - 1) / ctas > 16384) ctas *= 2;
  const int part = ((vocab + ctas - 1) / ctas + 7) / 8 * 8;
  SampleArgs a{logits, row_stride, uniform, temperature, top_p, min_p, top_k, temperature1, top_p1, min_p1, top_k1, rows, vocab,
               part, uniform64 != 0, reinterpret_cast<long long*>(tokens), logprobs};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == LB_F32 ? launch<float>(a, ctas, s) : dtype == LB_BF16 ? launch<__nv_bfloat16>(a, ctas, s)
                                                                                     : launch<__half>(a, ctas, s);
  return e == cudaSuccess ? LB_OK : LB_ERR_CUDA;
}
