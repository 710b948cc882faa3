// The first half of a gated feed-forward block with 4-bit weights, in one kernel:
//   out[t][o] = act(g) * u,  g = sum_k x[t][k] W[o][k],  u = sum_k x[t][k] W[f + o][k],  W = (n - 8) * s[row][k / group]
//
// Both products run on tcgen05 from one token to thousands, with the outputs as the rows of the MMA (128 gate rows and
// the 128 up rows that belong to them) and the tokens as its columns.  The weights are never rounded: the
// MMAs take the whole numbers n - 8, exact in each operand type (bf16 or fp16 for x of that type, e4m3 and int8 for 8-bit x, which
// goes to the tensor cores as it lies), and the sum of each group leaves the tensor memory and takes its scale in 32
// bits, where an output's lane makes the scale a register.
//
// Widened codes never see shared memory: warps read the codes that TMA brought, widen them in registers (12 or 13
// instructions for 8 codes, 6 to int8) and store them to the tensor memory, from where the MMAs take them as their A operand.
// Shared memory then only has to feed x to the MMAs.
//
// Warpgroups: 0 loads (warp 0: TMA; warp 2: x's scales of a group) and issues the MMAs (warps 1 and 3, a side each); 1 and 2 widen, a
// side each; 3 and 4 add up, half of the tokens each, and finish the tile.  A unit is one side's (gate or up) product over a block of
// K: while the one side's sums are taken out of the tensor memory the other side's MMAs run.
//
// Few tokens: the tiles of outputs are fewer than the SMs, so K is dealt out to the CTAs of a cluster.  Each sends its partial
// sums to the CTA that finishes the token (stores over the cluster), which adds them up in the order of K.
//
// Measured, 1536 x 6144 in groups of 128 (calls in one graph, weights out of L2): 2 rows of e4m3 12.1 us (9.8 MB at 0.8 TB/s: a
// chain of launch, first loads, six blocks of some 0.67 us, in which the widening warps set the pace, and the join; weights in L2
// 11.2), of bf16 10.8; bf16: 128 rows 15.4, 499 rows 28, 4096 rows 143 (1081 TFLOP/s, 65 % of the measured rate; 162 us where the
// power limit holds the clocks down); 4096 rows in fp16 153, int8 156, e4m3 178, with x's scales in groups of 128 213 and 206.
// What bounds the large ones is the work beside the MMAs: of some 5 thousand instructions for a tile of 128 tokens and a block of K
// the widening takes a third, sums a sixth and results a tenth.  A tile's results are not covered by the next one's MMAs, which
// stop two units ahead.  Groups of 64 and 32 take two and four times the sums: 204 and 327 us. On the way (4096 rows, the steps'
// own times): one lane issuing all MMAs 254 us, a warp that walks together 214, two widening warpgroups instead of one 192, a warp
// a side for the MMAs 164 (the waits of one were as long as its MMAs), results without a loop 145.
#include "../../include/listener_b200.h"
#include "common.cuh"
#include "kernels.h"
#include "rows.h"

namespace lb {
namespace {

constexpr int kThreads = 640, kFirstAdder = 12;  // warps
constexpr int kBlockO = 128;                   // outputs of a tile
constexpr int kBlockK = 128;                   // k of a stage
constexpr int kSideBytes = kBlockO * kBlockK / 2;
constexpr int kCodeBytes = 2 * kSideBytes;     // gate and up
constexpr int kABuffers = 4, kAColumn = 256, kAWidth = 64;  // widened codes in the tensor memory
constexpr int kScaleRing = 4;
constexpr int kWeightRing = 8;                 // units whose weights' scales are kept: more than the buffers reach ahead
constexpr int kSms = 148;
constexpr float kLog2e = 1.4426950408889634f, kLog2eRest = static_cast<float>(1.4426950408889634 - static_cast<double>(kLog2e));

enum XKind { kXBf16, kXF16, kXE4m3, kXI8 };

struct GatedArgs {
  const float* x_scale;       // or null
  const __half* w_scale;      // [2 f][k / group]
  void* out;
  long long ld_out;
  int* status;
  int x_group, m, f, k, group, out_dtype, gelu;
  int o_tiles, t_tiles, k_blocks;  // blocks of kBlockK
};

template <int X, int NT>
struct Shape {
  static constexpr bool kWide = X == kXBf16 || X == kXF16;    // 16-bit operands
  static constexpr int kXBytes = NT * kBlockK * (kWide ? 2 : 1);
  static constexpr int kStage = kCodeBytes + kXBytes;
  // partial sums of the groups of four tokens that a CTA finishes, from 2, 4 or 8 CTAs
  static constexpr int kParts = NT <= 64 ? 2 * (NT / 4) * kBlockO * 16 : 0;
  static constexpr int kRoom = 200 * 1024 - kParts;
  static constexpr int kStages = kRoom / kStage > 8 ? 8 : kRoom / kStage;
  static constexpr int kSmem = kStages * kStage + kParts + 1024;  // (up to 12 KB are declared beside it)
  static constexpr int kSideD = NT > 64 ? 1 : 2, kD = 2 * kSideD;  // accumulators in the tensor memory, of a side and in all
  static constexpr int kCols = NT / 2;                        // tokens of an adding warpgroup
  static constexpr int kSteps = kWide ? 16 : 32;              // k of an MMA
  // Registers a thread by role.  Wide tiles of 16-bit operands are best with 40 and 176 (4096 x 1536 x 6144 in bf16: 6 % less than with 48
  // and 168); the widening of 8-bit ones holds more constants (e4m3: 4 % less the other way), and narrow tiles wait for the widening (2 rows:
  // 5 % less).
  static constexpr bool kMoreSums = kWide && NT > 64;
  static constexpr int kLoadRegs = 40, kWidenRegs = kMoreSums ? 40 : 48, kAddRegs = kMoreSums ? 176 : 168;
  static_assert(kD * NT <= kAColumn, "tensor memory");
};

// two 32-bit values an instruction
typedef unsigned long long pair_t;

// D(tmem) (+)= A(tmem) * B(smem)^T
template <int X>
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
#define LB_TS(kind)                                                     \
  asm volatile(                                                         \
      "{\n\t.reg .pred p;\n\t"                                          \
      "setp.ne.b32 p, %4, 0;\n\t"                                       \
      "tcgen05.mma.cta_group::1.kind::" kind " [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) \
      : "memory")
  if constexpr (X == kXBf16 || X == kXF16) LB_TS("f16");
  else if constexpr (X == kXE4m3) LB_TS("f8f6f4");
  else LB_TS("i8");
#undef LB_TS
}
template <int X>
__host__ __device__ constexpr uint32_t idesc_of(int m, int n) {
  const uint32_t shape = static_cast<uint32_t>(n >> 3) << 17 | static_cast<uint32_t>(m >> 4) << 24;
  return X == kXBf16 ? shape | 1u << 4 | 1u << 7 | 1u << 10   // f32 sums, bf16
         : X == kXI8 ? shape | 2u << 4 | 1u << 7 | 1u << 10   // s32 sums, s8
                     : shape | 1u << 4;                        // f32 sums; format 0: f16, e4m3
}

// 32 lanes x 16 (or 8) columns, a lane's values from its registers
__device__ __forceinline__ void tmem_st(uint32_t at, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st(uint32_t at, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// 16 columns as pairs, and their wait in one statement
__device__ __forceinline__ void tmem_ld16(uint32_t at, pair_t (&r)[8]) {
  asm volatile(
      "{\n\t.reg .b32 t<16>;\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {t0,t1,t2,t3,t4,t5,t6,t7,t8,t9,t10,t11,t12,t13,t14,t15}, [%8];\n\t"
      "tcgen05.wait::ld.sync.aligned;\n\t"
      "mov.b64 %0, {t0, t1};\n\tmov.b64 %1, {t2, t3};\n\tmov.b64 %2, {t4, t5};\n\tmov.b64 %3, {t6, t7};\n\t"
      "mov.b64 %4, {t8, t9};\n\tmov.b64 %5, {t10, t11};\n\tmov.b64 %6, {t12, t13};\n\tmov.b64 %7, {t14, t15};\n\t}"
      : "=l"(r[0]), "=l"(r[1]), "=l"(r[2]), "=l"(r[3]), "=l"(r[4]), "=l"(r[5]), "=l"(r[6]), "=l"(r[7])
      : "r"(at)
      : "memory");
}

// Waits for a phase, with a limit of some 2.6 s (try_wait sleeps for up to the 20 us that it is given).  One look is in line.
constexpr int kPolls = 1 << 17;
__device__ __forceinline__ bool look(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(bar), "r"(parity), "r"(20000u)
      : "memory");
  return done != 0;
}
__device__ __forceinline__ bool wait_on(uint32_t bar, uint32_t parity) {
#pragma unroll 1
  for (int n = 0; n < kPolls; ++n)
    if (look(bar, parity)) return true;
  return false;
}
__device__ __forceinline__ bool wait_one(uint64_t* bar, uint32_t parity) {
  return look(smem_u32(bar), parity) || wait_on(smem_u32(bar), parity);
}
// by a whole warp: the same answer for every lane
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity) {
  if (__all_sync(0xffffffffu, look(smem_u32(bar), parity))) return true;
  return __all_sync(0xffffffffu, wait_on(smem_u32(bar), parity));
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t peer_address(uint32_t at, uint32_t rank) {
  uint32_t peer;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(at), "r"(rank));
  return peer;
}
__device__ __forceinline__ void peer_store(uint32_t at, pair_t a, pair_t b) {
  asm volatile("st.shared::cluster.v2.b64 [%0], {%1, %2};" ::"r"(at), "l"(a), "l"(b) : "memory");
}

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
__device__ __forceinline__ pair_t add2(pair_t a, pair_t b) {
  pair_t p;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(p) : "l"(a), "l"(b));
  return p;
}

template <typename H>
__device__ __forceinline__ uint32_t bits_of(H v) { return *reinterpret_cast<const uint32_t*>(&v); }

// 8 codes n (lowest bits first) as n - 8 in the operand's type and in their order.  The logic runs on a pipe of half rate
// that bounds the widening, so the constants are held in registers that the compiler cannot know (it made them anew for each use).
__device__ __forceinline__ uint32_t held(uint32_t v) {
  uint32_t r;
  asm volatile("mov.b32 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
__device__ __forceinline__ uint32_t look_up(uint32_t low, uint32_t high, uint32_t w) {  // (__byte_perm has no sign mode)
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(low), "r"(high), "r"(w));
  return r;
}
template <int X>
struct Widen;
// bf16, fp16: two codes under the exponent of 128 or 1024, where they count in ones, less 136 or 1032 (fp16: the odd
// codes as they lie, in sixteens, come down by the product).
template <>
struct Widen<kXBf16> {
  uint32_t mask = held(0x000f000fu), exponent = held(0x43004300u);
  __device__ __forceinline__ void operator()(uint32_t w, uint32_t* r) const {
    const __nv_bfloat162 bias = __floats2bfloat162_rn(136.0f, 136.0f);
    const uint32_t odd = w >> 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t pair = and_or(__byte_perm(w, odd, 0x0400 + 0x0101 * i), mask, exponent);
      r[i] = bits_of(__hsub2(*reinterpret_cast<const __nv_bfloat162*>(&pair), bias));
    }
  }
};
template <>
struct Widen<kXF16> {
  uint32_t mask = held(0x00f0000fu), exponent = held(0x64006400u);
  __device__ __forceinline__ void operator()(uint32_t w, uint32_t* r) const {
    const __half2 factor = __floats2half2_rn(1.0f, 0.0625f), bias = __floats2half2_rn(-1032.0f, -72.0f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t pair = and_or(__byte_perm(w, w, 0x0101 * i), mask, exponent);
      r[i] = bits_of(__hfma2(*reinterpret_cast<const __half2*>(&pair), factor, bias));
    }
  }
};
// e4m3: below 16 the bits count in steps of 2^-9 (a sign and four bits), so a code becomes the sign and the size of n - 8
// and the scale 2^9 larger.  A byte permute looks a code's lower three bits up in a table of eight, and where the fourth
// is set gives the looked-up byte's sign instead: 0 in these tables.
template <>
struct Widen<kXE4m3> {
  uint32_t b0 = held(0x05060708u), b1 = held(0x01020304u), a0 = held(0x03020100u), a1 = held(0x07060504u), low = held(0x7f7f7f7fu),
           top = held(0x80808080u);
  __device__ __forceinline__ uint32_t four(uint32_t w, uint32_t turned) const {
    const uint32_t below = look_up(b0, b1, w);       // n < 8: 8 - n
    const uint32_t above = look_up(a0, a1, turned);  // n >= 8: n - 8
    const uint32_t sign = look_up(low, low, w);      // n < 8: 0x7f
    return and_or(sign + sign, top, below | above);
  }
  __device__ __forceinline__ void operator()(uint32_t w, uint32_t* r) const {
    const uint32_t turned = w ^ 0x88888888u;
    r[0] = four(w, turned);
    r[1] = four(w >> 16, turned >> 16);
  }
};
// int8: 16 (n - 8), a code with its top bit turned as the byte's upper half
template <>
struct Widen<kXI8> {
  uint32_t high = held(0xf0f0f0f0u), top = held(0x80808080u);
  __device__ __forceinline__ uint32_t upper(uint32_t w) const {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(r) : "r"(w), "r"(high), "r"(top));  // (w & high) ^ top
    return r;
  }
  __device__ __forceinline__ void operator()(uint32_t w, uint32_t* r) const {
    const uint32_t odd = upper(w), even = upper(w << 4);
    r[0] = __byte_perm(even, odd, 0x5140);
    r[1] = __byte_perm(even, odd, 0x7362);
  }
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// g / (1 + exp(-z)): silu with z = g, gelu's tanh form with z = 2 sqrt(2 / pi) (g + 0.044715 g^3), as
// (1 + tanh(a)) / 2 = 1 / (1 + exp(-2 a)).  The rounding of the exponent z log2(e) costs |z| 2^-24 of the result, below 2^-17 where
// it is not 0 in 16 bits.  For 32-bit outputs (kFine) it comes back: the product's remainder, by a multiply-add, and that of log2(e)
// itself.  silu is then good to some 2^-21 of itself, gelu to that and z's own rounding, |z| 2^-21.  Both end at z = -87.3, where
// the reciprocal of 1 + e leaves the normal numbers and is flushed: what is below |g| 2^-126 becomes 0.  (Going on down to the smallest
// numbers by 2^64 / e, one more choice a value, made registers spill: 4096 x 1536 x 6144 149 us instead of 138, 32-bit outputs 165 instead of 143.)
template <bool kGelu, bool kFine>
__device__ __forceinline__ float activated(float g) {
  float z = g;
  if constexpr (kGelu) z = 1.5957691216057308f * fmaf(0.044715f * g * g, g, g);
  const float y = -kLog2e * z;
  float e = exp2_fast(y);
  if constexpr (kFine) {
    const float rest = fmaf(-kLog2e, z, -y) - z * kLog2eRest;
    e = fabsf(y) < 126.0f ? fmaf(e, rest * 0.6931471805599453f, e) : e;
  }
  return g * rcp_fast(1.0f + e);
}
__device__ __forceinline__ void put(float* at, float v) { *at = v; }
__device__ __forceinline__ void put(__nv_bfloat16* at, float v) { *at = __float2bfloat16_rn(v); }
__device__ __forceinline__ void put(__half* at, float v) { *at = __float2half_rn(v); }

template <int X, int NT, int SUBS>
__global__ void __launch_bounds__(kThreads, 1) gated_kernel(const GatedArgs a, const __grid_constant__ CUtensorMap w_map,
                                                            const __grid_constant__ CUtensorMap x_map) {
  using S = Shape<X, NT>;
  extern __shared__ unsigned char gated_raw[];
  unsigned char* smem = gated_raw + ((1024 - (smem_u32(gated_raw) & 1023)) & 1023);
  unsigned char* x_stages = smem;                             // [stage][half of k][token][128 bytes], swizzled
  unsigned char* c_stages = smem + S::kStages * S::kXBytes;   // [stage][side][row][64 bytes], swizzled
  unsigned char* parts = smem + S::kStages * S::kStage;
  __shared__ uint64_t c_full[S::kStages], c_empty[S::kStages], x_full[S::kStages], x_empty[S::kStages];
  __shared__ uint64_t a_full[kABuffers], a_empty[kABuffers], d_full[S::kD], d_empty[S::kD];
  __shared__ uint64_t s_full[kScaleRing], s_empty[kScaleRing];
  __shared__ __align__(16) float xs_s[kScaleRing][NT];
  __shared__ uint16_t ws_s[kWeightRing][SUBS][kBlockO];  // f16, by unit
  __shared__ uint32_t tmem_slot;

  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  uint32_t splits;
  asm volatile("mov.u32 %0, %cluster_nctarank;" : "=r"(splits));
  const int split = static_cast<int>(cluster_rank());
  if (tid == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(&c_full[i], 1);
      mbar_init(&c_empty[i], 8);
      mbar_init(&x_full[i], 1);
      mbar_init(&x_empty[i], 2);
    }
    for (int i = 0; i < kABuffers; ++i) {
      mbar_init(&a_full[i], 4);
      mbar_init(&a_empty[i], 1);
    }
    for (int i = 0; i < S::kD; ++i) {
      mbar_init(&d_full[i], 1);
      mbar_init(&d_empty[i], 8);
    }
    for (int i = 0; i < kScaleRing; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_empty[i], 8);
    }
    fence_barrier_init();
    tma_prefetch_desc(&w_map);
    tma_prefetch_desc(&x_map);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  // this CTA's blocks of K and its tiles (one, where K is dealt out)
  const int kb0 = a.k_blocks * split / static_cast<int>(splits), kb1 = a.k_blocks * (split + 1) / static_cast<int>(splits);
  const int first = blockIdx.x / splits, step = gridDim.x / splits, tiles = a.o_tiles * a.t_tiles;
  const bool grouped = a.x_group != 0;
  bool ok = true, joined = splits == 1 || NT > 64;
  if (!joined) cluster_arrive();

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::kLoadRegs));
    if (warp == 0 && lane == 0) {
      // ---------------- loads
      int st = 0;
      uint32_t ph = 0;
      int held = 0;  // stages that were requested
      for (int tile = first; tile < tiles && ok; tile += step) {
        const int o0 = tile % a.o_tiles * kBlockO, t0 = tile / a.o_tiles * NT;
        for (int kb = kb0; kb < kb1; ++kb) {
          ok = wait_one(&c_empty[st], ph ^ 1);
          if (!ok) break;
          mbar_arrive_expect_tx(&c_full[st], kCodeBytes);
          unsigned char* c = c_stages + st * kCodeBytes;
          asm volatile(
              "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(c)),
              "l"(reinterpret_cast<uint64_t>(&w_map)), "r"(smem_u32(&c_full[st])), "r"(kb * (kBlockK / 2)), "r"(o0)
              : "memory");
          asm volatile(
              "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
                  smem_u32(c + kSideBytes)),
              "l"(reinterpret_cast<uint64_t>(&w_map)), "r"(smem_u32(&c_full[st])), "r"(kb * (kBlockK / 2)), "r"(a.f + o0)
              : "memory");
          ok = wait_one(&x_empty[st], ph ^ 1);
          if (!ok) break;
          mbar_arrive_expect_tx(&x_full[st], S::kXBytes);
          unsigned char* x = x_stages + st * S::kXBytes;
#pragma unroll
          for (int h = 0; h < (S::kWide ? 2 : 1); ++h)
            asm volatile(
                "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
                    smem_u32(x + h * NT * 128)),
                "l"(reinterpret_cast<uint64_t>(&x_map)), "r"(smem_u32(&x_full[st])), "r"(kb * kBlockK + 64 * h), "r"(t0)
                : "memory");
          ++held;
          if (++st == S::kStages) {
            st = 0;
            ph ^= 1;
          }
        }
      }
      if (!ok) {  // the copies in flight, before the CTA may end: every stage's last request
        for (int i = 0; i < S::kStages && i < held; ++i) {
          st = st == 0 ? S::kStages - 1 : st - 1;
          if (st == S::kStages - 1) ph ^= 1;
          wait_one(&c_full[st], ph);
          wait_one(&x_full[st], ph);
        }
      }
    } else if (warp & 1) {
      // ---------------- MMAs, a warp a side: each one's waits and commits pass while the other's MMAs run.  The warp walks together
      // and one lane issues, so that descriptors and barriers stay uniform (a lane by itself took twice as long).
      const int side = warp >> 1;
      int st = 0, unit = side;
      uint32_t ph = 0;
      constexpr uint32_t idesc = idesc_of<X>(kBlockO, NT);
      const bool leader = elect_one();
      for (int tile = first; tile < tiles && ok; tile += step) {
        for (int kb = kb0; kb < kb1 && ok; ++kb) {
          const int ab = unit & (kABuffers - 1);
          ok = wait_warp(&x_full[st], ph) && wait_warp(&a_full[ab], unit / kABuffers & 1);
          const uint64_t x = smem_desc_k128(smem_u32(x_stages + st * S::kXBytes));
          const uint32_t wide = tmem + kAColumn + ab * kAWidth;
#pragma unroll
          for (int sub = 0; sub < SUBS; ++sub) {
            const int turn = unit / 2 * SUBS + sub, db = side * S::kSideD + (turn & (S::kSideD - 1));
            ok = ok && wait_warp(&d_empty[db], (turn / S::kSideD & 1) ^ 1);
            if (!ok) break;
            tc_fence_after();
            const uint32_t d = tmem + db * NT;
            constexpr int kPer = kBlockK / SUBS / S::kSteps;  // MMAs of a group
            if (leader) {
#pragma unroll
              for (int i = 0; i < kPer; ++i) {
                const int j = sub * kPer + i;  // of the block: 32 bytes of a row of x, 8 columns of the codes
                const int at = S::kWide ? (j >> 2) * (NT * 128) + (j & 3) * 32 : j * 32;
                umma_ts<X>(d, wide + j * 8, x + (at >> 4), idesc, i > 0);
              }
              umma_commit(&d_full[db]);
              if (sub == SUBS - 1) {
                umma_commit(&a_empty[ab]);
                umma_commit(&x_empty[st]);
              }
            }
            __syncwarp();
          }
          unit += 2;
          if (++st == S::kStages) {
            st = 0;
            ph ^= 1;
          }
        }
      }
    } else if (warp == 2 && grouped) {
      // ---------------- x's scales of a block's group
      int ring = 0;
      uint32_t ph = 0;
      const int groups = a.k / a.x_group;
      for (int tile = first; tile < tiles && ok; tile += step) {
        const int t0 = tile / a.o_tiles * NT;
        for (int kb = kb0; kb < kb1; ++kb) {
          float v[NT / 32];
          const int g = kb * kBlockK / a.x_group;
#pragma unroll
          for (int i = 0; i < NT / 32; ++i) {
            const int t = t0 + 32 * i + lane;
            v[i] = t < a.m ? a.x_scale[static_cast<long long>(t) * groups + g] : 0.0f;
          }
          ok = wait_warp(&s_empty[ring], ph ^ 1);
          if (!ok) break;
#pragma unroll
          for (int i = 0; i < NT / 32; ++i) xs_s[ring][32 * i + lane] = v[i];
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_full[ring]);
          if (++ring == kScaleRing) {
            ring = 0;
            ph ^= 1;
          }
        }
      }
    }
    __syncwarp();
  } else if (warp < kFirstAdder) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::kWidenRegs));
    // ---------------- codes -> operands, a warpgroup a side; a lane has a row, and brings the row's scales too
    const int side = (warp - 4) >> 2, row = 32 * (warp & 3) + lane, groups = a.k / a.group;
    const Widen<X> widen;
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // 32 lanes, in the address's upper half
    int st = 0, unit = side;
    uint32_t ph = 0;
    for (int tile = first; tile < tiles && ok; tile += step) {
      const int o = tile % a.o_tiles * kBlockO + row;
      const bool there = o < a.f;
      const uint16_t* scale = reinterpret_cast<const uint16_t*>(a.w_scale) + static_cast<long long>(there ? side * a.f + o : 0) * groups;
      uint16_t next[SUBS];
      const auto fetch = [&](int kb) {
#pragma unroll
        for (int i = 0; i < SUBS; ++i) next[i] = there && kb < kb1 && kb * SUBS + i < groups ? scale[kb * SUBS + i] : 0;
      };
      fetch(kb0);
      for (int kb = kb0; kb < kb1; ++kb) {
        const int ab = unit & (kABuffers - 1);
        // the ring's place is free: MMAs of the unit four back are over, so the adders have left all before the last two (or
        // four) of them.  They read it after those of this unit, which come after this warp's arrival.
        ok = wait_warp(&c_full[st], ph) && wait_warp(&a_empty[ab], (unit / kABuffers & 1) ^ 1);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int i = 0; i < SUBS; ++i) ws_s[unit & (kWeightRing - 1)][i][row] = next[i];
        fetch(kb + 1);
        constexpr int kRegs = S::kWide ? 16 : 8;  // of 32 codes
        uint32_t wide = tmem + lanes + kAColumn + ab * kAWidth;
        const unsigned char* c = c_stages + st * kCodeBytes + side * kSideBytes + row * 64;
        uint4 raw[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) raw[i] = *reinterpret_cast<const uint4*>(c + ((i ^ ((row >> 1) & 3)) << 4));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t r[kRegs];
          widen(raw[i].x, r);
          widen(raw[i].y, r + kRegs / 4);
          widen(raw[i].z, r + kRegs / 2);
          widen(raw[i].w, r + kRegs * 3 / 4);
          tmem_st(wide + i * kRegs, r);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&a_full[ab]);
          mbar_arrive(&c_empty[st]);
        }
        unit += 2;
        if (++st == S::kStages) {
          st = 0;
          ph ^= 1;
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::kAddRegs));
    // ---------------- sums and results
    const int half = (warp - kFirstAdder) >> 2, row = 32 * (warp & 3) + lane;
    const uint32_t from = tmem + (static_cast<uint32_t>(warp & 3) << 21) + half * S::kCols;
    int turn = 0, ring = 0, unit = 0;
    uint32_t rph = 0;
    constexpr float kUnit = X == kXE4m3 ? 512.0f : X == kXI8 ? 0.0625f : 1.0f;  // of the widened codes
    for (int tile = first; tile < tiles && ok; tile += step) {
      const int o = tile % a.o_tiles * kBlockO + row, t0 = tile / a.o_tiles * NT + half * S::kCols;
      // 8-bit x with a scale a row: a lane keeps those of two tokens for the end
      float row_scale[2] = {1.0f, 1.0f};
      if (!S::kWide && !grouped) {
#pragma unroll
        for (int i = 0; i < 2; ++i) row_scale[i] = 32 * i + lane < S::kCols && t0 + 32 * i + lane < a.m ? a.x_scale[t0 + 32 * i + lane] : 0.0f;
      }
      pair_t acc[2][S::kCols / 2];
#pragma unroll
      for (int j = 0; j < S::kCols / 2; ++j) acc[0][j] = acc[1][j] = 0;
      for (int kb = kb0; kb < kb1 && ok; ++kb) {
        if (grouped) ok = wait_warp(&s_full[ring], rph);
#pragma unroll
        for (int sub = 0; sub < SUBS; ++sub) {
#pragma unroll
          for (int side = 0; side < 2; ++side) {
            const int db = side * S::kSideD + (turn & (S::kSideD - 1));
            ok = ok && wait_warp(&d_full[db], turn / S::kSideD & 1);
            if (!ok) break;
            tc_fence_after();
            const float s = __half2float(__ushort_as_half(ws_s[(unit + side) & (kWeightRing - 1)][sub][row])) * kUnit;
            const pair_t s2 = pair_of(s, s);
            const uint32_t d = from + db * NT;
#pragma unroll
            for (int j0 = 0; j0 < S::kCols; j0 += 16) {
              pair_t r[8];
              [[maybe_unused]] ulonglong2 xs{};  // x's scales of four tokens
              tmem_ld16(d + j0, r);
              if (j0 + 16 == S::kCols) {  // the sums are in registers
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&d_empty[db]);
              }
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                pair_t v = r[j];
                if constexpr (!S::kWide) {
                  if (grouped && j % 2 == 0) xs = *reinterpret_cast<const ulonglong2*>(&xs_s[ring][half * S::kCols + j0 + 2 * j]);
                }
                if constexpr (X == kXI8) {  // sums below 2^22, under the exponent of 3 * 2^22
                  float lo, hi;
                  unpair(v, lo, hi);
                  v = add2(pair_of(__uint_as_float(0x4b400000u + __float_as_uint(lo)), __uint_as_float(0x4b400000u + __float_as_uint(hi))),
                           pair_of(-12582912.0f, -12582912.0f));
                }
                if constexpr (!S::kWide) {
                  if (grouped) v = mul2(v, j % 2 ? xs.y : xs.x);
                }
                acc[side][j0 / 2 + j] = fma2(v, s2, acc[side][j0 / 2 + j]);
              }
            }
          }
          ++turn;
        }
        unit += 2;
        if (grouped) {
          __syncwarp();
          if (lane == 0 && ok) mbar_arrive(&s_empty[ring]);
          if (++ring == kScaleRing) {
            ring = 0;
            rph ^= 1;
          }
        }
      }
      if (!ok) break;
      if (splits == 1) {
        const int live = o < a.f ? a.m - t0 : 0;  // tokens from t0 on
        const long long pitch = a.ld_out * (a.out_dtype == LB_F32 ? 4 : 2);
        unsigned char* at = static_cast<unsigned char*>(a.out) + t0 * pitch + static_cast<long long>(o) * (a.out_dtype == LB_F32 ? 4 : 2);
        // up to 32 tokens are computed before they are stored, without a branch between them.  (A loop over turns, with the rest moving up
        // to the first registers, took 18 us more of 163 for 4096 rows of 1536 x 6144.)
        const bool whole = tile % a.o_tiles * kBlockO + kBlockO <= a.f && t0 + S::kCols <= a.m;
        const auto turn = [&](auto gelu, auto type) {
          using Out = decltype(type);
          constexpr int kTurn = S::kCols % 32 == 0 ? 32 : 16;
#pragma unroll
          for (int j0 = 0; j0 < S::kCols; j0 += kTurn) {
            float v[kTurn];
#pragma unroll
            for (int j = 0; j < kTurn; ++j) {
              float g[2], u[2];
              unpair(acc[0][(j0 + j) / 2], g[0], g[1]);
              unpair(acc[1][(j0 + j) / 2], u[0], u[1]);
              float gate = g[j & 1], up = u[j & 1];
              if (!S::kWide && !grouped) {
                const float xs = __shfl_sync(0xffffffffu, j0 + j >= 32 ? row_scale[1] : row_scale[0], (j0 + j) & 31);
                gate *= xs;
                up *= xs;
              }
              v[j] = activated<decltype(gelu)::value, sizeof(Out) == 4>(gate) * up;
            }
            if (whole) {
#pragma unroll
              for (int j = 0; j < kTurn; ++j) put(reinterpret_cast<Out*>(at + j * pitch), v[j]);
            } else {
#pragma unroll
              for (int j = 0; j < kTurn; ++j)
                if (j0 + j < live) put(reinterpret_cast<Out*>(at + j * pitch), v[j]);
            }
            at += kTurn * pitch;
          }
        };
        const auto typed = [&](auto gelu) {
          if (a.out_dtype == LB_F32) turn(gelu, float{});
          else if (a.out_dtype == LB_BF16) turn(gelu, __nv_bfloat16{});
          else turn(gelu, __half{});
        };
        if (a.gelu) typed(std::true_type{});
        else typed(std::false_type{});
      } else {
        // the tile's four tokens from 4 q on are finished by CTA q % splits, as its group q / splits: [source][side][group][row][4]
        // (stores of 16 bytes: a warp's store over the cluster takes some 27 cycles whatever its width)
        if (!joined) {  // (the others have begun)
          cluster_wait();
          joined = true;
        }
        if constexpr (NT <= 64) {
          const int n = static_cast<int>(splits), own = (NT / 4 + n - 1) / n, first_q = half * S::kCols / 4;
          const int live = (min(S::kCols, a.m - t0) + 3) / 4;
          int to = first_q % n, i = first_q / n;
          const uint32_t at = smem_u32(parts) + (split * 2 * own * kBlockO + row) * 16;
#pragma unroll
          for (int q = 0; q < S::kCols / 4; ++q) {
            if (q < live) {
              const uint32_t peer = peer_address(at + i * kBlockO * 16, to);
              peer_store(peer, acc[0][2 * q], acc[0][2 * q + 1]);
              peer_store(peer + own * kBlockO * 16, acc[1][2 * q], acc[1][2 * q + 1]);
            }
            if (++to == n) {
              to = 0;
              ++i;
            }
          }
        }
      }
    }
  }
  if (!ok && a.status) atomicOr(a.status, static_cast<int>(kStatusWaitTimeout));
  __syncwarp();
  if (NT <= 64 && splits > 1) {
    if (!joined) cluster_wait();
    cluster_arrive();
    cluster_wait();
    if (warp >= kFirstAdder) {
      const int row = 32 * (warp & 3) + lane, o = first % a.o_tiles * kBlockO + row, t0 = first / a.o_tiles * NT;
      const int n = static_cast<int>(splits), own = (NT / 4 + n - 1) / n;
      const float4* part = reinterpret_cast<const float4*>(parts) + row;
      for (int i = (warp - kFirstAdder) >> 2; i < own; i += 2) {
        const int j = 4 * (split + i * n), t = t0 + j;
        if (j >= NT || t >= a.m) break;
        float g[4] = {0.0f, 0.0f, 0.0f, 0.0f}, u[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int r = 0; r < n; ++r) {
          const float4 x = part[(r * 2 * own + i) * kBlockO], y = part[((r * 2 + 1) * own + i) * kBlockO];
          g[0] += x.x, g[1] += x.y, g[2] += x.z, g[3] += x.w;
          u[0] += y.x, u[1] += y.y, u[2] += y.z, u[3] += y.w;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (o >= a.f || t + e >= a.m) break;
          if (!S::kWide && !grouped) {
            const float xs = a.x_scale[t + e];
            g[e] *= xs;
            u[e] *= xs;
          }
          const float v = (a.gelu ? activated<true, true>(g[e]) : activated<false, true>(g[e])) * u[e];
          const long long to = (t + e) * a.ld_out + o;
          if (a.out_dtype == LB_F32) put(static_cast<float*>(a.out) + to, v);
          else if (a.out_dtype == LB_BF16) put(static_cast<__nv_bfloat16*>(a.out) + to, v);
          else put(static_cast<__half*>(a.out) + to, v);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int X, int NT, int SUBS>
cudaError_t launch(const GatedArgs& a, int splits, const CUtensorMap& w_map, const CUtensorMap& x_map, cudaStream_t s) {
  using S = Shape<X, NT>;
  const auto kernel = gated_kernel<X, NT, SUBS>;
  static std::atomic<unsigned long long> done{0};
  static std::atomic<int> registers{0};
  cudaError_t e = ensure_smem(done, reinterpret_cast<const void*>(kernel), S::kSmem);
  if (e != cudaSuccess) return e;
  if (registers.load(std::memory_order_relaxed) == 0) {
    // the five warpgroups' shares of the registers have to fit what the block is launched with: more would be waited for without end
    cudaFuncAttributes f;
    if ((e = cudaFuncGetAttributes(&f, reinterpret_cast<const void*>(kernel))) != cudaSuccess) return e;
    registers.store(f.numRegs, std::memory_order_relaxed);
  }
  if (registers.load(std::memory_order_relaxed) * 5 < S::kLoadRegs + 2 * S::kWidenRegs + 2 * S::kAddRegs) return cudaErrorInvalidConfiguration;
  const int tiles = a.o_tiles * a.t_tiles;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = static_cast<unsigned>(splits > 1 ? tiles * splits : tiles < kSms ? tiles : kSms);
  cfg.blockDim = kThreads;
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {static_cast<unsigned>(splits), 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kernel, a, w_map, x_map);
  return e == cudaSuccess ? cudaGetLastError() : e;
}
template <int X, int NT>
cudaError_t launch(const GatedArgs& a, int splits, const CUtensorMap& w_map, const CUtensorMap& x_map, cudaStream_t s) {
  if (a.group == 128) return launch<X, NT, 1>(a, splits, w_map, x_map, s);
  if (a.group == 64) return launch<X, NT, 2>(a, splits, w_map, x_map, s);
  return launch<X, NT, 4>(a, splits, w_map, x_map, s);
}
template <int X>
cudaError_t launch(const GatedArgs& a, int nt, int splits, const CUtensorMap& w_map, const CUtensorMap& x_map, cudaStream_t s) {
  if (nt == 32) return launch<X, 32>(a, splits, w_map, x_map, s);
  if (nt == 64) return launch<X, 64>(a, splits, w_map, x_map, s);
  if (nt == 96) return launch<X, 96>(a, splits, w_map, x_map, s);
  return launch<X, 128>(a, splits, w_map, x_map, s);
}

}  // namespace
}  // namespace lb

extern "C" int lb_op_w4_gated(const void* x, int64_t x_ld, int x_dtype, const float* x_scale, int x_group, int m,
                              const void* codes, const void* w_scale, int group, int ffn, int k, int activation, void* out,
                              int64_t ld_out, int out_dtype, int32_t* status, void* stream) {
  using namespace lb;
  if (!x || !codes || !w_scale || !out || m < 1 || ffn < 1 || k < 1 || x_ld < k || ld_out < ffn || activation < 0 || activation > 1)
    return LB_ERR_INVALID_ARGUMENT;
  if ((group != 32 && group != 64 && group != 128) || k % group != 0) return LB_ERR_INVALID_ARGUMENT;
  const bool eight = x_dtype == LB_E4M3 || x_dtype == LB_I8;
  if ((!eight && x_dtype != LB_BF16 && x_dtype != LB_F16) || eight != (x_scale != nullptr)) return LB_ERR_INVALID_ARGUMENT;
  if (x_group < 0 || (x_group && (!eight || x_group % 128 != 0 || k % x_group != 0))) return LB_ERR_INVALID_ARGUMENT;
  if (out_dtype != LB_F32 && out_dtype != LB_BF16 && out_dtype != LB_F16) return LB_ERR_INVALID_ARGUMENT;
  const int64_t size = eight ? 1 : 2;
  if (reinterpret_cast<uintptr_t>(codes) % 16 != 0 || reinterpret_cast<uintptr_t>(x) % 16 != 0 || (m > 1 && x_ld * size % 16 != 0))
    return LB_ERR_INVALID_ARGUMENT;
  if (ffn > (1 << 24) || m > (1 << 24) || x_ld > (1ll << 36)) return LB_ERR_CAPACITY;
  const int64_t out_size = out_dtype == LB_F32 ? 4 : 2;
  if (rows_meet({x, x_ld * size, 0, m, 1, k * size}, {out, ld_out * out_size, 0, m, 1, ffn * out_size})) return LB_ERR_INVALID_ARGUMENT;
  GatedArgs a{x_scale, static_cast<const __half*>(w_scale), out, ld_out, status, x_group == k ? 0 : x_group, m, ffn, k, group, out_dtype,
              activation, 0, 0, 0};
  a.o_tiles = (ffn + kBlockO - 1) / kBlockO;
  a.k_blocks = (k + kBlockK - 1) / kBlockK;
  // The width of a tile and the dealing out of K by an estimate of the time in tenths of a microsecond: a wave of tiles takes 4
  // us and for each block of K 0.67, 0.7, 0.85 or 1 at 32, 64, 96 or 128 tokens (1536 x 6144 in groups of 128, bf16, where all
  // five were measured: 128 rows as 48 tiles of 128 tokens take 1.3 times as long as 96 of 64; finer groups and 8-bit x cost more at
  // each width, which the estimate leaves out).  K is dealt out where all clusters fit the GPU at once: 2 rows of 1536 x
  // 6144 take 1.4 times as long whole as in clusters of two, and 1.5 times in clusters of three, not all of which fit.
  int nt = 0, splits = 1;
  long long best = 0;
  for (const int width : {32, 64, 96, 128}) {
    const long long t_tiles = (m + width - 1) / width, tiles = a.o_tiles * t_tiles;
    const int split = width > 64 ? 1 : tiles <= 16 && a.k_blocks >= 8 ? 8 : tiles <= 32 && a.k_blocks >= 4 ? 4 : tiles <= 74 && a.k_blocks >= 2 ? 2 : 1;
    const long long time = (tiles * split + kSms - 1) / kSms * (40 + (width == 32 ? 67 : width == 64 ? 70 : width == 96 ? 85 : 100) * ((a.k_blocks + split - 1) / split) / 10);
    if (nt == 0 || time < best) {
      nt = width;
      splits = split;
      best = time;
    }
  }
  if (static_cast<long long>(a.o_tiles) * ((m + nt - 1) / nt) > 0x3fffffffll) return LB_ERR_CAPACITY;
  a.t_tiles = (m + nt - 1) / nt;
  CUtensorMap w_map, x_map;
  const int64_t x_row = m > 1 ? x_ld * size : (static_cast<int64_t>(k) * size + 15) / 16 * 16;
  if (make_tensor_map_u8(&w_map, codes, k / 2, 2ull * ffn, 64, kBlockO) != 0 ||
      make_tensor_map_2d(&x_map, x, static_cast<int>(size), k, m, x_row, eight ? 128 : 64, nt, true, x_dtype == LB_F16) != 0)
    return LB_ERR_CUDA;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (x_dtype == LB_BF16) e = launch<kXBf16>(a, nt, splits, w_map, x_map, s);
  else if (x_dtype == LB_F16) e = launch<kXF16>(a, nt, splits, w_map, x_map, s);
  else if (x_dtype == LB_E4M3) e = launch<kXE4m3>(a, nt, splits, w_map, x_map, s);
  else e = launch<kXI8>(a, nt, splits, w_map, x_map, s);
  return e == cudaSuccess ? LB_OK : LB_ERR_CUDA;
}
