// Page plans on the GPU: block tables, token positions and cache slots of one
// step from the request lengths, and their commit and release.
//
// Row i adds new_i tokens to a session that holds L0_i.  With P tokens a page it
// has p0_i = ceil(L0_i / P) pages and needs p1_i - p0_i more, p1_i = ceil((L0_i +
// new_i) / P).  The j-th of them is the (rank_i + j)-th lowest free page, rank_i =
// sum of the needs of the rows before it: the rule of the session packer (the
// k-th new row gets the k-th lowest free slot), applied to pages.
//
// plan_kernel is one launch without any exchange between CTAs: each CTA takes the
// prefix sums over all rows and over the free bits of the whole pool for itself
// (8 bytes a row and a bit a page, both small beside what is written) and then
// fills its share of the row tables and of the tokens.  A second launch, or a
// wait of CTAs for one another, would cost more than the repeated sums.  The floor is a launch (2048 rows
// move 2.5 MB, 0.4 us at the copy rate); 16 rows take 6.8 us inside a graph, the chain of the two scans, 2048 rows 12 us.
// A commit is two launches (the check, then the writing): some 6 us.
#include "../../include/listener_b200.h"
#include "common.cuh"

namespace lb {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kMaxPlanRows = 8192;
constexpr int kMaxPlanSessions = 262144;
constexpr int kMaxPlanTokens = 1 << 26;  // 8192 rows of them stay below 2^40 (the packed sums)
constexpr int kStatusPagesExhausted = LB_DEV_PAGES_EXHAUSTED;

// Exclusive prefix sum over the block's threads; *total is the sum.
__device__ long long block_scan(long long v, long long* total, long long* sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) sh[warp] = x;
  __syncthreads();
  if (warp == 0) {
    long long w = sh[lane];  // kPlanThreads / 32 == 32 warps
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    sh[lane] = w;
  }
  __syncthreads();
  const long long before = warp > 0 ? sh[warp - 1] : 0;
  *total = sh[31];
  __syncthreads();
  return before + x - v;
}

struct PlanArgs {
  int n, n_sessions, max_pages, n_pages, page_tokens, max_tokens;
  const int *sessions, *new_tokens, *tables, *lengths;
  const unsigned* used;
  int *row_tables, *kv_len, *cu_tokens, *positions, *token_rows, *status;
  long long* slots;
  int* planned;  // a copy of the sessions, or null
};

__device__ __forceinline__ unsigned free_bits(const PlanArgs& a, int word) {
  unsigned w = ~a.used[word];
  const int left = a.n_pages - word * 32;
  if (left < 32) w &= (1u << left) - 1u;
  return w;
}

// The k-th lowest free page: the thread chunk of the bitmap whose prefix count
// holds it, then its word, then its bit.
__device__ int select_free(const PlanArgs& a, const int* free_before, int words_each, int k) {
  int lo = 0, hi = kPlanThreads - 1;
  while (lo < hi) {  // last chunk with free_before[chunk] <= k
    const int mid = (lo + hi + 1) >> 1;
    if (free_before[mid] <= k) lo = mid; else hi = mid - 1;
  }
  int left = k - free_before[lo];
  const int words = (a.n_pages + 31) / 32;
  const int end = min(words, (lo + 1) * words_each);
  for (int w = lo * words_each; w < end; ++w) {
    unsigned bits = free_bits(a, w);
    const int c = __popc(bits);
    if (left < c) {
      while (left-- > 0) bits &= bits - 1;
      return w * 32 + __ffs(bits) - 1;
    }
    left -= c;
  }
  return -1;  // not reached: the plan is refused when the pages run out
}

__global__ void __launch_bounds__(kPlanThreads) plan_kernel(PlanArgs a) {
  extern __shared__ int plan_smem[];
  int* cu = plan_smem;               // n + 1: tokens before the row
  int* rank = cu + a.n + 1;          // n: pages needed by the rows before it
  int* before = rank + a.n;          // n: tokens the session held
  int* free_before = before + a.n;   // kPlanThreads
  unsigned* seen = reinterpret_cast<unsigned*>(free_before + kPlanThreads);  // a bit per session
  __shared__ long long sh[32];
  __shared__ int bad;
  const int tid = threadIdx.x, P = a.page_tokens;
  if (tid == 0) bad = 0;
  for (int i = tid; i < (a.n_sessions + 31) / 32; i += kPlanThreads) seen[i] = 0u;
  __syncthreads();

  // rows: thread t has the rows [t * each, (t + 1) * each); both sums in one scan
  // (tokens in the low 40 bits, pages above them: a sum of pages that does not fit
  // there comes with a sum of tokens that is refused)
  const int each = (a.n + kPlanThreads - 1) / kPlanThreads;
  const int r0 = min(a.n, tid * each), r1 = min(a.n, r0 + each);
  long long mine = 0;
  int wrong = 0;
  for (int r = r0; r < r1; ++r) {
    const int s = a.sessions[r], add = a.new_tokens[r];
    int held = 0;
    if (s < 0 || s >= a.n_sessions) {
      wrong |= LB_DEV_BAD_HANDLE;
    } else {
      if (atomicOr(&seen[s >> 5], 1u << (s & 31)) >> (s & 31) & 1u) wrong |= LB_DEV_DUPLICATE_ROW;
      held = a.lengths[s];
    }
    const long long room = static_cast<long long>(a.max_pages) * P;
    if (add < 0 || add > a.max_tokens || held < 0 || held > room) {
      wrong |= LB_DEV_BAD_ROW_COUNT;
    } else if (held + static_cast<long long>(add) > room) {
      wrong |= kStatusPagesExhausted;
    } else {
      const int need = (held + add + P - 1) / P - (held + P - 1) / P;
      mine += add + (static_cast<long long>(need) << 40);
    }
    before[r] = held;
  }
  if (wrong) atomicOr(&bad, wrong);
  long long total;
  long long run = block_scan(mine, &total, sh);
  const long long tokens = total & ((1ll << 40) - 1);
  const long long need_all = total >> 40;
  if (bad == 0) {  // (no early refusal past the scan's barriers: `bad` is final here)
    for (int r = r0; r < r1; ++r) {
      const int held = before[r], add = a.new_tokens[r];
      cu[r] = static_cast<int>(run & ((1ll << 40) - 1));
      rank[r] = static_cast<int>(run >> 40);
      run += add + (static_cast<long long>((held + add + P - 1) / P - (held + P - 1) / P) << 40);
    }
    if (tid == 0) cu[a.n] = static_cast<int>(tokens);
  }

  // free pages before each thread's chunk of the bitmap
  const int words = (a.n_pages + 31) / 32;
  const int words_each = (words + kPlanThreads - 1) / kPlanThreads;
  int count = 0;
  if (need_all > 0)
    for (int w = tid * words_each; w < min(words, (tid + 1) * words_each); ++w) count += __popc(free_bits(a, w));
  long long free_all;
  free_before[tid] = static_cast<int>(block_scan(count, &free_all, sh));
  int status = bad;
  if (status == 0 && tokens > a.max_tokens) status = LB_DEV_BAD_ROW_COUNT;
  if (status == 0 && need_all > free_all) status = kStatusPagesExhausted;
  __syncthreads();
  if (blockIdx.x == 0 && tid == 0) *a.status = status;

  const long long stride = static_cast<long long>(gridDim.x) * kPlanThreads;
  const long long first = static_cast<long long>(blockIdx.x) * kPlanThreads + tid;
  for (long long i = first; i <= a.n; i += stride) {
    a.cu_tokens[i] = status ? 0 : cu[i];
    if (i < a.n) {
      a.kv_len[i] = status ? 0 : before[i] + (cu[i + 1] - cu[i]);
      if (a.planned) a.planned[i] = a.sessions[i];
    }
  }
  for (long long i = first; i < static_cast<long long>(a.n) * a.max_pages; i += stride) {
    const int r = static_cast<int>(i / a.max_pages), c = static_cast<int>(i - static_cast<long long>(r) * a.max_pages);
    int page = -1;
    if (status == 0) {
      const int p0 = (before[r] + P - 1) / P, p1 = (before[r] + (cu[r + 1] - cu[r]) + P - 1) / P;
      if (c < p0) page = a.tables[static_cast<long long>(a.sessions[r]) * a.max_pages + c];
      else if (c < p1) page = select_free(a, free_before, words_each, rank[r] + c - p0);
    }
    a.row_tables[i] = page;
  }
  for (long long t = first; t < a.max_tokens; t += stride) {
    int row = -1, pos = -1;
    long long slot = -1;
    if (status == 0 && t < tokens) {
      int lo = 0, hi = a.n - 1;  // last row with cu[row] <= t (rows without tokens end where they begin)
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (cu[mid] <= t) lo = mid; else hi = mid - 1;
      }
      row = lo;
      pos = before[row] + static_cast<int>(t) - cu[row];
      const int c = pos / P, p0 = (before[row] + P - 1) / P;
      const int page = c < p0 ? a.tables[static_cast<long long>(a.sessions[row]) * a.max_pages + c]
                              : select_free(a, free_before, words_each, rank[row] + c - p0);
      slot = static_cast<long long>(page) * P + (pos - c * P);
    }
    a.slots[t] = slot;
    a.positions[t] = pos;
    a.token_rows[t] = row;
  }
}

// Does the plan still fit the directory?  One warp a row, before anything is written: the session must hold the tokens
// and pages that it held when the plan was made, and the pages it would get must still be free.  (Another launch
// than the commit's, so that no row is installed unless all fit.)
__global__ void check_kernel(int n, const int* sessions, int n_sessions, int max_pages, int n_pages, int P,
                             const int* row_tables, const int* kv_len, const int* cu_tokens, const int* tables,
                             const int* lengths, const unsigned* used, int* status) {
  const int r = (blockIdx.x * blockDim.x + threadIdx.x) >> 5, lane = threadIdx.x & 31;
  if (r >= n) return;
  const int s = sessions[r];
  bool stale = s < 0 || s >= n_sessions;
  if (!stale) {
    const long long held = lengths[s], now = kv_len[r], room = static_cast<long long>(max_pages) * P;
    stale = held < 0 || now < held || now > room || (cu_tokens && now - held != static_cast<long long>(cu_tokens[r + 1]) - cu_tokens[r]);
    if (!stale) {
      const int p0 = static_cast<int>((held + P - 1) / P), p1 = static_cast<int>((now + P - 1) / P);
      for (int c = lane; c < p1; c += 32) {
        const int page = row_tables[static_cast<long long>(r) * max_pages + c];
        stale = stale || (c < p0 ? page != tables[static_cast<long long>(s) * max_pages + c]
                                 : page < 0 || page >= n_pages || (used[page >> 5] >> (page & 31) & 1u));
      }
    }
  }
  // (a refused plan has its reason there already, and is all the same not installed)
  if (__any_sync(0xffffffffu, stale) && lane == 0 && *static_cast<volatile int*>(status) == 0) atomicOr(status, LB_DEV_STALE_COMMIT);
}

// One warp a row: the pages past the held ones become the session's.
__global__ void commit_kernel(int n, const int* sessions, int n_sessions, int max_pages, int n_pages, int P,
                              const int* row_tables, const int* kv_len, const int* status, int* tables,
                              int* lengths, unsigned* used) {
  const int r = (blockIdx.x * blockDim.x + threadIdx.x) >> 5, lane = threadIdx.x & 31;
  if (r >= n || *status != 0) return;
  const int s = sessions[r];
  if (s < 0 || s >= n_sessions) return;
  const int p0 = (lengths[s] + P - 1) / P, p1 = min(max_pages, (kv_len[r] + P - 1) / P);
  for (int c = p0 + lane; c < p1; c += 32) {
    const int page = row_tables[static_cast<long long>(r) * max_pages + c];
    tables[static_cast<long long>(s) * max_pages + c] = page;
    if (page >= 0 && page < n_pages) atomicOr(&used[page >> 5], 1u << (page & 31));
  }
  __syncwarp();
  if (lane == 0) lengths[s] = kv_len[r];
}

__global__ void release_kernel(int n, const int* sessions, int n_sessions, int max_pages, int n_pages, int P,
                               int* tables, int* lengths, unsigned* used, int* status) {
  const int r = (blockIdx.x * blockDim.x + threadIdx.x) >> 5, lane = threadIdx.x & 31;
  if (r >= n) return;
  const int s = sessions[r];
  if (s < 0 || s >= n_sessions) {
    if (lane == 0) atomicOr(status, static_cast<int>(LB_DEV_BAD_HANDLE));
    return;
  }
  const int held = min(max_pages, (lengths[s] + P - 1) / P);
  for (int c = lane; c < held; c += 32) {
    int* at = &tables[static_cast<long long>(s) * max_pages + c];
    const int page = *at;
    if (page >= 0 && page < n_pages) atomicAnd(&used[page >> 5], ~(1u << (page & 31)));
    *at = -1;
  }
  __syncwarp();
  if (lane == 0) lengths[s] = 0;
}

bool bad_shape(int n, int n_sessions, int max_pages, int n_pages, int page_tokens) {
  return n < 1 || n_sessions < 1 || n_sessions > kMaxPlanSessions || max_pages < 1 || n_pages < 1 ||
         page_tokens < 16 || page_tokens > 256 || page_tokens % 16 != 0 ||
         static_cast<long long>(max_pages) * page_tokens > 0x7fffffffll;
}

}  // namespace
}  // namespace lb

extern "C" {

int lb_plan_step(int n, const int32_t* sessions, const int32_t* new_tokens, int n_sessions, int max_pages,
                 int n_pages, int page_tokens, const int32_t* tables, const int32_t* lengths,
                 const int32_t* used, int max_tokens, int32_t* row_tables, int32_t* kv_len,
                 int32_t* cu_tokens, int64_t* slots, int32_t* positions, int32_t* token_rows,
                 int32_t* planned_sessions, int32_t* status, void* stream) {
  using namespace lb;
  if (bad_shape(n, n_sessions, max_pages, n_pages, page_tokens) || n > kMaxPlanRows || max_tokens < 1 || max_tokens > kMaxPlanTokens)
    return LB_ERR_INVALID_ARGUMENT;
  if (!sessions || !new_tokens || !tables || !lengths || !used || !row_tables || !kv_len || !cu_tokens || !slots ||
      !positions || !token_rows || !status)
    return LB_ERR_INVALID_ARGUMENT;
  PlanArgs a{n, n_sessions, max_pages, n_pages, page_tokens, max_tokens, sessions, new_tokens, tables, lengths,
             reinterpret_cast<const unsigned*>(used), row_tables, kv_len, cu_tokens, positions, token_rows, status,
             reinterpret_cast<long long*>(slots), planned_sessions};
  const size_t smem = sizeof(int) * (3 * static_cast<size_t>(n) + 1 + kPlanThreads + (n_sessions + 31) / 32);
  constexpr size_t kMost = sizeof(int) * (3 * kMaxPlanRows + 1 + kPlanThreads + kMaxPlanSessions / 32);
  static std::atomic<unsigned long long> done{0};
  if (smem > 48 * 1024 &&
      ensure_smem(done, reinterpret_cast<const void*>(plan_kernel), static_cast<int>(kMost)) != cudaSuccess)
    return LB_ERR_CUDA;
  // a CTA for each 4096 values written, at most one per SM
  const long long values = static_cast<long long>(n) * max_pages + 3ll * max_tokens;
  const int grid = static_cast<int>(values / 4096 < 1 ? 1 : values / 4096 > 148 ? 148 : values / 4096);
  plan_kernel<<<grid, kPlanThreads, smem, static_cast<cudaStream_t>(stream)>>>(a);
  return cudaGetLastError() == cudaSuccess ? LB_OK : LB_ERR_CUDA;
}

int lb_plan_pages(int n, const int32_t* sessions, const int32_t* new_tokens, int n_sessions, int max_pages,
                  int n_pages, int page_tokens, const int32_t* tables, const int32_t* lengths,
                  const int32_t* used, int max_tokens, int32_t* row_tables, int32_t* kv_len,
                  int32_t* cu_tokens, int64_t* slots, int32_t* positions, int32_t* token_rows,
                  int32_t* status, void* stream) {
  return lb_plan_step(n, sessions, new_tokens, n_sessions, max_pages, n_pages, page_tokens, tables, lengths, used,
                      max_tokens, row_tables, kv_len, cu_tokens, slots, positions, token_rows, nullptr, status, stream);
}

int lb_commit_step(int n, const int32_t* sessions, int n_sessions, int max_pages, int n_pages, int page_tokens,
                   const int32_t* row_tables, const int32_t* kv_len, const int32_t* cu_tokens, int32_t* status,
                   int32_t* tables, int32_t* lengths, int32_t* used, void* stream) {
  using namespace lb;
  if (bad_shape(n, n_sessions, max_pages, n_pages, page_tokens) || !sessions || !row_tables || !kv_len || !status ||
      !tables || !lengths || !used)
    return LB_ERR_INVALID_ARGUMENT;
  unsigned* bits = reinterpret_cast<unsigned*>(used);
  check_kernel<<<(n + 7) / 8, 256, 0, static_cast<cudaStream_t>(stream)>>>(
      n, sessions, n_sessions, max_pages, n_pages, page_tokens, row_tables, kv_len, cu_tokens, tables, lengths, bits, status);
  if (cudaGetLastError() != cudaSuccess) return LB_ERR_CUDA;
  commit_kernel<<<(n + 7) / 8, 256, 0, static_cast<cudaStream_t>(stream)>>>(
      n, sessions, n_sessions, max_pages, n_pages, page_tokens, row_tables, kv_len, status, tables, lengths, bits);
  return cudaGetLastError() == cudaSuccess ? LB_OK : LB_ERR_CUDA;
}

int lb_commit_pages(int n, const int32_t* sessions, int n_sessions, int max_pages, int n_pages, int page_tokens,
                    const int32_t* row_tables, const int32_t* kv_len, int32_t* status, int32_t* tables,
                    int32_t* lengths, int32_t* used, void* stream) {
  return lb_commit_step(n, sessions, n_sessions, max_pages, n_pages, page_tokens, row_tables, kv_len, nullptr, status,
                        tables, lengths, used, stream);
}

int lb_release_pages(int n, const int32_t* sessions, int n_sessions, int max_pages, int n_pages, int page_tokens,
                     int32_t* tables, int32_t* lengths, int32_t* used, int32_t* status, void* stream) {
  using namespace lb;
  if (bad_shape(n, n_sessions, max_pages, n_pages, page_tokens) || !sessions || !tables || !lengths || !used || !status)
    return LB_ERR_INVALID_ARGUMENT;
  release_kernel<<<(n + 7) / 8, 256, 0, static_cast<cudaStream_t>(stream)>>>(
      n, sessions, n_sessions, max_pages, n_pages, page_tokens, tables, lengths, reinterpret_cast<unsigned*>(used), status);
  return cudaGetLastError() == cudaSuccess ? LB_OK : LB_ERR_CUDA;
}

}  // extern "C"
