// One step of a batch of sequences over a page pool, besides its attention: page tables and slot maps from the sequences' lengths, and
// the new tokens' K / V rows into the pool.
//
// The pool is that of the paged cache, [max_pages][2 (K, V)][page_len][n_kv_heads][head_dim] a layer; sequence b's row p sits in page
// block_table[b][p / page_len] at token p % page_len, its slot is page * page_len + p % page_len.
#include "common.h"
#include <algorithm>

namespace subspec {

// ---------------------------------------------------------------------------------------------------------------- plan
// With L cached and n new rows a sequence holds h = ceil(L / P) pages and takes a = ceil((L + n) / P) - h more; tokens and pages are
// numbered by the exclusive sums of n and a over the sequences, and the free pages are a stack, so new page r of the step is
// free[n_free - 1 - r].  Nothing a workgroup needs is written by another: a token whose page is new computes it from the rank, and table
// entries below h are only read.  So every workgroup scans the lengths for itself (8 bytes a sequence, 32 KB at most, out of the L2) and ONE launch does all,
// where a scan, a table update and a slot map would be three.  There is next to nothing to move (8 sequences 0.3 KB, 500 sequences, sixteen of them with chunks,
// 400 KB): the kernel is its chain of dependent reads, 4.4 and 6.8 us (the launch that appends 61 tokens takes 2.6).
constexpr int kPlanThreads = 1024;
constexpr int kPlanItems = SUBSPEC_MAX_BATCH / kPlanThreads;

struct PlanArgs {
  const int32_t* kv_lens;
  const int32_t* new_lens;
  const int32_t* free_pages;
  const int32_t* n_free;
  int32_t* block_table;
  int32_t* query_starts;
  int32_t* total_lens;
  int32_t* positions;
  int64_t* slots;
  int32_t* sequences;
  int32_t* counts;
  int64_t free_capacity, max_blocks, table_stride;
  int batch, page_shift, n_tokens;
};

__device__ __forceinline__ int64_t wave_scan64(int64_t v) {          // inclusive
  const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const int64_t u = __shfl_up(v, o, kWave);
    if (lane >= o) v += u;
  }
  return v;
}

__global__ __launch_bounds__(kPlanThreads) void paged_plan_kernel(PlanArgs a) {
  __shared__ int32_t starts[SUBSPEC_MAX_BATCH + 1], page_starts[SUBSPEC_MAX_BATCH + 1];
  __shared__ int64_t wave_tokens[kPlanThreads / kWave], wave_pages[kPlanThreads / kWave];
  __shared__ int bad;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  if (tid == 0) bad = 0;
  __syncthreads();
  const int items = (a.batch + kPlanThreads - 1) / kPlanThreads, b0 = tid * items;
  const int page_mask = (1 << a.page_shift) - 1;
  int64_t n[kPlanItems], pages[kPlanItems], sum_n = 0, sum_p = 0;
  int flaws = 0;
#pragma unroll
  for (int i = 0; i < kPlanItems; ++i) {
    n[i] = pages[i] = 0;
    if (i < items && b0 + i < a.batch) {
      const int64_t held = a.kv_lens[b0 + i], more = a.new_lens[b0 + i];
      if (held < 0 || more < 0) {
        flaws |= SUBSPEC_PLAN_NEGATIVE;
      } else {
        const int64_t need = (held + more + page_mask) >> a.page_shift;
        if (need > a.max_blocks || held + more > INT32_MAX) flaws |= SUBSPEC_PLAN_TABLE;
        n[i] = more;
        pages[i] = need - ((held + page_mask) >> a.page_shift);
      }
    }
    sum_n += n[i];
    sum_p += pages[i];
  }
  const int64_t upto_n = wave_scan64(sum_n), upto_p = wave_scan64(sum_p);
  if (lane == kWave - 1) {
    wave_tokens[wave] = upto_n;
    wave_pages[wave] = upto_p;
  }
  if (flaws) atomicOr(&bad, flaws);
  __syncthreads();
  int64_t at_n = upto_n - sum_n, at_p = upto_p - sum_p, tokens = 0, taken = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / kWave; ++w) {
    if (w < wave) {
      at_n += wave_tokens[w];
      at_p += wave_pages[w];
    }
    tokens += wave_tokens[w];
    taken += wave_pages[w];
  }
  const int64_t n_free = *a.n_free;
  int status = bad;
  if (tokens > a.n_tokens) status |= SUBSPEC_PLAN_TOKENS;
  if (n_free > a.free_capacity || taken > n_free) status |= SUBSPEC_PLAN_PAGES;
  if (status) {                                          // (the same in every thread of every workgroup) nothing is handed out
    if (blockIdx.x == 0) {
      for (int b = tid; b < a.batch; b += kPlanThreads) a.total_lens[b] = a.kv_lens[b];
      for (int b = tid; b <= a.batch; b += kPlanThreads) a.query_starts[b] = 0;
      if (tid < 4) a.counts[tid] = tid == 2 ? (int32_t)n_free : tid == 3 ? status : 0;
    }
    const int64_t t = (int64_t)blockIdx.x * kPlanThreads + tid;
    if (t < a.n_tokens) {
      a.positions[t] = 0;
      a.slots[t] = -1;
      a.sequences[t] = -1;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < kPlanItems; ++i) {
    if (i < items && b0 + i < a.batch) {
      starts[b0 + i] = (int32_t)at_n;
      page_starts[b0 + i] = (int32_t)at_p;
      if (blockIdx.x == 0) {
        a.query_starts[b0 + i] = (int32_t)at_n;
        a.total_lens[b0 + i] = a.kv_lens[b0 + i] + (int32_t)n[i];
      }
    }
    at_n += n[i];
    at_p += pages[i];
  }
  if (blockIdx.x == 0 && tid < 5) {
    if (tid == 4) a.query_starts[a.batch] = (int32_t)tokens;
    else a.counts[tid] = tid == 0 ? (int32_t)tokens : tid == 1 ? (int32_t)taken : tid == 2 ? (int32_t)(n_free - taken) : 0;
  }
  __syncthreads();
  // the last sequence whose start is not behind x: the one that x lies in (those that bring nothing share their start with the next)
  auto owner = [&](const int32_t* s, int x) {
    int lo = 0, hi = a.batch;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s[mid] <= x) lo = mid;
      else hi = mid;
    }
    return lo;
  };
  const int32_t* stack = a.free_pages + n_free - 1;
  for (int64_t r = (int64_t)blockIdx.x * kPlanThreads + tid; r < taken; r += (int64_t)gridDim.x * kPlanThreads) {
    const int b = owner(page_starts, (int)r);
    const int64_t held = ((int64_t)a.kv_lens[b] + page_mask) >> a.page_shift;
    a.block_table[b * a.table_stride + held + r - page_starts[b]] = stack[-r];
  }
  const int64_t t = (int64_t)blockIdx.x * kPlanThreads + tid;
  if (t >= a.n_tokens) return;
  if (t >= tokens) {
    a.positions[t] = 0;
    a.slots[t] = -1;
    a.sequences[t] = -1;
    return;
  }
  const int b = owner(starts, (int)t);
  const int64_t len = a.kv_lens[b], pos = len + t - starts[b], held = (len + page_mask) >> a.page_shift;
  const int64_t block = pos >> a.page_shift;
  const int page = block < held ? a.block_table[b * a.table_stride + block] : stack[-(page_starts[b] + block - held)];
  a.positions[t] = (int32_t)pos;
  a.slots[t] = page < 0 ? -1 : ((int64_t)page << a.page_shift) + (pos & page_mask);
  a.sequences[t] = b;
}

// ---------------------------------------------------------------------------------------------------------------- append
// Pure data movement.  `lanes` (a power of two) lanes carry one token, K and V side by side, `Piece` bytes each at a time, so that a
// wavefront is busy also where a token's K is a few pieces only.  8191 tokens of 8 heads of 128, 67 MB out and back: 11.0 us, 6.1 TB/s, where a
// large copy reaches 5.2 (the rows come out of the caches where they were just written); 61 tokens: a launch.
struct AppendArgs {
  const char* k;
  const char* v;
  char* pool;
  const int64_t* slots;
  int64_t k_token, k_head, v_token, v_head;      // strides, bytes
  int64_t row_bytes, head_bytes, page_bytes;     // a token's K in the pool, a head's part of it, a page's K
  int64_t n_slots;
  int n_tokens, page_shift, lane_shift;
};

template <typename Piece>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendArgs a) {
  const int lanes = 1 << a.lane_shift;
  const int64_t t = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> a.lane_shift;
  if (t >= a.n_tokens) return;
  const int64_t slot = a.slots[t];
  if (slot < 0 || slot >= a.n_slots) return;             // a padded row, or a bad map: nothing is written
  char* row = a.pool + (slot >> a.page_shift) * 2 * a.page_bytes + (slot & ((1 << a.page_shift) - 1)) * a.row_bytes;
  const char* k = a.k + t * a.k_token;
  const char* v = a.v + t * a.v_token;
  const int head_bytes = (int)a.head_bytes;
  for (int i = (int)(threadIdx.x & (lanes - 1)) * (int)sizeof(Piece); i < a.row_bytes; i += lanes * (int)sizeof(Piece)) {
    const int head = i / head_bytes, in = i - head * head_bytes;
    const Piece kp = *(const Piece*)(k + head * a.k_head + in), vp = *(const Piece*)(v + head * a.v_head + in);
    *(Piece*)(row + i) = kp;
    *(Piece*)(row + a.page_bytes + i) = vp;
  }
}

static int page_shift_of(int64_t page_len) {
  int shift = 0;
  while ((1ll << shift) < page_len) ++shift;
  return shift;
}

}  // namespace subspec

using namespace subspec;

extern "C" int subspec_paged_batch_plan(const int32_t* kv_lens, const int32_t* new_lens, int64_t batch, const int32_t* free_pages,
                                        const int32_t* n_free, int64_t free_capacity, int32_t* block_table, int64_t max_blocks,
                                        int64_t table_stride, int64_t page_len, int64_t n_tokens, int32_t* query_starts,
                                        int32_t* total_lens, int32_t* positions, int64_t* slots, int32_t* sequences, int32_t* counts,
                                        void* stream) {
  const char* what = "paged_batch_plan";
  if (!kv_lens || !new_lens || !n_free || !block_table || !query_starts || !total_lens || !counts || (free_capacity > 0 && !free_pages) ||
      (n_tokens > 0 && (!positions || !slots || !sequences)))
    SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: null pointer argument", what);
  if (batch < 1 || batch > SUBSPEC_MAX_BATCH)
    SUBSPEC_FAIL(SUBSPEC_ERR_LIMIT, "%s: batch=%lld outside [1, %d]", what, (long long)batch, SUBSPEC_MAX_BATCH);
  if (page_len < 1 || page_len > (1 << 20) || (page_len & (page_len - 1)))
    SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: page_len=%lld is no power of two up to 2^20", what, (long long)page_len);
  if (max_blocks < 1 || table_stride < max_blocks || max_blocks > INT32_MAX)
    SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: a table of %lld columns with a row stride of %lld", what, (long long)max_blocks,
                 (long long)table_stride);
  if (free_capacity < 0 || free_capacity > INT32_MAX || n_tokens < 0 || n_tokens > (1ll << 30))
    SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: free_capacity=%lld, n_tokens=%lld", what, (long long)free_capacity, (long long)n_tokens);
  PlanArgs a{kv_lens, new_lens, free_pages, n_free, block_table, query_starts, total_lens, positions, slots, sequences, counts,
             free_capacity, max_blocks, table_stride, (int)batch, page_shift_of(page_len), (int)n_tokens};
  const int64_t groups = std::max<int64_t>(1, (n_tokens + kPlanThreads - 1) / kPlanThreads);
  DominantKernelTimer timer((hipStream_t)stream);
  hipLaunchKernelGGL(paged_plan_kernel, dim3((unsigned)groups), dim3(kPlanThreads), 0, (hipStream_t)stream, a);
  SUBSPEC_CHECK_HIP(hipGetLastError());
  return SUBSPEC_OK;
}

extern "C" int subspec_kv_append_paged(const void* k, int64_t k_token_stride, int64_t k_head_stride, const void* v, int64_t v_token_stride,
                                       int64_t v_head_stride, void* kv_pool_layer, int dtype, int64_t max_pages, int64_t page_len,
                                       int64_t n_kv_heads, int64_t head_dim, const int64_t* slots, int64_t n_tokens, void* stream) {
  const char* what = "kv_append_paged";
  if (!dtype_ok(dtype)) SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: dtype %d not supported", what, dtype);
  if (n_tokens < 0 || n_tokens > (1ll << 30)) SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: n_tokens=%lld", what, (long long)n_tokens);
  if (n_tokens == 0) return SUBSPEC_OK;
  if (!k || !v || !kv_pool_layer || !slots) SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: null pointer argument", what);
  if (page_len < 1 || page_len > (1 << 20) || (page_len & (page_len - 1)))
    SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: page_len=%lld is no power of two up to 2^20", what, (long long)page_len);
  if (max_pages < 1 || max_pages > INT32_MAX || n_kv_heads < 1 || head_dim < 1 || n_kv_heads * head_dim > (1 << 24))
    SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: %lld pages of %lld heads of %lld", what, (long long)max_pages, (long long)n_kv_heads,
                 (long long)head_dim);
  if (k_token_stride < 0 || k_head_stride < 0 || v_token_stride < 0 || v_head_stride < 0)
    SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: negative stride", what);
  const int64_t es = (int64_t)dtype_size(dtype);
  AppendArgs a;
  a.k = (const char*)k; a.v = (const char*)v; a.pool = (char*)kv_pool_layer; a.slots = slots;
  a.k_token = k_token_stride * es; a.k_head = k_head_stride * es; a.v_token = v_token_stride * es; a.v_head = v_head_stride * es;
  a.head_bytes = head_dim * es; a.row_bytes = n_kv_heads * a.head_bytes; a.page_bytes = page_len * a.row_bytes;
  a.n_slots = max_pages * page_len;
  a.n_tokens = (int)n_tokens; a.page_shift = page_shift_of(page_len);
  if (((uintptr_t)k | (uintptr_t)v | (uintptr_t)kv_pool_layer) % es) SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: misaligned tensors", what);
  // the widest piece that every row and head starts at
  const uint64_t all = (uint64_t)(uintptr_t)k | (uint64_t)(uintptr_t)v | (uint64_t)(uintptr_t)kv_pool_layer | (uint64_t)a.k_token |
                       (uint64_t)a.k_head | (uint64_t)a.v_token | (uint64_t)a.v_head | (uint64_t)a.head_bytes;
  const int piece = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 2;
  const int64_t pieces = a.row_bytes / piece;
  a.lane_shift = 0;
  while (a.lane_shift < 6 && (1 << a.lane_shift) < pieces) ++a.lane_shift;
  const int64_t per_group = 256 >> a.lane_shift;
  const dim3 grid((unsigned)((n_tokens + per_group - 1) / per_group));
  hipStream_t st = (hipStream_t)stream;
  DominantKernelTimer timer(st);
  if (piece == 16) hipLaunchKernelGGL(kv_append_kernel<uint4>, grid, dim3(256), 0, st, a);
  else if (piece == 4) hipLaunchKernelGGL(kv_append_kernel<uint32_t>, grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(kv_append_kernel<uint16_t>, grid, dim3(256), 0, st, a);
  SUBSPEC_CHECK_HIP(hipGetLastError());
  return SUBSPEC_OK;
}
