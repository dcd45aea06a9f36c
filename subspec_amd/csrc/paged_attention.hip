// Attention of the new tokens of a batch of sequences over a page pool.
#include "common.h"
#include <algorithm>

namespace subspec {

struct PagedParams {
  const uint16_t* q;
  const uint16_t* pool;
  const int32_t* table;
  const int32_t* starts;
  const int32_t* lens;
  uint16_t* out;
  int64_t q_token, q_head;                 // strides, elements
  int64_t table_stride, page_elems;        // page_elems: a page's K (V follows it)
  int batch, n_tokens, hq, hkv, group, max_new, max_kv, window, sinks, page_shift, max_pages, max_blocks;
  float scale_log2;
};

// keys a row at position pos sees: j <= pos, and with a window w only j > pos - w or j < sinks
__device__ __forceinline__ bool paged_sees(const PagedParams& p, int pos, int j) {
  return j <= pos && (p.window == 0 || j > pos - p.window || j < p.sinks);
}

// One workgroup per (token, query head): 256 keys at a time, a thread per key for the scores, then a thread per head dimension.
template <int DT, int D>
__global__ __launch_bounds__(256) void paged_attention_row_kernel(PagedParams p) {
  __shared__ float qs[D], prob[256], scratch[4], half[D];
  __shared__ int64_t row_at[256];
  const int t = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
  int b = 0;
  while (b < p.batch && p.starts[b + 1] <= t) ++b;
  if (b == p.batch || p.starts[b] > t) return;
  const int first = p.starts[b], n = min(p.starts[b + 1] - first, p.max_new);
  if (t - first >= n) return;
  const int len = min(min(p.lens[b], p.max_kv), (int)min((int64_t)p.max_blocks << p.page_shift, (int64_t)INT32_MAX));
  const int pos = len - n + t - first;
  for (int d = tid; d < D; d += 256) qs[d] = Elem<DT>::load(p.q, t * p.q_token + h * p.q_head + d);
  const int kvh = h / p.group;
  float m = -INFINITY, l = 0.f, o = 0.f;
  const int d = tid % D, part = tid / D;
  for (int j0 = 0; j0 <= pos; j0 += 256) {
    const int j = j0 + tid;
    float s = -INFINITY;
    __syncthreads();
    if (paged_sees(p, pos, j)) {
      const int page = min(max(p.table[b * p.table_stride + (j >> p.page_shift)], 0), p.max_pages - 1);
      const int64_t at = (int64_t)page * 2 * p.page_elems + ((int64_t)(j & ((1 << p.page_shift) - 1)) * p.hkv + kvh) * D;
      row_at[tid] = at;
      s = 0.f;
      for (int i = 0; i < D; ++i) s = fmaf(qs[i], Elem<DT>::load(p.pool, at + i), s);
      s *= p.scale_log2;
    }
    const float mx = fmaxf(m, block_max<256>(s, scratch));
    const float e = s == -INFINITY ? 0.f : exp2f(s - mx);
    prob[tid] = e;
    const float alpha = m == -INFINITY ? 0.f : exp2f(m - mx);
    l = l * alpha + block_sum<256>(e, scratch);
    o *= alpha;
    m = mx;
    for (int i = part; i < 256; i += 256 / D)
      if (prob[i] > 0.f) o = fmaf(prob[i], Elem<DT>::load(p.pool, row_at[i] + p.page_elems + d), o);
  }
  for (int w = 1; w < 256 / D; ++w) {
    __syncthreads();
    if (part == w) half[d] = o;
    __syncthreads();
    if (part == 0) o += half[d];
  }
  if (part == 0) Elem<DT>::store(p.out, ((int64_t)t * p.hq + h) * D + d, l > 0.f ? o / l : 0.f);
}

}  // namespace subspec

using namespace subspec;

extern "C" size_t subspec_paged_attention_workspace(int64_t batch, int64_t n_tokens, int64_t n_q_heads, int64_t n_kv_heads,
                                                    int64_t head_dim, int64_t max_new, int64_t max_kv, int64_t window, int64_t sinks) {
  return 256;
}

extern "C" int subspec_paged_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* kv_pool_layer,
                                       int64_t max_pages, int64_t page_len, const int32_t* block_table, int64_t max_blocks,
                                       int64_t table_stride, const int32_t* query_starts, const int32_t* kv_lens, void* out, int dtype,
                                       int64_t batch, int64_t n_tokens, int64_t n_q_heads, int64_t n_kv_heads, int64_t head_dim,
                                       int64_t max_new, int64_t max_kv, int64_t window, int64_t sinks, float scale, void* workspace,
                                       size_t workspace_bytes, void* stream) {
  const char* what = "paged_attention";
  if (dtype != SUBSPEC_BF16 && dtype != SUBSPEC_F16)
    SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: dtype %d not supported (bf16 / fp16 only)", what, dtype);
  if (head_dim != 64 && head_dim != 128)
    SUBSPEC_FAIL(SUBSPEC_ERR_LIMIT, "%s: head_dim=%lld (built for 64 and 128)", what, (long long)head_dim);
  if (n_tokens < 0 || n_tokens > (1ll << 30) || max_new < 0 || max_kv < 0 || max_kv > (1ll << 30))
    SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: n_tokens=%lld max_new=%lld max_kv=%lld", what, (long long)n_tokens, (long long)max_new,
                 (long long)max_kv);
  if (batch < 1 || batch > SUBSPEC_MAX_BATCH)
    SUBSPEC_FAIL(SUBSPEC_ERR_LIMIT, "%s: batch=%lld outside [1, %d]", what, (long long)batch, SUBSPEC_MAX_BATCH);
  if (n_q_heads < 1 || n_kv_heads < 1 || n_q_heads % n_kv_heads || n_q_heads > 1024)
    SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: heads=%lld/%lld", what, (long long)n_q_heads, (long long)n_kv_heads);
  if (page_len < 1 || page_len > (1 << 20) || (page_len & (page_len - 1)))
    SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: page_len=%lld is no power of two up to 2^20", what, (long long)page_len);
  if (max_pages < 1 || max_pages > INT32_MAX || max_blocks < 1 || max_blocks > INT32_MAX || table_stride < max_blocks)
    SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: %lld pages, a table of %lld columns with a row stride of %lld", what, (long long)max_pages,
                 (long long)max_blocks, (long long)table_stride);
  if (window < 0 || sinks < 0 || (window == 0 && sinks != 0))
    SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: window=%lld sinks=%lld", what, (long long)window, (long long)sinks);
  if (!(scale > 0.f) || scale > 1e30f) SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: scale=%g must be positive", what, (double)scale);
  if (n_tokens == 0 || max_new == 0 || max_kv == 0) return SUBSPEC_OK;
  if (!q || !kv_pool_layer || !block_table || !query_starts || !kv_lens || !out)
    SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: null pointer argument", what);
  if ((uintptr_t)q % 16 || (uintptr_t)kv_pool_layer % 16 || (uintptr_t)out % 16 || q_token_stride % 8 || q_head_stride % 8 ||
      q_token_stride < 0 || q_head_stride < 0)
    SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: q, the pool and out must be 16-byte aligned, q's strides multiples of 8 elements", what);
  PagedParams p;
  p.q = (const uint16_t*)q; p.pool = (const uint16_t*)kv_pool_layer; p.table = block_table; p.starts = query_starts; p.lens = kv_lens;
  p.out = (uint16_t*)out;
  p.q_token = q_token_stride; p.q_head = q_head_stride; p.table_stride = table_stride;
  p.page_elems = page_len * n_kv_heads * head_dim;
  p.batch = (int)batch; p.n_tokens = (int)n_tokens; p.hq = (int)n_q_heads; p.hkv = (int)n_kv_heads; p.group = (int)(n_q_heads / n_kv_heads);
  p.max_new = (int)std::min<int64_t>(max_new, n_tokens); p.max_kv = (int)max_kv;
  p.window = (int)std::min<int64_t>(window, 1ll << 30); p.sinks = (int)std::min<int64_t>(sinks, 1ll << 30);
  p.page_shift = 0;
  while ((1ll << p.page_shift) < page_len) ++p.page_shift;
  p.max_pages = (int)max_pages; p.max_blocks = (int)max_blocks;
  p.scale_log2 = scale * kLog2e;
  const dim3 grid((unsigned)n_tokens, (unsigned)n_q_heads);
  hipStream_t st = (hipStream_t)stream;
#define SUBSPEC_PAGED(DT, D) hipLaunchKernelGGL((paged_attention_row_kernel<DT, D>), grid, dim3(256), 0, st, p)
  DominantKernelTimer timer(st);
  if (dtype == SUBSPEC_BF16) { if (head_dim == 128) SUBSPEC_PAGED(SUBSPEC_BF16, 128); else SUBSPEC_PAGED(SUBSPEC_BF16, 64); }
  else { if (head_dim == 128) SUBSPEC_PAGED(SUBSPEC_F16, 128); else SUBSPEC_PAGED(SUBSPEC_F16, 64); }
#undef SUBSPEC_PAGED
  SUBSPEC_CHECK_HIP(hipGetLastError());
  return SUBSPEC_OK;
}
