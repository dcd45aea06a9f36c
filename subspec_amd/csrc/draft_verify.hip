// Drafted tokens of a batch of sequences against the target's probabilities, from given numbers, for gfx950.
//
// Row i of a sequence's logits gives the distribution p_i of the token behind its token i (softmax at a temperature, after the filters of a draw, see
// sample.hip); the draft x_i behind it was drawn from q_i.  x_i stays if u_i q_i(x_i) < p_i(x_i), which happens with probability min(1, p_i / q_i); at the
// first that does not the next token is drawn from max(p_i - q_i, 0), after the last row from p itself.  What comes out is distributed like the target's own
// draws (Y. Leviathan, M. Kalman, Y. Matias, "Fast inference from transformers via speculative decoding", 2023).  A draft without q is one
// that nothing was drawn for: q_i(x_i) = 1.
//
// Masses are the whole numbers of a draw (2^-42 of the largest, see mass_series.h).  With m_j an entry's mass and Z the row's, the test is u q Z < m, and the rest
// max(m_j - q_j Z, 0) is rounded to such units again, so its sums are exact, no order of addition changes a token, and the token is the first in the
// order of the vocabulary whose sum exceeds v times the whole.
#include "sample.h"
#include <algorithm>

namespace subspec {

constexpr int kVerifyThreads = 256;
constexpr int kVerifyRound = 8 * kVerifyThreads;       // entries that a workgroup takes at a time, eight a thread

// A slice's mass, relative to its own largest logit: rows without filters need no more than the sums of these.
struct SliceMass {
  double mass;
  float top;
  int first;                       // index of the first entry that equals it
};
// The row that a sequence ends with.
struct EndRecord {
  RowCut cut;
  int row, sequence_row;           // row of the call (-1: the sequence has none), row of the sequence
  int last;                        // no draft stands behind it
  int draft;                       // ... or the one that did not stay (-1: none of the vocabulary)
};
struct RestSum { uint64_t rest, all; };
struct VerifyArgs {
  SampleArgs s;
  const int64_t* drafts;
  const int32_t* starts;
  const float* draws;
  const void* q;
  int64_t q_stride;
  int32_t* accepted;
  RowCut* cuts;                    // of every row, where `slices` is 0
  SliceMass* masses;               // [row][slices]
  EndRecord* ends;
  RestSum* sums;                   // [sequence][end_slices]
  int q_dtype, slices, length, end_slices, end_length, batch, n_rows, wide, q_wide;
};

struct VerifySpan { int first, n; };
__device__ __forceinline__ VerifySpan verify_span(const VerifyArgs& a, int b) {
  const int first = min(max(a.starts[b], 0), a.n_rows), end = min(max(a.starts[b + 1], 0), a.n_rows);
  return VerifySpan{first, max(end - first, 0)};
}
template <int DT>
__device__ __forceinline__ const char* verify_row(const VerifyArgs& a, int row) {
  return (const char*)a.s.logits + (int64_t)row * a.s.row_stride * Elem<DT>::kBytes;
}
// Entries i .. i + 7 of a row of n; `fill` behind its end.  wide: rows start at multiples of 16 bytes.
template <int DT>
__device__ __forceinline__ void load_eight(const void* row, int i, int n, int wide, float fill, float* x) {
  if (wide && i + 8 <= n) {
    const dec_u4* p = (const dec_u4*)((const char*)row + (size_t)i * Elem<DT>::kBytes);
    if constexpr (DT == SUBSPEC_F32) {
      const dec_u4 a = p[0], b = p[1];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = __uint_as_float(a[e]);
        x[4 + e] = __uint_as_float(b[e]);
      }
    } else {
      unpack8<DT>(p[0], x);
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = i + e < n ? Elem<DT>::load(row, i + e) : fill;
}
__device__ __forceinline__ void load_eight_q(const VerifyArgs& a, int row, int i, float* x) {
  const int n = a.s.vocab;
  if (a.q_dtype == SUBSPEC_F32) load_eight<SUBSPEC_F32>((const char*)a.q + row * a.q_stride * 4, i, n, a.q_wide, 0.f, x);
  else if (a.q_dtype == SUBSPEC_F16) load_eight<SUBSPEC_F16>((const char*)a.q + row * a.q_stride * 2, i, n, a.q_wide, 0.f, x);
  else load_eight<SUBSPEC_BF16>((const char*)a.q + row * a.q_stride * 2, i, n, a.q_wide, 0.f, x);
}
__device__ __forceinline__ double draft_prob(float q) { return q > 0.f ? (double)q : 0.0; }       // (a NaN is none)
__device__ __forceinline__ float load_q(const VerifyArgs& a, int row, int i) {
  const int64_t at = row * a.q_stride + i;
  return a.q_dtype == SUBSPEC_F32 ? ((const float*)a.q)[at] : a.q_dtype == SUBSPEC_F16 ? Elem<SUBSPEC_F16>::load(a.q, at) : Elem<SUBSPEC_BF16>::load(a.q, at);
}
// The mass that an entry keeps, before rounding
template <int DT>
__device__ __forceinline__ double kept_mass(float l, int i, const RowCut& cut, const RowTop& top, const RowRule& r, const Series& series) {
  if (!(entry_distance(l, top, r) < kReach)) return 0.0;
  const double m = entry_mass(l, top, r, series);
  if (r.min_p > 0.0 && m < r.min_p * (double)(1ull << kMassBits)) return 0.0;
  return cut.last != ~0ull && order_key<DT>(l, i) > cut.last ? 0.0 : m;
}
__device__ __forceinline__ uint64_t block_sum_u64(uint64_t v, uint64_t* scratch) {
  v = wave_scan_u64(v);
  if ((threadIdx.x & (kWave - 1)) == kWave - 1) scratch[threadIdx.x / kWave] = v;
  __syncthreads();
  uint64_t sum = 0;
#pragma unroll
  for (int w = 0; w < kVerifyThreads / kWave; ++w) sum += scratch[w];
  __syncthreads();
  return sum;
}

// ---------------------------------------------------------------------------------------------------------------- rows without filters
template <int DT, int ROUNDS>
__global__ __launch_bounds__(kVerifyThreads) void verify_mass_kernel(VerifyArgs a) {
  __shared__ float tops[kVerifyThreads / kWave];
  __shared__ int firsts[kVerifyThreads / kWave];
  __shared__ uint64_t sums[kVerifyThreads / kWave];
  const int row = blockIdx.x / a.slices, slice = blockIdx.x % a.slices;
  if (row < a.starts[0] || row >= a.starts[a.batch]) return;           // a row of no sequence
  const RowRule r = row_rule(a.s, row);
  const char* src = verify_row<DT>(a, row);
  const int i0 = slice * a.length + 8 * (int)threadIdx.x;
  float x[8 * ROUNDS], top = -INFINITY;
#pragma unroll
  for (int k = 0; k < ROUNDS; ++k) load_eight<DT>(src, i0 + k * kVerifyRound, a.s.vocab, a.wide, -INFINITY, x + 8 * k);
#pragma unroll
  for (int e = 0; e < 8 * ROUNDS; ++e) top = x[e] > top ? x[e] : top;   // (a NaN never is)
  top = block_max<kVerifyThreads>(top, tops);
  const RowTop t = row_top_of(top, r);
  const Series series;
  uint64_t sum = 0;
  int first = INT32_MAX;
  if (top > -INFINITY) {
#pragma unroll
    for (int e = 0; e < 8 * ROUNDS; ++e) {
      if (entry_distance(x[e], t, r) < kReach) sum += whole(entry_mass(x[e], t, r, series));
      if (r.greedy && x[e] == top) first = min(first, i0 + (e / 8) * kVerifyRound + e % 8);
    }
  }
  if (r.greedy) first = block_min_i<kVerifyThreads>(first, firsts);     // (uniform)
  sum = block_sum_u64(sum, sums);
  if (threadIdx.x == 0) a.masses[blockIdx.x] = SliceMass{(double)sum, top, first};
}

// A row's cut from its slices (a wavefront; the same in all its lanes)
template <int DT>
__device__ RowCut row_cut(const VerifyArgs& a, int row, const RowRule& r, const Series& series) {
  if (a.slices == 0) return a.cuts[row];
  const int lane = threadIdx.x & (kWave - 1);
  const SliceMass* of = a.masses + (int64_t)row * a.slices;
  float top = -INFINITY;
  for (int s = lane; s < a.slices; s += kWave) top = fmaxf(top, of[s].top);
  top = wave_max(top);
  if (top == -INFINITY) return RowCut{0.0, 0, top};
  const RowTop t = row_top_of(top, r);
  if (r.greedy) {                                                       // the first of the largest alone
    int first = INT32_MAX;
    for (int s = lane; s < a.slices; s += kWave)
      if (of[s].top == top) first = min(first, of[s].first);
    return RowCut{(double)(1ull << kMassBits), order_key<DT>(top, wave_min_i(first)), top};
  }
  double z = 0.0;
  for (int s = lane; s < a.slices; s += kWave) {
    const SliceMass m = of[s];
    if (entry_distance(m.top, t, r) < kReach) z = fma(m.mass, entry_mass(m.top, t, r, series) * 0x1p-42, z);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) z += __shfl_xor(z, o, kWave);
  return RowCut{z, ~0ull, top};
}

// ---------------------------------------------------------------------------------------------------------------- which drafts stay
// A workgroup a sequence, a wavefront a row at a time; one more for the rows of nobody.
template <int DT>
__global__ __launch_bounds__(kVerifyThreads) void verify_accept_kernel(VerifyArgs a) {
  __shared__ int end;
  if ((int)blockIdx.x == a.batch) {
    const int begin = min(max(a.starts[0], 0), a.n_rows), behind = min(max(a.starts[a.batch], 0), a.n_rows);
    for (int t = threadIdx.x; t < a.n_rows; t += kVerifyThreads)
      if (t < begin || t >= behind) {
        a.s.tokens[t] = -1;
        a.s.probs[t] = 0.f;
      }
    return;
  }
  const VerifySpan sp = verify_span(a, blockIdx.x);
  if (sp.n == 0) {
    if (threadIdx.x == 0) {
      a.accepted[blockIdx.x] = 0;
      a.ends[blockIdx.x].row = -1;
    }
    return;
  }
  if (threadIdx.x == 0) end = sp.n - 1;
  __syncthreads();
  const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
  const Series series;
  for (int i = wave; i < sp.n - 1; i += kVerifyThreads / kWave) {
    const int row = sp.first + i;
    const RowRule r = row_rule(a.s, row);
    const int64_t x = a.drafts[row + 1];
    const bool known = x >= 0 && x < a.s.vocab;
    const float l = known ? Elem<DT>::load(verify_row<DT>(a, row), x) : -INFINITY;
    const double q = !a.q ? 1.0 : known ? draft_prob(load_q(a, row, (int)x)) : 0.0;
    const RowCut cut = row_cut<DT>(a, row, r, series);
    const double m = cut.mass > 0.0 ? kept_mass<DT>(l, (int)x, cut, row_top_of(cut.top, r), r, series) : 0.0;
    if (lane == 0) {
      a.s.probs[row] = cut.mass > 0.0 ? (float)(m / cut.mass) : 0.f;
      if (!(r.u * q * cut.mass < m)) atomicMin(&end, i);
    }
  }
  __syncthreads();
  const int stop = end;
  for (int i = threadIdx.x; i < sp.n; i += kVerifyThreads) {            // (the row it ends with is the draw's)
    if (i < stop) {
      a.s.tokens[sp.first + i] = a.drafts[sp.first + i + 1];
    } else if (i > stop) {
      a.s.tokens[sp.first + i] = -1;
      a.s.probs[sp.first + i] = 0.f;
    }
  }
  if (wave != 0) return;
  const int row = sp.first + stop;
  const RowCut cut = row_cut<DT>(a, row, row_rule(a.s, row), series);
  if (lane == 0) {
    const int64_t x = stop == sp.n - 1 ? -1 : a.drafts[row + 1];
    a.accepted[blockIdx.x] = stop;
    a.ends[blockIdx.x] = EndRecord{cut, row, stop, stop == sp.n - 1, x >= 0 && x < a.s.vocab ? (int)x : -1};
  }
}

// ---------------------------------------------------------------------------------------------------------------- the token behind them
// What the draw gives an entry: its rest, or (all) its mass.
template <int DT>
struct RestOf {
  const EndRecord& e;
  RowRule r;
  RowTop top;
  Series series;
  __device__ __forceinline__ RestOf(const VerifyArgs& a, const EndRecord& end) : e(end), r(row_rule(a.s, end.row)), top(row_top_of(end.cut.top, r)) {}
  __device__ __forceinline__ double mass(float l, int i) const { return kept_mass<DT>(l, i, e.cut, top, r, series); }
  __device__ __forceinline__ uint64_t rest(double m, float q) const {
    const double left = fma(-draft_prob(q), e.cut.mass, m);
    return left > 0.0 ? whole(left) : 0;
  }
};
// the draft's probabilities of eight entries
__device__ __forceinline__ void eight_drafts(const VerifyArgs& a, const EndRecord& e, int i, float* q) {
  if (e.last) return;
  if (a.q) {
    load_eight_q(a, e.row, i, q);
    return;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) q[k] = i + k == e.draft ? 1.f : 0.f;
}

template <int DT>
__global__ __launch_bounds__(kVerifyThreads) void verify_rest_kernel(VerifyArgs a) {
  __shared__ uint64_t scratch[kVerifyThreads / kWave];
  const int b = blockIdx.x / a.end_slices, slice = blockIdx.x % a.end_slices;
  const EndRecord e = a.ends[b];
  if (e.row < 0 || !(e.cut.mass > 0.0)) return;
  const RestOf<DT> of(a, e);
  const char* src = verify_row<DT>(a, e.row);
  const int end = min((slice + 1) * a.end_length, a.s.vocab);
  uint64_t rest = 0, all = 0;
  for (int i = slice * a.end_length + 8 * (int)threadIdx.x; i < end; i += kVerifyRound) {
    float x[8], q[8];
    load_eight<DT>(src, i, a.s.vocab, a.wide, -INFINITY, x);
    eight_drafts(a, e, i, q);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const double m = of.mass(x[k], i + k);
      all += whole(m);
      if (!e.last) rest += of.rest(m, q[k]);
    }
  }
  rest = block_sum_u64(rest, scratch);
  all = block_sum_u64(all, scratch);
  if (threadIdx.x == 0) a.sums[blockIdx.x] = RestSum{rest, all};
}

// sum over the threads before this one, and over all of them
__device__ __forceinline__ uint64_t block_before_u64(uint64_t v, uint64_t* scratch, uint64_t* total) {
  const uint64_t upto = wave_scan_u64(v);
  if ((threadIdx.x & (kWave - 1)) == kWave - 1) scratch[threadIdx.x / kWave] = upto;
  __syncthreads();
  uint64_t before = upto - v, sum = 0;
#pragma unroll
  for (int w = 0; w < kVerifyThreads / kWave; ++w) {
    if (w < (int)threadIdx.x / kWave) before += scratch[w];
    sum += scratch[w];
  }
  __syncthreads();
  *total = sum;
  return before;
}

template <int DT>
__global__ __launch_bounds__(kVerifyThreads) void verify_draw_kernel(VerifyArgs a) {
  __shared__ uint64_t scratch[kVerifyThreads / kWave], goal_left;
  __shared__ int found;
  const EndRecord e = a.ends[blockIdx.x];
  if (e.row < 0) return;                                                // (uniform, as the other return below)
  if (threadIdx.x == 0) {                                               // (what stays where nothing can be drawn)
    a.s.tokens[e.row] = -1;
    a.s.probs[e.row] = 0.f;
    found = 0;
    goal_left = 0;
  }
  if (!(e.cut.mass > 0.0)) return;
  // the slice that the number falls into: a thread has consecutive ones
  const RestSum* sums = a.sums + (int64_t)blockIdx.x * a.end_slices;
  const int each = (a.end_slices + kVerifyThreads - 1) / kVerifyThreads, s0 = threadIdx.x * each;
  uint64_t rest = 0, all = 0, total;
  for (int s = s0; s < min(s0 + each, a.end_slices); ++s) {
    rest += sums[s].rest;
    all += sums[s].all;
  }
  const uint64_t rest_before = block_before_u64(rest, scratch, &total);
  const bool by_rest = total > 0;
  uint64_t all_total;
  const uint64_t all_before = block_before_u64(all, scratch, &all_total);
  if (!by_rest) total = all_total;
  const float v = a.draws[blockIdx.x];
  const uint64_t goal = draw_goal(v > 0.f ? (double)v : 0.0, total);
  uint64_t before = by_rest ? rest_before : all_before;
  if (before <= goal && goal < before + (by_rest ? rest : all)) {        // (one thread: the goal is below the total)
    int s = s0;
    for (;; ++s) {
      const uint64_t here = by_rest ? sums[s].rest : sums[s].all;
      if (s + 1 >= min(s0 + each, a.end_slices) || goal < before + here) break;
      before += here;
    }
    found = s;
    goal_left = goal - before;
  }
  __syncthreads();
  // ... and the entry in it: a thread has consecutive ones again
  const RestOf<DT> of(a, e);
  const char* src = verify_row<DT>(a, e.row);
  const int per = a.end_length / kVerifyThreads, i0 = found * a.end_length + (int)threadIdx.x * per;
  const uint64_t left = goal_left;
  auto weight = [&](const float* x, const float* q, int k, int i) {
    const double m = of.mass(x[k], i + k);
    return by_rest ? of.rest(m, q[k]) : whole(m);
  };
  uint64_t sum = 0;
  float x[8], q[8];
  for (int i = i0; i < i0 + per; i += 8) {
    load_eight<DT>(src, i, a.s.vocab, a.wide, -INFINITY, x);
    eight_drafts(a, e, i, q);
#pragma unroll
    for (int k = 0; k < 8; ++k) sum += weight(x, q, k, i);
  }
  uint64_t at = block_before_u64(sum, scratch, &total);
  if (!(at <= left && left < at + sum)) return;                          // (one thread is left)
  for (int i = i0; i < i0 + per; i += 8) {
    load_eight<DT>(src, i, a.s.vocab, a.wide, -INFINITY, x);
    eight_drafts(a, e, i, q);
    for (int k = 0; k < 8; ++k) {
      at += weight(x, q, k, i);
      if (at > left) {
        a.s.tokens[e.row] = i + k;
        a.s.probs[e.row] = (float)(of.mass(x[k], i + k) / e.cut.mass);
        return;
      }
    }
  }
}

// Entries of a slice: a round or more of a workgroup's threads, so that `rows` rows make some thousands of workgroups.
static int verify_slice_length(int64_t rows, int64_t vocab) {
  int64_t length = kVerifyRound;
  while (length < 4 * kVerifyRound && rows * ((vocab + 2 * length - 1) / (2 * length)) >= 2048) length *= 2;
  return (int)length;
}

struct VerifyPlan {
  int length, slices, end_length, end_slices;
  size_t search, masses, cuts, ends, sums, bytes;
};
static VerifyPlan verify_plan(int64_t n_rows, int64_t batch, int64_t vocab, bool filtered) {
  VerifyPlan p{};
  p.length = verify_slice_length(n_rows, vocab);
  p.slices = (int)((vocab + p.length - 1) / p.length);
  p.end_length = verify_slice_length(batch, vocab);
  p.end_slices = (int)((vocab + p.end_length - 1) / p.end_length);
  if (filtered && n_rows > 0) p.search = align_up(row_search_workspace(n_rows, vocab), 256);
  else p.masses = align_up((size_t)n_rows * p.slices * sizeof(SliceMass), 256);
  p.cuts = filtered ? align_up((size_t)n_rows * sizeof(RowCut), 256) : 0;
  p.ends = align_up((size_t)batch * sizeof(EndRecord), 256);
  p.sums = align_up((size_t)batch * p.end_slices * sizeof(RestSum), 256);
  p.bytes = p.search + p.masses + p.cuts + p.ends + p.sums;
  return p;
}

template <int DT>
static void launch_verify(const VerifyArgs& a, hipStream_t st) {
  if (a.n_rows > 0) {
    if (a.slices) {
      DominantKernelTimer timer(st);
      const dim3 grid((unsigned)((int64_t)a.n_rows * a.slices)), block(kVerifyThreads);
      if (a.length == kVerifyRound) hipLaunchKernelGGL((verify_mass_kernel<DT, 1>), grid, block, 0, st, a);
      else if (a.length == 2 * kVerifyRound) hipLaunchKernelGGL((verify_mass_kernel<DT, 2>), grid, block, 0, st, a);
      else hipLaunchKernelGGL((verify_mass_kernel<DT, 4>), grid, block, 0, st, a);
    }
  }
  hipLaunchKernelGGL(verify_accept_kernel<DT>, dim3((unsigned)a.batch + 1), dim3(kVerifyThreads), 0, st, a);
  if (a.n_rows > 0) {
    hipLaunchKernelGGL(verify_rest_kernel<DT>, dim3((unsigned)(a.batch * a.end_slices)), dim3(kVerifyThreads), 0, st, a);
    hipLaunchKernelGGL(verify_draw_kernel<DT>, dim3((unsigned)a.batch), dim3(kVerifyThreads), 0, st, a);
  }
}

}  // namespace subspec

using namespace subspec;

extern "C" size_t subspec_verify_drafts_workspace(int64_t n_rows, int64_t batch, int64_t vocab, int filtered) {
  if (n_rows < 0 || n_rows > (1 << 20) || batch < 1 || batch > SUBSPEC_MAX_BATCH || vocab < 1 || vocab > (1 << 20)) return 256;
  return verify_plan(n_rows, batch, vocab, filtered != 0).bytes;
}

extern "C" int subspec_verify_drafts(const void* logits, int dtype, int64_t n_rows, int64_t vocab, int64_t row_stride, const int64_t* drafts,
                                     const int32_t* query_starts, int64_t batch, const float* uniforms, const float* draws,
                                     const void* draft_probs, int draft_dtype, int64_t draft_stride, const float* temperatures,
                                     float temperature, const int32_t* top_ks, int32_t top_k, const float* top_ps, float top_p,
                                     const float* min_ps, float min_p, void* workspace, size_t workspace_bytes, int64_t* tokens, float* probs,
                                     int32_t* accepted, void* stream) {
  const char* what = "verify_drafts";
  if (!dtype_ok(dtype) || (draft_probs && !dtype_ok(draft_dtype)))
    SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: dtype %d / %d not supported", what, dtype, draft_dtype);
  if (n_rows < 0 || n_rows > (1 << 20)) SUBSPEC_FAIL(SUBSPEC_ERR_LIMIT, "%s: n_rows=%lld outside [0, 2^20]", what, (long long)n_rows);
  if (vocab < 1 || vocab > (1 << 20)) SUBSPEC_FAIL(SUBSPEC_ERR_LIMIT, "%s: vocab=%lld outside [1, 2^20]", what, (long long)vocab);
  if (batch < 1 || batch > SUBSPEC_MAX_BATCH)
    SUBSPEC_FAIL(SUBSPEC_ERR_LIMIT, "%s: batch=%lld outside [1, %d]", what, (long long)batch, SUBSPEC_MAX_BATCH);
  if (row_stride < vocab || (draft_probs && draft_stride < vocab))
    SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: rows of %lld entries are %lld and %lld apart", what, (long long)vocab, (long long)row_stride,
                 (long long)draft_stride);
  if (!query_starts || !accepted || (n_rows > 0 && (!logits || !drafts || !uniforms || !draws || !tokens || !probs)))
    SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: null pointer argument", what);
  if ((uintptr_t)logits % dtype_size(dtype) || (draft_probs && (uintptr_t)draft_probs % dtype_size(draft_dtype)))
    SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: misaligned logits or draft_probs", what);
  const bool filtered = top_ks || top_ps || min_ps || (top_k > 0 && top_k < vocab) || top_p < 1.f || min_p > 0.f;
  const VerifyPlan p = verify_plan(n_rows, batch, vocab, filtered);
  if (!workspace || workspace_bytes < p.bytes)
    SUBSPEC_FAIL(SUBSPEC_ERR_WORKSPACE, "%s: workspace of %zu bytes is smaller than the %zu required", what, workspace_bytes, p.bytes);
  if ((uintptr_t)workspace % 16) SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: workspace must be 16-byte aligned", what);
  if (n_rows * p.slices > INT32_MAX || batch * p.end_slices > INT32_MAX)
    SUBSPEC_FAIL(SUBSPEC_ERR_LIMIT, "%s: too large (%lld rows of %lld)", what, (long long)n_rows, (long long)vocab);
  VerifyArgs a{};
  a.s = SampleArgs{logits, uniforms, temperatures, top_ks, top_ps, min_ps, tokens, probs, row_stride, (int)vocab, top_k, temperature, top_p, min_p};
  a.drafts = drafts; a.starts = query_starts; a.draws = draws; a.q = draft_probs; a.q_stride = draft_stride; a.accepted = accepted;
  char* ws = (char*)workspace;
  void* search = ws;
  ws += p.search;
  a.masses = (SliceMass*)ws; ws += p.masses;
  a.cuts = (RowCut*)ws; ws += p.cuts;
  a.ends = (EndRecord*)ws; ws += p.ends;
  a.sums = (RestSum*)ws;
  a.q_dtype = draft_dtype; a.slices = filtered ? 0 : p.slices; a.length = p.length; a.end_slices = p.end_slices; a.end_length = p.end_length;
  a.batch = (int)batch; a.n_rows = (int)n_rows;
  const int64_t es = (int64_t)dtype_size(dtype), qs = (int64_t)dtype_size(draft_dtype);
  a.wide = (uintptr_t)logits % 16 == 0 && row_stride * es % 16 == 0;
  a.q_wide = (uintptr_t)draft_probs % 16 == 0 && draft_stride * qs % 16 == 0;
  hipStream_t st = (hipStream_t)stream;
  if (filtered && n_rows > 0) launch_row_cuts(a.s, dtype, n_rows, a.cuts, search, st);
  if (dtype == SUBSPEC_F32) launch_verify<SUBSPEC_F32>(a, st);
  else if (dtype == SUBSPEC_F16) launch_verify<SUBSPEC_F16>(a, st);
  else launch_verify<SUBSPEC_BF16>(a, st);
  SUBSPEC_CHECK_HIP(hipGetLastError());
  return SUBSPEC_OK;
}
