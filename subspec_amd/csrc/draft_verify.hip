// Drafted tokens of a batch of sequences against the target's probabilities, from given numbers, for gfx950.
//
// Row i of a sequence's logits gives the distribution p_i of the token behind its token i (softmax at a temperature, after the filters of a draw, see
// sample.hip); the draft x_i behind it was drawn from q_i.  x_i stays if u_i q_i(x_i) < p_i(x_i), which happens with probability min(1, p_i / q_i); at the
// first that does not the next token is drawn from max(p_i - q_i, 0), after the last row from p itself.  What comes out is distributed like the target's own
// draws (Y. Leviathan, M. Kalman, Y. Matias, "Fast inference from transformers via speculative decoding", 2023).  A draft without q is one
// that nothing was drawn for: q_i(x_i) = 1.
//
// Masses are the whole numbers of a draw (2^-42 of the largest, see mass_series.h).  With m_j an entry's mass and Z the row's, the test is u q Z < m, and of the
// rest max(m_j - q_j Z, 0) the token is the first in the order of the vocabulary whose sum exceeds v times the whole.  The rest is whole numbers too, whose sums are exact: with
// filters every entry's is rounded, without them that of 512 entries (from exact sums of masses and a sum of q in 64 bits and a fixed order, see kOpen below), and
// within the 512 that the token falls to every entry's.
// 48 sequences of up to 8 drafts, 346 rows of 152064 bf16 (105 MB): the statistics of all rows 20.5 us (5.1 TB/s), acceptance and the end rows' masses 20.6, the draws 10.4; one sequence
// of 4 drafts in fp32 4.0 + 5.9 + 4.2.  With filters the cuts of all rows come first (sample.hip): 63 rows' 42 us are most of 16 sequences' 54.
#include "sample.h"
#include <algorithm>

namespace subspec {

constexpr int kVerifyThreads = 256;
constexpr int kVerifyWaves = kVerifyThreads / kWave;
constexpr int kVerifyRound = 8 * kVerifyThreads;       // entries that a workgroup takes at a time, eight a thread
constexpr int kChunk = 8 * kWave;                      // ... a wavefront: sums are kept of these
constexpr int kMostChunks = (1 << 20) / kChunk;

// A slice of a row without filters, in 32 bits: its largest logit, the masses relative to it, the first entry that equals it.
struct SliceStats {
  float top, sum;
  int first, unused;
};
// The row that a sequence ends with.
struct EndRecord {
  RowCut cut;                      // (its mass is that of the chunks: it counts for rows with filters)
  int row;                         // of the call (-1: the sequence has none)
  int last;                        // no draft stands behind it
  int draft;                       // ... or the one that did not stay (-1: none of the vocabulary)
};
struct VerifyArgs {
  SampleArgs s;
  const int64_t* drafts;
  const int32_t* starts;
  const float* draws;
  const void* q;
  int64_t q_stride;
  int32_t* accepted;
  RowCut* cuts;                    // of every row, with filters
  SliceStats* stats;               // [row][slices], without
  EndRecord* ends;
  uint64_t* all;                   // [sequence][chunks] masses of the row that it ends with
  uint64_t* part;                  // ... of the entries of which the draft leaves something (kOpen beside it: of some it is not clear whether)
  double* taken;                   // ... what the draft has of these, in probabilities: part - taken * the row's mass is left
  int q_dtype, slices, end_slices, end_length, chunks, batch, n_rows, wide, q_wide, filtered;
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
// ROUNDS chunks of a row of n entries from c0 on, `apart` entries from one to the next: lane l has entries 8 l .. 8 l + 7 of each, `fill` behind the row's end.  wide:
// rows start at multiples of 16 bytes.  All are asked for before the first is looked at, which takes that nothing branches between the requests: a lane's
// own end of the row is the business of the last chunk alone.
template <int DT, int ROUNDS>
__device__ __forceinline__ void load_chunks(const void* row, int c0, int apart, int n, int wide, float fill, float (&x)[ROUNDS][8]) {
  const int at = c0 + 8 * (int)(threadIdx.x & (kWave - 1));
  constexpr int kPieces = Elem<DT>::kBytes / 2;
  if (wide && c0 + (ROUNDS - 1) * apart + kChunk <= n) {                 // (uniform)
    dec_u4 raw[ROUNDS][kPieces];
#pragma unroll
    for (int k = 0; k < ROUNDS; ++k)
#pragma unroll
      for (int p = 0; p < kPieces; ++p) raw[k][p] = ((const dec_u4*)((const char*)row + (size_t)(at + k * apart) * Elem<DT>::kBytes))[p];
#pragma unroll
    for (int k = 0; k < ROUNDS; ++k) {
      if constexpr (DT == SUBSPEC_F32) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[k][e] = __uint_as_float(raw[k][e / 4][e % 4]);
      } else {
        unpack8<DT>(raw[k][0], x[k]);
      }
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < ROUNDS; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = at + k * apart + e;
      const float v = Elem<DT>::load(row, min(i, n - 1));
      x[k][e] = i < n ? v : fill;
    }
}
// the draft's probabilities of the same entries
template <int ROUNDS>
__device__ __forceinline__ void load_drafts(const VerifyArgs& a, int row, int draft, int c0, int apart, float (&x)[ROUNDS][8]) {
  const int n = a.s.vocab;
  if (!a.q) {
#pragma unroll
    for (int k = 0; k < ROUNDS; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) x[k][e] = c0 + k * apart + 8 * (int)(threadIdx.x & (kWave - 1)) + e == draft ? 1.f : 0.f;
  } else if (a.q_dtype == SUBSPEC_F32) {
    load_chunks<SUBSPEC_F32, ROUNDS>((const char*)a.q + row * a.q_stride * 4, c0, apart, n, a.q_wide, 0.f, x);
  } else if (a.q_dtype == SUBSPEC_F16) {
    load_chunks<SUBSPEC_F16, ROUNDS>((const char*)a.q + row * a.q_stride * 2, c0, apart, n, a.q_wide, 0.f, x);
  } else {
    load_chunks<SUBSPEC_BF16, ROUNDS>((const char*)a.q + row * a.q_stride * 2, c0, apart, n, a.q_wide, 0.f, x);
  }
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
// ... of eight entries from i on, without a branch an entry: what is 60 or more below the largest (in bits), and a NaN, is taken to be at 60, which rounds
// to nothing
template <int DT>
__device__ __forceinline__ void eight_masses(const float* l, int i, const RowCut& cut, const RowTop& top, const RowRule& r, const Series& series, double* m) {
  if (top.only) {                                                        // (uniform)
#pragma unroll
    for (int k = 0; k < 8; ++k) m[k] = l[k] == top.value ? (double)(1ull << kMassBits) : 0.0;
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const double x = fmax(((double)l[k] - top.wide) * r.inv_t_log2e, -60.0), n = rint(x);
      m[k] = ldexp(series(x - n), (int)n);
    }
  }
  if (r.min_p > 0.0) {
    const double least = r.min_p * (double)(1ull << kMassBits);
#pragma unroll
    for (int k = 0; k < 8; ++k) m[k] = m[k] < least ? 0.0 : m[k];
  }
  if (cut.last != ~0ull) {
#pragma unroll
    for (int k = 0; k < 8; ++k) m[k] = order_key<DT>(l[k], i + k) > cut.last ? 0.0 : m[k];
  }
}
__device__ __forceinline__ uint64_t block_sum_u64(uint64_t v, uint64_t* scratch) {
  v = wave_sum_u64(v);
  if ((threadIdx.x & (kWave - 1)) == 0) scratch[threadIdx.x / kWave] = v;
  __syncthreads();
  uint64_t sum = 0;
#pragma unroll
  for (int w = 0; w < kVerifyWaves; ++w) sum += scratch[w];
  __syncthreads();
  return sum;
}

// ---------------------------------------------------------------------------------------------------------------- rows without filters
// A row's mass in 32 bits says of nearly every draft whether it stays, so all rows are read once, as fast as they come; masses in 64 bits are worked out
// for the one row that a sequence ends with (and for a row whose draft the 32 bits leave undecided, see kUnsure).
// A slice is a wavefront's, so nobody waits for anybody.
constexpr int kSliceChunks = 4;
// (l - top) / (T ln 2), from half of top and twice 1 / (T ln 2).  The difference comes first, and of halves: products of logits and 1 / T can be of any size (a mask
// of -1e30, a T of 1e-20), and two of them leave nothing of it; so can the difference of two of the lowest and largest numbers.  (Beside the row's way out of memory it costs
// nothing: 20.5 us for 48 sequences' rows, as with one product less.)
__device__ __forceinline__ float bits_below(float l, float half_top, float twice) { return fmaf(l, 0.5f, -half_top) * twice; }
template <int DT>
__global__ __launch_bounds__(kVerifyThreads) void verify_stats_kernel(VerifyArgs a) {
  constexpr int ROUNDS = kSliceChunks, kLength = kSliceChunks * kChunk;
  const uint32_t unit = blockIdx.x * kVerifyWaves + threadIdx.x / kWave;
  const int row = __builtin_amdgcn_readfirstlane(unit / (uint32_t)a.slices), slice = (int)(unit - (uint32_t)row * a.slices), lane = threadIdx.x & (kWave - 1);
  if (row < a.starts[0] || row >= min(a.starts[a.batch], a.n_rows)) return;      // a row of no sequence, or none
  const char* src = verify_row<DT>(a, row);
  float of[ROUNDS][8], top = -INFINITY, sum = 0.f;
  load_chunks<DT, ROUNDS>(src, slice * kLength, kChunk, a.s.vocab, a.wide, -INFINITY, of);
  const RowRule r = row_rule(a.s, row);
  float* x = of[0];
#pragma unroll
  for (int e = 0; e < 8 * ROUNDS; ++e) top = fmaxf(top, x[e]);           // (a NaN never is)
  top = wave_max(top);
  int first = INT32_MAX;
  if (r.greedy || top == INFINITY) {                                   // only entries that equal the largest have mass
#pragma unroll
    for (int e = 8 * ROUNDS - 1; e >= 0; --e) {
      if (x[e] != top) continue;
      sum += 1.f;
      first = slice * kLength + 8 * lane + (e / 8) * kChunk + e % 8;
    }
    first = wave_min_i(first);
    sum = wave_sum(sum);
  } else if (top > -INFINITY) {
    const float twice = 2.f * (float)r.inv_t_log2e, half = 0.5f * top;
#pragma unroll
    for (int e = 0; e < 8 * ROUNDS; ++e) sum += __builtin_amdgcn_exp2f(bits_below(x[e], half, twice));
    sum = wave_sum(sum);
    if (sum != sum) {                                                  // there is a NaN, which has no mass
      sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8 * ROUNDS; ++e) sum += x[e] != x[e] ? 0.f : __builtin_amdgcn_exp2f(bits_below(x[e], half, twice));
      sum = wave_sum(sum);
    }
  }
  if (lane == 0) a.stats[unit] = SliceStats{top, sum, first, 0};
}

// A row from its slices (kRowLanes lanes; the same in all of them): the cut, with the mass relative to the largest and in 32 bits.
constexpr int kRowLanes = 16, kRowsAtOnce = kVerifyThreads / kRowLanes;
template <int DT>
__device__ RowCut row_from_slices(const VerifyArgs& a, int row, const RowRule& r) {
  const int lane = threadIdx.x % kRowLanes;
  const SliceStats* of = a.stats + (int64_t)row * a.slices;
  // (a row of up to 262144 in one trip to memory)
  constexpr int kHeld = 8;
  SliceStats held[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) held[i] = of[min(lane + i * kRowLanes, a.slices - 1)];
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kHeld; ++i) top = fmaxf(top, held[i].top);
  for (int s = lane + kHeld * kRowLanes; s < a.slices; s += kRowLanes) top = fmaxf(top, of[s].top);
#pragma unroll
  for (int o = kRowLanes / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, kWave));
  const float twice = 2.f * (float)r.inv_t_log2e, half = 0.5f * top;
  float z = 0.f;
  int first = INT32_MAX;
  auto add = [&](const SliceStats& m) {
    z = fmaf(m.sum, m.top == top ? 1.f : __builtin_amdgcn_exp2f(fmaxf(bits_below(m.top, half, twice), -200.f)), z);
    first = m.top == top ? min(first, m.first) : first;
  };
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
    if (lane + i * kRowLanes < a.slices) add(held[i]);
  for (int s = lane + kHeld * kRowLanes; s < a.slices; s += kRowLanes) add(of[s]);
#pragma unroll
  for (int o = kRowLanes / 2; o > 0; o >>= 1) {
    z += __shfl_xor(z, o, kWave);
    first = min(first, __shfl_xor(first, o, kWave));
  }
  if (top == -INFINITY) return RowCut{0.0, 0, top};
  if (r.greedy) return RowCut{1.0, order_key<DT>(top, first), top};      // the first of the largest alone
  return RowCut{(double)z, ~0ull, top};
}
// The row's mass in 64 bits (a workgroup)
template <int DT>
__device__ uint64_t exact_mass(const VerifyArgs& a, int row, const RowCut& cut, const RowTop& top, const RowRule& r, const Series& series,
                               uint64_t* scratch) {
  uint64_t sum = 0;
#pragma unroll 1
  for (int c = (int)threadIdx.x / kWave * kChunk; c < a.s.vocab; c += kVerifyRound) {
    float x[1][8];
    load_chunks<DT, 1>(verify_row<DT>(a, row), c, 0, a.s.vocab, a.wide, -INFINITY, x);
    double m[8];
    eight_masses<DT>(x[0], c + 8 * (int)(threadIdx.x & (kWave - 1)), cut, top, r, series, m);
#pragma unroll
    for (int k = 0; k < 8; ++k) sum += whole(m[k]);
  }
  return block_sum_u64(sum, scratch);
}

// ---------------------------------------------------------------------------------------------------------------- the row a sequence ends with
// What a draft leaves of an entry's mass
__device__ __forceinline__ uint64_t rest_of(double m, float q, double z) { return whole(fmax(fma(-draft_prob(q), z, m), 0.0)); }
// How far u q Z and m may be apart, relative to m, for 32 bits to say which is larger.  With d = (l - top) / (T ln 2) a term 2^d is off by 3 |d| 2^-24 ln 2
// (the difference's rounding, the product's, the factor's; what a slice's largest logit is below the row's is a part of d, with the same three) and 2^-23; 2^20 terms of a size below 2^-20 make no more than one, so by
// 20 * 3 * 2^-24 * 0.7 on average; a lane adds 32 terms, a wavefront 64 sums in a tree, a row 512 of these, 32 a
// lane: 2.5e-6 + 2^-23 + 74 * 2^-24 < 2^-17.
constexpr double kUnsure = 0x1p-17;
constexpr uint64_t kOpen = 1ull << 63;               // (a chunk's masses stay below 2^51)

// What the draft leaves of a row, sum over j of max(m_j - q_j Z, 0), takes Z, which is complete only when all slices have been seen; but which terms are above zero
// the mass in 32 bits says already, up to those within kUnsure of it, and the sum of these terms is sum m_j - Z sum q_j.  So a chunk keeps both
// sums, the row is read once, and a chunk that has a term too near to call is looked at again when Z is there (one or two of 300 where p and q
// are those of two models; a pass of its own for Z took 13 us of 56 for 48 rows of 152064).
// A workgroup a slice of that row.  Each looks for itself which drafts of the sequence stay (kRowsAtOnce rows at a time: few words, out of the caches), which
// is cheaper than a launch of its own for that; the first of a sequence's writes it down.  Then the masses of the slice's chunks, and where the
// row's mass is known (with filters) what the draft leaves of them.  One more workgroup is for the rows of nobody.
template <int DT, bool FILTERED, int ROUNDS>
__global__ __launch_bounds__(kVerifyThreads) void verify_end_kernel(VerifyArgs a) {
  __shared__ uint64_t scratch[kVerifyWaves];
  __shared__ RowCut cuts[kRowsAtOnce];
  __shared__ int stop;                                                  // 2 i: the sequence ends with row i; 2 i + 1: 32 bits do not say
  const int b = blockIdx.x / a.end_slices, slice = blockIdx.x % a.end_slices;
  if (b == a.batch) {
    const int begin = min(max(a.starts[0], 0), a.n_rows), behind = min(max(a.starts[a.batch], 0), a.n_rows);
    for (int t = threadIdx.x; t < a.n_rows; t += kVerifyThreads)
      if (t < begin || t >= behind) {
        a.s.tokens[t] = -1;
        a.s.probs[t] = 0.f;
      }
    return;
  }
  const VerifySpan sp = verify_span(a, b);
  if (sp.n == 0) {
    if (slice == 0 && threadIdx.x == 0) {
      a.accepted[b] = 0;
      a.ends[b].row = -1;
    }
    return;
  }
  const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1), end = slice == 0;
  const Series series;
  int base = 0, here;
  if (threadIdx.x == 0) stop = INT32_MAX;
  __syncthreads();
  for (;;) {
    const int i = base + (int)threadIdx.x / kRowLanes;
    if (i < sp.n) {
      const int row = sp.first + i, last = i == sp.n - 1;
      const RowRule r = row_rule(a.s, row);
      const int64_t x = last ? -1 : a.drafts[row + 1];
      const bool known = x >= 0 && x < a.s.vocab;
      const float l = known ? Elem<DT>::load(verify_row<DT>(a, row), x) : -INFINITY;
      const double q = !a.q ? 1.0 : known ? draft_prob(load_q(a, row, (int)x)) : 0.0;
      const RowCut cut = FILTERED ? a.cuts[row] : row_from_slices<DT>(a, row, r);
      if (threadIdx.x % kRowLanes == 0) {
        const double unit = FILTERED ? 1.0 : 0x1p-42;                    // (masses in 32 bits are relative to the largest)
        const double m = cut.mass > 0.0 ? kept_mass<DT>(l, (int)x, cut, row_top_of(cut.top, r), r, series) * unit : 0.0;
        const double goal = r.u * q * cut.mass;
        const bool unsure = !FILTERED && !r.greedy && !last && m > 0.0 && fabs(goal - m) <= kUnsure * m;
        if (unsure) atomicMin(&stop, 2 * i + 1);
        else if (last || !(goal < m)) atomicMin(&stop, 2 * i);
        if (end && !last) a.s.probs[row] = cut.mass > 0.0 ? (float)(m / cut.mass) : 0.f;
        cuts[threadIdx.x / kRowLanes] = cut;
      }
    }
    __syncthreads();
    here = stop;
    if (here == INT32_MAX) {                                             // (uniform) the next rows
      __syncthreads();
      base += kRowsAtOnce;
      continue;
    }
    if (FILTERED || !(here & 1)) break;
    const int row = sp.first + here / 2;
    const RowRule r = row_rule(a.s, row);
    const RowCut cut = cuts[here / 2 - base];
    const RowTop top = row_top_of(cut.top, r);
    const double z = (double)exact_mass<DT>(a, row, cut, top, r, series, scratch);
    const int64_t x = a.drafts[row + 1];                                 // (one of the vocabulary: it has mass)
    const double m = kept_mass<DT>(Elem<DT>::load(verify_row<DT>(a, row), x), (int)x, cut, top, r, series);
    if (!(r.u * (!a.q ? 1.0 : draft_prob(load_q(a, row, (int)x))) * z < m)) break;
    base = here / 2 + 1;
    if (threadIdx.x == 0) stop = INT32_MAX;                              // (all have read it: exact_mass has barriers)
    __syncthreads();
  }
  const int stays = here / 2, row = sp.first + stays, last = stays == sp.n - 1;
  const RowRule r = row_rule(a.s, row);
  const RowCut cut = cuts[stays - base];
  const int64_t x = last ? -1 : a.drafts[row + 1];
  const int draft = x >= 0 && x < a.s.vocab ? (int)x : -1;
  if (end) {
    for (int i = threadIdx.x; i < sp.n; i += kVerifyThreads) {          // (the row it ends with is the draw's)
      if (i < stays) {
        a.s.tokens[sp.first + i] = a.drafts[sp.first + i + 1];
      } else if (i > stays) {
        a.s.tokens[sp.first + i] = -1;
        a.s.probs[sp.first + i] = 0.f;
      }
    }
    if (threadIdx.x == 0) {
      a.accepted[b] = stays;
      a.ends[b] = EndRecord{cut, row, last, draft};
    }
  }
  const RowTop top = row_top_of(cut.top, r);
  const char* src = verify_row<DT>(a, row);
  // (all of the wavefront's entries asked for before the first is looked at)
  const int c0 = slice * a.end_length + wave * kChunk;
  float l[ROUNDS][8], q[ROUNDS][8];
  load_chunks<DT, ROUNDS>(src, c0, kVerifyRound, a.s.vocab, a.wide, -INFINITY, l);
  if (!last) load_drafts<ROUNDS>(a, row, draft, c0, kVerifyRound, q);
  const double z = FILTERED ? cut.mass : cut.mass * (double)(1ull << kMassBits);
#pragma unroll
  for (int k = 0; k < ROUNDS; ++k) {
    const int c = c0 + k * kVerifyRound;
    if (c >= a.s.vocab) break;
    uint64_t all = 0, part = 0;
    double m[8], taken = 0.0;
    bool open = false;
    eight_masses<DT>(l[k], c + 8 * lane, cut, top, r, series, m);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint64_t w = whole(m[e]);
      all += w;
      if (last) continue;
      if (FILTERED) {                                        // (the row's mass is known)
        part += rest_of(m[e], q[k][e], z);
      } else {
        const double p = draft_prob(q[k][e]), left = fma(-p, z, m[e]);
        const bool some = left > 0.0;
        part += some ? w : 0;
        taken += some ? p : 0.0;
        open |= fabs(left) < kUnsure * m[e];                  // (not where there is no mass: nothing is left of it)
      }
    }
    all = wave_sum_u64(all);
    part = wave_sum_u64(part);
    if (!FILTERED) {
      taken = wave_sum_f64(taken);
      if (__any(open) && !last) part |= kOpen;
    }
    if (lane == 0) {
      const int64_t at = (int64_t)b * a.chunks + c / kChunk;
      a.all[at] = all;
      a.part[at] = part;
      a.taken[at] = taken;
    }
  }
}

// The token: the chunk that the number falls into, then the entry.  A workgroup a sequence, whose wavefronts share the chunks that have to be looked at again;
// one of them finds the entry.
template <int DT>
__global__ __launch_bounds__(kVerifyThreads) void verify_draw_kernel(VerifyArgs a) {
  __shared__ uint64_t alls[kMostChunks], rests[kMostChunks], scratch[kVerifyWaves];
  const int b = blockIdx.x, lane = threadIdx.x & (kWave - 1);
  const EndRecord e = a.ends[b];
  if (e.row < 0) return;
  const RowRule r = row_rule(a.s, e.row);
  const RowTop top = row_top_of(e.cut.top, r);
  const Series series;
  const char* src = verify_row<DT>(a, e.row);
  const int64_t first = (int64_t)b * a.chunks;
  uint64_t z_units = 0;
  for (int c = threadIdx.x; c < a.chunks; c += kVerifyThreads) z_units += alls[c] = a.all[first + c];
  z_units = block_sum_u64(z_units, scratch);
  const double z = a.filtered ? e.cut.mass : (double)z_units;
  uint64_t rest = 0;
  if (!e.last) {
    for (int c = (int)threadIdx.x / kWave * kWave; c < a.chunks; c += kVerifyThreads) {
      const int at = c + lane;
      const uint64_t part = at < a.chunks ? a.part[first + at] : 0;
      const double left = (double)(part & ~kOpen) - z * (at < a.chunks ? a.taken[first + at] : 0.0);
      uint64_t mine = whole(fmax(left, 0.0));
      for (uint64_t open = __ballot(part >= kOpen); open; open &= open - 1) {                  // once more, with Z
        const int which = __ffsll((unsigned long long)open) - 1;
        float l[1][8], q[1][8];
        double m[8];
        load_chunks<DT, 1>(src, (c + which) * kChunk, 0, a.s.vocab, a.wide, -INFINITY, l);
        load_drafts<1>(a, e.row, e.draft, (c + which) * kChunk, 0, q);
        eight_masses<DT>(l[0], (c + which) * kChunk + 8 * lane, e.cut, top, r, series, m);
        uint64_t exact = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) exact += rest_of(m[k], q[0][k], z);
        exact = wave_sum_u64(exact);
        if (lane == which) mine = exact;
      }
      if (at < a.chunks) rests[at] = mine;
      rest += mine;
    }
    rest = block_sum_u64(rest, scratch);
  }
  __syncthreads();
  if (threadIdx.x >= kWave) return;
  const bool by_rest = rest > 0;
  const uint64_t* sums = by_rest ? rests : alls;
  // a lane has consecutive chunks
  const int per = (a.chunks + kWave - 1) / kWave, c0 = min(lane * per, a.chunks), c1 = min(c0 + per, a.chunks);
  uint64_t mine = 0;
  for (int c = c0; c < c1; ++c) mine += sums[c];
  const uint64_t upto = wave_scan_u64(mine), total = lane_u64(upto, kWave - 1);
  int64_t token = -1;
  float prob = 0.f;
  if (total > 0) {
    const float v = a.draws[b];
    const uint64_t goal = draw_goal(v > 0.f ? (double)v : 0.0, total);
    const int owner = __ffsll((unsigned long long)__ballot(goal < upto)) - 1;       // (the last lane's is the total)
    int chunk = c0;
    uint64_t before = upto - mine;
    for (; chunk + 1 < c1; ++chunk) {
      const uint64_t next = before + sums[chunk];
      if (goal < next) break;
      before = next;
    }
    chunk = __shfl(chunk, owner, kWave);
    uint64_t left = goal - __shfl((unsigned long long)before, owner, kWave);
    const int i = chunk * kChunk + 8 * lane;
    float l[1][8], q[1][8];
    load_chunks<DT, 1>(src, chunk * kChunk, 0, a.s.vocab, a.wide, -INFINITY, l);
    if (by_rest) load_drafts<1>(a, e.row, e.draft, chunk * kChunk, 0, q);
    uint64_t w[8], sum = 0;
    double m[8];
    eight_masses<DT>(l[0], i, e.cut, top, r, series, m);
#pragma unroll
    for (int k = 0; k < 8; ++k) sum += w[k] = by_rest ? rest_of(m[k], q[0][k], z) : whole(m[k]);
    const uint64_t here = wave_sum_u64(sum);
    if (here == 0) {                                           // (a chunk whose terms round to nothing, one by one: its masses)
      sum = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) sum += w[k] = whole(m[k]);
      left = 0;
    } else {
      left = min(left, here - 1);                              // (the chunk's sum was of its terms before rounding)
    }
    uint64_t at = wave_scan_u64(sum) - sum;
    const uint64_t hit = __ballot(at <= left && left < at + sum);
    double mass = 0.0;
    int k_hit = 0;
#pragma unroll
    for (int k = 7; k >= 0; --k) {
      const uint64_t ahead = at + (sum -= w[k]);                                    // mass before entry k
      if (ahead <= left && left < ahead + w[k]) {
        mass = m[k];
        k_hit = k;
      }
    }
    const int finder = hit ? __ffsll((unsigned long long)hit) - 1 : 0;
    if (hit) {
      token = __shfl(i + k_hit, finder, kWave);
      prob = __shfl((float)(mass / z), finder, kWave);
    }
  }
  if (lane == 0) {
    a.s.tokens[e.row] = token;
    a.s.probs[e.row] = prob;
  }
}

// Entries of a slice of the rows that sequences end with: one round of a workgroup's threads, two or four, while there are more workgroups than fit at once
static int verify_end_length(int64_t batch, int64_t vocab) {
  int64_t length = kVerifyRound;
  while (length < 4 * kVerifyRound && batch * ((vocab + 2 * length - 1) / (2 * length)) >= 768) length *= 2;
  return (int)length;
}

struct VerifyPlan {
  int slices, end_length, end_slices, chunks;
  size_t search, stats, cuts, ends, sums, bytes;
};
static VerifyPlan verify_plan(int64_t n_rows, int64_t batch, int64_t vocab, bool filtered) {
  VerifyPlan p{};
  p.slices = (int)((vocab + kSliceChunks * kChunk - 1) / (kSliceChunks * kChunk));
  p.end_length = verify_end_length(batch, vocab);
  p.end_slices = (int)((vocab + p.end_length - 1) / p.end_length);
  p.chunks = (int)((vocab + kChunk - 1) / kChunk);
  if (filtered && n_rows > 0) p.search = align_up(row_search_workspace(n_rows, vocab), 256);
  if (filtered) p.cuts = align_up((size_t)n_rows * sizeof(RowCut), 256);
  else p.stats = align_up((size_t)n_rows * p.slices * sizeof(SliceStats), 256);
  p.ends = align_up((size_t)batch * sizeof(EndRecord), 256);
  p.sums = align_up((size_t)batch * p.chunks * sizeof(uint64_t), 256);
  p.bytes = p.search + p.stats + p.cuts + p.ends + 3 * p.sums;
  return p;
}

template <int DT, int ROUNDS>
static void launch_ends(const VerifyArgs& a, hipStream_t st) {
  const dim3 block(kVerifyThreads), ends_and_nobody((unsigned)(a.batch * a.end_slices + 1));
  if (a.filtered) hipLaunchKernelGGL((verify_end_kernel<DT, true, ROUNDS>), ends_and_nobody, block, 0, st, a);
  else hipLaunchKernelGGL((verify_end_kernel<DT, false, ROUNDS>), ends_and_nobody, block, 0, st, a);
}
template <int DT>
static void launch_verify(const VerifyArgs& a, hipStream_t st) {
  if (!a.filtered && a.n_rows > 0) {
    DominantKernelTimer timer(st);
    const dim3 grid((unsigned)(((int64_t)a.n_rows * a.slices + kVerifyWaves - 1) / kVerifyWaves)), block(kVerifyThreads);
    hipLaunchKernelGGL(verify_stats_kernel<DT>, grid, block, 0, st, a);
  }
  if (a.end_length == kVerifyRound) launch_ends<DT, 1>(a, st);
  else if (a.end_length == 2 * kVerifyRound) launch_ends<DT, 2>(a, st);
  else launch_ends<DT, 4>(a, st);
  if (a.n_rows > 0) hipLaunchKernelGGL(verify_draw_kernel<DT>, dim3((unsigned)a.batch), dim3(kVerifyThreads), 0, st, a);
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
  // (a launch has below 2^32 threads; the other ones, of a workgroup a row or an end row's slice, are far below)
  if (!filtered && (n_rows * p.slices + kVerifyWaves - 1) / kVerifyWaves * kVerifyThreads > UINT32_MAX)
    SUBSPEC_FAIL(SUBSPEC_ERR_LIMIT, "%s: too large (%lld rows of %lld)", what, (long long)n_rows, (long long)vocab);
  VerifyArgs a{};
  a.s = SampleArgs{logits, uniforms, temperatures, top_ks, top_ps, min_ps, tokens, probs, row_stride, (int)vocab, top_k, temperature, top_p, min_p};
  a.drafts = drafts; a.starts = query_starts; a.draws = draws; a.q = draft_probs; a.q_stride = draft_stride; a.accepted = accepted;
  char* ws = (char*)workspace;
  void* search = ws;
  ws += p.search;
  a.stats = (SliceStats*)ws; ws += p.stats;
  a.cuts = (RowCut*)ws; ws += p.cuts;
  a.ends = (EndRecord*)ws; ws += p.ends;
  a.all = (uint64_t*)ws; ws += p.sums;
  a.part = (uint64_t*)ws; ws += p.sums;
  a.taken = (double*)ws;
  a.q_dtype = draft_dtype; a.slices = p.slices; a.end_slices = p.end_slices; a.end_length = p.end_length; a.chunks = p.chunks;
  a.batch = (int)batch; a.n_rows = (int)n_rows; a.filtered = filtered;
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
