// Sampling from a language model's logits after temperature, top-k, top-p and min-p, from one given number a row.
//
// Entries are ordered by logit, larger first, equal ones by index; entry j has the mass m_j = exp((l_j - l_max) / T).  Each filter keeps a
// prefix of that order: top-k the first k, top-p the entries with less than p times the mass of those k before them, min-p those with
// m_j >= min_p.  The token drawn is the first entry whose mass, added to that of all before it, exceeds u times the mass of what stays.
// So a row needs no sort: it needs the entry at a rank (top-k) and twice the entry at a mass (top-p, the draw).  A histogram of
// (l_max - l) / T with counts and masses says in which bin each of the three lies; the entries of those bins alone are put in order.
//
// Masses are whole numbers, round(m * 2^42), of an exponential evaluated in 64 bits: their sums are exact and do not depend on the
// order in which wavefronts add them, 2^20 entries stay below 2^62, and what rounds to zero (less than 2^-43 of the largest) is drawn with a
// probability below 2^-23 even if a million such entries are there.  In fp32 the sum over a flat row of 150000 entries is off by more
// than the step between two of them.
#include "common.h"
#include <algorithm>

namespace subspec {

constexpr int kSampleThreads = 1024;      // of a workgroup that has a whole row
constexpr int kSliceThreads = 512;        // ... a slice of one
constexpr int kBins = 1024;
constexpr int kMassBits = 42;
constexpr float kReach = 29.9f;           // 43 ln 2 = 29.81: masses beyond round to zero
constexpr int kCandidates = 4096;
constexpr int kSliceCandidates = 1024;

struct SampleArgs {
  const void* logits;
  const float* uniforms;
  const float* temperatures;     // null: the scalar below, for these four
  const int32_t* top_ks;
  const float* top_ps;
  const float* min_ps;
  int64_t* tokens;
  float* probs;
  int64_t row_stride;
  int vocab, top_k;
  float temperature, top_p, min_p;
};

// What a row is drawn with.
struct RowRule { double inv_t; float inv_tf; bool greedy; int k; double p, min_p, u; };
__device__ __forceinline__ RowRule row_rule(const SampleArgs& a, int row) {
  RowRule r;
  const float t = a.temperatures ? a.temperatures[row] : a.temperature;
  const int k = a.top_ks ? a.top_ks[row] : a.top_k;
  const float p = a.top_ps ? a.top_ps[row] : a.top_p, q = a.min_ps ? a.min_ps[row] : a.min_p, u = a.uniforms[row];
  r.greedy = !(t > 0.f);
  r.inv_t = r.greedy ? 1.0 : 1.0 / (double)t;
  r.inv_tf = (float)r.inv_t;
  r.k = r.greedy ? 1 : k <= 0 ? INT32_MAX : k;
  r.p = p < 1.f ? (double)p : 1.0;                       // (a NaN filters nothing)
  r.min_p = q > 0.f ? fmin((double)q, 1.0) : 0.0;
  r.u = u > 0.f ? (double)u : 0.0;
  return r;
}

// 2^x for x <= 0 times 2^42, rounded to a whole number: x = n + f, |f| <= 1/2, the Taylor series of e^(f ln 2) to the tenth power
// (remainder (ln 2 / 2)^11 / 11! = 2.2e-13 of the value).
__device__ __forceinline__ double exp2_part(double f) {
  const double y = f * 0.69314718055994530942;
  double s = 1.0 / 3628800.0;
  s = fma(s, y, 1.0 / 362880.0);
  s = fma(s, y, 1.0 / 40320.0);
  s = fma(s, y, 1.0 / 5040.0);
  s = fma(s, y, 1.0 / 720.0);
  s = fma(s, y, 1.0 / 120.0);
  s = fma(s, y, 1.0 / 24.0);
  s = fma(s, y, 1.0 / 6.0);
  s = fma(s, y, 0.5);
  s = fma(s, y, 1.0);
  return fma(s, y, 1.0);
}
// How far entry l is below the largest in units of T, in 32 bits: what the bins go by (falls as l rises, so bins keep the order; kReach or more,
// or NaN: no mass).  With T = 0 only entries that equal the largest are near.
__device__ __forceinline__ float entry_distance(float l, float top, const RowRule& r) {
  if (l == top) return 0.f;
  return r.greedy ? INFINITY : (top - l) * r.inv_tf;
}
__device__ __forceinline__ int bin_of(float d) { return min((int)(d * (kBins / kReach)), kBins - 1); }
// The mass of an entry less than about kReach below the largest, in units of 2^-42 and before rounding.
__device__ __forceinline__ double entry_mass(float l, float top, const RowRule& r) {
  const double x = l == top ? 0.0 : ((double)l - (double)top) * r.inv_t * 1.44269504088896340736, n = rint(x);
  return ldexp(exp2_part(x - n), (int)n + kMassBits);
}
__device__ __forceinline__ uint64_t whole(double m) { return (uint64_t)rint(m); }
// f(bin, mass before rounding, mass) for an entry that has any
template <typename F>
__device__ __forceinline__ void with_mass(float l, float top, const RowRule& r, F f) {
  const float d = entry_distance(l, top, r);
  if (!(d < kReach)) return;
  const double m = entry_mass(l, top, r);
  const uint64_t w = whole(m);
  if (w != 0) f(bin_of(d), m, w);
}
// larger logits first, then lower indexes: ascending 64-bit keys
__device__ __forceinline__ uint64_t order_key(float l, int i) {
  uint32_t b = __float_as_uint(l == 0.f ? 0.f : l);      // (-0 is 0)
  b = b >> 31 ? b : ~b & 0x7fffffffu;                     // larger first: positive values below, negative ones with the sign bit above
  return (uint64_t)b << 32 | (uint32_t)i;
}
__device__ __forceinline__ float key_logit(uint64_t key) {
  const uint32_t b = (uint32_t)(key >> 32);
  return __uint_as_float(b >> 31 ? b : ~b & 0x7fffffffu);
}

struct Hist {
  uint64_t mass[kBins];            // a bin's own, or inclusive sums after scan_bins
  uint32_t count[kBins];
};
struct Candidates {
  uint64_t key[kCandidates];
  uint64_t upto[kCandidates];      // inclusive mass over the ordered candidates
};
struct SampleShared {
  Hist bins;
  union {
    Candidates c;
    Hist digits;                   // a search without candidates
  };
  uint64_t wave_mass[kSampleThreads / kWave];
  uint32_t wave_count[kSampleThreads / kWave];
  float scratch[kSampleThreads / kWave];
  unsigned long long min_p_mass;
  int n_candidates;
};

__device__ __forceinline__ uint64_t wave_scan_u64(uint64_t v) {      // inclusive
  const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const uint64_t u = __shfl_up((unsigned long long)v, o, kWave);
    if (lane >= o) v += u;
  }
  return v;
}
__device__ __forceinline__ uint32_t wave_scan_u32(uint32_t v) {
  const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const uint32_t u = __shfl_up(v, o, kWave);
    if (lane >= o) v += u;
  }
  return v;
}

// counts and masses of the bins -> inclusive sums (all threads; ends with a barrier)
template <int THREADS>
__device__ void scan_bins(Hist& h, uint64_t* wave_mass, uint32_t* wave_count) {
  constexpr int kEach = kBins / THREADS;
  const int tid = threadIdx.x, wave = tid / kWave, lane = tid & (kWave - 1);
  uint64_t m[kEach], sum = 0;
  uint32_t c[kEach], n = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    m[i] = sum += h.mass[tid * kEach + i];
    c[i] = n += h.count[tid * kEach + i];
  }
  const uint64_t wm = wave_scan_u64(sum);
  const uint32_t wc = wave_scan_u32(n);
  if (lane == kWave - 1) {
    wave_mass[wave] = wm;
    wave_count[wave] = wc;
  }
  __syncthreads();
  uint64_t bm = wm - sum;
  uint32_t bc = wc - n;
  for (int w = 0; w < wave; ++w) {
    bm += wave_mass[w];
    bc += wave_count[w];
  }
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    h.mass[tid * kEach + i] = bm + m[i];
    h.count[tid * kEach + i] = bc + c[i];
  }
  __syncthreads();
}
template <int THREADS>
__device__ __forceinline__ void clear_hist(Hist& h) {
  for (int i = threadIdx.x; i < kBins; i += THREADS) {
    h.mass[i] = 0;
    h.count[i] = 0;
  }
}

// first bin whose inclusive mass (count) exceeds t, which one does (uniform; every thread searches)
__device__ __forceinline__ int bin_at(const Hist& h, bool by_count, uint64_t t) {
  int lo = 0, hi = kBins - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if ((by_count ? (uint64_t)h.count[mid] : h.mass[mid]) > t) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// f(logit, index) for a workgroup's part of a row: 16 bytes a load between the row's aligned addresses, four of them in flight a thread (one
// in flight is 16 KB a compute unit, which a round trip of a microsecond turns into 16 GB/s)
template <int DT, int THREADS, typename F>
__device__ __forceinline__ void each_entry(const void* row, int i0, int i1, F f) {
  constexpr int kVec = 16 / Elem<DT>::kBytes, kFlight = 4;
  const int tid = threadIdx.x;
  const size_t address = (size_t)(uintptr_t)row + (size_t)i0 * Elem<DT>::kBytes;
  const int first = min(i0 + (int)((16 - address % 16) % 16) / Elem<DT>::kBytes, i1);
  const int pieces = (i1 - first) / kVec, rest = first + pieces * kVec;
  if (i0 + tid < first) f(Elem<DT>::load(row, i0 + tid), i0 + tid);
  const dec_u4* src = (const dec_u4*)((const char*)row + (size_t)first * Elem<DT>::kBytes);
  for (int p0 = tid; p0 < pieces; p0 += kFlight * THREADS) {
    dec_u4 v[kFlight];
#pragma unroll
    for (int u = 0; u < kFlight; ++u) v[u] = src[min(p0 + u * THREADS, pieces - 1)];
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      const int p = p0 + u * THREADS, at = first + p * kVec;
      if (p >= pieces) break;
      if constexpr (DT == SUBSPEC_F32) {
#pragma unroll
        for (int e = 0; e < 4; ++e) f(__uint_as_float(v[u][e]), at + e);
      } else {
        float x[8];
        unpack8<DT>(v[u], x);
#pragma unroll
        for (int e = 0; e < 8; ++e) f(x[e], at + e);
      }
    }
  }
  if (rest + tid < i1) f(Elem<DT>::load(row, rest + tid), rest + tid);
}

// The bins of a part of a row, and the mass that min-p keeps of it (a thread's own, returned).  Counts are wanted with a top-k only.
template <int DT, int THREADS>
__device__ __forceinline__ uint64_t fill_bins(Hist& h, const void* row, int i0, int i1, int vocab, float top, const RowRule& r) {
  const double least = r.min_p * (double)(1ull << kMassBits);
  const bool counted = r.k < vocab;
  uint64_t kept = 0;
  each_entry<DT, THREADS>(row, i0, i1, [&](float l, int) {
    with_mass(l, top, r, [&](int bin, double m, uint64_t w) {
      atomicAdd((unsigned long long*)&h.mass[bin], (unsigned long long)w);
      if (counted) atomicAdd(&h.count[bin], 1u);
      if (!(m < least)) kept += w;
    });
  });
  return kept;
}

// Where the three entries can lie, from the bins alone: the mass of the top k is known up to the bin of its last entry, so the other two are
// intervals of bins.
struct BinRanges { int lo[3], hi[3]; bool by_k, by_p; };
__device__ __forceinline__ uint64_t below(const Hist& h, int b) { return b > 0 ? h.mass[b - 1] : 0; }
__device__ __forceinline__ uint64_t top_p_goal(double p, uint64_t z) { return (uint64_t)fmax(ceil(p * (double)z), 1.0) - 1; }
__device__ __forceinline__ uint64_t draw_goal(double u, uint64_t z) {
  const uint64_t t = (uint64_t)(u * (double)z);
  return z > 0 ? min(t, z - 1) : 0;
}
__device__ __forceinline__ BinRanges bin_ranges(const Hist& h, uint64_t min_p_mass, const RowRule& r) {
  BinRanges g;
  uint64_t z_lo = h.mass[kBins - 1], z_hi = z_lo;
  g.by_k = (uint32_t)r.k < h.count[kBins - 1];
  g.by_p = r.p < 1.0;
  g.lo[0] = g.lo[1] = 1;
  g.hi[0] = g.hi[1] = 0;
  if (g.by_k) {
    g.lo[0] = g.hi[0] = bin_at(h, true, (uint32_t)r.k - 1);
    z_lo = below(h, g.lo[0]) + 1;
    z_hi = h.mass[g.hi[0]];
  }
  if (g.by_p) {
    g.lo[1] = bin_at(h, false, top_p_goal(r.p, z_lo));
    g.hi[1] = bin_at(h, false, top_p_goal(r.p, z_hi));
    z_lo = below(h, g.lo[1]) + 1;
    z_hi = h.mass[g.hi[1]];
  }
  z_lo = min(z_lo, min_p_mass);
  z_hi = min(z_hi, min_p_mass);
  g.lo[2] = bin_at(h, false, draw_goal(r.u, z_lo));
  g.hi[2] = bin_at(h, false, draw_goal(r.u, z_hi));
  return g;
}
__device__ __forceinline__ bool in_ranges(const BinRanges& g, int b) {
  return (b >= g.lo[0] && b <= g.hi[0]) || (b >= g.lo[1] && b <= g.hi[1]) || (b >= g.lo[2] && b <= g.hi[2]);
}

// The entries of those bins in a part of a row; *n counts them, `most` of them are kept.
template <int DT, int THREADS>
__device__ __forceinline__ void gather(uint64_t* keys, int most, int* n, const void* row, int i0, int i1, float top, const RowRule& r,
                                       const BinRanges& g) {
  each_entry<DT, THREADS>(row, i0, i1, [&](float l, int i) {
    const float d = entry_distance(l, top, r);
    if (!(d < kReach) || !in_ranges(g, bin_of(d)) || whole(entry_mass(l, top, r)) == 0) return;
    const int at = atomicAdd(n, 1);
    if (at < most) keys[at] = order_key(l, i);
  });
}

// The candidates in order, with the inclusive sums of their masses (all threads; ends with a barrier).
__device__ void order_candidates(SampleShared& s, int n, float top, const RowRule& r) {
  const int tid = threadIdx.x, wave = tid / kWave, lane = tid & (kWave - 1);
  int size = kWave;
  while (size < n) size <<= 1;
  for (int i = tid; i < size; i += kSampleThreads)
    if (i >= n) s.c.key[i] = ~0ull;
  __syncthreads();
  for (int span = 2; span <= size; span <<= 1) {             // bitonic
    for (int step = span >> 1; step > 0; step >>= 1) {
      for (int i = tid; i < size / 2; i += kSampleThreads) {
        const int lo = (i & (step - 1)) | (i & ~(step - 1)) << 1, hi = lo | step;
        const uint64_t a = s.c.key[lo], b = s.c.key[hi];
        if ((a > b) == ((lo & span) == 0)) {
          s.c.key[lo] = b;
          s.c.key[hi] = a;
        }
      }
      __syncthreads();
    }
  }
  uint64_t before = 0;
  for (int i0 = 0; i0 < n; i0 += kSampleThreads) {
    const int i = i0 + tid;
    const uint64_t w = wave_scan_u64(i < n ? whole(entry_mass(key_logit(s.c.key[i]), top, r)) : 0);
    if (lane == kWave - 1) s.wave_mass[wave] = w;
    __syncthreads();
    uint64_t base = before;
    for (int v = 0; v < kSampleThreads / kWave; ++v) {
      if (v < wave) base += s.wave_mass[v];
      before += s.wave_mass[v];
    }
    if (i < n) s.c.upto[i] = base + w;
    __syncthreads();
  }
}

// The first entry in order whose rank (by_count) or inclusive mass exceeds t: its key, and the inclusive mass there.  (uniform)
struct Found { uint64_t key, upto; };
__device__ Found find_ordered(const SampleShared& s, int n, bool by_count, uint64_t t, float top, const RowRule& r) {
  const int b = bin_at(s.bins, by_count, t);
  int lo = 0, hi = n;                                         // first candidate of bin b
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (bin_of(entry_distance(key_logit(s.c.key[mid]), top, r)) >= b) hi = mid;
    else lo = mid + 1;
  }
  const uint64_t passed = below(s.bins, b) - (lo > 0 ? s.c.upto[lo - 1] : 0);        // mass before the bin that is not in the list
  if (by_count) {
    lo = min(lo + (int)(t - (b > 0 ? s.bins.count[b - 1] : 0)), n - 1);
  } else {
    hi = n - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (s.c.upto[mid] + passed > t) hi = mid;
      else lo = mid + 1;
    }
  }
  return Found{s.c.key[lo], s.c.upto[lo] + passed};
}

// The same over the whole row, for bins that hold more entries than the list (thousands of equal logits): digit by digit of the
// order's key, a pass over the row for each.
template <int DT>
__device__ Found find_in_row(SampleShared& s, const void* row, int vocab, bool by_count, uint64_t t, float top, const RowRule& r) {
  const int b = bin_at(s.bins, by_count, t);
  t -= by_count ? (uint64_t)(b > 0 ? s.bins.count[b - 1] : 0) : below(s.bins, b);
  uint64_t prefix = 0, upto = below(s.bins, b);
  const int shifts[6] = {54, 44, 34, 32, 10, 0}, widths[6] = {10, 10, 10, 2, 10, 10};        // 32 bits of the logit, 20 of the index
  for (int level = 0; level < 6; ++level) {
    const int shift = shifts[level], width = widths[level];
    __syncthreads();
    clear_hist<kSampleThreads>(s.digits);
    __syncthreads();
    each_entry<DT, kSampleThreads>(row, 0, vocab, [&](float l, int i) {
      const float d = entry_distance(l, top, r);
      if (!(d < kReach) || bin_of(d) != b) return;
      const uint64_t key = order_key(l, i);
      if (level > 0 && ((key ^ prefix) >> (shift + width)) != 0) return;
      const uint64_t m = whole(entry_mass(l, top, r));
      if (m == 0) return;
      const int digit = (int)(key >> shift) & ((1 << width) - 1);
      atomicAdd((unsigned long long*)&s.digits.mass[digit], (unsigned long long)m);
      atomicAdd(&s.digits.count[digit], 1u);
    });
    __syncthreads();
    scan_bins<kSampleThreads>(s.digits, s.wave_mass, s.wave_count);
    const int digit = bin_at(s.digits, by_count, t);
    t -= by_count ? (uint64_t)(digit > 0 ? s.digits.count[digit - 1] : 0) : below(s.digits, digit);
    upto += level == 5 ? s.digits.mass[digit] : below(s.digits, digit);
    prefix |= (uint64_t)digit << shift;
  }
  __syncthreads();
  return Found{prefix, upto};
}

// The row's token from the scanned bins and, where they fit, the candidates (n > kCandidates: they do not).
template <int DT>
__device__ void draw_row(SampleShared& s, const SampleArgs& a, int row_index, const void* row, float top, const RowRule& r, bool by_k, bool by_p,
                         uint64_t min_p_mass, int n) {
  const bool listed = n <= kCandidates;
  if (listed) order_candidates(s, n, top, r);
  auto find = [&](bool by_count, uint64_t t) {
    return listed ? find_ordered(s, n, by_count, t, top, r) : find_in_row<DT>(s, row, a.vocab, by_count, t, top, r);
  };
  uint64_t z = s.bins.mass[kBins - 1];
  if (by_k) z = find(true, (uint32_t)r.k - 1).upto;
  if (by_p) z = find(false, top_p_goal(r.p, z)).upto;
  z = min(z, min_p_mass);
  const Found drawn = find(false, draw_goal(r.u, z));
  if (threadIdx.x == 0) {
    a.tokens[row_index] = (int64_t)(uint32_t)drawn.key;
    a.probs[row_index] = (float)(entry_mass(key_logit(drawn.key), top, r) / (double)z);
  }
}
__device__ __forceinline__ void nothing_to_draw(const SampleArgs& a, int row_index) {
  if (threadIdx.x == 0) {
    a.tokens[row_index] = -1;
    a.probs[row_index] = 0.f;
  }
}

__device__ __forceinline__ float larger(float m, float l) { return l > m ? l : m; }      // a NaN never is
template <int DT>
__device__ __forceinline__ const void* row_of(const SampleArgs& a, int row_index) {
  return (const char*)a.logits + (int64_t)row_index * a.row_stride * Elem<DT>::kBytes;
}

// One workgroup a row, the row read three times: the largest, the bins, the entries of the bins that matter.
template <int DT>
__global__ __launch_bounds__(kSampleThreads) void sample_row_kernel(SampleArgs a) {
  __shared__ SampleShared s;
  const int row_index = blockIdx.x;
  const void* row = row_of<DT>(a, row_index);
  const RowRule r = row_rule(a, row_index);
  float top = -INFINITY;
  each_entry<DT, kSampleThreads>(row, 0, a.vocab, [&](float l, int) { top = larger(top, l); });
  top = block_max<kSampleThreads>(top, s.scratch);
  if (top == -INFINITY) return nothing_to_draw(a, row_index);              // (uniform)
  clear_hist<kSampleThreads>(s.bins);
  if (threadIdx.x == 0) {
    s.min_p_mass = 0;
    s.n_candidates = 0;
  }
  __syncthreads();
  const uint64_t kept = wave_scan_u64(fill_bins<DT, kSampleThreads>(s.bins, row, 0, a.vocab, a.vocab, top, r));
  if ((threadIdx.x & (kWave - 1)) == kWave - 1) atomicAdd(&s.min_p_mass, (unsigned long long)kept);
  __syncthreads();
  scan_bins<kSampleThreads>(s.bins, s.wave_mass, s.wave_count);
  const BinRanges g = bin_ranges(s.bins, s.min_p_mass, r);
  gather<DT, kSampleThreads>(s.c.key, kCandidates, &s.n_candidates, row, 0, a.vocab, top, r, g);
  __syncthreads();
  draw_row<DT>(s, a, row_index, row, top, r, g.by_k, g.by_p, s.min_p_mass, s.n_candidates);
}

// Few long rows: a row is cut into slices so that all compute units have a part of one, and the steps are launches: the slices' largest; their
// bins; the row's bins from its slices' (every slice adds them up for itself) and the candidates of a slice; the draw, a workgroup a row.
struct SliceRecord {
  Hist bins;
  unsigned long long min_p_mass;
  float top;
  int n_candidates;
  uint64_t key[kSliceCandidates];
};
struct RowRecord {
  Hist bins;                       // inclusive sums
  unsigned long long min_p_mass;
  int by_k, by_p;
};
struct SliceArgs {
  SliceRecord* slices;             // [rows][count]
  RowRecord* rows;
  int count, length;
};
template <int THREADS>
__device__ __forceinline__ float row_top(const SliceArgs& c, int row_index, float* scratch) {
  float top = -INFINITY;
  for (int i = threadIdx.x; i < c.count; i += THREADS) top = fmaxf(top, c.slices[(int64_t)row_index * c.count + i].top);
  return block_max<THREADS>(top, scratch);
}

template <int DT>
__global__ __launch_bounds__(kSliceThreads) void sample_top_kernel(SampleArgs a, SliceArgs c) {
  __shared__ float scratch[kSliceThreads / kWave];
  const int row_index = blockIdx.x / c.count, slice = blockIdx.x % c.count;
  float top = -INFINITY;
  each_entry<DT, kSliceThreads>(row_of<DT>(a, row_index), slice * c.length, min((slice + 1) * c.length, a.vocab),
                                [&](float l, int) { top = larger(top, l); });
  top = block_max<kSliceThreads>(top, scratch);
  if (threadIdx.x == 0) c.slices[blockIdx.x].top = top;
}

template <int DT>
__global__ __launch_bounds__(kSliceThreads) void sample_bins_kernel(SampleArgs a, SliceArgs c) {
  __shared__ Hist h;
  __shared__ float scratch[kSliceThreads / kWave];
  __shared__ unsigned long long min_p_mass;
  const int row_index = blockIdx.x / c.count, slice = blockIdx.x % c.count;
  clear_hist<kSliceThreads>(h);
  if (threadIdx.x == 0) min_p_mass = 0;
  const RowRule r = row_rule(a, row_index);
  const float top = row_top<kSliceThreads>(c, row_index, scratch);          // (its barriers also stand between the clearing and the sums)
  const uint64_t kept = wave_scan_u64(fill_bins<DT, kSliceThreads>(h, row_of<DT>(a, row_index), slice * c.length,
                                                                   min((slice + 1) * c.length, a.vocab), a.vocab, top, r));
  if ((threadIdx.x & (kWave - 1)) == kWave - 1) atomicAdd(&min_p_mass, (unsigned long long)kept);
  __syncthreads();
  SliceRecord& out = c.slices[blockIdx.x];
  for (int i = threadIdx.x; i < kBins; i += kSliceThreads) {
    out.bins.mass[i] = h.mass[i];
    out.bins.count[i] = h.count[i];
  }
  if (threadIdx.x == 0) out.min_p_mass = min_p_mass;
}

template <int DT>
__global__ __launch_bounds__(kSliceThreads) void sample_gather_kernel(SampleArgs a, SliceArgs c) {
  __shared__ Hist h;
  __shared__ float scratch[kSliceThreads / kWave];
  __shared__ uint64_t wave_mass[kSliceThreads / kWave];
  __shared__ uint32_t wave_count[kSliceThreads / kWave];
  __shared__ int n;
  const int row_index = blockIdx.x / c.count, slice = blockIdx.x % c.count;
  if (threadIdx.x == 0) n = 0;
  const RowRule r = row_rule(a, row_index);
  const SliceRecord* of = c.slices + (int64_t)row_index * c.count;
  const float top = row_top<kSliceThreads>(c, row_index, scratch);
  if (top == -INFINITY) return;                                             // (uniform) the last launch says so
  for (int i = threadIdx.x; i < kBins; i += kSliceThreads) {
    uint64_t m = 0;
    uint32_t k = 0;
#pragma unroll 8
    for (int j = 0; j < c.count; ++j) {
      m += of[j].bins.mass[i];
      k += of[j].bins.count[i];
    }
    h.mass[i] = m;
    h.count[i] = k;
  }
  uint64_t kept = 0;
  for (int j = 0; j < c.count; ++j) kept += of[j].min_p_mass;
  __syncthreads();
  scan_bins<kSliceThreads>(h, wave_mass, wave_count);
  const BinRanges g = bin_ranges(h, kept, r);
  SliceRecord& out = c.slices[blockIdx.x];
  gather<DT, kSliceThreads>(out.key, kSliceCandidates, &n, row_of<DT>(a, row_index), slice * c.length, min((slice + 1) * c.length, a.vocab), top, r, g);
  if (slice == 0) {
    RowRecord& rec = c.rows[row_index];
    for (int i = threadIdx.x; i < kBins; i += kSliceThreads) {
      rec.bins.mass[i] = h.mass[i];
      rec.bins.count[i] = h.count[i];
    }
    if (threadIdx.x == 0) {
      rec.min_p_mass = kept;
      rec.by_k = g.by_k;
      rec.by_p = g.by_p;
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) out.n_candidates = n;
}

template <int DT>
__global__ __launch_bounds__(kSampleThreads) void sample_draw_kernel(SampleArgs a, SliceArgs c) {
  __shared__ SampleShared s;
  const int row_index = blockIdx.x;
  const RowRule r = row_rule(a, row_index);
  const SliceRecord* of = c.slices + (int64_t)row_index * c.count;
  const float top = row_top<kSampleThreads>(c, row_index, s.scratch);
  if (top == -INFINITY) return nothing_to_draw(a, row_index);               // (uniform)
  const RowRecord& rec = c.rows[row_index];
  for (int i = threadIdx.x; i < kBins; i += kSampleThreads) {
    s.bins.mass[i] = rec.bins.mass[i];
    s.bins.count[i] = rec.bins.count[i];
  }
  int n = 0;
  bool whole_list = true;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
  for (int j = 0; j < c.count; ++j) {                                       // a wavefront a slice
    const int some = of[j].n_candidates;
    whole_list = whole_list && some <= kSliceCandidates && n + some <= kCandidates;
    if (whole_list && j % (kSampleThreads / kWave) == wave)
      for (int i = lane; i < some; i += kWave) s.c.key[n + i] = of[j].key[i];
    n += some;
  }
  __syncthreads();
  draw_row<DT>(s, a, row_index, row_of<DT>(a, row_index), top, r, rec.by_k, rec.by_p, rec.min_p_mass, whole_list ? n : kCandidates + 1);
}

// Slices a row is cut into: as many as give every compute unit two, of 4096 entries and more, 32 at most (each adds up the bins of all); 1:
// the row stays whole, which is one launch in the place of four.
static int sample_slices(int64_t rows, int64_t vocab) {
  if (vocab < 16384 || rows >= 512) return 1;
  return (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(512 / rows, 32), vocab / 4096));
}

}  // namespace subspec

using namespace subspec;

extern "C" size_t subspec_sample_filtered_workspace(int64_t rows, int64_t vocab) {
  if (rows < 1 || vocab < 1 || vocab > (1 << 20)) return 256;
  const int count = sample_slices(rows, vocab);
  if (count == 1) return 256;
  return 256 + align_up((size_t)rows * count * sizeof(SliceRecord), 256) + (size_t)rows * sizeof(RowRecord);
}

extern "C" int subspec_sample_filtered(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t row_stride, const float* uniforms,
                                       const float* temperatures, float temperature, const int32_t* top_ks, int32_t top_k,
                                       const float* top_ps, float top_p, const float* min_ps, float min_p, void* workspace,
                                       size_t workspace_bytes, int64_t* tokens, float* probs, void* stream) {
  const char* what = "sample_filtered";
  if (!dtype_ok(dtype)) SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: dtype %d not supported", what, dtype);
  if (rows < 0 || rows > (1 << 20)) SUBSPEC_FAIL(SUBSPEC_ERR_LIMIT, "%s: rows=%lld outside [0, 2^20]", what, (long long)rows);
  if (vocab < 1 || vocab > (1 << 20)) SUBSPEC_FAIL(SUBSPEC_ERR_LIMIT, "%s: vocab=%lld outside [1, 2^20]", what, (long long)vocab);
  if (row_stride < vocab) SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: rows of %lld logits are %lld apart", what, (long long)vocab, (long long)row_stride);
  if (rows == 0) return SUBSPEC_OK;
  if (!logits || !uniforms || !tokens || !probs) SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: null pointer argument", what);
  if ((uintptr_t)logits % dtype_size(dtype)) SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: misaligned logits", what);
  const size_t need = subspec_sample_filtered_workspace(rows, vocab);
  if (need > 256 && (!workspace || workspace_bytes < need))
    SUBSPEC_FAIL(SUBSPEC_ERR_WORKSPACE, "%s: workspace of %zu bytes is smaller than the %zu required", what, workspace_bytes, need);
  if ((uintptr_t)workspace % 16) SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: workspace must be 16-byte aligned", what);
  const SampleArgs a{logits, uniforms, temperatures, top_ks, top_ps, min_ps, tokens, probs, row_stride, (int)vocab, top_k, temperature, top_p, min_p};
  SliceArgs c;
  c.count = sample_slices(rows, vocab);
  c.length = (int)((vocab + c.count - 1) / c.count);
  c.slices = (SliceRecord*)workspace;
  c.rows = (RowRecord*)((char*)workspace + align_up((size_t)rows * c.count * sizeof(SliceRecord), 256));
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)rows), slices((unsigned)(rows * c.count));
#define SUBSPEC_SAMPLE(DT)                                                                                                 \
  do {                                                                                                                     \
    if (c.count == 1) {                                                                                                    \
      DominantKernelTimer timer(st);                                                                                       \
      hipLaunchKernelGGL(sample_row_kernel<DT>, grid, dim3(kSampleThreads), 0, st, a);                                     \
    } else {                                                                                                               \
      hipLaunchKernelGGL(sample_top_kernel<DT>, slices, dim3(kSliceThreads), 0, st, a, c);                                 \
      {                                                                                                                    \
        DominantKernelTimer timer(st);                                                                                     \
        hipLaunchKernelGGL(sample_bins_kernel<DT>, slices, dim3(kSliceThreads), 0, st, a, c);                              \
      }                                                                                                                    \
      hipLaunchKernelGGL(sample_gather_kernel<DT>, slices, dim3(kSliceThreads), 0, st, a, c);                              \
      hipLaunchKernelGGL(sample_draw_kernel<DT>, grid, dim3(kSampleThreads), 0, st, a, c);                                 \
    }                                                                                                                      \
  } while (0)
  if (dtype == SUBSPEC_F32) SUBSPEC_SAMPLE(SUBSPEC_F32);
  else if (dtype == SUBSPEC_F16) SUBSPEC_SAMPLE(SUBSPEC_F16);
  else SUBSPEC_SAMPLE(SUBSPEC_BF16);
#undef SUBSPEC_SAMPLE
  SUBSPEC_CHECK_HIP(hipGetLastError());
  return SUBSPEC_OK;
}
