// Sampling from a language model's logits after temperature, top-k, top-p and min-p, from one given number a row.
//
// Entries are ordered by logit, larger first, equal ones by index; entry j has the mass m_j = exp((l_j - l_max) / T).  Each filter keeps a
// prefix of that order: top-k the first k, top-p the entries with less than p times the mass of those k before them, min-p those with
// m_j >= min_p.  The token drawn is the first entry whose mass, added to that of all before it, exceeds u times the mass of what stays.
// So a row needs no sort: it needs the entry at a rank (top-k) and twice the entry at a mass (top-p, the draw).  A histogram of
// (l_max - l) / T with counts and masses says in which bin each of the three lies; the entries of those bins alone are put in order.
//
// Masses are whole numbers, m * 2^42 rounded, of an exponential evaluated in 64 bits (within 0.54 of such a unit, see mass_series.h): their sums are
// exact and do not depend on the order in which wavefronts add them, 2^20 entries stay below 2^62, and what rounds to zero (less than 2^-43 of the
// largest) is drawn with a probability below 2^-23 even if a million such entries are there.  In fp32 the sum over a flat row of 150000 entries is off
// by more than the step between two of them.
// One row of 152064 fp32: 28 us, four dependent launches of 3 + 7 + 10 + 8; 64 rows bf16 (19.5 MB): 50, the largest 6, the exponentials in 64 bits
// 16, the sums of the slices' bins and the second pass 15, the search among the candidates 15.
// A row of more candidates than kCandidates (or a slice's share of them) is searched by one workgroup, which reads it again for every ten bits of
// every search: 152064 logits of deviation 2 at T = 3 and top-p 0.95 310 us (32 at T = 1; a row of bf16 46), 64 rows of bf16 363 to 382 (55); rows of equal logits
// 0.65 to 1.3 ms, with a top-k of 70000 and a top-p 3.5.
#include "sample.h"
#include <algorithm>

namespace subspec {

constexpr int kSampleThreads = 1024;      // of a workgroup that has a whole row
constexpr int kSliceThreads = 512;        // ... a slice of one
constexpr int kBins = 1024;
constexpr int kCandidates = 4096;
constexpr int kSliceCandidates = 2048;

__device__ __forceinline__ int bin_of(float d) { return (int)(d * (0.999999f * kBins / kReach)); }      // (below kBins, rounding or not)

struct Hist {
  uint64_t mass[kBins];            // a bin's own, or inclusive sums after scan_bins
  uint32_t count[kBins];
};
// What a search works with.
struct Search {
  Hist digits;
  uint64_t wave_mass[kSampleThreads / kWave];
  uint32_t wave_count[kSampleThreads / kWave];
  uint64_t list[kWave];
  uint64_t key, upto;              // its answer
  int n;
};

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

// First index below n at which `over` holds (it then holds behind it too); n if nowhere.  64 probes at a time: two or three trips to LDS where
// halving takes ten to twelve.  (Every wavefront searches for itself; all its lanes are active.)
template <typename F>
__device__ __forceinline__ int first_over(int n, F over) {
  const int lane = threadIdx.x & (kWave - 1);
  int lo = 0, hi = n;                                         // the answer lies in [lo, hi]
  while (hi > lo) {
    const int step = (hi - lo + kWave - 1) / kWave, at = lo + (lane + 1) * step - 1;        // the last of the lane's stretch
    const uint64_t hit = __ballot(at >= hi || over(min(at, hi - 1)));
    const int f = hit ? __ffsll((unsigned long long)hit) - 1 : kWave;
    if (step == 1) return min(lo + f, hi);
    hi = min(lo + (f + 1) * step - 1, hi);                    // (its last one is over, or there is none: the answer is at most there)
    lo = min(lo + f * step, hi);
  }
  return lo;
}
// first bin whose inclusive mass (count) exceeds t, which one does
__device__ __forceinline__ int bin_at(const Hist& h, bool by_count, uint64_t t) {
  return min(first_over(kBins, [&](int i) { return (by_count ? (uint64_t)h.count[i] : h.mass[i]) > t; }), kBins - 1);
}

// A workgroup's part [i0, i1) of a row: pieces of 16 bytes between the row's aligned addresses, and the ragged ends, less than a piece each.
template <int DT>
struct Part {
  static constexpr int kVec = 16 / Elem<DT>::kBytes;
  const void* row;
  const dec_u4* src;
  int i0, i1, first, pieces, rest;
  __device__ __forceinline__ Part(const void* r, int b, int e) : row(r), i0(b), i1(e) {
    const size_t address = (size_t)(uintptr_t)row + (size_t)i0 * Elem<DT>::kBytes;
    first = min(i0 + (int)((16 - address % 16) % 16) / Elem<DT>::kBytes, i1);
    pieces = (i1 - first) / kVec;
    rest = first + pieces * kVec;
    src = (const dec_u4*)((const char*)row + (size_t)first * Elem<DT>::kBytes);
  }
  __device__ __forceinline__ dec_u4 piece(int p) const {                  // (past the end: the last one again)
    return pieces > 0 ? src[min(p, pieces - 1)] : dec_u4{0, 0, 0, 0};
  }
  template <int THREADS, typename F>
  __device__ __forceinline__ void ends(F f) const {
#pragma unroll 1
    for (int e = threadIdx.x; e < first - i0 + i1 - rest; e += THREADS) {
      const int i = e < first - i0 ? i0 + e : rest + e - (first - i0);
      f(Elem<DT>::load(row, i), i);
    }
  }
};
// A thread's pieces of a part of a row, the first two asked for where this is made, before what has to be known of the row is (four or six: no faster).
template <int DT, int THREADS>
struct Pieces {
  const Part<DT> part;
  dec_u4 next[2];
  __device__ __forceinline__ Pieces(const void* row, int i0, int i1) : part(row, i0, i1) {
#pragma unroll
    for (int u = 0; u < 2; ++u) next[u] = part.piece(threadIdx.x + u * THREADS);
  }
  // the piece of turn p, and one more asked for
  __device__ __forceinline__ dec_u4 take(int p) {
    const dec_u4 v = next[0];
    next[0] = next[1];
    next[1] = part.piece(p + 2 * THREADS);
    return v;
  }
};
// f(logit, index) for a part of a row, the next pieces asked for before the last are worked on.  One copy of f in the code (two for pairs of 16-bit
// logits): it is long, and a slice takes few turns.
template <int DT, int THREADS, typename F>
__device__ __forceinline__ void each_entry(Pieces<DT, THREADS>& pieces, F f) {
  const Part<DT>& part = pieces.part;
#pragma unroll 1
  for (int p = threadIdx.x; p < part.pieces; p += THREADS) {
    dec_u4 v = pieces.take(p);
#pragma unroll 1
    for (int j = 0; j < 4; ++j) {
      const uint32_t bits = v[0];
      v = dec_u4{v[1], v[2], v[3], bits};
      if constexpr (DT == SUBSPEC_F32) {
        f(__uint_as_float(bits), part.first + p * 4 + j);
      } else {
        float x[2];
        unpack2<DT>(bits, x);
        f(x[0], part.first + p * 8 + 2 * j);
        f(x[1], part.first + p * 8 + 2 * j + 1);
      }
    }
  }
  part.template ends<THREADS>(f);
}
// The largest of a part of a row (a thread's own)
template <int DT, int THREADS>
__device__ __forceinline__ float part_top(const void* row, int i0, int i1) {
  constexpr int kFlight = 4;
  const Part<DT> part(row, i0, i1);
  float top = -INFINITY;
  for (int p0 = threadIdx.x; p0 < part.pieces; p0 += kFlight * THREADS) {
    dec_u4 v[kFlight];
#pragma unroll
    for (int u = 0; u < kFlight; ++u) v[u] = part.piece(p0 + u * THREADS);
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      if constexpr (DT == SUBSPEC_F32) {
#pragma unroll
        for (int e = 0; e < 4; ++e) top = larger(top, __uint_as_float(v[u][e]));
      } else {
        float x[8];
        unpack8<DT>(v[u], x);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = larger(top, x[e]);
      }
    }
  }
  part.template ends<THREADS>([&](float l, int) { top = larger(top, l); });
  return top;
}

// The bins of a part of a row, and the mass that min-p keeps of it (a thread's own, returned).  Counts are wanted with a top-k only.
template <int DT, int THREADS>
__device__ __forceinline__ uint64_t fill_bins(Hist& h, Pieces<DT, THREADS>& pieces, int vocab, const RowTop& top, const RowRule& r) {
  const double least = r.min_p * (double)(1ull << kMassBits);
  const bool counted = r.k < vocab, sorted_out = r.min_p > 0.0;
  const Series series;
  uint64_t kept = 0;
  each_entry<DT, THREADS>(pieces, [&](float l, int) {
    const float d = entry_distance(l, top, r);
    if (!(d < kReach)) return;
    const double m = entry_mass(l, top, r, series);
    const uint64_t w = whole(m);
    const int bin = bin_of(d);
    atomicAdd((unsigned long long*)&h.mass[bin], (unsigned long long)w);
    if (counted) atomicAdd(&h.count[bin], 1u);
    if (sorted_out) kept += m < least ? 0 : w;
  });
  return kept;
}

// Where the three entries can lie, from the bins alone: the mass of the top k is known up to the bin of its last entry, so the other two are
// intervals of bins.
struct BinRanges { int lo[3], hi[3]; bool by_k, by_p; };
__device__ __forceinline__ uint64_t below(const Hist& h, int b) { return b > 0 ? h.mass[b - 1] : 0; }
__device__ __forceinline__ uint64_t top_p_goal(double p, uint64_t z) { return (uint64_t)fmax(ceil(p * (double)z), 1.0) - 1; }
template <bool DRAW>
__device__ __forceinline__ BinRanges bin_ranges(const Hist& h, uint64_t min_p_mass, const RowRule& r) {      // (min_p_mass counts with a min-p only)
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
  if constexpr (!DRAW) {
    g.lo[2] = 1;
    g.hi[2] = 0;
    return g;
  }
  if (r.min_p > 0.0) {
    z_lo = min(z_lo, min_p_mass);
    z_hi = min(z_hi, min_p_mass);
  }
  g.lo[2] = bin_at(h, false, draw_goal(r.u, z_lo));
  g.hi[2] = bin_at(h, false, draw_goal(r.u, z_hi));
  return g;
}
__device__ __forceinline__ bool in_ranges(const BinRanges& g, int b) {
  return (b >= g.lo[0] && b <= g.hi[0]) || (b >= g.lo[1] && b <= g.hi[1]) || (b >= g.lo[2] && b <= g.hi[2]);
}

// The entries of those bins in a part of a row; *n counts them, `most` of them are kept.  Few are, so a piece is first looked over in 32 bits:
// within a bin of one of the ranges, |top - l - centre| <= width, nine instructions an entry (a NaN, and infinities among them, passes).
template <int DT, int THREADS, bool DRAW>
__device__ __forceinline__ void gather(uint64_t* keys, int most, int* n, Pieces<DT, THREADS>& pieces, const RowTop& top, const RowRule& r,
                                       const BinRanges& g) {
  if (!DRAW && !g.by_k && !g.by_p) return;                                // (uniform: nothing is looked for)
  float centre[3], width[3];
  const float bin = kReach / kBins / r.inv_t;                             // width of a bin in logits
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    centre[k] = 0.5f * (float)(g.lo[k] + g.hi[k] + 1) * bin;
    width[k] = g.lo[k] > g.hi[k] ? -1.f : (0.5f * (float)(g.hi[k] - g.lo[k] + 1) + 1.f) * bin;
  }
  auto near = [&](float l) {
    const float x = top.value - l;
    return !(fabsf(x - centre[0]) > width[0]) || !(fabsf(x - centre[1]) > width[1]) || (DRAW && !(fabsf(x - centre[2]) > width[2]));
  };
  auto take = [&](float l, int i) {
    const float d = entry_distance(l, top, r);
    if (!(d < kReach) || !in_ranges(g, bin_of(d))) return;
    const int at = atomicAdd(n, 1);
    if (at < most) keys[at] = order_key<DT>(l, i);
  };
  constexpr int kVec = 16 / Elem<DT>::kBytes;
  const Part<DT>& part = pieces.part;
#pragma unroll 1
  for (int p = threadIdx.x; p < part.pieces; p += THREADS) {
    const dec_u4 v = pieces.take(p);
    float x[kVec];
    if constexpr (DT == SUBSPEC_F32) {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = __uint_as_float(v[e]);
    } else {
      unpack8<DT>(v, x);
    }
    uint32_t hits = 0;
#pragma unroll
    for (int e = 0; e < kVec; ++e) hits |= (near(x[e]) ? 1u : 0u) << e;
    if (top.only) hits = (1u << kVec) - 1;
    while (hits) {                                                        // (one turn for most wavefronts that have any)
      const int e = __ffs(hits) - 1;
      hits &= hits - 1;
      float l = x[0];
#pragma unroll
      for (int k = 1; k < kVec; ++k) l = e == k ? x[k] : l;
      take(l, part.first + p * kVec + e);
    }
  }
  part.template ends<THREADS>(take);
}

// The first entry in order whose rank (by_count) or inclusive mass exceeds t: its key, and the inclusive mass there.  `each` hands its argument
// the keys among which the entries of that bin are (all threads; ends with a barrier).  While more than 64 are left, the next ten bits of the
// keys tell them apart by a histogram like the bins'; 64 are put in order by one wavefront.
struct Found { uint64_t key, upto; };
template <int DT, int THREADS, typename Each>
__device__ Found find_entry(Search& s, const Hist& bins, bool by_count, uint64_t t, const RowTop& top, const RowRule& r, int most, Each each) {
  const Series series;
  const int b = bin_at(bins, by_count, t);
  uint64_t prefix = 0, upto = below(bins, b);
  t -= by_count ? (uint64_t)(b > 0 ? bins.count[b - 1] : 0) : upto;
  // the keys of a bin (and of its neighbours, for what rounding there is) agree in their leading bits
  const float wide = kReach / kBins / r.inv_t;
  const uint64_t first = order_key<DT>(top.only ? top.value : top.value - (float)(b - 1) * wide, 0);
  const uint64_t last = order_key<DT>(top.only ? top.value : top.value - (float)(b + 2) * wide, (1 << 20) - 1);
  int shift = 64 - __clzll((long long)((first ^ last) | 1));
  prefix = last >> shift << shift;
  int left = most <= kWave ? 0 : most;                        // at most how many there are (0: look)
  auto mine = [&](uint64_t key) { return (key ^ prefix) >> shift == 0 && bin_of(entry_distance(key_logit<DT>(key), top, r)) == b; };
  for (;;) {
    if (left <= kWave) {
      if (threadIdx.x == 0) s.n = 0;
      __syncthreads();
      each([&](uint64_t key) {
        if (!mine(key)) return;
        const int at = atomicAdd(&s.n, 1);
        if (at < kWave) s.list[at] = key;
      });
      __syncthreads();
      left = s.n;
      if (left <= kWave) break;
    }
    clear_hist<THREADS>(s.digits);
    __syncthreads();
    const int width = min(10, shift), next = shift - width;
    each([&](uint64_t key) {
      if (!mine(key)) return;
      const int digit = (int)(key >> next) & ((1 << width) - 1);
      atomicAdd((unsigned long long*)&s.digits.mass[digit], (unsigned long long)whole(entry_mass(key_logit<DT>(key), top, r, series)));
      atomicAdd(&s.digits.count[digit], 1u);
    });
    __syncthreads();
    scan_bins<THREADS>(s.digits, s.wave_mass, s.wave_count);
    const int digit = bin_at(s.digits, by_count, t);
    const uint32_t ahead = digit > 0 ? s.digits.count[digit - 1] : 0;
    left = (int)(s.digits.count[digit] - ahead);
    t -= by_count ? (uint64_t)ahead : below(s.digits, digit);
    upto += below(s.digits, digit);
    prefix |= (uint64_t)digit << next;
    shift = next;
    __syncthreads();
  }
  if (threadIdx.x < kWave) {
    const int lane = threadIdx.x;
    uint64_t k = lane < left ? s.list[lane] : ~0ull;
    for (int span = 2; span / 2 < left; span <<= 1) {         // bitonic, over as many lanes as there are entries
      for (int step = span >> 1; step > 0; step >>= 1) {
        const uint64_t other = __shfl_xor((unsigned long long)k, step, kWave);
        k = ((lane & step) == 0) == ((lane & span) == 0) ? min(k, other) : max(k, other);
      }
    }
    const uint64_t sum = wave_scan_u64(lane < left ? whole(entry_mass(key_logit<DT>(k), top, r, series)) : 0);
    const uint64_t over = __ballot(lane < left && (by_count ? (uint64_t)lane : sum) >= t + (by_count ? 0 : 1));
    if (lane == (over ? __ffsll((unsigned long long)over) - 1 : max(left - 1, 0))) {
      s.key = k;
      s.upto = upto + sum;
    }
  }
  __syncthreads();
  return Found{s.key, s.upto};
}

// The row's token from the scanned bins and the candidates (`n` of them, or more than `most`: then from the row itself).  Without DRAW: what the filters
// leave, into the row's RowCut.
template <int DT, int THREADS, bool DRAW>
__device__ void draw_row(Search& s, const Hist& bins, const uint64_t* keys, int n, int most, const SampleArgs& a, RowCut* cuts, int row_index,
                         const void* row, const RowTop& top, const RowRule& r, bool by_k, bool by_p, uint64_t min_p_mass) {
  uint64_t z = bins.mass[kBins - 1];
  Found found{~0ull, 0};
#pragma unroll 1
  for (int which = by_k ? 0 : by_p ? 1 : 2; which < (DRAW ? 3 : 2); which += which == 0 && !by_p ? 2 : 1) {       // (one copy of the search in the code)
    if (which == 2 && r.min_p > 0.0) z = min(z, min_p_mass);
    const uint64_t t = which == 0 ? (uint32_t)r.k - 1 : which == 1 ? top_p_goal(r.p, z) : draw_goal(r.u, z);
    found = find_entry<DT, THREADS>(s, bins, which == 0, t, top, r, n <= most ? n : a.vocab, [&](auto f) {
      if (n <= most) {
        for (int i = threadIdx.x; i < n; i += THREADS) f(keys[i]);
      } else {
        Pieces<DT, THREADS> pieces(row, 0, a.vocab);
        each_entry<DT, THREADS>(pieces, [&](float l, int i) {
          if (entry_distance(l, top, r) < kReach) f(order_key<DT>(l, i));
        });
      }
    });
    if (which < 2) z = found.upto;
  }
  if (threadIdx.x != 0) return;
  if constexpr (DRAW) {
    a.tokens[row_index] = (int64_t)(found.key & 0xfffff);
    a.probs[row_index] = (float)(entry_mass(key_logit<DT>(found.key), top, r, Series()) / (double)z);
  } else {
    cuts[row_index] = RowCut{(double)(r.min_p > 0.0 ? min(z, min_p_mass) : z), found.key, top.value};
  }
}
template <bool DRAW>
__device__ __forceinline__ void nothing_to_draw(const SampleArgs& a, RowCut* cuts, int row_index) {
  if (threadIdx.x != 0) return;
  if constexpr (DRAW) {
    a.tokens[row_index] = -1;
    a.probs[row_index] = 0.f;
  } else {
    cuts[row_index] = RowCut{0.0, 0, -INFINITY};
  }
}

template <int DT>
__device__ __forceinline__ const void* row_of(const SampleArgs& a, int row_index) {
  return (const char*)a.logits + (int64_t)row_index * a.row_stride * Elem<DT>::kBytes;
}

// One workgroup a row, the row read three times: the largest, the bins, the entries of the bins that matter.
template <int DT, bool DRAW>
__global__ __launch_bounds__(kSampleThreads) void sample_row_kernel(SampleArgs a, RowCut* cuts) {
  __shared__ Hist bins;
  __shared__ Search s;
  __shared__ uint64_t keys[kCandidates];
  __shared__ float scratch[kSampleThreads / kWave];
  __shared__ unsigned long long min_p_mass;
  __shared__ int n;
  const int row_index = blockIdx.x;
  const void* row = row_of<DT>(a, row_index);
  const RowRule r = row_rule(a, row_index);
  const RowTop top = row_top_of(block_max<kSampleThreads>(part_top<DT, kSampleThreads>(row, 0, a.vocab), scratch), r);
  if (top.value == -INFINITY) return nothing_to_draw<DRAW>(a, cuts, row_index);              // (uniform)
  clear_hist<kSampleThreads>(bins);
  if (threadIdx.x == 0) {
    min_p_mass = 0;
    n = 0;
  }
  __syncthreads();
  Pieces<DT, kSampleThreads> first(row, 0, a.vocab);
  const uint64_t kept = wave_scan_u64(fill_bins<DT, kSampleThreads>(bins, first, a.vocab, top, r));
  if ((threadIdx.x & (kWave - 1)) == kWave - 1) atomicAdd(&min_p_mass, (unsigned long long)kept);
  __syncthreads();
  scan_bins<kSampleThreads>(bins, s.wave_mass, s.wave_count);
  const BinRanges g = bin_ranges<DRAW>(bins, min_p_mass, r);
  Pieces<DT, kSampleThreads> again(row, 0, a.vocab);
  gather<DT, kSampleThreads, DRAW>(keys, kCandidates, &n, again, top, r, g);
  __syncthreads();
  draw_row<DT, kSampleThreads, DRAW>(s, bins, keys, n, kCandidates, a, cuts, row_index, row, top, r, g.by_k, g.by_p, min_p_mass);
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
  const float top = block_max<kSliceThreads>(
      part_top<DT, kSliceThreads>(row_of<DT>(a, row_index), slice * c.length, min((slice + 1) * c.length, a.vocab)), scratch);
  if (threadIdx.x == 0) c.slices[blockIdx.x].top = top;
}

template <int DT, int THREADS>
__global__ __launch_bounds__(THREADS) void sample_bins_kernel(SampleArgs a, SliceArgs c) {
  __shared__ Hist h;
  __shared__ float scratch[THREADS / kWave];
  __shared__ unsigned long long min_p_mass;
  const int row_index = blockIdx.x / c.count, slice = blockIdx.x % c.count;
  Pieces<DT, THREADS> pieces(row_of<DT>(a, row_index), slice * c.length, min((slice + 1) * c.length, a.vocab));
  clear_hist<THREADS>(h);
  if (threadIdx.x == 0) min_p_mass = 0;
  const RowRule r = row_rule(a, row_index);
  const RowTop top = row_top_of(row_top<THREADS>(c, row_index, scratch), r);          // (its barriers also stand between the clearing and the sums)
  const uint64_t kept = wave_scan_u64(fill_bins<DT, THREADS>(h, pieces, a.vocab, top, r));
  if ((threadIdx.x & (kWave - 1)) == kWave - 1) atomicAdd(&min_p_mass, (unsigned long long)kept);
  __syncthreads();
  SliceRecord& out = c.slices[blockIdx.x];
  for (int i = threadIdx.x; i < kBins; i += THREADS) {
    out.bins.mass[i] = h.mass[i];
    out.bins.count[i] = h.count[i];
  }
  if (threadIdx.x == 0) out.min_p_mass = min_p_mass;
}

template <int DT, bool DRAW, int THREADS>
__global__ __launch_bounds__(THREADS) void sample_gather_kernel(SampleArgs a, SliceArgs c) {
  __shared__ Hist h;
  __shared__ float scratch[THREADS / kWave];
  __shared__ uint64_t wave_mass[THREADS / kWave];
  __shared__ uint32_t wave_count[THREADS / kWave];
  __shared__ int n;
  const int row_index = blockIdx.x / c.count, slice = blockIdx.x % c.count;
  Pieces<DT, THREADS> pieces(row_of<DT>(a, row_index), slice * c.length, min((slice + 1) * c.length, a.vocab));
  if (threadIdx.x == 0) n = 0;
  const RowRule r = row_rule(a, row_index);
  const SliceRecord* of = c.slices + (int64_t)row_index * c.count;
  const int lane = threadIdx.x & (kWave - 1);
  uint64_t kept = lane < c.count ? of[lane].min_p_mass : 0;                                  // (at most 16 slices)
  const RowTop top = row_top_of(row_top<THREADS>(c, row_index, scratch), r);
  if (top.value == -INFINITY) return;                                             // (uniform) the last launch says so
  constexpr int kEach = kBins / THREADS;                  // bins that a thread adds up
  typedef uint64_t Masses __attribute__((ext_vector_type(kEach)));
  typedef uint32_t Counts __attribute__((ext_vector_type(kEach)));
  const int first = threadIdx.x * kEach;
  Masses m = 0;
#pragma unroll 16
  for (int j = 0; j < c.count; ++j) m += *(const Masses*)&of[j].bins.mass[first];
  *(Masses*)&h.mass[first] = m;
  Counts k = 0;
  if (r.k < a.vocab) {
#pragma unroll 16
    for (int j = 0; j < c.count; ++j) k += *(const Counts*)&of[j].bins.count[first];
  }
  *(Counts*)&h.count[first] = k;
  kept = __shfl((unsigned long long)wave_scan_u64(kept), kWave - 1, kWave);
  __syncthreads();
  scan_bins<THREADS>(h, wave_mass, wave_count);
  const BinRanges g = bin_ranges<DRAW>(h, kept, r);
  SliceRecord& out = c.slices[blockIdx.x];
  gather<DT, THREADS, DRAW>(out.key, kSliceCandidates, &n, pieces, top, r, g);
  if (slice == 0) {
    RowRecord& rec = c.rows[row_index];
    for (int i = threadIdx.x; i < kBins; i += THREADS) {
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

template <int DT, bool DRAW>
__global__ __launch_bounds__(kSliceThreads) void sample_draw_kernel(SampleArgs a, SliceArgs c, RowCut* cuts) {
  __shared__ Hist bins;
  __shared__ Search s;
  __shared__ uint64_t keys[kCandidates];
  __shared__ float scratch[kSliceThreads / kWave];
  const int row_index = blockIdx.x;
  const RowRule r = row_rule(a, row_index);
  const SliceRecord* of = c.slices + (int64_t)row_index * c.count;
  const RowRecord& rec = c.rows[row_index];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
  const int some = lane < c.count ? of[lane].n_candidates : 0;                               // (at most 16 slices)
  const RowTop top = row_top_of(row_top<kSliceThreads>(c, row_index, scratch), r);
  if (top.value == -INFINITY) return nothing_to_draw<DRAW>(a, cuts, row_index);               // (uniform)
  for (int i = threadIdx.x; i < kBins; i += kSliceThreads) {
    bins.mass[i] = rec.bins.mass[i];
    bins.count[i] = rec.bins.count[i];
  }
  const int upto = (int)wave_scan_u32((uint32_t)some), n = __shfl(upto, kWave - 1, kWave);
  const bool all = !__any(some > kSliceCandidates) && n <= kCandidates;
  if (all) {
    for (int j = wave; j < c.count; j += kSliceThreads / kWave) {                            // a wavefront a slice
      const int to = __shfl(upto, j, kWave), len = __shfl(some, j, kWave);
      for (int i = lane; i < len; i += kWave) keys[to - len + i] = of[j].key[i];
    }
  }
  __syncthreads();
  draw_row<DT, kSliceThreads, DRAW>(s, bins, keys, all ? n : 1, all ? kCandidates : 0, a, cuts, row_index, row_of<DT>(a, row_index), top, r, rec.by_k,
                                    rec.by_p, rec.min_p_mass);
}

// Slices a row is cut into; 1: the row stays whole, which is one launch in the place of four.  More slices shorten the two passes over the row, but
// each adds up the bins of all for itself.  1 / 4 / 8 / 16 / 32 slices, us (top-p 0.95, min-p 0.02): one row of 152064 fp32 92 53 41 34 32, 16 rows bf16
// 87 53 45 39 45, 64 89 58 57 59 77, 128 93 75 81 88 124, 256 99 110 124 141 215; fp32, one row of 32000 31 28 27 26 27, 64 38 36 42 47 67; one of 16384
// 21 23 24 23 -.
// From 32 rows on slices of twice the threads, half as many, where that leaves as many threads: every workgroup of the second pass reads the bins of all its row's slices (63 rows of
// 152064: 48 MB, now 12; bins 17.4 -> 15.8 us, the second pass 16.5 -> 13.3; 107 of 32000 12.3 -> 9.8 and 11.5 -> 10.8; 16 rows 8.9 -> 8.4 and 10.2 -> 11.1, 100 rows in two
// instead of five 63.6 and 59.9).  From 171 rows on that is the whole row (170 rows in three slices 80, whole 84, 190 in two 100 and 86).
static bool wide_slices(int64_t rows) { return rows >= 32 && 512 / rows == 2 * (256 / rows); }
static int sample_slices(int64_t rows, int64_t vocab) {
  if (vocab < 24576) return 1;
  return (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>((wide_slices(rows) ? 256 : 512) / rows, 16), vocab / (rows <= 8 ? 2048 : 8192)));
}

size_t row_search_workspace(int64_t rows, int64_t vocab) {
  const int count = sample_slices(rows, vocab);
  if (count == 1) return 256;
  return 256 + align_up((size_t)rows * count * sizeof(SliceRecord), 256) + (size_t)rows * sizeof(RowRecord);
}
template <int DT, bool DRAW>
static void launch_row_search_of(const SampleArgs& a, int64_t rows, RowCut* cuts, void* workspace, hipStream_t st) {
  SliceArgs c;
  c.count = sample_slices(rows, a.vocab);
  c.length = (a.vocab + c.count - 1) / c.count;
  c.slices = (SliceRecord*)workspace;
  c.rows = (RowRecord*)((char*)workspace + align_up((size_t)rows * c.count * sizeof(SliceRecord), 256));
  const dim3 grid((unsigned)rows), slices((unsigned)(rows * c.count));
  if (c.count == 1) {
    DominantKernelTimer timer(st);
    hipLaunchKernelGGL((sample_row_kernel<DT, DRAW>), grid, dim3(kSampleThreads), 0, st, a, cuts);
    return;
  }
  hipLaunchKernelGGL(sample_top_kernel<DT>, slices, dim3(kSliceThreads), 0, st, a, c);
  {
    DominantKernelTimer timer(st);
    if (!wide_slices(rows)) hipLaunchKernelGGL((sample_bins_kernel<DT, kSliceThreads>), slices, dim3(kSliceThreads), 0, st, a, c);
    else hipLaunchKernelGGL((sample_bins_kernel<DT, 2 * kSliceThreads>), slices, dim3(2 * kSliceThreads), 0, st, a, c);
  }
  if (!wide_slices(rows)) hipLaunchKernelGGL((sample_gather_kernel<DT, DRAW, kSliceThreads>), slices, dim3(kSliceThreads), 0, st, a, c);
  else hipLaunchKernelGGL((sample_gather_kernel<DT, DRAW, 2 * kSliceThreads>), slices, dim3(2 * kSliceThreads), 0, st, a, c);
  hipLaunchKernelGGL((sample_draw_kernel<DT, DRAW>), grid, dim3(kSliceThreads), 0, st, a, c, cuts);
}
template <bool DRAW>
static void launch_row_search(const SampleArgs& a, int dtype, int64_t rows, RowCut* cuts, void* workspace, hipStream_t st) {
  if (dtype == SUBSPEC_F32) launch_row_search_of<SUBSPEC_F32, DRAW>(a, rows, cuts, workspace, st);
  else if (dtype == SUBSPEC_F16) launch_row_search_of<SUBSPEC_F16, DRAW>(a, rows, cuts, workspace, st);
  else launch_row_search_of<SUBSPEC_BF16, DRAW>(a, rows, cuts, workspace, st);
}
void launch_row_cuts(const SampleArgs& a, int dtype, int64_t rows, RowCut* cuts, void* workspace, hipStream_t st) {
  launch_row_search<false>(a, dtype, rows, cuts, workspace, st);
}

}  // namespace subspec

using namespace subspec;

extern "C" size_t subspec_sample_filtered_workspace(int64_t rows, int64_t vocab) {
  if (rows < 1 || vocab < 1 || vocab > (1 << 20)) return 256;
  return row_search_workspace(rows, vocab);
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
  launch_row_search<true>(a, dtype, rows, nullptr, workspace, (hipStream_t)stream);
  SUBSPEC_CHECK_HIP(hipGetLastError());
  return SUBSPEC_OK;
}
