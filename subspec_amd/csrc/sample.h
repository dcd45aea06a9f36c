// What the kernels that draw from a row of logits share: a row's settings, the masses of its entries and their order (see sample.hip).
#pragma once
#include "common.h"
#include "mass_series.h"

namespace subspec {

constexpr float kReach = 29.9f;           // 43 ln 2 = 29.81: masses beyond round to zero

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
struct RowRule { double inv_t_log2e; float inv_t; bool greedy; int k; double p, min_p, u; };
__device__ __forceinline__ RowRule row_rule(const SampleArgs& a, int row) {
  RowRule r;
  const float t = a.temperatures ? a.temperatures[row] : a.temperature;
  const int k = a.top_ks ? a.top_ks[row] : a.top_k;
  const float p = a.top_ps ? a.top_ps[row] : a.top_p, q = a.min_ps ? a.min_ps[row] : a.min_p, u = a.uniforms[row];
  r.greedy = !(t >= 1.17549435e-38f);                    // (below the smallest normal number 1 / T is infinite)
  const double inv_t = r.greedy ? 1.0 : 1.0 / (double)t;
  r.inv_t_log2e = inv_t * 1.44269504088896340736;
  r.inv_t = (float)inv_t;
  r.k = r.greedy ? 1 : k <= 0 ? INT32_MAX : k;
  r.p = p < 1.f ? (double)p : 1.0;                       // (a NaN filters nothing)
  r.min_p = q > 0.f ? fmin((double)q, 1.0) : 0.0;
  r.u = u > 0.f ? (double)u : 0.0;
  return r;
}
// The largest logit, and whether only entries that equal it have mass (T = 0, or it is infinite).
struct RowTop { float value; double wide; bool only; };
__device__ __forceinline__ RowTop row_top_of(float top, const RowRule& r) { return RowTop{top, (double)top, r.greedy || top == INFINITY}; }

// 2^f * 2^42 for |f| <= 1/2.  (The coefficients are held in registers of the wavefront: left to itself the compiler copies each into the result before
// it adds.)
struct Series {
  double c[kSeriesTerms];
  __device__ __forceinline__ Series() {
    constexpr SeriesTable of = series_table();
#pragma unroll
    for (int i = 0; i < kSeriesTerms; ++i) {
      c[i] = of.c[i];
      asm("" : "+v"(c[i]));
    }
  }
  __device__ __forceinline__ double operator()(double f) const { return series_value(c, f); }
};
// How far entry l is below the largest in units of T, in 32 bits: what the bins go by (falls as l rises, so bins keep the order).  Entries at kReach
// and beyond, and NaN, have no mass and no bin.
__device__ __forceinline__ float entry_distance(float l, const RowTop& top, const RowRule& r) {
  if (top.only) return l == top.value ? 0.f : INFINITY;
  return (top.value - l) * r.inv_t;
}
// The mass of an entry less than kReach below the largest, in units of 2^-42 and before rounding.
__device__ __forceinline__ double entry_mass(float l, const RowTop& top, const RowRule& r, const Series& exp2_part) {
  if (top.only) return (double)(1ull << kMassBits);
  const double x = ((double)l - top.wide) * r.inv_t_log2e, n = rint(x);
  return ldexp(exp2_part(x - n), (int)n);
}
// ... rounded (to even): below 2^52 a sum with 2^52 has no bits behind the point
__device__ __forceinline__ uint64_t whole(double m) { return (uint64_t)__double_as_longlong(m + 4503599627370496.0) & 0xfffffffffffffull; }

// Larger logits first, then lower indexes, as ascending keys: the bits of the value that its type has (a bf16's or fp16's float is zero behind
// them), turned round, and 20 bits of the index.
template <int DT> constexpr int kDropped = DT == SUBSPEC_F32 ? 0 : DT == SUBSPEC_F16 ? 13 : 16;
template <int DT>
__device__ __forceinline__ uint64_t order_key(float l, int i) {
  uint32_t b = __float_as_uint(l == 0.f ? 0.f : l);      // (-0 is 0)
  b = b >> 31 ? b : ~b & 0x7fffffffu;                     // positive values below, negative ones with the sign bit above
  return (uint64_t)(b >> kDropped<DT>) << 20 | (uint32_t)i;
}
template <int DT>
__device__ __forceinline__ float key_logit(uint64_t key) {
  const uint32_t b = (uint32_t)(key >> 20) << kDropped<DT>;
  return __uint_as_float(b >> 31 ? b : ~(b | ((1u << kDropped<DT>) - 1)) & 0x7fffffffu);
}

// Sums up to each lane (all lanes active), by lanes that neighbour in a row of sixteen and the rows' last ones: registers alone, where exchanges through LDS wait
// for one another.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t lanes_shifted_u64(uint64_t v) {
  const int lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xf, false);
  const int hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xf, false);
  return (uint64_t)(uint32_t)hi << 32 | (uint32_t)lo;
}
__device__ __forceinline__ uint64_t wave_scan_u64(uint64_t v) {
  v += lanes_shifted_u64<0x111, 0xf>(v);
  v += lanes_shifted_u64<0x112, 0xf>(v);
  v += lanes_shifted_u64<0x114, 0xf>(v);
  v += lanes_shifted_u64<0x118, 0xf>(v);
  v += lanes_shifted_u64<0x142, 0xa>(v);
  v += lanes_shifted_u64<0x143, 0xc>(v);
  return v;
}
__device__ __forceinline__ uint64_t lane_u64(uint64_t v, int lane) {        // (the lane is the same in all)
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
}
__device__ __forceinline__ uint64_t wave_sum_u64(uint64_t v) { return lane_u64(wave_scan_u64(v), kWave - 1); }
__device__ __forceinline__ double wave_sum_f64(double v) {
  auto add = [&](uint64_t u) { v += __longlong_as_double((long long)u); };
  add(lanes_shifted_u64<0x111, 0xf>((uint64_t)__double_as_longlong(v)));
  add(lanes_shifted_u64<0x112, 0xf>((uint64_t)__double_as_longlong(v)));
  add(lanes_shifted_u64<0x114, 0xf>((uint64_t)__double_as_longlong(v)));
  add(lanes_shifted_u64<0x118, 0xf>((uint64_t)__double_as_longlong(v)));
  add(lanes_shifted_u64<0x142, 0xa>((uint64_t)__double_as_longlong(v)));
  add(lanes_shifted_u64<0x143, 0xc>((uint64_t)__double_as_longlong(v)));
  return __longlong_as_double((long long)lane_u64((uint64_t)__double_as_longlong(v), kWave - 1));
}
__device__ __forceinline__ float larger(float m, float l) { return l > m ? l : m; }      // a NaN never is
__device__ __forceinline__ uint64_t draw_goal(double u, uint64_t z) {
  const uint64_t t = (uint64_t)(u * (double)z);
  return z > 0 ? min(t, z - 1) : 0;
}

// What the filters leave of a row: its mass (in units of 2^-42 of the largest entry's; 0: nothing), the key of the last entry in order that top-k and
// top-p keep, the largest logit.  (Of those entries min-p keeps the ones whose mass reaches it.)
struct RowCut {
  double mass;
  uint64_t last;
  float top;
};
// The cuts of all rows, with the steps of a draw up to its last (sample.hip); the workspace is that of as many draws.
size_t row_search_workspace(int64_t rows, int64_t vocab);
void launch_row_cuts(const SampleArgs& a, int dtype, int64_t rows, RowCut* cuts, void* workspace, hipStream_t st);

}  // namespace subspec
