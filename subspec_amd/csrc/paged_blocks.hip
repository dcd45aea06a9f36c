// Attention of the new tokens of a batch over the blocks of their sequences that matter to them, for gfx950: bounds of every full page's keys, the
// blocks that a token's queries score highest by these, and attention over those blocks.
//
// The pool is that of the paged cache, [max_pages][2 (K, V)][page_len][n_kv_heads][head_dim] a layer.  A block is a sequence's rows j page_len .. of
// one page, block_table[sequence][j].  A token at position pos sees rows 0 .. pos, so blocks 0 .. c = pos / page_len, of which all but c
// are full and hold nothing behind it.
#include "paged.h"
#include "sample.h"
#include <algorithm>
#include <cmath>

namespace subspec {

static int block_shift_of(int64_t page_len) {
  int shift = 0;
  while ((1ll << shift) < page_len) ++shift;
  return shift;
}

// ---------------------------------------------------------------------------------------------------------------- bounds
// low_d = min over the page's rows of K_d, high_d = max, of every page whose last row is among the slots: the rows of a page are
// written in order, so it is full then, and its bounds come from the page alone (nothing is read, changed and written back).
// A wavefront takes a slice of 16 pieces (16 bytes each; 8 where a row has no more) of the pages whose last rows are among up to eight slots (32 of long pages), several rows at a time with up
// to sixteen requests a lane under way.  Its lanes meet through registers, so nobody waits for anybody, and a wavefront without such a page leaves.
// As whole numbers that rise with the value: the bits of a negative value but its sign turned round.  A NaN is then above +infinity or below -infinity, so the
// least and the largest say if there is one, and two values of either type take five instructions where a comparison in 32 bits that keeps a NaN takes sixteen.
// Bound by the trips slots -> rows -> bounds: 61 slots 2.6 to 3 us, of which a launch is 2; 8191 rows of 8 heads of 128 in pages of 16 rows (18.9 MB) 6.1 (3.1 TB/s), of 1 row (50 MB)
// 15.4, of 256 (16.4 MB) 7 to 8.3, 4000 rows in pages of 64 (8.4 MB) 4.1 to 4.6.  With a workgroup a slot, all of a page's pieces in it: 6.0, 7.5, 27, 64 and 33.
constexpr int kBoundsThreads = 256;
typedef short dec_s2 __attribute__((ext_vector_type(2)));
struct BoundsArgs {
  const uint16_t* pool;
  uint16_t* bounds;              // [max_pages][n_kv_heads][2 (low, high)][head_dim]
  const int64_t* slots;
  int64_t n_slots, page_elems;
  int n_tokens, page_shift, pieces, head_pieces, slices, slices_shift, infinity, per;      // slots of a wavefront; 16-byte pieces of a token's K, of a head's; slices of a workgroup, as a power of two
};
__device__ __forceinline__ dec_s2 ordered(dec_s2 v) { return v ^ (v >> 15 & 0x7fff); }          // (and back)

// With SPLIT a workgroup's four wavefronts have the same slice and a quarter of the rows each, and meet through LDS.
template <int LANES, int AT_ONCE, bool SPLIT>
__global__ __launch_bounds__(kBoundsThreads) void page_bounds_kernel(BoundsArgs a) {
  constexpr int kWaves = kBoundsThreads / kWave, kRows = kWave / LANES * (SPLIT ? kWaves : 1);
  __shared__ dec_s2 sides[SPLIT ? kWaves : 1][8][SPLIT ? LANES : 1];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave, page_len = 1 << a.page_shift, half = lane / LANES;
  const int row = half + (SPLIT ? wave * (kWave / LANES) : 0);
  const int slice = SPLIT ? blockIdx.y : (blockIdx.y << a.slices_shift) + (wave & ((1 << a.slices_shift) - 1)), piece = slice * LANES + lane % LANES, from = min(piece, a.pieces - 1);
  if (slice >= a.slices) return;
  // a prompt's last rows come at equal distances: every XCD (each eighth workgroup) has neighbouring groups, or one of them would have all the work
  const int64_t of_block = SPLIT ? 1 : kWaves >> a.slices_shift;
  const int64_t apart = (int64_t)gridDim.x * of_block, block = (int64_t)(blockIdx.x % 8) * (gridDim.x / 8) + blockIdx.x / 8;
  for (int64_t group = block * of_block + (SPLIT ? 0 : wave >> a.slices_shift); group * a.per < a.n_tokens; group += apart) {
    const int64_t t = group * a.per + lane;
    const int64_t slot = lane < a.per && t < a.n_tokens ? a.slots[t] : -1;
    uint64_t last_rows = __ballot(slot >= 0 && slot < a.n_slots && (slot & (page_len - 1)) == page_len - 1);
    for (; last_rows; last_rows &= last_rows - 1) {
      const int64_t page = (int64_t)lane_u64((uint64_t)slot, __ffsll((unsigned long long)last_rows) - 1) >> a.page_shift;
      const dec_u4* rows = (const dec_u4*)(a.pool + page * 2 * a.page_elems) + from;
      dec_s2 low[4], high[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        low[e] = dec_s2{32767, 32767};
        high[e] = dec_s2{-32768, -32768};
      }
      for (int r0 = 0; r0 < page_len; r0 += kRows * AT_ONCE) {
        dec_u4 raw[AT_ONCE];
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) raw[k] = rows[(int64_t)min(r0 + k * kRows + row, page_len - 1) * a.pieces];       // (past the end: the last row again)
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const dec_s2 x = ordered(__builtin_bit_cast(dec_s2, (uint32_t)raw[k][e]));
            low[e] = __builtin_elementwise_min(low[e], x);
            high[e] = __builtin_elementwise_max(high[e], x);
          }
      }
      if (page_len > 1) {
#pragma unroll
        for (int o = LANES; o < kWave; o <<= 1)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            low[e] = __builtin_elementwise_min(low[e], __builtin_bit_cast(dec_s2, __shfl_xor(__builtin_bit_cast(int, low[e]), o, kWave)));
            high[e] = __builtin_elementwise_max(high[e], __builtin_bit_cast(dec_s2, __shfl_xor(__builtin_bit_cast(int, high[e]), o, kWave)));
          }
      }
      if constexpr (SPLIT) {                                 // (all four have the same slots)
        if (half == 0)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            sides[wave][e][lane] = low[e];
            sides[wave][4 + e][lane] = high[e];
          }
        __syncthreads();
        if (wave == 0)
#pragma unroll
          for (int w = 1; w < kWaves; ++w)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              low[e] = __builtin_elementwise_min(low[e], sides[w][e][lane % LANES]);
              high[e] = __builtin_elementwise_max(high[e], sides[w][4 + e][lane % LANES]);
            }
        __syncthreads();
      }
      if (piece < a.pieces && half < 2 && (!SPLIT || wave == 0)) {
        dec_u4 out;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          dec_s2 v = ordered(half ? high[e] : low[e]);
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (high[e][i] > a.infinity || low[e][i] < ~a.infinity) v[i] = 0x7fff;                // (the order has -infinity at ~infinity)
          out[e] = __builtin_bit_cast(uint32_t, v);
        }
        dec_u4* to = (dec_u4*)(a.bounds + page * 2 * (a.page_elems >> a.page_shift)) + (piece / a.head_pieces) * 2 * a.head_pieces + piece % a.head_pieces;
        to[half * a.head_pieces] = out;
      }
    }
  }
}
template <int LANES>
static void launch_bounds(BoundsArgs a, hipStream_t st) {
  a.slices = (a.pieces + LANES - 1) / LANES;
  const int rows = (1 << a.page_shift) * LANES / kWave;      // of a lane, where a wavefront has them all
  const bool split = rows >= 16;
  a.slices_shift = split ? 0 : a.slices >= 4 ? 2 : a.slices >= 2 ? 1 : 0;
  // few slots a wavefront while there are few, whose pages may all fill up at once; of a prompt's many one in page_len is a last row
  a.per = std::min(std::max(a.n_tokens / 64, 1), split ? 32 : 8);
  const int64_t groups = ((int64_t)a.n_tokens + a.per - 1) / a.per, of_block = split ? 1 : kBoundsThreads / kWave >> a.slices_shift;
  const dim3 grid((unsigned)std::min<int64_t>(((groups + of_block - 1) / of_block + 7) / 8 * 8, 1 << 16), (unsigned)((a.slices + (1 << a.slices_shift) - 1) >> a.slices_shift)), block(kBoundsThreads);
  if (rows <= 1) hipLaunchKernelGGL((page_bounds_kernel<LANES, 1, false>), grid, block, 0, st, a);
  else if (!split) hipLaunchKernelGGL((page_bounds_kernel<LANES, 4, false>), grid, block, 0, st, a);
  else if (rows < 64) hipLaunchKernelGGL((page_bounds_kernel<LANES, 4, true>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((page_bounds_kernel<LANES, 16, true>), grid, block, 0, st, a);
}

// Sums up to each lane, and a wavefront's largest, by lanes that neighbour in a row of sixteen and the rows' last ones: a dozen instructions, where six exchanges
// through LDS one after the other take 0.3 us.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t shifted_in(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false); }
__device__ __forceinline__ uint32_t lanes_upto(uint32_t v) {
  v += shifted_in<0x111, 0xf>(v);
  v += shifted_in<0x112, 0xf>(v);
  v += shifted_in<0x114, 0xf>(v);
  v += shifted_in<0x118, 0xf>(v);
  v += shifted_in<0x142, 0xa>(v);
  v += shifted_in<0x143, 0xc>(v);
  return v;
}
__device__ __forceinline__ uint32_t lanes_largest(uint32_t v) {
  v = max(v, shifted_in<0x111, 0xf>(v));
  v = max(v, shifted_in<0x112, 0xf>(v));
  v = max(v, shifted_in<0x114, 0xf>(v));
  v = max(v, shifted_in<0x118, 0xf>(v));
  v = max(v, shifted_in<0x142, 0xa>(v));
  v = max(v, shifted_in<0x143, 0xc>(v));
  return (uint32_t)__builtin_amdgcn_readlane((int)v, kWave - 1);
}

// Tiles of up to `share` (a power of two) neighbouring tokens of one sequence, from the first of a run of them on: the m-th of those of tokens [first, end), and how
// many there are.  Tokens outside are nobody's neighbours, those of no sequence are in no tile.  Every wavefront looks for itself, 64 tokens at a time: for the few
// hundred tokens of a step less than a launch for it, or a workgroup for every token that is not the first of a tile, to leave at once.
struct TokenTile { int first, tokens, sequence, all; };
__device__ __forceinline__ TokenTile token_tile(const int32_t* sequences, int first, int end, int batch, int share, int m) {
  const int lane = threadIdx.x & (kWave - 1);
  const uint64_t upto = ~0ull >> (kWave - 1 - lane);
  TokenTile tile{0, 0, -1, 0};
  int run = first, before = -1;                              // where the last run began, the sequence of the token before
  int ahead = sequences[min(first + lane, end - 1)];
  for (int x0 = first; x0 < end; x0 += kWave) {
    const int x = x0 + lane, b = ahead;
    ahead = sequences[min(x + kWave, end - 1)];
    const int left = __shfl_up(b, 1, kWave);
    const uint64_t begins = __ballot(x == first || b != (lane ? left : before)) & upto;
    const int pos = begins ? lane - (kWave - 1 - __clzll((long long)begins)) : x - run;
    const bool counts = x < end && b >= 0 && b < batch;
    const uint64_t leads = __ballot(counts && (pos & (share - 1)) == 0);
    const uint64_t here = __ballot(counts && tile.all + __popcll(leads & upto) - 1 == m);
    if (here && tile.tokens == 0) {
      const int at = __ffsll((unsigned long long)here) - 1;
      tile.first = x0 + at;
      tile.sequence = __builtin_amdgcn_readlane(b, at);
    }
    tile.tokens += __popcll(here);
    tile.all += __popcll(leads);
    run = __builtin_amdgcn_readlane(x - pos, kWave - 1);
    before = __builtin_amdgcn_readlane(b, kWave - 1);
  }
  return tile;
}
constexpr int kTileTokens = 1024;          // tokens of a launch whose tiles are looked for
// Tiles of so many tokens where every sequence's are neighbours: as many are looked for at once, and then the next.
static int tiles_at_once(int64_t tokens, int64_t batch, int64_t share) { return (int)std::min(tokens, std::min(tokens, batch) + tokens / share); }

// ---------------------------------------------------------------------------------------------------------------- scores
// s_j = sum over the KV head's query heads g and dimensions d of max(q_gd low_jd, q_gd high_jd), which no sum of the heads' scores of a key of block j
// exceeds; with A_d = sum_g max(q_gd, 0) and B_d = sum_g min(q_gd, 0) it is sum_d A_d high_jd + B_d low_jd.  In 64 bits: which block comes out ahead must not
// hang on an order of addition, and the rows come out of memory no faster than that (4 D operations for 4 D bytes).
struct SelectArgs {
  const uint16_t* q;
  const uint16_t* bounds;
  const int32_t* table;
  const int32_t* sequences;
  const int32_t* positions;
  int32_t* blocks;               // [tokens][n_kv_heads][keep]
  double* scores;                // [token - first][n_kv_heads][most]
  int64_t q_token, q_head, table_stride, most;
  int batch, first, tokens, hkv, group, page_shift, max_pages, keep, recent, last_row, span, spans, spans_at_once, tiles_at_once;
};
// Blocks that a token sees (0: none), and of these the first so many that compete.
struct TokenBlocks { int seen, scored; };
__device__ __forceinline__ TokenBlocks token_blocks(const SelectArgs& a, int b, int position) {
  const int last = min(position, a.last_row);
  if (b < 0 || b >= a.batch || last < 0) return TokenBlocks{0, 0};
  const int seen = (last >> a.page_shift) + 1;
  return TokenBlocks{seen, seen > a.keep ? seen - a.recent : 0};
}
constexpr int kScoreTokens = 8;           // tokens of a sequence that share a reading of the bounds
constexpr int kScoreThreads = 256;
constexpr int kScoreBlocks = 1536;        // workgroups from which on they take several spans each, a third of these
constexpr int kSharedDepth = 4;           // readings of a wavefront then (1 / 2 / 4: 20.4 / 15.2 / 10.5 us for 72 drafts)

// a double from another lane of sixteen (a DPP control)
template <int CTRL>
__device__ __forceinline__ double from_lane(double v) {
  const uint64_t u = (uint64_t)__double_as_longlong(v);
  const int lo = __builtin_amdgcn_mov_dpp((int)(uint32_t)u, CTRL, 0xf, 0xf, true), hi = __builtin_amdgcn_mov_dpp((int)(uint32_t)(u >> 32), CTRL, 0xf, 0xf, true);
  return __longlong_as_double((long long)((uint64_t)(uint32_t)hi << 32 | (uint32_t)lo));
}
constexpr int kPair = 0xB1, kTwoPairs = 0x4E, kTurnFour = 0x124, kTurnEight = 0x128, kMirrorEight = 0x141;
// Sums of eight values over LANES neighbouring lanes: lane p, p % 4 = r, ends up with those of values r and 4 + r.  Where lanes swap values, each keeps half
// of them, so the later steps have fewer to add: 54 instructions in the place of 96.
template <int LANES>
__device__ __forceinline__ void sum_eight(double (&v)[8], int lane, double* out) {
  if constexpr (LANES == 8) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += from_lane<kMirrorEight>(v[i]);
  }
  double w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const double keep = lane & 1 ? v[2 * i + 1] : v[2 * i], give = lane & 1 ? v[2 * i] : v[2 * i + 1];
    w[i] = keep + from_lane<kPair>(give);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const double keep = lane & 2 ? w[2 * i + 1] : w[2 * i], give = lane & 2 ? w[2 * i] : w[2 * i + 1];
    out[i] = keep + from_lane<kTwoPairs>(give);
    if constexpr (LANES == 16) {
      out[i] += from_lane<kTurnFour>(out[i]);
      out[i] += from_lane<kTurnEight>(out[i]);
    }
  }
}

// The query heads of `tokens` tokens added up by a workgroup, into LDS: (of high, of low) of each.  A thread has DIMS neighbouring dimensions; where there are more
// threads than these, every team of them has a part of the heads, and the teams' sums are added in their order.  Ends with a barrier.
// (`meanwhile` runs before the first barrier)
template <int DT, int D, int TOKENS, int THREADS, int DIMS, typename F>
__device__ __forceinline__ void score_weights(const SelectArgs& a, int t, int tokens, int kvh, double* weight, F meanwhile) {
  constexpr int kTeam = TOKENS * D / DIMS, kTeams = THREADS / kTeam;
  const int team = threadIdx.x / kTeam, k = threadIdx.x / (D / DIMS) % TOKENS, d = threadIdx.x % (D / DIMS) * DIMS;
  const int heads = k < tokens ? a.group : 0;                 // (a token that is not there has the weights 0)
  double up[DIMS], down[DIMS];
#pragma unroll
  for (int e = 0; e < DIMS; ++e) up[e] = down[e] = 0.0;
  const uint16_t* q = a.q + (t + min(k, tokens - 1)) * a.q_token + (int64_t)kvh * a.group * a.q_head + d;
#pragma unroll 4
  for (int g = team; g < heads; g += kTeams) {
    const uint32_t* src = (const uint32_t*)(q + g * a.q_head);
#pragma unroll
    for (int p = 0; p < DIMS / 2; ++p) {
      float x[2];
      unpack2<DT>(src[p], x);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        // (a NaN goes into both: its blocks all score NaN)
        up[2 * p + e] += x[e] < 0.f ? 0.0 : (double)x[e];
        down[2 * p + e] += x[e] > 0.f ? 0.0 : (double)x[e];
      }
    }
  }
  double* mine = weight + ((team * TOKENS + k) * 2) * D + d;
#pragma unroll
  for (int e = 0; e < DIMS; ++e) {
    mine[e] = up[e];
    mine[D + e] = down[e];
  }
  meanwhile();
  __syncthreads();
  if constexpr (kTeams > 1) {
    const int teams = min(kTeams, a.group);
    for (int i = threadIdx.x; i < TOKENS * 2 * D; i += THREADS) {
      double sum = weight[i];
      for (int m = 1; m < teams; ++m) sum += weight[m * TOKENS * 2 * D + i];
      weight[i] = sum;
    }
    __syncthreads();
  }
}
// Bounds of DEPTH * kAtOnce blocks from j0 on (below j1; past it the last one again), all asked for at once: 16-byte pieces of `low` and `high` a lane.  A step reads
// them once, as streaming data: 64 tokens of up to 32768 rows, 193 MB, 43.6 -> 38.9 us (5.0 TB/s; a large copy reaches 5.1).
template <int D, int DEPTH>
__device__ __forceinline__ void load_bounds(const SelectArgs& a, int page, int kvh, dec_u4* low, dec_u4* high) {
  constexpr int kLanes = D / 8, kAtOnce = kWave / kLanes;
  static_assert(DEPTH * kAtOnce <= kWave, "a lane holds a page number");
  const int lane = threadIdx.x & (kWave - 1), page_of = min(max(page, 0), a.max_pages - 1);
  const dec_u4* bounds = (const dec_u4*)(a.bounds + (int64_t)kvh * 2 * D) + lane % kLanes;
#pragma unroll
  for (int i = 0; i < DEPTH; ++i) {
    const dec_u4* src = bounds + (int64_t)__shfl(page_of, i * kAtOnce + lane / kLanes, kWave) * a.hkv * 2 * kLanes;
    low[i] = __builtin_nontemporal_load(src);
    high[i] = __builtin_nontemporal_load(src + kLanes);
  }
}
__device__ __forceinline__ double score_of(double s) { return s != s ? INFINITY : s; }

// A workgroup takes `span` blocks of (token, KV head), a wavefront a quarter of them: D / 8 lanes a block, all requests of a wavefront under way before
// the first score; meanwhile the four of them add the query heads up.  One token of 2048 blocks 5.7 us (5.3 at best); 64 tokens, 193 MB, 39 (4.9 TB/s).
template <int DT, int D>
__global__ __launch_bounds__(kScoreThreads) void block_score_kernel(SelectArgs a) {
  constexpr int kLanes = D / 8, kAtOnce = kWave / kLanes, kDepth = 8;
  __shared__ __attribute__((aligned(16))) double weight[kScoreThreads / (D / 2) * 2 * D];
  const uint32_t unit = blockIdx.x;
  const int kvh = (int)(unit % (uint32_t)a.hkv), span = (int)(unit / (uint32_t)a.hkv % (uint32_t)a.spans);
  const int local = (int)(unit / (uint32_t)a.hkv / (uint32_t)a.spans), t = a.first + local, b = a.sequences[t];
  const int most = token_blocks(a, b, a.positions[t]).scored;
  if (span * a.span >= most) return;                         // (the whole workgroup)
  const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1), part = lane % kLanes, which = lane / kLanes;
  const int j0 = span * a.span + wave * kAtOnce * kDepth, j1 = min(j0 + kAtOnce * kDepth, most);
  dec_u4 low[kDepth], high[kDepth];
  const int page = a.table[b * a.table_stride + max(min(j0 + lane, j1 - 1), 0)];
  if (j0 < j1) load_bounds<D, kDepth>(a, page, kvh, low, high);
  score_weights<DT, D, 1, kScoreThreads, 2>(a, t, 1, kvh, weight, [] {});
  if (j0 >= j1) return;
  double up[8], down[8], s[kDepth], out[2];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    up[e] = weight[part * 8 + e];
    down[e] = weight[D + part * 8 + e];
  }
#pragma unroll
  for (int i = 0; i < kDepth; ++i) {
    float l[8], h[8];
    unpack8<DT>(low[i], l);
    unpack8<DT>(high[i], h);
    s[i] = 0.0;
#pragma unroll
    for (int e = 0; e < 8; ++e) s[i] = fma(up[e], (double)h[e], fma(down[e], (double)l[e], s[i]));
  }
  sum_eight<kLanes>(s, lane, out);
  if (part >= 4) return;
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    const int j = j0 + (4 * m + part) * kAtOnce + which;
    if (j < j1) a.scores[((int64_t)local * a.hkv + kvh) * a.most + j] = score_of(out[m]);
  }
}

// The same for up to kScoreTokens neighbouring tokens of one sequence: the bounds are read and converted once for all, the weights come out of LDS again
// for every block.  (72 drafts of 16 sequences, 32 : 8 heads, up to 255 blocks: a conversion a token 17.4 us, this 9.2 to 10.2.)
// With MORE a workgroup goes on to the next spans, so that the weights are added up for several of them, and asks for their bounds while it looks at these.  Both fit
// two wavefronts a SIMD; the loop costs registers, though, and where the spans fit at once nothing is gained: 128 tiles' 512 spans 9.0 us and 12.4, 504 tiles' 2016 of
// two tokens each 26 and 17, 512 tiles' 16384 216 and 131.
template <int DT, int D, bool MORE>
__global__ __launch_bounds__(kScoreThreads, 2) void block_score_shared_kernel(SelectArgs a) {
  constexpr int kLanes = D / 8, kAtOnce = kWave / kLanes, kAtOnceTokens = 8 / kSharedDepth;            // (tokens that make eight sums)
  __shared__ __attribute__((aligned(16))) double weight[kScoreThreads / (D / 4) * 2 * D];
  const uint32_t unit = blockIdx.x;
  const int kvh = (int)(unit % (uint32_t)a.hkv), span = (int)(unit / (uint32_t)a.hkv % (uint32_t)a.spans_at_once);
  const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1), part = lane % kLanes, which = lane / kLanes;
  for (int m = (int)(unit / (uint32_t)a.hkv / (uint32_t)a.spans_at_once);; m += a.tiles_at_once) {
    const TokenTile tile = token_tile(a.sequences, a.first, a.first + a.tokens, a.batch, kScoreTokens, m);
    if (!tile.tokens) return;
    const int t = tile.first, local = t - a.first;
    // a lane has a token's number of blocks
    const int mine = lane < tile.tokens ? token_blocks(a, tile.sequence, a.positions[t + lane]).scored : 0;
    const int most = (int)lanes_largest((uint32_t)mine);
    const int first = span * a.span, step = a.spans_at_once * a.span;
    if (first < most) {                                       // (the whole workgroup)
      auto page_of = [&](int from) { return a.table[tile.sequence * a.table_stride + min(from + wave * kAtOnce * kSharedDepth + lane, most - 1)]; };
      dec_u4 low[kSharedDepth], high[kSharedDepth];
      int page = page_of(first);
      score_weights<DT, D, kScoreTokens, kScoreThreads, 4>(a, t, tile.tokens, kvh, weight, [&]() {
        load_bounds<D, kSharedDepth>(a, page, kvh, low, high);
        if (MORE) page = page_of(first + step);
      });
      for (int from = first; from < most; from += step) {
        const int j0 = from + wave * kAtOnce * kSharedDepth;
        double low_of[kSharedDepth][8], high_of[kSharedDepth][8];
#pragma unroll
        for (int i = 0; i < kSharedDepth; ++i) {
          float l[8], h[8];
          unpack8<DT>(low[i], l);
          unpack8<DT>(high[i], h);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            low_of[i][e] = (double)l[e];
            high_of[i][e] = (double)h[e];
          }
        }
        if (MORE && from + step < most) {
          load_bounds<D, kSharedDepth>(a, page, kvh, low, high);
          page = page_of(from + 2 * step);
        }
#pragma unroll
        for (int k0 = 0; k0 < kScoreTokens; k0 += kAtOnceTokens) {
          if (k0 >= tile.tokens || j0 >= most) break;
          double s[8], out[2];
#pragma unroll
          for (int k = 0; k < kAtOnceTokens; ++k) {
            // (a token that is not there has the weights 0, and nobody takes what comes of it)
            const double* of = weight + (k0 + k) * 2 * D + part * 8;
#pragma unroll
            for (int i = 0; i < kSharedDepth; ++i) {
              double above = 0.0, below = 0.0;                // (two chains of sums: a wavefront has few others to wait beside)
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                above = fma(of[e], high_of[i][e], above);
                below = fma(of[D + e], low_of[i][e], below);
              }
              s[k * kSharedDepth + i] = above + below;
            }
          }
          sum_eight<kLanes>(s, lane, out);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int v = 4 * i + part, k = k0 + v / kSharedDepth, j = j0 + v % kSharedDepth * kAtOnce + which;
            const int n = __shfl(mine, k & 7, kWave);
            if (part < 4 && j < n) a.scores[((int64_t)(local + k) * a.hkv + kvh) * a.most + j] = score_of(out[i]);
          }
        }
        if (!MORE) break;
      }
    }
    if (m + a.tiles_at_once >= tile.all) return;
    __syncthreads();                                          // (the weights have been read)
  }
}

// ---------------------------------------------------------------------------------------------------------------- the best of them
// The keep - recent blocks of largest score, equal ones from the lowest on, without sorting: the scores as ordered whole numbers, and the digits (eleven bits at
// a time, from the first that differs) of the smallest that stays; the few entries that share them are ranked one by one.  What stays is a bit each, and the
// bits in order are the list.  2048 blocks: 6.2 us (its launch and loads alone 2.8).
constexpr int kMostBlocks = 1 << 17;
constexpr int kDigits = 2048;
constexpr int kHeld = 8;                 // scores of a thread that stay in registers
constexpr int kRanked = 256;
__device__ __forceinline__ uint64_t score_key(double s) {             // ascending
  const uint64_t u = (uint64_t)__double_as_longlong(s + 0.0);          // (-0 is 0)
  return u >> 63 ? ~u : u | 1ull << 63;
}

template <int THREADS>
__global__ __launch_bounds__(THREADS) void block_select_kernel(SelectArgs a) {
  constexpr int kWaves = THREADS / kWave;
  __shared__ uint64_t stays[kMostBlocks / 64];
  __shared__ uint64_t even[kMostBlocks / 64];          // equal to the smallest that stays, where too many are
  __shared__ uint32_t digits[kDigits];
  __shared__ uint64_t list[kRanked];
  __shared__ int list_at[kRanked];
  __shared__ uint32_t lows[kWaves], highs[kWaves];
  __shared__ uint32_t counts[kWaves];
  __shared__ int n_list, digit_at;
  __shared__ uint32_t above_at;
  const int tid = threadIdx.x, wave = tid / kWave, lane = tid & (kWave - 1);
  const int local = blockIdx.x / a.hkv, kvh = blockIdx.x % a.hkv, t = a.first + local;
  int32_t* out = a.blocks + ((int64_t)t * a.hkv + kvh) * a.keep;
  const double* scores = a.scores + ((int64_t)local * a.hkv + kvh) * a.most;
  double early[kHeld];                                  // asked for before it is known how many there are
#pragma unroll
  for (int i = 0; i < kHeld; ++i) early[i] = i * THREADS < a.most ? scores[min((int64_t)tid + i * THREADS, a.most - 1)] : 0.0;
  const TokenBlocks tb = token_blocks(a, a.sequences[t], a.positions[t]);
  if (tb.seen <= a.keep) {
    for (int i = tid; i < a.keep; i += THREADS) out[i] = i < tb.seen ? i : -1;
    return;
  }
  const int n = tb.scored;
  int need = a.keep - a.recent;
  for (int i = tid; i < a.recent; i += THREADS) out[need + i] = n + i;
  if (need == 0) return;
  uint64_t held[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) held[i] = score_key(early[i]);
  // f(key, j, whether there is one) for all entries, every wavefront's lanes together
  auto each = [&](auto f) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (i * THREADS < n) f(held[i], tid + i * THREADS, tid + i * THREADS < n);
    for (int j0 = kHeld * THREADS; j0 < n; j0 += THREADS) {
      const int j = j0 + tid;
      f(j < n ? score_key(scores[j]) : 0, j, j < n);
    }
  };
  // (the keys' upper halves say well enough from which bit on they agree)
  uint32_t low = 0, high = 0;                            // (of the complements, so that both are largest ones)
  each([&](uint64_t key, int, bool there) {
    if (!there) return;
    low = max(low, ~(uint32_t)(key >> 32));
    high = max(high, (uint32_t)(key >> 32));
  });
  low = lanes_largest(low);
  high = lanes_largest(high);
  if (lane == 0) {
    lows[wave] = low;
    highs[wave] = high;
  }
  for (int i = tid; i < kDigits; i += THREADS) digits[i] = 0;
  if (tid == 0) n_list = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    low = max(low, lows[w]);
    high = max(high, highs[w]);
  }
  low = ~low;
  int top = 32 + (low == high ? 0 : 32 - __clz((int)(low ^ high)));      // bits from here on agree in all entries
  int shift = max(0, top - 11);
  uint64_t prefix = top >= 64 ? 0 : (uint64_t)low << 32 >> top << top;
  // each turn: of the entries that agree with `prefix` from `top` on, the digit that the last one to stay has
  int in_digit = 0;
  for (;;) {
    auto mine = [&](uint64_t key) { return top >= 64 || (key ^ prefix) >> top == 0; };
    each([&](uint64_t key, int, bool there) {
      if (there && mine(key)) atomicAdd(&digits[(int)(key >> shift) & (kDigits - 1)], 1u);
    });
    __syncthreads();
    constexpr int kEach = kDigits / THREADS;             // digits from the largest down: thread 0 has the largest ones
    uint32_t mine_n = 0, of[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) mine_n += of[i] = digits[kDigits - 1 - (tid * kEach + i)];
    const uint32_t upto = lanes_upto(mine_n);
    if (lane == kWave - 1) counts[wave] = upto;
    __syncthreads();
    uint32_t before = upto - mine_n;
    for (int w = 0; w < wave; ++w) before += counts[w];
    if (before < (uint32_t)need && (uint32_t)need <= before + mine_n) {
      uint32_t at = before;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        if (at < (uint32_t)need && (uint32_t)need <= at + of[i]) {
          digit_at = kDigits - 1 - (tid * kEach + i);
          above_at = at;
        }
        at += of[i];
      }
    }
    __syncthreads();
    const int digit = digit_at;
    need -= (int)above_at;
    in_digit = (int)digits[digit];
    prefix |= (uint64_t)digit << shift;
    top = shift;
    __syncthreads();
    if (in_digit == need || in_digit <= kRanked || top == 0) break;
    shift = max(0, top - 11);
    for (int i = tid; i < kDigits; i += THREADS) digits[i] = 0;
    __syncthreads();
  }
  // larger ones stay; of those that agree with the prefix all, or the `need` first in order
  const bool all = in_digit == need, ranked = !all && in_digit <= kRanked;
  each([&](uint64_t key, int j, bool there) {
    const uint64_t over = key >> top, border = prefix >> top;
    const bool same = there && over == border;
    const uint64_t in = __ballot((there && over > border) || (same && all)), equal = __ballot(same && !all && !ranked);
    if (same && ranked) {
      const int at = atomicAdd(&n_list, 1);
      list[at] = key;
      list_at[at] = j;
    }
    if (lane == 0) {
      stays[j >> 6] = in;
      even[j >> 6] = equal;
    }
  });
  __syncthreads();
  if (ranked) {
    if (tid < in_digit) {
      int rank = 0;
      for (int i = 0; i < in_digit; ++i) rank += list[i] > list[tid] || (list[i] == list[tid] && list_at[i] < list_at[tid]);
      if (rank < need) atomicOr((unsigned long long*)&stays[list_at[tid] >> 6], 1ull << (list_at[tid] & 63));
    }
    __syncthreads();
  }
  // a thread takes consecutive words
  const int words = (n + 63) / 64, per = (words + THREADS - 1) / THREADS, w0 = tid * per, w1 = min(w0 + per, words);
  auto before_of = [&](uint32_t v) {
    const uint32_t upto = lanes_upto(v);
    if (lane == kWave - 1) counts[wave] = upto;
    __syncthreads();
    uint32_t before = upto - v;
    for (int w = 0; w < wave; ++w) before += counts[w];
    __syncthreads();
    return before;
  };
  if (!all && !ranked) {
    uint32_t v = 0;
    for (int w = w0; w < w1; ++w) v += __popcll(even[w]);
    int left = need - (int)before_of(v);
    for (int w = w0; w < w1; ++w)
      for (uint64_t m = even[w]; m && left > 0; m &= m - 1, --left) stays[w] |= m & (~m + 1);
  }
  uint32_t v = 0;
  for (int w = w0; w < w1; ++w) v += __popcll(stays[w]);
  int at = (int)before_of(v);
  for (int w = w0; w < w1; ++w)
    for (uint64_t m = stays[w]; m; m &= m - 1) out[at++] = w * 64 + __ffsll((unsigned long long)m) - 1;
}

// ---------------------------------------------------------------------------------------------------------------- attention
// As the attention of few rows over a whole cache (paged_attention.hip): a unit is (token, KV head, chunk of the listed rows) and one wavefront, whose
// rows travel straight into its own ring of LDS stages, 32 keys each; S^T = K Q^T and O^T = V^T P^T by 16x16x32 products; a row's
// probabilities are relative to a reference that follows its largest score by at most 2^8.  A probability goes into its product as two numbers
// of the type, what it rounds to and what that leaves (2^-17 of it in bf16): a few rows carry most of a selected context, so that roundings do not cancel, and the
// second product costs nothing beside the rows' way out of memory (2-norm against 64 bits with one number 0.0026, with two 0.0016, which is
// the output's own rounding).  A listed row that the token does not see (behind it, of no block) is a row of zeros and has no probability: what the
// cache holds there never comes near a product.
// Tokens of one sequence list much the same blocks, so where a call has more tokens than sequences up to eight of them share a unit (32 rows of a KV head): its
// blocks are those that any of them lists, ascending, each with a bit a token (block_union_kernel), and a row sees a key by its token's bit and position.
// 72 drafts of 16 sequences, 32 blocks of 64 rows each, 32 : 8 heads: a unit a token reads 600 MB, out of the caches, in 92 us; their union, 192 MB, takes 42 (4.6 TB/s).  64 tokens
// by themselves, 134 MB: 26.8 (5.0 TB/s); one of 1024 rows: 5.5, five trips to memory and the launch.  A stage of 32 keys and 32 rows is 1.3 us of a wavefront's work.
constexpr int kAttendKeys = 32;
constexpr int kAttendStages = 2;
constexpr int kAttendSegment = 512;        // keys whose row offsets are in LDS at a time
constexpr int kShareRows = 32;             // rows of a unit that several tokens share
typedef int dec_i4 __attribute__((ext_vector_type(4)));
__device__ __attribute__((aligned(16))) uint32_t zero_piece[4];

struct AttendArgs {
  const uint16_t* q;
  const uint16_t* pool;
  const int32_t* table;
  const int32_t* blocks;
  const int32_t* sequences;
  const int32_t* positions;
  uint16_t* out;
  float* part_o;                 // [token][n_kv_heads][chunks][group][D], fp32
  float* part_ml;                // (reference, sum)
  int2* merged;                  // [n_kv_heads][token][keep], from a tile's first token on: the blocks of the tile, a bit for each token that lists them
  int32_t* parts;                // [n_kv_heads][token]: chunks of the token's tile
  int4* tiles;                   // [tile][n_kv_heads]: first token, tokens (0: there is no such tile), blocks, how many tiles there are
  int64_t q_token, q_head, table_stride, page_elems;
  int batch, first, tokens, hq, hkv, group, page_shift, max_pages, keep, last_row, keys, chunk_keys, chunks, share, tiles_at_once;
  float scale_log2;
};
// Chunks of a tile of `keys` keys where there are so many tiles: as many units as the GPU holds at once (four of 39 KB a CU) end together, and some more wait for a round of
// their own (128 tiles of 2933 keys, 8 heads' tiles of 16 sequences: 5 / 6 / 7 / 8 chunks 47.0 / 45.4 / 45.0 / 42.6 us, 9 / 10 54.5 / 52.2), so units are as many as that or a
// multiple of it.  Short ones are a few trips to memory for little: a chunk has 64 keys at least, and 0.5 sqrt of all the tiles' keys.
constexpr int kSharedKeys = 1024;
constexpr int kUnitsAtOnce = 4 * 256;
__host__ __device__ __forceinline__ int tile_chunks(int keys, int tiles) {
  const int64_t rounds = ((int64_t)tiles * ((keys + kSharedKeys - 1) / kSharedKeys) + kUnitsAtOnce - 1) / kUnitsAtOnce;
  const float least = fmaxf(64.f, 0.5f * sqrtf((float)tiles * (float)keys));
  const int64_t chunks = rounds * kUnitsAtOnce / (tiles > 0 ? tiles : 1), most = (int64_t)((float)keys / least);
  return (int)(chunks < most ? chunks > 0 ? chunks : 1 : most > 0 ? most : 1);
}
__device__ __forceinline__ int attend_last(const AttendArgs& a, int t) { return min(a.positions[t], a.last_row); }

// ---- tiles of up to `share` neighbouring tokens of a sequence, and their blocks: a byte a block in LDS, a bit of it a token, then the bytes in order
constexpr int kUnionThreads = 256;
constexpr int kUnionBlocks = 1 << 15;
__global__ __launch_bounds__(kUnionThreads) void block_union_kernel(AttendArgs a) {
  __shared__ uint32_t marks[kUnionBlocks / 4];
  __shared__ int sums[kUnionThreads / kWave], places[8];
  const int kvh = blockIdx.x % a.hkv, tid = threadIdx.x, lane = tid & (kWave - 1);
  for (int m = blockIdx.x / a.hkv;; m += a.tiles_at_once) {
    const TokenTile tile = token_tile(a.sequences, a.first, a.first + a.tokens, a.batch, a.share, m);
    const int t = tile.first, tokens = tile.tokens, at = kvh * a.tokens + t - a.first;
    if (tokens == 0) {                                       // (the whole workgroup; the tiles of a later m are looked for only if there are any)
      if (tid == 0) a.tiles[m * a.hkv + kvh] = make_int4(0, 0, 0, 0);
      return;
    }
    // the tokens' places and the first entries of their lists, asked for together
    const int entries = tokens * a.keep, place = attend_last(a, t + min(lane, tokens - 1));
    auto entry = [&](int n) {
      const int i = n / a.keep;
      return a.blocks[((int64_t)(t + i) * a.hkv + kvh) * a.keep + (n - i * a.keep)];
    };
    int block = entry(min(tid, entries - 1));
    const int most = (int)lanes_largest((uint32_t)max((place >> a.page_shift) + 1, 0)), words = (most + 3) / 4;
    if (tid < 8) places[tid] = place;
    for (int w = tid; w < words; w += kUnionThreads) marks[w] = 0;
    __syncthreads();
    for (int n = tid; n < entries; n += kUnionThreads) {
      const int i = n / a.keep, last = places[i];
      if (n != tid) block = entry(n);
      if (block >= 0 && last >= 0 && block <= last >> a.page_shift) atomicOr(&marks[block >> 2], 1u << (8 * (block & 3) + i));
    }
    __syncthreads();
    const int per = (words + kUnionThreads - 1) / kUnionThreads, w0 = min(tid * per, words), w1 = min(w0 + per, words);
    int mine = 0;
    for (int w = w0; w < w1; ++w)
#pragma unroll
      for (int k = 0; k < 4; ++k) mine += (marks[w] >> 8 * k & 0xff) != 0;
    const int upto = (int)lanes_upto((uint32_t)mine);
    if (lane == kWave - 1) sums[tid / kWave] = upto;
    __syncthreads();
    int before = upto - mine, count = 0;
#pragma unroll
    for (int w = 0; w < kUnionThreads / kWave; ++w) {
      if (w < tid / kWave) before += sums[w];
      count += sums[w];
    }
    int2* out = a.merged + (int64_t)at * a.keep;
    for (int w = w0; w < w1; ++w)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (const int mark = marks[w] >> 8 * k & 0xff) out[before++] = make_int2(4 * w + k, mark);
    if (tid == 0) a.tiles[m * a.hkv + kvh] = make_int4(t - a.first, tokens, count, tile.all);
    if (m + a.tiles_at_once >= tile.all) return;
    __syncthreads();                                         // (marks and sums have been read)
  }
}

template <int D> __device__ __forceinline__ int attend_k_swap(int row) { return D == 128 ? row & 15 : (row >> 1) & 7; }
template <int D> __device__ __forceinline__ int attend_v_swap(int row) { return D == 128 ? 2 * (row & 7) : 2 * ((row >> 1) & 3); }

// Chunk `chunk` of the rows listed for `tokens` tokens from t on.  Where several share it, a row of the pool that one of them does not see has the probability 0 for it, and 0
// times an infinity or a NaN is no 0: true then (and nothing written), for the tokens' results to be found one after the other, `alone`, with zeros in such rows.
template <int DT, int D, int ROWT, bool SHARED>
__device__ __forceinline__ bool attend_unit(const AttendArgs& a, int kvh, int chunk, int t, int b, int tokens, int keys, int chunk_keys, int alone) {
  constexpr int kRowBytes = D * 2, kPieces = kRowBytes / 16, kRowsPerCopy = 64 / kPieces, kCopies = kAttendKeys / kRowsPerCopy;
  constexpr int kHalf = kAttendKeys * kRowBytes, kStage = 2 * kHalf;
  __shared__ __attribute__((aligned(1024))) uint8_t ring[kAttendStages * kStage];
  __shared__ int64_t row_at[kAttendSegment];
  __shared__ uint32_t seen_at[kAttendSegment / kAttendKeys];
  __shared__ __attribute__((aligned(16))) int place_at[SHARED ? kAttendSegment : 4];        // a key's row of the sequence, and its block's bits
  __shared__ uint32_t bits_at[SHARED ? kAttendSegment / 4 : 1];
  const int v_begin = chunk * chunk_keys, v_end = min(v_begin + chunk_keys, keys), local = t - a.first;
  const int lane = threadIdx.x, lq = lane & 15, lg = lane >> 4, rows = tokens * a.group;
  const int32_t* list = a.blocks + ((int64_t)t * a.hkv + kvh) * a.keep;
  const int2* merged = a.merged + ((int64_t)kvh * a.tokens + local) * a.keep;
  const int32_t* row_pages = a.table + b * a.table_stride;
  // The blocks of a segment's rows, and then their pages: each asked for all at once.  One after the other they are a trip to memory for every 64 rows and more
  // than the rows' own way takes.
  int block[kAttendSegment / 64], bits[kAttendSegment / 64];
  auto look_at = [&](int v0) {
#pragma unroll
    for (int u = 0; u < kAttendSegment / 64; ++u) {
      block[u] = -1;
      bits[u] = 1;
      if (u * 64 >= v_end - v0) continue;
      const int at = min(v0 + u * 64 + lane, v_end - 1) >> a.page_shift;
      if constexpr (SHARED) {
        const int2 entry = merged[at];
        block[u] = entry.x;
        bits[u] = entry.y;
      } else {
        block[u] = list[at];
      }
    }
  };
  look_at(v_begin);

  dec_u4 q[ROWT][D / 32];
  int token[ROWT], place[ROWT];                              // of a row: its token in the tile, the last row it sees
  int last = -1, least = INT32_MAX;
#pragma unroll
  for (int nt = 0; nt < ROWT; ++nt) {
    const int r = min(nt * 16 + lq, rows - 1), i = SHARED ? r / a.group : 0;
    token[nt] = i;
    place[nt] = attend_last(a, t + i);
    const uint16_t* src = a.q + (t + i) * a.q_token + (int64_t)(kvh * a.group + r - i * a.group) * a.q_head + lg * 8;
#pragma unroll
    for (int ks = 0; ks < D / 32; ++ks) q[nt][ks] = nt * 16 + lq < rows ? *(const dec_u4*)(src + ks * 32) : dec_u4{0, 0, 0, 0};
    last = max(last, place[nt]);
    least = min(least, place[nt]);
  }
  if constexpr (SHARED) {
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) {
      last = max(last, __shfl_xor(last, o, kWave));
      least = min(least, __shfl_xor(least, o, kWave));
    }
    if (alone >= 0) last = attend_last(a, t + alone);
  }
  v4f o[ROWT][D / 16];
  float ref[ROWT], l[ROWT];                                  // ref in units of exp2's argument
#pragma unroll
  for (int nt = 0; nt < ROWT; ++nt) {
    ref[nt] = -INFINITY;
    l[nt] = 0.f;
#pragma unroll
    for (int mt = 0; mt < D / 16; ++mt) o[nt][mt] = v4f{0.f, 0.f, 0.f, 0.f};
  }
  const uint32_t ring0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)ring;
  const char* kbase = (const char*)(a.pool + kvh * D);
  const int64_t v_bytes = a.page_elems * 2;
  const int crow = lane / kPieces, cpiece = lane % kPieces;
  const uint32_t koff = ring0 + lq * kRowBytes;
  const uint32_t voff = ring0 + kHalf + (4 * lg + (lq >> 2)) * kRowBytes + (lq & 1) * 8;
  const int kswap = attend_k_swap<D>(lq), vswap = attend_v_swap<D>(4 * lg + (lq >> 2)), vpiece = (lq >> 1) & 1;

  for (int v0 = v_begin; v0 < v_end; v0 += kAttendSegment) {
    int stages = 0;                                          // up to the last one of which something is seen
    if (v0 > v_begin) look_at(v0);
    uint32_t sees = 0;                                       // a bit for each of the lane's rows
    int page[kAttendSegment / 64];
#pragma unroll
    for (int u = 0; u < kAttendSegment / 64; ++u) {
      page[u] = 0;
      if (u * 64 >= v_end - v0) continue;
      const int v = v0 + u * 64 + lane, in = v & ((1 << a.page_shift) - 1);
      bool there = v < v_end && block[u] >= 0 && last >= 0 && block[u] <= last >> a.page_shift && (block[u] << a.page_shift) + in <= last;
      if (SHARED && alone >= 0) there = there && (bits[u] >> alone & 1);
      sees |= (uint32_t)there << u;
      page[u] = row_pages[there ? block[u] : 0];
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int u = 0; u < kAttendSegment / 64; ++u) {
      if (u * 64 >= v_end - v0) continue;
      const bool there = sees >> u & 1;
      const int in = (v0 + u * 64 + lane) & ((1 << a.page_shift) - 1);
      row_at[u * 64 + lane] = there ? 2 * ((int64_t)min(max(page[u], 0), a.max_pages - 1) * 2 * a.page_elems + (int64_t)a.hkv * D * in) : -1;
      const uint64_t some = __ballot(there);
      uint64_t all = some;                                   // (shared: seen by all rows)
      if constexpr (SHARED) {
        const int row = there ? (block[u] << a.page_shift) + in : INT32_MAX;
        place_at[u * 64 + lane] = row;
        ((uint8_t*)bits_at)[u * 64 + lane] = (uint8_t)bits[u];
        all = __ballot(row <= least && bits[u] == (1 << tokens) - 1);
      }
      if (lane < 2) seen_at[u * 2 + lane] = (uint32_t)(all >> (32 * lane));
      if (some) stages = u * 2 + (some >> 32 ? 2 : 1);
    }
    __builtin_amdgcn_s_waitcnt(0);                           // rows' offsets and the queries; from here on only copies are counted
    int64_t from[kCopies];                                   // of the copies to be asked for next: read together, well before their use
    auto look_up = [&](int st) {
#pragma unroll
      for (int c = 0; c < kCopies; ++c) from[c] = row_at[st * kAttendKeys + c * kRowsPerCopy + crow];
    };
    auto request = [&](int st) {
      const uint32_t at = ring0 + (uint32_t)(st % kAttendStages) * kStage;
#pragma unroll
      for (int c = 0; c < kCopies; ++c) {
        const int row = c * kRowsPerCopy + crow;
        const char* src = kbase + from[c];
        const char* k = from[c] < 0 ? (const char*)zero_piece : src + ((cpiece ^ attend_k_swap<D>(row)) << 4);
        const char* v = from[c] < 0 ? (const char*)zero_piece : src + v_bytes + ((cpiece ^ attend_v_swap<D>(row)) << 4);
        dma16_nt(at + c * 1024, k);
        dma16_nt(at + kHalf + c * 1024, v);
      }
    };
    for (int st = 0; st < min(kAttendStages, stages); ++st) {
      look_up(st);
      request(st);
    }
    for (int st = 0; st < stages; ++st) {
      if (st + kAttendStages <= stages) wait_vmcnt<(kAttendStages - 1) * 2 * kCopies>();
      else wait_vmcnt<0>();
      look_up(min(st + kAttendStages, stages - 1));
      const uint32_t at = (uint32_t)(st % kAttendStages) * kStage;
      const uint32_t seen = __builtin_amdgcn_readfirstlane(seen_at[st]);
      v4f s[ROWT][2];
#pragma unroll
      for (int nt = 0; nt < ROWT; ++nt) s[nt][0] = s[nt][1] = v4f{0.f, 0.f, 0.f, 0.f};
      // a stage's pieces asked for together: left to itself the compiler waits for each before it asks for the next
      dec_u4 kt[D / 32][2], vt[D / 16];
#pragma unroll
      for (int ks = 0; ks < D / 32; ++ks)
#pragma unroll
        for (int h = 0; h < 2; ++h) kt[ks][h] = lds_16(koff + at + h * 16 * kRowBytes + (((ks * 4 + lg) ^ kswap) << 4));
#pragma unroll
      for (int mt = 0; mt < D / 16; ++mt) {
        const uint32_t va = voff + at + (((mt * 2 + vpiece) ^ vswap) << 4);
        const uint2 lo = lds_tr16(va), hi = lds_tr16(va + 16 * kRowBytes);
        vt[mt] = dec_u4{lo.x, lo.y, hi.x, hi.y};
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int ks = 0; ks < D / 32; ++ks)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int nt = 0; nt < ROWT; ++nt) s[nt][h] = mfma16x16x32<DT>(kt[ks][h], q[nt][ks], s[nt][h]);
      dec_i4 places[2] = {};
      uint32_t bits[2] = {};
      if (SHARED && seen != ~0u) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          places[h] = *(const dec_i4*)&place_at[st * kAttendKeys + h * 16 + 4 * lg];
          bits[h] = bits_at[(st * kAttendKeys + h * 16) / 4 + lg];
        }
      }
      dec_u4 pb[ROWT], rest[ROWT];
#pragma unroll
      for (int nt = 0; nt < ROWT; ++nt) {
        float x[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) x[r] = s[nt][r >> 2][r & 3];
        if (seen != ~0u) {
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            const int key = (r >> 2) * 16 + 4 * lg + (r & 3);
            bool there = seen >> key & 1;
            if constexpr (SHARED) there = places[r >> 2][r & 3] <= place[nt] && (bits[r >> 2] >> (8 * (r & 3) + token[nt]) & 1);
            if (!there) x[r] = -INFINITY;
          }
        }
        const float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7]))) * a.scale_log2;
        if (__any(top > ref[nt] + kSlack)) {                 // (also where the reference is still -inf)
          float m = fmaxf(top, __shfl_xor(top, 16, kWave));
          m = fmaxf(m, __shfl_xor(m, 32, kWave));
          const float next = m > ref[nt] + kSlack ? m : ref[nt];
          const float alpha = next == ref[nt] ? 1.f : __builtin_amdgcn_exp2f(ref[nt] - next);
          ref[nt] = next;
          l[nt] *= alpha;
#pragma unroll
          for (int mt = 0; mt < D / 16; ++mt) o[nt][mt] *= alpha;
        }
        const float base = ref[nt] == -INFINITY ? 0.f : ref[nt];
        float e[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) e[r] = __builtin_amdgcn_exp2f(fmaf(x[r], a.scale_log2, -base));
        l[nt] += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
        pb[nt] = pack8<DT>(e);
        float near[8];
        unpack8<DT>(pb[nt], near);
#pragma unroll
        for (int r = 0; r < 8; ++r) e[r] -= near[r];
        rest[nt] = pack8<DT>(e);
#pragma unroll
        for (int mt = 0; mt < D / 16; ++mt) {
          o[nt][mt] = mfma16x16x32<DT>(vt[mt], pb[nt], o[nt][mt]);
          o[nt][mt] = mfma16x16x32<DT>(vt[mt], rest[nt], o[nt][mt]);
        }
      }
      if (st + kAttendStages < stages) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the stage has been read
        request(st + kAttendStages);
      }
    }
  }

  if (SHARED && alone < 0 && tokens > 1) {
    float none = 0.f;                                        // (NaN where a sum is infinite or NaN)
#pragma unroll
    for (int nt = 0; nt < ROWT; ++nt)
#pragma unroll
      for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e) none = fmaf(o[nt][mt][e], 0.f, none);
    if (__any(none != none)) return true;
  }
#pragma unroll
  for (int nt = 0; nt < ROWT; ++nt) {
    float sum = l[nt] + __shfl_xor(l[nt], 16, kWave);
    sum += __shfl_xor(sum, 32, kWave);
    const int r = nt * 16 + lq;
    if (r >= rows || (SHARED && alone >= 0 && token[nt] != alone)) continue;
    const int head = r - token[nt] * a.group;
    if (a.chunks == 1) {
      const float inv = sum > 0.f ? 1.0f / sum : 0.f;
      uint16_t* dst = a.out + ((int64_t)(t + token[nt]) * a.hq + kvh * a.group + head) * D + lg * 4;
#pragma unroll
      for (int mt = 0; mt < D / 16; ++mt)
        *(uint2*)(dst + mt * 16) = make_uint2(pack2<DT>(o[nt][mt][0] * inv, o[nt][mt][1] * inv), pack2<DT>(o[nt][mt][2] * inv, o[nt][mt][3] * inv));
    } else {
      const int64_t slot = (((int64_t)(local + token[nt]) * a.hkv + kvh) * a.chunks + chunk) * a.group + head;
      float* dst = a.part_o + slot * D + lg * 4;
#pragma unroll
      for (int mt = 0; mt < D / 16; ++mt) *(v4f*)(dst + mt * 16) = o[nt][mt];
      if (lg == 0) *(v2f*)(a.part_ml + slot * 2) = v2f{ref[nt], sum};
    }
  }
  return false;
}

template <int DT, int D, int ROWT, bool SHARED>
__global__ __launch_bounds__(kWave) void block_attention_kernel(AttendArgs a) {
  const uint32_t unit = blockIdx.x, tc = unit / (uint32_t)a.hkv;
  const int kvh = (int)(unit % (uint32_t)a.hkv), chunk = (int)(tc % (uint32_t)a.chunks), local = (int)(tc / (uint32_t)a.chunks);
  if constexpr (!SHARED) {
    const int b = a.sequences[a.first + local];
    if (b >= 0 && b < a.batch) attend_unit<DT, D, ROWT, false>(a, kvh, chunk, a.first + local, b, 1, a.keys, a.chunk_keys, -1);
  } else {
    // its first token, how many it has, their blocks; the tiles of the call
    auto tile_of = [&](int m) {
      const int4 v = a.tiles[m * a.hkv + kvh];
      return make_int4(__builtin_amdgcn_readfirstlane(v.x), __builtin_amdgcn_readfirstlane(v.y), __builtin_amdgcn_readfirstlane(v.z),
                       __builtin_amdgcn_readfirstlane(v.w));
    };
    int4 tile = tile_of(local);
    if (tile.y == 0) return;
    for (int m = local, alone = -1;;) {
      const int t = a.first + tile.x, keys = tile.z << a.page_shift, chunks = min(tile_chunks(keys, tile.w * a.hkv), a.chunks);
      if (chunk < chunks) {
        if (chunk == 0 && (int)threadIdx.x < tile.y) a.parts[kvh * a.tokens + tile.x + threadIdx.x] = chunks;
        const int each = ((keys + chunks - 1) / chunks + kAttendKeys - 1) / kAttendKeys * kAttendKeys;
        const bool apart = attend_unit<DT, D, ROWT, true>(a, kvh, chunk, t, a.sequences[t], tile.y, keys, each, alone);
        alone = alone < 0 && !apart ? tile.y : alone + 1;
        if (alone < tile.y) continue;
      }
      alone = -1;
      m += a.tiles_at_once;
      if (m >= tile.w) return;
      tile = tile_of(m);
    }
  }
}

// out = sum_c 2^(ref_c - max ref) O_c / sum_c 2^(ref_c - max ref) l_c, a wavefront a row
template <int DT, int D>
__global__ __launch_bounds__(256) void block_merge_kernel(AttendArgs a, int64_t rows) {
  constexpr int kLanes = D / 4, kSide = kWave / kLanes;
  const int64_t id = (int64_t)blockIdx.x * 4 + threadIdx.x / kWave;              // (token, KV head, row)
  if (id >= rows) return;
  const int lane = threadIdx.x & (kWave - 1), r = (int)(id % a.group);
  const int64_t tk = id / a.group;
  const int t = a.first + (int)(tk / a.hkv), kvh = (int)(tk % a.hkv);
  const int b = a.sequences[t];
  const int64_t slot = tk * a.chunks * a.group + r;
  const float* ml = a.part_ml + slot * 2;
  const float* po = a.part_o + slot * D + (lane % kLanes) * 4;
  const int side = lane / kLanes;
  // the first chunks' parts, and every lane's chunk's reference and sum, on their way before anything is known of them
  constexpr int kHeld = 16 / kSide;
  v4f early[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) early[i] = *(const v4f*)(po + (int64_t)min(i * kSide + side, a.chunks - 1) * a.group * D);
  v2f mine = *(const v2f*)(ml + (int64_t)min(lane, a.chunks - 1) * a.group * 2);
  if (b < 0 || b >= a.batch) return;
  int chunks = a.chunks;
  if (a.share) chunks = min(max(a.parts[kvh * a.tokens + (t - a.first)], 1), a.chunks);
  float top = lane < chunks ? mine[0] : -INFINITY;
  for (int c = lane + kWave; c < chunks; c += kWave) top = fmaxf(top, ml[(int64_t)c * a.group * 2]);
  top = wave_max(top);
  const float base = top == -INFINITY ? 0.f : top;
  v4f num = {0.f, 0.f, 0.f, 0.f};
  float den = 0.f;
  for (int c0 = 0; c0 < chunks; c0 += kWave) {
    if (c0 > 0) mine = *(const v2f*)(ml + (int64_t)min(c0 + lane, chunks - 1) * a.group * 2);
    const float weight = c0 + lane < chunks ? __builtin_amdgcn_exp2f(mine[0] - base) : 0.f;
    den = fmaf(weight, c0 + lane < chunks ? mine[1] : 0.f, den);
    const int some = min(kWave, chunks - c0);
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      if (c0 > 0 || i * kSide >= some) break;                // (uniform)
      const float w = __shfl(weight, i * kSide + side, kWave);
#pragma unroll
      for (int e = 0; e < 4; ++e) num[e] = i * kSide + side < some ? fmaf(w, early[i][e], num[e]) : num[e];
    }
    for (int c = c0 > 0 ? 0 : kHeld * kSide; c < some; c += 4 * kSide) {
      v4f part[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) part[i] = *(const v4f*)(po + (int64_t)(c0 + min(c + i * kSide + side, some - 1)) * a.group * D);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int from = c + i * kSide + side;
        const float w = __shfl(weight, min(from, kWave - 1), kWave);
#pragma unroll
        for (int e = 0; e < 4; ++e) num[e] = from < some ? fmaf(w, part[i][e], num[e]) : num[e];
      }
    }
  }
  den = wave_sum(den);
#pragma unroll
  for (int s = kLanes; s < kWave; s <<= 1)
#pragma unroll
    for (int e = 0; e < 4; ++e) num[e] += __shfl_xor(num[e], s, kWave);
  if (lane >= kLanes) return;
  const float inv = den > 0.f ? 1.f / den : 0.f;
  *(uint2*)(a.out + ((int64_t)t * a.hq + kvh * a.group + r) * D + lane * 4) =
      make_uint2(pack2<DT>(num[0] * inv, num[1] * inv), pack2<DT>(num[2] * inv, num[3] * inv));
}

// Tokens of a sequence that share a unit (1: none do), chunks of a unit's rows, tokens whose partial results are held at a time.
struct AttendPlan { int share, chunk_keys, chunks; int64_t tokens; size_t part_o, part_ml, tiles, merged, parts, bytes; };
static AttendPlan attend_plan(int64_t batch, int64_t n_tokens, int64_t hq, int64_t hkv, int64_t head_dim, int64_t page_len, int64_t max_blocks, int64_t keep) {
  AttendPlan p{};
  const int64_t group = hq / hkv;
  p.share = 1;
  if (n_tokens > batch && max_blocks <= kUnionBlocks)
    while (p.share < 8 && 2 * p.share * group <= kShareRows) p.share *= 2;
  // rows of a unit: those of a token, or, of several, as many as lists that agree in most blocks have together
  const int64_t most = std::min(p.share * keep, std::max(max_blocks, keep)) * page_len, keys = p.share > 1 ? std::min(most, 2 * keep * page_len) : keep * page_len;
  // (where several share: as many tiles as sequences, or as their tokens fill)
  const int64_t units = (p.share > 1 ? std::max<int64_t>(std::min<int64_t>(n_tokens, batch), std::min<int64_t>(n_tokens, kTileTokens) / p.share) : n_tokens) * hkv;
  int64_t per;
  if (p.share > 1) {
    const int64_t chunks = tile_chunks((int)keys, (int)units);
    per = (keys + chunks - 1) / chunks;
  } else {
    per = ((int64_t)(0.65 * std::sqrt((double)units * (double)keys)) + kAttendKeys - 1) / kAttendKeys * kAttendKeys;
    per = std::min<int64_t>(std::max<int64_t>(per, 64), 384);
  }
  while (keys > per * 256) per *= 2;
  p.chunk_keys = (int)per;
  p.chunks = (int)((keys + per - 1) / per);
  p.tokens = p.share > 1 ? std::min<int64_t>(n_tokens, kTileTokens) : n_tokens;
  if (p.chunks > 1) p.tokens = std::min<int64_t>(p.tokens, std::max<int64_t>(8, (1 << 20) / (hq * p.chunks)));      // half a gigabyte at 128 a head
  p.tokens = std::min<int64_t>(p.tokens, (1 << 25) / (p.chunks * hkv));        // (a launch has below 2^32 threads, a unit 64 of them)
  const size_t slots = (size_t)p.tokens * hq * p.chunks;
  if (p.chunks > 1) {
    p.part_o = align_up(slots * head_dim * sizeof(float), 256);
    p.part_ml = align_up(slots * 2 * sizeof(float), 256);
  }
  if (p.share > 1) {
    p.tiles = align_up((size_t)p.tokens * hkv * sizeof(int4), 256);
    p.merged = align_up((size_t)p.tokens * hkv * keep * sizeof(int2), 256);
    p.parts = align_up((size_t)p.tokens * hkv * sizeof(int32_t), 256);
  }
  p.bytes = 256 + p.part_o + p.part_ml + p.tiles + p.merged + p.parts;
  return p;
}

// Tokens of a pass: their scores are a quarter of a gigabyte, and their lists, a workgroup of up to 512 threads each, no more than a launch can have (below 2^32 threads).
static int64_t select_tokens(int64_t n_tokens, int64_t hkv, int64_t most) {
  const int64_t fit = std::max<int64_t>(kScoreTokens, std::min((1 << 25) / (hkv * std::max<int64_t>(most, 1)), (1 << 22) / hkv) / kScoreTokens * kScoreTokens);
  return std::min(n_tokens, fit);
}

// More tokens than sequences: some have several, which share readings.
template <int DT, int D>
static void launch_scores(SelectArgs a, hipStream_t st) {
  const bool shared = a.tokens > a.batch;
  a.span = kScoreThreads / (D / 8) * (shared ? kSharedDepth : 8);
  a.spans = (int)((a.most + a.span - 1) / a.span);
  a.tiles_at_once = tiles_at_once(a.tokens, a.batch, kScoreTokens);
  const int64_t tiles = std::max<int64_t>(a.batch, a.tokens / kScoreTokens) * a.hkv;
  const bool more = tiles * a.spans > kScoreBlocks;
  a.spans_at_once = more ? (int)std::max<int64_t>(1, kScoreBlocks / 3 / tiles) : a.spans;
  const dim3 grid((unsigned)((int64_t)(shared ? (int64_t)a.tiles_at_once * a.spans_at_once : (int64_t)a.tokens * a.spans) * a.hkv)), block(kScoreThreads);
  if (shared && more) hipLaunchKernelGGL((block_score_shared_kernel<DT, D, true>), grid, block, 0, st, a);
  else if (shared) hipLaunchKernelGGL((block_score_shared_kernel<DT, D, false>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((block_score_kernel<DT, D>), grid, block, 0, st, a);
}

template <int DT, int D>
static void launch_attend_of(const AttendArgs& a, int64_t tokens, hipStream_t st) {
  const dim3 grid((unsigned)((a.share ? a.tiles_at_once : tokens) * a.chunks * a.hkv)), block(kWave);
  if (a.share) {
    if (a.share * a.group <= 16) hipLaunchKernelGGL((block_attention_kernel<DT, D, 1, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((block_attention_kernel<DT, D, 2, true>), grid, block, 0, st, a);
  } else {
    if (a.group <= 16) hipLaunchKernelGGL((block_attention_kernel<DT, D, 1, false>), grid, block, 0, st, a);
    else if (a.group <= 32) hipLaunchKernelGGL((block_attention_kernel<DT, D, 2, false>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((block_attention_kernel<DT, D, 4, false>), grid, block, 0, st, a);
  }
}
template <int DT, int D>
static void launch_block_merge_of(const AttendArgs& a, int64_t tokens, hipStream_t st) {
  const int64_t rows = tokens * a.hq;
  hipLaunchKernelGGL((block_merge_kernel<DT, D>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, a, rows);
}

}  // namespace subspec

using namespace subspec;

static int check_pool_shape(const char* what, int dtype, int64_t head_dim, int64_t max_pages, int64_t page_len) {
  if (dtype != SUBSPEC_BF16 && dtype != SUBSPEC_F16)
    SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: dtype %d not supported (bf16 / fp16 only)", what, dtype);
  if (head_dim != 64 && head_dim != 128)
    SUBSPEC_FAIL(SUBSPEC_ERR_LIMIT, "%s: head_dim=%lld (built for 64 and 128)", what, (long long)head_dim);
  if (page_len < 1 || page_len > (1 << 20) || (page_len & (page_len - 1)))
    SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: page_len=%lld is no power of two up to 2^20", what, (long long)page_len);
  if (max_pages < 1 || max_pages > INT32_MAX) SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: %lld pages", what, (long long)max_pages);
  return SUBSPEC_OK;
}
static int check_batch(const char* what, int64_t batch, int64_t n_tokens, int64_t hq, int64_t hkv, int64_t max_blocks, int64_t table_stride) {
  if (batch < 1 || batch > SUBSPEC_MAX_BATCH)
    SUBSPEC_FAIL(SUBSPEC_ERR_LIMIT, "%s: batch=%lld outside [1, %d]", what, (long long)batch, SUBSPEC_MAX_BATCH);
  if (n_tokens < 0 || n_tokens > (1 << 20)) SUBSPEC_FAIL(SUBSPEC_ERR_LIMIT, "%s: n_tokens=%lld outside [0, 2^20]", what, (long long)n_tokens);
  if (hq < 1 || hkv < 1 || hq % hkv || hq > 1024) SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: heads=%lld/%lld", what, (long long)hq, (long long)hkv);
  if (max_blocks < 1 || max_blocks > INT32_MAX || table_stride < max_blocks)
    SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: a table of %lld columns with a row stride of %lld", what, (long long)max_blocks, (long long)table_stride);
  return SUBSPEC_OK;
}

extern "C" int subspec_kv_page_bounds(const void* kv_pool_layer, void* bounds, int dtype, int64_t max_pages, int64_t page_len,
                                      int64_t n_kv_heads, int64_t head_dim, const int64_t* slots, int64_t n_tokens, void* stream) {
  const char* what = "kv_page_bounds";
  if (const int code = check_pool_shape(what, dtype, head_dim, max_pages, page_len)) return code;
  if (n_kv_heads < 1 || n_kv_heads > 1024) SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: %lld heads", what, (long long)n_kv_heads);
  if (n_tokens < 0 || n_tokens > (1ll << 30)) SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: n_tokens=%lld", what, (long long)n_tokens);
  if (n_tokens == 0) return SUBSPEC_OK;
  if (!kv_pool_layer || !bounds || !slots) SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: null pointer argument", what);
  if ((uintptr_t)kv_pool_layer % 16 || (uintptr_t)bounds % 16) SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: the pool and bounds must be 16-byte aligned", what);
  BoundsArgs a;
  a.pool = (const uint16_t*)kv_pool_layer; a.bounds = (uint16_t*)bounds; a.slots = slots;
  a.n_slots = max_pages * page_len; a.page_elems = page_len * n_kv_heads * head_dim;
  a.n_tokens = (int)n_tokens; a.page_shift = block_shift_of(page_len);
  a.pieces = (int)(n_kv_heads * head_dim / 8); a.head_pieces = (int)(head_dim / 8);
  a.infinity = dtype == SUBSPEC_BF16 ? 0x7f80 : 0x7c00;
  hipStream_t st = (hipStream_t)stream;
  DominantKernelTimer timer(st);
  if (a.pieces <= 8) launch_bounds<8>(a, st);
  else launch_bounds<16>(a, st);
  SUBSPEC_CHECK_HIP(hipGetLastError());
  return SUBSPEC_OK;
}

// blocks that any token of a call can see
static int64_t most_blocks(int64_t page_len, int64_t max_blocks, int64_t max_kv) {
  return std::min(max_blocks, (max_kv + page_len - 1) / page_len);
}

extern "C" size_t subspec_select_blocks_workspace(int64_t n_tokens, int64_t n_kv_heads, int64_t page_len, int64_t max_blocks, int64_t max_kv) {
  if (n_tokens < 1 || n_tokens > (1 << 20) || n_kv_heads < 1 || n_kv_heads > 1024 || page_len < 1 || max_blocks < 1 || max_kv < 0 ||
      max_kv > (1ll << 30) || max_blocks > INT32_MAX)
    return 256;
  const int64_t most = most_blocks(page_len, max_blocks, max_kv);
  if (most > kMostBlocks) return 256;
  return 256 + (size_t)select_tokens(n_tokens, n_kv_heads, most) * n_kv_heads * most * sizeof(double);
}

extern "C" int subspec_select_blocks(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* bounds, int dtype,
                                     int64_t max_pages, int64_t page_len, const int32_t* block_table, int64_t max_blocks,
                                     int64_t table_stride, const int32_t* sequences, const int32_t* positions, int64_t batch,
                                     int64_t n_tokens, int64_t n_q_heads, int64_t n_kv_heads, int64_t head_dim, int64_t max_kv,
                                     int64_t keep, int64_t recent, int32_t* blocks, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "select_blocks";
  if (const int code = check_pool_shape(what, dtype, head_dim, max_pages, page_len)) return code;
  if (const int code = check_batch(what, batch, n_tokens, n_q_heads, n_kv_heads, max_blocks, table_stride)) return code;
  if (max_kv < 0 || max_kv > (1ll << 30)) SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: max_kv=%lld outside [0, 2^30]", what, (long long)max_kv);
  if (recent < 1 || keep < recent || keep > kMostBlocks)
    SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: keep=%lld (at most 2^17), recent=%lld (1 to keep)", what, (long long)keep, (long long)recent);
  const int64_t most = most_blocks(page_len, max_blocks, max_kv);
  if (most > kMostBlocks)
    SUBSPEC_FAIL(SUBSPEC_ERR_LIMIT, "%s: %lld blocks a sequence (at most 2^17): larger pages, or a smaller max_kv", what, (long long)most);
  if (n_tokens == 0) return SUBSPEC_OK;
  if (!q || !bounds || !block_table || !sequences || !positions || !blocks) SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: null pointer argument", what);
  if ((uintptr_t)q % 16 || (uintptr_t)bounds % 16 || q_token_stride % 8 || q_head_stride % 8 || q_token_stride < 0 || q_head_stride < 0)
    SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: q and bounds must be 16-byte aligned, q's strides multiples of 8 elements", what);
  const size_t need = subspec_select_blocks_workspace(n_tokens, n_kv_heads, page_len, max_blocks, max_kv);
  if (need > 256 && (!workspace || workspace_bytes < need))
    SUBSPEC_FAIL(SUBSPEC_ERR_WORKSPACE, "%s: workspace of %zu bytes is smaller than the %zu required", what, workspace_bytes, need);
  if ((uintptr_t)workspace % 16) SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: workspace must be 16-byte aligned", what);
  SelectArgs a;
  a.q = (const uint16_t*)q; a.bounds = (const uint16_t*)bounds; a.table = block_table; a.sequences = sequences; a.positions = positions;
  a.blocks = blocks; a.scores = (double*)workspace;
  a.q_token = q_token_stride; a.q_head = q_head_stride; a.table_stride = table_stride; a.most = most;
  a.batch = (int)batch; a.hkv = (int)n_kv_heads; a.group = (int)(n_q_heads / n_kv_heads);
  a.page_shift = block_shift_of(page_len); a.max_pages = (int)max_pages; a.keep = (int)keep; a.recent = (int)recent;
  a.last_row = (int)(std::min(max_kv, max_blocks * page_len) - 1);
  int64_t at_once = select_tokens(n_tokens, n_kv_heads, most);
  if (n_tokens > batch && most > keep) at_once = std::min<int64_t>(at_once, kTileTokens);
  hipStream_t st = (hipStream_t)stream;
  for (int64_t first = 0; first < n_tokens; first += at_once) {
    const int64_t some = std::min(at_once, n_tokens - first);
    a.first = (int)first;
    a.tokens = (int)some;
    if (most > keep) {
      DominantKernelTimer timer(st);
      if (dtype == SUBSPEC_BF16) {
        if (head_dim == 128) launch_scores<SUBSPEC_BF16, 128>(a, st);
        else launch_scores<SUBSPEC_BF16, 64>(a, st);
      } else {
        if (head_dim == 128) launch_scores<SUBSPEC_F16, 128>(a, st);
        else launch_scores<SUBSPEC_F16, 64>(a, st);
      }
    }
    // (up to 255 blocks 5.4 us with 256 threads, a wave's steps fewer; 2048 blocks 6.2 with 512, two rounds of entries fewer: 6.8 and 9.0, 8.6 and 7.6 when these were compared)
    const dim3 lists((unsigned)(some * n_kv_heads));
    if (most <= 512) hipLaunchKernelGGL(block_select_kernel<256>, lists, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(block_select_kernel<512>, lists, dim3(512), 0, st, a);
  }
  SUBSPEC_CHECK_HIP(hipGetLastError());
  return SUBSPEC_OK;
}

extern "C" size_t subspec_block_attention_workspace(int64_t batch, int64_t n_tokens, int64_t n_q_heads, int64_t n_kv_heads, int64_t head_dim,
                                                    int64_t page_len, int64_t max_blocks, int64_t keep) {
  if (batch < 1 || max_blocks < 1 || max_blocks > INT32_MAX || n_tokens < 1 || n_tokens > (1 << 20) || n_kv_heads < 1 || n_q_heads < n_kv_heads || n_q_heads > 1024 || head_dim < 1 || head_dim > 1024 ||
      page_len < 1 || page_len > (1 << 20) || keep < 1 || keep > kMostBlocks || keep * page_len > (1 << 30))
    return 256;
  return attend_plan(batch, n_tokens, n_q_heads, n_kv_heads, head_dim, page_len, most_blocks(page_len, max_blocks, 1ll << 30), keep).bytes;
}

extern "C" int subspec_block_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* kv_pool_layer, int dtype,
                                       int64_t max_pages, int64_t page_len, const int32_t* block_table, int64_t max_blocks,
                                       int64_t table_stride, const int32_t* blocks, int64_t keep, const int32_t* sequences,
                                       const int32_t* positions, int64_t batch, int64_t n_tokens, int64_t n_q_heads, int64_t n_kv_heads,
                                       int64_t head_dim, float scale, void* out, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "block_attention";
  if (const int code = check_pool_shape(what, dtype, head_dim, max_pages, page_len)) return code;
  if (const int code = check_batch(what, batch, n_tokens, n_q_heads, n_kv_heads, max_blocks, table_stride)) return code;
  if (n_q_heads / n_kv_heads > 64)
    SUBSPEC_FAIL(SUBSPEC_ERR_LIMIT, "%s: %lld query heads a KV head (at most 64)", what, (long long)(n_q_heads / n_kv_heads));
  if (keep < 1 || keep > kMostBlocks || keep * page_len > (1 << 30))
    SUBSPEC_FAIL(SUBSPEC_ERR_LIMIT, "%s: %lld blocks of %lld rows a token (2^17 blocks, 2^30 rows at most)", what, (long long)keep,
                 (long long)page_len);
  if (!(scale > 0.f) || scale > 1e30f) SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: scale=%g must be positive", what, (double)scale);
  if (n_tokens == 0) return SUBSPEC_OK;
  if (!q || !kv_pool_layer || !block_table || !blocks || !sequences || !positions || !out)
    SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: null pointer argument", what);
  if ((uintptr_t)q % 16 || (uintptr_t)kv_pool_layer % 16 || (uintptr_t)out % 16 || q_token_stride % 8 || q_head_stride % 8 ||
      q_token_stride < 0 || q_head_stride < 0)
    SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: q, the pool and out must be 16-byte aligned, q's strides multiples of 8 elements", what);
  const AttendPlan p = attend_plan(batch, n_tokens, n_q_heads, n_kv_heads, head_dim, page_len, most_blocks(page_len, max_blocks, 1ll << 30), keep);
  if (p.bytes > 256 && (!workspace || workspace_bytes < p.bytes))
    SUBSPEC_FAIL(SUBSPEC_ERR_WORKSPACE, "%s: workspace of %zu bytes is smaller than the %zu required", what, workspace_bytes, p.bytes);
  if ((uintptr_t)workspace % 16) SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: workspace must be 16-byte aligned", what);
  AttendArgs a;
  a.q = (const uint16_t*)q; a.pool = (const uint16_t*)kv_pool_layer; a.table = block_table; a.blocks = blocks; a.sequences = sequences;
  a.positions = positions; a.out = (uint16_t*)out;
  char* ws = (char*)workspace;
  a.part_o = (float*)ws; ws += p.part_o;
  a.part_ml = (float*)ws; ws += p.part_ml;
  a.tiles = (int4*)ws; ws += p.tiles;
  a.merged = (int2*)ws; ws += p.merged;
  a.parts = (int32_t*)ws;
  a.share = p.share > 1 ? p.share : 0;
  a.q_token = q_token_stride; a.q_head = q_head_stride; a.table_stride = table_stride; a.page_elems = page_len * n_kv_heads * head_dim;
  a.batch = (int)batch; a.hq = (int)n_q_heads; a.hkv = (int)n_kv_heads; a.group = (int)(n_q_heads / n_kv_heads);
  a.page_shift = block_shift_of(page_len); a.max_pages = (int)max_pages; a.keep = (int)keep;
  a.last_row = (int)(std::min<int64_t>(max_blocks * page_len, 1ll << 30) - 1);
  a.keys = (int)(keep * page_len); a.chunk_keys = p.chunk_keys; a.chunks = p.chunks;
  a.scale_log2 = scale * kLog2e;
  hipStream_t st = (hipStream_t)stream;
  for (int64_t first = 0; first < n_tokens; first += p.tokens) {
    const int64_t some = std::min(p.tokens, n_tokens - first);
    a.first = (int)first;
    a.tokens = (int)some;
    if (a.share) {
      a.tiles_at_once = tiles_at_once(some, batch, a.share);
      hipLaunchKernelGGL(block_union_kernel, dim3((unsigned)(a.tiles_at_once * n_kv_heads)), dim3(kUnionThreads), 0, st, a);
    }
    {
      DominantKernelTimer timer(st);
      if (dtype == SUBSPEC_BF16) {
        if (head_dim == 128) launch_attend_of<SUBSPEC_BF16, 128>(a, some, st);
        else launch_attend_of<SUBSPEC_BF16, 64>(a, some, st);
      } else {
        if (head_dim == 128) launch_attend_of<SUBSPEC_F16, 128>(a, some, st);
        else launch_attend_of<SUBSPEC_F16, 64>(a, some, st);
      }
    }
    if (p.chunks > 1) {
      if (dtype == SUBSPEC_BF16) {
        if (head_dim == 128) launch_block_merge_of<SUBSPEC_BF16, 128>(a, some, st);
        else launch_block_merge_of<SUBSPEC_BF16, 64>(a, some, st);
      } else {
        if (head_dim == 128) launch_block_merge_of<SUBSPEC_F16, 128>(a, some, st);
        else launch_block_merge_of<SUBSPEC_F16, 64>(a, some, st);
      }
    }
  }
  SUBSPEC_CHECK_HIP(hipGetLastError());
  return SUBSPEC_OK;
}
