// Attention of the new tokens of a batch of sequences over a page pool, for gfx950.
//
// The new tokens are packed; sequence b's are query_starts[b] .. query_starts[b + 1] - 1, and the row r = (token i of them) * group + head of
// a KV head's query heads is a row of that KV head's products, so that all query heads of a group share a key's way out of memory.
// Every length is read on the device; the host knows bounds only (max_new, max_kv) and lays out launches and workspace by them.
#include "paged.h"
#include <algorithm>
#include <cmath>

namespace subspec {

// ---------------------------------------------------------------------------------------------------------------- few rows
// Sequences whose new tokens make at most 16 ROWT rows a KV head (one token of up to 64 query heads, a handful of tokens of a few): the
// call is the K / V rows' way out of memory, and everything is arranged for that.  A unit is (sequence, KV head, chunk of the keys) and ONE
// wavefront: it has no barrier to meet anyone at, so four of them share a compute unit and each waits for its own rows only.  Rows
// travel from memory straight into the wavefront's ring of LDS stages, 32 keys each, which the transposing reads of V need anyway; a stage is
// asked for again as soon as it has been read.  The rows are read once and copied as streaming data: 64 tokens of up to 4096 rows, 28 : 4
// heads, 348 MB: 70.8 us against 79.6, 16 of up to 32768 rows, 32 : 8, 1.3 GB: 243 against 262 (5.5 TB/s; a large copy reaches 5.2 here).
// A probability is rounded once, to the type of the product with V; the row's sum takes it before that, in fp32 (the tiles' kernel takes it after, where
// one instruction adds a rounded pair).  The two differ by half a step of the type at most (in fp16 and 2^-25 a key), mostly far less: roundings cancel.
// S^T = K Q^T and O^T = V^T P^T by 16x16x32 products: the two accumulators of a stage (eight keys of one query a lane) are, packed, the
// operand of the second, with its keys taken in the same order from V.
// A row's probabilities are relative to a reference that follows its largest score by at most 2^8 (see kSlack), so that a stage without a
// new maximum needs no step across lanes.  Rows of a stage: the 16-byte pieces are swapped (XOR) so that 16 rows' reads of one piece, and the
// transposing reads of 8 rows' two pieces, cover all banks.
constexpr int kFewKeys = 32;
constexpr int kFewStages = 2;
constexpr int kSegment = 512;             // keys whose row offsets are in LDS at a time

// where the stored piece of a row is, in pieces: K is read a piece of 16 rows at a time, V two pieces of 8 rows
template <int D> __device__ __forceinline__ int few_k_swap(int row) { return D == 128 ? row & 15 : (row >> 1) & 7; }
template <int D> __device__ __forceinline__ int few_v_swap(int row) { return D == 128 ? 2 * (row & 7) : 2 * ((row >> 1) & 3); }

template <int DT, int D, int ROWT>
__global__ __launch_bounds__(64) void paged_few_kernel(PagedParams p) {
  constexpr int kRowBytes = D * 2, kPieces = kRowBytes / 16, kRowsPerCopy = 64 / kPieces, kCopies = kFewKeys / kRowsPerCopy;
  constexpr int kHalf = kFewKeys * kRowBytes, kStage = 2 * kHalf;
  __shared__ __attribute__((aligned(1024))) uint8_t ring[kFewStages * kStage];
  __shared__ int64_t row_at[kSegment];
  const uint32_t unit = blockIdx.x;
  const int kvh = (int)(unit % (uint32_t)p.hkv);
  const uint32_t bc = unit / (uint32_t)p.hkv;
  const int chunk = (int)(bc % (uint32_t)p.few.chunks), b = (int)(bc / (uint32_t)p.few.chunks);
  const PagedSequence sq = paged_sequence(p, b);
  const int rows = sq.n * p.group;
  if (sq.n <= 0 || rows > p.few.rows) return;
  const PagedSpan sp = paged_span(p, sq.len, sq.pos0, sq.pos0 + sq.n - 1, kFewKeys);
  const int chunks = paged_chunks(sp, p.few.chunk_keys);
  if (chunk >= chunks) return;
  const int lane = threadIdx.x, lq = lane & 15, lg = lane >> 4;

  dec_u4 q[ROWT][D / 32];
  int pos[ROWT];
  int64_t out_at[ROWT];                                     // row (token, head) of the output
#pragma unroll
  for (int nt = 0; nt < ROWT; ++nt) {
    const int r = nt * 16 + lq, i = r / p.group;
    const bool ok = r < rows;
    const int token = sq.first + (ok ? i : 0), head = kvh * p.group + (ok ? r - i * p.group : 0);
    pos[nt] = ok ? max(sq.pos0 + i, -1) : -1;
    out_at[nt] = (int64_t)token * p.hq + head;
    const uint16_t* src = p.q + token * p.q_token + head * p.q_head + lg * 8;
#pragma unroll
    for (int ks = 0; ks < D / 32; ++ks) q[nt][ks] = ok ? *(const dec_u4*)(src + ks * 32) : dec_u4{0, 0, 0, 0};
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
  const int v_begin = chunk * p.few.chunk_keys, v_end = min(v_begin + p.few.chunk_keys, sp.length);
  const uint32_t ring0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)ring;
  const char* kbase = (const char*)(p.pool + kvh * D);
  const int64_t v_bytes = p.page_elems * 2;
  const int crow = lane / kPieces, cpiece = lane % kPieces;
  const uint32_t koff = ring0 + lq * kRowBytes;
  const uint32_t voff = ring0 + kHalf + (4 * lg + (lq >> 2)) * kRowBytes + (lq & 1) * 8;
  const int kswap = few_k_swap<D>(lq), vswap = few_v_swap<D>(4 * lg + (lq >> 2)), vpiece = (lq >> 1) & 1;

  for (int v0 = v_begin; v0 < v_end; v0 += kSegment) {
    const int v1 = min(v0 + kSegment, v_end), stages = (v1 - v0 + kFewKeys - 1) / kFewKeys;
#pragma unroll
    for (int u = 0; u < kSegment / 64; ++u) {
      const int v = v0 + u * 64 + lane;                     // past the end: the last row again, which nobody sees there
      if (u * 64 < v1 - v0) row_at[u * 64 + lane] = paged_row_bytes(p, sq, sp, min(v, v1 - 1));
    }
    __builtin_amdgcn_s_waitcnt(0);                           // rows' offsets and the queries; from here on only copies are counted
    int64_t from[kCopies];                                   // of the copies to be asked for next: read together, well before their use
    auto look_up = [&](int st) {
#pragma unroll
      for (int c = 0; c < kCopies; ++c) from[c] = row_at[st * kFewKeys + c * kRowsPerCopy + crow];
    };
    auto request = [&](int st) {
      const uint32_t at = ring0 + (uint32_t)(st % kFewStages) * kStage;
#pragma unroll
      for (int c = 0; c < kCopies; ++c) {
        const int row = c * kRowsPerCopy + crow;
        const char* src = kbase + from[c];
        dma16_nt(at + c * 1024, src + ((cpiece ^ few_k_swap<D>(row)) << 4));
        dma16_nt(at + kHalf + c * 1024, src + v_bytes + ((cpiece ^ few_v_swap<D>(row)) << 4));
      }
    };
    for (int st = 0; st < min(kFewStages, stages); ++st) {
      look_up(st);
      request(st);
    }
    for (int st = 0; st < stages; ++st) {
      if (st + kFewStages <= stages) wait_vmcnt<(kFewStages - 1) * 2 * kCopies>();
      else wait_vmcnt<0>();
      look_up(min(st + kFewStages, stages - 1));
      const uint32_t at = (uint32_t)(st % kFewStages) * kStage;
      const int kb = paged_real(sp, v0 + st * kFewKeys);
      v4f s[ROWT][2];
#pragma unroll
      for (int nt = 0; nt < ROWT; ++nt) s[nt][0] = s[nt][1] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < D / 32; ++ks)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const dec_u4 a = lds_16(koff + at + t * 16 * kRowBytes + (((ks * 4 + lg) ^ kswap) << 4));
#pragma unroll
          for (int nt = 0; nt < ROWT; ++nt) s[nt][t] = mfma16x16x32<DT>(a, q[nt][ks], s[nt][t]);
        }
      dec_u4 vt[D / 16];
#pragma unroll
      for (int mt = 0; mt < D / 16; ++mt) {
        const uint32_t va = voff + at + (((mt * 2 + vpiece) ^ vswap) << 4);
        const uint2 lo = lds_tr16(va), hi = lds_tr16(va + 16 * kRowBytes);
        vt[mt] = dec_u4{lo.x, lo.y, hi.x, hi.y};
      }
      const bool plain = kb + kFewKeys - 1 <= min(sq.pos0, sq.len - 1) &&
                         (p.window == 0 || kb > sq.pos0 + sq.n - 1 - p.window || kb + kFewKeys <= p.sinks);
      dec_u4 pb[ROWT];
#pragma unroll
      for (int nt = 0; nt < ROWT; ++nt) {
        float x[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) x[r] = s[nt][r >> 2][r & 3] * p.scale_log2;
        if (!plain) {
#pragma unroll
          for (int r = 0; r < 8; ++r)
            if (!paged_sees(p, sq.len, pos[nt], kb + (r >> 2) * 16 + 4 * lg + (r & 3))) x[r] = -INFINITY;
        }
        const float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
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
        for (int r = 0; r < 8; ++r) e[r] = __builtin_amdgcn_exp2f(x[r] - base);
        l[nt] += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
        pb[nt] = pack8<DT>(e);
      }
#pragma unroll
      for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
        for (int nt = 0; nt < ROWT; ++nt) o[nt][mt] = mfma16x16x32<DT>(vt[mt], pb[nt], o[nt][mt]);
      if (st + kFewStages < stages) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the stage has been read
        request(st + kFewStages);
      }
    }
  }

#pragma unroll
  for (int nt = 0; nt < ROWT; ++nt) {
    float sum = l[nt] + __shfl_xor(l[nt], 16, kWave);
    sum += __shfl_xor(sum, 32, kWave);
    const int r = nt * 16 + lq;
    if (r >= rows) continue;
    if (chunks == 1) {
      const float inv = sum > 0.f ? 1.0f / sum : 0.f;
      uint16_t* dst = p.out + out_at[nt] * D + lg * 4;
#pragma unroll
      for (int mt = 0; mt < D / 16; ++mt)
        *(uint2*)(dst + mt * 16) = make_uint2(pack2<DT>(o[nt][mt][0] * inv, o[nt][mt][1] * inv), pack2<DT>(o[nt][mt][2] * inv, o[nt][mt][3] * inv));
    } else {
      const int64_t slot = (((int64_t)b * p.hkv + kvh) * p.few.chunks + chunk) * p.few.rows + r;
      float* dst = p.few.part_o + slot * D + lg * 4;
#pragma unroll
      for (int mt = 0; mt < D / 16; ++mt) *(v4f*)(dst + mt * 16) = o[nt][mt];
      if (lg == 0) *(v2f*)(p.few.part_ml + slot * 2) = v2f{ref[nt], sum};
    }
  }
}
// ---------------------------------------------------------------------------------------------------------------- merge
// out = sum_c 2^(ref_c - max ref) O_c / sum_c 2^(ref_c - max ref) l_c, a row of WAVES wavefronts: the chunks' weights go through LDS,
// kMergeWeights of them at a time, then every kLanes lanes take the chunks in turn, 16 bytes of their row a lane.
constexpr int kMergeWeights = 1024;
template <int DT, int D, int WAVES>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedParams p) {
  constexpr int kLanes = D / 4, kSide = WAVES * kWave / kLanes, kTeams = 4 / WAVES, kThreads = WAVES * kWave;
  __shared__ float weight[kTeams][kMergeWeights / kTeams];
  __shared__ __attribute__((aligned(16))) float part[kTeams][WAVES][D + 4];
  __shared__ float tops[4];
  const int team = threadIdx.x / kThreads, tid = threadIdx.x % kThreads, wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
  const int64_t id = (int64_t)blockIdx.x * kTeams + team;    // (sequence, KV head, row)
  const int r = (int)(id % p.few_most), bk = (int)(id / p.few_most), kvh = bk % p.hkv, rows = p.few.rows;
  bool mine = bk / p.hkv < p.batch;
  const int64_t slot = (int64_t)bk * p.few.chunks * rows + r;
  const float* ml = p.few.part_ml + slot * 2;
  // the first chunks' references and sums, on their way before it is known how many chunks there are
  const v2f early = mine && tid < p.few.chunks ? *(const v2f*)(ml + (int64_t)tid * rows * 2) : v2f{-INFINITY, 0.f};
  const PagedSequence sq = paged_sequence(p, mine ? bk / p.hkv : 0);
  mine = mine && r < sq.n * p.group && sq.n * p.group <= rows;
  int chunks = 1;
  if (mine) chunks = paged_chunks(paged_span(p, sq.len, sq.pos0, sq.pos0 + sq.n - 1, kFewKeys), p.few.chunk_keys);
  mine = mine && chunks > 1;                                 // (one chunk: complete already)
  if (WAVES == 4 && !mine) return;                           // (the whole workgroup)
  const int d4 = (tid % kLanes) * 4, side = tid / kLanes;
  const float* po = p.few.part_o + slot * D + d4;
  float top = tid < chunks ? early[0] : -INFINITY;
  if (mine)
    for (int c = tid + kThreads; c < chunks; c += kThreads) top = fmaxf(top, ml[(int64_t)c * rows * 2]);
  top = wave_max(top);
  if constexpr (WAVES == 4) {
    if (lane == 0) tops[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  }
  const float base = top == -INFINITY ? 0.f : top;
  v4f num = {0.f, 0.f, 0.f, 0.f};
  float den = 0.f;
  constexpr int kAtOnce = kMergeWeights / kTeams;
  for (int c0 = 0; mine && c0 < chunks; c0 += kAtOnce) {     // (uniform in a team)
    const int some = min(kAtOnce, chunks - c0);
    for (int c = tid; c < some; c += kThreads) {
      const v2f m = c0 + c < kThreads ? early : *(const v2f*)(ml + (int64_t)(c0 + c) * rows * 2);
      const float w = __builtin_amdgcn_exp2f(m[0] - base);
      weight[team][c] = w;
      den = fmaf(w, m[1], den);
    }
    if constexpr (WAVES == 4) __syncthreads();
    else __builtin_amdgcn_wave_barrier();
#pragma unroll 8
    for (int c = side; c < some; c += kSide) {
      const v4f o = *(const v4f*)(po + (int64_t)(c0 + c) * rows * D);
      const float w = weight[team][c];
#pragma unroll
      for (int e = 0; e < 4; ++e) num[e] = fmaf(w, o[e], num[e]);
    }
    if constexpr (WAVES == 4) __syncthreads();
    else __builtin_amdgcn_wave_barrier();
  }
  den = wave_sum(den);
#pragma unroll
  for (int s = kLanes; s < kWave; s <<= 1)
#pragma unroll
    for (int e = 0; e < 4; ++e) num[e] += __shfl_xor(num[e], s, kWave);
  if constexpr (WAVES == 4) {
    if (lane < kLanes) *(v4f*)&part[0][wave][d4] = num;
    if (lane == 0) part[0][wave][D] = den;
    __syncthreads();
    if (wave != 0 || lane >= kLanes) return;
    for (int w = 1; w < WAVES; ++w) {
      num += *(const v4f*)&part[0][w][d4];
      den += part[0][w][D];
    }
  }
  if (!mine || lane >= kLanes) return;
  const float inv = den > 0.f ? 1.f / den : 0.f;
  *(uint2*)(p.out + ((int64_t)(sq.first + r / p.group) * p.hq + kvh * p.group + r % p.group) * D + d4) =
      make_uint2(pack2<DT>(num[0] * inv, num[1] * inv), pack2<DT>(num[2] * inv, num[3] * inv));
}

// Chunks of `blocks` key blocks each for `units` (tile, KV head) pairs.  In blocks (1.6 us): a compute unit takes one workgroup at a time, whose start and
// end cost about three; a launch for the merge two and 0.4 for every chunk that it adds up; a chunk's partial results, 128 KB out and back, a
// thirtieth.  Both launches at 1 / 2 / 3 / 4 / 5 / 8 / 16 chunks, 28 : 4 heads, us: 512 tokens behind 4096 rows (56 pairs, 72 blocks) 120 73 56 49 68 61 87,
// 33 behind 7967 (4, 125) 195 105 75 60 50 37 29, 2048 behind 6144 (224, 128) 218 240 241 243 243 291 407, four of 200 behind 2800, 32 : 8 heads (72, 47)
// 86 58 52 59 61 67 97, sixteen of up to 33 behind 4000 (64, 63) 109 70 56 60 63 69 84, of which this takes 63.
static int64_t paged_tile_chunks(int64_t blocks, int64_t units) {
  double best = 1e30;
  int64_t chunks = 1;
  for (int64_t c = 1; c <= std::min<int64_t>(blocks, 32); ++c) {
    const int64_t per = (blocks + c - 1) / c;
    if ((blocks + per - 1) / per != c) continue;
    const double cost = (double)((units * c + 255) / 256) * (double)(per + 3) + (c > 1 ? 2 + 0.4 * (double)c + (double)(units * c) / 30 : 0);
    if (cost < best) {
      best = cost;
      chunks = c;
    }
  }
  return chunks;
}

// No key behind this many rows is read (max_kv), so a window or sinks beyond it say no more than it does: the plan and the kernels both take the smaller
// number (the plan's sums with a window of 2^63 - 1 would wrap).
constexpr int64_t kMostRows = 1ll << 30;

// How a call is cut, from the bounds alone.  Keys of a row: at most max_kv, or a window's, its sinks and the row's fellow tokens'.
struct PagedPlan { int few_rows, few_keys, few_chunks, tile_keys, tile_chunks; int64_t tiles; size_t few_o, few_ml, tile_o, tile_ml, bytes; };
static PagedPlan paged_plan(int64_t batch, int64_t n_tokens, int64_t hq, int64_t hkv, int64_t head_dim, int64_t max_new, int64_t max_kv,
                            int64_t window, int64_t sinks) {
  PagedPlan pl{};
  const int64_t group = hq / hkv, most = max_new * group;
  auto span = [&](int64_t tokens, int64_t block) {
    return window ? std::min(max_kv, window + tokens + (sinks + block - 1) / block * block + block) : max_kv;
  };
  // one token's rows, or all of a short call's: 16, 32 or 64; none where the only sequence may bring more
  const int64_t few = most <= 64 ? most : batch > 1 ? group : 65;
  pl.few_rows = few <= 16 ? 16 : few <= 32 ? 32 : few <= 64 ? 64 : 0;
  if (pl.few_rows) {
    const int64_t keys = std::max<int64_t>(1, span(pl.few_rows / group, kFewKeys)), units = batch * hkv;
    // A unit's stages follow one another (16 copies and the products of 32 keys each), so short calls want short chunks; a partial result costs
    // the merge as much as 7 keys of 28 : 4 heads, so long ones want long ones.  Both launches, chunks of 64 / 128 / 256 / 384 / 512 keys, us:
    // one token of 1000 rows, 32 : 8 heads of 64: 8.2 8.6 10.3 12.1 14.1; of 32768, 28 : 4: 27.0 20.2 18.8 20.9 19.4; 32 tokens of up to 1000:
    // 19.3 15.9 15.2 17.4 18.0; 64 of up to 4096: 95 85 81 70 74; 16 of up to 32768, 32 : 8: 330 283 253 244 241
    int64_t per = ((int64_t)(0.65 * std::sqrt((double)units * (double)keys)) + kFewKeys - 1) / kFewKeys * kFewKeys;
    per = std::min<int64_t>(std::max<int64_t>(per, 64), 384);
    while (per < keys && units * ((keys + per - 1) / per) * pl.few_rows > (1 << 21)) per *= 2;         // a gigabyte of partial results at 128 a head
    pl.few_keys = (int)per;
    pl.few_chunks = (int)((keys + per - 1) / per);
    const size_t slots = (size_t)units * pl.few_chunks * pl.few_rows;
    if (pl.few_chunks > 1) {
      pl.few_o = align_up(slots * head_dim * sizeof(float), 256);
      pl.few_ml = align_up(slots * 2 * sizeof(float), 256);
    }
  }
  if (most > pl.few_rows) {
    pl.tiles = n_tokens * group / kTileRows + batch;
    const int64_t keys = std::max<int64_t>(1, span(std::min(max_new, kTileRows / group + 2), kTileKeys)), blocks = (keys + kTileKeys - 1) / kTileKeys;
    int64_t chunks = paged_tile_chunks(blocks, (n_tokens * group + kTileRows - 1) / kTileRows * hkv);      // (tiles of all tokens, none part empty)
    while (chunks > 1 && pl.tiles * hkv * chunks > (1 << 13)) --chunks;                  // a gigabyte of partial results at 128 a head
    const int64_t per = (blocks + chunks - 1) / chunks * kTileKeys;
    pl.tile_keys = (int)per;
    pl.tile_chunks = (int)((keys + per - 1) / per);
    const size_t slots = (size_t)pl.tiles * hkv * pl.tile_chunks * kTileRows;
    if (pl.tile_chunks > 1) {
      pl.tile_o = align_up(slots * head_dim * sizeof(float), 256);
      pl.tile_ml = align_up(slots * 2 * sizeof(float), 256);
    }
  }
  pl.bytes = 256 + pl.few_o + pl.few_ml + pl.tile_o + pl.tile_ml;
  return pl;
}

template <int DT, int D>
static void launch_few_of(const PagedParams& p, int tiles, unsigned units, hipStream_t st) {
  if (tiles == 1) hipLaunchKernelGGL((paged_few_kernel<DT, D, 1>), dim3(units), dim3(64), 0, st, p);
  else if (tiles == 2) hipLaunchKernelGGL((paged_few_kernel<DT, D, 2>), dim3(units), dim3(64), 0, st, p);
  else hipLaunchKernelGGL((paged_few_kernel<DT, D, 4>), dim3(units), dim3(64), 0, st, p);
}
static void launch_few(const PagedParams& p, int tiles, int dtype, unsigned units, hipStream_t st) {
  if (dtype == SUBSPEC_BF16) {
    if (p.head_dim == 128) launch_few_of<SUBSPEC_BF16, 128>(p, tiles, units, st);
    else launch_few_of<SUBSPEC_BF16, 64>(p, tiles, units, st);
  } else {
    if (p.head_dim == 128) launch_few_of<SUBSPEC_F16, 128>(p, tiles, units, st);
    else launch_few_of<SUBSPEC_F16, 64>(p, tiles, units, st);
  }
}
// A workgroup a row where there are many chunks to add up, a wavefront a row where there are few.
template <int DT, int D>
static void launch_few_merge_of(const PagedParams& p, int64_t rows, hipStream_t st) {
  if (p.few.chunks > 12) hipLaunchKernelGGL((paged_merge_kernel<DT, D, 4>), dim3((unsigned)rows), dim3(256), 0, st, p);
  else hipLaunchKernelGGL((paged_merge_kernel<DT, D, 1>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, p);
}
static void launch_few_merge(const PagedParams& p, int dtype, int64_t rows, hipStream_t st) {
  if (dtype == SUBSPEC_BF16) {
    if (p.head_dim == 128) launch_few_merge_of<SUBSPEC_BF16, 128>(p, rows, st);
    else launch_few_merge_of<SUBSPEC_BF16, 64>(p, rows, st);
  } else {
    if (p.head_dim == 128) launch_few_merge_of<SUBSPEC_F16, 128>(p, rows, st);
    else launch_few_merge_of<SUBSPEC_F16, 64>(p, rows, st);
  }
}

}  // namespace subspec

using namespace subspec;

extern "C" size_t subspec_paged_attention_workspace(int64_t batch, int64_t n_tokens, int64_t n_q_heads, int64_t n_kv_heads,
                                                    int64_t head_dim, int64_t max_new, int64_t max_kv, int64_t window,
                                                    int64_t sinks) {
  if (batch < 1 || batch > SUBSPEC_MAX_BATCH || n_kv_heads < 1 || n_q_heads < n_kv_heads || n_q_heads % n_kv_heads || n_q_heads > 1024 || max_kv < 0 ||
      max_kv > kMostRows || n_tokens < 1 || n_tokens > (1ll << 30) || max_new < 0 || window < 0 || sinks < 0 || head_dim < 1 || head_dim > 1024)
    return 256;
  return paged_plan(batch, n_tokens, n_q_heads, n_kv_heads, head_dim, std::min(max_new, n_tokens), max_kv, std::min(window, kMostRows),
                    std::min(sinks, kMostRows)).bytes;
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
  if (n_tokens < 0 || n_tokens > (1ll << 30) || max_new < 0 || max_kv < 0 || max_kv > kMostRows)
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
  max_new = std::min(max_new, n_tokens);
  if (max_new * (n_q_heads / n_kv_heads) > INT32_MAX - kTileRows)        // (the kernels number a sequence's rows of a KV head in 32 bits)
    SUBSPEC_FAIL(SUBSPEC_ERR_LIMIT, "%s: %lld tokens of %lld query heads a KV head in one sequence", what, (long long)max_new,
                 (long long)(n_q_heads / n_kv_heads));
  window = std::min(window, kMostRows);
  sinks = std::min(sinks, kMostRows);
  const PagedPlan pl = paged_plan(batch, n_tokens, n_q_heads, n_kv_heads, head_dim, max_new, max_kv, window, sinks);
  if (pl.bytes > 256 && (!workspace || workspace_bytes < pl.bytes))
    SUBSPEC_FAIL(SUBSPEC_ERR_WORKSPACE, "%s: workspace of %zu bytes is smaller than the %zu required", what, workspace_bytes, pl.bytes);
  if ((uintptr_t)workspace % 16) SUBSPEC_FAIL(SUBSPEC_ERR_ARG, "%s: workspace must be 16-byte aligned", what);
  PagedParams p;
  p.q = (const uint16_t*)q; p.pool = (const uint16_t*)kv_pool_layer; p.table = block_table; p.starts = query_starts; p.lens = kv_lens;
  p.out = (uint16_t*)out;
  p.q_token = q_token_stride; p.q_head = q_head_stride; p.table_stride = table_stride;
  p.page_elems = page_len * n_kv_heads * head_dim;
  p.batch = (int)batch; p.n_tokens = (int)n_tokens; p.hq = (int)n_q_heads; p.hkv = (int)n_kv_heads; p.group = (int)(n_q_heads / n_kv_heads);
  p.head_dim = (int)head_dim; p.max_new = (int)max_new; p.max_kv = (int)std::min(max_kv, max_blocks * page_len);
  p.window = (int)window; p.sinks = (int)sinks;
  p.page_shift = 0;
  while ((1ll << p.page_shift) < page_len) ++p.page_shift;
  p.max_pages = (int)max_pages;
  p.scale_log2 = scale * kLog2e;
  char* ws = (char*)workspace;
  p.few = PagedCut{pl.few_rows, pl.few_keys, pl.few_chunks, (float*)ws, (float*)(ws + pl.few_o)};
  ws += pl.few_o + pl.few_ml;
  p.tile = PagedCut{kTileRows, pl.tile_keys, pl.tile_chunks, (float*)ws, (float*)(ws + pl.tile_o)};
  p.tiles = (int)pl.tiles;
  p.few_most = (int)std::max<int64_t>(1, std::min<int64_t>(pl.few_rows, max_new * p.group));
  hipStream_t st = (hipStream_t)stream;
  const int64_t merge_rows = batch * n_kv_heads * p.few_most;
  const int64_t few_units = batch * n_kv_heads * pl.few_chunks, tile_units = pl.tiles * n_kv_heads * pl.tile_chunks;
  if (few_units > INT32_MAX || tile_units * 8 > INT32_MAX || merge_rows > INT32_MAX)
    SUBSPEC_FAIL(SUBSPEC_ERR_LIMIT, "%s: too large (%lld tokens of %lld heads, %lld sequences)", what, (long long)n_tokens, (long long)n_q_heads,
                 (long long)batch);
  if (pl.tiles) {
    {
      DominantKernelTimer timer(st);
      launch_paged_tile(p, dtype, st);
    }
    if (pl.tile_chunks > 1) launch_paged_tile_merge(p, dtype, st);
  }
  if (pl.few_rows) {
    if (pl.tiles) {
      launch_few(p, pl.few_rows / 16, dtype, (unsigned)few_units, st);
    } else {
      DominantKernelTimer timer(st);
      launch_few(p, pl.few_rows / 16, dtype, (unsigned)few_units, st);
    }
    if (pl.few_chunks > 1) launch_few_merge(p, dtype, merge_rows, st);
  }
  SUBSPEC_CHECK_HIP(hipGetLastError());
  return SUBSPEC_OK;
}
