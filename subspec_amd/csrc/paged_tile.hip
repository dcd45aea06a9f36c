// Attention over a page pool, chunks of prompts: 256 packed rows (token, query head of one KV head) and a chunk of the keys a workgroup.
//
// The matrix work is that of a prompt: S^T = K Q^T and O^T = V^T P^T by 32x32x16 products, a wavefront 32 rows, a block 64 keys; S^T's accumulators
// (sixteen keys of one row a lane) are, packed, the operand of O^T, so probabilities never leave registers.  Left to themselves the
// eight wavefronts run in step, all in the products and then all in the softmax, with the matrix pipe idle meanwhile.  So a block is two
// phases between barriers, M (O^T of the block before, S^T of this one) and V (softmax), and the second wavefront of every SIMD enters the
// loop one barrier later: one of the two is in M while the other is in V.
// K and V rows are copied from memory straight into a ring of four LDS stages, asked for two blocks ahead, a quarter of the copies at a time
// between the products.  The copies are inline assembly, waited for by count: the compiler would wait for all of them before any LDS read.
// A row's address comes from its page number: the chunk's part of the page table is in LDS before the loop.  Where a wavefront's eight rows of a
// block lie in one page (pages of 8 rows and more) that is one number for all lanes.
// Packing (token, head) rows lets a key block serve the whole group: 28 : 4 heads, 256 rows are 37 tokens of 7 heads, and one copy of a block is
// read where a workgroup for each head would read seven.
// 2048 tokens behind 6144 rows, 28 : 4 heads of 128: 217 to 224 us, 0.97 to 0.94 PFLOP/s; 8192 tokens, 16 : 8 heads: 257, 1.07; 2048 behind 6144, 32 : 8
// heads of 64: 156, 0.77.  The matrix pipes of a compute unit are busy for 0.54 of its cycles (a block takes 3800, its products' own are 2048); with
// heads of 64 and a window 0.24.  The products of a phase stand at 47 cycles each instead of 32 even without an LDS read between them.
// Operands asked for earlier, other priorities and copies in the softmax phase changed nothing.
#include "paged.h"

namespace subspec {

typedef float v16f __attribute__((ext_vector_type(16)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));

template <int DT>
__device__ __forceinline__ v16f mfma32x32x16(dec_u4 a, dec_u4 b, v16f c) {
  if constexpr (DT == SUBSPEC_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

constexpr int kStages = 4;
template <int D> struct TileShape {
  static constexpr int kRowBytes = D * 2, kPieces = kRowBytes / 16, kRowsPerCopy = 64 / kPieces;
  static constexpr int kCopies = 8 / kRowsPerCopy;                     // copies of a wavefront's eight K rows (as many for V)
  static constexpr int kHalf = kTileKeys * kRowBytes;                  // K of a stage; the V ring follows the K ring
  static constexpr int kVRing = kStages * kHalf, kPages = 2 * kVRing, kLds = kPages + kTilePages * 4;
  static constexpr int kKSteps = D / 16, kDTiles = D / 32;
  // Stored place of a row's 16-byte pieces.  K: one piece of 16 consecutive rows at a time; V: 64 bytes of 4 consecutive rows.
  static __device__ __forceinline__ int k_swap(int row) { return D == 128 ? row & 15 : (row >> 1) & 7; }
  static __device__ __forceinline__ int v_swap(int row) { return D == 128 ? 4 * (row & 3) : 4 * ((row >> 1) & 1); }
};

// The copies of a wavefront's eight rows of one block.  In one page: a scalar address and the lane's offset in the rows.  (The address comes out of
// scalar instructions and has its five wait states behind them.)
struct TileCopy {
  const char* k;                                                       // the first row's K
  const char* v;
  uint32_t at;                                                         // place in the stage; V's is kVRing behind
  int block;                                                           // of the chunk
  bool one_page;
};
__device__ __forceinline__ void dma16_row(uint32_t lds_base, uint32_t offset, const char* base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds_base), "v"(offset), "s"(base) : "memory", "m0");
}
template <int D>
__device__ __forceinline__ void wait_block() { wait_vmcnt<2 * TileShape<D>::kCopies>(); }     // all but the newest block's copies

// M phase.  MODE 2: even steps are O^T of the previous block, odd ones S^T of this one, so that no accumulator comes up twice in a row; MODE 0: S^T
// alone (first block), MODE 1: O^T alone (after the last).  Operands are asked for kAhead steps before their use; scheduling fences
// keep that distance.
struct TileAddress { uint32_t vst, kst, vx, kx; };
template <int MODE> __device__ __forceinline__ constexpr bool step_is_pv(int k) { return MODE == 1 || (MODE == 2 && (k & 1) == 0); }
template <int MODE> __device__ __forceinline__ constexpr int step_index(int k) { return MODE == 2 ? k >> 1 : k; }
template <int D, int MODE>
__device__ __forceinline__ dec_u4 load_step(int k, const uint32_t (&kaddr)[D / 16], const uint32_t (&vaddr)[D / 32]) {
  using S = TileShape<D>;
  const int j = step_index<MODE>(k);
  if (step_is_pv<MODE>(k)) {
    const int ts = j / S::kDTiles, dt = j % S::kDTiles;                // keys 16 ts .. of the block
    const uint32_t va = vaddr[dt] + (uint32_t)(ts * 16 * S::kRowBytes);
    const uint2 lo = lds_tr16(va), hi = lds_tr16(va + 8 * S::kRowBytes);
    return dec_u4{lo.x, lo.y, hi.x, hi.y};
  }
  return lds_16(kaddr[j >> 1] + (uint32_t)((j & 1) * 32 * S::kRowBytes));
}
// between(k) is what else the phase does behind step k.
template <int DT, int D, int MODE, typename Between>
__device__ __forceinline__ void matrix_phase(const TileAddress& ad, v16f (&o)[D / 32], v16f (&s)[2], const v16f& cinit, const dec_u4 (&pb)[4],
                                             const dec_u4 (&q)[D / 16], Between between) {
  using S = TileShape<D>;
  constexpr int kOne = 2 * S::kKSteps, kSteps = MODE == 2 ? 2 * kOne : kOne, kAhead = 4;
  __builtin_amdgcn_s_setprio(1);                                       // the wavefront that multiplies goes first
  uint32_t kaddr[S::kKSteps], vaddr[S::kDTiles];
  if (MODE != 1) {
#pragma unroll
    for (int ks = 0; ks < S::kKSteps; ++ks) kaddr[ks] = ad.kst + (ad.kx ^ (uint32_t)(ks << 5));
  }
  if (MODE != 0) {
#pragma unroll
    for (int dt = 0; dt < S::kDTiles; ++dt) vaddr[dt] = ad.vst + (ad.vx ^ (uint32_t)(dt << 6));
  }
  dec_u4 ring[kAhead];
#pragma unroll
  for (int k = 0; k < kAhead; ++k) ring[k] = load_step<D, MODE>(k, kaddr, vaddr);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    const dec_u4 a = ring[k % kAhead];
    const int j = step_index<MODE>(k);
    if (step_is_pv<MODE>(k)) {
      const int ts = j / S::kDTiles, dt = j % S::kDTiles;
      o[dt] = mfma32x32x16<DT>(a, pb[ts], o[dt]);
    } else {
      s[j & 1] = mfma32x32x16<DT>(a, q[j >> 1], (j >> 1) == 0 ? cinit : s[j & 1]);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (k + kAhead < kSteps) ring[k % kAhead] = load_step<D, MODE>(k + kAhead, kaddr, vaddr);
    between(k, kSteps);
    __builtin_amdgcn_sched_barrier(0);
  }
  __builtin_amdgcn_s_setprio(0);
}

// V phase.  A probability is rounded once, to the type of the product with V, and the row's sum is that of the rounded ones in fp32: one instruction
// adds a pair of them, and what V is multiplied by adds up to what the result is divided by.  The accumulators hold raw scores relative to the row's
// reference, which follows the largest score by at most kSlack (in units of exp2's argument) and moves rarely once the first blocks are through.
template <int DT>
__device__ __forceinline__ float pair_sum(uint32_t packed, float acc) {
  if constexpr (DT == SUBSPEC_BF16) return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2bf, packed), __builtin_bit_cast(v2bf, 0x3f803f80u), acc, false);
  else return __builtin_amdgcn_fdot2(__builtin_bit_cast(v2h, packed), __builtin_bit_cast(v2h, 0x3c003c00u), acc, false);
}
__device__ __forceinline__ float max_halves(float x) {                 // of lanes i and i ^ 32, in both
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
struct TileRow { int pos; float ref, l; bool have; };
// keys kb .. kb + 63 that a row at `pos` sees of `len`, as bits (paged_sees)
__device__ __forceinline__ uint64_t seen_bits(const PagedParams& p, int len, int pos, int kb) {
  const int left = min(pos, len - 1) - kb;
  uint64_t bits = left < 0 ? 0ull : left >= 63 ? ~0ull : (2ull << left) - 1ull;
  if (p.window) {
    const int low = pos - p.window + 1 - kb, first = p.sinks - kb;
    const uint64_t recent = low <= 0 ? ~0ull : low > 63 ? 0ull : ~0ull << low;
    const uint64_t sink = first <= 0 ? 0ull : first > 63 ? ~0ull : (1ull << first) - 1ull;
    bits &= recent | sink;
  }
  return bits;
}
template <int DT, int D>
__device__ __forceinline__ void softmax_phase(const PagedParams& p, int len, int kb, bool plain, int g, TileRow& row, v16f (&s)[2], v16f (&o)[D / 32],
                                              v16f& cinit, dec_u4 (&pb)[4]) {
  if (!plain) {
    const uint64_t bits = seen_bits(p, len, row.pos, kb);
    const uint32_t half[2] = {(uint32_t)bits >> (4 * g), (uint32_t)(bits >> 32) >> (4 * g)};
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const uint32_t keep = (uint32_t)__builtin_amdgcn_sbfe((int)half[t], (r >> 2) * 8 + (r & 3), 1);
        s[t][r] = __uint_as_float((__float_as_uint(s[t][r]) & keep) | (0xff800000u & ~keep));
      }
  }
  float m[2] = {-INFINITY, -INFINITY};
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int r = 0; r < 16; r += 2) m[t] = fmaxf(fmaxf(s[t][r], s[t][r + 1]), m[t]);
  const float top = max_halves(fmaxf(m[0], m[1]));                     // raw units, relative to the reference
  const bool move = top > -INFINITY && (!row.have || top * p.scale_log2 > kSlack);
  if (__any(move)) {
    const float d = move ? top : 0.f;
    const float alpha = __builtin_amdgcn_exp2f(fminf(-d * p.scale_log2, 0.f));     // (down only the first time: nothing to rescale)
    row.ref += d;
    row.l *= alpha;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) o[dt] *= alpha;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[t][r] -= d;
#pragma unroll
    for (int r = 0; r < 16; ++r) cinit[r] = -row.ref;
  }
  row.have = row.have || top > -INFINITY;
  float sum[4];
#pragma unroll
  for (int ts = 0; ts < 4; ++ts) {
    float e[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) e[k] = __builtin_amdgcn_exp2f(s[ts >> 1][8 * (ts & 1) + k] * p.scale_log2);
    pb[ts] = pack8<DT>(e);
    sum[ts] = pair_sum<DT>(pb[ts][3], pair_sum<DT>(pb[ts][2], pair_sum<DT>(pb[ts][1], pair_sum<DT>(pb[ts][0], 0.f))));
  }
  row.l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

// Where tile u lies, and whether it has rows.  A tile before the first sequence's (tokens before starts[0]: nobody's), like one behind the last of its
// sequence, has none.
struct TilePlace { PagedSequence sq; int tile, rows, row0, row1, pos_lo, pos_hi; };
__device__ __forceinline__ bool tile_place(const PagedParams& p, int u, TilePlace* t) {
  t->sq = paged_sequence(p, __builtin_amdgcn_readfirstlane(paged_tile_owner(p, u)));
  t->tile = u - paged_first_tile(p, t->sq.b);
  t->rows = t->sq.n * p.group;
  t->row0 = t->tile * kTileRows;
  if (t->sq.n <= 0 || t->rows <= p.few.rows || t->tile < 0 || t->row0 >= t->rows) return false;
  t->row1 = min(t->rows, t->row0 + kTileRows);
  t->pos_lo = t->sq.pos0 + t->row0 / p.group;
  t->pos_hi = t->sq.pos0 + (t->row1 - 1) / p.group;
  return true;
}

template <int DT, int D>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) void paged_tile_kernel(PagedParams p) {
  using S = TileShape<D>;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[S::kLds];
  // KV heads fastest: workgroups are dealt to the XCDs in turn, so that those of a KV head meet in the same L2s.  The longest first: whole chunks
  // before what is left over behind them, the last tiles, whose rows see the most keys, before the first.
  const int kvh = (int)(blockIdx.x % (uint32_t)p.hkv);
  const uint32_t rest = blockIdx.x / (uint32_t)p.hkv;
  const int chunk = (int)(rest / (uint32_t)p.tiles), u = p.tiles - 1 - (int)(rest % (uint32_t)p.tiles);
  TilePlace tp;
  if (!tile_place(p, u, &tp)) return;
  const PagedSpan sp = paged_span(p, tp.sq.len, tp.pos_lo, tp.pos_hi, kTileKeys);
  const int chunks = paged_chunks(sp, p.tile.chunk_keys);
  if (chunk >= chunks) return;
  const int v_begin = chunk * p.tile.chunk_keys, v_end = min(v_begin + p.tile.chunk_keys, sp.length);

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 31, g = lane >> 5;
  const int wrow = tp.row0 + wave * 32, r = wrow + lr;                 // packed rows of the sequence
  const bool live = wrow < tp.rows, row_ok = r < tp.rows;
  const bool second = wave >= 4;                                       // the second wavefront of its SIMD
  const int pos0 = tp.sq.pos0, len = tp.sq.len;
  const int token = tp.sq.first + (row_ok ? r / p.group : 0), head = kvh * p.group + (row_ok ? r % p.group : 0);
  const int wave_lo = pos0 + wrow / p.group, wave_hi = pos0 + (min(tp.rows, wrow + 32) - 1) / p.group;

  dec_u4 q[D / 16];
  {
    const uint16_t* src = p.q + token * p.q_token + head * p.q_head + g * 8;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) q[ks] = row_ok ? *(const dec_u4*)(src + ks * 16) : dec_u4{0, 0, 0, 0};
  }
  v16f o[D / 32], s[2], cinit;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) o[dt][i] = 0.f;
    s[0][i] = s[1][i] = cinit[i] = 0.f;
  }
  dec_u4 pb[4] = {};
  TileRow row{row_ok ? max(pos0 + r / p.group, -1) : -1, 0.f, 0.f, false};

  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
  const int crow = lane / S::kPieces, cpiece = lane % S::kPieces;
  const int64_t tok_bytes = (int64_t)p.hkv * S::kRowBytes, page_bytes = p.page_elems * 2;
  const char* kbase = (const char*)(p.pool + kvh * D);
  const int tok_mask = (1 << p.page_shift) - 1;
  // lane offsets of the wavefront's copies from its first row's
  uint32_t kfrom[S::kCopies], vfrom[S::kCopies];
#pragma unroll
  for (int c = 0; c < S::kCopies; ++c) {
    const int in = c * S::kRowsPerCopy + crow;
    kfrom[c] = (uint32_t)(in * (int)tok_bytes) + (uint32_t)((cpiece ^ S::k_swap(wave * 8 + in)) << 4);
    vfrom[c] = (uint32_t)(in * (int)tok_bytes) + (uint32_t)((cpiece ^ S::v_swap(wave * 8 + in)) << 4);
  }
  TileCopy cp;
  int asked = 0;
  // A stretch of the chunk: as many keys as there is room for page numbers (all of them but where pages hold a row or two).  pages[]: those of the
  // keys before the gap between sinks and window, then those behind it.
  int* pages = (int*)(lds + S::kPages);
  const int64_t stretch = (int64_t)(kTilePages - 64) << p.page_shift;
  int v0 = v_begin, nb = 0, base1 = 0, count1 = 0, base2 = 0;
  auto load_pages = [&](int nkeys) {
    const int split = min(max(sp.skip - v0, 0), nkeys);                // keys before the gap
    const int real2 = paged_real(sp, v0 + split);
    nb = (nkeys + kTileKeys - 1) / kTileKeys;
    base1 = v0 >> p.page_shift;
    count1 = split > 0 ? ((v0 + split - 1) >> p.page_shift) - base1 + 1 : 0;
    base2 = real2 >> p.page_shift;
    const int count2 = split < nkeys ? ((real2 + nkeys - split - 1) >> p.page_shift) - base2 + 1 : 0;
    const int32_t* table = p.table + tp.sq.b * p.table_stride;
    for (int e = tid; e < count1 + count2; e += 512) pages[e] = min(max(table[e < count1 ? base1 + e : base2 + e - count1], 0), p.max_pages - 1);
  };
  // The next copies are those of block J -> stage J % 4; blocks past the last repeat it (every wavefront's count of copies is the same on every
  // path).  ask() reads the page number that plan() uses a few products later.
  auto place = [&](int J, int* v, int* j, int* shift) {
    *v = v0 + min(J, nb - 1) * kTileKeys + wave * 8;                   // the wavefront's eight keys
    *j = paged_real(sp, *v);
    *shift = *v < sp.skip ? -base1 : count1 - base2;                   // page number of key j: pages[(j >> page_shift) + shift]
  };
  auto ask = [&](int J) {
    int v, j, shift;
    place(J, &v, &j, &shift);
    asked = pages[(j >> p.page_shift) + shift];
  };
  auto plan = [&](int J) {
    int v, j, shift;
    place(J, &v, &j, &shift);
    cp.block = J;
    cp.at = lds0 + (uint32_t)(J & (kStages - 1)) * S::kHalf + (uint32_t)(wave * 8 * S::kRowBytes);
    cp.one_page = p.page_shift >= 3 && j + 7 < sp.high && (j >= sp.low || j + 7 < p.sinks);
    cp.k = kbase + (int64_t)__builtin_amdgcn_readfirstlane(asked) * 2 * page_bytes + (j & tok_mask) * tok_bytes;
    cp.v = cp.k + page_bytes;
  };
  auto copy_one = [&](int c) {                                         // c: K's, then V's
    if (c < S::kCopies) dma16_row(cp.at + c * 1024, kfrom[c < S::kCopies ? c : 0], cp.k);
    else dma16_row(cp.at + S::kVRing + (c - S::kCopies) * 1024, vfrom[c < S::kCopies ? 0 : c - S::kCopies], cp.v);
  };
  // small pages, the end of the keys, the gap: row by row.  A key that no row sees stands for one that some row does, what it holds must not reach
  // a product, not even multiplied by zero.
  auto copy_rows = [&]() {
    int v, j, shift;
    place(cp.block, &v, &j, &shift);
    int self = lane;
    asm volatile("" : "+v"(self));                                     // (what follows from the lane is worked out here, not kept for the whole loop)
    const int crow = self / S::kPieces, cpiece = self % S::kPieces;
#pragma unroll
    for (int c = 0; c < S::kCopies; ++c) {
      const int in = c * S::kRowsPerCopy + crow;
      int key = j + in;
      if (v < sp.skip) key = min(key, p.sinks - 1);
      else key = min(key >= p.sinks ? max(key, sp.low) : key, sp.high - 1);
      const char* at = kbase + (int64_t)pages[(key >> p.page_shift) + shift] * 2 * page_bytes + (key & tok_mask) * tok_bytes;
      dma16_from(cp.at + c * 1024, at + ((cpiece ^ S::k_swap(wave * 8 + in)) << 4));
      dma16_from(cp.at + S::kVRing + c * 1024, at + page_bytes + ((cpiece ^ S::v_swap(wave * 8 + in)) << 4));
    }
  };
  auto copy_all = [&]() {
    if (cp.one_page) {
#pragma unroll
      for (int c = 0; c < 2 * S::kCopies; ++c) copy_one(c);
    } else {
      copy_rows();
    }
  };
  // behind step k of an M phase: a copy every so many steps, then what the next ones need
  auto between = [&](int J, int k, int steps) {
    const int each = steps / (2 * S::kCopies);
    if (k % each == 1 && cp.one_page) copy_one(k / each);
    if (k == 2) ask(J);
    if (k == steps - each + 2) {
      if (!cp.one_page) copy_rows();
      plan(J);
    }
  };
  // operand addresses inside a stage.  K: key 32 t + lr, piece 2 ks + g.  V^T: of 16 lanes, lane i supplies the 8 bytes of key 4 g + i / 4 at
  // d = 32 dt + 16 h + 4 (i % 4)
  const int r16 = lane & 15, hh = (lane >> 4) & 1;
  const uint32_t klane = lds0 + lr * S::kRowBytes;
  const uint32_t vlane = lds0 + S::kVRing + (4 * g + (r16 >> 2)) * S::kRowBytes + (2 * hh + ((r16 & 3) >> 1)) * 16 + (r16 & 1) * 8;
  TileAddress ad;
  ad.kx = (uint32_t)((g ^ S::k_swap(lr)) << 4);
  ad.vx = (uint32_t)(S::v_swap(r16 >> 2) << 4);
  auto stages = [&](int i) {
    ad.vst = vlane + (uint32_t)((i - 1) & (kStages - 1)) * S::kHalf;
    ad.kst = klane + (uint32_t)(i & (kStages - 1)) * S::kHalf;
  };
  auto softmax = [&](int i) {
    const int kb = paged_real(sp, v0 + i * kTileKeys);
    const bool plain = kb + kTileKeys - 1 <= min(wave_lo, len - 1) && (p.window == 0 || kb > wave_hi - p.window || kb + kTileKeys <= p.sinks);
    softmax_phase<DT, D>(p, len, kb, plain, g, row, s, o, cinit, pb);
  };

  for (; v0 < v_end; v0 = (int)min((int64_t)v_end, v0 + stretch)) {
    load_pages((int)min((int64_t)(v_end - v0), stretch));
    __builtin_amdgcn_s_waitcnt(0);                                     // page numbers (and queries); from here on only copies are counted
    __syncthreads();
    ask(0);
    plan(0);
    copy_all();
    ask(1);
    plan(1);
    copy_all();
    ask(2);
    plan(2);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (second) __syncthreads();
    if (live) {
      stages(0);
      matrix_phase<DT, D, 0>(ad, o, s, cinit, pb, q, [&](int k, int steps) { between(3, k, steps); });
    } else {
      copy_all();
      ask(3);
      plan(3);
    }
    if (second) wait_block<D>();
    __syncthreads();
    if (live) softmax(0);
    if (!second) wait_block<D>();
    __syncthreads();
    for (int i = 1; i < nb; ++i) {
      if (live) {
        stages(i);
        matrix_phase<DT, D, 2>(ad, o, s, cinit, pb, q, [&](int k, int steps) { between(i + 3, k, steps); });
      } else {
        copy_all();
        ask(i + 3);
        plan(i + 3);
      }
      if (second) wait_block<D>();
      __syncthreads();
      if (live) softmax(i);
      if (!second) wait_block<D>();
      __syncthreads();
    }
    if (live) {
      stages(nb);
      matrix_phase<DT, D, 1>(ad, o, s, cinit, pb, q, [](int, int) {});
    }
    __syncthreads();
    if (!second) __syncthreads();
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                   // no copy may be on its way into LDS when the workgroup ends, or begins anew
    __syncthreads();
  }

  const float l = row.l + __shfl_xor(row.l, 32, kWave);
  if (!live) return;
  if (chunks == 1) {
    if (!row_ok) return;
    const float inv = l > 0.f ? 1.0f / l : 0.f;
    uint16_t* dst = p.out + ((int64_t)token * p.hq + head) * D + g * 4;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4)
        *(uint2*)(dst + dt * 32 + q4 * 8) = make_uint2(pack2<DT>(o[dt][4 * q4] * inv, o[dt][4 * q4 + 1] * inv),
                                                       pack2<DT>(o[dt][4 * q4 + 2] * inv, o[dt][4 * q4 + 3] * inv));
  } else {
    // [unit][chunk][wavefront][16 bytes of a lane, D / 8 of them]: every store writes a kilobyte
    const int64_t slot = (((int64_t)u * p.hkv + kvh) * p.tile.chunks + chunk) * 8 + wave;
    float* dst = p.tile.part_o + slot * (32 * D) + lane * 4;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4)
        *(v4f*)(dst + (dt * 4 + q4) * 256) = v4f{o[dt][4 * q4], o[dt][4 * q4 + 1], o[dt][4 * q4 + 2], o[dt][4 * q4 + 3]};
    if (g == 0) *(v2f*)(p.tile.part_ml + (slot * 32 + lr) * 2) = v2f{row.have ? row.ref * p.scale_log2 : -INFINITY, l};
  }
}

// out = sum_c 2^(ref_c - max ref) O_c / sum_c 2^(ref_c - max ref) l_c: a workgroup per (tile, KV head, wavefront of it) and 32 dimensions, a
// thread four of a row's; the loads of four chunks are on their way together.
template <int DT, int D>
__global__ __launch_bounds__(256) void paged_tile_merge_kernel(PagedParams p) {
  const int wave = (int)(blockIdx.x % 8u), kvh = (int)(blockIdx.x / 8u % (uint32_t)p.hkv), u = (int)(blockIdx.x / 8u / (uint32_t)p.hkv);
  TilePlace tp;
  if (!tile_place(p, u, &tp)) return;
  const int lane = threadIdx.x & 63, lr = lane & 31, g = lane >> 5, piece = blockIdx.y * 4 + threadIdx.x / 64;
  const int r = tp.row0 + wave * 32 + lr;
  if (tp.row0 + wave * 32 >= tp.rows) return;
  const PagedSpan sp = paged_span(p, tp.sq.len, tp.pos_lo, tp.pos_hi, kTileKeys);
  const int chunks = paged_chunks(sp, p.tile.chunk_keys);
  if (chunks == 1 || r >= tp.rows) return;
  const int64_t slot = (((int64_t)u * p.hkv + kvh) * p.tile.chunks) * 8 + wave;
  const float* ml = p.tile.part_ml + (slot * 32 + lr) * 2;
  const float* po = p.tile.part_o + slot * (32 * D) + piece * 256 + lane * 4;
  float top = -INFINITY, den = 0.f;
  v4f num = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int c = 0; c < chunks; ++c) top = fmaxf(top, ml[(int64_t)c * 8 * 64]);
  const float base = top == -INFINITY ? 0.f : top;
#pragma unroll 4
  for (int c = 0; c < chunks; ++c) {
    const v2f m = *(const v2f*)(ml + (int64_t)c * 8 * 64);
    const v4f o = *(const v4f*)(po + (int64_t)c * 8 * 32 * D);
    const float w = __builtin_amdgcn_exp2f(m[0] - base);
#pragma unroll
    for (int e = 0; e < 4; ++e) num[e] = fmaf(w, o[e], num[e]);
    den = fmaf(w, m[1], den);
  }
  const float inv = den > 0.f ? 1.f / den : 0.f;
  const int token = tp.sq.first + r / p.group, head = kvh * p.group + r % p.group;
  uint16_t* dst = p.out + ((int64_t)token * p.hq + head) * D + piece / 4 * 32 + piece % 4 * 8 + g * 4;
  *(uint2*)dst = make_uint2(pack2<DT>(num[0] * inv, num[1] * inv), pack2<DT>(num[2] * inv, num[3] * inv));
}

void launch_paged_tile(const PagedParams& p, int dtype, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)p.tiles * p.tile.chunks * p.hkv));
#define SUBSPEC_PAGED_TILE(DT, D) hipLaunchKernelGGL((paged_tile_kernel<DT, D>), grid, dim3(512), 0, st, p)
  if (dtype == SUBSPEC_BF16) { if (p.head_dim == 128) SUBSPEC_PAGED_TILE(SUBSPEC_BF16, 128); else SUBSPEC_PAGED_TILE(SUBSPEC_BF16, 64); }
  else { if (p.head_dim == 128) SUBSPEC_PAGED_TILE(SUBSPEC_F16, 128); else SUBSPEC_PAGED_TILE(SUBSPEC_F16, 64); }
#undef SUBSPEC_PAGED_TILE
}
void launch_paged_tile_merge(const PagedParams& p, int dtype, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)p.tiles * p.hkv * 8), (unsigned)(p.head_dim / 32));
#define SUBSPEC_PAGED_TILE(DT, D) hipLaunchKernelGGL((paged_tile_merge_kernel<DT, D>), grid, dim3(256), 0, st, p)
  if (dtype == SUBSPEC_BF16) { if (p.head_dim == 128) SUBSPEC_PAGED_TILE(SUBSPEC_BF16, 128); else SUBSPEC_PAGED_TILE(SUBSPEC_BF16, 64); }
  else { if (p.head_dim == 128) SUBSPEC_PAGED_TILE(SUBSPEC_F16, 128); else SUBSPEC_PAGED_TILE(SUBSPEC_F16, 64); }
#undef SUBSPEC_PAGED_TILE
}

}  // namespace subspec
