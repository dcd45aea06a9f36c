// What the kernels of attention over a page pool share: the batch's description, the keys a tile of rows sees, products and LDS reads.
#pragma once
#include "common.h"
#include "dma.h"

namespace subspec {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));

// How one of the kernels cuts its sequences: `rows` packed rows a tile, the keys in chunks; partial results [unit][chunk][rows][D], fp32,
// with (reference, sum) of each row.
struct PagedCut {
  int rows, chunk_keys, chunks;
  float* part_o;
  float* part_ml;
};
struct PagedParams {
  const uint16_t* q;
  const uint16_t* pool;
  const int32_t* table;
  const int32_t* starts;
  const int32_t* lens;
  uint16_t* out;
  int64_t q_token, q_head;                 // strides, elements
  int64_t table_stride, page_elems;        // page_elems: a page's K (V follows it)
  int batch, n_tokens, hq, hkv, group, head_dim, max_new, max_kv, window, sinks, page_shift, max_pages;
  float scale_log2;
  PagedCut few;                            // sequences of at most few.rows rows a KV head (0 rows: none)
  int few_most;                            // rows a KV head that one of them can have
  PagedCut tile;                           // the others
  int tiles;                               // tiles of a KV head that the launch has room for
};

// A sequence's tokens that the call computes, `n` from `first` on, the position of the first of them, and the keys that there are.  The bounds max_new
// and max_kv leave tokens and keys out; they move no position, so pos0 comes from the lengths as they are.  (No token of a sequence can be more
// than 2^30 behind its first: below -2^30 a position is as good as there.)
struct PagedSequence { int b, first, n, pos0, len; };
__device__ __forceinline__ PagedSequence paged_sequence(const PagedParams& p, int b) {
  PagedSequence s;
  s.b = b;
  const int end = p.starts[b + 1], rows = max(p.lens[b], 0);
  s.first = min(max(p.starts[b], 0), p.n_tokens);
  s.n = min(min(end, p.n_tokens) - s.first, p.max_new);
  s.pos0 = (int)max((int64_t)rows - ((int64_t)end - s.first), -(1ll << 30));
  s.len = min(rows, p.max_kv);                     // (max_kv is within the table: the host saw to it)
  return s;
}
// keys a row at position pos (-1: none) sees: j <= pos, and with a window w only j > pos - w or j < sinks
__device__ __forceinline__ bool paged_sees(const PagedParams& p, int len, int pos, int j) {
  return j <= min(pos, len - 1) && (p.window == 0 || j > pos - p.window || j < p.sinks);
}

// The keys that rows at positions pos_lo .. pos_hi see between them: [0, sinks) and [low, high), as one range of `length` virtual keys in
// blocks of `block`: the first `skip` of them are keys 0 .., the others keys `start` .. (start and skip are multiples of the block).  Where all windows
// begin behind the last key there are the sinks alone, keys [0, high).
struct PagedSpan { int skip, start, low, high, length; };
__device__ __forceinline__ PagedSpan paged_span(const PagedParams& p, int len, int pos_lo, int pos_hi, int block) {
  PagedSpan s;
  s.low = p.window ? max(0, max(pos_lo, 0) - p.window + 1) : 0;
  s.high = max(0, min(pos_hi + 1, len));
  if (s.low >= s.high) {
    s.low = 0;
    if (p.window) s.high = min(s.high, p.sinks);
  }
  s.start = s.low & -block;
  s.skip = min((int)(((int64_t)p.sinks + block - 1) & -block), s.start);
  s.length = s.skip + s.high - s.start;
  return s;
}
__device__ __forceinline__ int paged_real(const PagedSpan& s, int v) { return v < s.skip ? v : v - s.skip + s.start; }
__device__ __forceinline__ int paged_chunks(const PagedSpan& s, int chunk_keys) { return max(1, (s.length + chunk_keys - 1) / chunk_keys); }
// Byte offset of virtual key v's K row of KV head 0.  A key inside a block that no row sees (between the sinks and the window) stands for
// one that some row does: what it holds must not reach a product, not even multiplied by zero.
__device__ __forceinline__ int64_t paged_row_bytes(const PagedParams& p, const PagedSequence& sq, const PagedSpan& s, int v) {
  const int real = paged_real(s, v), j = real >= p.sinks && real < s.low ? s.low : real;
  const int page = min(max(p.table[sq.b * p.table_stride + (j >> p.page_shift)], 0), p.max_pages - 1);
  const int64_t row = ((int64_t)p.hkv * p.head_dim) * (j & ((1 << p.page_shift) - 1));
  return 2 * ((int64_t)page * 2 * p.page_elems + row);
}

constexpr float kSlack = 8.0f;            // 2^8 above the reference is within the range of fp16, and costs no bits of a float's

template <int DT>
__device__ __forceinline__ v4f mfma16x16x32(dec_u4 a, dec_u4 b, v4f c) {
  if constexpr (DT == SUBSPEC_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}
typedef __attribute__((address_space(3))) v4s lds_v4s;
typedef __attribute__((address_space(3))) dec_u4 lds_u4;
__device__ __forceinline__ uint2 lds_tr16(uint32_t address) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(uintptr_t)address));
}
__device__ __forceinline__ dec_u4 lds_16(uint32_t address) { return *(const lds_u4*)(uintptr_t)address; }
__device__ __forceinline__ void dma16_nt(uint32_t lds_base, const void* src) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off nt" ::"s"(lds_base), "v"(src) : "memory", "m0");
}
__device__ __forceinline__ void dma16_from(uint32_t lds_base, const void* src) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds_base), "v"(src) : "memory", "m0");
}

// Tiles are numbered across the batch without a scan over it: sequence b's first tile is starts[b] * group / rows + b (rounded down), which leaves
// room for ceil(n * group / rows) of them before the next sequence's and for starts[batch] * group / rows + batch in all.  The sequence that
// tile u falls to is the last whose first tile is not behind it (every wavefront looks for itself, 64 sequences a load).
__device__ __forceinline__ int paged_first_tile(const PagedParams& p, int b) {
  return (int)((int64_t)min(max(p.starts[b], 0), p.n_tokens) * p.group / p.tile.rows) + b;
}
__device__ __forceinline__ int paged_tile_owner(const PagedParams& p, int u) {
  const int lane = threadIdx.x & (kWave - 1);
  int owners = 0;
  for (int b0 = 0; b0 < p.batch; b0 += kWave) {
    const int b = b0 + lane;
    owners += __popcll(__ballot(b < p.batch && paged_first_tile(p, b) <= u));
  }
  return max(owners - 1, 0);
}

constexpr int kTileRows = 256;             // eight wavefronts of 32 rows
constexpr int kTileKeys = 64;              // keys of a block
constexpr int kTilePages = 4096;           // page numbers of a chunk that are held in LDS
// products of sequences with more rows than p.few.rows (paged_tile.hip)
void launch_paged_tile(const PagedParams& p, int dtype, hipStream_t st);
void launch_paged_tile_merge(const PagedParams& p, int dtype, hipStream_t st);

}  // namespace subspec
