#pragma once
// Attention of sequences that share a prefix, over the paged cache: the
// workgroup of one work item, and the merge of split rows.
//
// An item (PrefixItem, le_internal.h) is a tile of query columns (row, head of
// one kv head) against a range of keys of one block table: the shared keys,
// attended by the rows of every sequence of a group, or the keys that follow
// them, by one sequence's rows under the causal mask. For a column c
//     s_k = q_c . k_k scale,  m = max_k s_k,  l = sum_k e^(s_k - m),
//     o = sum_k e^(s_k - m) v_k
// over the item's keys; a row with one item is done (out = o / l), the others
// leave (m, l, o) in fp32 and the merge adds them up:
//     out = sum_i o_i e^(m_i - M) / sum_i l_i e^(m_i - M),  M = max_i m_i.
//
// Four waves bring 64 keys at a time into LDS (16 each; double buffered, the
// next tile's loads in registers meanwhile) and share them in one of two ways:
//   * tiles of more than 32 columns: a wave has 32 columns and all 64 keys
//     (32x32x16 MFMA), one barrier a tile;
//   * up to 32 columns, where three waves would idle: a wave has all columns
//     and the 16 keys that it loads itself (16x16 MFMAs, no barrier), and the
//     four waves' (m, l, o) are merged at the end. A single row is this case:
//     it is bound by its keys' bytes, not by the products. Items of a few keys,
//     where there are many, take a wave each, in the same way but for the merge.
// S^T = K Q^T and O^T = V^T P^T: a lane holds one column, and its scores are
// the second product's B operand as they are (A and B only have to agree on
// the order of keys). q enters as it is and the scale is applied to the fp32
// scores, so 16-bit products are exact.
//
// Arithmetic: q, K and V of one 16-bit type use that type's MFMA, and the
// softmax weights are rounded to it (the row sum is of the rounded weights; in
// the key-sharing case, which has the matrix cores to spare, they are two
// 16-bit terms instead). fp32 q over a bf16 cache, and their weights, are three
// bf16 terms each: products of 24 bits, in a fifth of the fp32 MFMA's cycles (256
// rows behind 16384 keys and 64 to 1024 of their own, 32/8 heads x 128: 318 us, on
// the fp32 MFMA 868).
// Anything else uses the fp32 MFMA on widened operands.
//
// What bounds it: narrow tiles, HBM (256 sequences of 64 to 1024 keys, 8 kv
// heads x 128, bf16: 108 us, 5.4 TB/s of K and V); wide ones, the products and
// the softmax beside them, at the clock that they leave (122 rows after 131072
// keys, 32/8 heads x 128: 327 us, 800 TFLOP/s; on zeros 264); small steps, the
// chain of two launches (block ids, q, keys, record, merge: 7 us at least).
#include <float.h>

#include <type_traits>

#include "le_common.h"
#include "le_internal.h"

namespace le {
namespace pfx {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr int kKeys = kPrefixTileKeys;  // keys of an LDS tile
constexpr int kNarrow = kPrefixNarrow;  // columns up to which the waves share keys
constexpr float kSlack = 8.f;           // log2 units that scores may pass a column's base by

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef short bf16raw4 __attribute__((ext_vector_type(4)));

// The operand type: the 16-bit type of both, bf16 also under fp32 activations, or
// float.
template <typename ACT, typename KV>
using operand = std::conditional_t<(std::is_same_v<ACT, KV> && sizeof(KV) == 2) ||
                                       (std::is_same_v<ACT, float> && std::is_same_v<KV, bf16_t>), KV, float>;
// Terms of the operand type that a q element is given in; softmax weights have
// as many (one: rounded; 16 keys a wave: two).
template <typename ACT, typename KV> constexpr int kTerms = !std::is_same_v<ACT, KV> && sizeof(operand<ACT, KV>) == 2 ? 3 : 1;

// Products over 16 (wide: 32x32 tiles) or 32 (narrow: 16x16 tiles) dims, a
// lane holding eight consecutive ones of its row of A and column of B; and
// over keys, four of a lane's scores at a time (nt) or eight (wt).
template <typename X> struct mm;
template <> struct mm<bf16_t> {
  using frag = bf16x8;
  using scalar = __bf16;
  typedef __bf16 pair __attribute__((ext_vector_type(2)));
  // c + a[0] + a[1], for the row sum of rounded weights
  __device__ __forceinline__ static float sum2(pair a, float c) {
    const pair ones = {static_cast<__bf16>(1.f), static_cast<__bf16>(1.f)};
    return __builtin_amdgcn_fdot2_f32_bf16(a, ones, c, false);
  }
  __device__ __forceinline__ static frag load(const char* p) { return *reinterpret_cast<const frag*>(p); }
  __device__ __forceinline__ static f32x16 wide(frag a, frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  __device__ __forceinline__ static f32x4 narrow(frag a, frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  __device__ __forceinline__ static f32x4 keys16(bf16x4 a, bf16x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(bf16raw4, a), __builtin_bit_cast(bf16raw4, b),
                                                     c, 0, 0, 0);
  }
};
template <> struct mm<f16_t> {
  using frag = f16x8;
  using scalar = _Float16;
  typedef _Float16 pair __attribute__((ext_vector_type(2)));
  __device__ __forceinline__ static float sum2(pair a, float c) {
    const pair ones = {static_cast<_Float16>(1.f), static_cast<_Float16>(1.f)};
    return __builtin_amdgcn_fdot2(a, ones, c, false);
  }
  __device__ __forceinline__ static frag load(const char* p) { return *reinterpret_cast<const frag*>(p); }
  __device__ __forceinline__ static f32x16 wide(frag a, frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  __device__ __forceinline__ static f32x4 narrow(frag a, frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  __device__ __forceinline__ static f32x4 keys16(f16x4 a, f16x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, c, 0, 0, 0);
  }
};
template <> struct mm<float> {
  using frag = f32x8;
  using scalar = float;
  __device__ __forceinline__ static f32x16 wide(const frag& a, const frag& b, f32x16 c) {
#pragma unroll
    for (int e = 0; e < 8; e++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
  __device__ __forceinline__ static f32x4 narrow(const frag& a, const frag& b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 8; e++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
};

// A tile in LDS: 64 K rows, then 64 V rows, no padding (a wave's 16-byte stores
// fill 1 KB in lane order). Piece s of row r holds the row's piece s ^ f(r), so
// that neither the 16-byte fragment reads of consecutive rows nor the
// transposing reads of four rows x 64 bytes meet on a bank.
template <typename KV, int HD> struct Geo {
  static constexpr int ES = static_cast<int>(sizeof(KV));
  static constexpr int ROW = HD * ES;
  static constexpr int CPR = ROW / 16;         // pieces of a row
  static constexpr int RPI = kWave / CPR;      // rows that a wave's load covers
  static constexpr int IPW = 16 / RPI;         // loads of a wave's 16 rows
  static constexpr int K_BYTES = kKeys * ROW;
  static constexpr int BYTES = 2 * K_BYTES;
  __device__ __forceinline__ static int f(int row) {
    return CPR == 8 ? ((row & 2) << 1) | ((row >> 2) & 3) : ((row & 3) << 2) | ((row >> 2) & 3);
  }
};
template <typename KV, int HD> struct Smem {
  __attribute__((aligned(16))) char lds[2][Geo<KV, HD>::BYTES];
  float2 ml[kWaves][kNarrow];  // a wave's (max, sum) of each column, at the end
  int2 row[kNarrow];           // token and first record of each row, for the end
};
// a row of the end's accumulators, in the tiles' place
template <int HD> constexpr int kAccRow = HD + 4;

// eight elements from piece `piece` of an LDS row on, as an operand
template <typename X, typename KV, int HD>
__device__ __forceinline__ typename mm<X>::frag lds_frag(const char* row, int f, int piece) {
  const char* p = row + ((piece ^ f) << 4);
  if constexpr (!std::is_same_v<X, float>) {
    return mm<X>::load(p);
  } else {
    float v[8];
    elem<KV>::widen(ld16(p), v);
    if constexpr (sizeof(KV) == 4) elem<KV>::widen(ld16(row + (((piece + 1) ^ f) << 4)), v + 4);
    f32x8 r;
#pragma unroll
    for (int e = 0; e < 8; e++) r[e] = v[e];
    return r;
  }
}
// one element of an LDS row
template <typename KV, int HD> __device__ __forceinline__ float lds_elem(const char* row, int f, int i) {
  constexpr int PE = 16 / static_cast<int>(sizeof(KV));
  return elem<KV>::load1(reinterpret_cast<const KV*>(row + (((i / PE) ^ f) << 4)) + i % PE);
}

__device__ __forceinline__ float vmax3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
__device__ __forceinline__ float halves_max(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return vmax2(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float halves_sum(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// The last product's result may be read: the compiler counts the wait states of
// an MFMA result up to its first reader, but not up to one in inline assembly,
// and not along every way around a conditional block.
template <typename X> __device__ __forceinline__ void settle() {
  __builtin_amdgcn_sched_barrier(0);
  if constexpr (std::is_same_v<X, float>) asm volatile("s_nop 15\n\ts_nop 3");
  else asm volatile("s_nop 11");
  __builtin_amdgcn_sched_barrier(0);
}

// A query column: its row's token and first record, its head, and the last key
// that it sees, relative to the item's first (negative: none of them).
struct Column {
  int token, part0, head, lim;
  bool ok;  // the column exists
};
// A column's row among its item's: c / G (c < 128, G <= 8: exact).
__device__ __forceinline__ int row_index(const PrefixParams& p, int c) { return (c * p.per_row) >> 16; }
// The item's row of a column (past its last: the list repeats that one).
__device__ __forceinline__ PrefixRow row_of(const PrefixParams& p, int item, int c) {
  return p.rows[static_cast<int64_t>(item) * p.rows_stride + min(row_index(p, c), p.rows_stride - 1)];
}
__device__ __forceinline__ Column column_of(const PrefixParams& p, const PrefixItem& it, const PrefixRow& row, int kvh, int c) {
  const int G = p.q_heads / p.kv_heads;
  const int r = row_index(p, c);
  Column o;
  o.ok = r < it.n_rows;
  o.token = row.token;
  o.part0 = row.part0;
  o.head = kvh * G + c - r * G;
  o.lim = o.ok ? min(it.key_end - 1, row.pos) - it.key_begin : -1;
  return o;
}

// x as N terms of type S, the largest first. What they leave is 2^-25 of x with
// three bf16 ones (an infinity is in the first alone).
template <int N, typename S> __device__ __forceinline__ void split(float x, S (&t)[N]) {
#pragma unroll
  for (int k = 0; k < N; k++) {
    t[k] = static_cast<S>(x);
    const float y = static_cast<float>(t[k]);
    if (k + 1 < N) x = y - y == 0.f ? x - y : 0.f;
  }
}
// the same of a weight, which is at most some hundreds
template <int N, typename S> __device__ __forceinline__ void split_weight(float x, S (&t)[N]) {
#pragma unroll
  for (int k = 0; k < N; k++) {
    t[k] = static_cast<S>(x);
    if (k + 1 < N) x -= static_cast<float>(t[k]);
  }
}

// eight elements of a column's q from dim d on, with the scale's sign
template <typename ACT, typename X, int TERMS>
__device__ __forceinline__ void q_frag(const PrefixParams& p, const Column& c, int hd, int d, typename mm<X>::frag (&r)[TERMS]) {
  const ACT* q = static_cast<const ACT*>(p.q) + (static_cast<int64_t>(c.token) * p.q_heads + c.head) * hd + d;
  if constexpr (sizeof(X) == 2 && TERMS == 1) {  // the same type: bits
    u32x4 raw = *reinterpret_cast<const u32x4*>(q);
    const uint32_t sign = p.negate ? 0x80008000u : 0u, keep = c.ok ? ~0u : 0u;
#pragma unroll
    for (int e = 0; e < 4; e++) raw[e] = (raw[e] ^ sign) & keep;
    r[0] = __builtin_bit_cast(typename mm<X>::frag, raw);
  } else {
    float f[8];
    elem<ACT>::load8(q, f);
#pragma unroll
    for (int e = 0; e < 8; e++) {
      typename mm<X>::scalar t[TERMS];
      split(c.ok ? (p.negate ? -f[e] : f[e]) : 0.f, t);
#pragma unroll
      for (int k = 0; k < TERMS; k++) r[k][e] = t[k];
    }
  }
}

// Where a row's part is written: its record's accumulator and (m, l).
__device__ __forceinline__ int64_t record_of(const PrefixParams& p, const PrefixItem& it, int part0, int head) {
  return (static_cast<int64_t>(part0) + it.part) * p.q_heads + head;
}

// A wave's 16 rows of every tile. The rows' blocks are the wave's (16 keys from
// a multiple of 16 on lie in one block, or in two of 8), so their addresses are
// scalars and a lane adds its place in the rows. The block ids of 64 blocks at a
// time wait in a register, a block a lane (first_id: the first ones, as listed).
template <typename KV, int HD, bool SOLO = false> struct Loader {
  using L = Geo<KV, HD>;
  static constexpr int kStep = SOLO ? kKeys / kWaves : kKeys;  // keys of a tile
  const char* kbase;
  const char* vbase;
  const int32_t* ids;
  uint32_t row_bytes, block_bytes, num_blocks;  // a block is less than 4 GiB, the caller checks
  int n_keys, wave, row0, bs_shift, last_blk, window;  // row0: the wave's first row of a tile
  int32_t id_now, id_next;  // lane i: block 64 * window + i's id, and 64 further
  uint32_t off[L::IPW];
  struct Stage {  // a tile in flight
    u32x4 k[L::IPW], v[L::IPW];
    uint32_t gone;  // bits 0 and 1: its rows 0-7 and 8-15 have no block
  };

  __device__ __forceinline__ Loader(const PrefixParams& p, const PrefixItem& it, int kvh, int32_t first_id) {
    const int lane = threadIdx.x & (kWave - 1);
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    row0 = SOLO ? 0 : wave * 16;
    kbase = static_cast<const char*>(p.k_cache) + static_cast<int64_t>(kvh) * L::ROW;
    vbase = static_cast<const char*>(p.v_cache) + static_cast<int64_t>(kvh) * L::ROW;
    ids = p.ids + it.ids_off;
    row_bytes = static_cast<uint32_t>(p.kv_heads) * L::ROW;
    block_bytes = row_bytes * p.block_size;
    num_blocks = static_cast<uint32_t>(min(p.num_cache_blocks, static_cast<int64_t>(INT32_MAX) + 1));
    n_keys = it.key_end - it.key_begin;
    bs_shift = __builtin_ctz(p.block_size);
    last_blk = (n_keys - 1) >> bs_shift;
    window = 0;
    id_now = first_id;
    id_next = last_blk >= kWave ? ids[min(kWave + lane, last_blk)] : 0;
#pragma unroll
    for (int j = 0; j < L::IPW; j++) {
      const int row = j * L::RPI + lane / L::CPR;
      off[j] = static_cast<uint32_t>((row & 7) * row_bytes) + (((lane % L::CPR) ^ L::f(row)) << 4);
    }
  }
  // eight consecutive rows of a block as a buffer: a scalar descriptor, and a
  // lane's 32-bit offset is all it adds
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t rows8(const char* base) const {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, 8 * row_bytes, 0x00027000);
  }
  // requests the tile whose first key, relative to the item's, is rel
  __device__ __forceinline__ void issue(Stage& st, int rel) {
    const int w = (rel >> bs_shift) >> 6;
    if (w != window) {
      window = w;
      id_now = id_next;
      id_next = ids[min((w + 1) * kWave + static_cast<int>(threadIdx.x & (kWave - 1)), last_blk)];
    }
    st.gone = 0;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      // eight keys (past the range: its last eight again)
      const int key = min(rel + row0 + h * 8, (n_keys - 1) & ~7);
      const int id = __builtin_amdgcn_readlane(id_now, (key >> bs_shift) & (kWave - 1));
      const bool in = static_cast<uint32_t>(id) < num_blocks;
      st.gone |= in ? 0u : 1u << h;
      const uint64_t at = static_cast<uint64_t>(in ? id : 0) * block_bytes + (key & ((1 << bs_shift) - 1)) * row_bytes;
      const auto kr = rows8(kbase + at), vr = rows8(vbase + at);
#pragma unroll
      for (int j = h * L::IPW / 2; j < (h + 1) * L::IPW / 2; j++) {
        st.k[j] = __builtin_amdgcn_raw_buffer_load_b128(kr, off[j], 0, 0);
        st.v[j] = __builtin_amdgcn_raw_buffer_load_b128(vr, off[j], 0, 0);
      }
    }
  }
  // Puts it into LDS. V rows past the range become zeros (a weight of 0 times
  // what the cache holds there need not be 0), and K and V rows without a block.
  __device__ __forceinline__ void stash(const Stage& st, char* buf, int rel) const {
    const int lane = threadIdx.x & (kWave - 1);
    const int live = n_keys - (rel + row0);
    char* dst = buf + wave * L::IPW * 1024 + lane * 16;
#pragma unroll
    for (int j = 0; j < L::IPW; j++) {
      *reinterpret_cast<u32x4*>(dst + j * 1024) = st.k[j];
      *reinterpret_cast<u32x4*>(dst + j * 1024 + L::K_BYTES) = st.v[j];
    }
    if (live < 16 || st.gone != 0) {
#pragma unroll
      for (int j = 0; j < L::IPW; j++) {
        const int row = j * L::RPI + lane / L::CPR;
        const bool none = (st.gone >> (row >> 3)) & 1u;
        if (none) *reinterpret_cast<uint4*>(dst + j * 1024) = make_uint4(0, 0, 0, 0);
        if (none || row >= live) *reinterpret_cast<uint4*>(dst + j * 1024 + L::K_BYTES) = make_uint4(0, 0, 0, 0);
      }
    }
  }
};

// Calls tile(LDS buffer, first key) for the tiles of an item; stage a holds the
// first one's loads. Shared rows: one tile in flight beside the one in use, and
// a barrier a tile.
template <typename KV, int HD, typename F>
__device__ __forceinline__ void shared_tiles(Loader<KV, HD>& ld, typename Loader<KV, HD>::Stage& a, Smem<KV, HD>& sm,
                                             F tile) {
  const int n_tiles = (ld.n_keys + kKeys - 1) / kKeys;
  ld.stash(a, sm.lds[0], 0);
  for (int t = 0; t < n_tiles; t++) {
    __syncthreads();  // all rows of tile t are there, and tile t - 1 is no longer read
    if (t + 1 < n_tiles) ld.issue(a, (t + 1) * kKeys);
    tile(sm.lds[t & 1], t * kKeys);
    if (t + 1 < n_tiles) ld.stash(a, sm.lds[(t + 1) & 1], (t + 1) * kKeys);
  }
}
// A wave's own rows: two tiles in flight beside the one in use (what bounds
// such items is how many bytes are on their way), no barrier.
template <typename KV, int HD, bool SOLO, typename F>
__device__ __forceinline__ void own_tiles(Loader<KV, HD, SOLO>& ld, typename Loader<KV, HD, SOLO>::Stage& a,
                                          Smem<KV, HD>& sm, F tile) {
  constexpr int kStep = Loader<KV, HD, SOLO>::kStep;
  typename Loader<KV, HD, SOLO>::Stage b;
  const int n_tiles = (ld.n_keys + kStep - 1) / kStep;
  if (n_tiles > 1) ld.issue(b, kStep);
  for (int t = 0; t < n_tiles; t += 2) {
    const int rel = t * kStep;
    ld.stash(a, sm.lds[0], rel);
    if (t + 2 < n_tiles) ld.issue(a, rel + 2 * kStep);
    tile(sm.lds[0], rel);
    if (t + 1 >= n_tiles) break;
    ld.stash(b, sm.lds[1], rel + kStep);
    if (t + 3 < n_tiles) ld.issue(b, rel + 3 * kStep);
    tile(sm.lds[1], rel + kStep);
  }
}

// ---- more than 32 columns: 32 a wave ----
template <typename ACT, typename KV, int HD>
__device__ __forceinline__ void wide_item(const PrefixParams& p, const PrefixItem& it, const PrefixRow& row, int kvh,
                                          int32_t first_id, Smem<KV, HD>& sm) {
  using X = operand<ACT, KV>;
  using M = mm<X>;
  using L = Geo<KV, HD>;
  constexpr int KS = HD / 16, DT = HD / 32, U = kKeys / 32;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
  const int col = lane & 31, half = lane >> 5, l16 = lane & 15;
  Loader<KV, HD> ld(p, it, kvh, first_id);
  typename Loader<KV, HD>::Stage first;
  ld.issue(first, 0);
  const Column c = column_of(p, it, row, kvh, wave * 32 + col);
  constexpr int TERMS = kTerms<ACT, KV>;
  typename M::frag qb[KS][TERMS];
#pragma unroll
  for (int ks = 0; ks < KS; ks++) q_frag<ACT, X>(p, c, HD, ks * 16 + half * 8, qb[ks]);
  // the wave's keys: none past the last one that any of its columns sees, and
  // no mask up to the first that one does not (columns without a row aside)
  const bool any = row_index(p, wave * 32) < it.n_rows;
  int wave_lim = c.lim, free_lim = c.ok ? c.lim : INT32_MAX;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    wave_lim = max(wave_lim, __shfl_xor(wave_lim, d, kWave));
    free_lim = min(free_lim, __shfl_xor(free_lim, d, kWave));
  }
  wave_lim = __builtin_amdgcn_readfirstlane(any ? wave_lim : -1);
  free_lim = __builtin_amdgcn_readfirstlane(free_lim);

  f32x16 acc[DT];
#pragma unroll
  for (int d = 0; d < DT; d++)
#pragma unroll
    for (int e = 0; e < 16; e++) acc[d][e] = 0.f;
  float base = 0.f, thr = -FLT_MAX, lsum = 0.f;  // thr -FLT_MAX: no key yet
  const float scale = p.scale_log2;
  // Where a lane's fragments lie in the tile, piece 0's: a piece further on is
  // an xor away, and so is the other buffer.
  const int fk = L::f(col), vrow = 4 * half + (l16 >> 2), vpiece = ((lane >> 4) & 1) * 2 + ((l16 & 3) >> 1);
  int k_at = col * L::ROW + ((half ^ fk) << 4);
  int v_at = vrow * L::ROW + ((vpiece ^ L::f(vrow)) << 4) + (l16 & 1) * 8;
  shared_tiles(ld, first, sm, [&](const char* b, int rel) {
    if (rel > wave_lim) return;
    f32x16 s[U];
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int e = 0; e < 16; e++) s[u][e] = 0.f;
    // 16-bit products go in the order written: each with the read of the
    // fragment four products on. (Left to it, the compiler reads two fragments
    // and waits for them.)
    constexpr int kAhead = 4, N = U * KS;
    typename M::frag kf[kAhead];
    auto k_frag = [&](int i) {
      if constexpr (sizeof(X) == 2) return M::load(&sm.lds[0][0] + (k_at ^ ((i / U) * 32)) + (i % U) * 32 * L::ROW);
      else return lds_frag<X, KV, HD>(b + ((i % U) * 32 + col) * L::ROW, fk, ((i / U) * 16 + half * 8) * L::ES / 16);
    };
#pragma unroll
    for (int i = 0; i < kAhead; i++) kf[i] = k_frag(i);
    if constexpr (sizeof(X) == 2) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < N; i++) {
#pragma unroll
      for (int k = 0; k < TERMS; k++) s[i % U] = M::wide(kf[i % kAhead], qb[i / U][k], s[i % U]);
      if (i + kAhead < N) kf[i % kAhead] = k_frag(i + kAhead);
      if constexpr (sizeof(X) == 2) __builtin_amdgcn_sched_barrier(0);
    }
    settle<X>();
    // accumulator e of a lane is key 8 (e / 4) + 4 half + e % 4
    if (rel + kKeys - 1 > free_lim) {
      const int m = c.lim - rel - half * 4;
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int e = 0; e < 16; e++)
          if (32 * u + 8 * (e / 4) + e % 4 > m) s[u][e] = -INFINITY;
    }
    float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int e = 0; e < 16; e += 4)
#pragma unroll
      for (int i = 0; i < 4; i++) m4[i] = vmax3(m4[i], s[i >> 1][e + 2 * (i & 1)], s[i >> 1][e + 2 * (i & 1) + 1]);
    const float mt = vmax2(vmax3(m4[0], m4[1], m4[2]), m4[3]);
    const float y = __builtin_fmaf(mt, scale, -base);
    if (__builtin_amdgcn_ballot_w64(y > thr)) {
      // A column's first keys set its base to their maximum; later ones
      // move it when they pass it by more than kSlack.
      const float m = halves_max(y);
      const bool go = m > thr;
      const float shift = go ? m : 0.f;
      const float alpha = go && thr != -FLT_MAX ? __builtin_amdgcn_exp2f(-shift) : 1.f;
      base += shift;
      thr = go ? kSlack : thr;
      lsum *= alpha;
#pragma unroll
      for (int d = 0; d < DT; d++) acc[d] *= alpha;
    }
    if constexpr (std::is_same_v<X, float>) {
#pragma unroll
      for (int u = 0; u < U; u++) {
#pragma unroll
        for (int e = 0; e < 16; e++) {
          s[u][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][e], scale, -base));
          lsum += s[u][e];
        }
#pragma unroll
        for (int e = 0; e < 16; e++) {
          const int row = 8 * (e / 4) + 4 * half + e % 4;
#pragma unroll
          for (int d = 0; d < DT; d++) {
            const float a = lds_elem<KV, HD>(b + L::K_BYTES + (u * 32 + row) * L::ROW, L::f(row), d * 32 + col);
            acc[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, s[u][e], acc[d], 0, 0, 0);
          }
        }
      }
    } else {
      // weights g: those of accumulators 8 (g % 2) .. + 7 of s[g / 2]
      typename M::frag pb[2 * U][TERMS];
      auto weights = [&](int g, int e) {
        const f32x16& x = s[g / 2];
        const int at = 8 * (g % 2) + e;
        const float w0 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[at], scale, -base));
        const float w1 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[at + 1], scale, -base));
        typename M::scalar t0[TERMS], t1[TERMS];
        split_weight(w0, t0);
        split_weight(w1, t1);
#pragma unroll
        for (int k = 0; k < TERMS; k++) {
          pb[g][k][e] = t0[k];
          pb[g][k][e + 1] = t1[k];
        }
        if constexpr (TERMS == 1) lsum = M::sum2(typename M::pair{t0[0], t1[0]}, lsum);
        else lsum += w0 + w1;
      };
      // Beside each product: the read of the fragment two products on, and its
      // share of the next 16 keys' weights.
      // V^T operand of 16 keys: lane (dim 16 (lane / 16 % 2) + lane % 16,
      // half) holds the keys of weights g
      constexpr int kAheadV = 2, NV = 2 * U * DT;
      typename M::frag vf[kAheadV];
      auto v_frag = [&](int i) {
        const int g = i / DT, d = i % DT;
        const char* vp = &sm.lds[0][0] + L::K_BYTES + 16 * g * L::ROW;
        const auto lo = lds_read_tr16<KV>(vp + (v_at ^ (d * 64)));
        const auto hi = lds_read_tr16<KV>(vp + 8 * L::ROW + (v_at ^ (d * 64 + 32)));  // f(row + 8) = f(row) ^ 2
        return typename M::frag{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      };
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < kAheadV; i++) vf[i] = v_frag(i);
#pragma unroll
      for (int e = 0; e < 8; e += 2) weights(0, e);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < NV; i++) {
        const int g = i / DT, d = i % DT;
#pragma unroll
        for (int k = 0; k < TERMS; k++) acc[d] = M::wide(vf[i % kAheadV], pb[g][k], acc[d]);
        if (i + kAheadV < NV) vf[i % kAheadV] = v_frag(i + kAheadV);
        if (g + 1 < 2 * U) {
#pragma unroll
          for (int e = d * 8 / DT; e < (d + 1) * 8 / DT; e += 2) weights(g + 1, e);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    k_at ^= L::BYTES;
    v_at ^= L::BYTES;
  });

  // acc[d][e] = O[column][dim 32 d + 8 (e / 4) + 4 half + e % 4]
  const float l = halves_sum(lsum);
  if (!c.ok) return;
  if (it.part < 0) {
    ACT* out = static_cast<ACT*>(p.out) + (static_cast<int64_t>(c.token) * p.q_heads + c.head) * HD + half * 4;
    const float inv = 1.f / l;
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const float f[4] = {acc[d][e] * inv, acc[d][e + 1] * inv, acc[d][e + 2] * inv, acc[d][e + 3] * inv};
        elem<ACT>::store4(out + d * 32 + e * 2, f);
      }
    return;
  }
  const int64_t rec = record_of(p, it, c.part0, c.head);
  float* o = p.acc + rec * HD + half * 4;
#pragma unroll
  for (int d = 0; d < DT; d++)
#pragma unroll
    for (int e = 0; e < 16; e += 4)
      *reinterpret_cast<float4*>(o + d * 32 + e * 2) = make_float4(acc[d][e], acc[d][e + 1], acc[d][e + 2], acc[d][e + 3]);
  if (half == 0) p.ml[rec] = make_float2(l > 0.f ? base : -FLT_MAX, l);
}

// ---- up to 32 columns: 16 of the 64 keys a wave ----
// NC column tiles of 16, known at compile time: with a branch around the second
// tile's products the compiler left the first one's result a wait too short on
// the way past the branch (fp32: a score without its last product).
// SOLO: the wave has the item for itself, all keys.
template <typename ACT, typename KV, int HD, int NC, bool SOLO>
__device__ __forceinline__ void narrow_item(const PrefixParams& p, const PrefixItem& it, const PrefixRow* rows, int kvh,
                                            int32_t first_id, Smem<KV, HD>& sm) {
  using X = operand<ACT, KV>;
  using M = mm<X>;
  using L = Geo<KV, HD>;
  constexpr int KS = HD / 32, DT = HD / 16;
  const int lane = threadIdx.x & (kWave - 1);
  const int l16 = lane & 15, g = lane >> 4;
  const int G = p.q_heads / p.kv_heads;
  Loader<KV, HD, SOLO> ld(p, it, kvh, first_id);
  const int wave = ld.wave;
  typename Loader<KV, HD, SOLO>::Stage first;
  ld.issue(first, 0);
  Column c[NC];
  constexpr int TERMS = kTerms<ACT, KV>;
  typename M::frag qb[NC][KS][TERMS];
#pragma unroll
  for (int n = 0; n < NC; n++) {
    c[n] = column_of(p, it, rows[n], kvh, n * 16 + l16);
#pragma unroll
    for (int ks = 0; ks < KS; ks++) q_frag<ACT, X>(p, c[n], HD, ks * 32 + g * 8, qb[n][ks]);
  }
  if (!SOLO && wave == 0 && g == 0) {
#pragma unroll
    for (int n = 0; n < NC; n++)
      if (c[n].ok) sm.row[row_index(p, n * 16 + l16)] = make_int2(c[n].token, c[n].part0);
  }

  f32x4 acc[NC][DT];
  float m[NC], lsum[NC];
#pragma unroll
  for (int n = 0; n < NC; n++) {
    m[n] = -FLT_MAX;
    lsum[n] = 0.f;
#pragma unroll
    for (int d = 0; d < DT; d++) acc[n][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const float scale = p.scale_log2;
  own_tiles(ld, first, sm, [&](const char* tile, int rel) {
    const int key0 = rel + ld.row0;  // this wave's keys
    if (key0 >= ld.n_keys) return;
    const char* b = tile + wave * 16 * L::ROW;
    const char* bv = b + L::K_BYTES;
    const int fk = L::f(l16);
    f32x4 s[NC];
#pragma unroll
    for (int n = 0; n < NC; n++) s[n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
      const auto ka = lds_frag<X, KV, HD>(b + l16 * L::ROW, fk, (ks * 32 + g * 8) * L::ES / 16);
#pragma unroll
      for (int n = 0; n < NC; n++)
#pragma unroll
        for (int k = 0; k < TERMS; k++) s[n] = M::narrow(ka, qb[n][ks][k], s[n]);
    }
    // accumulator i of a lane is key 4 g + i
    float w[NC][4];
#pragma unroll
    for (int n = 0; n < NC; n++) {
      const int lim = c[n].lim - key0 - 4 * g;
      float x[4], mt = -FLT_MAX;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        x[i] = i > lim ? -INFINITY : s[n][i] * scale;
        mt = vmax2(mt, x[i]);
      }
      const float mn = vmax2(m[n], rows_max(mt));
      if (__builtin_amdgcn_ballot_w64(mn > m[n])) {
        const float alpha = __builtin_amdgcn_exp2f(m[n] - mn);
        m[n] = mn;
        lsum[n] *= alpha;
#pragma unroll
        for (int d = 0; d < DT; d++) acc[n][d] *= alpha;
      }
#pragma unroll
      for (int i = 0; i < 4; i++) {
        w[n][i] = __builtin_amdgcn_exp2f(x[i] - m[n]);
        lsum[n] += w[n][i];
      }
    }
    if constexpr (std::is_same_v<X, float>) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int row = 4 * g + i;
#pragma unroll
        for (int d = 0; d < DT; d++) {
          const float a = lds_elem<KV, HD>(bv + row * L::ROW, L::f(row), d * 16 + l16);
#pragma unroll
          for (int n = 0; n < NC; n++) acc[n][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(a, w[n][i], acc[n][d], 0, 0, 0);
        }
      }
    } else {
      constexpr int WT = TERMS == 1 ? 2 : TERMS;
      typename mma16<KV>::v4 wt[NC][WT];
#pragma unroll
      for (int n = 0; n < NC; n++) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
          typename M::scalar t[WT];
          split_weight(w[n][i], t);
#pragma unroll
          for (int k = 0; k < WT; k++) wt[n][k][i] = t[k];
        }
      }
      const int row = 4 * g + (l16 >> 2), piece = (l16 & 3) >> 1, f = L::f(row);
      const char* vp = bv + row * L::ROW + (l16 & 1) * 8;
#pragma unroll
      for (int d = 0; d < DT; d++) {
        const auto va = lds_read_tr16<KV>(vp + (((d * 2 + piece) ^ f) << 4));
#pragma unroll
        for (int n = 0; n < NC; n++) {
#pragma unroll
          for (int k = 0; k < WT; k++) acc[n][d] = M::keys16(va, wt[n][k], acc[n][d]);
        }
      }
    }
  });

  if constexpr (SOLO) {
    // acc[n][d][i] = O[column 16 n + l16][dim 16 d + 4 g + i]
#pragma unroll
    for (int n = 0; n < NC; n++) {
      const float l = rows_sum(lsum[n]);
      if (!c[n].ok) continue;
      if (it.part < 0) {
        ACT* out = static_cast<ACT*>(p.out) + (static_cast<int64_t>(c[n].token) * p.q_heads + c[n].head) * HD + g * 4;
        const float inv = 1.f / l;
#pragma unroll
        for (int d = 0; d < DT; d++) {
          const float f[4] = {acc[n][d][0] * inv, acc[n][d][1] * inv, acc[n][d][2] * inv, acc[n][d][3] * inv};
          elem<ACT>::store4(out + d * 16, f);
        }
      } else {
        const int64_t rec = record_of(p, it, c[n].part0, c[n].head);
#pragma unroll
        for (int d = 0; d < DT; d++) *reinterpret_cast<f32x4*>(p.acc + rec * HD + d * 16 + g * 4) = acc[n][d];
        if (g == 0) p.ml[rec] = make_float2(m[n], l);
      }
    }
    return;
  }
  // ---- the four waves' results, in the tiles' place: 16 columns at a time,
  // waves 0 and 1 in the first buffer, 2 and 3 in the second ----
  // acc[n][d][i] = O[column 16 n + l16][dim 16 d + 4 g + i]
  constexpr int AR = kAccRow<HD>, PIECES = HD / 4;
  static_assert(2 * 16 * AR * 4 <= L::BYTES);
  float* mine = reinterpret_cast<float*>(wave < 2 ? sm.lds[0] : sm.lds[1]) + (wave & 1) * 16 * AR;
#pragma unroll
  for (int n = 0; n < NC; n++) {
    const float l = rows_sum(lsum[n]);
    if (g == 0) sm.ml[wave][n * 16 + l16] = make_float2(m[n], l);
  }
#pragma unroll
  for (int n = 0; n < NC; n++) {
    __syncthreads();
#pragma unroll
    for (int d = 0; d < DT; d++) *reinterpret_cast<f32x4*>(mine + l16 * AR + d * 16 + 4 * g) = acc[n][d];
    __syncthreads();
    const int cols = min(16, it.n_rows * G - n * 16);
    for (int i = threadIdx.x; i < cols * PIECES; i += kThreads) {
      const int cl = i / PIECES, cc = n * 16 + cl, d = (i - cl * PIECES) * 4;
      const int row = row_index(p, cc), head = kvh * G + cc - row * G;
      const int2 o = sm.row[row];
      float M4 = -FLT_MAX;
#pragma unroll
      for (int w = 0; w < kWaves; w++) M4 = fmaxf(M4, sm.ml[w][cc].x);
      float l = 0.f;
      f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWaves; w++) {
        const float2 x = sm.ml[w][cc];
        const float f = __builtin_amdgcn_exp2f(x.x - M4);
        const float* all = reinterpret_cast<const float*>(w < 2 ? sm.lds[0] : sm.lds[1]) + (w & 1) * 16 * AR;
        l += x.y * f;
        a += *reinterpret_cast<const f32x4*>(all + cl * AR + d) * f;
      }
      if (it.part < 0) {
        const float inv = 1.f / l;
        const float f[4] = {a[0] * inv, a[1] * inv, a[2] * inv, a[3] * inv};
        elem<ACT>::store4(static_cast<ACT*>(p.out) + (static_cast<int64_t>(o.x) * p.q_heads + head) * HD + d, f);
      } else {
        const int64_t rec = record_of(p, it, o.y, head);
        *reinterpret_cast<f32x4*>(p.acc + rec * HD + d) = a;
        if (d == 0) p.ml[rec] = make_float2(M4, l);
      }
    }
  }
}

template <typename ACT, typename KV, int HD>
__global__ __launch_bounds__(kThreads, (HD > 64 && (std::is_same_v<operand<ACT, KV>, float> || kTerms<ACT, KV> > 1) ? 1 : 2)) void prefix_kernel(PrefixParams p) {
  __shared__ Smem<KV, HD> sm;
  // an item's kv heads lie side by side: their rows are neighbours in the cache
  const uint32_t shared = static_cast<uint32_t>(p.n_items - p.n_solo) * p.kv_heads;
  uint32_t unit = blockIdx.x;
  if (unit >= shared) {  // an item a wave
    unit = shared + (unit - shared) * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (unit >= static_cast<uint32_t>(p.n_items) * p.kv_heads) return;
  }
  const int item = unit / p.kv_heads, kvh = unit - item * p.kv_heads;
  const int lane = threadIdx.x & (kWave - 1);
  const int32_t first_id = p.item_ids[static_cast<int64_t>(item) * p.ids_stride +
                                      min(lane, p.ids_stride - 1)];
  // the rows of a lane's columns, of every kind of tile: asked for beside the item
  const PrefixRow wide_row = row_of(p, item, threadIdx.x / kWave * 32 + (lane & 31));
  const PrefixRow rows[2] = {row_of(p, item, lane & 15), row_of(p, item, 16 + (lane & 15))};
  const PrefixItem it = p.items[item];
  const int cols = it.n_rows * (p.q_heads / p.kv_heads);
  if (blockIdx.x >= shared) {
    if (cols <= 16) narrow_item<ACT, KV, HD, 1, true>(p, it, rows, kvh, first_id, sm);
    else narrow_item<ACT, KV, HD, 2, true>(p, it, rows, kvh, first_id, sm);
  } else if (cols <= 16) {
    narrow_item<ACT, KV, HD, 1, false>(p, it, rows, kvh, first_id, sm);
  } else if (cols <= kNarrow) {
    narrow_item<ACT, KV, HD, 2, false>(p, it, rows, kvh, first_id, sm);
  } else {
    wide_item<ACT, KV, HD>(p, it, wide_row, kvh, first_id, sm);
  }
}

// ---- rows of several parts: a wave for each (row, head) ----
// The parts' factors are formed by the lanes together (a part each, 64 at a
// time); then a lane has four dims of every 64 / (HD / 4)-th part, four loads in
// flight beside the four in use. (One thread per four dims that went through all parts by itself took
// 21.7 us for 64 rows x 14 heads x 64 of 34 parts.)
template <typename ACT, int HD>
__global__ __launch_bounds__(kThreads) void prefix_merge_kernel(PrefixParams p) {
  constexpr int DL = HD / 4, GROUPS = kWave / DL;
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t rh = static_cast<int64_t>(blockIdx.x) * kWaves + (threadIdx.x >> 6);
  if (rh >= static_cast<int64_t>(p.n_tokens) * p.q_heads) return;
  const int token = static_cast<int>(rh / p.q_heads), head = static_cast<int>(rh - static_cast<int64_t>(token) * p.q_heads);
  const int n = p.row_parts[token];
  if (n <= 1) return;
  const int64_t rec0 = static_cast<int64_t>(p.part0[token]) * p.q_heads + head;
  const float2* ml = p.ml + rec0;
  const float* acc = p.acc + rec0 * HD + (lane & (DL - 1)) * 4;
  const int64_t step = static_cast<int64_t>(p.q_heads) * HD;
  const int group = lane / DL;
  // the parts' factors, 64 at a time, and beside them the first parts' loads
  float2 x = ml[static_cast<int64_t>(min(lane, n - 1)) * p.q_heads];
  f32x4 v[4];
  auto load = [&](int k) {
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = *reinterpret_cast<const f32x4*>(acc + min(k + j * GROUPS + group, n - 1) * step);
  };
  load(0);
  float M = x.x;
  for (int k = lane + kWave; k < n; k += kWave) M = fmaxf(M, ml[static_cast<int64_t>(k) * p.q_heads].x);
  M = wave_max(M);
  float l = 0.f;
  f32x4 a = {0.f, 0.f, 0.f, 0.f};
  for (int k0 = 0; k0 < n; k0 += kWave) {
    if (k0 > 0) x = ml[static_cast<int64_t>(min(k0 + lane, n - 1)) * p.q_heads];
    const float f = k0 + lane < n ? __builtin_amdgcn_exp2f(x.x - M) : 0.f;
    l += x.y * f;
    const int end = min(n - k0, kWave);
    for (int i = 0; i < end; i += 4 * GROUPS) {  // (all lanes: a part's factor may be any lane's)
      f32x4 now[4];
#pragma unroll
      for (int j = 0; j < 4; j++) now[j] = v[j];
      if (k0 + i + 4 * GROUPS < n) load(k0 + i + 4 * GROUPS);
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float w = __shfl(f, i + j * GROUPS + group, kWave);
        a += w > 0.f ? now[j] * w : f32x4{0.f, 0.f, 0.f, 0.f};
      }
    }
  }
  l = wave_sum(l);
#pragma unroll
  for (int d = DL; d < kWave; d <<= 1)
#pragma unroll
    for (int e = 0; e < 4; e++) a[e] += __shfl_xor(a[e], d, kWave);
  if (group != 0) return;
  const float inv = 1.f / l;
  const float f[4] = {a[0] * inv, a[1] * inv, a[2] * inv, a[3] * inv};
  elem<ACT>::store4(static_cast<ACT*>(p.out) + rh * HD + lane * 4, f);
}

template <typename ACT, typename KV, int HD>
hipError_t launch_prefix(const PrefixParams& p, hipStream_t stream) {
  const int64_t solo = static_cast<int64_t>(p.n_solo) * p.kv_heads, units = static_cast<int64_t>(p.n_items) * p.kv_heads;
  prefix_kernel<ACT, KV, HD><<<static_cast<unsigned>(units - solo + (solo + kWaves - 1) / kWaves), kThreads, 0, stream>>>(p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.n_parts == 0) return e;
  const int64_t waves = static_cast<int64_t>(p.n_tokens) * p.q_heads;
  prefix_merge_kernel<ACT, HD><<<static_cast<unsigned>((waves + kWaves - 1) / kWaves), kThreads, 0, stream>>>(p);
  return hipGetLastError();
}

}  // namespace
}  // namespace pfx
}  // namespace le
