// What the packed-attention kernels share: which rows of which sequence a
// workgroup takes, and the LDS layout of their tiles.
//
// Rows. Sequences lie one behind the other: queries [cu_q[b], cu_q[b + 1]),
// keys [cu_k[b], cu_k[b + 1]). The G = H / Hkv query heads of a key head are
// rows beside each other: row r of sequence b and key head h is query r / G of
// it, head h G + r % G. So K and V are read once for a group, the rows of a
// tile lie on one diagonal as far as they can (128 / G queries instead of 128),
// and dK and dV add up over the group inside a workgroup. A tile is 128 rows.
//
// Tiles without lengths on the host. Sequence i of the list below owns the
// slots from S(i) = floor(begin(i) G / 128) + i on, which are enough for its
// rows (ceil(n / 128) <= floor((a + n) / 128) - floor(a / 128) + 1), so a launch
// has floor(T G / 128) + sequences slots for each key head, and a workgroup
// finds its sequence by a search for the last i with S(i) <= slot. The list is
// the B sequences between two of no keys, the rows before cu[0] and the rows
// from cu[B] on, whose outputs are zeros.
#pragma once

#include "veda_pipeline.h"

namespace veda {

constexpr int kRows = 128;                       // query rows, or keys, of a workgroup

struct Packing {
  const int32_t* cu_q;
  const int32_t* cu_k;
  int32_t n_seq;
  int32_t q_rows, k_rows;  // rows of q and of k, v
  int32_t n_kv, group;     // key heads; query heads of each
  int32_t causal;
};

// A tile's place: its sequence's queries and keys, and the tile's index in it.
struct Span {
  int32_t q0, nq, k0, nk, tile;
};

__device__ __forceinline__ int32_t cu_at(const int32_t* cu, int i, int n_seq, int32_t rows) {
  return i < 0 ? 0 : i > n_seq ? rows : min(max(cu[i], 0), rows);
}

// The sequence of slot `slot` (of rows with `mult` rows a packed row), by all
// lanes of a wave at once: 64 candidates a round. Offsets that do not ascend
// give some sequence, whose rows are within the tensors all the same.
__device__ __forceinline__ int seq_of_slot(const int32_t* cu, int n_seq, int32_t rows, int mult,
                                           int slot, int lane) {
  int lo = 0, count = n_seq + 2;
  while (count > 1) {
    const int stride = (count + 63) >> 6;
    const int i = lo + lane * stride;
    const bool in = i < lo + count;
    const int64_t at = ((int64_t)cu_at(cu, in ? i - 1 : lo - 1, n_seq, rows) * mult) / kRows + i;
    const uint64_t below = __ballot(in && at <= slot);
    const int hits = max((int)__builtin_popcountll(below), 1);
    const int next = lo + (hits - 1) * stride;
    count = min(stride, lo + count - next);
    lo = next;
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

// The span of a slot; of_keys: slots count tiles of keys, not of query rows.
__device__ __forceinline__ Span span_of_slot(const Packing& p, bool of_keys, int slot, int lane) {
  const int32_t* cu = of_keys ? p.cu_k : p.cu_q;
  const int32_t rows = of_keys ? p.k_rows : p.q_rows;
  const int mult = of_keys ? 1 : p.group;
  const int i = seq_of_slot(cu, p.n_seq, rows, mult, slot, lane);
  Span s;
  s.q0 = cu_at(p.cu_q, i - 1, p.n_seq, p.q_rows);
  s.nq = max(cu_at(p.cu_q, i, p.n_seq, p.q_rows) - s.q0, 0);
  s.k0 = cu_at(p.cu_k, i - 1, p.n_seq, p.k_rows);
  s.nk = max(cu_at(p.cu_k, i, p.n_seq, p.k_rows) - s.k0, 0);
  const int32_t begin = of_keys ? s.k0 : s.q0;
  s.tile = slot - (int)(((int64_t)begin * mult) / kRows + i);
  if (i == 0 || i == p.n_seq + 1) {  // rows of no sequence: no key, no query
    if (of_keys) s.nq = 0;
    else s.nk = 0;
  }
  return s;
}

__host__ __device__ inline int64_t slots_of(int64_t rows, int64_t mult, int64_t n_seq) {
  return rows * mult / kRows + n_seq + 2;
}

// Keys that row r of a span sees (the first so many of them).
__device__ __forceinline__ int visible_keys(const Packing& p, const Span& s, int r) {
  if (!p.causal) return s.nk;
  return min(max(r / p.group + 1 + s.nk - s.nq, 0), s.nk);
}

// LDS tiles of 64 rows of D bf16, 16-byte chunks permuted by row so that a
// wave's 16-byte row reads and its transposed reads both meet every bank once
// (gfx950 serves a ds_read_b128 in 4 cycles of 16 lanes and a transposed read
// in 2 of 32): chunk c of row r lies at c ^ swz<D>(r).
template <int D>
__device__ __forceinline__ int swz_row(int r) {  // tiles read by rows
  return D == 128 ? r & 15 : (r >> 1) & 7;
}
template <int D>
__device__ __forceinline__ int swz_tr(int r) {  // tiles read transposed
  return D == 128 ? (r & 3) << 2 : ((r >> 1) & 1) << 2;
}
// both ways (a swizzle of its own, as the rows of a row read and the rows of a
// transposed read differ in other bits)
template <int D>
__device__ __forceinline__ int swz_both(int r) {
  return D == 128 ? ((r & 3) << 2) | ((r >> 2) & 3) : (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
}

template <int D>
struct Tile {
  static constexpr int kPitch = 2 * D;                // bytes of a row
  static constexpr int kChunks = D / 8;               // 16-byte chunks of a row
  static constexpr int kSegRows = 64 / kChunks;       // rows of a wave's 1 KB load
  static constexpr int kSegs = 16 / kSegRows;         // such loads of a wave for 64 rows
  static constexpr int kBytes = 64 * kPitch;          // 64 rows
  static constexpr int kK = D / 16;                   // k-steps of a product over D
  static constexpr int kT = D / 32;                   // 32-wide blocks of D
};

// Offset in a tile of the transposed read (rows 4 hi + i / 4, columns 32 dt +
// 16 dh + 4 (i % 4) .. + 3) that gives lane (dh, i) row 32 dt + 16 dh + i of
// the transposed 16-row block; the next 8 rows of it are at + 8 kPitch where
// the swizzle does not change there.
template <int D, typename Swz>
__device__ __forceinline__ uint32_t tr_offset(int lane, int dt, int row_add, Swz swz) {
  const int i = lane & 15, dh = (lane >> 4) & 1, hi = lane >> 5;
  const int r = 4 * hi + (i >> 2) + row_add;
  const int c = 4 * dt + 2 * dh + ((i >> 1) & 1);
  return (uint32_t)(r * Tile<D>::kPitch + ((c ^ swz(r)) << 4) + 8 * (i & 1));
}

__device__ __forceinline__ bf16x8 join_tr(const lds_u8* lo, const lds_u8* up) {
  const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)lo);
  const i16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)up);
  return __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

__device__ __forceinline__ f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ bf16x8 lds_frag(const lds_u8* p) {
  return as_bf16x8(*reinterpret_cast<const __attribute__((address_space(3))) u32x4*>(p));
}

__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int e = 0; e < 16; ++e) z[e] = 0.f;
  return z;
}

inline bool rows16(const void* p, int64_t s, int64_t h) {
  return ((reinterpret_cast<uintptr_t>(p) & 15) | ((s | h) & 7)) == 0;
}

}  // namespace veda
