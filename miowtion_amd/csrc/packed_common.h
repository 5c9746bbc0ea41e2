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
  int32_t ranked_q, ranked_k;  // tiles of query rows, of keys, by their sequences' length
};

// A tile's place: its sequence's queries and keys, the tile's index in it, and the
// sequence's in the list.
struct Span {
  int32_t q0, nq, k0, nk, tile, seq;
};

// A tile past every row, for workgroups that have none (its first row is 2^30).
constexpr int32_t kNoTile = 1 << 23;

// The first slot of query tiles of a span's sequence.
__device__ __forceinline__ int first_q_slot(const Packing& p, const Span& s) {
  return (int)(((int64_t)s.q0 * p.group) / kRows) + s.seq;
}

// Read without a branch, so that several are under way at once.
__device__ __forceinline__ int32_t cu_at(const int32_t* cu, int i, int n_seq, int32_t rows) {
  const int32_t at = cu[min(max(i, 0), n_seq)];
  return i < 0 ? 0 : i > n_seq ? rows : min(max(at, 0), rows);
}

// The span of slot `slot`, by all lanes of a wave at once, 64 candidates a round;
// the last round's lanes hold the offsets of both sides, so the sequence's own
// come from the lanes beside each other. of_keys: slots count tiles of keys, not
// of query rows. Offsets that do not ascend give some sequence, whose rows are
// within the tensors all the same, or no tile.
__device__ __forceinline__ Span span_of_slot(const Packing& p, bool of_keys, int slot, int lane) {
  const int32_t* cu = of_keys ? p.cu_k : p.cu_q;
  const int32_t* other = of_keys ? p.cu_q : p.cu_k;
  const int32_t rows = of_keys ? p.k_rows : p.q_rows, other_rows = of_keys ? p.q_rows : p.k_rows;
  const int mult = of_keys ? 1 : p.group;
  const int last = p.n_seq + 1;
  int lo = 0, count = last + 1;
  while (count > 64) {
    const int stride = (count + 63) >> 6;
    const int i = min(lo + lane * stride, lo + count - 1);
    const int64_t at = ((int64_t)cu_at(cu, i - 1, p.n_seq, rows) * mult) / kRows + i;
    const uint64_t below = __ballot(lane * stride < count && at <= slot);
    const int next = lo + (max((int)__builtin_popcountll(below), 1) - 1) * stride;
    count = min(stride, lo + count - next);
    lo = next;
  }
  // lane: where sequence lo + lane begins, which is where the one before it ends
  const int32_t mine = cu_at(cu, lo + lane - 1, p.n_seq, rows);
  const int32_t its = cu_at(other, lo + lane - 1, p.n_seq, other_rows);
  const int64_t at = ((int64_t)mine * mult) / kRows + lo + lane;
  const uint64_t below = __ballot(lane < count && at <= slot);
  const int hit = max((int)__builtin_popcountll(below), 1) - 1;
  const int i = __builtin_amdgcn_readfirstlane(lo + hit);
  const int32_t begin = __builtin_amdgcn_readlane(mine, hit);
  const int32_t other_begin = __builtin_amdgcn_readlane(its, hit);
  const int32_t end = hit < 63 ? __builtin_amdgcn_readlane(mine, hit + 1) : cu_at(cu, i, p.n_seq, rows);
  const int32_t other_end =
      hit < 63 ? __builtin_amdgcn_readlane(its, hit + 1) : cu_at(other, i, p.n_seq, other_rows);
  Span s;
  s.q0 = of_keys ? other_begin : begin;
  s.nq = max(of_keys ? other_end - other_begin : end - begin, 0);
  s.k0 = of_keys ? begin : other_begin;
  s.nk = max(of_keys ? end - begin : other_end - other_begin, 0);
  s.tile = slot - (int)(((int64_t)begin * mult) / kRows + i);
  if (s.tile < 0) s.tile = kNoTile;  // offsets do not ascend
  s.seq = i;
  if (i == 0 || i == last) {  // rows of no sequence: no key, no query
    if (of_keys) s.nq = 0;
    else s.nk = 0;
  }
  return s;
}

// The tile at place `rank` when the sequences are taken from the longest walk to
// the shortest, for a long tile that starts late ends a launch alone: 30 prompts of
// 20 to 1,500, 1,380 workgroups, took 73 us in the order given, 68 in this (42 and
// 34 units of a step by list scheduling on 512 places); training on 20, 541 and
// 515 us. Taking the tiles themselves in the order of their work mixes the
// sequences, whose tiles then share no keys in the L2: 32 prompts of 512 took 79 us
// so, 68 by sequence.
//
// By all lanes of a wave, two sequences each (the two of no sequence among them).
// The place's level (walks of as many steps of 64) is found by bisection, its
// sequence within the level by a prefix sum. Within a level a sequence's tiles begin
// an eighth further on than the one's before: workgroups go round the XCDs and
// their shader engines, and where sequences of one length have as many tiles as the
// round, one engine would get the longest tile of each (the 32 prompts: 73 us).
// Launches that are resident at once, two workgroups to a CU, take the second half
// from the shortest on: a CU has a long and a short one (training on 32 of 512, 512
// workgroups to a kernel: 287 and 275 us). Up to one to a CU, the order is all the
// same. `each`: workgroups of a tile, heads and splits.
constexpr int kRankedSeqs = 126;
constexpr int64_t kRankedTiles = 256;

// Each lane's sum (or maximum, of none below 0) of its own and all lanes' before
// it: rows of 16 lanes in four steps, then over the rows' last lanes.
template <bool MAX>
__device__ __forceinline__ int lanes_upto(int x) {
  auto put = [&](int y) { x = MAX ? max(x, y) : x + y; };
  put(__builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false));  // row_shr:1
  put(__builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false));
  put(__builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false));
  put(__builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false));
  put(__builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));  // row_bcast:15
  put(__builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));  // row_bcast:31
  return x;
}

__device__ __forceinline__ Span span_of_rank(const Packing& p, bool of_keys, int rank, int each,
                                             int lane) {
  const int last = p.n_seq + 1;
  int32_t q0[2], nq[2], k0[2], nk[2], tiles[2], steps[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = lane + 64 * h;
    q0[h] = cu_at(p.cu_q, i - 1, p.n_seq, p.q_rows);
    k0[h] = cu_at(p.cu_k, i - 1, p.n_seq, p.k_rows);
    const int32_t q1 = cu_at(p.cu_q, i, p.n_seq, p.q_rows), k1 = cu_at(p.cu_k, i, p.n_seq, p.k_rows);
    nq[h] = i > last ? 0 : max(q1 - q0[h], 0);
    nk[h] = i > last ? 0 : max(k1 - k0[h], 0);
    const uint32_t rows = (uint32_t)(nq[h] * p.group);  // < 2^31
    tiles[h] = (int)(((of_keys ? (uint32_t)nk[h] : rows) + kRows - 1) / kRows);
    if (i == 0 || i == last) {  // rows of no sequence: no key, no query
      if (of_keys) nq[h] = 0;
      else nk[h] = 0;
    }
    steps[h] = (int)(((of_keys ? (uint32_t)(nq[h] * p.group) : (uint32_t)nk[h]) + 63u) >> 6);
  }
  // tiles of walks of `level` steps or more
  auto total = [&](int level) {
    const int n = (steps[0] >= level ? tiles[0] : 0) + (steps[1] >= level ? tiles[1] : 0);
    return __builtin_amdgcn_readlane(lanes_upto<false>(n), 63);
  };
  Span s{0, 0, 0, 0, kNoTile, 0};
  const int n_tiles = total(0);
  if (rank >= n_tiles) return s;
  if (n_tiles * each <= 512 && rank >= 256 / each) rank = n_tiles - 1 - (rank - 256 / each);
  int lo = 0, hi = __builtin_amdgcn_readlane(lanes_upto<true>(max(steps[0], steps[1])), 63) + 1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (total(mid) > rank) lo = mid;
    else hi = mid;
  }
  int left = rank - total(lo + 1);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int upto = lanes_upto<false>(steps[h] == lo ? tiles[h] : 0);
    const int at = (int)__builtin_popcountll(__ballot(upto <= left));
    if (at < 64) {
      const int n = __builtin_amdgcn_readlane(tiles[h], at);
      int in = left - (__builtin_amdgcn_readlane(upto, at) - n);
      s.q0 = __builtin_amdgcn_readlane(q0[h], at);
      s.nq = __builtin_amdgcn_readlane(nq[h], at);
      s.k0 = __builtin_amdgcn_readlane(k0[h], at);
      s.nk = __builtin_amdgcn_readlane(nk[h], at);
      s.seq = __builtin_amdgcn_readfirstlane(at + 64 * h);
      if (in < 0 || in >= n) return s;  // not where offsets ascend
      const uint64_t level = __ballot(steps[h] == lo && lane < at);
      in += (n * ((int)__builtin_popcountll(level) & 7)) >> 3;
      if (in >= n) in -= n;
      s.tile = of_keys ? in : n - 1 - in;
      return s;
    }
    left -= __builtin_amdgcn_readlane(upto, 63);
  }
  return s;
}

// The tile of a workgroup; slots are taken from the last one where they count
// query rows (causal: the last rows of a sequence see the most), from the first
// where they count keys.
__device__ __forceinline__ Span span_of(const Packing& p, bool of_keys, int item, int n_slots, int each,
                                        int lane) {
  if (of_keys ? p.ranked_k : p.ranked_q) return span_of_rank(p, of_keys, item, each, lane);
  return span_of_slot(p, of_keys, of_keys ? item : n_slots - 1 - item, lane);
}

// Whether a launch over `tiles` workgroups takes the sequences by their length.
inline int ranked(int64_t n_seq, int64_t tiles) {
  return n_seq >= 2 && n_seq <= kRankedSeqs && tiles >= kRankedTiles && tiles < (1 << 20);
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

// A wave's 32 packed rows r0 .. of a tensor [rows, heads, D] (`x` at the span's
// first row and the group's first head), zeros past `rows`: read as whole rows
// into registers, kSegRows a load. A fragment read straight from memory takes 32
// bytes of each of 32 rows, so a line comes in four times over once the rows of
// the waves beside it have pushed it out of L1.
template <int D>
struct RowLoads {
  u32x4 x[32 / Tile<D>::kSegRows];
};

template <int D>
__device__ __forceinline__ RowLoads<D> load_rows(const uint16_t* x, int64_t stride_s, int64_t stride_h,
                                                 int group, uint32_t per_group, int r0, int rows,
                                                 int lane) {
  using T = Tile<D>;
  RowLoads<D> res;
  const int t0 = r0 / group, rem = r0 - t0 * group;  // wave-uniform
#pragma unroll
  for (int i = 0; i < 32 / T::kSegRows; ++i) {
    const int rr = i * T::kSegRows + lane / T::kChunks;
    const uint32_t y = (uint32_t)(rr + rem);
    const uint32_t t = group == 1 ? y : __umulhi(y, per_group), g = y - t * (uint32_t)group;
    res.x[i] = u32x4{0, 0, 0, 0};
    if (r0 + rr < rows)
      res.x[i] = ld16(x + (t0 + (int64_t)t) * stride_s + (int64_t)g * stride_h + 8 * (lane % T::kChunks));
  }
  return res;
}

// 2^32 / group, rounded up, for divisions by it (0 for one). The quotient of x is
// exact for a row of a wave or of a step, at most group + 62, with every group up to
// 65,536 (each of them tried), and one too large for row group - 1 of 65,537, whose
// head would wrap below zero.
constexpr int64_t kMaxGroup = 1 << 16;
__host__ __device__ inline uint32_t per_group_of(uint32_t group) { return 0xffffffffu / group + 1; }

// Those rows as B operand fragments (lane: row lane % 32, chunk 2 s + lane / 32),
// by way of the wave's own 32 rows of LDS.
template <int D>
__device__ __forceinline__ void frags_of_rows(const RowLoads<D>& r, lds_u8* box, int lane,
                                              bf16x8 (&f)[Tile<D>::kK]) {
  using T = Tile<D>;
  typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
  const int li = lane & 31, hi = lane >> 5;
#pragma unroll
  for (int i = 0; i < 32 / T::kSegRows; ++i) {
    const int rr = i * T::kSegRows + lane / T::kChunks, pos = lane % T::kChunks;
    *reinterpret_cast<lds_u32x4*>(box + rr * T::kPitch + ((pos ^ swz_row<D>(rr)) << 4)) = r.x[i];
  }
  asm volatile("" ::: "memory");
#pragma unroll
  for (int s = 0; s < T::kK; ++s)
    f[s] = lds_frag(box + li * T::kPitch + (((2 * s + hi) ^ swz_row<D>(li)) << 4));
  asm volatile("" ::: "memory");
}

inline bool rows16(const void* p, int64_t s, int64_t h) {
  return ((reinterpret_cast<uintptr_t>(p) & 15) | ((s | h) & 7)) == 0;
}

}  // namespace veda
