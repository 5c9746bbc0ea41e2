// Attention of a chunk of new tokens of every sequence over a paged cache that holds
// them already, for gfx950: queries [cu[b], cu[b + 1]) of sequence b, n_q of them, see
// the first n_k = lengths[b] positions of its cache, query i the keys up to
// i + n_k - n_q when causal. Formulas, rows and the walk are those of the packed
// forward (packed_walk.h); keys and values come from the cache's pages as they lie
// (paged_common.h), in bf16 or e4m3.
//
// A wave loads 16 of a step's 64 keys, which lie in one page: pages have 16 rows at
// least and begin where a block of 16 keys does. A lane holds where the keys of one step
// lie for its wave, 64 steps at a time, so a step's place is one lane's registers.
//   bf16: rows go from the page straight into LDS.
//   e4m3: codes wait for one iteration, while they come (V's in registers, K's in LDS),
//         and are decoded (times the row's power of two: exact) on their way into the
//         slots, once for the workgroup's 128 rows. (Products of the codes themselves, by
//         the instructions that take e4m3 with a scale for a row and Q as two terms of
//         it, took 7 to 8 % less time, but cut a product off at 2^-13 of the largest of eight:
//         an LSE off by 1e-5 where it is off by 1e-7.)
// A key in a page outside the cache draws no weight.
//
// Where rows are many, bound as the packed forward is, by power (two chunks of 2,048 onto
// 32,768 and 20,001, 32 heads on 8, head_dim 128: 1,460 to 1,520 us, 1.14 PFLOP/s; 1,640 in
// e4m3, which takes a tenth more LDS accesses and a fifth more vector instructions);
// where they are few, by the cache's bytes (four tokens of eight sequences over 40,103
// positions in all, 8 key heads: 34 us, 4.8 TB/s); between them in e4m3 by latency, of an
// iteration's chain and of its loads (9 tokens of 64 sequences of 4,096: 152 us, 3.6 TB/s, 2.3
// us an iteration, of half of bf16's bytes, which takes 220 us, 4.9 TB/s; with codes asked for
// two steps ahead, but no products among the softmax, as LDS has not room for both: 179 us).
// A few rows over e4m3 are bound by latency too: the four tokens of eight sequences above, with
// their join, take 26 us for 37 in bf16, 3.2 TB/s, with one tile a wave on its way in either type.
// A workgroup takes one unit. Equal shares of all tiles' steps for as many workgroups as
// are resident, tiles cut where a share ends, took longer (40 on 8 heads, 16 tokens of 48
// sequences: 62 us for 53; four chunks of 512, head_dim 64: 162 for 131): starts and ends
// cost 6 to 11 us each, and the tiles of a sequence read their keys at different times.
#include <type_traits>

#include "packed_walk.h"
#include "paged_common.h"

namespace veda {
namespace {

constexpr int kThreads = 256;

struct ChunkArgs {
  Packing pk;  // cu_k is cu_q: the keys' lengths are apart
  const uint16_t* q;
  int64_t qs, qh;
  Pages kp, vp;
  Table tab;
  const int32_t* lengths;
  uint16_t* out;
  int64_t os, oh;
  float* lse;   // [q_rows, H] or NULL
  float* part;  // n_split > 1: [n_split][q_rows, H][D] sums, [n_split][q_rows, H] pairs of
                // reference (log2) and sum of weights, [q_rows, H] numbers of splits
  float scale_log2;
  int32_t n_slots, n_split;
  int32_t units;  // splits of a key head beyond one of each tile at most, or 0: a slot's
                  // splits lie side by side
  int32_t resident;  // workgroups at once of a key head's share of the GPU
  uint32_t per_group;
};

// A workgroup's share: its tile, and which of how many splits of the keys.
struct Unit {
  Span sp;
  int split, splits;
};

constexpr int kMinSteps = 4;  // of 64 keys, of a split
// What a split costs beside its steps, in steps: its start, and its rows' sums written
// and read again.
constexpr float kStart = 5.f, kStartRows = 20.f / 128, kStartFew = 15.f;
constexpr int64_t kEarlyRows = 4096;

// Rows r0 .. r0 + 127 of a span: their queries, without a division each. (Products with
// 2^32 / group, rounded up, are exact up to group + 127: each group was tried.)
struct Queries {
  int first, rem, group;
  uint32_t per_group;
  __device__ __forceinline__ Queries(const ChunkArgs& p, int r0)
      : first(r0 / p.pk.group), rem(r0 - first * p.pk.group), group(p.pk.group), per_group(p.per_group) {}
  // of row r0 + x, and the row's head of the group
  __device__ __forceinline__ int query(int x) const {
    return group == 1 ? first + x : first + (int)__umulhi((uint32_t)(rem + x), per_group);
  }
  __device__ __forceinline__ int head(int x) const { return rem + x - (query(x) - first) * group; }
};

// Keys that query i of a span sees.
__device__ __forceinline__ int seen(const ChunkArgs& p, const Span& s, int i) {
  return p.pk.causal ? min(max(i + 1 + s.nk - s.nq, 0), s.nk) : s.nk;
}

// Keys of sequence b; none of the rows of no sequence (b -1 or n_seq).
__device__ __forceinline__ int cached(const ChunkArgs& p, int b) {
  if (p.pk.n_seq == 0) return 0;  // lengths holds none
  const int n = p.lengths[min(max(b, 0), p.pk.n_seq - 1)];
  return b < 0 || b >= p.pk.n_seq || p.tab.pages == 0 ? 0 : min(max(n, 0), p.tab.width << p.tab.shift);
}

// Up to 126 sequences, two to a lane: unit `rank` of those that all tiles' splits make,
// sequences with long units first where not all are resident at once (span_of_rank has
// the order and why). Splits follow the sequences' lengths, which the host does not
// know: with W steps in all on R places, splits of n steps that cost s more each take
// W (1 + s / n) / R and on average half of a split longer until the last one ends, which
// is least at n = sqrt(2 s W / R). By all lanes of a wave.
__device__ __forceinline__ Unit unit_of_rank(const ChunkArgs& p, int rank, int lane) {
  const int last = p.pk.n_seq + 1;
  const bool two = last >= 64;  // sequences in a lane's second place
  int32_t q0[2] = {}, nq[2] = {}, nk[2] = {}, tiles[2] = {}, steps[2] = {}, splits[2] = {1, 1}, units[2] = {};
  float work = 0.f, base = 0.f, all = 0.f;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (h == 1 && !two) break;
    const int i = lane + 64 * h;
    q0[h] = cu_at(p.pk.cu_q, i - 1, p.pk.n_seq, p.pk.q_rows);
    const int32_t q1 = cu_at(p.pk.cu_q, i, p.pk.n_seq, p.pk.q_rows);
    nk[h] = cached(p, i - 1);
    nq[h] = i > last ? 0 : max(q1 - q0[h], 0);
    tiles[h] = (int)(((uint32_t)(nq[h] * p.pk.group) + kRows - 1) / kRows);
    steps[h] = (int)(((uint32_t)nk[h] + 63u) >> 6);
    work += (float)tiles[h] * (float)steps[h];
    base += (float)tiles[h];
    all += (float)nq[h] * (float)p.pk.group;
  }
  work = wave_reduce<false>(work);
  base = wave_reduce<false>(base);
  all = wave_reduce<false>(all);
  const float each_rows = all * __builtin_amdgcn_rcpf(fmaxf(base, 1.f));  // of a tile
  const float start = each_rows <= 32.f ? kStartFew : kStart + kStartRows * each_rows;
  const float best = __builtin_amdgcn_sqrtf(2.f * start * work * __builtin_amdgcn_rcpf((float)p.resident));
  // (the grid has room for work / per more units than tiles; a few roundings of 2^-23)
  const float per = fmaxf(fmaxf(best, work * 1.0001f * __builtin_amdgcn_rcpf((float)p.units)), (float)kMinSteps);
  const float per_inv = __builtin_amdgcn_rcpf(per);
  float level[2] = {0.f, 0.f};  // steps of a split
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    splits[h] = (int)fminf((float)steps[h] * per_inv * 0.99999f + 1.f, (float)p.n_split);
    units[h] = tiles[h] * splits[h];
    level[h] = (float)steps[h] * __builtin_amdgcn_rcpf((float)splits[h]);
  }
  int n_units = __builtin_amdgcn_readlane(lanes_upto<false>(units[0]), 63);
  if (two) n_units += __builtin_amdgcn_readlane(lanes_upto<false>(units[1]), 63);
  Unit x{{0, 0, 0, 0, kNoTile, 0}, 0, 1};
  if (rank >= n_units) return x;
  int left = rank;
  if (n_units * p.pk.n_kv > 512) {  // not all are resident at once
    steps[0] = (int)level[0];
    steps[1] = (int)level[1];
    auto total = [&](int from) {
      const int n = (steps[0] >= from ? units[0] : 0) + (steps[1] >= from ? units[1] : 0);
      return __builtin_amdgcn_readlane(lanes_upto<false>(n), 63);
    };
    int lo = 0, hi = __builtin_amdgcn_readlane(lanes_upto<true>(max(steps[0], steps[1])), 63) + 1;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (total(mid) > rank) lo = mid;
      else hi = mid;
    }
    left -= total(lo + 1);
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (steps[h] != lo) units[h] = 0;
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int upto = lanes_upto<false>(units[h]);
    const int at = (int)__builtin_popcountll(__ballot(upto <= left));
    if (at < 64) {
      const int n = __builtin_amdgcn_readlane(units[h], at);
      const uint32_t in = (uint32_t)(left - (__builtin_amdgcn_readlane(upto, at) - n));
      x.sp.q0 = __builtin_amdgcn_readlane(q0[h], at);
      x.sp.nq = __builtin_amdgcn_readlane(nq[h], at);
      x.sp.nk = __builtin_amdgcn_readlane(nk[h], at);
      x.sp.seq = __builtin_amdgcn_readfirstlane(at + 64 * h);
      if (in >= (uint32_t)n) return x;  // not where offsets ascend
      x.splits = __builtin_amdgcn_readlane(splits[h], at);
      const int tile = (int)(in / (uint32_t)x.splits);
      x.split = (int)in - tile * x.splits;
      x.sp.tile = __builtin_amdgcn_readlane(tiles[h], at) - 1 - tile;
      return x;
    }
    left -= __builtin_amdgcn_readlane(upto, 63);
  }
  return x;
}

// More sequences: the tile of a slot, its splits side by side in the grid, in the order given.
// That ends with the longest sequence: 1 to 8,021 keys each, 4 tokens, 40 on 8 heads, 126
// sequences by rank 123 us (e4m3 73), 127 by slot 201 (141), 256 287 (203).
__device__ __forceinline__ Unit unit_of_slot(const ChunkArgs& p, int item, int lane) {
  Unit x;
  x.sp = span_of_slot(p.pk, false, p.n_slots - 1 - item / p.n_split, lane);
  x.sp.k0 = 0;
  x.sp.nk = cached(p, x.sp.seq - 1);
  x.splits = min(max((((x.sp.nk + 63) >> 6) + kMinSteps - 1) / kMinSteps, 1), p.n_split);
  x.split = item % p.n_split;
  if (x.split >= x.splits) x.sp.tile = kNoTile;
  return x;
}

// A row whose O came out with a NaN though its sum of weights has none, again, key by
// key, as redo_row of the packed forward: `limit` keys from `first` on. kx, vx, ke and
// ve: at the key head; table: at the sequence. (By single values: a struct would be
// kept in memory for it, by every walk.)
template <int D, bool F8>
__device__ __noinline__ void redo_paged_row(const uint16_t* q, const uint8_t* kx, const uint8_t* vx,
                                            const uint8_t* ke, const uint8_t* ve, int64_t sp, int64_t ss,
                                            int64_t ep, int64_t es, const int32_t* table, int pages, int shift,
                                            int first, int limit, float c, float mu, float inv, uint16_t* out,
                                            float* part, int lane) {
  const int mask = (1 << shift) - 1;
  float acc[D / 64] = {};
  for (int j0 = 0; j0 < limit; j0 += 64) {
    const int j = first + j0 + lane;
    const int at = j & mask;
    int page = -1;
    if (j0 + lane < limit) {
      page = table[j >> shift];
      if (page >= pages) page = -1;
    }
    float pr = 0.f;
    if (page >= 0) {
      const int64_t off = page * sp + at * ss;
      float s = 0.f;
      for (int d = 0; d < D; d += 8) {
        const u32x4 a = ld16(q + d);
        u32x4 k;
        if (F8) {
          const u32x2 w = *reinterpret_cast<const u32x2*>(kx + off + d);
          const float e = scale_of(ke[page * ep + at * es]);
          k = u32x4{decode2<false>(w[0], e), decode2<true>(w[0], e), decode2<false>(w[1], e),
                    decode2<true>(w[1], e)};
        } else {
          k = *reinterpret_cast<const u32x4*>(kx + 2 * (off + d));
        }
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          s = fmaf(bf16_to_f32(a[m] & 0xffffu), bf16_to_f32(k[m] & 0xffffu), s);
          s = fmaf(bf16_to_f32(a[m] >> 16), bf16_to_f32(k[m] >> 16), s);
        }
      }
      pr = __builtin_amdgcn_exp2f(fmaf(s, c, -mu));
    }
    for (int i = 0; i < min(64, limit - j0); ++i) {
      const float pi = __shfl(pr, i);
      const int64_t pg = __shfl(page, i);
      if (pi == 0.f) continue;  // (no page: no weight)
      const int row = (first + j0 + i) & mask;
#pragma unroll
      for (int m = 0; m < D / 64; ++m) {
        const int64_t off = pg * sp + row * ss + lane + 64 * m;
        const uint32_t v = F8 ? decode2<false>(vx[off], scale_of(ve[pg * ep + row * es])) & 0xffffu
                              : reinterpret_cast<const uint16_t*>(vx)[off];
        acc[m] = fmaf(pi, bf16_to_f32(v), acc[m]);
      }
    }
  }
#pragma unroll
  for (int m = 0; m < D / 64; ++m) {
    if (part != nullptr) part[lane + 64 * m] = acc[m];
    else out[lane + 64 * m] = (uint16_t)f32_to_bf16(acc[m] * inv);
  }
}

// A row's exponent, held as the aligned word with its byte and the byte's place: a value
// of a byte that waits through an iteration of a loop is widened at its end, which would
// wait for it there.
struct Exponent {
  uint32_t word, bit;
};
// The byte at x + off.
__device__ __forceinline__ Exponent exponent_at(const uint8_t* x, uint32_t off) {
  const uint32_t low = (uint32_t)reinterpret_cast<uintptr_t>(x) & 3u, at = off + low;
  return Exponent{*reinterpret_cast<const uint32_t*>(x - low + (at & ~3u)), 8 * (at & 3u)};
}
__device__ __forceinline__ uint32_t byte_of(const Exponent& x) { return __builtin_amdgcn_ubfe(x.word, x.bit, 8); }

// Scores of keys in blocks of 16 that have no page: bit 0 the sub-block's first.
__device__ __forceinline__ void mask_blocks(f32x16& s, uint32_t bad) {
#pragma unroll
  for (int e = 0; e < 16; ++e)
    if ((bad >> (e >> 3)) & 1) s[e] = -INFINITY;
}

// A step's 16 keys of a wave: where their first row lies in K and V (bytes) and in the
// exponents, the rows from there to the sequence's end, and the step's blocks of 16
// without a page (bits 0 to 3).
struct Place {
  int64_t at, exp;
  int rows;
  uint32_t bad;
};

typedef __attribute__((address_space(3))) u32x4 lds_u32x4;

// ---------------------------------------------------------------------------
// A sequence of at most 32 rows (few new tokens), 16 NB at most: each wave takes tiles of 32 keys of its
// own, every fourth of the unit's, for all rows, and nothing waits for another wave
// until the end, as in the attention of one token (paged.hip has the layout of its
// 16x16 products): K goes from memory straight into the operand, V through the wave's
// own LDS, both asked for again once their registers are free. In the walk of 128 rows
// one wave would have all the work of such a tile and three none (eight sequences of
// 2,000 to 8,192, 16 rows: 39 us there and 37 here, in e4m3 41 and 27).

template <int D, bool F8, int NB>
__device__ __forceinline__ void few_rows(const ChunkArgs& p, const Unit& unit, const Queries& of, int head, int rows,
                                         int from, int n_steps, int last, int wave, int lane, lds_u8* s0) {
  constexpr int kPitch = 2 * D;               // a V row in LDS, bf16
  constexpr int kTileBytes = 32 * kPitch;
  constexpr int kPer = F8 ? 16 : 8;           // elements of a 16-byte load
  constexpr int kBytes = F8 ? 1 : 2;
  constexpr int kKLoads = D / (4 * kPer);     // of a lane, for a K row
  constexpr int kSteps = D / 32;              // k-steps of a score
  constexpr int kLanes = D / kPer;            // lanes of a V row
  constexpr int kVRows = 64 / kLanes;         // V rows of a load
  constexpr int kVLoads = 32 / kVRows;
  constexpr int kDB = D / 16;
  typedef __attribute__((address_space(3))) f32x4 lds_f32x4;
  __shared__ float red_m[4][16 * NB], red_l[4][16 * NB];
  const Span& sp = unit.sp;
  const int n = lane & 15, g = lane >> 4, b = sp.seq - 1;
  const int begin = 64 * from, end = min(64 * (from + n_steps), last);
  const int last_block = max(sp.nk - 1, 0) >> 4, mask = (1 << p.tab.shift) - 1;
  const int64_t n_heads = (int64_t)p.pk.n_kv * p.pk.group, all_rows = p.pk.q_rows * n_heads;
  const int64_t row0 = sp.q0 * n_heads + (int64_t)head * p.pk.group;
  // Q: row 16 nb + n, in the order of the K loads' elements; the keys that it sees
  bf16x8 qf[NB][kSteps];
  int lim[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int r = min(16 * nb + n, rows - 1);
    lim[nb] = min(seen(p, sp, of.query(r)), end);
    const uint16_t* qrow = p.q + (sp.q0 + of.query(r)) * p.qs + ((int64_t)head * p.pk.group + of.head(r)) * p.qh;
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      qf[nb][s] = as_bf16x8(ld16(qrow + (F8 ? 64 * (s >> 1) + 16 * g + 8 * (s & 1) : 32 * s + 8 * g)));
  }
  const int see_all = min(seen(p, sp, 0), end);  // keys that every row sees
  const uint8_t* const kx = p.kp.x + head * p.kp.sh * kBytes;
  const uint8_t* const vx = p.vp.x + head * p.kp.sh * kBytes;
  const uint8_t* const kex = F8 ? p.kp.e + head * p.kp.eh : nullptr;
  const uint8_t* const vex = F8 ? p.vp.e + head * p.kp.eh : nullptr;
  const uint32_t row_bytes = (uint32_t)(p.kp.ss * kBytes), row_exps = (uint32_t)p.kp.es;
  const int vr = lane / kLanes, vd = kPer * (lane % kLanes);
  // Pages of a tile's two blocks, -1 where there is none; lane i: of the wave's i-th tile
  // from `window` on
  int pages[2], window = 0;
  auto look = [&](int tile) __attribute__((always_inline)) {
    window = tile;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int block = min(((begin + 32 * wave) >> 4) + 8 * (tile + lane) + i, last_block);
      const int x = p.tab.t[b * p.tab.ld + (block >> (p.tab.shift - 4))];
      pages[i] = x >= 0 && x < p.tab.pages ? x : -1;
    }
  };
  u32x4 kreg[2][kKLoads], vreg[kVLoads];
  Exponent ke[2], ve[kVLoads];
  auto load_k = [&](int j0, const int (&pg)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t page = max(pg[i], 0);
      const uint32_t at = (uint32_t)((j0 + 16 * i + n) & mask);
      const uint8_t* x = kx + page * p.kp.sp * kBytes;
      const uint32_t off = at * row_bytes + 16 * g;
#pragma unroll
      for (int s = 0; s < kKLoads; ++s) kreg[i][s] = *reinterpret_cast<const u32x4*>(x + (off + 64 * s));
      if (F8) ke[i] = exponent_at(kex + page * p.kp.ep, at * row_exps);
    }
  };
  auto load_v = [&](int j0, const int (&pg)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < kVLoads; ++u) {
      const int64_t page = max(pg[kVRows * u < 16 ? 0 : 1], 0);
      const uint32_t at = (uint32_t)((j0 + kVRows * u + vr) & mask);
      vreg[u] = *reinterpret_cast<const u32x4*>(vx + page * p.kp.sp * kBytes + (at * row_bytes + vd * kBytes));
      if (F8) ve[u] = exponent_at(vex + page * p.kp.ep, at * row_exps);
    }
  };
  lds_u8* const mine = s0 + wave * kTileBytes;
  // transposed reads: rows 4 g + n / 4 (and 16 on), column block db at xor 32 db
  const int tr_row = 4 * g + (n >> 2);
  const uint32_t tr = (uint32_t)(tr_row * kPitch + ((((n >> 1) & 1) ^ swz_v<D>(tr_row)) << 4) + 8 * (n & 1));
  f32x4 o[NB][kDB];
  float m_run[NB], l_run[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
    for (int db = 0; db < kDB; ++db) o[nb][db] = f32x4{0.f, 0.f, 0.f, 0.f};
    m_run[nb] = -INFINITY;
    l_run[nb] = 0.f;
  }
  const float c = p.scale_log2;
  int j = begin + 32 * wave, tile = 0;
  int now[2] = {-1, -1}, next[2] = {-1, -1};
  if (j < end) {
    look(0);
#pragma unroll
    for (int i = 0; i < 2; ++i) now[i] = __builtin_amdgcn_readlane(pages[i], 0);
    load_k(j, now);
    load_v(j, now);
  }
  for (; j < end; j += 128, ++tile) {
    const bool more = j + 128 < end;
    if (more) {
      if (tile + 1 - window >= 64) look(tile + 1);
#pragma unroll
      for (int i = 0; i < 2; ++i) next[i] = __builtin_amdgcn_readlane(pages[i], tile + 1 - window);
    }
    f32x4 s[NB][2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      u32x4 a[kSteps];
#pragma unroll
      for (int t = 0; t < kKLoads; ++t) {
        if (F8) decode16(kreg[i][t], scale_of(byte_of(ke[i])), a[(2 * t) % kSteps], a[(2 * t + 1) % kSteps]);
        else a[t % kSteps] = kreg[i][t];
      }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        s[nb][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < kSteps; ++t)
          s[nb][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(a[t]), qf[nb][t], s[nb][i], 0, 0, 0);
      }
      if (F8) __builtin_amdgcn_sched_barrier(0);  // one block's decoded keys in registers
    }
    if (more) load_k(j + 128, next);
    // rows of V that some row sees
    const int live[2] = {now[0] >= 0 ? end - j : 0, now[1] >= 0 ? end - j - 16 : 0};
    const bool masked = j + 32 > see_all || now[0] < 0 || now[1] < 0;
    u32x4 pb[NB];
    float alpha[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      if (masked) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int l = now[i] >= 0 ? lim[nb] - j - 16 * i - 4 * g : 0;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (e >= l) s[nb][i][e] = -INFINITY;
        }
      }
      float top = -INFINITY;
#pragma unroll
      for (int e = 0; e < 4; ++e) top = fmaxf(top, fmaxf(s[nb][0][e], s[nb][1][e]));
      const float m_new = fmaxf(m_run[nb], over_groups<true>(top) * c);
      const float mu = m_new == -INFINITY ? 0.f : m_new;
      alpha[nb] = __builtin_amdgcn_exp2f(m_run[nb] - mu);
      m_run[nb] = m_new;
      float pr[8], sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        pr[e] = __builtin_amdgcn_exp2f(fmaf(s[nb][e >> 2][e & 3], c, -mu));
        sum += pr[e];
      }
      l_run[nb] = fmaf(l_run[nb], alpha[nb], sum);
      pb[nb] = u32x4{pack_bf16x2(pr[0], pr[1]), pack_bf16x2(pr[2], pr[3]), pack_bf16x2(pr[4], pr[5]),
                     pack_bf16x2(pr[6], pr[7])};
    }
    // V into LDS, zero where there is no key
#pragma unroll
    for (int u = 0; u < kVLoads; ++u) {
      const int row = kVRows * u + vr;
      const bool ok = (row & 15) < live[kVRows * u < 16 ? 0 : 1];
      lds_u8* const to = mine + row * kPitch;
      const int ch = vd / 8, sw = swz_v<D>(row);
      const u32x4 none = u32x4{0, 0, 0, 0};
      if (F8) {
        u32x4 x, y;
        decode16(vreg[u], scale_of(byte_of(ve[u])), x, y);
        *reinterpret_cast<lds_u32x4*>(to + ((ch ^ sw) << 4)) = ok ? x : none;
        *reinterpret_cast<lds_u32x4*>(to + (((ch + 1) ^ sw) << 4)) = ok ? y : none;
      } else {
        *reinterpret_cast<lds_u32x4*>(to + ((ch ^ sw) << 4)) = ok ? vreg[u] : none;
      }
    }
    if (more) load_v(j + 128, next);
    asm volatile("" ::: "memory");  // the V rows are written before they are read
#pragma unroll
    for (int db = 0; db < kDB; ++db) {
      const lds_u8* const x = mine + (tr ^ (32 * db));
      const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)x);
      const i16x4 up = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(x + 16 * kPitch));
      const bf16x8 a = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, up, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nb][db][e] *= alpha[nb];
        o[nb][db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, as_bf16x8(pb[nb]), o[nb][db], 0, 0, 0);
      }
      if ((db & 3) == 3) __builtin_amdgcn_sched_barrier(0);  // not all of V^T in registers at once
    }
    asm volatile("" ::: "memory");  // and read before the next tile's are written
    now[0] = next[0];
    now[1] = next[1];
  }

  // The waves' sums, at the largest of their references, by way of LDS: O^T of lane
  // (n, g) is head-dims 16 db + 4 g .. + 3 of row 16 nb + n.
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    l_run[nb] = over_groups<false>(l_run[nb]);
    if (g == 0) {
      red_m[wave][16 * nb + n] = m_run[nb];
      red_l[wave][16 * nb + n] = l_run[nb];
    }
  }
  const int tid = 64 * wave + lane, qn = tid >> 4;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    __syncthreads();
    {
      float m = -INFINITY;
#pragma unroll
      for (int w = 0; w < 4; ++w) m = fmaxf(m, red_m[w][16 * nb + n]);
      const float f = __builtin_amdgcn_exp2f(m_run[nb] - (m == -INFINITY ? 0.f : m));
#pragma unroll
      for (int db = 0; db < kDB; ++db) {
        f32x4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = f == 0.f ? 0.f : o[nb][db][e] * f;
        *reinterpret_cast<lds_f32x4*>(s0 + ((wave * 16 + n) * (D / 4) + ((4 * db + g) ^ n)) * 16) = y;
      }
    }
    __syncthreads();
    // 16 threads a row, D / 64 times four head-dims each
    const int r = 16 * nb + qn;
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) m = fmaxf(m, red_m[w][r]);
    const float mu = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int w = 0; w < 4; ++w)  // (a wave whose scores are all NaN has no reference, but a sum that is NaN)
      l = fmaf(red_l[w][r], __builtin_amdgcn_exp2f(red_m[w][r] - mu), l);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int rr = min(r, rows - 1);
    const int64_t tok = of.query(rr), hd = of.head(rr);
    const int64_t row = row0 + tok * n_heads + hd;
    uint16_t* const out = p.out + (sp.q0 + tok) * p.os + ((int64_t)head * p.pk.group + hd) * p.oh;
    float* const part = unit.splits > 1 ? p.part + (unit.split * all_rows + row) * D : nullptr;
    f32x4 y[D / 64];
    bool bad = false;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      const int ch = 16 * i + (tid & 15);
      y[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < 4; ++w)
        y[i] += *reinterpret_cast<const lds_f32x4*>(s0 + ((w * 16 + qn) * (D / 4) + (ch ^ qn)) * 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) bad |= y[i][e] != y[i][e];
    }
    // (a wave has four rows, 16 lanes each)
    const uint64_t bads = __ballot(bad && l == l && r < rows);
    const bool again = ((bads >> (lane & 48)) & 0xffff) != 0;
    if (r < rows && !again) {
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        const int ch = 16 * i + (tid & 15);
        if (unit.splits == 1)
          *reinterpret_cast<u32x2*>(out + 4 * ch) =
              u32x2{pack_bf16x2(y[i][0] * inv, y[i][1] * inv), pack_bf16x2(y[i][2] * inv, y[i][3] * inv)};
        else
          *reinterpret_cast<f32x4*>(part + 4 * ch) = y[i];
      }
    }
    if (r < rows && (tid & 15) == 0) {
      if (unit.splits > 1)
        *reinterpret_cast<f32x2*>(p.part + p.n_split * all_rows * D + 2 * (unit.split * all_rows + row)) = f32x2{m, l};
      else if (p.lse != nullptr)
        p.lse[row] = l == 0.f ? -INFINITY : (m + __log2f(l)) * kLn2;
      if (p.n_split > 1 && unit.split == 0)
        reinterpret_cast<int32_t*>(p.part + p.n_split * all_rows * (D + 2))[row] = unit.splits;
    }
    for (int i = 0; i < 4; ++i) {
      if (((bads >> (16 * i)) & 0xffff) == 0) continue;
      const int which = 16 * nb + 4 * wave + i;
      const int64_t t = of.query(which), h = of.head(which);
      redo_paged_row<D, F8>(
          p.q + (sp.q0 + t) * p.qs + ((int64_t)head * p.pk.group + h) * p.qh, kx, vx, kex, vex, p.kp.sp, p.kp.ss,
          p.kp.ep, p.kp.es, p.tab.t + b * p.tab.ld, p.tab.pages, p.tab.shift, begin,
          max(min(seen(p, sp, of.query(which)), end) - begin, 0), c, __shfl(mu, 16 * i), __shfl(inv, 16 * i),
          p.out + (sp.q0 + t) * p.os + ((int64_t)head * p.pk.group + h) * p.oh,
          unit.splits > 1 ? p.part + (unit.split * all_rows + row0 + t * n_heads + h) * D : nullptr, lane);
    }
  }
}

template <int D, bool F8>
__global__ void __launch_bounds__(kThreads, D == 64 ? 3 : 2) chunk_kernel(ChunkArgs p) {
  using T = Tile<D>;
  constexpr int kSlot = 2 * T::kBytes;        // K and V of a step, in bf16
  constexpr int kRaw = F8 ? 64 * D : 0;       // K's codes of a step
  __shared__ __attribute__((aligned(1024))) uint8_t ring[2 * kSlot + kRaw];
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int li = lane & 31, hi = lane >> 5;
  const int head = blockIdx.x % p.pk.n_kv;
  const int item = (int)(blockIdx.x / p.pk.n_kv);
  const Unit unit = p.units > 0 ? unit_of_rank(p, item, lane) : unit_of_slot(p, item, lane);
  const Span sp = unit.sp;
  const int b = sp.seq - 1;
  const int rows = sp.nq * p.pk.group;
  const int r0 = sp.tile * kRows;
  if (r0 >= rows) return;

  const int r = r0 + 32 * wave + li;
  const bool real = r < rows;
  const Queries of(p, r0);
  const int last = seen(p, sp, of.query(min(kRows, rows - r0) - 1));
  // this split's steps of 64 keys; from here on keys count from its first
  const int all_steps = (last + 63) >> 6;
  // (in 32-bit floats, whose roundings are the same in each split of a row)
  auto begins = [&](int i) {
    return i == unit.splits ? all_steps : (int)((float)(all_steps * i) * __builtin_amdgcn_rcpf((float)unit.splits));
  };
  const int from = begins(unit.split);
  const int n_steps = begins(unit.split + 1) - from;
  if (rows <= 16) return few_rows<D, F8, 1>(p, unit, of, head, rows, from, n_steps, last, wave, lane, (lds_u8*)ring);
  if (rows <= 32) return few_rows<D, F8, 2>(p, unit, of, head, rows, from, n_steps, last, wave, lane, (lds_u8*)ring);
  const int end = 64 * n_steps;
  const int limit = min(max((real ? seen(p, sp, of.query(r - r0)) : last) - 64 * from, 0), end);
  const int n_plain = min(max(seen(p, sp, of.first) - 64 * from, 0), end) >> 6;  // seen whole by every row
  // keys that every row of the wave sees (its rows see more and more)
  const int wave_all = __builtin_amdgcn_readfirstlane(
      min(max((r0 + 32 * wave < rows ? seen(p, sp, of.query(32 * wave)) : last) - 64 * from, 0), end));
  const RowLoads<D> qrows =
      load_rows<D>(p.q + (int64_t)sp.q0 * p.qs + (int64_t)head * p.pk.group * p.qh, p.qs, p.qh, p.pk.group,
                   p.per_group, r0 + 32 * wave, rows, lane);
  Wave<D> w;

  // Places. Lane i: of step window + i, where this wave's 16 keys lie, and in the low bits,
  // as rows begin on 16 bytes, the blocks without a page (which are read from page 0).
  // Blocks past the sequence's last repeat it.
  const int last_block = max(sp.nk - 1, 0) >> 4, page_mask = (1 << p.tab.shift) - 1;
  constexpr int kBytes = F8 ? 1 : 2;
  const uint8_t* const kx = p.kp.x + kBytes * head * p.kp.sh;
  const uint8_t* const vx = p.vp.x + kBytes * head * p.kp.sh;  // (V lies as K does)
  int window = -64;
  uint64_t ats = 0, exp_ats = 0;
  auto lane_of = [](uint64_t x, int i) {
    const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)x, i), up = __builtin_amdgcn_readlane((uint32_t)(x >> 32), i);
    return (uint64_t)up << 32 | lo;
  };
  auto place = [&](int u) __attribute__((always_inline)) {
    if (u - window >= 64) {
      window = u;
      uint32_t bads = 0;
      int page = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int block = min(4 * (from + u + lane) + i, last_block);
        const int g = p.tab.t[b * p.tab.ld + (block >> (p.tab.shift - 4))];
        const bool ok = g >= 0 && g < p.tab.pages;
        bads |= ok ? 0u : 1u << i;
        if (i == wave) page = ok ? g : 0;
      }
      const int row = (16 * min(4 * (from + u + lane) + wave, last_block)) & page_mask;
      ats = (uint64_t)(kBytes * (page * p.kp.sp + row * p.kp.ss)) | bads;
      if (F8) exp_ats = (uint64_t)(page * p.kp.ep + row * p.kp.es);
    }
    Place x;
    const uint64_t at = lane_of(ats, u - window);
    x.bad = (uint32_t)at & 15u;
    x.at = (int64_t)(at & ~(uint64_t)15);
    x.exp = F8 ? (int64_t)lane_of(exp_ats, u - window) : 0;
    x.rows = sp.nk - 16 * min(4 * (from + u) + wave, last_block);
    return x;
  };
  lds_u8* const s0 = (lds_u8*)ring;
  // bf16 rows go into LDS as they lie. This wave's loads of a step's K or V, a segment is
  // 1 KB of its 16 rows; `clamp`: rows past the sequence's last key read that key again.
  // e4m3: K's codes, each lane's 16 where it reads them again.
  constexpr int kSegs = F8 ? D / 64 : T::kSegs;
  struct Src {
    const char* base;
    uint32_t off[kSegs];
  };
  auto src_of = [&](bool is_v, const Place& y, bool clamp) __attribute__((always_inline)) {
    Src r;
    r.base = reinterpret_cast<const char*>(is_v ? vx : kx) + y.at;
    constexpr int kChunks = kBytes * D / 16, kSegRows = 64 / kChunks;
#pragma unroll
    for (int s = 0; s < kSegs; ++s) {
      const int row = s * kSegRows + lane / kChunks, pos = lane % kChunks;
      const uint32_t src = (uint32_t)(clamp ? min(row, y.rows - 1) : row);
      const int swz = F8 ? 0 : is_v ? swz_tr<D>(row) : swz_row<D>(row);
      r.off[s] = src * (uint32_t)(kBytes * p.kp.ss) + ((pos ^ swz) << 4);
    }
    return r;
  };
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(s0 + (F8 ? 2 * kSlot : 0) + kSegs * 1024 * wave));
  auto issue = [&](const Src& x, int s, uint32_t to) { dma16_m0(x.base, x.off[s], to + s * 1024); };
  // e4m3 rows are decoded (times the row's power of two: exact) on their way into the
  // slots, once for the workgroup's 128 rows: 16 codes of a lane, kCodeLanes lanes a row. V's
  // codes wait in registers while they come, K's in the wave's part of LDS, as there are
  // not registers for both.
  constexpr int kCodeLanes = D / 16, kCodes = kCodeLanes / 4;
  struct Exponents {
    Exponent of[kCodes > 0 ? kCodes : 1];
  };
  struct Codes {
    u32x4 x[kCodes > 0 ? kCodes : 1];
    Exponents e;
  };
  auto code_row = [&](int s) { return s * (64 / kCodeLanes) + lane / kCodeLanes; };
  auto exponents = [&](const uint8_t* x, const Place& y, bool clamp) __attribute__((always_inline)) {
    Exponents r;
#pragma unroll
    for (int s = 0; s < kCodes; ++s) {
      const int row = clamp ? min(code_row(s), y.rows - 1) : code_row(s);
      r.of[s] = exponent_at(x + y.exp + head * p.kp.eh, (uint32_t)row * (uint32_t)p.kp.es);
    }
    return r;
  };
  auto fetch = [&](const Place& y, bool clamp) __attribute__((always_inline)) {
    Codes r;
#pragma unroll
    for (int s = 0; s < kCodes; ++s) {
      const uint32_t src = (uint32_t)(clamp ? min(code_row(s), y.rows - 1) : code_row(s));
      r.x[s] = *reinterpret_cast<const u32x4*>(vx + y.at + (src * (uint32_t)p.kp.ss + 16 * (lane % kCodeLanes)));
    }
    r.e = exponents(p.vp.e, y, clamp);
    return r;
  };
  auto put = [&](u32x4 x, const Exponent& e, int s, uint32_t slot, bool is_v) __attribute__((always_inline)) {
    u32x4 a, c;
    decode16(x, scale_of(byte_of(e)), a, c);
    const int row = 16 * wave + code_row(s), ch = 2 * (lane % kCodeLanes);
    const int swz = is_v ? swz_tr<D>(row) : swz_row<D>(row);
    lds_u8* const to = s0 + slot + (is_v ? T::kBytes : 0) + row * T::kPitch;
    *reinterpret_cast<lds_u32x4*>(to + ((ch ^ swz) << 4)) = a;
    *reinterpret_cast<lds_u32x4*>(to + (((ch + 1) ^ swz) << 4)) = c;
  };
  auto put_v = [&](const Codes& x, int s, uint32_t slot) __attribute__((always_inline)) {
    put(x.x[s], x.e.of[s], s, slot, true);
  };
  // (K's exponents are asked for behind its codes, and loads arrive in order: once the
  // former are here so are the latter)
  auto put_k = [&](Exponents& e, int s, uint32_t slot) __attribute__((always_inline)) {
    asm volatile("" : "+v"(e.of[s].word) : : "memory");
    const u32x4 x = *reinterpret_cast<const lds_u32x4*>(s0 + 2 * kSlot + 1024 * (kSegs * wave + s) + 16 * lane);
    put(x, e.of[s], s, slot, false);
  };

  Frags<D> f;
#pragma unroll
  for (int s = 0; s < T::kK; ++s)
    f.k[s] = (uint32_t)(li * T::kPitch + (((2 * s + hi) ^ swz_row<D>(li)) << 4));
#pragma unroll
  for (int t = 0; t < T::kT; ++t) f.v[t] = T::kBytes + tr_offset<D>(lane, t, 0, swz_tr<D>);
#pragma unroll
  for (int t = 0; t < T::kT; ++t) w.o[t] = zero16();
  w.m_run = -INFINITY;
  w.l_run = w.mu = w.first_sum = 0.f;
  w.alpha = 1.f;
  w.have_ref = false;
  const float c = p.scale_log2;

  // The walk of the packed forward: iteration u multiplies K of step u + 1 and V of step
  // u, and brings K of step u + 2 (over K of step u) and V of step u + 1 into LDS. bf16:
  // as loads that have an iteration to arrive. e4m3: as codes that were asked for an
  // iteration before, which it asks for again, a step on.
  constexpr int kSub = 32 * T::kPitch;
  auto sync = [&]() {
    if (F8) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the rows that it put into LDS
    else VEDA_WAIT_VM(0);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  f32x16 sa, sb;
  u32x4 pa[2], pb[2];
  Place p1, p2;   // of steps u + 1 and u + 2 (e4m3)
  Codes vc;       // e4m3: V of step u + 1
  Exponents ke;   // e4m3: of K of step u + 2
  constexpr int kAhead = F8 ? 3 : 2;  // the step that K is asked for
  // Part j of what an iteration brings. e4m3: what is there goes into the slots before
  // anything is asked for again: V's loads are waited for by their number, and loads into
  // LDS, which hipcc does not count, would be waited for with them.
  auto bring = [&](int j, const Src& ks, const Src& vs, const Place& next, bool clamp, uint32_t cur, uint32_t nxt)
      __attribute__((always_inline)) {
    if constexpr (F8) {
      if (j < kCodes) put_k(ke, j, cur);
      else if (j < 2 * kCodes) put_v(vc, j - kCodes, nxt);
      else if (j == 2 * kCodes) {
#pragma unroll
        for (int s = 0; s < kSegs; ++s) issue(ks, s, lds0);
        ke = exponents(p.kp.e, next, clamp);
      } else if (j == 2 * kCodes + 1) {
        vc = fetch(p2, clamp);
      }
    } else {
      if (j < kSegs) issue(ks, j, lds0 + cur);
      else if (j < 2 * kSegs) issue(vs, j - kSegs, lds0 + nxt + T::kBytes);
    }
  };
  auto iter = [&](auto masked, int u, uint32_t cur, uint32_t nxt) __attribute__((always_inline)) {
    // MASKED: step u + 1 holds keys that some row does not see, or a step that is asked
    // for may be past the last
    constexpr bool MASKED = decltype(masked)::value;
    const Place next = place(MASKED ? min(u + kAhead, n_steps - 1) : u + kAhead);
    const uint32_t bad = p1.bad;
    const Src ks = src_of(false, next, MASKED);
    Src vs;
    if constexpr (!F8) vs = src_of(true, p1, MASKED);
    sync();
    Next<D> ahead;
    constexpr int kGive = F8 ? kNoNext : kReadNext, kTake = F8 ? kNoNext : kTakeNext;
    stage<D, true, kSmSecond, true, kGive>(s0 + nxt, s0 + cur, f, c, sa, sb, pb, pa, w,
                                           [&](int j) { bring(j, ks, vs, next, MASKED, cur, nxt); }, &ahead);
    if (MASKED && 64 * (u + 1) + 32 > wave_all) mask_scores(sa, limit - 64 * (u + 1), hi);
    if (__builtin_expect((bad & 3) != 0, 0)) mask_blocks(sa, bad);
    stage<D, true, kSmFirst, true, kTake>(s0 + nxt + kSub, s0 + cur + kSub, f, c, sb, sa, pa, pb, w, NoHook{},
                                          &ahead);
    if (MASKED && 64 * (u + 1) + 64 > wave_all) mask_scores(sb, limit - 64 * (u + 1) - 32, hi);
    if (__builtin_expect((bad & 12) != 0, 0)) mask_blocks(sb, bad >> 2);
    p1 = F8 ? p2 : next;
    p2 = next;
  };
  const bool idle = r0 + 32 * wave >= rows;  // without rows, in a sequence's last tile: only brings keys and values
  if (n_steps > 0) {
    const Place p0 = place(0);
    p1 = place(min(1, n_steps - 1));
    p2 = place(min(2, n_steps - 1));
    const Src k0 = src_of(false, p0, true);
#pragma unroll
    for (int s = 0; s < kSegs; ++s) issue(k0, s, lds0);
    if constexpr (F8) {
      ke = exponents(p.kp.e, p0, true);
      vc = fetch(p0, true);
#pragma unroll
      for (int s = 0; s < kCodes; ++s) {
        put_k(ke, s, 0);
        put_v(vc, s, 0);
      }
      const Src k1 = src_of(false, p1, true);
#pragma unroll
      for (int s = 0; s < kSegs; ++s) issue(k1, s, lds0);
      ke = exponents(p.kp.e, p1, true);
      vc = fetch(p1, true);
    } else {
      const Src v0 = src_of(true, p0, true);
#pragma unroll
      for (int s = 0; s < kSegs; ++s) issue(v0, s, lds0 + T::kBytes);
    }
    // Q by way of slot 1, which K of step 1 comes into after the barrier
    frags_of_rows<D>(qrows, s0 + kSlot + wave * 32 * T::kPitch, lane, w.qf);
#pragma unroll
    for (int s = 0; s < T::kK; ++s) asm volatile("" : : "v"(w.qf[s]));
    sync();
    if constexpr (F8) {
#pragma unroll
      for (int s = 0; s < kCodes; ++s) put_k(ke, s, kSlot);
      const Src k2 = src_of(false, p2, true);
#pragma unroll
      for (int s = 0; s < kSegs; ++s) issue(k2, s, lds0);
      ke = exponents(p.kp.e, p2, true);
    } else if (n_steps > 1) {
      const Src k1 = src_of(false, p1, true);
#pragma unroll
      for (int s = 0; s < kSegs; ++s) issue(k1, s, lds0 + kSlot);
    }
    if (idle) {
#pragma unroll 1
      for (int u = 0; u + 1 < n_steps; ++u) {
        const uint32_t cur = (u & 1) * kSlot, nxt = kSlot - cur;
        const Place next = place(min(u + kAhead, n_steps - 1));
        const Src ks = src_of(false, next, true);
        Src vs;
        if constexpr (!F8) vs = src_of(true, p1, true);
        sync();
#pragma unroll
        for (int j = 0; j < 8; ++j) bring(j, ks, vs, next, true, cur, nxt);
        p1 = F8 ? p2 : next;
        p2 = next;
      }
      sync();
    } else {
      stage<D, true, kNoSm, false>(s0, s0, f, c, sa, sb, pa, pb, w, NoHook{});
      stage<D, true, kNoSm, false>(s0 + kSub, s0, f, c, sb, sa, pa, pb, w, NoHook{});
      if (n_plain == 0) {
        mask_scores(sa, limit, hi);
        mask_scores(sb, limit - 32, hi);
      }
      if (p0.bad != 0) {
        mask_blocks(sa, p0.bad);
        mask_blocks(sb, p0.bad >> 2);
      }
      first_reference<D>(sa, sb, c, w);
      stage<D, false, kSmFirst, false>(s0, s0, f, c, sb, sa, pa, pb, w, NoHook{});
      int u = 0;
      for (; u + kAhead + 1 < n_plain; u += 2) {
        iter(std::false_type{}, u, 0, kSlot);
        iter(std::false_type{}, u + 1, kSlot, 0);
      }
#pragma unroll 1
      for (; u + 1 < n_steps; ++u) {
        const uint32_t to = (u & 1) * kSlot;
        iter(std::true_type{}, u, to, kSlot - to);
      }
      const lds_u8* const cur = s0 + ((n_steps - 1) & 1) * kSlot;
      sync();
      stage<D, false, kSmSecond, true>(s0, cur, f, c, sb, sb, pb, pa, w, NoHook{});
      stage<D, false, kNoSm, true>(s0, cur + kSub, f, c, sa, sb, pa, pb, w, NoHook{});
    }
    if (F8) VEDA_WAIT_VM(0);  // codes that no step takes are on their way into LDS, which is another's after the end
  }
  if (p.n_split > 1 && unit.split == 0 && real && hi == 0) {
    const int64_t n_heads = (int64_t)p.pk.n_kv * p.pk.group, all_rows = p.pk.q_rows * n_heads;
    const int64_t row = (sp.q0 + of.query(r - r0)) * n_heads + (int64_t)head * p.pk.group + of.head(r - r0);
    reinterpret_cast<int32_t*>(p.part + p.n_split * all_rows * (D + 2))[row] = unit.splits;
  }
  leave_rows<D>(p, w, sp, unit.split, unit.splits, head, r0, rows, limit, wave, lane, s0,
                [&](int64_t tok, int64_t hd, int lim, float mu, float inv, float* part) {
                  redo_paged_row<D, F8>(p.q + tok * p.qs + hd * p.qh, kx, vx, p.kp.e + head * p.kp.eh,
                                        p.vp.e + head * p.vp.eh, p.kp.sp, p.kp.ss, p.kp.ep, p.kp.es,
                                        p.tab.t + b * p.tab.ld, p.tab.pages, p.tab.shift, 64 * from, lim, c,
                                        mu, inv, p.out + tok * p.os + hd * p.oh, part, lane);
                });
}

// The splits of a row joined, where it has more than one: D / 4 threads a row, four
// head-dims each. EARLY: the first splits are asked for before their number is known
// (what lies there is the workspace's, and not used), which saves a load's time where
// rows are few and costs reads where they are many.
template <int D, bool EARLY>
__global__ void __launch_bounds__(256) chunk_merge_kernel(ChunkArgs p) {
  constexpr int kEarly = EARLY ? 8 : 1;
  const int64_t n_heads = (int64_t)p.pk.n_kv * p.pk.group, all_rows = p.pk.q_rows * n_heads;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = i / (D / 4);
  const int d = 4 * (int)(i % (D / 4));
  if (row >= all_rows) return;
  const f32x2* ml = reinterpret_cast<const f32x2*>(p.part + p.n_split * all_rows * D) + row;
  const float* part = p.part + row * D + d;
  const int found = reinterpret_cast<const int32_t*>(p.part + p.n_split * all_rows * (D + 2))[row];
  f32x2 x[kEarly];
  f32x4 y[kEarly];
  if (EARLY) {
#pragma unroll
    for (int s = 0; s < kEarly; ++s) {
      const int64_t at = min(s, p.n_split - 1) * all_rows;
      x[s] = ml[at];
      y[s] = *reinterpret_cast<const f32x4*>(part + at * D);
    }
  }
  const int n = min(found, p.n_split);
  if (n <= 1) return;
  float m = -INFINITY;
  if (EARLY) {
#pragma unroll
    for (int s = 0; s < kEarly; ++s) m = s < n ? fmaxf(m, x[s][0]) : m;
  }
#pragma unroll 4
  for (int s = EARLY ? kEarly : 0; s < n; ++s) m = fmaxf(m, ml[s * all_rows][0]);
  const float mu = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
  auto add = [&](f32x2 a, f32x4 b) {
    const float w = __builtin_amdgcn_exp2f(a[0] - mu);
    l = fmaf(w, a[1], l);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = w == 0.f ? o[e] : fmaf(w, b[e], o[e]);
  };
  if (EARLY) {
#pragma unroll
    for (int s = 0; s < kEarly; ++s)
      if (s < n) add(x[s], y[s]);
  }
#pragma unroll 4
  for (int s = EARLY ? kEarly : 0; s < n; ++s)
    add(ml[s * all_rows], *reinterpret_cast<const f32x4*>(part + s * all_rows * D));
  const float inv = l == 0.f ? 0.f : 1.f / l;
  *reinterpret_cast<u32x2*>(p.out + (row / n_heads) * p.os + (row % n_heads) * p.oh + d) =
      u32x2{pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv)};
  if (d == 0 && p.lse != nullptr) p.lse[row] = l == 0.f ? -INFINITY : (m + __log2f(l)) * kLn2;
}

}  // namespace
}  // namespace veda

using namespace veda;

extern "C" int veda_chunk_fwd(const void* q, int64_t q_stride_s, int64_t q_stride_h, int64_t q_rows,
                              int64_t n_heads, int64_t n_kv_heads, int64_t head_dim, const int32_t* cu,
                              int64_t n_seq, const void* k_pages, const void* v_pages, int64_t stride_p,
                              int64_t stride_s, int64_t stride_h, int e4m3, const uint8_t* k_exp,
                              const uint8_t* v_exp, int64_t exp_stride_p, int64_t exp_stride_s,
                              int64_t exp_stride_h, int64_t n_pages, int64_t page, const int32_t* table,
                              int64_t table_ld, int64_t width, const int32_t* lengths, int causal, float scale,
                              int64_t n_split, int64_t units, void* out, int64_t o_stride_s,
                              int64_t o_stride_h, float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* const what = "chunk_fwd";
  ChunkArgs p{};
  p.kp = pages_of(k_pages, stride_p, stride_s, stride_h, k_exp, exp_stride_p, exp_stride_s, exp_stride_h);
  p.vp = pages_of(v_pages, stride_p, stride_s, stride_h, v_exp, exp_stride_p, exp_stride_s, exp_stride_h);
  if (int rc = check_cache(what, head_dim, n_kv_heads, n_pages, page, width, e4m3, p.kp, p.vp)) return rc;
  VEDA_REQUIRE(n_heads > 0 && n_heads % n_kv_heads == 0,
               "%s: %lld query heads are no multiple of %lld key heads", what, (long long)n_heads,
               (long long)n_kv_heads);
  VEDA_REQUIRE(n_heads / n_kv_heads <= kMaxGroup, "%s: at most %lld query heads to a key head, got %lld", what,
               (long long)kMaxGroup, (long long)(n_heads / n_kv_heads));
  VEDA_REQUIRE(q_rows >= 0 && n_seq >= 0, "%s: negative size", what);
  VEDA_REQUIRE(q_rows * n_heads <= 0x7fffff00 && n_seq < (1 << 20),
               "%s: q_rows x heads past 2^31 - 256, or 2^20 sequences", what);
  VEDA_REQUIRE(width * page <= 0x7fff0000, "%s: a table row holds nearly 2^31 keys", what);
  // a page's rows are addressed with 32-bit byte offsets
  VEDA_REQUIRE(stride_s >= 0 && exp_stride_s >= 0 && stride_s < (1 << 22) && exp_stride_s < (1 << 22),
               "%s: row stride of the cache negative or too large", what);
  VEDA_REQUIRE(scale > 0.f && scale < INFINITY, "%s: scale must be positive and finite", what);
  VEDA_REQUIRE(rows16(q, q_stride_s, q_stride_h) && rows16(out, o_stride_s, o_stride_h),
               "%s: q and out rows must be 16-byte aligned", what);
  VEDA_REQUIRE(n_split >= 1 && n_split <= 64, "%s: n_split %lld outside [1, 64]", what, (long long)n_split);
  VEDA_REQUIRE(units >= 1 && units <= (1 << 20), "%s: units %lld outside [1, 2^20]", what, (long long)units);
  if (q_rows == 0) return VEDA_OK;
  const int64_t group = n_heads / n_kv_heads, slots = slots_of(q_rows, group, n_seq);
  const bool by_rank = n_seq <= kRankedSeqs && slots < (1 << 20);
  // (a launch holds less than 2^32 threads)
  const int64_t items = by_rank ? slots + (n_split > 1 ? units : 0) : slots * n_split;
  VEDA_REQUIRE(items * n_kv_heads < (1 << 24) && (n_split == 1 || q_rows * n_heads < (1 << 27)),
               "%s: too many rows for one launch", what);
  const int64_t need = n_split == 1 ? 0 : q_rows * n_heads * (n_split * (head_dim + 2) + 1) * 4;
  VEDA_REQUIRE(need == 0 || (workspace != nullptr && rows16(workspace, 0, 0) && workspace_bytes >= need),
               "%s: workspace needs %lld bytes (16-byte aligned), got %lld", what, (long long)need,
               (long long)workspace_bytes);
  p.pk = Packing{cu, cu, (int32_t)n_seq, (int32_t)q_rows, (int32_t)q_rows, (int32_t)n_kv_heads, (int32_t)group,
                 causal ? 1 : 0, 0, 0};
  p.q = static_cast<const uint16_t*>(q);
  p.qs = q_stride_s; p.qh = q_stride_h;
  p.tab = table_of(table, table_ld, width, n_pages, page);
  p.lengths = lengths;
  p.out = static_cast<uint16_t*>(out);
  p.os = o_stride_s; p.oh = o_stride_h;
  p.lse = lse;
  p.part = static_cast<float*>(workspace);
  p.scale_log2 = scale * 1.4426950408889634f;
  p.n_split = (int32_t)n_split;
  p.per_group = per_group_of((uint32_t)group);
  p.n_slots = (int32_t)slots;
  p.units = by_rank ? (int32_t)units : 0;
  p.resident = (int32_t)((head_dim == 128 ? 512 : 768) / n_kv_heads);
  if (p.resident == 0) p.resident = 1;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const unsigned grid = (unsigned)(items * n_kv_heads);
  if (head_dim == 128) {
    if (e4m3) chunk_kernel<128, true><<<grid, kThreads, 0, s>>>(p);
    else chunk_kernel<128, false><<<grid, kThreads, 0, s>>>(p);
  } else {
    if (e4m3) chunk_kernel<64, true><<<grid, kThreads, 0, s>>>(p);
    else chunk_kernel<64, false><<<grid, kThreads, 0, s>>>(p);
  }
  if (n_split > 1) {
    if (int rc = check_launch(what)) return rc;
    const unsigned join = (unsigned)((q_rows * n_heads * (head_dim / 4) + 255) / 256);
    const bool early = q_rows * n_heads <= kEarlyRows;
    if (head_dim == 128 && early) chunk_merge_kernel<128, true><<<join, 256, 0, s>>>(p);
    else if (head_dim == 128) chunk_merge_kernel<128, false><<<join, 256, 0, s>>>(p);
    else if (early) chunk_merge_kernel<64, true><<<join, 256, 0, s>>>(p);
    else chunk_merge_kernel<64, false><<<join, 256, 0, s>>>(p);
  }
  return check_launch(what);
}
