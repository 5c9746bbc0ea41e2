// A paged key-value cache for gfx950: rows written as they come, read back, and
// the attention of one new token of every sequence over them.
//
// The cache holds pages of `page` rows (a power of two, 16 to 256) of every key
// head, in bf16 or in e4m3 with one power of two for a row: a row x is held as
// codes c and an exponent byte b with x = c 2^(b - 127), b the least that
// brings the row's largest finite magnitude to 448 or less. With a power of two
// the scaling rounds nothing: a code is the row's value rounded once, to e4m3's
// three bits, and its bf16 value is exact (a magnitude that rounds to 2^128
// reads back as infinity). A NaN or an infinity is held as NaN.
//
// Position i of sequence b lies in page table[b][i / page], row i % page. A
// page number outside the cache, or a position past the table, is no row: it is
// not written, reads as zeros and draws no weight.
#include <type_traits>

#include "veda_pipeline.h"

namespace veda {
namespace {

constexpr float kLn2 = 0.6931471805599453f;

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// One of the cache's two tensors. Strides in elements: page, row, head.
struct Pages {
  uint8_t* x;
  int64_t sp, ss, sh;
  uint8_t* e;  // exponent bytes (e4m3), or NULL
  int64_t ep, es, eh;
};

struct Table {
  const int32_t* t;
  int64_t ld;
  int32_t width;   // pages of a sequence at most
  int32_t pages;   // pages of the cache
  int32_t shift;   // log2 of the page's rows
};

// The page of position `pos` of sequence b, or -1.
__device__ __forceinline__ int page_of(const Table& t, int b, int64_t pos) {
  const int64_t i = pos >> t.shift;
  if (pos < 0 || i >= t.width) return -1;
  const int g = t.t[b * t.ld + i];
  return g >= 0 && g < t.pages ? g : -1;
}

// The sequence whose rows [cu[b], cu[b + 1]) hold row r, or -1; by all lanes of
// a wave for one r, 64 offsets a round.
__device__ __forceinline__ int seq_of_row(const int32_t* cu, int n_seq, int r, int lane) {
  int lo = 0, count = n_seq + 1;  // the last i in [0, n_seq] with cu[i] <= r
  int32_t first = 0;
  while (count > 1) {
    const int stride = (count + 63) >> 6;
    const int i = lo + lane * stride;
    const bool in = i < lo + count;
    const int32_t c = cu[in ? i : lo];
    const uint64_t below = __ballot(in && c <= r);
    const int hits = (int)__builtin_popcountll(below);
    if (hits == 0) return -1;
    const int next = lo + (hits - 1) * stride;
    count = min(stride, lo + count - next);
    lo = next;
    first = __shfl(c, hits - 1);
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  return lo < n_seq && first <= r ? lo : -1;
}

// Two e4m3 codes of `word` (the low or the high pair), times the power of two
// whose biased exponent is `byte`, as bf16: exact but for subnormal results.
template <bool HI>
__device__ __forceinline__ uint32_t decode2(uint32_t word, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, scale, HI));
}
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

// Sixteen codes as sixteen bf16.
__device__ __forceinline__ void decode16(u32x4 w, float scale, u32x4& a, u32x4& b) {
  a = u32x4{decode2<false>(w[0], scale), decode2<true>(w[0], scale), decode2<false>(w[1], scale),
            decode2<true>(w[1], scale)};
  b = u32x4{decode2<false>(w[2], scale), decode2<true>(w[2], scale), decode2<false>(w[3], scale),
            decode2<true>(w[3], scale)};
}

// ---------------------------------------------------------------------------
// Writing. A wave takes one token: D / 8 lanes a row, the rows of all key heads
// of K, then of V.

struct AppendArgs {
  const uint16_t* k;
  const uint16_t* v;
  int64_t ks, kh, vs, vh;
  Pages kp, vp;
  Table tab;
  const int32_t* cu;
  const int32_t* start;
  int32_t n_seq, rows, n_kv;
};

// The row's eight values of a lane as e4m3 codes, and its exponent byte.
template <int LANES>
__device__ __forceinline__ u32x2 encode8(u32x4 x, uint32_t& byte) {
  // largest finite magnitude: bf16 magnitudes order as integers
  uint32_t top = 0;
  bool odd = false;  // a NaN or an infinity
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    const uint32_t lo = x[m] & 0x7fffu, up = (x[m] >> 16) & 0x7fffu;
    odd |= lo >= 0x7f80u || up >= 0x7f80u;
    top = max(top, max(lo < 0x7f80u ? lo : 0u, up < 0x7f80u ? up : 0u));
  }
#pragma unroll
  for (int off = LANES / 2; off >= 1; off >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off));
  // 448 = 1.75 2^8: the exponent less 8, one more where the mantissa is past 1.75
  const int e = (int)(top >> 7) - 8 + ((top & 0x7fu) > 0x60u ? 1 : 0);
  byte = (uint32_t)max(e, 0);
  const float s = __uint_as_float((254u - byte) << 23);  // 2^(127 - byte)
  u32x2 w;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float f[4];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      f[2 * m] = bf16_to_f32(x[2 * h + m] & 0xffffu) * s;
      f[2 * m + 1] = bf16_to_f32(x[2 * h + m] >> 16) * s;
    }
    int c = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
    w[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], c, true);
    if (odd) {
#pragma unroll
      for (int m = 0; m < 4; ++m)
        if (!(fabsf(f[m]) < INFINITY)) w[h] |= 0x7fu << (8 * m);
    }
  }
  return w;
}

// Bound by memory where there are rows enough (4,096 rows of 8 key heads in bf16:
// 9.0 us, 3.7 TB/s), by its start at a row for each of 32 sequences (7.4 us).
template <int D, bool F8>
__global__ void __launch_bounds__(256) append_kernel(AppendArgs p) {
  constexpr int kLanes = D / 8, kRowsAtOnce = 64 / kLanes;
  const int lane = threadIdx.x & 63;
  const int64_t r64 = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r64 >= p.rows) return;
  const int r = __builtin_amdgcn_readfirstlane((int)r64);
  const int b = seq_of_row(p.cu, p.n_seq, r, lane);
  if (b < 0) return;
  const int64_t pos = (int64_t)p.start[b] + (r - p.cu[b]);
  const int page = page_of(p.tab, b, pos);
  if (page < 0) return;
  const int64_t at = pos & ((1 << p.tab.shift) - 1);
  const int sub = lane / kLanes, d = 8 * (lane % kLanes);
  for (int i = sub; i < 2 * p.n_kv; i += kRowsAtOnce) {
    const bool is_v = i >= p.n_kv;
    const int h = is_v ? i - p.n_kv : i;
    const u32x4 x = is_v ? ld16(p.v + r * p.vs + h * p.vh + d) : ld16(p.k + r * p.ks + h * p.kh + d);
    const Pages& to = is_v ? p.vp : p.kp;
    const int64_t off = page * to.sp + at * to.ss + h * to.sh + d;
    if (F8) {
      uint32_t byte;
      const u32x2 w = encode8<kLanes>(x, byte);
      *reinterpret_cast<u32x2*>(to.x + off) = w;
      if (d == 0) to.e[page * to.ep + at * to.es + h * to.eh] = (uint8_t)byte;
    } else {
      *reinterpret_cast<u32x4*>(to.x + 2 * off) = x;
    }
  }
}

// ---------------------------------------------------------------------------
// Reading back. A wave takes one row of the packed result, as above. Bound by
// memory (52,769 rows of 8 key heads in bf16: 432 MB in 77.8 us, 5.6 TB/s).

struct GatherArgs {
  Pages kp, vp;
  Table tab;
  const int32_t* cu;
  int32_t n_seq, rows, n_kv;
  uint16_t* k;
  uint16_t* v;
};

template <int D, bool F8>
__global__ void __launch_bounds__(256) gather_cache_kernel(GatherArgs p) {
  constexpr int kLanes = D / 8, kRowsAtOnce = 64 / kLanes;
  const int lane = threadIdx.x & 63;
  const int64_t r64 = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r64 >= p.rows) return;
  const int r = __builtin_amdgcn_readfirstlane((int)r64);
  const int b = seq_of_row(p.cu, p.n_seq, r, lane);
  int page = -1;
  int64_t at = 0;
  if (b >= 0) {
    const int64_t pos = r - p.cu[b];
    page = page_of(p.tab, b, pos);
    at = pos & ((1 << p.tab.shift) - 1);
  }
  const int sub = lane / kLanes, d = 8 * (lane % kLanes);
  for (int i = sub; i < 2 * p.n_kv; i += kRowsAtOnce) {
    const bool is_v = i >= p.n_kv;
    const int h = is_v ? i - p.n_kv : i;
    u32x4 x = u32x4{0, 0, 0, 0};
    if (page >= 0) {
      const Pages& from = is_v ? p.vp : p.kp;
      const int64_t off = page * from.sp + at * from.ss + h * from.sh + d;
      if (F8) {
        const u32x2 w = *reinterpret_cast<const u32x2*>(from.x + off);
        const float s = scale_of(from.e[page * from.ep + at * from.es + h * from.eh]);
        x = u32x4{decode2<false>(w[0], s), decode2<true>(w[0], s), decode2<false>(w[1], s),
                  decode2<true>(w[1], s)};
      } else {
        x = *reinterpret_cast<const u32x4*>(from.x + 2 * off);
      }
    }
    uint16_t* to = (is_v ? p.v : p.k) + ((int64_t)r * p.n_kv + h) * D + d;
    *reinterpret_cast<u32x4*>(to) = x;
  }
}

// ---------------------------------------------------------------------------
// One new token of every sequence. Workgroup = (sequence, key head, up to 16 of
// its query heads, `chunk` keys of the sequence), W waves (4, or 8 where a whole
// sequence is one chunk); each wave has tiles of 32 keys of its own, every W-th
// of the chunk, and nothing waits for another wave until the end. With v_mfma_f32_16x16x32_bf16 (A[i][k] in lane
// i + 16 (k / 8) and B[k][j] in lane j + 16 (k / 8), element k % 8; D[i][j] in
// lane j + 16 (i / 4), element i % 4) the scores are S^T = K Q^T: lane n + 16 g
// holds keys 4 g .. + 3 of both 16-key blocks of query head n, which are the
// B operand of O^T += V^T P^T when k index e of lane group g stands for key
// 16 (e / 4) + 4 g + e % 4. K goes from memory straight into the A operand; V
// passes through the wave's own LDS, to be read transposed.
//
// Bound by the cache's bytes: a tile's K is asked for once the last tile's
// scores are formed, its V once the last one's is in LDS, so a wave has a tile in
// flight at all times in the registers of one. The chunk's page numbers are in
// two registers from the start (lane i: pages i and 64 + i of the chunk).

struct TokenArgs {
  const uint16_t* q;
  int64_t qs, qh;
  Pages kp, vp;
  Table tab;
  const int32_t* lengths;
  int32_t n_kv, group, chunk, n_split;
  float scale_log2;
  uint16_t* out;
  int64_t os, oh;
  float* lse;   // [B, H] or NULL
  float* part;  // [B, H, n_split, D + 4]: O, then the reference (log2) and the sum
};

template <int D>
__device__ __forceinline__ int swz_v(int r) {
  return D == 128 ? ((r & 3) << 2) | ((((r >> 2) ^ (r >> 3)) & 1) << 1) | ((r >> 3) & 1)
                  : (((r >> 1) & 1) << 2) | (((r >> 2) & 1) << 1);
}

// Maximum and sum over the four lane groups of a query head (lanes n + 16 g).
template <bool MAX>
__device__ __forceinline__ float over_groups(float v) {
  const float w = __uint_as_float(__builtin_amdgcn_ds_swizzle(__float_as_uint(v), 0x401F));
  v = MAX ? fmaxf(v, w) : v + w;
  return MAX ? half_swap_max(v) : half_swap_sum(v);
}

__device__ __forceinline__ int length_of(const TokenArgs& p, int b) {
  return min(max(p.lengths[b], 0), p.tab.width << p.tab.shift);
}

// Bound by memory: four tokens over 386,613 positions in bf16, 8 key heads, 279 us,
// 5.7 TB/s; 64 over 73,366 in e4m3 33.8 us, 4.5 TB/s, the start and the uneven end
// of a short kernel among it; one over 1,500, 5.4 us of latency.
template <int D, bool F8, int W>
__global__ void __launch_bounds__(64 * W, W == 4 ? 3 : 2) token_kernel(TokenArgs p) {
  constexpr int kStride = 32 * W;             // keys of a round of the waves
  constexpr int kPitch = 2 * D;               // a V row in LDS, bf16
  constexpr int kTileBytes = 32 * kPitch;
  constexpr int kPer = F8 ? 16 : 8;           // elements of a 16-byte load
  constexpr int kBytes = F8 ? 1 : 2;
  constexpr int kKLoads = D / (4 * kPer);     // of a lane, for a K row
  constexpr int kSteps = D / 32;              // k-steps of a score
  constexpr int kLanes = D / kPer;            // lanes of a V row
  constexpr int kVRows = 64 / kLanes;         // V rows of a load (at most 16: one block of keys)
  constexpr int kVLoads = 32 / kVRows;
  constexpr int kDB = D / 16;
  typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
  typedef __attribute__((address_space(3))) f32x4 lds_f32x4;
  __shared__ __attribute__((aligned(1024))) uint8_t vt[W * kTileBytes];
  __shared__ float red_m[W][16], red_l[W][16];
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int n = lane & 15, g = lane >> 4;
  const int heads = p.n_kv * p.group;
  const int b = blockIdx.y;
  const int head = blockIdx.x % p.n_kv;
  const int g0 = 16 * blockIdx.z;             // first query head of the group here
  const int split = blockIdx.x / p.n_kv;
  const int begin = split * p.chunk;
  const int len = length_of(p, b);
  if (begin >= len && split > 0) return;      // the join does not read it
  const int end = min(begin + p.chunk, len);
  const int nq = min(p.group - g0, 16);

  // the chunk's pages, -1 where there is none (128 at most)
  const int first_page = begin >> p.tab.shift;
  int pages[2] = {-1, -1};
  if (begin < len) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int at = min(first_page + 64 * i + lane, (len - 1) >> p.tab.shift);
      const int g = p.tab.t[b * p.tab.ld + at];
      pages[i] = g >= 0 && g < p.tab.pages ? g : -1;
    }
  }
  // Q: query head n, in the order of the K loads' elements
  bf16x8 qf[kSteps];
  const uint16_t* qrow = p.q + b * p.qs + ((int64_t)head * p.group + g0 + min(n, nq - 1)) * p.qh;
#pragma unroll
  for (int s = 0; s < kSteps; ++s)
    qf[s] = as_bf16x8(ld16(qrow + (F8 ? 64 * (s >> 1) + 16 * g + 8 * (s & 1) : 32 * s + 8 * g)));

  const int mask = (1 << p.tab.shift) - 1;
  const int vr = lane / kLanes, vd = kPer * (lane % kLanes);
  // a head's first row of a page, wave-uniform; a lane's row and columns from
  // there are 32-bit offsets (the launcher checks)
  const uint8_t* const kx = p.kp.x + head * p.kp.sh * kBytes;
  const uint8_t* const vx = p.vp.x + head * p.vp.sh * kBytes;
  const uint8_t* const kex = F8 ? p.kp.e + head * p.kp.eh : nullptr;
  const uint8_t* const vex = F8 ? p.vp.e + head * p.vp.eh : nullptr;
  const uint32_t row_bytes = (uint32_t)(p.kp.ss * kBytes), row_exps = (uint32_t)p.kp.es;
  auto page_at = [&](int j) {
    const int i = (j >> p.tab.shift) - first_page;
    return i < 64 ? __builtin_amdgcn_readlane(pages[0], i) : __builtin_amdgcn_readlane(pages[1], i - 64);
  };
  // Block i of 16 keys of the tile at j0 lies in one page. Past the sequence's
  // end its rows are the rest of the last page, which no row's score or
  // probability takes in.
  u32x4 kreg[2][kKLoads], vreg[kVLoads];
  uint32_t ke[2], ve[kVLoads];
  auto load_k = [&](int j0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t pg = max(page_at(j0 + 16 * i), 0);
      const uint32_t at = (uint32_t)((j0 + 16 * i + n) & mask);
      const uint8_t* page = kx + pg * p.kp.sp * kBytes;
      const uint32_t off = at * row_bytes + 16 * g;
#pragma unroll
      for (int s = 0; s < kKLoads; ++s) kreg[i][s] = *reinterpret_cast<const u32x4*>(page + (off + 64 * s));
      if (F8) ke[i] = (kex + pg * p.kp.ep)[at * row_exps];
    }
  };
  auto load_v = [&](int j0) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < kVLoads; ++u) {
      const int64_t pg = max(page_at(j0 + (kVRows * u < 16 ? 0 : 16)), 0);
      const uint32_t at = (uint32_t)((j0 + kVRows * u + vr) & mask);
      vreg[u] = *reinterpret_cast<const u32x4*>(vx + pg * p.vp.sp * kBytes + (at * row_bytes + vd * kBytes));
      if (F8) ve[u] = (vex + pg * p.vp.ep)[at * row_exps];
    }
  };

  lds_u8* const mine = (lds_u8*)vt + wave * kTileBytes;
  // transposed reads: rows 4 g + n / 4 (and 16 on), column block db at xor 32 db
  const int tr_row = 4 * g + (n >> 2);
  const uint32_t tr = (uint32_t)(tr_row * kPitch + ((((n >> 1) & 1) ^ swz_v<D>(tr_row)) << 4) + 8 * (n & 1));
  f32x4 o[kDB];
#pragma unroll
  for (int db = 0; db < kDB; ++db) o[db] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m_run = -INFINITY, l_run = 0.f;
  const float c = p.scale_log2;

  int j = begin + 32 * wave;
  if (p.tab.pages == 0) j = end;
  if (j < end) {
    load_k(j);
    load_v(j);
  }
  for (; j < end; j += kStride) {
    const bool more = j + kStride < end;
    const int live[2] = {page_at(j) >= 0 ? end - j : 0, page_at(j + 16) >= 0 ? end - j - 16 : 0};
    f32x4 s[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      s[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      u32x4 a[kSteps];
#pragma unroll
      for (int t = 0; t < kKLoads; ++t) {
        if (F8) decode16(kreg[i][t], scale_of(ke[i]), a[(2 * t) % kSteps], a[(2 * t + 1) % kSteps]);
        else a[t % kSteps] = kreg[i][t];
      }
#pragma unroll
      for (int t = 0; t < kSteps; ++t)
        s[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(a[t]), qf[t], s[i], 0, 0, 0);
      if (F8) __builtin_amdgcn_sched_barrier(0);  // one block's decoded keys in registers
    }
    if (more) load_k(j + kStride);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (4 * g + e >= live[i]) s[i][e] = -INFINITY;
    float top = -INFINITY;
#pragma unroll
    for (int e = 0; e < 4; ++e) top = fmaxf(top, fmaxf(s[0][e], s[1][e]));
    const float m_new = fmaxf(m_run, over_groups<true>(top) * c);
    const float mu = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(m_run - mu);
    m_run = m_new;
    float pr[8], sum = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      pr[e] = __builtin_amdgcn_exp2f(fmaf(s[e >> 2][e & 3], c, -mu));
      sum += pr[e];
    }
    l_run = fmaf(l_run, alpha, sum);
    const u32x4 pb = u32x4{pack_bf16x2(pr[0], pr[1]), pack_bf16x2(pr[2], pr[3]),
                           pack_bf16x2(pr[4], pr[5]), pack_bf16x2(pr[6], pr[7])};
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
        decode16(vreg[u], scale_of(ve[u]), x, y);
        *reinterpret_cast<lds_u32x4*>(to + ((ch ^ sw) << 4)) = ok ? x : none;
        *reinterpret_cast<lds_u32x4*>(to + (((ch + 1) ^ sw) << 4)) = ok ? y : none;
      } else {
        *reinterpret_cast<lds_u32x4*>(to + ((ch ^ sw) << 4)) = ok ? vreg[u] : none;
      }
    }
    if (more) load_v(j + kStride);
    asm volatile("" ::: "memory");  // the V rows are written before they are read
#pragma unroll
    for (int db = 0; db < kDB; ++db) {
#pragma unroll
      for (int e = 0; e < 4; ++e) o[db][e] *= alpha;
      const lds_u8* const x = mine + (tr ^ (32 * db));
      const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)x);
      const i16x4 up = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(x + 16 * kPitch));
      const bf16x8 a =
          __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, up, 0, 1, 2, 3, 4, 5, 6, 7));
      o[db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, as_bf16x8(pb), o[db], 0, 0, 0);
      if ((db & 3) == 3) __builtin_amdgcn_sched_barrier(0);  // not all of V^T in registers at once
    }
    asm volatile("" ::: "memory");  // and read before the next tile's are written
  }

  // The waves' sums, at the largest of their references, by way of LDS: O^T
  // of lane (n, g) is head-dims 16 db + 4 g .. + 3 of query head n.
  l_run = over_groups<false>(l_run);
  if (g == 0) {
    red_m[wave][n] = m_run;
    red_l[wave][n] = l_run;
  }
  __syncthreads();
  {
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) m = fmaxf(m, red_m[w][n]);
    const float f = __builtin_amdgcn_exp2f(m_run - (m == -INFINITY ? 0.f : m));
#pragma unroll
    for (int db = 0; db < kDB; ++db) {
      f32x4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = f == 0.f ? 0.f : o[db][e] * f;
      *reinterpret_cast<lds_f32x4*>((lds_u8*)vt + ((wave * 16 + n) * (D / 4) + ((4 * db + g) ^ n)) * 16) = y;
    }
  }
  __syncthreads();
  // 16 threads a query head, D / 64 times four head-dims each
  const int qn = tid >> 4;
  if (qn >= nq) return;
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int w = 0; w < W; ++w) m = fmaxf(m, red_m[w][qn]);
  const float mu = m == -INFINITY ? 0.f : m;
#pragma unroll
  for (int w = 0; w < W; ++w) l += red_l[w][qn] * __builtin_amdgcn_exp2f(red_m[w][qn] - mu);
  const int hq = head * p.group + g0 + qn;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  float* const part = p.part + (((int64_t)b * heads + hq) * p.n_split + split) * (D + 4);
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
    const int ch = 16 * i + (tid & 15);
    f32x4 y = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < W; ++w)
      y += *reinterpret_cast<const lds_f32x4*>((lds_u8*)vt + ((w * 16 + qn) * (D / 4) + (ch ^ qn)) * 16);
    if (p.n_split == 1)
      *reinterpret_cast<u32x2*>(p.out + b * p.os + hq * p.oh + 4 * ch) =
          u32x2{pack_bf16x2(y[0] * inv, y[1] * inv), pack_bf16x2(y[2] * inv, y[3] * inv)};
    else
      *reinterpret_cast<f32x4*>(part + 4 * ch) = y;
  }
  if ((tid & 15) == 0) {
    if (p.n_split > 1) {
      part[D] = m;
      part[D + 1] = l;
    } else if (p.lse != nullptr) {
      p.lse[(int64_t)b * heads + hq] = l == 0.f ? -INFINITY : (m + __log2f(l)) * kLn2;
    }
  }
}

// The parts of a row joined, up to 64 of them: wave = (sequence, query head),
// lane i has part i's reference and sum, and D / 64 head-dims of every part, eight
// parts at a time; the first eight are asked for before the length is known.
// (2,560 rows of up to 21 parts: 4.8 us; 15.4 with four parts at a time, 9.3 with
// two waves a row.)
constexpr int kBatch = 8;

template <int D>
__global__ void __launch_bounds__(256) join_few_kernel(TokenArgs p, int64_t rows) {
  const int heads = p.n_kv * p.group;
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (row >= rows) return;
  const int b = (int)(row / heads), hq = (int)(row % heads);
  const float* part = p.part + row * p.n_split * (D + 4);
  float m = -INFINITY, sum = 0.f;
  if (lane < p.n_split) {
    m = part[lane * (D + 4) + D];
    sum = part[lane * (D + 4) + D + 1];
  }
  float x[kBatch][D / 64];
  auto fetch = [&](int i0) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
#pragma unroll
      for (int e = 0; e < D / 64; ++e)
        x[i][e] = part[min(i0 + i, p.n_split - 1) * (D + 4) + lane + 64 * e];
  };
  fetch(0);
  const int n = min(max((length_of(p, b) + p.chunk - 1) / p.chunk, 1), p.n_split);
  m = lane < n ? m : -INFINITY;
  const float top = wave_reduce<true>(m);
  const float w = lane < n ? __builtin_amdgcn_exp2f(m - (top == -INFINITY ? 0.f : top)) : 0.f;
  const float l = wave_reduce<false>(lane < n ? w * sum : 0.f);
  float acc[D / 64] = {};
  for (int i0 = 0; i0 < n; i0 += kBatch) {
    if (i0 > 0) fetch(i0);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const float wi = i0 + i < n ? __shfl(w, i0 + i) : 0.f;
#pragma unroll
      for (int e = 0; e < D / 64; ++e) acc[e] = wi == 0.f ? acc[e] : fmaf(wi, x[i][e], acc[e]);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int e = 0; e < D / 64; ++e)
    p.out[b * p.os + hq * p.oh + lane + 64 * e] = (uint16_t)f32_to_bf16(acc[e] * inv);
  if (lane == 0 && p.lse != nullptr) p.lse[row] = l == 0.f ? -INFINITY : (top + __log2f(l)) * kLn2;
}

// More parts: workgroup = (sequence, query head), a wave every W-th part, a lane
// D / 64 head-dims of it. Two passes over the references, as the weights need
// their maximum (224 rows of 128 parts: 67 us with one wave, 18 with eight).
template <int D, int W>
__global__ void __launch_bounds__(64 * W) join_kernel(TokenArgs p) {
  __shared__ float box[W][D + 2];
  const int heads = p.n_kv * p.group;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hq = blockIdx.x, b = blockIdx.y;
  const int n = min(max((length_of(p, b) + p.chunk - 1) / p.chunk, 1), p.n_split);
  const float* part = p.part + ((int64_t)b * heads + hq) * p.n_split * (D + 4);
  // this wave's parts: wave, wave + W, ..; lane i has the i-th one's reference
  float m = -INFINITY;
  for (int i = wave + W * lane; i < n; i += 64 * W) m = fmaxf(m, part[(int64_t)i * (D + 4) + D]);
  m = wave_reduce<true>(m);
  const float mu = m == -INFINITY ? 0.f : m;
  float l = 0.f, acc[D / 64] = {};
  for (int i0 = wave; i0 < n; i0 += 64 * W) {
    const int mine = i0 + W * lane;
    float w = 0.f;
    if (mine < n) {
      const float* x = part + (int64_t)mine * (D + 4) + D;
      w = __builtin_amdgcn_exp2f(x[0] - mu);
      l = fmaf(w, x[1], l);
    }
    const int count = min(64, (n - i0 + W - 1) / W);
    for (int k = 0; k < count; k += kBatch) {
      float y[kBatch][D / 64];
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
#pragma unroll
        for (int e = 0; e < D / 64; ++e)
          y[i][e] = part[(int64_t)(i0 + W * min(k + i, count - 1)) * (D + 4) + lane + 64 * e];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const float wi = k + i < count ? __shfl(w, k + i) : 0.f;
#pragma unroll
        for (int e = 0; e < D / 64; ++e) acc[e] = wi == 0.f ? acc[e] : fmaf(wi, y[i][e], acc[e]);
      }
    }
  }
  l = wave_reduce<false>(l);
#pragma unroll
  for (int e = 0; e < D / 64; ++e) box[wave][lane + 64 * e] = acc[e];
  if (lane == 0) {
    box[wave][D] = m;
    box[wave][D + 1] = l;
  }
  __syncthreads();
  const int d = threadIdx.x;
  if (d >= D) return;
  m = -INFINITY;
#pragma unroll
  for (int w = 0; w < W; ++w) m = fmaxf(m, box[w][D]);
  float y = 0.f;
  l = 0.f;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const float f = __builtin_amdgcn_exp2f(box[w][D] - (m == -INFINITY ? 0.f : m));
    l = fmaf(f, box[w][D + 1], l);
    y = f == 0.f ? y : fmaf(f, box[w][d], y);
  }
  p.out[b * p.os + hq * p.oh + d] = (uint16_t)f32_to_bf16(l == 0.f ? 0.f : y / l);
  if (d == 0 && p.lse != nullptr)
    p.lse[(int64_t)b * heads + hq] = l == 0.f ? -INFINITY : (m + __log2f(l)) * kLn2;
}

bool whole(const void* p, int64_t mult, int64_t a, int64_t b, int64_t c) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && a % mult == 0 && b % mult == 0 && c % mult == 0;
}

int check_cache(const char* what, int64_t head_dim, int64_t n_kv, int64_t n_pages, int64_t page,
                int64_t width, int f8, const Pages& k, const Pages& v) {
  VEDA_REQUIRE(head_dim == 64 || head_dim == 128, "%s: head_dim must be 64 or 128, got %lld", what,
               (long long)head_dim);
  VEDA_REQUIRE(n_kv > 0 && n_kv <= 65535, "%s: 1 to 65535 key heads, got %lld", what, (long long)n_kv);
  VEDA_REQUIRE(page >= 16 && page <= 256 && (page & (page - 1)) == 0,
               "%s: pages of 16, 32, 64, 128 or 256 rows, got %lld", what, (long long)page);
  VEDA_REQUIRE(n_pages >= 0 && n_pages < (1ll << 31) && width >= 0 && width < (1ll << 31),
               "%s: page count or table width out of range", what);
  const int64_t mult = f8 ? 16 : 8;
  VEDA_REQUIRE(whole(k.x, mult, k.sp, k.ss, k.sh) && whole(v.x, mult, v.sp, v.ss, v.sh),
               "%s: cache rows must be 16-byte aligned", what);
  VEDA_REQUIRE(!f8 || n_pages == 0 || (k.e != nullptr && v.e != nullptr),
               "%s: an e4m3 cache needs its exponents", what);
  return VEDA_OK;
}

Pages pages_of(const void* x, int64_t sp, int64_t ss, int64_t sh, const uint8_t* e, int64_t ep,
               int64_t es, int64_t eh) {
  return Pages{static_cast<uint8_t*>(const_cast<void*>(x)), sp, ss, sh, const_cast<uint8_t*>(e),
               ep, es, eh};
}

Table table_of(const int32_t* table, int64_t ld, int64_t width, int64_t n_pages, int64_t page) {
  return Table{table, ld, (int32_t)width, (int32_t)n_pages, __builtin_ctzll((uint64_t)page)};
}

}  // namespace
}  // namespace veda

using namespace veda;

extern "C" int veda_cache_append(const void* k, int64_t k_stride_s, int64_t k_stride_h,
                                 const void* v, int64_t v_stride_s, int64_t v_stride_h, int64_t rows,
                                 int64_t n_kv_heads, int64_t head_dim, const int32_t* cu,
                                 const int32_t* start, int64_t n_seq, void* k_pages, void* v_pages,
                                 int64_t stride_p, int64_t stride_s, int64_t stride_h, int e4m3,
                                 uint8_t* k_exp, uint8_t* v_exp, int64_t exp_stride_p,
                                 int64_t exp_stride_s, int64_t exp_stride_h, int64_t n_pages,
                                 int64_t page, const int32_t* table, int64_t table_ld, int64_t width,
                                 void* stream) {
  AppendArgs p{};
  p.kp = pages_of(k_pages, stride_p, stride_s, stride_h, k_exp, exp_stride_p, exp_stride_s, exp_stride_h);
  p.vp = pages_of(v_pages, stride_p, stride_s, stride_h, v_exp, exp_stride_p, exp_stride_s, exp_stride_h);
  if (int rc = check_cache("cache_append", head_dim, n_kv_heads, n_pages, page, width, e4m3, p.kp, p.vp))
    return rc;
  // (a wave a row, and a launch holds less than 2^32 threads)
  VEDA_REQUIRE(rows >= 0 && rows < (1 << 26) && n_seq >= 0 && n_seq < (1 << 20),
               "cache_append: 2^26 rows or 2^20 sequences, or negative");
  VEDA_REQUIRE(whole(k, 8, k_stride_s, k_stride_h, 0) && whole(v, 8, v_stride_s, v_stride_h, 0),
               "cache_append: k and v rows must be 16-byte aligned");
  if (rows == 0 || n_seq == 0) return VEDA_OK;
  p.k = static_cast<const uint16_t*>(k);
  p.v = static_cast<const uint16_t*>(v);
  p.ks = k_stride_s; p.kh = k_stride_h;
  p.vs = v_stride_s; p.vh = v_stride_h;
  p.tab = table_of(table, table_ld, width, n_pages, page);
  p.cu = cu;
  p.start = start;
  p.n_seq = (int32_t)n_seq;
  p.rows = (int32_t)rows;
  p.n_kv = (int32_t)n_kv_heads;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const unsigned grid = (unsigned)((rows + 3) / 4);
  if (head_dim == 128) {
    if (e4m3) append_kernel<128, true><<<grid, 256, 0, s>>>(p);
    else append_kernel<128, false><<<grid, 256, 0, s>>>(p);
  } else {
    if (e4m3) append_kernel<64, true><<<grid, 256, 0, s>>>(p);
    else append_kernel<64, false><<<grid, 256, 0, s>>>(p);
  }
  return check_launch("veda_cache_append");
}

extern "C" int veda_cache_gather(const void* k_pages, const void* v_pages, int64_t stride_p,
                                 int64_t stride_s, int64_t stride_h, int e4m3, const uint8_t* k_exp,
                                 const uint8_t* v_exp, int64_t exp_stride_p, int64_t exp_stride_s,
                                 int64_t exp_stride_h, int64_t n_pages, int64_t page,
                                 const int32_t* table, int64_t table_ld, int64_t width,
                                 const int32_t* cu, int64_t n_seq, int64_t rows, int64_t n_kv_heads,
                                 int64_t head_dim, void* k, void* v, void* stream) {
  GatherArgs p{};
  p.kp = pages_of(k_pages, stride_p, stride_s, stride_h, k_exp, exp_stride_p, exp_stride_s, exp_stride_h);
  p.vp = pages_of(v_pages, stride_p, stride_s, stride_h, v_exp, exp_stride_p, exp_stride_s, exp_stride_h);
  if (int rc = check_cache("cache_gather", head_dim, n_kv_heads, n_pages, page, width, e4m3, p.kp, p.vp))
    return rc;
  VEDA_REQUIRE(rows >= 0 && rows < (1 << 26) && n_seq >= 0 && n_seq < (1 << 20),
               "cache_gather: 2^26 rows or 2^20 sequences, or negative");
  VEDA_REQUIRE(whole(k, 8, 0, 0, 0) && whole(v, 8, 0, 0, 0), "cache_gather: k and v must be 16-byte aligned");
  if (rows == 0) return VEDA_OK;
  p.tab = table_of(table, table_ld, width, n_pages, page);
  p.cu = cu;
  p.n_seq = (int32_t)n_seq;
  p.rows = (int32_t)rows;
  p.n_kv = (int32_t)n_kv_heads;
  p.k = static_cast<uint16_t*>(k);
  p.v = static_cast<uint16_t*>(v);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const unsigned grid = (unsigned)((rows + 3) / 4);
  if (head_dim == 128) {
    if (e4m3) gather_cache_kernel<128, true><<<grid, 256, 0, s>>>(p);
    else gather_cache_kernel<128, false><<<grid, 256, 0, s>>>(p);
  } else {
    if (e4m3) gather_cache_kernel<64, true><<<grid, 256, 0, s>>>(p);
    else gather_cache_kernel<64, false><<<grid, 256, 0, s>>>(p);
  }
  return check_launch("veda_cache_gather");
}

extern "C" int veda_paged_fwd(const void* q, int64_t q_stride_s, int64_t q_stride_h, int64_t n_seq,
                              int64_t n_heads, int64_t n_kv_heads, int64_t head_dim,
                              const void* k_pages, const void* v_pages, int64_t stride_p,
                              int64_t stride_s, int64_t stride_h, int e4m3, const uint8_t* k_exp,
                              const uint8_t* v_exp, int64_t exp_stride_p, int64_t exp_stride_s,
                              int64_t exp_stride_h, int64_t n_pages, int64_t page,
                              const int32_t* table, int64_t table_ld, int64_t width,
                              const int32_t* lengths, float scale, int64_t chunk, void* out,
                              int64_t o_stride_s, int64_t o_stride_h, float* lse, void* workspace,
                              int64_t workspace_bytes, void* stream) {
  TokenArgs p{};
  p.kp = pages_of(k_pages, stride_p, stride_s, stride_h, k_exp, exp_stride_p, exp_stride_s, exp_stride_h);
  p.vp = pages_of(v_pages, stride_p, stride_s, stride_h, v_exp, exp_stride_p, exp_stride_s, exp_stride_h);
  if (int rc = check_cache("paged_fwd", head_dim, n_kv_heads, n_pages, page, width, e4m3, p.kp, p.vp))
    return rc;
  VEDA_REQUIRE(n_heads > 0 && n_heads % n_kv_heads == 0,
               "paged_fwd: %lld query heads are no multiple of %lld key heads", (long long)n_heads,
               (long long)n_kv_heads);
  VEDA_REQUIRE(n_seq >= 0 && n_seq <= 65535, "paged_fwd: at most 65535 sequences, got %lld",
               (long long)n_seq);
  VEDA_REQUIRE(width * page <= 0x7fff0000, "paged_fwd: a table row holds nearly 2^31 keys");
  // a page's rows are addressed with 32-bit byte offsets
  VEDA_REQUIRE(stride_s >= 0 && exp_stride_s >= 0 && stride_s < (1 << 22) && exp_stride_s < (1 << 22),
               "paged_fwd: row stride of the cache negative or too large");
  VEDA_REQUIRE(scale > 0.f && scale < INFINITY, "paged_fwd: scale must be positive and finite");
  VEDA_REQUIRE(whole(q, 8, q_stride_s, q_stride_h, 0) && whole(out, 8, o_stride_s, o_stride_h, 0),
               "paged_fwd: q and out rows must be 16-byte aligned");
  VEDA_REQUIRE(chunk >= page && chunk % page == 0 && chunk % 32 == 0 && chunk <= 128 * page,
               "paged_fwd: chunk must be a multiple of 32 and 1 to 128 whole pages, got %lld",
               (long long)chunk);
  if (n_seq == 0) return VEDA_OK;
  const int64_t group = n_heads / n_kv_heads, capacity = width * page;
  const int64_t n_split = capacity > chunk ? (capacity + chunk - 1) / chunk : 1;
  const int64_t need = n_split == 1 ? 0 : n_seq * n_heads * n_split * (head_dim + 4) * 4;
  VEDA_REQUIRE(need == 0 || ((reinterpret_cast<uintptr_t>(workspace) & 15) == 0 &&
                             workspace != nullptr && workspace_bytes >= need),
               "paged_fwd: workspace needs %lld bytes (16-byte aligned), got %lld", (long long)need,
               (long long)workspace_bytes);
  VEDA_REQUIRE(n_split * n_kv_heads < (1 << 24) && group <= 16 * 65535 && n_heads * n_seq < (1 << 26) &&
                   n_heads < (1 << 23),
               "paged_fwd: too many heads for one launch");
  p.q = static_cast<const uint16_t*>(q);
  p.qs = q_stride_s; p.qh = q_stride_h;
  p.tab = table_of(table, table_ld, width, n_pages, page);
  p.lengths = lengths;
  p.n_kv = (int32_t)n_kv_heads;
  p.group = (int32_t)group;
  p.chunk = (int32_t)chunk;
  p.n_split = (int32_t)n_split;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.out = static_cast<uint16_t*>(out);
  p.os = o_stride_s; p.oh = o_stride_h;
  p.lse = lse;
  p.part = static_cast<float*>(workspace);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)(n_split * n_kv_heads), (unsigned)n_seq, (unsigned)((group + 15) / 16));
  auto launch = [&](auto d, auto f8) {
    // eight waves where they are all that a sequence gets and the launch leaves room
    if (n_split == 1 && capacity > 128 && grid.x * grid.y * grid.z < 256)
      token_kernel<decltype(d)::value, decltype(f8)::value, 8><<<grid, 512, 0, s>>>(p);
    else
      token_kernel<decltype(d)::value, decltype(f8)::value, 4><<<grid, 256, 0, s>>>(p);
  };
  using D128 = std::integral_constant<int, 128>;
  using D64 = std::integral_constant<int, 64>;
  if (head_dim == 128 && e4m3) launch(D128{}, std::true_type{});
  else if (head_dim == 128) launch(D128{}, std::false_type{});
  else if (e4m3) launch(D64{}, std::true_type{});
  else launch(D64{}, std::false_type{});
  if (n_split > 1) {
    if (int rc = check_launch("veda_paged_fwd")) return rc;
    const dim3 jgrid((unsigned)n_heads, (unsigned)n_seq);
    const int64_t rows = n_seq * n_heads;
    const unsigned few = (unsigned)((rows + 3) / 4);
    if (head_dim == 128) {
      if (n_split <= 64) join_few_kernel<128><<<few, 256, 0, s>>>(p, rows);
      else join_kernel<128, 8><<<jgrid, 512, 0, s>>>(p);
    } else {
      if (n_split <= 64) join_few_kernel<64><<<few, 256, 0, s>>>(p, rows);
      else join_kernel<64, 8><<<jgrid, 512, 0, s>>>(p);
    }
  }
  return check_launch("veda_paged_fwd");
}
