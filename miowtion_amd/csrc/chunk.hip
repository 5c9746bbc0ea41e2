// Attention of a chunk of new tokens of every sequence over a paged cache that holds
// them already, for gfx950: queries [cu[b], cu[b + 1]) of sequence b, n_q of them, see
// the first n_k = lengths[b] positions of its cache, query i the keys up to
// i + n_k - n_q when causal. Formulas, rows and the walk are those of the packed
// forward (packed_walk.h); keys and values come from the cache's pages as they lie
// (paged_common.h), in bf16 or e4m3.
//
// A wave loads 16 of a step's 64 keys, which lie in one page: pages have 16 rows at
// least and begin where a block of 16 keys does. A lane holds the page of one step
// for its wave, 64 steps at a time, so a step's page is one lane's register.
//   bf16: rows go from the page straight into LDS.
//   e4m3: codes of a step wait in registers for one iteration, while they come, and
//         are decoded (times the row's power of two: exact) on their way into LDS, once
//         for the workgroup's 128 rows.
// A key in a page outside the cache draws no weight.
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
  float* part;  // n_split > 1: [n_split][q_rows, H][D] sums, then [n_split][q_rows, H]
                // pairs of reference (log2) and sum of weights
  float scale_log2;
  int32_t n_slots, n_split;
  uint32_t per_group;
};

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

// Scores of keys in blocks of 16 that have no page: bit 0 the sub-block's first.
__device__ __forceinline__ void mask_blocks(f32x16& s, uint32_t bad) {
#pragma unroll
  for (int e = 0; e < 16; ++e)
    if ((bad >> (e >> 3)) & 1) s[e] = -INFINITY;
}

// A step's 16 keys of a wave: the page, the block of 16 keys, and the step's blocks
// without a page (bits 0 to 3).
struct Place {
  int page, block;
  uint32_t bad;
};

template <int D, bool F8>
__global__ void __launch_bounds__(kThreads, 2) chunk_kernel(ChunkArgs p) {
  using T = Tile<D>;
  constexpr int kSlot = 2 * T::kBytes;  // K and V of a step
  constexpr int kAhead = F8 ? 3 : 2;    // steps from a step's scores to K's load
  typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
  __shared__ __attribute__((aligned(1024))) uint8_t ring[2][kSlot];
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int li = lane & 31, hi = lane >> 5;
  const int head = blockIdx.x % p.pk.n_kv;
  const int item = (int)(blockIdx.x / p.pk.n_kv);
  const int split = item % p.n_split;
  Span sp = span_of_slot(p.pk, false, p.n_slots - 1 - item / p.n_split, lane);
  const int b = sp.seq - 1;
  const bool none = b < 0 || b >= p.pk.n_seq || p.tab.pages == 0;
  sp.k0 = 0;
  sp.nk = none ? 0 : min(max(p.lengths[b], 0), p.tab.width << p.tab.shift);
  const int rows = sp.nq * p.pk.group;
  const int r0 = sp.tile * kRows;
  if (r0 >= rows) return;

  const int r = r0 + 32 * wave + li;
  const bool real = r < rows;
  const int last = visible_keys(p.pk, sp, min(r0 + kRows, rows) - 1);
  // this split's steps of 64 keys; from here on keys count from its first
  const int all_steps = (last + 63) >> 6;
  const int from = (int)((int64_t)all_steps * split / p.n_split);
  const int n_steps = (int)((int64_t)all_steps * (split + 1) / p.n_split) - from;
  const int end = 64 * n_steps;
  const int limit = min(max((real ? visible_keys(p.pk, sp, r) : last) - 64 * from, 0), end);
  const int n_plain = min(max(visible_keys(p.pk, sp, r0) - 64 * from, 0), end) >> 6;  // seen whole by every row
  // keys that every row of the wave sees (its rows see more and more)
  const int wave_all = __builtin_amdgcn_readfirstlane(
      min(max((r0 + 32 * wave < rows ? visible_keys(p.pk, sp, r0 + 32 * wave) : last) - 64 * from, 0), end));
  const RowLoads<D> qrows =
      load_rows<D>(p.q + (int64_t)sp.q0 * p.qs + (int64_t)head * p.pk.group * p.qh, p.qs, p.qh, p.pk.group,
                   p.per_group, r0 + 32 * wave, rows, lane);
  Wave<D> w;

  // Pages. Lane i: of step window + i, the page of this wave's 16 keys and the blocks
  // without one. Blocks past the sequence's last repeat it.
  const int last_block = max(sp.nk - 1, 0) >> 4, page_mask = (1 << p.tab.shift) - 1;
  int pages = 0, window = -64;
  uint32_t bads = 0;
  auto place = [&](int u) __attribute__((always_inline)) {
    if (u - window >= 64) {
      window = u;
      bads = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int block = min(4 * (from + u + lane) + i, last_block);
        const int g = p.tab.t[b * p.tab.ld + (block >> (p.tab.shift - 4))];
        const bool ok = g >= 0 && g < p.tab.pages;
        bads |= ok ? 0u : 1u << i;
        if (i == wave) pages = ok ? g : 0;
      }
    }
    Place x;
    x.page = __builtin_amdgcn_readlane(pages, u - window);
    x.bad = __builtin_amdgcn_readlane(bads, u - window);
    x.block = min(4 * (from + u) + wave, last_block);
    return x;
  };
  // where a place's first row lies in K or V, in elements
  auto at = [&](const Pages& x, const Place& y) __attribute__((always_inline)) {
    return y.page * x.sp + ((16 * y.block) & page_mask) * x.ss + head * x.sh;
  };
  // bf16: this wave's loads of a step, segment s (1 KB) rows kSegRows s on of its 16;
  // `clamp`: rows past the sequence's last key read that key again
  struct Src {
    const char* base;
    uint32_t off[T::kSegs];
  };
  auto src_of = [&](const Pages& x, const Place& y, bool is_v, bool clamp) __attribute__((always_inline)) {
    Src r;
    r.base = reinterpret_cast<const char*>(x.x) + 2 * at(x, y);
#pragma unroll
    for (int s = 0; s < T::kSegs; ++s) {
      const int row = s * T::kSegRows + lane / T::kChunks, pos = lane % T::kChunks;
      const uint32_t src = (uint32_t)(clamp ? min(row, sp.nk - 1 - 16 * y.block) : row);
      r.off[s] = src * (uint32_t)(2 * x.ss) + ((pos ^ (is_v ? swz_tr<D>(row) : swz_row<D>(row))) << 4);
    }
    return r;
  };
  // e4m3: 16 codes of a lane, kCodeLanes lanes a row, and the row's exponent
  constexpr int kCodeLanes = D / 16, kCodes = 16 * kCodeLanes / 64;
  struct Codes {
    u32x4 x[kCodes];
    uint32_t e[kCodes];
  };
  auto fetch = [&](const Pages& x, const Place& y, bool clamp) __attribute__((always_inline)) {
    Codes r;
    const uint8_t* base = x.x + at(x, y);
    const uint8_t* exps = x.e + y.page * x.ep + ((16 * y.block) & page_mask) * x.es + head * x.eh;
#pragma unroll
    for (int s = 0; s < kCodes; ++s) {
      const int row = s * (64 / kCodeLanes) + lane / kCodeLanes;
      const uint32_t src = (uint32_t)(clamp ? min(row, sp.nk - 1 - 16 * y.block) : row);
      r.x[s] = *reinterpret_cast<const u32x4*>(base + src * (uint32_t)x.ss + 16 * (lane % kCodeLanes));
      r.e[s] = exps[src * (uint32_t)x.es];
    }
    return r;
  };
  lds_u8* const s0 = (lds_u8*)ring[0];
  auto put = [&](const Codes& x, int s, lds_u8* to, bool is_v) __attribute__((always_inline)) {
    u32x4 a, c;
    decode16(x.x[s], scale_of(x.e[s]), a, c);
    const int row = 16 * wave + s * (64 / kCodeLanes) + lane / kCodeLanes, ch = 2 * (lane % kCodeLanes);
    const int swz = is_v ? swz_tr<D>(row) : swz_row<D>(row);
    *reinterpret_cast<lds_u32x4*>(to + row * T::kPitch + ((ch ^ swz) << 4)) = a;
    *reinterpret_cast<lds_u32x4*>(to + row * T::kPitch + (((ch + 1) ^ swz) << 4)) = c;
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
  // u, and brings K of step u + 2 (over K of step u) and V of step u + 1 into LDS: bf16
  // as loads that have an iteration to arrive, e4m3 from registers that were asked for
  // an iteration before.
  constexpr int kSub = 32 * T::kPitch;
  const uint32_t lds0 =
      __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(s0 + T::kSegs * 1024 * wave));
  auto issue = [&](const Src& x, int s, uint32_t to) { dma16_m0(x.base, x.off[s], to + s * 1024); };
  auto sync = [&]() {
    if (F8) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the rows that it put into LDS
    else VEDA_WAIT_VM(0);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  f32x16 sa, sb;
  u32x4 pa[2], pb[2];
  Place p1, p2;      // of steps u + 1 and u + 2 (e4m3)
  Codes kc, vc;      // e4m3: K of step u + 2, V of step u + 1
  auto iter = [&](auto masked, int u, uint32_t cur, uint32_t nxt) __attribute__((always_inline)) {
    // MASKED: step u + 1 holds keys that some row does not see, or a step that is
    // asked for may be past the last
    constexpr bool MASKED = decltype(masked)::value;
    const Place next = place(MASKED ? min(u + kAhead, n_steps - 1) : u + kAhead);
    const uint32_t bad = p1.bad;
    Src ks, vs;
    if constexpr (!F8) {
      ks = src_of(p.kp, next, false, MASKED);
      vs = src_of(p.vp, p1, true, MASKED);
    }
    sync();
    auto first = [&](int j) {
      if constexpr (F8) {
        if (j < kCodes) put(kc, j, s0 + cur, false);
        else if (j == kCodes) kc = fetch(p.kp, next, MASKED);
      } else {
        if (j < T::kSegs) issue(ks, j, lds0 + cur);
        else if (j < 2 * T::kSegs) issue(vs, j - T::kSegs, lds0 + nxt + T::kBytes);
      }
    };
    auto second = [&](int j) {
      if constexpr (F8) {
        if (j < kCodes) put(vc, j, s0 + nxt + T::kBytes, true);
        else if (j == kCodes) vc = fetch(p.vp, p2, MASKED);
      }
    };
    constexpr int kGive = F8 ? kNoNext : kReadNext, kTake = F8 ? kNoNext : kTakeNext;
    Next<D> ahead;
    stage<D, true, kSmSecond, true, kGive>(s0 + nxt, s0 + cur, f, c, sa, sb, pb, pa, w, first, &ahead);
    if (MASKED && 64 * (u + 1) + 32 > wave_all) mask_scores(sa, limit - 64 * (u + 1), hi);
    if (__builtin_expect((bad & 3) != 0, 0)) mask_blocks(sa, bad);
    stage<D, true, kSmFirst, true, kTake>(s0 + nxt + kSub, s0 + cur + kSub, f, c, sb, sa, pa, pb, w, second,
                                          &ahead);
    if (MASKED && 64 * (u + 1) + 64 > wave_all) mask_scores(sb, limit - 64 * (u + 1) - 32, hi);
    if (__builtin_expect((bad & 12) != 0, 0)) mask_blocks(sb, bad >> 2);
    p1 = F8 ? p2 : next;
    p2 = next;
  };
  if (n_steps > 0) {
    const Place p0 = place(0);
    p1 = place(min(1, n_steps - 1));
    p2 = place(min(2, n_steps - 1));
    if constexpr (F8) {
      kc = fetch(p.kp, p0, true);
      vc = fetch(p.vp, p0, true);
#pragma unroll
      for (int s = 0; s < kCodes; ++s) {
        put(kc, s, s0, false);
        put(vc, s, s0 + T::kBytes, true);
      }
    } else {
      const Src k0 = src_of(p.kp, p0, false, true), v0 = src_of(p.vp, p0, true, true);
#pragma unroll
      for (int s = 0; s < T::kSegs; ++s) issue(k0, s, lds0);
#pragma unroll
      for (int s = 0; s < T::kSegs; ++s) issue(v0, s, lds0 + T::kBytes);
    }
    // Q by way of slot 1, which K of step 1 comes into after the barrier
    frags_of_rows<D>(qrows, s0 + kSlot + wave * 32 * T::kPitch, lane, w.qf);
#pragma unroll
    for (int s = 0; s < T::kK; ++s) asm volatile("" : : "v"(w.qf[s]));
    if constexpr (F8) kc = fetch(p.kp, p1, true);
    sync();
    if constexpr (F8) {
#pragma unroll
      for (int s = 0; s < kCodes; ++s) put(kc, s, s0 + kSlot, false);
      kc = fetch(p.kp, p2, true);
      vc = fetch(p.vp, p1, true);
    } else if (n_steps > 1) {
      const Src k1 = src_of(p.kp, p1, false, true);
#pragma unroll
      for (int s = 0; s < T::kSegs; ++s) issue(k1, s, lds0 + kSlot);
    }
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
  leave_rows<D>(p, w, sp, split, head, r0, rows, limit, wave, lane, s0,
                [&](int64_t tok, int64_t hd, int lim, float mu, float inv, float* part) {
                  constexpr int kBytes = F8 ? 1 : 2;
                  redo_paged_row<D, F8>(p.q + tok * p.qs + hd * p.qh, p.kp.x + kBytes * head * p.kp.sh,
                                        p.vp.x + kBytes * head * p.vp.sh, p.kp.e + head * p.kp.eh,
                                        p.vp.e + head * p.vp.eh, p.kp.sp, p.kp.ss, p.kp.ep, p.kp.es,
                                        p.tab.t + b * p.tab.ld, p.tab.pages, p.tab.shift, 64 * from, lim, c,
                                        mu, inv, p.out + tok * p.os + hd * p.oh, part, lane);
                });
}

// The splits of a row joined, as the packed forward's.
template <int D>
__global__ void __launch_bounds__(256) chunk_merge_kernel(ChunkArgs p) {
  const int64_t n_heads = (int64_t)p.pk.n_kv * p.pk.group, all_rows = p.pk.q_rows * n_heads;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = i / (D / 4);
  const int d = 4 * (int)(i % (D / 4));
  if (row >= all_rows) return;
  const f32x2* ml = reinterpret_cast<const f32x2*>(p.part + p.n_split * all_rows * D) + row;
  float m = -INFINITY;
#pragma unroll 4
  for (int s = 0; s < p.n_split; ++s) m = fmaxf(m, ml[s * all_rows][0]);
  const float mu = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < p.n_split; ++s) {
    const f32x2 x = ml[s * all_rows];
    const float w = __builtin_amdgcn_exp2f(x[0] - mu);
    const f32x4 y = *reinterpret_cast<const f32x4*>(p.part + (s * all_rows + row) * D + d);
    l = fmaf(w, x[1], l);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = w == 0.f ? o[e] : fmaf(w, y[e], o[e]);
  }
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
                              int64_t n_split, void* out, int64_t o_stride_s, int64_t o_stride_h, float* lse,
                              void* workspace, int64_t workspace_bytes, void* stream) {
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
  if (q_rows == 0) return VEDA_OK;
  const int64_t group = n_heads / n_kv_heads, slots = slots_of(q_rows, group, n_seq);
  // a launch holds less than 2^32 threads
  VEDA_REQUIRE(slots * n_kv_heads * n_split < (1 << 24) && (n_split == 1 || q_rows * n_heads < (1 << 27)),
               "%s: too many rows for one launch", what);
  const int64_t need = n_split == 1 ? 0 : n_split * q_rows * n_heads * (head_dim + 2) * 4;
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
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const unsigned grid = (unsigned)(slots * n_kv_heads * n_split);
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
    if (head_dim == 128) chunk_merge_kernel<128><<<join, 256, 0, s>>>(p);
    else chunk_merge_kernel<64><<<join, 256, 0, s>>>(p);
  }
  return check_launch(what);
}
