// Attention of packed sequences for gfx950 (bf16, head_dim 64 or 128, grouped
// heads, causal or not): for query i of a sequence with n_q queries and n_k keys
//   S_j = scale q_i . k_j  over the keys j it sees (causal: j <= i + n_k - n_q)
//   O_i = sum_j exp(S_j - LSE_i) v_j,   LSE_i = log sum_j exp(S_j)
// A row that sees no key has O = 0 and LSE = -inf.
//
// Workgroup = 128 packed rows of one key head (packed_common.h), 4 waves; wave
// w owns rows 32 w .. + 31 and walks the keys in steps of 64. Scores are
// computed transposed (S^T = K Q^T, 32x32x16 products), so a lane owns one
// query row, its softmax needs one exchange between the wave's halves, and P^T
// goes from the accumulators into the B operand of O^T += V^T P^T.
#include <type_traits>

#include "packed_walk.h"

namespace veda {
namespace {

constexpr int kThreads = 256;

struct FwdArgs {
  Packing pk;
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  int64_t qs, qh, ks, kh, vs, vh;
  uint16_t* out;
  int64_t os, oh;
  float* lse;  // [q_rows, H] or NULL
  float* part;  // n_split > 1: [n_split][q_rows, H][D] sums, then [n_split][q_rows, H]
                // pairs of reference (log2) and sum of weights
  float scale_log2;
  int32_t n_slots, n_split;
  uint32_t per_group;
};

// A row whose O came out with a NaN though its sum of weights has none, again, key
// by key: a key that the row does not see, or whose probability is zero, adds
// nothing whatever its V holds (a product with a zero probability makes a NaN of an
// infinity or a NaN). All lanes of the wave work on the row; lane l has head-dims l
// and l + 64. To out as bf16, or, where part is given, there in 32 bits.
// A row costs some 200 times its share of the walk (4,096 tokens, 8 heads on 2: all
// rows 14 ms, the walk 67 us), so rows that the walk has right are left out: an
// infinity is one of a key with a weight, and a sum of weights that is NaN, as any
// score that is NaN makes it, gives a NaN in every column either way.
template <int D>
__device__ __noinline__ void redo_row(const uint16_t* q, const uint16_t* k, const uint16_t* v,
                                      int64_t ks, int64_t vs, int limit, float c, float mu, float inv,
                                      uint16_t* out, float* part, int lane) {
  float acc[D / 64] = {};
  for (int j0 = 0; j0 < limit; j0 += 64) {
    const int j = j0 + lane;
    float s = 0.f;
    if (j < limit) {
      for (int d = 0; d < D; d += 8) {
        const u32x4 a = ld16(q + d), b = ld16(k + j * ks + d);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          s = fmaf(bf16_to_f32(a[m] & 0xffffu), bf16_to_f32(b[m] & 0xffffu), s);
          s = fmaf(bf16_to_f32(a[m] >> 16), bf16_to_f32(b[m] >> 16), s);
        }
      }
    }
    const float pr = j < limit ? __builtin_amdgcn_exp2f(fmaf(s, c, -mu)) : 0.f;
    for (int i = 0; i < min(64, limit - j0); ++i) {
      const float pi = __shfl(pr, i);
      if (pi == 0.f) continue;
#pragma unroll
      for (int m = 0; m < D / 64; ++m)
        acc[m] = fmaf(pi, bf16_to_f32(v[(j0 + i) * vs + lane + 64 * m]), acc[m]);
    }
  }
#pragma unroll
  for (int m = 0; m < D / 64; ++m) {
    if (part != nullptr) part[lane + 64 * m] = acc[m];
    else out[lane + 64 * m] = (uint16_t)f32_to_bf16(acc[m] * inv);
  }
}

// Bound by power at head_dim 128 (16,384 tokens, 16 heads on 4: 966 us, 1.14
// PFLOP/s; the matrix cores are busy 69 % of a clock that falls to 1.6 GHz), by the
// vector units at 64 (four chunks of 512 onto up to 8,192 keys, 32 on 8: 106 us a
// call, 0.80 PFLOP/s; about half of their cycles are exponentials, and the longest
// sequence's tiles end last). A prompt of 77 is
// launch and latency: 10 us.
template <int D>
__global__ void __launch_bounds__(kThreads, 2) packed_fwd_kernel(FwdArgs p) {
  using T = Tile<D>;
  constexpr int kSlot = 2 * T::kBytes;  // K and V of a step
  __shared__ __attribute__((aligned(1024))) uint8_t ring[2][kSlot];
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int li = lane & 31, hi = lane >> 5;
  const int head = blockIdx.x % p.pk.n_kv;
  const int item = (int)(blockIdx.x / p.pk.n_kv);
  const int split = item % p.n_split;
  const Span sp = span_of(p.pk, false, item / p.n_split, p.n_slots, p.pk.n_kv * p.n_split, lane);
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
  const int nk = sp.nk - 64 * from;
  const RowLoads<D> qrows =
      load_rows<D>(p.q + (int64_t)sp.q0 * p.qs + (int64_t)head * p.pk.group * p.qh, p.qs, p.qh, p.pk.group,
                   p.per_group, r0 + 32 * wave, rows, lane);
  Wave<D> w;

  const uint16_t* kbase = p.k + (int64_t)(sp.k0 + 64 * from) * p.ks + head * p.kh;
  const uint16_t* vbase = p.v + (int64_t)(sp.k0 + 64 * from) * p.vs + head * p.vh;
  // This wave's loads of K or V of step u (past the last step that one again):
  // segment s is 1 KB, rows kSegRows (kSegs wave + s) on; rows past the
  // sequence's last key read that key again.
  struct Src {
    const char* base;
    uint32_t off[T::kSegs];
  };
  auto src_of = [&](const uint16_t* x, int64_t stride, int u, bool is_v, bool clamp) {
    u = clamp ? min(u, n_steps - 1) : u;
    Src r;
    r.base = reinterpret_cast<const char*>(x + (int64_t)u * 64 * stride);
#pragma unroll
    for (int s = 0; s < T::kSegs; ++s) {
      const int row = (T::kSegs * wave + s) * T::kSegRows + lane / T::kChunks, pos = lane % T::kChunks;
      const uint32_t src = (uint32_t)(clamp ? min(row, nk - 1 - 64 * u) : row);
      r.off[s] = src * (uint32_t)(2 * stride) +
                 ((pos ^ (is_v ? swz_tr<D>(row) : swz_row<D>(row))) << 4);
    }
    return r;
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

  // The walk. K and V of step u have their halves of slot u % 2, and V runs one
  // step behind K: iteration u multiplies K of step u + 1 and V of step u, and
  // loads K of step u + 2 (over K of step u) and V of step u + 1, so a load has
  // an iteration to arrive.
  constexpr int kSub = 32 * T::kPitch;
  lds_u8* const s0 = (lds_u8*)ring[0];
  const uint32_t lds0 =
      __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(s0 + T::kSegs * 1024 * wave));
  auto issue = [&](const Src& x, int s, uint32_t to) { dma16_m0(x.base, x.off[s], to + s * 1024); };
  auto sync = [&]() {
    VEDA_WAIT_VM(0);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  f32x16 sa, sb;
  u32x4 pa[2], pb[2];
  auto iter = [&](auto masked, int u, uint32_t cur, uint32_t nxt) __attribute__((always_inline)) {
    // MASKED: step u + 1 holds keys that some row does not see, or step u + 2 may
    // be past the last
    constexpr bool MASKED = decltype(masked)::value;
    const Src ks = src_of(kbase, p.ks, u + 2, false, MASKED);
    const Src vs = src_of(vbase, p.vs, u + 1, true, MASKED);
    sync();
    auto hook = [&](int j) {
      if (j < T::kSegs) issue(ks, j, lds0 + cur);
      else if (j < 2 * T::kSegs) issue(vs, j - T::kSegs, lds0 + nxt + T::kBytes);
    };
    Next<D> next;
    stage<D, true, kSmSecond, true, kReadNext>(s0 + nxt, s0 + cur, f, c, sa, sb, pb, pa, w, hook, &next);
    if (MASKED && 64 * (u + 1) + 32 > wave_all) mask_scores(sa, limit - 64 * (u + 1), hi);
    stage<D, true, kSmFirst, true, kTakeNext>(s0 + nxt + kSub, s0 + cur + kSub, f, c, sb, sa, pa, pb, w,
                                              NoHook{}, &next);
    if (MASKED && 64 * (u + 1) + 64 > wave_all) mask_scores(sb, limit - 64 * (u + 1) - 32, hi);
  };
  if (n_steps > 0) {
    const Src k0 = src_of(kbase, p.ks, 0, false, true), k1 = src_of(kbase, p.ks, 1, false, true);
    const Src v0 = src_of(vbase, p.vs, 0, true, true);
#pragma unroll
    for (int s = 0; s < T::kSegs; ++s) issue(k0, s, lds0);
#pragma unroll
    for (int s = 0; s < T::kSegs; ++s) issue(v0, s, lds0 + T::kBytes);
    // Q by way of slot 1, which K of step 1 is loaded into after the barrier
    frags_of_rows<D>(qrows, s0 + kSlot + wave * 32 * T::kPitch, lane, w.qf);
#pragma unroll
    for (int s = 0; s < T::kK; ++s) asm volatile("" : : "v"(w.qf[s]));
    sync();
    if (n_steps > 1) {
#pragma unroll
      for (int s = 0; s < T::kSegs; ++s) issue(k1, s, lds0 + kSlot);
    }
    stage<D, true, kNoSm, false>(s0, s0, f, c, sa, sb, pb, pa, w, NoHook{});
    stage<D, true, kNoSm, false>(s0 + kSub, s0, f, c, sb, sa, pa, pb, w, NoHook{});
    if (n_plain == 0) {
      mask_scores(sa, limit, hi);
      mask_scores(sb, limit - 32, hi);
    }
    first_reference<D>(sa, sb, c, w);
    stage<D, false, kSmFirst, false>(s0, s0, f, c, sb, sa, pa, pb, w, NoHook{});
    int u = 0;
    for (; u + 3 < n_plain; u += 2) {
      iter(std::false_type{}, u, 0, kSlot);
      iter(std::false_type{}, u + 1, kSlot, 0);
    }
#pragma unroll 1
    for (; u + 1 < n_steps; ++u) {
      const uint32_t at = (u & 1) * kSlot;
      iter(std::true_type{}, u, at, kSlot - at);
    }
    const lds_u8* const cur = s0 + ((n_steps - 1) & 1) * kSlot;
    sync();
    stage<D, false, kSmSecond, true>(s0, cur, f, c, sb, sb, pb, pa, w, NoHook{});
    stage<D, false, kNoSm, true>(s0, cur + kSub, f, c, sa, sb, pa, pb, w, NoHook{});
  }
  leave_rows<D>(p, w, sp, split, p.n_split, head, r0, rows, limit, wave, lane, s0,
                [&](int64_t tok, int64_t hd, int lim, float mu, float inv, float* part) {
                  redo_row<D>(p.q + tok * p.qs + hd * p.qh, kbase, vbase, p.ks, p.vs, lim, c, mu, inv,
                              p.out + tok * p.os + hd * p.oh, part, lane);
                });
}

// The splits of a row joined: D / 4 threads a row, four head-dims each. Bound by
// memory (512 rows of 32 heads, four splits, head_dim 128: 7.8 us, 4.9 TB/s).
template <int D>
__global__ void __launch_bounds__(256) packed_merge_kernel(FwdArgs p) {
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

extern "C" int veda_packed_fwd(const void* q, int64_t q_stride_s, int64_t q_stride_h, const void* k,
                               int64_t k_stride_s, int64_t k_stride_h, const void* v,
                               int64_t v_stride_s, int64_t v_stride_h, int64_t q_rows,
                               int64_t k_rows, int64_t n_heads, int64_t n_kv_heads, int64_t head_dim,
                               const int32_t* cu_q, const int32_t* cu_k, int64_t n_seq, int causal,
                               float scale, int64_t n_split, void* out, int64_t o_stride_s,
                               int64_t o_stride_h, float* lse, void* workspace,
                               int64_t workspace_bytes, void* stream) {
  VEDA_REQUIRE(head_dim == 64 || head_dim == 128, "packed_fwd: head_dim must be 64 or 128, got %lld",
               (long long)head_dim);
  VEDA_REQUIRE(n_kv_heads > 0 && n_heads > 0 && n_heads % n_kv_heads == 0,
               "packed_fwd: %lld query heads are no multiple of %lld key heads", (long long)n_heads,
               (long long)n_kv_heads);
  VEDA_REQUIRE(n_heads / n_kv_heads <= kMaxGroup, "packed_fwd: at most %lld query heads to a key head, got %lld",
               (long long)kMaxGroup, (long long)(n_heads / n_kv_heads));
  VEDA_REQUIRE(q_rows >= 0 && k_rows >= 0 && n_seq >= 0, "packed_fwd: negative size");
  VEDA_REQUIRE(q_rows * n_heads <= 0x7fffff00 && k_rows <= 0x7fffff00 && n_seq < (1 << 20),
               "packed_fwd: q_rows x heads or k_rows past 2^31 - 256, or 2^20 sequences");
  VEDA_REQUIRE(scale > 0.f && scale < INFINITY, "packed_fwd: scale must be positive and finite");
  VEDA_REQUIRE(rows16(q, q_stride_s, q_stride_h) && rows16(k, k_stride_s, k_stride_h) &&
                   rows16(v, v_stride_s, v_stride_h) && rows16(out, o_stride_s, o_stride_h),
               "packed_fwd: q, k, v and out rows must be 16-byte aligned");
  // the LDS loads address a 64-row step with 32-bit byte offsets
  VEDA_REQUIRE(k_stride_s >= 0 && v_stride_s >= 0 && k_stride_s < (1 << 24) && v_stride_s < (1 << 24),
               "packed_fwd: row stride of k or v negative or too large");
  if (q_rows == 0) return VEDA_OK;
  FwdArgs p{};
  p.pk = Packing{cu_q, cu_k, (int32_t)n_seq, (int32_t)q_rows, (int32_t)k_rows, (int32_t)n_kv_heads,
                 (int32_t)(n_heads / n_kv_heads), causal ? 1 : 0,
                 ranked(n_seq, q_rows * n_heads / kRows * n_split), 0};
  p.q = static_cast<const uint16_t*>(q);
  p.k = static_cast<const uint16_t*>(k);
  p.v = static_cast<const uint16_t*>(v);
  p.qs = q_stride_s; p.qh = q_stride_h;
  p.ks = k_stride_s; p.kh = k_stride_h;
  p.vs = v_stride_s; p.vh = v_stride_h;
  p.out = static_cast<uint16_t*>(out);
  p.os = o_stride_s; p.oh = o_stride_h;
  p.lse = lse;
  p.scale_log2 = scale * 1.4426950408889634f;
  const int64_t slots = slots_of(q_rows, p.pk.group, n_seq);
  VEDA_REQUIRE(n_split >= 1 && n_split <= 64, "packed_fwd: n_split %lld outside [1, 64]",
               (long long)n_split);
  // a launch holds less than 2^32 threads
  VEDA_REQUIRE(slots * n_kv_heads * n_split < (1 << 24) &&
                   (n_split == 1 || q_rows * n_heads < (1 << 27)),
               "packed_fwd: too many rows for one launch");
  const int64_t need = n_split == 1 ? 0 : n_split * q_rows * n_heads * (head_dim + 2) * 4;
  VEDA_REQUIRE(need == 0 || (workspace != nullptr && rows16(workspace, 0, 0) && workspace_bytes >= need),
               "packed_fwd: workspace needs %lld bytes (16-byte aligned), got %lld", (long long)need,
               (long long)workspace_bytes);
  p.part = static_cast<float*>(workspace);
  p.n_split = (int32_t)n_split;
  p.per_group = per_group_of((uint32_t)p.pk.group);
  p.n_slots = (int32_t)slots;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const unsigned grid = (unsigned)(slots * n_kv_heads * n_split);
  if (head_dim == 128)
    packed_fwd_kernel<128><<<grid, kThreads, 0, s>>>(p);
  else
    packed_fwd_kernel<64><<<grid, kThreads, 0, s>>>(p);
  if (n_split > 1) {
    if (int rc = check_launch("packed_fwd")) return rc;
    const unsigned join = (unsigned)((q_rows * n_heads * (head_dim / 4) + 255) / 256);
    if (head_dim == 128)
      packed_merge_kernel<128><<<join, 256, 0, s>>>(p);
    else
      packed_merge_kernel<64><<<join, 256, 0, s>>>(p);
  }
  return check_launch("packed_fwd");
}
