// The walk over keys of the packed and paged forwards: scores, softmax and products
// of a wave's 32 rows with 32 keys at a time, pipelined over three of them; and how
// its results leave.
#pragma once

#include "packed_common.h"

namespace veda {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr float kLn2 = 0.6931471805599453f;

// ---------------------------------------------------------------------------
// The walk of the dense forward (attention.hip, head_dim 128 alone: what is mended in
// one is for the other too), with its own tiles and masks.
//
// A stage works on three consecutive 32-key sub-blocks at once: the score
// products of sub-block n + 1 (QK: K rows at `kb` into sn), the softmax of n (SM:
// scores sp into the packed probabilities pn) and the P V products of n - 1 (PV: V
// rows at `vb`, probabilities pp), written out in turn with scheduling fences, so
// that a wave's vector and matrix work run at once. A stage is one basic block:
// a branch inside it would make the compiler move the softmax out of it or keep
// O twice, so O's rescale waits for the next stage's start (alpha).
//
// The reference of a row is the maximum of its first step; later probabilities
// are taken against it as it stands, with no maximum taken, unless a lane's 16
// sum to kLazyLimit or more, or are not finite, or a row has no reference yet:
// then the sub-block raises the references that a score passes by 2^8 and takes
// its probabilities again.

constexpr float kLazyLimit = 256.f;
constexpr float kRescaleSlack = 8.f;  // log2 units

template <int D>
struct Wave {
  bf16x8 qf[Tile<D>::kK];
  f32x16 o[Tile<D>::kT];
  float m_run, l_run, mu;  // mu: m_run, or 0 where there is none
  float alpha;             // what O is still to be scaled by
  bool have_ref;           // every row of the wave has a reference
  float first_sum;         // of a step's first sub-block, until the second's joins it
};

enum { kNoSm = 0, kSmFirst = 1, kSmSecond = 2 };

template <int D>
__device__ __forceinline__ void raise_reference(const f32x16& s, float c, u32x4 (&pk)[2], Wave<D>& w) {
  float top = -INFINITY;
#pragma unroll
  for (int e = 0; e < 16; ++e) top = fmaxf(top, s[e]);
  top = half_swap_max(top) * c;
  const float m_new = top > w.m_run + kRescaleSlack ? top : w.m_run;
  const float mu = m_new == -INFINITY ? 0.f : m_new;
  w.alpha = __builtin_amdgcn_exp2f(w.m_run - mu);
  w.m_run = m_new;
  w.mu = mu;
  float l4[4];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float a = __builtin_amdgcn_exp2f(fmaf(s[2 * j], c, -mu));
    const float b = __builtin_amdgcn_exp2f(fmaf(s[2 * j + 1], c, -mu));
    l4[j >> 1] = (j & 1) ? l4[j >> 1] + (a + b) : a + b;
    pk[j >> 2][j & 3] = pack_bf16x2(a, b);
  }
  w.l_run = fmaf(w.l_run, w.alpha, (l4[0] + l4[1]) + (l4[2] + l4[3]));
  w.have_ref = __ballot(m_new != -INFINITY) == ~0ull;
}

template <int D>
__device__ __forceinline__ void first_reference(const f32x16& sa, const f32x16& sb, float c, Wave<D>& w) {
  float top = -INFINITY;
#pragma unroll
  for (int e = 0; e < 16; ++e) top = fmaxf(top, fmaxf(sa[e], sb[e]));
  w.m_run = half_swap_max(top) * c;
  w.mu = w.m_run == -INFINITY ? 0.f : w.m_run;
  w.have_ref = __ballot(w.m_run != -INFINITY) == ~0ull;
}

// Scores of keys that a row does not see; lim: the row's keys less the
// sub-block's first one.
__device__ __forceinline__ void mask_scores(f32x16& s, int lim, int hi) {
  const int l = lim - 4 * hi;
#pragma unroll
  for (int e = 0; e < 16; ++e)
    if (8 * (e >> 2) + (e & 3) >= l) s[e] = -INFINITY;
}

template <int D>
struct Frags {
  uint32_t k[Tile<D>::kK];  // K row li, chunk 2 s + hi
  uint32_t v[Tile<D>::kT];  // transposed reads of V
};

// First fragments of the stage that follows on the same slots, read in the place
// of a stage's last reads, so that its products do not begin with a wait.
template <int D>
struct Next {
  bf16x8 k[Tile<D>::kK / 2];
  bf16x8 v;
};
enum { kNoNext = 0, kReadNext = 1, kTakeNext = 2 };

template <int D>
__device__ __forceinline__ bf16x8 vt_frag(const lds_u8* vb, const Frags<D>& f, int i) {
  const lds_u8* a = vb + (i / Tile<D>::kT) * 16 * Tile<D>::kPitch + f.v[i % Tile<D>::kT];
  return join_tr(a, a + 8 * Tile<D>::kPitch);
}

// The end of a sub-block's softmax: its sums l4 to the row's, or its probabilities again
// against a raised reference.
template <int D, int SM>
__device__ __forceinline__ void take_sums(const float (&l4)[4], const f32x16& sp, float c, u32x4 (&pn)[2],
                                          Wave<D>& w) {
  const float sum = (l4[0] + l4[1]) + (l4[2] + l4[3]);
  if (__builtin_expect(!(w.have_ref && __ballot(sum < kLazyLimit) == ~0ull), 0)) {
    if (SM == kSmSecond) w.l_run += w.first_sum;
    w.first_sum = 0.f;
    raise_reference<D>(sp, c, pn, w);
  } else if (SM == kSmFirst) {
    w.first_sum = sum;
  } else {
    w.l_run += w.first_sum + sum;
  }
}

template <int D, bool QK, int SM, bool PV, int NEXT = kNoNext, typename Hook>
__device__ __forceinline__ void stage(const lds_u8* kb, const lds_u8* vb, const Frags<D>& f, float c,
                                      f32x16& sn, const f32x16& sp, u32x4 (&pn)[2],
                                      const u32x4 (&pp)[2], Wave<D>& w, Hook hook,
                                      Next<D>* next = nullptr) {
  using T = Tile<D>;
  constexpr int kAhead = T::kK / 2;          // K fragments ahead of their products
  constexpr int kEvery = 8 / T::kK;          // pieces for a product of each kind
  constexpr int kSub = 32 * T::kPitch;       // bytes of 32 rows
  if (PV && __any(w.alpha != 1.f)) {
#pragma unroll
    for (int t = 0; t < T::kT; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) w.o[t][e] *= w.alpha;
  }
  bf16x8 kf[T::kK], va[T::kK];
  if (QK) {
    sn = zero16();
#pragma unroll
    for (int k = 0; k < kAhead; ++k) kf[k] = NEXT == kTakeNext ? next->k[k] : lds_frag(kb + f.k[k]);
  }
  if (PV) va[0] = NEXT == kTakeNext ? next->v : vt_frag<D>(vb, f, 0);
  float l4[4];
  const float mu = w.mu;
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    hook(j);
    const int i = j / kEvery;
    if (QK && j % kEvery == 0) {
      if (i + kAhead < T::kK) kf[i + kAhead] = lds_frag(kb + f.k[i + kAhead]);
      else if (NEXT == kReadNext) next->k[i - kAhead] = lds_frag(kb + kSub + f.k[i - kAhead]);
      sn = mfma32(kf[i], w.qf[i], sn);
    }
    if (SM != kNoSm) {
      const float a = __builtin_amdgcn_exp2f(fmaf(sp[2 * j], c, -mu));
      const float b = __builtin_amdgcn_exp2f(fmaf(sp[2 * j + 1], c, -mu));
      l4[j >> 1] = (j & 1) ? l4[j >> 1] + (a + b) : a + b;
      uint32_t pk = pack_bf16x2(a, b);
      asm volatile("" : "+v"(pk));  // kept here, not sunk to its use a stage later
      pn[j >> 2][j & 3] = pk;
    }
    if (PV && j % kEvery == kEvery - 1) {
      if (i + 1 < T::kK) va[i + 1] = vt_frag<D>(vb, f, i + 1);
      else if (NEXT == kReadNext) next->v = vt_frag<D>(vb + kSub, f, 0);
      w.o[i % T::kT] = mfma32(va[i], as_bf16x8(pp[i / T::kT]), w.o[i % T::kT]);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  w.alpha = 1.f;
  if (SM != kNoSm) take_sums<D, SM>(l4, sp, c, pn, w);
}

// A wave's rows once the walk is done: out and lse, or, of one of several `splits` of the
// keys, the split's O, reference (log2) and sum of weights; O leaves as whole rows, by way of
// the wave's part of the ring. again(token, head, limit, reference, 1 / l, part):
// forms a row anew whose O came out with a NaN though its sum of weights has none.
// limit: the keys that the lane's row sees.
template <int D, typename Args, typename Again>
__device__ __forceinline__ void leave_rows(const Args& p, const Wave<D>& w, const Span& sp, int split,
                                           int splits, int head, int r0, int rows, int limit, int wave, int lane,
                                           lds_u8* s0, Again again) {
  using T = Tile<D>;
  const int li = lane & 31, hi = lane >> 5;
  const int r = r0 + 32 * wave + li;
  const bool real = r < rows;
  const int64_t token = sp.q0 + r / p.pk.group;
  const int64_t qhead = (int64_t)head * p.pk.group + r % p.pk.group;
  const float m_run = w.m_run, l_run = w.l_run;
  const f32x16(&o)[T::kT] = w.o;
  const float l = half_swap_sum(l_run);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t n_heads = (int64_t)p.pk.n_kv * p.pk.group, all_rows = p.pk.q_rows * n_heads;
  if (p.lse != nullptr && hi == 0 && real && splits == 1)
    p.lse[token * n_heads + qhead] = l == 0.f ? -INFINITY : (m_run + __log2f(l)) * kLn2;
  bool bad = false;
#pragma unroll
  for (int t = 0; t < T::kT; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) bad |= o[t][e] != o[t][e];
  const uint64_t bad_lanes = __ballot(bad && l == l);
  uint32_t bad_rows = (uint32_t)bad_lanes | (uint32_t)(bad_lanes >> 32);
  auto redo = [&](uint32_t which) {
    while (which != 0) {
      const int rr = __builtin_ctz(which);
      which &= which - 1;
      const int row = r0 + 32 * wave + rr;
      if (row >= rows) continue;
      const int64_t tok = sp.q0 + row / p.pk.group, hd = (int64_t)head * p.pk.group + row % p.pk.group;
      const float m = __shfl(m_run, rr);
      again(tok, hd, __shfl(limit, rr), m == -INFINITY ? 0.f : m, __shfl(inv, rr),
            splits > 1 ? p.part + (split * all_rows + tok * n_heads + hd) * D : nullptr);
    }
  };
  if (splits > 1) {
    if (real) {
      const int64_t at = split * all_rows + token * n_heads + qhead;
      if (hi == 0)
        *reinterpret_cast<f32x2*>(p.part + p.n_split * all_rows * D + 2 * at) = f32x2{m_run, l};
      if (!((bad_rows >> li) & 1)) {
#pragma unroll
        for (int t = 0; t < T::kT; ++t)
#pragma unroll
          for (int g = 0; g < 4; ++g)
            *reinterpret_cast<f32x4*>(p.part + at * D + 32 * t + 8 * g + 4 * hi) =
                f32x4{o[t][4 * g], o[t][4 * g + 1], o[t][4 * g + 2], o[t][4 * g + 3]};
      }
    }
    redo(bad_rows);
    return;
  }
  __syncthreads();  // every wave is done with the ring
  lds_u8* const stage = s0 + wave * 32 * T::kPitch;
#pragma unroll
  for (int t = 0; t < T::kT; ++t)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<__attribute__((address_space(3))) u32x2*>(
          stage + li * T::kPitch + (((4 * t + g) ^ swz_row<D>(li)) << 4) + 8 * hi) =
          u32x2{pack_bf16x2(o[t][4 * g] * inv, o[t][4 * g + 1] * inv),
                pack_bf16x2(o[t][4 * g + 2] * inv, o[t][4 * g + 3] * inv)};
  asm volatile("" ::: "memory");
  uint16_t* const orow = p.out + token * p.os + qhead * p.oh;
  const uint64_t obits = reinterpret_cast<uintptr_t>(orow);
#pragma unroll
  for (int i = 0; i < 32 / T::kSegRows; ++i) {
    const int rr = i * T::kSegRows + lane / T::kChunks, pos = lane % T::kChunks;
    const u32x4 x = *reinterpret_cast<const __attribute__((address_space(3))) u32x4*>(
        stage + rr * T::kPitch + ((pos ^ swz_row<D>(rr)) << 4));
    const uint32_t lo = (uint32_t)__shfl((int)(uint32_t)obits, rr);
    const uint32_t up = (uint32_t)__shfl((int)(uint32_t)(obits >> 32), rr);
    if (r0 + 32 * wave + rr < rows && !((bad_rows >> rr) & 1))
      *reinterpret_cast<u32x4*>(
          reinterpret_cast<uint16_t*>((uintptr_t)(((uint64_t)up << 32) | lo)) + 8 * pos) = x;
  }
  redo(bad_rows);
}

}  // namespace veda
