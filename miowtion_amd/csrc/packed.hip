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
#include "packed_common.h"

namespace veda {
namespace {

constexpr int kThreads = 256;
constexpr float kLn2 = 0.6931471805599453f;

struct FwdArgs {
  Packing pk;
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  int64_t qs, qh, ks, kh, vs, vh;
  uint16_t* out;
  int64_t os, oh;
  float* lse;  // [q_rows, H] or NULL
  float scale_log2;
  int32_t n_slots;
};

// A row whose O came out with an infinity or a NaN, again, key by key: a key
// that the row does not see, or whose probability is zero, adds nothing
// whatever its V holds (a product with a zero probability makes a NaN of it).
// All lanes of the wave work on the row; lane l has head-dims l and l + 64.
template <int D>
__device__ __noinline__ void redo_row(const uint16_t* q, const uint16_t* k, const uint16_t* v,
                                      int64_t ks, int64_t vs, int limit, float c, float mu, float inv,
                                      uint16_t* out, int lane) {
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
  for (int m = 0; m < D / 64; ++m) out[lane + 64 * m] = (uint16_t)f32_to_bf16(acc[m] * inv);
}

template <int D>
__global__ void __launch_bounds__(kThreads, 2) packed_fwd_kernel(FwdArgs p) {
  using T = Tile<D>;
  constexpr int kSlot = 2 * T::kBytes;  // K and V of a step
  __shared__ __attribute__((aligned(1024))) uint8_t ring[2][kSlot];
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int li = lane & 31, hi = lane >> 5;
  const int head = blockIdx.x % p.pk.n_kv;
  const int slot = p.n_slots - 1 - (int)(blockIdx.x / p.pk.n_kv);
  const Span sp = span_of_slot(p.pk, false, slot, lane);
  const int rows = sp.nq * p.pk.group;
  const int r0 = sp.tile * kRows;
  if (r0 >= rows) return;

  const int r = r0 + 32 * wave + li;
  const bool real = r < rows;
  const int last = visible_keys(p.pk, sp, min(r0 + kRows, rows) - 1);
  const int limit = real ? visible_keys(p.pk, sp, r) : last;
  const int n_steps = (last + 63) >> 6;
  const int n_plain = visible_keys(p.pk, sp, r0) >> 6;  // steps that every row sees whole
  const int64_t token = sp.q0 + r / p.pk.group;
  const int64_t qhead = (int64_t)head * p.pk.group + r % p.pk.group;
  const uint16_t* qptr = p.q + token * p.qs + qhead * p.qh;
  bf16x8 qf[T::kK];
#pragma unroll
  for (int s = 0; s < T::kK; ++s)
    qf[s] = real ? as_bf16x8(ld16(qptr + 16 * s + 8 * hi)) : as_bf16x8(u32x4{0, 0, 0, 0});

  const uint16_t* kbase = p.k + (int64_t)sp.k0 * p.ks + head * p.kh;
  const uint16_t* vbase = p.v + (int64_t)sp.k0 * p.vs + head * p.vh;
  // K and V of step u; rows past the sequence's last key read that key again
  auto load_step = [&](int u, lds_u8* dst) {
    const char* kb = reinterpret_cast<const char*>(kbase + (int64_t)u * 64 * p.ks);
    const char* vb = reinterpret_cast<const char*>(vbase + (int64_t)u * 64 * p.vs);
#pragma unroll
    for (int s = 0; s < T::kSegs; ++s) {
      const int seg = T::kSegs * wave + s;
      const int row = seg * T::kSegRows + lane / T::kChunks, pos = lane % T::kChunks;
      const int src = min(row, sp.nk - 1 - 64 * u);
      dma16(kb, (uint32_t)src * (uint32_t)(2 * p.ks) + ((pos ^ swz_row<D>(row)) << 4), dst + seg * 1024);
      dma16(vb, (uint32_t)src * (uint32_t)(2 * p.vs) + ((pos ^ swz_tr<D>(row)) << 4),
            dst + T::kBytes + seg * 1024);
    }
  };
  uint32_t kro[T::kK], vro[T::kT];
#pragma unroll
  for (int s = 0; s < T::kK; ++s)
    kro[s] = (uint32_t)(li * T::kPitch + (((2 * s + hi) ^ swz_row<D>(li)) << 4));
#pragma unroll
  for (int t = 0; t < T::kT; ++t) vro[t] = T::kBytes + tr_offset<D>(lane, t, 0, swz_tr<D>);

  f32x16 o[T::kT];
#pragma unroll
  for (int t = 0; t < T::kT; ++t) o[t] = zero16();
  float m_run = -INFINITY, l_run = 0.f;
  const float c = p.scale_log2;

  lds_u8* const s0 = (lds_u8*)ring[0];
  if (n_steps > 0) load_step(0, s0);
  for (int u = 0; u < n_steps; ++u) {
    const lds_u8* cur = s0 + (u & 1) * kSlot;
    VEDA_WAIT_VM(0);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (u + 1 < n_steps) load_step(u + 1, s0 + ((u + 1) & 1) * kSlot);
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) {
      f32x16 s = zero16();
#pragma unroll
      for (int i = 0; i < T::kK; ++i)
        s = mfma32(lds_frag(cur + sub * 32 * T::kPitch + kro[i]), qf[i], s);
      if (u >= n_plain) {
        const int lim = limit - 64 * u - 32 * sub - 4 * hi;
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (8 * (e >> 2) + (e & 3) >= lim) s[e] = -INFINITY;
      }
      float top = -INFINITY;
#pragma unroll
      for (int e = 0; e < 16; ++e) top = fmaxf(top, s[e]);
      const float m_new = fmaxf(m_run, half_swap_max(top) * c);
      const float mu = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = __builtin_amdgcn_exp2f(m_run - mu);
      m_run = m_new;
      float sum = 0.f;
      u32x4 pb[2];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float a = __builtin_amdgcn_exp2f(fmaf(s[2 * j], c, -mu));
        const float b = __builtin_amdgcn_exp2f(fmaf(s[2 * j + 1], c, -mu));
        sum += a + b;
        pb[j >> 2][j & 3] = pack_bf16x2(a, b);
      }
      l_run = fmaf(l_run, alpha, sum);
#pragma unroll
      for (int t = 0; t < T::kT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[t][e] *= alpha;
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int t = 0; t < T::kT; ++t) {
          const lds_u8* a = cur + (sub * 32 + kk * 16) * T::kPitch + vro[t];
          o[t] = mfma32(join_tr(a, a + 8 * T::kPitch), as_bf16x8(pb[kk]), o[t]);
        }
    }
  }

  // O leaves as whole rows, by way of the wave's part of the ring
  const float l = half_swap_sum(l_run);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (p.lse != nullptr && hi == 0 && real)
    p.lse[token * ((int64_t)p.pk.n_kv * p.pk.group) + qhead] =
        l == 0.f ? -INFINITY : (m_run + __log2f(l)) * kLn2;
  bool bad = false;
#pragma unroll
  for (int t = 0; t < T::kT; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) bad |= !(fabsf(o[t][e]) < INFINITY);
  const uint64_t bad_lanes = __ballot(bad);
  uint32_t bad_rows = (uint32_t)bad_lanes | (uint32_t)(bad_lanes >> 32);
  __syncthreads();  // every wave is done with the ring
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
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
  while (bad_rows != 0) {
    const int rr = __builtin_ctz(bad_rows);
    bad_rows &= bad_rows - 1;
    const int row = r0 + 32 * wave + rr;
    if (row >= rows) continue;
    const int64_t tok = sp.q0 + row / p.pk.group, hd = (int64_t)head * p.pk.group + row % p.pk.group;
    const float m = __shfl(m_run, rr);
    redo_row<D>(p.q + tok * p.qs + hd * p.qh, kbase, vbase, p.ks, p.vs, __shfl(limit, rr), c,
                m == -INFINITY ? 0.f : m, __shfl(inv, rr), p.out + tok * p.os + hd * p.oh, lane);
  }
}

}  // namespace
}  // namespace veda

using namespace veda;

extern "C" int veda_packed_fwd(const void* q, int64_t q_stride_s, int64_t q_stride_h, const void* k,
                               int64_t k_stride_s, int64_t k_stride_h, const void* v,
                               int64_t v_stride_s, int64_t v_stride_h, int64_t q_rows,
                               int64_t k_rows, int64_t n_heads, int64_t n_kv_heads, int64_t head_dim,
                               const int32_t* cu_q, const int32_t* cu_k, int64_t n_seq, int causal,
                               float scale, void* out, int64_t o_stride_s, int64_t o_stride_h,
                               float* lse, void* stream) {
  VEDA_REQUIRE(head_dim == 64 || head_dim == 128, "packed_fwd: head_dim must be 64 or 128, got %lld",
               (long long)head_dim);
  VEDA_REQUIRE(n_kv_heads > 0 && n_heads > 0 && n_heads % n_kv_heads == 0,
               "packed_fwd: %lld query heads are no multiple of %lld key heads", (long long)n_heads,
               (long long)n_kv_heads);
  VEDA_REQUIRE(q_rows >= 0 && k_rows >= 0 && n_seq >= 0, "packed_fwd: negative size");
  VEDA_REQUIRE(q_rows * n_heads < (1ll << 31) && k_rows < (1ll << 31) && n_seq < (1 << 20),
               "packed_fwd: q_rows x heads or k_rows of 2^31 or more, or 2^20 sequences");
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
                 (int32_t)(n_heads / n_kv_heads), causal ? 1 : 0};
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
  VEDA_REQUIRE(slots * n_kv_heads < (1ll << 31), "packed_fwd: too many tiles");
  p.n_slots = (int32_t)slots;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const unsigned grid = (unsigned)(slots * n_kv_heads);
  if (head_dim == 128)
    packed_fwd_kernel<128><<<grid, kThreads, 0, s>>>(p);
  else
    packed_fwd_kernel<64><<<grid, kThreads, 0, s>>>(p);
  return check_launch("packed_fwd");
}
