// Gradients of the attention of packed sequences (packed.hip) for gfx950. With
// P = exp(S - LSE) as the forward had it and, for a query row,
// D = dO . O - dLSE:
//   dP = dO V^T,  dS = P (dP - D)
//   dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO
// dK and dV of a key head add up over the query heads of its group.
//
// Two kernels, none of them atomic: every gradient row is written by one
// workgroup, so the result does not depend on scheduling.
//   packed_dq_kernel   128 packed rows (packed_common.h) of one key head, the
//       keys in steps of 64. It forms D from its rows of O and dO and leaves
//       [LSE log2 e | -D] of every 64 rows as a record for the other kernel.
//       Transposed products (S^T = K Q^T): a lane owns a query row.
//       The dS of a row sum to dLSE. With D from the bf16 O they do not: D is
//       off by 2^-9 of |dO| |O| and every dS by 2^-9 of itself, and what their
//       sum is off by meets the row's mean key P K, which is no small vector
//       where keys have a direction in common. So the kernel adds up dS (exact,
//       which mends D for the records) and its rounded values, forms P K with
//       the products' A operand that dS K has read already, and takes the
//       rounded sum's excess times P K off dQ. Distance of dQ from 64 bits at
//       8,192 tokens x 28 heads: 1.1e-2 -> 2.1e-3 (bf16's own rounding is
//       1.7e-3), of dK 5e-3 -> 2.4e-3; the whole step 7 % longer.
//   packed_dkv_kernel  128 keys of one key head, the packed rows that see them
//       in steps of 64. Plain products (S = Q K^T): a lane owns a key.
// In both, P or dS goes from the accumulators straight into the B operand of
// its own accumulation (the products sum over their k index in any order, so a
// lane supplies the rows in the order in which it holds them).
#include <type_traits>

#include "packed_common.h"

namespace veda {
namespace {

constexpr int kThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kRecFloats = 128;                  // of 64 rows: LSE in log2 units, -D
constexpr int kRecBytes = 4 * kRecFloats;

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) u32x2 lds_u32x2;
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) f32x4 lds_f32x4;

struct BwdArgs {
  Packing pk;
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  const uint16_t* o;
  const uint16_t* dout;
  int64_t qs, qh, ks, kh, vs, vh, os, oh, dos, doh;
  const float* lse;   // [q_rows, H]
  const float* dlse;  // [q_rows, H] or NULL
  float* rec;         // [n_kv, q slots, 2] records
  uint16_t* dq;       // [q_rows, H, D]
  uint16_t* dk;       // [k_rows, n_kv, D]
  uint16_t* dv;
  float* part;        // [dv | dk][n_split][k_rows, n_kv, D] sums, with n_split > 1
  float scale, scale_log2;
  int32_t q_slots, k_slots, n_split;
  uint32_t per_group;  // 2^32 / group
};

// The lane's index, formed anew at each call, so that what is derived from it
// holds no register between its uses.
__device__ __forceinline__ int lane_anew() {
  int ln;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(ln));
  return ln;
}

// Offsets of a lane's reads in a tile of rows permuted by swz_both. Row reads:
// row lane % 32, chunk 2 s + lane / 32 is row_offset xor 32 s. Transposed reads:
// column block t is tr_offset xor 64 t, the next eight rows xor 8 kPitch + 32.
template <int D>
__device__ __forceinline__ uint32_t row_offset(int lane) {
  const int li = lane & 31;
  return (uint32_t)(li * Tile<D>::kPitch + (((lane >> 5) ^ swz_both<D>(li)) << 4));
}

// acc + the two bf16 of a word.
__device__ __forceinline__ float add_pair(uint32_t pair, float acc) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pair),
                                         __builtin_bit_cast(bf16x2, 0x3f803f80u), acc, false);
}

// 32 rows of a wave as whole rows from its accumulators (acc[t][e] = row
// lane % 32, column 32 t + 8 (e / 4) + 4 (lane / 32) + e % 4), by way of `stage`;
// row(i) is where row i goes, or NULL.
template <int D, typename Row>
__device__ __forceinline__ void store_rows(const f32x16 (&acc)[Tile<D>::kT], float scale,
                                           lds_u8* stage, int lane, Row row) {
  using T = Tile<D>;
  const int li = lane & 31, hi = lane >> 5;
#pragma unroll
  for (int t = 0; t < T::kT; ++t)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<lds_u32x2*>(stage + li * T::kPitch + (((4 * t + g) ^ swz_row<D>(li)) << 4) + 8 * hi) =
          u32x2{pack_bf16x2(acc[t][4 * g] * scale, acc[t][4 * g + 1] * scale),
                pack_bf16x2(acc[t][4 * g + 2] * scale, acc[t][4 * g + 3] * scale)};
  asm volatile("" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32 / T::kSegRows; ++i) {
    const int rr = i * T::kSegRows + lane / T::kChunks, pos = lane % T::kChunks;
    const u32x4 x =
        *reinterpret_cast<const lds_u32x4*>(stage + rr * T::kPitch + ((pos ^ swz_row<D>(rr)) << 4));
    uint16_t* to = row(rr);
    if (to != nullptr) *reinterpret_cast<u32x4*>(to + 8 * pos) = x;
  }
  asm volatile("" ::: "memory");
}

// Four products a pair. Bound by power as the forward is: 8,192 tokens, 28 heads on
// 4, 847 us, 1.14 PFLOP/s, the matrix cores busy 62 % of 1.8 GHz.
template <int D>
__global__ void __launch_bounds__(kThreads, 2) packed_dq_kernel(BwdArgs p) {
  using T = Tile<D>;
  constexpr int kSlot = 2 * T::kBytes;  // K and V of a step
  // of head_dim 128 half of the wave's Q fragments stay in LDS: with the two
  // sums of products a row has, all of them would not fit the registers
  constexpr int kQReg = D == 128 ? T::kK / 2 : T::kK;
  __shared__ __attribute__((aligned(1024))) uint8_t ring[2][kSlot];
  __shared__ __attribute__((aligned(1024))) uint8_t qbox[D == 128 ? 4 * 4096 : 16];
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int li = lane & 31, hi = lane >> 5;
  const int head = blockIdx.x % p.pk.n_kv;
  const Span sp = span_of(p.pk, false, (int)(blockIdx.x / p.pk.n_kv), p.q_slots, p.pk.n_kv, lane);
  const int group = p.pk.group, rows = sp.nq * group;
  const int r0 = sp.tile * kRows;
  if (r0 >= rows) return;

  const int r = r0 + 32 * wave + li;
  const bool real = r < rows;
  const int last = visible_keys(p.pk, sp, min(r0 + kRows, rows) - 1);
  const int limit = real ? visible_keys(p.pk, sp, r) : 0;
  const int n_steps = (last + 63) >> 6;
  const int n_plain = r0 + kRows <= rows ? visible_keys(p.pk, sp, r0) >> 6 : 0;
  const int64_t n_heads = (int64_t)p.pk.n_kv * group;
  lds_u8* const s0 = (lds_u8*)ring[0];
  bf16x8 qf[kQReg], dof[T::kK];
  lds_u8* const qmine = (lds_u8*)qbox + wave * 4096;
  float dot = 0.f;
  {
    // Q, dO and O by way of slot 1, which is loaded into after the first barrier
    auto rows_of = [&](const uint16_t* x, int64_t s, int64_t h) {
      return load_rows<D>(x + (int64_t)sp.q0 * s + (int64_t)head * group * h, s, h, group, p.per_group,
                          r0 + 32 * wave, rows, lane);
    };
    const RowLoads<D> a = rows_of(p.q, p.qs, p.qh), b = rows_of(p.dout, p.dos, p.doh),
                      c = rows_of(p.o, p.os, p.oh);
    lds_u8* const box = s0 + kSlot + wave * 32 * T::kPitch;
    bf16x8 x[T::kK];
    frags_of_rows<D>(a, box, lane, x);
#pragma unroll
    for (int s = 0; s < T::kK; ++s) {
      if (s < kQReg) qf[s] = x[s];
      else *reinterpret_cast<lds_u32x4*>(qmine + ((s - kQReg) * 64 + lane) * 16) = __builtin_bit_cast(u32x4, x[s]);
    }
    frags_of_rows<D>(b, box, lane, dof);
    frags_of_rows<D>(c, box, lane, x);
#pragma unroll
    for (int s = 0; s < T::kK; ++s) {
      const u32x4 y = __builtin_bit_cast(u32x4, dof[s]), z = __builtin_bit_cast(u32x4, x[s]);
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        dot = fmaf(bf16_to_f32(y[m] & 0xffffu), bf16_to_f32(z[m] & 0xffffu), dot);
        dot = fmaf(bf16_to_f32(y[m] >> 16), bf16_to_f32(z[m] >> 16), dot);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  dot = half_swap_sum(dot);
  // a row without keys, and a row past the last, has P = exp2(-inf) = 0
  float lse2 = INFINITY, nd = 0.f;
  if (real) {
    const int64_t at = (sp.q0 + r / group) * n_heads + (int64_t)head * group + r % group;
    const float l = p.lse[at];
    lse2 = l == -INFINITY ? INFINITY : l * kLog2e;
    nd = (p.dlse != nullptr ? p.dlse[at] : 0.f) - dot;
  }

  const uint16_t* kbase = p.k + (int64_t)sp.k0 * p.ks + head * p.kh;
  const uint16_t* vbase = p.v + (int64_t)sp.k0 * p.vs + head * p.vh;
  auto load_step = [&](int u, lds_u8* dst) {
    const int lane = lane_anew();
    const char* kb = reinterpret_cast<const char*>(kbase + (int64_t)u * 64 * p.ks);
    const char* vb = reinterpret_cast<const char*>(vbase + (int64_t)u * 64 * p.vs);
#pragma unroll
    for (int s = 0; s < T::kSegs; ++s) {
      const int seg = T::kSegs * wave + s;
      const int row = seg * T::kSegRows + lane / T::kChunks, pos = lane % T::kChunks;
      const uint32_t src = (uint32_t)min(row, sp.nk - 1 - 64 * u);
      dma16(kb, src * (uint32_t)(2 * p.ks) + ((pos ^ swz_both<D>(row)) << 4), dst + seg * 1024);
      dma16(vb, src * (uint32_t)(2 * p.vs) + ((pos ^ swz_both<D>(row)) << 4),
            dst + T::kBytes + seg * 1024);
    }
  };
  f32x16 acc[T::kT], mean[T::kT];  // dS K, P K
#pragma unroll
  for (int t = 0; t < T::kT; ++t) acc[t] = mean[t] = zero16();
  float sum = 0.f, sum_r = 0.f;  // of dS, and of dS as rounded
  const float c = p.scale_log2;

  if (n_steps > 0) load_step(0, s0);
  // MASK: some row does not see some key of the steps
  auto walk = [&](auto mask, int from, int to) __attribute__((always_inline)) {
    constexpr bool MASK = decltype(mask)::value;
#pragma unroll 1
    for (int u = from; u < to; ++u) {
      const lds_u8* cur = s0 + (u & 1) * kSlot;
      VEDA_WAIT_VM(0);
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (u + 1 < n_steps) load_step(u + 1, s0 + ((u + 1) & 1) * kSlot);
#pragma unroll 1
      for (int sub = 0; sub < 2; ++sub) {
        const int ln = lane_anew();
        const uint32_t ra = row_offset<D>(ln), ta = tr_offset<D>(ln, 0, 0, swz_both<D>);
        const lds_u8* ks = cur + sub * 32 * T::kPitch;
        const lds_u8* vs = ks + T::kBytes;
        f32x16 st = zero16(), dp;
#pragma unroll
        for (int e = 0; e < 16; ++e) dp[e] = nd;
        bf16x8 ka[T::kK], va[T::kK];
        ka[0] = lds_frag(ks + ra);
        ka[1] = lds_frag(ks + (ra ^ 32));
#pragma unroll
        for (int s = 0; s < T::kK; ++s) {
          if (s + 2 < T::kK) ka[s + 2] = lds_frag(ks + (ra ^ (32 * (s + 2))));
          else va[s + 2 - T::kK] = lds_frag(vs + (ra ^ (32 * (s + 2 - T::kK))));
          st = mfma32(ka[s], s < kQReg ? qf[s % kQReg] : lds_frag(qmine + ((s - kQReg) * 64 + ln) * 16), st);
          __builtin_amdgcn_sched_barrier(0);
        }
        // dP - D, and the probabilities under its products
        const int lim = limit - 64 * u - 32 * sub - 4 * hi;
        auto sees = [&](int e) { return !MASK || 8 * (e >> 2) + (e & 3) < lim; };
        constexpr int kPer = 16 / T::kK;
        float pr[16];
        u32x4 pb[2], db[2];
#pragma unroll
        for (int s = 0; s < T::kK; ++s) {
          if (s + 2 < T::kK) va[s + 2] = lds_frag(vs + (ra ^ (32 * (s + 2))));
          dp = mfma32(va[s], dof[s], dp);
#pragma unroll
          for (int m = 0; m < kPer; ++m) {
            const int e = kPer * s + m;
            const float x = __builtin_amdgcn_exp2f(fmaf(st[e], c, -lse2));
            pr[e] = sees(e) ? x : 0.f;
            if (e & 1) pb[e >> 3][(e >> 1) & 3] = pack_bf16x2(pr[e - 1], pr[e]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        auto tr = [&](int i) {  // keys 16 (i / kT), column block i % kT
          const lds_u8* a = ks + (i / T::kT) * 16 * T::kPitch;
          const uint32_t at = ta ^ (64 * (i % T::kT));
          return join_tr(a + at, a + (at ^ (8 * T::kPitch + 32)));
        };
        // dS of two keys (pair j of the lane's eight)
        auto pair = [&](int j) {
          float ds[2];
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            const int e = 2 * j + m;
            ds[m] = sees(e) ? pr[e] * dp[e] : 0.f;
          }
          const uint32_t y = pack_bf16x2(ds[0], ds[1]);
          db[j >> 2][j & 3] = y;
          sum += ds[0] + ds[1];
          sum_r = add_pair(y, sum_r);
        };
        // dS K and P K, the second 16 keys' dS under the first's products
        bf16x8 kt[2 * T::kT];
        kt[0] = tr(0);
#pragma unroll
        for (int j = 0; j < 4; ++j) pair(j);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 2 * T::kT; ++i) {
          if (i + 1 < 2 * T::kT) kt[i + 1] = tr(i + 1);
          acc[i % T::kT] = mfma32(kt[i], as_bf16x8(db[i / T::kT]), acc[i % T::kT]);
          if (i < T::kT) {
#pragma unroll
            for (int j = 0; j < 4 / T::kT; ++j) pair(4 + i * (4 / T::kT) + j);
          }
          mean[i % T::kT] = mfma32(kt[i], as_bf16x8(pb[i / T::kT]), mean[i % T::kT]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  };
  walk(std::false_type{}, 0, min(n_plain, n_steps));
  walk(std::true_type{}, min(n_plain, n_steps), n_steps);
  // (the row's place again, from the lane's index: held through the walk it
  // would cost the registers that the products need)
  const int ln = lane_anew();
  const int row = r0 + 32 * wave + (ln & 31);
  const int64_t at = (sp.q0 + row / group) * n_heads + (int64_t)head * group + row % group;
  // dS of a row sums to dLSE: what its rounded values sum to beside that has
  // gone to the row's mean key, and -D is off by what the exact ones do
  sum = half_swap_sum(sum);
  sum_r = half_swap_sum(sum_r);
  const float dl = row < rows && p.dlse != nullptr && lse2 != INFINITY ? p.dlse[at] : 0.f;
  if (ln < 32) {
    const int slot = first_q_slot(p.pk, sp) + sp.tile;
    float* rec = p.rec + (((int64_t)head * p.q_slots + slot) * 2 + (wave >> 1)) * kRecFloats;
    rec[32 * (wave & 1) + ln] = lse2;
    rec[64 + 32 * (wave & 1) + ln] = nd - (sum - dl);
  }
#pragma unroll
  for (int t = 0; t < T::kT; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[t][e] = fmaf(dl - sum_r, mean[t][e], acc[t][e]);
  __syncthreads();  // every wave is done with the ring
  const uint64_t bits = reinterpret_cast<uintptr_t>(p.dq + at * D);
  store_rows<D>(acc, p.scale, s0 + wave * 32 * T::kPitch, ln, [&](int rr) {
    const uint32_t lo = (uint32_t)__shfl((int)(uint32_t)bits, rr);
    const uint32_t up = (uint32_t)__shfl((int)(uint32_t)(bits >> 32), rr);
    return r0 + 32 * wave + rr < rows
               ? reinterpret_cast<uint16_t*>((uintptr_t)(((uint64_t)up << 32) | lo))
               : nullptr;
  });
}

// Four products a pair: the same tokens 889 us, 1.08 PFLOP/s, busy 58 %.
template <int D>
__global__ void __launch_bounds__(kThreads, 2) packed_dkv_kernel(BwdArgs p) {
  using T = Tile<D>;
  constexpr int kSlot = 2 * T::kBytes + 1024;  // Q, dO and the record of a step
  constexpr int kProducts = 2 * T::kT;         // of an accumulation over 32 rows
  __shared__ __attribute__((aligned(1024))) uint8_t ring[2][kSlot];
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int li = lane & 31, hi = lane >> 5;
  const int head = blockIdx.x % p.pk.n_kv;
  const int item = (int)(blockIdx.x / p.pk.n_kv);
  const int split = item % p.n_split;
  const Span sp = span_of(p.pk, true, item / p.n_split, p.k_slots, p.pk.n_kv * p.n_split, lane);
  const int j0 = sp.tile * kRows;
  if (j0 >= sp.nk) return;
  const int group = p.pk.group, rows = sp.nq * group;
  // key j is seen by the rows from first(j) on
  auto first = [&](int j) {
    const int64_t i = (int64_t)j - (sp.nk - sp.nq);
    return p.pk.causal ? (int)min(max(i * group, (int64_t)0), (int64_t)rows) : 0;
  };
  // The steps that see the tile, from the last row down, every n_split-th of
  // them here: the workgroups of a head then walk the same rows at about the same
  // time, and find them in L2 (from each tile's own first row up, they did not).
  const int first_step = first(j0) >> 6, end_step = (rows + 63) >> 6;
  const int top = end_step - 1 - split;
  const int n_steps = top >= first_step ? (top - first_step) / p.n_split + 1 : 0;
  auto step = [&](int k) { return top - k * p.n_split; };
  const int w0 = j0 + 32 * wave;                       // this wave's keys
  const int key = min(w0 + li, sp.nk - 1);
  const int mine = first(key);
  const int live_from = __builtin_amdgcn_readfirstlane(first(w0));
  const int full_from = __builtin_amdgcn_readfirstlane(first(w0 + 31));
  const bool live = w0 < sp.nk;

  bf16x8 kf[T::kK], vf[T::kK];
  {
    const uint16_t* kr = p.k + (int64_t)(sp.k0 + key) * p.ks + head * p.kh + 8 * hi;
    const uint16_t* vr = p.v + (int64_t)(sp.k0 + key) * p.vs + head * p.vh + 8 * hi;
#pragma unroll
    for (int s = 0; s < T::kK; ++s) {
      kf[s] = as_bf16x8(ld16(kr + 16 * s));
      vf[s] = as_bf16x8(ld16(vr + 16 * s));
    }
  }
  f32x16 acc_v[T::kT], acc_k[T::kT];
#pragma unroll
  for (int t = 0; t < T::kT; ++t) acc_v[t] = acc_k[t] = zero16();
  const float c = p.scale_log2;
  // records of the sequence's rows: its first query slot's on
  const float* recs = p.rec + ((int64_t)head * p.q_slots + first_q_slot(p.pk, sp)) * 2 * kRecFloats;
  const uint16_t* qhead = p.q + (int64_t)sp.q0 * p.qs + (int64_t)head * group * p.qh;
  const uint16_t* dhead = p.dout + (int64_t)sp.q0 * p.dos + (int64_t)head * group * p.doh;

  // The steps' rows are loaded in turn: t0, rem are the next step's first token
  // and head. Row x from there is token x / group by a product with 2^32 / group
  // (exact: x < 63 + group, kMaxGroup).
  int t0 = 0, rem = 0;
  if (n_steps > 0) {
    t0 = (int)((int64_t)64 * top / group);
    rem = (int)((int64_t)64 * top - (int64_t)t0 * group);
  }
  const int t_step = 64 * p.n_split / group, r_step = 64 * p.n_split - t_step * group;
  auto load_step = [&](int u, lds_u8* dst) {
    const int lane = lane_anew();
    const char* qb = reinterpret_cast<const char*>(qhead + (int64_t)t0 * p.qs);
    const char* db = reinterpret_cast<const char*>(dhead + (int64_t)t0 * p.dos);
#pragma unroll
    for (int s = 0; s < T::kSegs; ++s) {
      const int seg = T::kSegs * wave + s;
      const int row = seg * T::kSegRows + lane / T::kChunks, pos = lane % T::kChunks;
      const uint32_t x = (uint32_t)(min(row, rows - 1 - 64 * u) + rem);
      const uint32_t t = group == 1 ? x : __umulhi(x, p.per_group), g = x - t * (uint32_t)group;
      const uint32_t ch = (uint32_t)((pos ^ swz_both<D>(row)) << 4);
      dma16(qb, t * (uint32_t)(2 * p.qs) + g * (uint32_t)(2 * p.qh) + ch, dst + seg * 1024);
      dma16(db, t * (uint32_t)(2 * p.dos) + g * (uint32_t)(2 * p.doh) + ch,
            dst + T::kBytes + seg * 1024);
    }
    t0 -= t_step;
    rem -= r_step;
    if (rem < 0) {
      rem += group;
      --t0;
    }
    if (wave == 0)
      dma16(reinterpret_cast<const char*>(recs + (int64_t)u * kRecFloats), (uint32_t)((lane & 31) * 16),
            dst + 2 * T::kBytes);
  };

  // rows 32 b .. + 31 of step u; MASK: some of them do not see all of the keys
  auto compute = [&](auto mask, int u, int b, const lds_u8* cur) __attribute__((always_inline)) {
    constexpr bool MASK = decltype(mask)::value;
    const int ln = lane_anew(), hi = ln >> 5;
    const uint32_t ra = row_offset<D>(ln);
    const uint32_t ta = tr_offset<D>(ln, 0, 0, swz_both<D>);
    const lds_u8* qs = cur + b * 32 * T::kPitch;
    const lds_u8* ds = qs + T::kBytes;
    const lds_u8* rec = cur + 2 * T::kBytes + 128 * b + 16 * hi;  // rows 8 m + 4 hi + {0..3}: + 32 m
    f32x16 st = zero16(), dp;
    bf16x8 qa[T::kK], da[T::kK];
    qa[0] = lds_frag(qs + ra);
    qa[1] = lds_frag(qs + (ra ^ 32));
#pragma unroll
    for (int s = 0; s < T::kK; ++s) {
      if (s + 2 < T::kK) qa[s + 2] = lds_frag(qs + (ra ^ (32 * (s + 2))));
      else da[s + 2 - T::kK] = lds_frag(ds + (ra ^ (32 * (s + 2 - T::kK))));
      if (s >= T::kK - 4) {
        const int m = s - (T::kK - 4);
        const f32x4 nd = *reinterpret_cast<const lds_f32x4*>(rec + 256 + 32 * m);
#pragma unroll
        for (int e = 0; e < 4; ++e) dp[4 * m + e] = nd[e];
      }
      st = mfma32(qa[s], kf[s], st);
      __builtin_amdgcn_sched_barrier(0);
    }
    // dP - D, and the probabilities under its products
    constexpr int kPer = 16 / T::kK;
    u32x4 pp[2], pd[2];
    float pr[16];
    f32x4 l4;
    const int lim = mine - 64 * u - 32 * b - 4 * hi;
#pragma unroll
    for (int s = 0; s < T::kK; ++s) {
      if (s + 2 < T::kK) da[s + 2] = lds_frag(ds + (ra ^ (32 * (s + 2))));
      dp = mfma32(da[s], vf[s], dp);
#pragma unroll
      for (int m = 0; m < kPer; ++m) {
        const int e = kPer * s + m;
        if ((e & 3) == 0) l4 = *reinterpret_cast<const lds_f32x4*>(rec + 8 * e);
        pr[e] = __builtin_amdgcn_exp2f(fmaf(st[e], c, -l4[e & 3]));
        if (MASK) pr[e] = 8 * (e >> 2) + (e & 3) >= lim ? pr[e] : 0.f;
        if (e & 1) pp[e >> 3][(e >> 1) & 3] = pack_bf16x2(pr[e - 1], pr[e]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    auto tr = [&](const lds_u8* base, int i) {  // 16 rows i / kT, column block i % kT
      const uint32_t at = ta ^ (64 * (i % T::kT));
      const lds_u8* x = base + (i / T::kT) * 16 * T::kPitch;
      return join_tr(x + at, x + (at ^ (8 * T::kPitch + 32)));
    };
    // dV, and dS under its products
    constexpr int kEach = 16 / kProducts;
    bf16x8 tv[kProducts], tq[kProducts];
    tv[0] = tr(ds, 0);
    tv[1] = tr(ds, 1);
#pragma unroll
    for (int i = 0; i < kProducts; ++i) {
      if (i + 2 < kProducts) tv[i + 2] = tr(ds, i + 2);
      else tq[i + 2 - kProducts] = tr(qs, i + 2 - kProducts);
      acc_v[i % T::kT] = mfma32(tv[i], as_bf16x8(pp[i / T::kT]), acc_v[i % T::kT]);
#pragma unroll
      for (int m = 0; m < kEach; m += 2) {
        const int e = kEach * i + m;
        // (a probability of 0 by the mask meets whatever dP holds there)
        const float a = MASK && pr[e] == 0.f ? 0.f : pr[e] * dp[e];
        const float y = MASK && pr[e + 1] == 0.f ? 0.f : pr[e + 1] * dp[e + 1];
        pd[e >> 3][(e >> 1) & 3] = pack_bf16x2(a, y);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int i = 0; i < kProducts; ++i) {
      if (i + 2 < kProducts) tq[i + 2] = tr(qs, i + 2);
      acc_k[i % T::kT] = mfma32(tq[i], as_bf16x8(pd[i / T::kT]), acc_k[i % T::kT]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  lds_u8* const s0 = (lds_u8*)ring[0];
  if (n_steps > 0) load_step(top, s0);
  auto walk = [&](auto mask, int from, int to) __attribute__((always_inline)) {
#pragma unroll 1
    for (int k = from; k < to; ++k) {
      const lds_u8* cur = s0 + (k & 1) * kSlot;
      const int u = step(k);
      VEDA_WAIT_VM(0);
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (k + 1 < n_steps) load_step(step(k + 1), s0 + ((k + 1) & 1) * kSlot);
      if (!live) continue;
      if (decltype(mask)::value) {
#pragma unroll 1
        for (int b = 0; b < 2; ++b)
          if (64 * u + 32 * b + 32 > live_from) compute(mask, u, b, cur);
      } else {
        compute(mask, u, 0, cur);
        compute(mask, u, 1, cur);
      }
    }
  };
  // steps from full_step on see all of the wave's keys
  const int full_step = (full_from + 63) >> 6;
  const int n_plain = top >= full_step ? min((top - full_step) / p.n_split + 1, n_steps) : 0;
  walk(std::false_type{}, 0, n_plain);
  walk(std::true_type{}, n_plain, n_steps);

  __syncthreads();  // every wave is done with the ring
  const int64_t ld = (int64_t)p.pk.n_kv * D;
  const int64_t base = (int64_t)(sp.k0 + w0) * ld + (int64_t)head * D;
  lds_u8* const stage = s0 + wave * 32 * T::kPitch;
  const int ln = lane_anew();
  if (p.n_split > 1) {
    // sums in 32 bits, joined and rounded by packed_join_kernel
    if (w0 + (ln & 31) >= sp.nk) return;
    float* to = p.part + split * ((int64_t)p.pk.k_rows * ld) + base + (ln & 31) * ld + 4 * (ln >> 5);
#pragma unroll
    for (int pass = 0; pass < 2; ++pass) {
      const f32x16(&a)[T::kT] = pass == 0 ? acc_v : acc_k;
#pragma unroll
      for (int t = 0; t < T::kT; ++t)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<f32x4*>(to + 32 * t + 8 * g) =
              f32x4{a[t][4 * g], a[t][4 * g + 1], a[t][4 * g + 2], a[t][4 * g + 3]};
      to += (int64_t)p.n_split * p.pk.k_rows * ld;
    }
    return;
  }
  store_rows<D>(acc_v, 1.f, stage, ln,
                [&](int rr) { return w0 + rr < sp.nk ? p.dv + base + rr * ld : nullptr; });
  store_rows<D>(acc_k, p.scale, stage, ln,
                [&](int rr) { return w0 + rr < sp.nk ? p.dk + base + rr * ld : nullptr; });
}

// The splits' sums of dV and dK joined: a thread four values, in the order of
// the splits. Bound by memory (8,192 tokens, 4 key heads, three splits: 117 MB in
// 17 us, 6.9 TB/s, part of it from the cache that the sums were just written to).
__global__ void __launch_bounds__(256) packed_join_kernel(const float* part, int64_t n, int n_split,
                                                          float scale, uint16_t* dv, uint16_t* dk) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  const bool is_k = blockIdx.y != 0;
  const float* x = part + (is_k ? n_split * n : 0) + i;
  f32x4 s = *reinterpret_cast<const f32x4*>(x);
  for (int k = 1; k < n_split; ++k) s += *reinterpret_cast<const f32x4*>(x + k * n);
  const float m = is_k ? scale : 1.f;
  *reinterpret_cast<u32x2*>((is_k ? dk : dv) + i) =
      u32x2{pack_bf16x2(s[0] * m, s[1] * m), pack_bf16x2(s[2] * m, s[3] * m)};
}

}  // namespace
}  // namespace veda

using namespace veda;

extern "C" int veda_packed_bwd(
    const void* q, int64_t q_stride_s, int64_t q_stride_h, const void* k, int64_t k_stride_s,
    int64_t k_stride_h, const void* v, int64_t v_stride_s, int64_t v_stride_h, const void* out,
    int64_t o_stride_s, int64_t o_stride_h, const void* dout, int64_t do_stride_s,
    int64_t do_stride_h, const float* lse, const float* dlse, int64_t q_rows, int64_t k_rows,
    int64_t n_heads, int64_t n_kv_heads, int64_t head_dim, const int32_t* cu_q,
    const int32_t* cu_k, int64_t n_seq, int causal, float scale, int64_t n_split, void* dq, void* dk, void* dv,
    void* workspace, int64_t workspace_bytes, void* stream) {
  VEDA_REQUIRE(head_dim == 64 || head_dim == 128, "packed_bwd: head_dim must be 64 or 128, got %lld",
               (long long)head_dim);
  VEDA_REQUIRE(n_kv_heads > 0 && n_heads > 0 && n_heads % n_kv_heads == 0,
               "packed_bwd: %lld query heads are no multiple of %lld key heads", (long long)n_heads,
               (long long)n_kv_heads);
  VEDA_REQUIRE(q_rows >= 0 && k_rows >= 0 && n_seq >= 0, "packed_bwd: negative size");
  VEDA_REQUIRE(q_rows * n_heads <= 0x7fffff00 && k_rows <= 0x7fffff00 && n_seq < (1 << 20),
               "packed_bwd: q_rows x heads or k_rows past 2^31 - 256, or 2^20 sequences");
  VEDA_REQUIRE(scale > 0.f && scale < INFINITY, "packed_bwd: scale must be positive and finite");
  VEDA_REQUIRE(rows16(q, q_stride_s, q_stride_h) && rows16(k, k_stride_s, k_stride_h) &&
                   rows16(v, v_stride_s, v_stride_h) && rows16(out, o_stride_s, o_stride_h) &&
                   rows16(dout, do_stride_s, do_stride_h) && rows16(dq, 0, 0) && rows16(dk, 0, 0) &&
                   rows16(dv, 0, 0),
               "packed_bwd: q, k, v, out, dout and gradient rows must be 16-byte aligned");
  // the LDS loads address a 64-row step with 32-bit byte offsets
  // (of one key head's rows: with one query head to each, no head stride)
  const bool heads = n_heads > n_kv_heads;
  const int64_t strides[] = {q_stride_s, k_stride_s, v_stride_s, do_stride_s, heads ? q_stride_h : 0,
                             heads ? do_stride_h : 0};
  for (int64_t s : strides)
    VEDA_REQUIRE(s >= 0 && s < (1 << 24), "packed_bwd: stride negative or too large");
  BwdArgs p{};
  p.pk = Packing{cu_q, cu_k, (int32_t)n_seq, (int32_t)q_rows, (int32_t)k_rows, (int32_t)n_kv_heads,
                 (int32_t)(n_heads / n_kv_heads), causal ? 1 : 0,
                 ranked(n_seq, q_rows * n_heads / kRows),
                 ranked(n_seq, k_rows * n_kv_heads / kRows * n_split)};
  VEDA_REQUIRE(p.pk.group <= kMaxGroup, "packed_bwd: at most %lld query heads to a key head, got %lld",
               (long long)kMaxGroup, (long long)p.pk.group);
  VEDA_REQUIRE(p.pk.group <= 64 || (q_stride_h * p.pk.group < (1 << 30) &&
                                    do_stride_h * p.pk.group < (1 << 30)),
               "packed_bwd: the heads of a group are too far apart");
  const int64_t q_slots = slots_of(q_rows, p.pk.group, n_seq), k_slots = slots_of(k_rows, 1, n_seq);
  VEDA_REQUIRE(n_split >= 1 && n_split <= 64, "packed_bwd: n_split %lld outside [1, 64]",
               (long long)n_split);
  const int64_t n_out = k_rows * n_kv_heads * head_dim;
  // a launch holds less than 2^32 threads
  VEDA_REQUIRE(q_slots * n_kv_heads < (1 << 24) && k_slots * n_kv_heads * n_split < (1 << 24) &&
                   (n_split == 1 || n_out < (1ll << 33)),
               "packed_bwd: too many rows for one launch");
  const int64_t rec_bytes = q_slots * n_kv_heads * 2 * kRecBytes;
  const int64_t need = rec_bytes + (n_split > 1 ? 2 * n_split * n_out * 4 : 0);
  VEDA_REQUIRE(workspace != nullptr && rows16(workspace, 0, 0) && workspace_bytes >= need,
               "packed_bwd: workspace needs %lld bytes (16-byte aligned), got %lld", (long long)need,
               (long long)workspace_bytes);
  p.q = static_cast<const uint16_t*>(q);
  p.k = static_cast<const uint16_t*>(k);
  p.v = static_cast<const uint16_t*>(v);
  p.o = static_cast<const uint16_t*>(out);
  p.dout = static_cast<const uint16_t*>(dout);
  p.qs = q_stride_s; p.qh = q_stride_h;
  p.ks = k_stride_s; p.kh = k_stride_h;
  p.vs = v_stride_s; p.vh = v_stride_h;
  p.os = o_stride_s; p.oh = o_stride_h;
  p.dos = do_stride_s; p.doh = do_stride_h;
  p.lse = lse;
  p.dlse = dlse;
  p.rec = static_cast<float*>(workspace);
  p.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + rec_bytes);
  p.n_split = (int32_t)n_split;
  p.per_group = per_group_of((uint32_t)p.pk.group);
  p.dq = static_cast<uint16_t*>(dq);
  p.dk = static_cast<uint16_t*>(dk);
  p.dv = static_cast<uint16_t*>(dv);
  p.scale = scale;
  p.scale_log2 = scale * kLog2e;
  p.q_slots = (int32_t)q_slots;
  p.k_slots = (int32_t)k_slots;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const unsigned q_grid = (unsigned)(q_slots * n_kv_heads), k_grid = (unsigned)(k_slots * n_kv_heads * n_split);
  if (q_rows > 0) {
    if (head_dim == 128) packed_dq_kernel<128><<<q_grid, kThreads, 0, s>>>(p);
    else packed_dq_kernel<64><<<q_grid, kThreads, 0, s>>>(p);
    if (int rc = check_launch("veda_packed_bwd (dq)")) return rc;
  }
  if (k_rows > 0) {
    if (head_dim == 128) packed_dkv_kernel<128><<<k_grid, kThreads, 0, s>>>(p);
    else packed_dkv_kernel<64><<<k_grid, kThreads, 0, s>>>(p);
    if (n_split > 1) {
      if (int rc = check_launch("veda_packed_bwd (dk, dv)")) return rc;
      packed_join_kernel<<<dim3((unsigned)((n_out / 4 + 255) / 256), 2), 256, 0, s>>>(
          p.part, n_out, p.n_split, scale, p.dv, p.dk);
    }
  }
  return check_launch("veda_packed_bwd (dk, dv)");
}
