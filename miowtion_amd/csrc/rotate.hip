// Norms of query and key heads and their rotation by position, in one pass, with
// the gradients; and the same on the way into a paged cache.
//
// For a head's row x of D values, with a weight w and positions p of its token:
//   z = x r w,  r = (mean(x^2) + eps)^-1/2
//   (y_a, y_b) = (z_a cos f - z_b sin f, z_b cos f + z_a sin f),  f = rate p[axis]
// for the pairs (a, b) of dims, each with a rate and an axis of its own; dims of
// no pair stay as they are. Pairs are dims j and j + P of P pairs, or 2 j and
// 2 j + 1. Gradients, with dz the rotation back of dy:
//   dw = sum dz x r,  dx = r (g - x r mean(g x r)),  g = dz w
//
// All of it is bound by memory: a row is read once and written once. A wave takes
// a token (or a part of its heads, where tokens are few): D / 8 lanes a row, 16
// bytes each, four rows of each lane asked for at a time. The token's angles are
// formed once, a pair by each lane, in turns and in 64 bits (a product with a far
// position has no bits of the angle left in 32), less whole turns, and then in 32
// bits by the sine and cosine instructions, which take turns (within 1.3e-7 over a
// turn); they go to the lanes of the rows by way of the wave's LDS.
//
// A clip's layer, 57,720 tokens, 48 heads of q and of k, head_dim 128: 493 us, 5.8 TB/s
// (a copy has 4.5 to 4.8); 77 tokens of 40 and 8 heads 4.2 us, of latency; 4,096 rows into a
// cache 21 us, 4.7 TB/s. Values are held in 32 bits from the load to the one rounding.
#include <type_traits>

#include "paged_common.h"

namespace veda {
namespace {

// How positions turn the pairs of a head.
struct Turn {
  const void* pos;      // [rows, axes], or NULL
  int32_t kind;         // kInt32, kInt64, kFloat32
  int64_t st, sa;       // strides of a row, of an axis
  const double* turns;  // of each pair, turns for a step of its position
  const int32_t* axes;  // of each pair
  int32_t pairs, n_axes;
};
enum { kInt32 = 0, kInt64 = 1, kFloat32 = 2 };

// Heads of a token, to be normalised and rotated.
struct Heads {
  const uint16_t* x;
  int64_t xs, xh;
  const void* w;  // [D], or NULL
  int32_t w16;    // w is bf16, else fp32
  int32_t n;
};

// How rows are moved: past the caches where they would not stay there anyway. Rows that
// are written leave the GPU's L2 from some 32 MB on (a preview's 38 MB of q and k: 16.5 us
// kept, 15.6 past it; 153 MB 60 and 48), rows that are read all caches from 256 MB on (1.4
// GB: 516 us kept, 494 past them; 153 MB 48 and 58, for what a projection has just written is
// still there).
enum { kKept = 0, kStoresPast = 1, kAllPast = 2 };

template <int MOVE>
__device__ __forceinline__ u32x4 load_row(const uint16_t* x) {
  const u32x4* const p = reinterpret_cast<const u32x4*>(x);
  return MOVE == kAllPast ? __builtin_nontemporal_load(p) : *p;
}
template <int MOVE>
__device__ __forceinline__ void store_row(uint16_t* y, u32x4 v) {
  if (MOVE == kKept) *reinterpret_cast<u32x4*>(y) = v;
  else __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(y));
}

__device__ __forceinline__ float weight_at(const Heads& h, int d) {
  if (h.w == nullptr) return 1.f;
  return h.w16 ? bf16_to_f32(static_cast<const uint16_t*>(h.w)[d]) : static_cast<const float*>(h.w)[d];
}

__device__ __forceinline__ double position_at(const Turn& t, int64_t row, int axis) {
  const int64_t at = row * t.st + axis * t.sa;
  if (t.kind == kInt32) return (double)static_cast<const int32_t*>(t.pos)[at];
  if (t.kind == kInt64) return (double)static_cast<const int64_t*>(t.pos)[at];
  return (double)static_cast<const float*>(t.pos)[at];
}

typedef float f32x2 __attribute__((ext_vector_type(2)));

// Cosine and sine of an angle in turns.
__device__ __forceinline__ f32x2 turned(double turns) {
  const float f = (float)(turns - __builtin_rint(turns));
  return f32x2{__builtin_amdgcn_cosf(f), __builtin_amdgcn_sinf(f)};
}

// A lane's eight dims of a row: those of lane % (D / 8).
template <int D, bool ADJ>
struct Lane {
  static constexpr int kLanes = D / 8, kRows = 64 / kLanes;
  int lane, sub, d;
  int region;   // halves of pairs: 0 the first dims, 1 the second, 2 of no pair
  int partner;  // the lane of the other dims of the pairs
  int other;    // their first dim (adjacent pairs: d)
  int pair;     // the first pair
  uint32_t paired;  // all ones where its dims have pairs; adjacent: bit e where dim e has one
  float c[8], s[8];

  __device__ __forceinline__ Lane(int l, int pairs) : lane(l), sub(l / kLanes), d(8 * (l % kLanes)) {
    region = ADJ ? 0 : d < pairs ? 0 : d < 2 * pairs ? 1 : 2;
    const int step = ADJ || region == 2 ? 0 : region == 0 ? pairs : -pairs;
    partner = lane + step / 8;
    other = d + step;
    pair = ADJ ? d / 2 : region == 2 ? 0 : d - region * pairs;
    paired = ADJ ? (1u << min(max(2 * pairs - d, 0), 8)) - 1u : region == 2 ? 0u : ~0u;
  }

  // Angles from the wave's box; s has the sign that the partner's value takes.
  __device__ __forceinline__ void take(const f32x2* box) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const f32x2 a = box[pair + (ADJ ? e / 2 : e)];
      c[e] = region == 2 ? 1.f : a[0];
      s[e] = region == 2 ? 0.f : (ADJ ? (e & 1) : region) ? a[1] : -a[1];
    }
  }

  // The other dims of the pairs of a row of packed bf16; zero for a dim of no pair, whose
  // infinities and NaN are its own. Their weights too.
  __device__ __forceinline__ u32x4 partners(u32x4 x) const {
    u32x4 y;
#pragma unroll
    for (int m = 0; m < 4; ++m)
      y[m] = (ADJ ? (x[m] >> 16) | (x[m] << 16) : (uint32_t)__shfl((int)x[m], partner)) & mask(2 * m);
    return y;
  }
  __device__ __forceinline__ float other_weight(const float* weights, int e) const {
    return __uint_as_float(__float_as_uint(weights[other + e]) & mask(e));
  }
  // All ones where dim e has a pair.
  __device__ __forceinline__ uint32_t mask(int e) const {
    return ADJ ? (uint32_t)__builtin_amdgcn_sbfe((int)paired, e, 1) : paired;
  }
};

// The sum over the lanes of a row, to all of them.
template <int D>
__device__ __forceinline__ float row_sum(float v) {
  auto add = [&](int w) { v += __uint_as_float((uint32_t)w); };
  add(__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), 0xB1, 0xF, 0xF, false));   // lane ^ 1
  add(__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), 0x4E, 0xF, 0xF, false));   // lane ^ 2
  add(__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), 0x141, 0xF, 0xF, false));  // mirrored in 8
  if (D == 128)
    add(__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), 0x140, 0xF, 0xF, false));  // in 16
  return v;
}

__device__ __forceinline__ void unpack(u32x4 x, float (&f)[8]) {
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    f[2 * m] = bf16_to_f32(x[m] & 0xffffu);
    f[2 * m + 1] = __uint_as_float(x[m] & 0xffff0000u);
  }
}

__device__ __forceinline__ u32x4 pack(const float (&f)[8]) {
  return u32x4{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
               pack_bf16x2(f[6], f[7])};
}

// (mean(x^2) + eps)^-1/2 of a row. Squares past 32 bits are taken of x 2^-70 (by
// all lanes of the row: the sum is theirs together).
template <int D>
__device__ __forceinline__ float inverse_norm(const float (&x)[8], float eps) {
  float sum = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) sum = fmaf(x[e], x[e], sum);
  sum = row_sum<D>(sum);
  if (__builtin_expect(sum == INFINITY, 0)) {
    constexpr float kDown = 0x1p-70f;  // (all of 128 at 2^128 stay below 2^124)
    sum = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = fmaf(x[e] * kDown, x[e] * kDown, sum);
    return __builtin_amdgcn_rsqf(row_sum<D>(sum) * (1.f / D)) * kDown;
  }
  return __builtin_amdgcn_rsqf(fmaf(sum, 1.f / D, eps));
}

struct RotateArgs {
  Turn turn;
  Heads h[2];      // q and k
  uint16_t* y[2];  // [rows, heads, D] contiguous
  int32_t rows, parts, per_part;  // rows' parts: rounds of rows of heads each
  float eps;       // < 0: no norm
};

// A lane's pair: what its angle takes.
struct Rate {
  double turns;
  int axis;
};
__device__ __forceinline__ Rate rate_of(const Turn& t, int lane) {
  Rate r{0.0, 0};
  if (lane < t.pairs) {
    r.turns = t.turns[lane];
    r.axis = min(max(t.axes[lane], 0), t.n_axes - 1);
  }
  return r;
}

// (cos, sin) of every pair of a token into the wave's box, (1, 0) past the pairs.
template <int D>
__device__ __forceinline__ void put_turns(f32x2* box, const Rate& rate, double pos, int pairs, int lane) {
  asm volatile("" ::: "memory");
  if (D == 128 || lane < 32) box[lane] = lane < pairs ? turned(pos * rate.turns) : f32x2{1.f, 0.f};
  asm volatile("" ::: "memory");
}

// The row's eight values of a lane, normalised and rotated. w, wo: the weights of
// its dims and of the other dims of the pairs.
template <int D, bool ADJ>
__device__ __forceinline__ void rotate8(const Lane<D, ADJ>& l, u32x4 x, const float* w, const float* wo,
                                        float eps, float (&y)[8]) {
  float f[8], o[8];
  unpack(x, f);
  unpack(l.partners(x), o);
  const float r = eps < 0.f ? 1.f : inverse_norm<D>(f, eps);
#pragma unroll
  for (int e = 0; e < 8; ++e)
    y[e] = fmaf(f[e] * r, w[e] * l.c[e], (o[e] * r) * (wo[ADJ ? e ^ 1 : e] * l.s[e]));
}

template <int D, bool ADJ, int MOVE>
__global__ void __launch_bounds__(256) norm_rotate_kernel(RotateArgs p) {
  using L = Lane<D, ADJ>;
  constexpr int kAhead = 4;
  __shared__ __attribute__((aligned(16))) float weights[2][D];
  __shared__ __attribute__((aligned(16))) f32x2 boxes[4][D / 2];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (tid < 2 * D) weights[tid / D][tid % D] = weight_at(p.h[tid / D], tid % D);
  const Rate rate = rate_of(p.turn, lane);
  L l(lane, p.turn.pairs);
  __syncthreads();
  const int rounds[2] = {(p.h[0].n + L::kRows - 1) / L::kRows, (p.h[1].n + L::kRows - 1) / L::kRows};
  for (int item = blockIdx.x * 4 + wave; item < p.rows * p.parts; item += gridDim.x * 4) {
    const int row = item / p.parts, part = item - row * p.parts;
    put_turns<D>(boxes[wave], rate,
                 lane < p.turn.pairs ? position_at(p.turn, row, rate.axis) : 0.0, p.turn.pairs, lane);
    l.take(boxes[wave]);
    const int begin = part * p.per_part, end = min(begin + p.per_part, rounds[0] + rounds[1]);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const Heads& h = p.h[t];
      const int from = t == 0 ? begin : max(begin - rounds[0], 0);
      const int to = t == 0 ? min(end, rounds[0]) : end - rounds[0];
      float w[8], wo[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        w[e] = weights[t][l.d + e];
        wo[e] = l.other_weight(weights[t], e);
      }
      for (int i = from; i < to; i += kAhead) {
        u32x4 x[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int head = (i + u) * L::kRows + l.sub;
          x[u] = u32x4{0, 0, 0, 0};
          if (i + u < to && head < h.n) x[u] = load_row<MOVE>(h.x + row * h.xs + head * h.xh + l.d);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int head = (i + u) * L::kRows + l.sub;
          if (i + u >= to) break;
          float y[8];
          rotate8<D, ADJ>(l, x[u], w, wo, p.eps, y);
          if (head < h.n)
            store_row<MOVE>(p.y[t] + ((int64_t)row * h.n + head) * D + l.d, pack(y));
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Gradients (24,960 tokens of 48 and 48 heads: 337 us, 5.5 TB/s of x, dy and dx, and 5 us
// for the second launch; a rotation without a norm 331, for x is read there too, which
// it has no use for). A wave's sums for the weights stay in its lanes' registers over
// all of its tokens, and are joined over the lanes and waves of a workgroup, then over
// the workgroups by a second launch, in an order that the sizes alone set.

struct RotateBwdArgs {
  Turn turn;
  Heads h[2];
  const uint16_t* dy[2];
  int64_t ds[2], dh[2];
  uint16_t* dx[2];  // [rows, heads, D] contiguous
  float* part;      // [workgroups][2][D], or NULL
  int32_t rows, parts, per_part;
  float eps;
};

template <int D, bool ADJ, int MOVE>
__global__ void __launch_bounds__(256) norm_rotate_bwd_kernel(RotateBwdArgs p) {
  using L = Lane<D, ADJ>;
  constexpr int kAhead = 2;
  __shared__ __attribute__((aligned(16))) float weights[2][D];
  __shared__ __attribute__((aligned(16))) f32x2 boxes[4][D / 2];
  __shared__ float sums[4][2][D];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (tid < 2 * D) weights[tid / D][tid % D] = weight_at(p.h[tid / D], tid % D);
  const Rate rate = rate_of(p.turn, lane);
  L l(lane, p.turn.pairs);
  __syncthreads();
  const int rounds[2] = {(p.h[0].n + L::kRows - 1) / L::kRows, (p.h[1].n + L::kRows - 1) / L::kRows};
  float acc[2][8] = {};
  for (int item = blockIdx.x * 4 + wave; item < p.rows * p.parts; item += gridDim.x * 4) {
    const int row = item / p.parts, part = item - row * p.parts;
    put_turns<D>(boxes[wave], rate,
                 lane < p.turn.pairs ? position_at(p.turn, row, rate.axis) : 0.0, p.turn.pairs, lane);
    l.take(boxes[wave]);
    const int begin = part * p.per_part, end = min(begin + p.per_part, rounds[0] + rounds[1]);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const Heads& h = p.h[t];
      const int from = t == 0 ? begin : max(begin - rounds[0], 0);
      const int to = t == 0 ? min(end, rounds[0]) : end - rounds[0];
      float w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = weights[t][l.d + e];
      for (int i = from; i < to; i += kAhead) {
        u32x4 x[kAhead], g[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int head = (i + u) * L::kRows + l.sub;
          x[u] = g[u] = u32x4{0, 0, 0, 0};
          if (i + u < to && head < h.n) {
            x[u] = load_row<MOVE>(h.x + row * h.xs + head * h.xh + l.d);
            g[u] = load_row<MOVE>(p.dy[t] + row * p.ds[t] + head * p.dh[t] + l.d);
          }
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int head = (i + u) * L::kRows + l.sub;
          if (i + u >= to) break;
          float f[8], o[8], y[8];
          unpack(g[u], f);
          unpack(l.partners(g[u]), o);
          float dz[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) dz[e] = fmaf(f[e], l.c[e], -(o[e] * l.s[e]));
          if (p.eps < 0.f) {
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = dz[e];
          } else {
            unpack(x[u], f);
            const float r = inverse_norm<D>(f, p.eps);
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              f[e] *= r;
              acc[t][e] = head < h.n ? fmaf(dz[e], f[e], acc[t][e]) : acc[t][e];
              dz[e] *= w[e];
              sum = fmaf(dz[e], f[e], sum);
            }
            sum = row_sum<D>(sum) * (1.f / D);
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = r * fmaf(-f[e], sum, dz[e]);
          }
          if (head < h.n)
            store_row<MOVE>(p.dx[t] + ((int64_t)row * h.n + head) * D + l.d, pack(y));
        }
      }
    }
  }
  if (p.part == nullptr) return;
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float v = acc[t][e];
#pragma unroll
      for (int off = 32; off >= L::kLanes; off >>= 1) v += __shfl_xor(v, off);
      if (l.sub == 0) sums[wave][t][l.d + e] = v;
    }
  __syncthreads();
  if (tid < 2 * D) {
    const float* s = &sums[0][0][0] + tid;
    p.part[(int64_t)blockIdx.x * 2 * D + tid] = (s[0] + s[2 * D]) + (s[4 * D] + s[6 * D]);
  }
}

struct WeightArgs {
  const float* part;  // [n][2][D]
  int32_t n;
  void* dw[2];  // or NULL
  int32_t w16[2];
};

// The workgroups' sums joined: 16 columns a workgroup, 64 threads to a column.
template <int D>
__global__ void __launch_bounds__(1024) weight_grad_kernel(WeightArgs p) {
  __shared__ float box[64][17];
  const int col = threadIdx.x & 15, at = threadIdx.x >> 4, c = blockIdx.x * 16 + col;
  float sum = 0.f;
#pragma unroll 4
  for (int i = at; i < p.n; i += 64) sum += p.part[(int64_t)i * 2 * D + c];
  box[at][col] = sum;
  __syncthreads();
  if (threadIdx.x >= 16) return;
  float total = 0.f;
#pragma unroll 8
  for (int i = 0; i < 64; ++i) total += box[i][col];
  const int t = c / D, d = c % D;
  if (p.dw[t] == nullptr) return;
  if (p.w16[t]) static_cast<uint16_t*>(p.dw[t])[d] = (uint16_t)f32_to_bf16(total);
  else static_cast<float*>(p.dw[t])[d] = total;
}

// ---------------------------------------------------------------------------
// On the way into a cache: the rows of a token's query heads to q's result, those
// of its key heads, normalised and rotated, and of V into the token's page. A key
// in e4m3 is the value in 32 bits rounded once.

struct AppendRotatedArgs {
  Turn turn;     // pos NULL: the token's position in its sequence, on all axes
  Heads h[2];
  const uint16_t* v;
  int64_t vs, vh;
  uint16_t* y;   // q's result [rows, heads, D] contiguous
  Pages kp, vp;
  Table tab;
  const int32_t* cu;
  const int32_t* start;
  int32_t n_seq, rows, parts, per_part;
  float eps;
};

template <int D, bool ADJ, bool F8>
__global__ void __launch_bounds__(256) append_rotated_kernel(AppendRotatedArgs p) {
  using L = Lane<D, ADJ>;
  constexpr int kAhead = 4;
  __shared__ __attribute__((aligned(16))) float weights[2][D];
  __shared__ __attribute__((aligned(16))) f32x2 boxes[4][D / 2];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (tid < 2 * D) weights[tid / D][tid % D] = weight_at(p.h[tid / D], tid % D);
  const Rate rate = rate_of(p.turn, lane);
  L l(lane, p.turn.pairs);
  __syncthreads();
  const int nq = p.h[0].n, nkv = p.h[1].n;
  const int q_rounds = (nq + L::kRows - 1) / L::kRows, kv_rounds = (nkv + L::kRows - 1) / L::kRows;
  for (int item = blockIdx.x * 4 + wave; item < p.rows * p.parts; item += gridDim.x * 4) {
    const int row = item / p.parts, part = item - row * p.parts;
    const int begin = part * p.per_part, end = min(begin + p.per_part, q_rounds + 2 * kv_rounds);
    const int b = seq_of_row(p.cu, p.n_seq, row, lane);
    const int64_t pos = b < 0 ? 0 : (int64_t)p.start[b] + (row - p.cu[b]);
    const int page = b < 0 ? -1 : page_of(p.tab, b, pos);
    const int64_t at = pos & ((1 << p.tab.shift) - 1);
    put_turns<D>(boxes[wave], rate,
                 p.turn.pos == nullptr ? (double)pos
                 : lane < p.turn.pairs ? position_at(p.turn, row, rate.axis) : 0.0,
                 p.turn.pairs, lane);
    l.take(boxes[wave]);
    for (int t = 0; t < 3; ++t) {  // q, k, v
      const int first = t == 0 ? 0 : t == 1 ? q_rounds : q_rounds + kv_rounds;
      const int n = t == 0 ? nq : nkv;
      const int from = max(begin - first, 0), to = min(end - first, t == 0 ? q_rounds : kv_rounds);
      if (from >= to || (t > 0 && page < 0)) continue;
      const uint16_t* x0 = t == 2 ? p.v + row * p.vs : p.h[t].x + row * p.h[t].xs;
      const int64_t xh = t == 2 ? p.vh : p.h[t].xh;
      float w[8], wo[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        w[e] = weights[t & 1][l.d + e];
        wo[e] = l.other_weight(weights[t & 1], e);
      }
      for (int i = from; i < to; i += kAhead) {
        u32x4 x[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int head = (i + u) * L::kRows + l.sub;
          x[u] = u32x4{0, 0, 0, 0};
          if (i + u < to && head < n) x[u] = ld16(x0 + head * xh + l.d);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int head = (i + u) * L::kRows + l.sub;
          if (i + u >= to) break;
          float y[8];
          if (t < 2) rotate8<D, ADJ>(l, x[u], w, wo, p.eps, y);
          if (t == 0) {
            if (head < n)
              *reinterpret_cast<u32x4*>(p.y + ((int64_t)row * n + head) * D + l.d) =
                  b < 0 ? u32x4{0, 0, 0, 0} : pack(y);
            continue;
          }
          const Pages& to_pages = t == 1 ? p.kp : p.vp;
          const int64_t off = page * to_pages.sp + at * to_pages.ss + head * to_pages.sh + l.d;
          if (F8) {
            uint32_t byte;
            const u32x2 code = t == 1 ? encode8<L::kLanes>(y, byte) : encode8<L::kLanes>(x[u], byte);
            if (head < n) {
              *reinterpret_cast<u32x2*>(to_pages.x + off) = code;
              if (l.d == 0)
                to_pages.e[page * to_pages.ep + at * to_pages.es + head * to_pages.eh] = (uint8_t)byte;
            }
          } else if (head < n) {
            *reinterpret_cast<u32x4*>(to_pages.x + 2 * off) = t == 1 ? pack(y) : x[u];
          }
        }
      }
    }
  }
}

// Waves that fill the GPU; workgroups of a launch, which take their tokens in turn: many
// where each stands alone (a clip of 57,720 tokens, four a workgroup at a time: 514, 508
// and 496 us with 2,048, 4,096 and 16,384), few where each leaves sums (the gradients of
// 24,960 tokens: 407, 342 and 345 with 512, 768 and 1,024).
constexpr int64_t kEnough = 4096, kMostBlocks = 16384, kMostBwdBlocks = 768;

// A launch's parts: waves for `rounds` rounds of every row, all by one where rows
// are enough to fill the GPU.
struct Split {
  int32_t parts, per_part;
  unsigned grid;
};
Split split_of(int64_t rows, int rounds, int64_t enough, int64_t most) {
  int64_t parts = enough / (rows > 0 ? rows : 1);
  if (parts > rounds) parts = rounds;
  if (parts < 1) parts = 1;  // (no heads: no rounds)
  const int per = (int)((rounds + parts - 1) / parts);
  if (per > 0) parts = (rounds + per - 1) / per;
  const int64_t blocks = (rows * parts + 3) / 4;
  return Split{(int32_t)parts, per, (unsigned)(blocks < most ? blocks : most)};
}

int check_rows(const char* what, const char* name, const void* x, int64_t s, int64_t h, int64_t heads) {
  VEDA_REQUIRE(heads >= 0 && heads <= 65535, "%s: 0 to 65535 heads of %s, got %lld", what, name,
               (long long)heads);
  VEDA_REQUIRE(heads == 0 || whole(x, 8, s, h, 0), "%s: %s rows must be 16-byte aligned", what, name);
  return VEDA_OK;
}

int check_turn(const char* what, int64_t rows, int64_t head_dim, const void* positions, int64_t kind,
               int64_t stride_t, int64_t stride_a, const double* turns, const int32_t* axes, int64_t n_pairs,
               int64_t n_axes, int adjacent, bool own_positions, float eps, Turn& t) {
  VEDA_REQUIRE(head_dim == 64 || head_dim == 128, "%s: head_dim must be 64 or 128, got %lld", what,
               (long long)head_dim);
  VEDA_REQUIRE(rows >= 0 && rows < (1 << 26), "%s: 2^26 rows or more, or negative", what);
  // (below that, squares of small values are lost beside which eps is small too)
  VEDA_REQUIRE(eps < 0.f || (eps >= 1e-30f && eps < INFINITY), "%s: eps must be 1e-30 at least and finite", what);
  VEDA_REQUIRE(n_pairs >= 0 && 2 * n_pairs <= head_dim, "%s: %lld pairs in a head of %lld", what,
               (long long)n_pairs, (long long)head_dim);
  t = Turn{};
  if (n_pairs == 0) return VEDA_OK;
  VEDA_REQUIRE(adjacent || n_pairs % 8 == 0, "%s: pairs of dims apart must be a multiple of 8, got %lld", what,
               (long long)n_pairs);
  VEDA_REQUIRE(n_axes > 0 && n_axes <= 65535, "%s: 1 to 65535 axes, got %lld", what, (long long)n_axes);
  VEDA_REQUIRE(turns != nullptr && axes != nullptr && (own_positions || positions != nullptr || rows == 0),
               "%s: a rotation needs positions, rates and axes", what);
  VEDA_REQUIRE(kind == kInt32 || kind == kInt64 || kind == kFloat32, "%s: unknown kind of positions", what);
  t = Turn{positions, (int32_t)kind, stride_t, stride_a, turns, axes, (int32_t)n_pairs, (int32_t)n_axes};
  return VEDA_OK;
}

Heads heads_of(const void* x, int64_t s, int64_t h, int64_t n, const void* w, int w16) {
  return Heads{static_cast<const uint16_t*>(x), s, h, w, w16, (int32_t)n};
}

int rounds_of(int64_t heads, int64_t head_dim) {
  const int64_t at_once = 512 / head_dim;
  return (int)((heads + at_once - 1) / at_once);
}

using D128 = std::integral_constant<int, 128>;
using D64 = std::integral_constant<int, 64>;

// f(head_dim, adjacent) with both as constants.
template <typename F>
void by_kind(int64_t head_dim, int adjacent, F f) {
  if (head_dim == 128 && adjacent) f(D128{}, std::true_type{});
  else if (head_dim == 128) f(D128{}, std::false_type{});
  else if (adjacent) f(D64{}, std::true_type{});
  else f(D64{}, std::false_type{});
}

// And f(head_dim, adjacent, how rows are moved) for `bytes` of them.
template <typename F>
void by_kind_and_size(int64_t head_dim, int adjacent, int64_t bytes, F f) {
  by_kind(head_dim, adjacent, [&](auto d, auto adj) {
    if (bytes >= (1 << 28)) f(d, adj, std::integral_constant<int, kAllPast>{});
    else if (bytes >= (1 << 25)) f(d, adj, std::integral_constant<int, kStoresPast>{});
    else f(d, adj, std::integral_constant<int, kKept>{});
  });
}

}  // namespace
}  // namespace veda

using namespace veda;

extern "C" int veda_norm_rotate(const void* q, int64_t q_stride_s, int64_t q_stride_h, int64_t q_heads,
                                const void* k, int64_t k_stride_s, int64_t k_stride_h, int64_t k_heads,
                                int64_t rows, int64_t head_dim, const void* positions, int64_t kind,
                                int64_t stride_t, int64_t stride_a, const double* turns, const int32_t* axes,
                                int64_t n_pairs, int64_t n_axes, int adjacent, const void* q_weight,
                                int q_weight_bf16, const void* k_weight, int k_weight_bf16, float eps,
                                void* q_out, void* k_out, void* stream) {
  RotateArgs p{};
  if (int rc = check_turn("norm_rotate", rows, head_dim, positions, kind, stride_t, stride_a, turns, axes,
                          n_pairs, n_axes, adjacent, false, eps, p.turn))
    return rc;
  if (int rc = check_rows("norm_rotate", "q", q, q_stride_s, q_stride_h, q_heads)) return rc;
  if (int rc = check_rows("norm_rotate", "k", k, k_stride_s, k_stride_h, k_heads)) return rc;
  VEDA_REQUIRE(whole(q_out, 8, 0, 0, 0) && whole(k_out, 8, 0, 0, 0), "norm_rotate: results must be 16-byte aligned");
  const int rounds = rounds_of(q_heads, head_dim) + rounds_of(k_heads, head_dim);
  if (rows == 0 || rounds == 0) return VEDA_OK;
  p.h[0] = heads_of(q, q_stride_s, q_stride_h, q_heads, q_weight, q_weight_bf16);
  p.h[1] = heads_of(k, k_stride_s, k_stride_h, k_heads, k_weight, k_weight_bf16);
  p.y[0] = static_cast<uint16_t*>(q_out);
  p.y[1] = static_cast<uint16_t*>(k_out);
  const Split split = split_of(rows, rounds, kEnough, kMostBlocks);
  p.rows = (int32_t)rows;
  p.parts = split.parts;
  p.per_part = split.per_part;
  p.eps = eps;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t bytes = 2 * rows * (q_heads + k_heads) * head_dim;
  by_kind_and_size(head_dim, adjacent && n_pairs > 0, bytes, [&](auto d, auto adj, auto move) {
    norm_rotate_kernel<decltype(d)::value, decltype(adj)::value, decltype(move)::value>
        <<<split.grid, 256, 0, s>>>(p);
  });
  return check_launch("veda_norm_rotate");
}

extern "C" int veda_norm_rotate_bwd(const void* q, int64_t q_stride_s, int64_t q_stride_h, const void* dq_out,
                                    int64_t dq_stride_s, int64_t dq_stride_h, int64_t q_heads, const void* k,
                                    int64_t k_stride_s, int64_t k_stride_h, const void* dk_out,
                                    int64_t dk_stride_s, int64_t dk_stride_h, int64_t k_heads, int64_t rows,
                                    int64_t head_dim, const void* positions, int64_t kind, int64_t stride_t,
                                    int64_t stride_a, const double* turns, const int32_t* axes,
                                    int64_t n_pairs, int64_t n_axes, int adjacent, const void* q_weight,
                                    int q_weight_bf16, const void* k_weight, int k_weight_bf16, float eps,
                                    void* dq, void* dk, void* dq_weight, void* dk_weight, void* workspace,
                                    int64_t workspace_bytes, void* stream) {
  const char* const what = "norm_rotate_bwd";
  RotateBwdArgs p{};
  if (int rc = check_turn(what, rows, head_dim, positions, kind, stride_t, stride_a, turns, axes, n_pairs,
                          n_axes, adjacent, false, eps, p.turn))
    return rc;
  if (int rc = check_rows(what, "q", q, q_stride_s, q_stride_h, q_heads)) return rc;
  if (int rc = check_rows(what, "k", k, k_stride_s, k_stride_h, k_heads)) return rc;
  if (int rc = check_rows(what, "q's gradient", dq_out, dq_stride_s, dq_stride_h, q_heads)) return rc;
  if (int rc = check_rows(what, "k's gradient", dk_out, dk_stride_s, dk_stride_h, k_heads)) return rc;
  VEDA_REQUIRE(whole(dq, 8, 0, 0, 0) && whole(dk, 8, 0, 0, 0), "%s: results must be 16-byte aligned", what);
  const bool sums = dq_weight != nullptr || dk_weight != nullptr;
  VEDA_REQUIRE(!sums || eps >= 0.f, "%s: weights without a norm", what);
  const int rounds = rounds_of(q_heads, head_dim) + rounds_of(k_heads, head_dim);
  const Split split = split_of(rows, rounds, kEnough, kMostBwdBlocks);
  const int64_t need = sums ? (int64_t)split.grid * 2 * head_dim * 4 : 0;
  VEDA_REQUIRE(need == 0 || (workspace != nullptr && whole(workspace, 8, 0, 0, 0) && workspace_bytes >= need),
               "%s: workspace needs %lld bytes (16-byte aligned), got %lld", what, (long long)need,
               (long long)workspace_bytes);
  const bool work = rows > 0 && rounds > 0;
  if (!work && !sums) return VEDA_OK;
  p.h[0] = heads_of(q, q_stride_s, q_stride_h, q_heads, q_weight, q_weight_bf16);
  p.h[1] = heads_of(k, k_stride_s, k_stride_h, k_heads, k_weight, k_weight_bf16);
  p.dy[0] = static_cast<const uint16_t*>(dq_out);
  p.dy[1] = static_cast<const uint16_t*>(dk_out);
  p.ds[0] = dq_stride_s; p.dh[0] = dq_stride_h;
  p.ds[1] = dk_stride_s; p.dh[1] = dk_stride_h;
  p.dx[0] = static_cast<uint16_t*>(dq);
  p.dx[1] = static_cast<uint16_t*>(dk);
  p.part = sums ? static_cast<float*>(workspace) : nullptr;
  p.rows = (int32_t)rows;
  p.parts = split.parts;
  p.per_part = split.per_part;
  p.eps = eps;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (work) {
    const int64_t bytes = 2 * rows * (q_heads + k_heads) * head_dim;
    by_kind_and_size(head_dim, adjacent && n_pairs > 0, bytes, [&](auto d, auto adj, auto move) {
      norm_rotate_bwd_kernel<decltype(d)::value, decltype(adj)::value, decltype(move)::value>
          <<<split.grid, 256, 0, s>>>(p);
    });
    if (int rc = check_launch("veda_norm_rotate_bwd")) return rc;
  }
  if (!sums) return VEDA_OK;
  WeightArgs w{p.part, work ? (int32_t)split.grid : 0, {dq_weight, dk_weight}, {q_weight_bf16, k_weight_bf16}};
  const unsigned columns = (unsigned)(2 * head_dim / 16);
  if (head_dim == 128) weight_grad_kernel<128><<<columns, 1024, 0, s>>>(w);
  else weight_grad_kernel<64><<<columns, 1024, 0, s>>>(w);
  return check_launch("veda_norm_rotate_bwd");
}

extern "C" int veda_cache_append_rotated(
    const void* q, int64_t q_stride_s, int64_t q_stride_h, int64_t q_heads, const void* k, int64_t k_stride_s,
    int64_t k_stride_h, const void* v, int64_t v_stride_s, int64_t v_stride_h, int64_t rows,
    int64_t n_kv_heads, int64_t head_dim, const int32_t* cu, const int32_t* start, int64_t n_seq,
    void* k_pages, void* v_pages, int64_t stride_p, int64_t stride_s, int64_t stride_h, int e4m3,
    uint8_t* k_exp, uint8_t* v_exp, int64_t exp_stride_p, int64_t exp_stride_s, int64_t exp_stride_h,
    int64_t n_pages, int64_t page, const int32_t* table, int64_t table_ld, int64_t width,
    const void* positions, int64_t kind, int64_t stride_t, int64_t stride_a, const double* turns,
    const int32_t* axes, int64_t n_pairs, int64_t n_axes, int adjacent, const void* q_weight,
    int q_weight_bf16, const void* k_weight, int k_weight_bf16, float eps, void* q_out, void* stream) {
  const char* const what = "cache_append_rotated";
  AppendRotatedArgs p{};
  p.kp = pages_of(k_pages, stride_p, stride_s, stride_h, k_exp, exp_stride_p, exp_stride_s, exp_stride_h);
  p.vp = pages_of(v_pages, stride_p, stride_s, stride_h, v_exp, exp_stride_p, exp_stride_s, exp_stride_h);
  if (int rc = check_cache(what, head_dim, n_kv_heads, n_pages, page, width, e4m3, p.kp, p.vp)) return rc;
  if (int rc = check_turn(what, rows, head_dim, positions, kind, stride_t, stride_a, turns, axes, n_pairs,
                          n_axes, adjacent, true, eps, p.turn))
    return rc;
  if (int rc = check_rows(what, "q", q, q_stride_s, q_stride_h, q_heads)) return rc;
  if (int rc = check_rows(what, "k", k, k_stride_s, k_stride_h, n_kv_heads)) return rc;
  if (int rc = check_rows(what, "v", v, v_stride_s, v_stride_h, n_kv_heads)) return rc;
  VEDA_REQUIRE(n_seq >= 0 && n_seq < (1 << 20), "%s: 2^20 sequences or more, or negative", what);
  VEDA_REQUIRE(whole(q_out, 8, 0, 0, 0), "%s: q's result must be 16-byte aligned", what);
  if (rows == 0) return VEDA_OK;
  p.h[0] = heads_of(q, q_stride_s, q_stride_h, q_heads, q_weight, q_weight_bf16);
  p.h[1] = heads_of(k, k_stride_s, k_stride_h, n_kv_heads, k_weight, k_weight_bf16);
  p.v = static_cast<const uint16_t*>(v);
  p.vs = v_stride_s; p.vh = v_stride_h;
  p.y = static_cast<uint16_t*>(q_out);
  p.tab = table_of(table, table_ld, width, n_pages, page);
  p.cu = cu;
  p.start = start;
  p.n_seq = (int32_t)n_seq;
  const Split split = split_of(rows, rounds_of(q_heads, head_dim) + 2 * rounds_of(n_kv_heads, head_dim),
                               kEnough, kMostBlocks);
  p.rows = (int32_t)rows;
  p.parts = split.parts;
  p.per_part = split.per_part;
  p.eps = eps;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  by_kind(head_dim, adjacent && n_pairs > 0, [&](auto d, auto adj) {
    constexpr int kD = decltype(d)::value;
    constexpr bool kAdj = decltype(adj)::value;
    if (e4m3) append_rotated_kernel<kD, kAdj, true><<<split.grid, 256, 0, s>>>(p);
    else append_rotated_kernel<kD, kAdj, false><<<split.grid, 256, 0, s>>>(p);
  });
  return check_launch("veda_cache_append_rotated");
}
