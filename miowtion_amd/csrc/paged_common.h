// What the kernels over a paged key-value cache share: its pages, rows and formats.
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
#pragma once

#include "veda_pipeline.h"

namespace veda {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

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

// The same for eight values of a lane in 32 bits.
template <int LANES>
__device__ __forceinline__ u32x2 encode8(const float (&x)[8], uint32_t& byte) {
  uint32_t top = 0;
  bool odd = false;  // a NaN or an infinity
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t mag = __float_as_uint(x[e]) & 0x7fffffffu;
    odd |= mag >= 0x7f800000u;
    top = max(top, mag < 0x7f800000u ? mag : 0u);
  }
#pragma unroll
  for (int off = LANES / 2; off >= 1; off >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off));
  const int e = (int)(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
  byte = (uint32_t)max(e, 0);
  const float s = __uint_as_float((254u - byte) << 23);  // 2^(127 - byte)
  u32x2 w;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    int c = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * h] * s, x[4 * h + 1] * s, 0, false);
    w[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * h + 2] * s, x[4 * h + 3] * s, c, true);
    if (odd) {
#pragma unroll
      for (int m = 0; m < 4; ++m)
        if (!(fabsf(x[4 * h + m]) < INFINITY)) w[h] |= 0x7fu << (8 * m);
    }
  }
  return w;
}

// V rows of a wave's own in LDS that are read transposed by 16x16 products: the chunk's
// place is xor'ed with this.
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

inline bool whole(const void* p, int64_t mult, int64_t a, int64_t b, int64_t c) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && a % mult == 0 && b % mult == 0 && c % mult == 0;
}

inline int check_cache(const char* what, int64_t head_dim, int64_t n_kv, int64_t n_pages, int64_t page,
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

inline Pages pages_of(const void* x, int64_t sp, int64_t ss, int64_t sh, const uint8_t* e, int64_t ep,
                      int64_t es, int64_t eh) {
  return Pages{static_cast<uint8_t*>(const_cast<void*>(x)), sp, ss, sh, const_cast<uint8_t*>(e),
               ep, es, eh};
}

inline Table table_of(const int32_t* table, int64_t ld, int64_t width, int64_t n_pages, int64_t page) {
  return Table{table, ld, (int32_t)width, (int32_t)n_pages, __builtin_ctzll((uint64_t)page)};
}

}  // namespace veda
