// The key/value cache: pools [n_pages, n_heads, page, pitch] of rows of d values (pitch: d rounded up to 16), in the
// model's type or in 8 bits with one fp32 scale per row, a table of pages for each sequence, and its lengths.
#pragma once

#include <type_traits>

#include "row_device.h"

namespace tmac {

struct CacheArgs {
  uint8_t *k, *v;           // pools
  float *ks, *vs;           // scales [n_pages, n_heads, page]; null in the model's type
  const int32_t* table;     // [B, max_pages] at a pitch of table_stride
  const int32_t* lengths;   // [B]: positions held, the new rows included
  const int32_t* counts;    // [B]: new rows; null: T, or the length where that is less
  int64_t table_stride;
  int n_pages, n_heads, page_shift, pitch, d, max_pages;
  int T;                    // new rows of a sequence at most
};

// One sequence: `len` positions, the last n of them new. ok is false for numbers that the table cannot hold (nothing
// of such a sequence is read or written, and what is asked of it is NaN).
struct Seq {
  int len, n;
  bool ok;
};
__device__ __forceinline__ Seq seq_of(const CacheArgs& a, int b) {
  Seq s;
  s.len = a.lengths[b];
  s.n = a.counts ? a.counts[b] : (a.T < s.len ? a.T : s.len);
  s.ok = s.len >= 0 && s.len <= (static_cast<int64_t>(a.max_pages) << a.page_shift) && s.n >= 0 && s.n <= a.T &&
         s.n <= s.len;
  return s;
}

// The pool's row (in rows) of position pos (inside the table) for head h; −1 for a page outside the pool.
__device__ __forceinline__ int64_t cache_row(const CacheArgs& a, int b, int pos, int h) {
  const int page = a.table[b * a.table_stride + (pos >> a.page_shift)];
  if (page < 0 || page >= a.n_pages) return -1;
  return ((static_cast<int64_t>(page) * a.n_heads + h) << a.page_shift) + (pos & ((1 << a.page_shift) - 1));
}

constexpr int kCacheSame = TMAC_CACHE_SAME, kCacheInt8 = TMAC_CACHE_INT8, kCacheE4m3 = TMAC_CACHE_E4M3;

// Two codes (bytes 0 and 1 of w, or 2 and 3 with HI) as 16-bit values of DT: every code is exact in them.
template <int DT, int FMT, bool HI>
__device__ __forceinline__ uint32_t code2(uint32_t w) {
  if constexpr (FMT == kCacheInt8) {
    const float lo = static_cast<float>(static_cast<int8_t>(w >> (HI ? 16 : 0)));
    const float hi = static_cast<float>(static_cast<int8_t>(w >> (HI ? 24 : 8)));
    return Mfma<DT>::pack2(lo, hi);
  } else if constexpr (DT == TMAC_BF16) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI));
  } else {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI));
  }
}
// Four codes as fp32.
template <int FMT>
__device__ __forceinline__ f32x4 code4(uint32_t w) {
  if constexpr (FMT == kCacheInt8) {
    return f32x4{static_cast<float>(static_cast<int8_t>(w)), static_cast<float>(static_cast<int8_t>(w >> 8)),
                 static_cast<float>(static_cast<int8_t>(w >> 16)), static_cast<float>(static_cast<int8_t>(w >> 24))};
  } else {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    return f32x4{lo[0], lo[1], hi[0], hi[1]};
  }
}

// A row's scale from the bits of its largest magnitude; NaN (and codes of 0) for a row that is not finite.
// int8: amax / 127 rounded to fp32; e4m3: the least power of two with amax <= 448 scale (448 = 1.75 · 2^8). At least
// 2^-126, so that the scale and its reciprocal are normal numbers.
template <int FMT>
__device__ __forceinline__ float code_scale(uint32_t amax) {
  if (amax >= 0x7f800000u) return __builtin_nanf("");
  if constexpr (FMT == kCacheInt8) {
    return fmaxf(__uint_as_float(amax) / 127.0f, 0x1p-126f);
  } else {
    const int e = static_cast<int>(amax >> 23) - 8 + ((amax & 0x7fffffu) > 0x600000u);  // biased exponent
    return __uint_as_float(static_cast<uint32_t>(e > 1 ? e : 1) << 23);
  }
}

// Four values as codes of scale s, one byte each.
//
// int8: rne(x / s) for |x| <= 127 s (within a rounding), from an approximate quotient q, decided by the remainder x − q s.
// That is exact in an fma: for |x| >= s it is a multiple of s's last bit below 0.6 s, for q = 0 it is x, and for
// q = ±1 and |x| >= s/2 the operands are within a factor of two of each other; for q = ±1 and |x| < s/2 it may be
// rounded, to s/2 at the least, and a tie goes to 0 as |x| < s/2 does. q is one off, or the remainder a tie, for few
// rows: the others take one comparison for their four values.
template <int FMT>
__device__ __forceinline__ uint32_t to_code4(float a, float b, float c, float d, float s) {
  if (s != s) return 0;
  if constexpr (FMT == kCacheInt8) {
    const float x[4] = {a, b, c, d}, inv = __builtin_amdgcn_rcpf(s), h = 0.5f * s;
    float q[4], r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      q[i] = rintf(x[i] * inv);
      r[i] = fmaf(-q[i], s, x[i]);
    }
    int code[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) code[i] = static_cast<int>(q[i]);
    if (fmaxf(fmaxf(fabsf(r[0]), fabsf(r[1])), fmaxf(fabsf(r[2]), fabsf(r[3]))) >= h) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool odd = code[i] & 1;
        if (r[i] > h || (r[i] == h && odd))
          code[i] += 1;
        else if (r[i] < -h || (r[i] == -h && odd))
          code[i] -= 1;
      }
    }
    return (code[0] & 255) | (code[1] & 255) << 8 | (code[2] & 255) << 16 | static_cast<uint32_t>(code[3] & 255) << 24;
  } else {
    const float inv = __uint_as_float(0x7f000000u - __float_as_uint(s));  // 1 / s, a power of two: exact products
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c * inv, d * inv, w, true));
  }
}

// The kernels' arguments from the caller's, checked: sizes that the kernels' integers hold, pools they can read.
inline int cache_args(const tmac_cache* c, int B, int T, CacheArgs& a) {
  if (!c) return TMAC_ERR_NULL;
  if (c->dtype != TMAC_F32 && c->dtype != TMAC_BF16 && c->dtype != TMAC_F16) return TMAC_ERR_DTYPE;
  if (c->format != TMAC_CACHE_SAME && c->format != TMAC_CACHE_INT8 && c->format != TMAC_CACHE_E4M3)
    return TMAC_ERR_DTYPE;
  int shift = 4;
  while (shift < 8 && (1 << shift) != c->page) ++shift;
  if ((1 << shift) != c->page || c->n_heads <= 0 || c->n_heads > 65535 || c->d_head <= 0 || c->d_head > 128 ||
      c->pitch != (c->d_head + 15) / 16 * 16)
    return TMAC_ERR_SHAPE;
  // a page's bytes are counted in 32 bits
  if (static_cast<int64_t>(c->n_heads) * c->page * c->pitch >= (1 << 29)) return TMAC_ERR_SHAPE;
  if (c->n_pages <= 0 || c->n_pages >= (INT64_C(1) << 31) || c->n_pages * c->n_heads >= (INT64_C(1) << 40) / c->page)
    return TMAC_ERR_SHAPE;
  // positions are counted in 32 bits, and so are the threads of a launch (up to 32 a row)
  if (c->max_pages <= 0 || c->max_pages > (1 << 30) / c->page || B < 0 || B > (1 << 20) || T < 0 || T > (1 << 30) ||
      static_cast<int64_t>(T) * c->n_heads > (1 << 26) || (B > 1 && c->table_stride < c->max_pages))
    return TMAC_ERR_SHAPE;
  if (!c->d_k || !c->d_v || !c->d_table || !c->d_lengths) return TMAC_ERR_NULL;
  if (c->format != TMAC_CACHE_SAME && (!c->d_k_scale || !c->d_v_scale)) return TMAC_ERR_NULL;
  auto off = [](const void* p, int n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) != 0; };
  if (off(c->d_k, 16) || off(c->d_v, 16) || off(c->d_k_scale, 16) || off(c->d_v_scale, 16) || off(c->d_table, 4) ||
      off(c->d_lengths, 4) || off(c->d_counts, 4))
    return TMAC_ERR_ALIGN;
  const bool same = c->format == TMAC_CACHE_SAME;
  a = CacheArgs{static_cast<uint8_t*>(c->d_k), static_cast<uint8_t*>(c->d_v), same ? nullptr : c->d_k_scale,
                same ? nullptr : c->d_v_scale, c->d_table, c->d_lengths, c->d_counts, c->table_stride,
                static_cast<int>(c->n_pages), c->n_heads, shift, c->pitch, c->d_head, c->max_pages, T};
  return TMAC_OK;
}

}  // namespace tmac
