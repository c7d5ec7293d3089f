// Attention of new rows over the key/value cache.
//
// With G = query heads / key heads, the G·T query rows (t, g) that read key head hk of one sequence are taken 16 RT at a
// time; a workgroup holds one such block of rows and walks the keys that any of them sees, 32 at a time, tiles dealt to
// its waves in turn (and to `splits` workgroups). All products are on the matrix cores, whose 16 columns cost
// nothing beside the reading of the cache when one row is real:
//   S^T (16 keys x 16 rows) = K · Q^T    A = keys' rows, B = the queries, resident in registers
//   O^T (16 of d x 16 rows) += V^T · P^T  A = values, B = probabilities
// Lane l = 16 g + n of the first result holds keys 4 g .. 4 g + 3 of row n, twice (two groups of 16 keys). The
// second product's sum over keys may run in any order, so k index 8 g + i stands for key 4 g + i (i < 4) or
// 16 + 4 g + i - 4: a lane's own eight probabilities are its operand as they are, and a row's statistics are in the
// lanes that hold the row's results. The values' operand needs eight keys of one column: a lane reads whole pieces of
// its eight keys' rows (column n·NJ .. + NJ, so 16 lanes read a row) and transposes them in registers.
// No LDS and no barrier before the waves' results are joined.

#include "cache_device.h"

namespace {
using namespace tmac;

constexpr float kInf = __builtin_huge_valf();

template <int DT>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (DT == TMAC_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
}

// A piece of BYTES contiguous bytes in registers.
template <int BYTES>
struct Piece {
  uint32_t w[BYTES / 4];
  __device__ __forceinline__ void load(const uint8_t* p) {
    if constexpr (BYTES == 4) {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else if constexpr (BYTES == 8) {
      const u32x2 x = *reinterpret_cast<const u32x2*>(p);
      w[0] = x[0], w[1] = x[1];
    } else {
#pragma unroll
      for (int i = 0; i < BYTES / 16; ++i) {
        const u32x4 x = reinterpret_cast<const u32x4*>(p)[i];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[4 * i + j] = x[j];
      }
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < BYTES / 4; ++i) w[i] = 0;
  }
};

// What a kernel's types and head width mean for its loads. DT: the values' type; FMT: how the cache holds them; DP: 64
// or 128, at least the pitch.
template <int DT, int FMT, int DP>
struct Shape {
  static constexpr int kElem = FMT != kCacheSame ? 1 : DT == TMAC_F32 ? 4 : 2;  // bytes of a stored value
  static constexpr int kRun = 16 / kElem;           // values in 16 bytes: a lane's piece of a key
  static constexpr int kPieces = DP / (4 * kRun);   // of each key, per lane; piece c of group g: 4 kRun c + kRun g ..
  static constexpr int kOps = DT == TMAC_F32 ? kRun : kRun / 8;  // products per piece
  static constexpr int NJ = DP / 16;                // columns of the values per lane, products per 32 keys
  static constexpr bool kF32 = DT == TMAC_F32;
};

// operand e of a key's piece
template <int DT, int FMT, int DP>
__device__ __forceinline__ auto key_operand(const Piece<16>& p, int e) {
  if constexpr (DT == TMAC_F32) {
    if constexpr (FMT == kCacheSame)
      return __uint_as_float(p.w[e]);
    else
      return code4<FMT>(p.w[e >> 2])[e & 3];
  } else if constexpr (FMT == kCacheSame) {
    return u32x4{p.w[0], p.w[1], p.w[2], p.w[3]};
  } else {
    const uint32_t lo = p.w[2 * e], hi = p.w[2 * e + 1];
    return u32x4{code2<DT, FMT, false>(lo), code2<DT, FMT, true>(lo), code2<DT, FMT, false>(hi),
                 code2<DT, FMT, true>(hi)};
  }
}

// operand j of the values of eight keys (16 bit): the lane's column j of all of them
template <int DT, int FMT, int NB>
__device__ __forceinline__ u32x4 value_operand(const Piece<NB> (&v)[8], int j) {
  u32x4 r;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if constexpr (FMT == kCacheSame) {
      r[w] = __builtin_amdgcn_perm(v[2 * w + 1].w[j >> 1], v[2 * w].w[j >> 1], j & 1 ? 0x07060302u : 0x05040100u);
    } else {
      // bytes j, j of two keys beside those of column j ^ 1: one permutation serves two columns
      const uint32_t x = __builtin_amdgcn_perm(v[2 * w + 1].w[j >> 2], v[2 * w].w[j >> 2],
                                               j & 2 ? 0x07030602u : 0x05010400u);
      r[w] = j & 1 ? code2<DT, FMT, true>(x) : code2<DT, FMT, false>(x);
    }
  }
  return r;
}
// one value in fp32
template <int FMT, int NB>
__device__ __forceinline__ float value_f32(const Piece<NB>& v, int j) {
  if constexpr (FMT == kCacheSame)
    return __uint_as_float(v.w[j]);
  else
    return code4<FMT>(v.w[j >> 2])[j & 3];
}

struct AttnArgs {
  CacheArgs c;
  const uint8_t* q;
  int64_t qb, qh, qt;
  const int64_t* tree;
  int64_t tree_stride;
  uint8_t* out;
  float* ws;
  int B, Hq, G, g_shift, n_rb, splits, np, row_cap;  // g_shift: log2 of G, or -1
  int window;  // INT_MAX / 2 and above: none
  float scale2;  // scale · log2 e
  bool q_vec, out_vec;
};

// A division costs a wave a few dozen instructions, in a kernel that may be done in a few hundred.
__device__ __forceinline__ int by_group(const AttnArgs& a, int r) {
  return a.g_shift >= 0 ? r >> a.g_shift : static_cast<int>(static_cast<unsigned>(r) / static_cast<unsigned>(a.G));
}

// What a row sees: j < np, lo <= j <= hi, and drafted rows by bits.
struct Row {
  int np, lo, hi;
  uint64_t bits;
};

__device__ __forceinline__ bool sees(const Row& r, int j, int base, bool tree) {
  bool v = (j < r.np) | ((j >= r.lo) & (j <= r.hi));
  if (tree) {
    const uint32_t s = static_cast<uint32_t>(j - base);
    v |= s < 64u && ((r.bits >> (s & 63u)) & 1);
  }
  return v;
}

__device__ __forceinline__ int bits_set(int64_t x) { return static_cast<int>(__popcll(static_cast<uint64_t>(x))); }

// Row t of sequence s. Without a tree position p = base + t.
__device__ __forceinline__ Row row_of(const AttnArgs& a, const Seq& s, int b, int t) {
  Row r{0, 1, 0, 0};
  if (t >= s.n) return r;
  const int base = s.len - s.n, np = a.np < s.len ? a.np : s.len;
  if (!a.tree) {
    const int p = base + t;
    r.np = np;
    if (p >= a.np) {
      r.lo = p - a.window > 0 ? p - a.window : 0;
      r.hi = p;
    }
    return r;
  }
  const int64_t* const tree = a.tree + b * a.tree_stride;
  const uint64_t have = s.n >= 64 ? ~0ull : (1ull << s.n) - 1;
  const int p = base + bits_set(tree[t]) - 1;
  r.np = np < base ? np : base;
  r.lo = p - a.window > 0 ? p - a.window : 0;
  r.hi = base - 1;
  r.bits = static_cast<uint64_t>(tree[t]) & have;
  if (a.window < 2 * TMAC_CACHE_MAX_TREE) {  // drafted rows may be behind the window: their places differ by up to 64
    for (int u = 0; u < s.n; ++u)
      if (base + bits_set(tree[u]) - 1 < p - a.window && base + u >= a.np) r.bits &= ~(1ull << u);
  }
  return r;
}

// w with what is not finite in it (two 16-bit values, or one fp32) replaced by zeros
template <int DT>
__device__ __forceinline__ uint32_t finite_only(uint32_t w) {
  if constexpr (DT == TMAC_F32) return (w & 0x7f800000u) == 0x7f800000u ? 0u : w;
  constexpr uint32_t kExp = DT == TMAC_BF16 ? 0x7f807f80u : 0x7c007c00u, kLow = DT == TMAC_BF16 ? 0x00800080u : 0x04000400u;
  const uint32_t top = ((w & kExp) + kLow) & 0x80008000u;  // the top bit of a half whose exponent is all ones
  return w & ~((top >> 15) * 0xffffu);
}

// o / sum; zeros for a row that sees nothing or is none, NaN where the sequence's numbers do not fit
template <int N>
__device__ __forceinline__ void row_finish(const Seq& s, int t, float sum, float (&o)[N]) {
  const float f = !s.ok ? __builtin_nanf("") : 1.f / sum;
  const bool none = s.ok && (t >= s.n || sum == 0.f);
#pragma unroll
  for (int e = 0; e < N; ++e) o[e] = none ? 0.f : o[e] * f;
}

// values i0 .. i0 + 3 of the result for row t of head h
template <int DT>
__device__ __forceinline__ void row_out(const AttnArgs& a, int b, int t, int h, int i0, const float (&o)[4]) {
  uint8_t* const to = a.out + (((static_cast<int64_t>(b) * a.c.T + t) * a.Hq + h) * a.c.d + i0) * kRowSize<DT>;
  if (a.out_vec) {  // d a multiple of 4
    if (i0 >= a.c.d) return;
    if constexpr (DT == TMAC_F32)
      *reinterpret_cast<f32x4*>(to) = f32x4{o[0], o[1], o[2], o[3]};
    else
      *reinterpret_cast<u32x2*>(to) = u32x2{Mfma<DT>::pack2(o[0], o[1]), Mfma<DT>::pack2(o[2], o[3])};
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float one[1] = {o[e]};
    if (i0 + e < a.c.d) row_store<DT, 1>(to + e * kRowSize<DT>, one);
  }
}

template <int DT, int FMT, int DP, int RT, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 1) void cached_attn_kernel(AttnArgs a) {
  using S = Shape<DT, FMT, DP>;
  constexpr int NJ = S::NJ, kRows = 16 * RT, NB = NJ * S::kElem;
  extern __shared__ float sh[];
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr int n_waves = WAVES;
  const int b = blockIdx.x, hk = blockIdx.y, rb = a.splits == 1 ? blockIdx.z : blockIdx.z / static_cast<unsigned>(a.splits),
            split = blockIdx.z - rb * a.splits;
  const Seq s = seq_of(a.c, b);
  const int rows_all = a.c.T * a.G, row0 = rb * kRows;
  const int G = a.G;
  const int t_lo = by_group(a, row0), t_end = by_group(a, row0 + kRows - 1);
  const int t_hi = t_end < s.n - 1 ? t_end : s.n - 1;
  const int base = s.len - s.n, len = s.len;
  const bool tree = a.tree != nullptr;
  const bool work = s.ok && t_lo < s.n;

  // the keys that any row sees: [0, np) and [lo, hi]; lo_all, hi_all: seen by all rows
  const int np = a.np < len ? a.np : len;
  int np_all = np, lo, hi, lo_all, hi_all;
  if (tree) {  // places from base - 1 (a row that sees no drafted row) to base + 63
    lo = base - 1 - a.window;
    lo_all = base + 63 - a.window;
    hi = len - 1;
    hi_all = base - 1;
    np_all = np < base ? np : base;
  } else {
    lo = base + t_lo - a.window;
    lo_all = base + t_hi - a.window;
    hi = base + t_hi;
    hi_all = base + t_lo;
    if (hi < a.np) hi = -1;            // only persistent rows
    if (hi_all < a.np) hi_all = -1;    // some
  }
  if (lo < np) lo = np;
  int n_a = (np + 31) >> 5, b0 = lo >> 5, n_b = 0;
  if (b0 < n_a) b0 = n_a;
  if (hi >= lo) n_b = (hi >> 5) - b0 + 1;
  if (n_b < 0) n_b = 0;
  const int n_tiles = work ? n_a + n_b : 0;
  int tile0 = 0, tile1 = n_tiles;
  if (a.splits > 1) {
    const int per = (n_tiles + a.splits - 1u) / static_cast<unsigned>(a.splits);
    tile0 = per * split < n_tiles ? per * split : n_tiles;
    tile1 = tile0 + per < n_tiles ? tile0 + per : n_tiles;
  }

  // this lane's rows, one of each 16
  Row row[RT];
  u32x4 q16[RT][S::kF32 ? 1 : S::kPieces * S::kOps];
  float q32[RT][S::kF32 ? S::kPieces * S::kRun : 1];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = row0 + 16 * rt + n, t = by_group(a, r), gg = r - t * G;
    const bool real = r < rows_all;  // read whatever the sequence's numbers are, which arrive later
    row[rt] = work && t < s.n ? row_of(a, s, b, t) : Row{0, 1, 0, 0};
    const uint8_t* const src = a.q + (b * a.qb + (hk * G + gg) * a.qh + t * a.qt) * kRowSize<DT>;
#pragma unroll
    for (int c = 0; c < S::kPieces; ++c) {
      float x[S::kRun];
#pragma unroll
      for (int u = 0; u < S::kRun; ++u) x[u] = 0.f;
      const int i0 = 4 * S::kRun * c + S::kRun * g;
      if (real) {
        if (a.q_vec) {
          constexpr int N = kRowVec<DT>;
#pragma unroll
          for (int u = 0; u < S::kRun; u += N) {
            if (i0 + u >= a.c.d) continue;
            float y[N];
            row_load<DT, N>(src + (i0 + u) * kRowSize<DT>, y);
#pragma unroll
            for (int e = 0; e < N; ++e) x[u + e] = y[e];
          }
        } else {
#pragma unroll
          for (int u = 0; u < S::kRun; ++u) {
            float y[1] = {0.f};
            if (i0 + u < a.c.d) row_load<DT, 1>(src + (i0 + u) * kRowSize<DT>, y);
            x[u] = y[0];
          }
        }
      }
      if constexpr (S::kF32) {
#pragma unroll
        for (int u = 0; u < S::kRun; ++u) q32[rt][c * S::kRun + u] = x[u];
      } else {
#pragma unroll
        for (int e = 0; e < S::kOps; ++e) {
          u32x4 w;
#pragma unroll
          for (int u = 0; u < 4; ++u) w[u] = Mfma<DT>::pack2(x[8 * e + 2 * u], x[8 * e + 2 * u + 1]);
          q16[rt][c * S::kOps + e] = w;
        }
      }
    }
  }

  f32x4 acc[RT][NJ];
  float m[RT], l[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m[rt] = -kInf;
    l[rt] = 0.f;
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[rt][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const int page_mask = (1 << a.c.page_shift) - 1, pitch_b = a.c.pitch * S::kElem;
  const int k_off = n * pitch_b + g * 16;                  // of a key's first piece, in a group of 16 keys
  const int v_off = 4 * g * pitch_b + n * NB;              // of the values' pieces, likewise
  const bool v_in = n * NJ < a.c.pitch;                    // columns of d: others are not read
  const int32_t* const table = a.c.table + b * a.c.table_stride;
  constexpr bool kScaled16 = DT == TMAC_F16 && FMT != kCacheSame;
  float v_ref = 0x1p-126f;
  bool cleaned = false;

  // The next tile's pages are looked up while this one is worked on; its keys are asked for when this one's have been
  // multiplied, its values when this one's have.
  Piece<16> kp[2][S::kPieces];
  Piece<NB> vp[8];
  float ks[8], vs[8];
  int page_next[2];
  auto look_up = [&](int it) {
    const int key0 = (it < n_a ? it : b0 + it - n_a) << 5;
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int key = key0 + 16 * hf;
      page_next[hf] = it < tile1 && key < len ? table[key >> a.c.page_shift] : 0;
    }
  };
  auto group_row = [&](int it, int hf, int page) {  // the pool's row of a group of 16 keys
    const int key = ((it < n_a ? it : b0 + it - n_a) << 5) + 16 * hf;
    if (page < 0 || page >= a.c.n_pages) page = 0;
    return ((static_cast<int64_t>(page) * a.c.n_heads + hk) << a.c.page_shift) + (key & page_mask);
  };
  auto load_keys = [&](const int64_t (&r)[2]) {
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const uint8_t* const kb = a.c.k + r[hf] * pitch_b;
#pragma unroll
      for (int c = 0; c < S::kPieces; ++c) {
        if (4 * S::kRun * c + S::kRun * g < a.c.pitch)
          kp[hf][c].load(kb + k_off + 64 * c);
        else
          kp[hf][c].clear();
      }
      if constexpr (FMT != kCacheSame) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(a.c.ks + r[hf] + 4 * g);
#pragma unroll
        for (int i = 0; i < 4; ++i) ks[4 * hf + i] = x[i];
      }
    }
  };
  auto load_values = [&](const int64_t (&r)[2]) {
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const uint8_t* const vb = a.c.v + r[hf] * pitch_b;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (v_in)
          vp[4 * hf + i].load(vb + v_off + i * pitch_b);
        else
          vp[4 * hf + i].clear();
      }
      if constexpr (FMT != kCacheSame) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(a.c.vs + r[hf] + 4 * g);
#pragma unroll
        for (int i = 0; i < 4; ++i) vs[4 * hf + i] = x[i];
      }
    }
  };
  int64_t at[2];
  if (tile0 + wave < tile1) {
    look_up(tile0 + wave);
    at[0] = group_row(tile0 + wave, 0, page_next[0]);
    at[1] = group_row(tile0 + wave, 1, page_next[1]);
    load_keys(at);
    load_values(at);
  }
  for (int it = tile0 + wave; it < tile1; it += n_waves) {
    const int key0 = (it < n_a ? it : b0 + it - n_a) << 5;
    bool bad[2];
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) bad[hf] = page_next[hf] < 0 || page_next[hf] >= a.c.n_pages;
    const bool more = it + n_waves < tile1;
    look_up(it + n_waves);
    // every row sees the whole tile (rows that are none see it too: their results are not used)
    const bool full = !bad[0] && !bad[1] && (key0 + 31 < np_all || (key0 >= lo_all && key0 + 31 <= hi_all));
    bool seen[8];  // by any row
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int key = key0 + 16 * (i >> 2) + 4 * g + (i & 3);
      seen[i] = full || (!bad[i >> 2] && (key < np || (key >= lo && key <= hi)));
    }
    // fp16 probabilities times a scale of the values: relative to a power of two above all scales so far
    if constexpr (kScaled16) {
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, seen[i] ? vs[i] : 0.f);
      top = fmaxf(top, lane_xor<16>(top));
      top = fmaxf(top, lane_xor<32>(top));
      if (top > v_ref) {  // the same in all lanes
        const float to = __uint_as_float(((__float_as_uint(top) >> 23) + (top < 0x1p126f)) << 23);
        const float f = v_ref / to;
        v_ref = to;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int j = 0; j < NJ; ++j) acc[rt][j] *= f;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) vs[i] *= 1.f / v_ref;
    }
    float p[RT][8], ks_now[8];
    f32x4 sc[RT][2];
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) sc[rt][hf] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < S::kPieces; ++c)
#pragma unroll
        for (int e = 0; e < S::kOps; ++e) {
          const auto key = key_operand<DT, FMT, DP>(kp[hf][c], e);
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            if constexpr (S::kF32)
              sc[rt][hf] = __builtin_amdgcn_mfma_f32_16x16x4f32(key, q32[rt][c * S::kRun + e], sc[rt][hf], 0, 0, 0);
            else
              sc[rt][hf] = mfma16<DT>(key, q16[rt][c * S::kOps + e], sc[rt][hf]);
          }
        }
    }
    if constexpr (FMT != kCacheSame) {
#pragma unroll
      for (int i = 0; i < 8; ++i) ks_now[i] = ks[i];
    }
    if (more) {
      at[0] = group_row(it + n_waves, 0, page_next[0]);
      at[1] = group_row(it + n_waves, 1, page_next[1]);
      load_keys(at);
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float x[8], mx = -kInf;
      uint32_t vis = 0xff;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = sc[rt][i >> 2][i & 3] * a.scale2;
        if constexpr (FMT != kCacheSame) x[i] *= ks_now[i];
      }
      if (!full) {
        vis = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int key = key0 + 16 * (i >> 2) + 4 * g + (i & 3);
          const bool v = sees(row[rt], key, base, tree);
          if (bad[i >> 2]) x[i] = __builtin_nanf("");
          if (!v) x[i] = -kInf;
          vis |= static_cast<uint32_t>(v) << i;
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) mx = fmaxf(mx, x[i]);
      if (__any(mx > m[rt])) {
        mx = fmaxf(mx, lane_xor<16>(mx));
        mx = fmaxf(mx, lane_xor<32>(mx));
        const float to = fmaxf(m[rt], mx);
        const float f = to == m[rt] ? 1.f : __builtin_amdgcn_exp2f(m[rt] - to);
        m[rt] = to;
        l[rt] *= f;
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[rt][j] *= f;
      }
      const float mu = m[rt] == -kInf ? 0.f : m[rt];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float e = __builtin_amdgcn_exp2f(x[i] - mu);
        l[rt] += e;
        if constexpr (FMT != kCacheSame) e = vis >> i & 1 ? e * vs[i] : 0.f;
        p[rt][i] = e;
      }
    }
    // Values of keys that no row sees may be anything: zeros in their place. So may be those that some rows see and
    // others do not (0 times infinity): zeros here, added after the loop for the rows that see them.
    if (!full) {
      uint32_t changed = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (!seen[i]) vp[i].clear();
        if (FMT == kCacheSame && a.c.T > 1) {
#pragma unroll
          for (int w = 0; w < NB / 4; ++w) {
            const uint32_t x = finite_only<DT>(vp[i].w[w]);
            changed |= x ^ vp[i].w[w];
            vp[i].w[w] = x;
          }
        }
      }
      if (FMT == kCacheSame && __any(changed != 0)) cleaned = true;
    }
    u32x4 pw[RT];
    if constexpr (!S::kF32) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int w = 0; w < 4; ++w) pw[rt][w] = Mfma<DT>::pack2(p[rt][2 * w], p[rt][2 * w + 1]);
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      if constexpr (S::kF32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float v = value_f32<FMT, NB>(vp[i], j);
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
            acc[rt][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, p[rt][i], acc[rt][j], 0, 0, 0);
        }
      } else {
        const u32x4 v = value_operand<DT, FMT, NB>(vp, j);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) acc[rt][j] = mfma16<DT>(v, pw[rt], acc[rt][j]);
      }
    }
    if (more) load_values(at);
  }

  if constexpr (kScaled16) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[rt][j] *= v_ref;
  }
  if (FMT == kCacheSame && cleaned) {
    // What was taken for zeros and is not finite, to the rows that see it.
    for (int it = tile0 + wave; it < tile1; it += n_waves) {
      const int key0 = (it < n_a ? it : b0 + it - n_a) << 5;
      if (key0 + 31 < np_all || (key0 >= lo_all && key0 + 31 <= hi_all)) continue;
      for (int key = key0; key < key0 + 32 && key < len; ++key) {
        const int64_t r = cache_row(a.c, b, key, hk);
        if (r < 0) continue;
        const uint8_t* const vb = a.c.v + r * pitch_b;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < NJ; ++j) {
            const int col = (4 * g + i) * NJ + j;
            float v[1] = {0.f};
            if (col < a.c.d) row_load<DT, 1>(vb + col * S::kElem, v);
            if (__builtin_isfinite(v[0])) continue;
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
              if (sees(row[rt], key, base, tree)) acc[rt][j][i] += v[0];
          }
      }
    }
  }

  // The waves' results are joined in LDS: first the rows' maxima and sums, by which every wave scales what it has, then
  // the scaled results, summed in the waves' order. Rows of kPitchO floats: 16 rows begin at different banks.
  constexpr int kPitchO = DP + 4;
  const int cap = a.row_cap;
  float* const so = sh + wave * cap * kPitchO;
  float2* const sm = reinterpret_cast<float2*>(sh + WAVES * cap * kPitchO);  // [WAVES][cap]
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = 16 * rt + n;
    float sum = l[rt] + lane_xor<16>(l[rt]);
    sum += lane_xor<32>(sum);
    if (r < cap && g == 0) sm[wave * cap + r] = float2{m[rt], sum};
  }
  __syncthreads();
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = 16 * rt + n;
    if (r >= cap) continue;
    float top = -kInf;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, sm[w * cap + r].x);
    const float f = m[rt] == top ? 1.f : __builtin_amdgcn_exp2f(m[rt] - top);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < NJ; j += 4)
        *reinterpret_cast<f32x4*>(so + r * kPitchO + (4 * g + i) * NJ + j) =
            f32x4{acc[rt][j][i] * f, acc[rt][j + 1][i] * f, acc[rt][j + 2][i] * f, acc[rt][j + 3][i] * f};
  }
  __syncthreads();
  const int live = rows_all - row0 < cap ? rows_all - row0 : cap;
  for (int u = threadIdx.x; u < live * (DP / 4); u += 64 * WAVES) {
    const int r = u / (DP / 4), i0 = u % (DP / 4) * 4;
    float top = -kInf, sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, sm[w * cap + r].x);
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float2 x = sm[w * cap + r];
      sum += x.y * (x.x == top ? 1.f : __builtin_amdgcn_exp2f(x.x - top));
    }
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(sh + (w * cap + r) * kPitchO + i0);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += x[e];
    }
    if (a.splits > 1) {
      const int64_t at = ((static_cast<int64_t>(b) * a.c.n_heads + hk) * a.splits + split) * rows_all + row0 + r;
      float* const po = a.ws + at * (DP + 4);
      *reinterpret_cast<f32x4*>(po + i0) = f32x4{o[0], o[1], o[2], o[3]};
      if (i0 == 0) {
        po[DP] = top;
        po[DP + 1] = sum;
      }
      continue;
    }
    const int t = by_group(a, row0 + r), gg = row0 + r - t * G;
    row_finish(s, t, sum, o);
    row_out<DT>(a, b, t, hk * G + gg, i0, o);
  }
}

// The parts of a row: one group of DP / N lanes joins them in order.
template <int DT, int DP>
__global__ __launch_bounds__(256) void cached_attn_join_kernel(AttnArgs a) {
  constexpr int N = 4, L = DP / N;
  const int64_t u = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int rows_all = a.c.T * a.G;
  const int64_t r_all = u / L;
  const int i0 = static_cast<int>(u % L) * N;
  const int64_t bh = r_all / rows_all;
  const int r = static_cast<int>(r_all % rows_all);
  if (bh >= static_cast<int64_t>(a.B) * a.c.n_heads || i0 >= a.c.d) return;
  const int b = static_cast<int>(bh / a.c.n_heads), hk = static_cast<int>(bh % a.c.n_heads);
  const float* const p0 = a.ws + (bh * a.splits * rows_all + r) * (DP + 4);
  const int64_t step = static_cast<int64_t>(rows_all) * (DP + 4);
  float top = -kInf, sum = 0.f;
  float o[N] = {0.f, 0.f, 0.f, 0.f};
  for (int w = 0; w < a.splits; ++w) top = fmaxf(top, p0[w * step + DP]);
  for (int w = 0; w < a.splits; ++w) {
    const float mw = p0[w * step + DP], lw = p0[w * step + DP + 1];
    if (mw == -kInf && lw == 0.f) continue;
    const float f = mw == top ? 1.f : __builtin_amdgcn_exp2f(mw - top);
    sum += lw * f;
    const f32x4 x = *reinterpret_cast<const f32x4*>(p0 + w * step + i0);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += x[e] * f;
  }
  const int t = by_group(a, r), gg = r - t * a.G;
  row_finish(seq_of(a.c, b), t, sum, o);
  row_out<DT>(a, b, t, hk * a.G + gg, i0, o);
}

struct Plan {
  int rt, waves, n_rb, splits, row_cap;
  size_t ws;
};

// rows: query rows per key head; blocks of rows of all sequences and heads; tiles of keys that a block may have to walk
Plan plan(const CacheArgs& c, int dtype, int B, int rows, int64_t window, int np) {
  Plan p{};
  const int dp = c.pitch <= 64 ? 64 : 128;
  p.rt = rows <= 16 ? 1 : dtype == TMAC_F32 ? 2 : 4;
  const int cap = 16 * p.rt;
  p.n_rb = (rows + cap - 1) / cap;
  p.row_cap = rows < cap ? rows : cap;
  const int64_t len = static_cast<int64_t>(c.max_pages) << c.page_shift;
  int64_t keys = window + c.T + np;
  if (keys > len) keys = len;
  const int64_t tiles = keys / 32 + 2;
  const int most = p.rt > 1 ? 4 : dtype != TMAC_F32 && dp == 64 ? 16 : 8;
  p.waves = tiles >= 2 * 8 && most == 16 ? 16 : tiles > 4 && most >= 8 ? 8 : 4;
  const int64_t blocks = static_cast<int64_t>(B) * c.n_heads * p.n_rb;
  // enough workgroups for every CU, each wave with 4 tiles at least
  int64_t s = (1024 + blocks - 1) / blocks;
  const int64_t by_len = tiles / (4 * p.waves);
  if (s > by_len) s = by_len;
  if (s > 64) s = 64;
  p.splits = s < 1 ? 1 : static_cast<int>(s);
  p.ws = p.splits > 1 ? static_cast<size_t>(B) * c.n_heads * p.splits * rows * (dp + 4) * 4 : 0;
  return p;
}

int check(const tmac_cache* cache, int B, int T, int Hq, int64_t window, int np, CacheArgs& c) {
  const int st = cache_args(cache, B, T, c);
  if (st != TMAC_OK) return st;
  if (Hq <= 0 || Hq > 65535 || Hq % c.n_heads || static_cast<int64_t>(T) * Hq > (1 << 26)) return TMAC_ERR_SHAPE;
  if (window < 0 || np < 0) return TMAC_ERR_VALUE;
  return TMAC_OK;
}

// Most waves of a workgroup with one tile of rows: as many as leave each the registers that it needs.
template <int DT, int DP>
constexpr int kMostWaves = DT != TMAC_F32 && DP == 64 ? 16 : 8;

template <int DT, int FMT, int DP>
void launch(const AttnArgs& a, const Plan& p, hipStream_t s) {
  const dim3 grid(a.B, a.c.n_heads, p.n_rb * p.splits);
  const size_t lds = static_cast<size_t>(p.waves) * p.row_cap * (DP + 4 + 2) * 4;
  constexpr int kMany = DT == TMAC_F32 ? 2 : 4, kMost = kMostWaves<DT, DP>;
  if (p.rt > 1)
    cached_attn_kernel<DT, FMT, DP, kMany, 4><<<grid, 64 * 4, lds, s>>>(a);
  else if (p.waves == 4)
    cached_attn_kernel<DT, FMT, DP, 1, 4><<<grid, 64 * 4, lds, s>>>(a);
  else if (p.waves == 8)
    cached_attn_kernel<DT, FMT, DP, 1, 8><<<grid, 64 * 8, lds, s>>>(a);
  else
    cached_attn_kernel<DT, FMT, DP, 1, kMost><<<grid, 64 * kMost, lds, s>>>(a);
  if (p.splits > 1) {
    const int64_t threads = static_cast<int64_t>(a.B) * a.c.n_heads * a.c.T * a.G * (DP / 4);
    cached_attn_join_kernel<DT, DP><<<static_cast<unsigned>((threads + 255) / 256), 256, 0, s>>>(a);
  }
}

template <int DT, int FMT>
void by_width(const AttnArgs& a, const Plan& p, hipStream_t s) {
  if (a.c.pitch <= 64)
    launch<DT, FMT, 64>(a, p, s);
  else
    launch<DT, FMT, 128>(a, p, s);
}

template <int DT>
void by_format(int format, const AttnArgs& a, const Plan& p, hipStream_t s) {
  if (format == TMAC_CACHE_SAME)
    by_width<DT, kCacheSame>(a, p, s);
  else if (format == TMAC_CACHE_INT8)
    by_width<DT, kCacheInt8>(a, p, s);
  else
    by_width<DT, kCacheE4m3>(a, p, s);
}

}  // namespace

extern "C" int tmac_cached_attn_workspace(const tmac_cache* cache, int B, int T, int n_q_heads, int64_t window,
                                          int n_persistent, size_t* ws_bytes) {
  CacheArgs c;
  if (!ws_bytes) return TMAC_ERR_NULL;
  const int st = check(cache, B, T, n_q_heads, window, n_persistent, c);
  if (st != TMAC_OK) return st;
  *ws_bytes = B && T ? plan(c, cache->dtype, B, T * (n_q_heads / c.n_heads), window, n_persistent).ws : 0;
  return TMAC_OK;
}

extern "C" int tmac_cached_attn(const tmac_cache* cache, const void* d_q, const int64_t* h_q_strides,
                                const int64_t* d_tree, int64_t tree_stride, void* d_out, void* d_ws, size_t ws_bytes,
                                int B, int T, int n_q_heads, int64_t window, int n_persistent, float scale,
                                void* stream) {
  AttnArgs a{};
  const int st = check(cache, B, T, n_q_heads, window, n_persistent, a.c);
  if (st != TMAC_OK) return st;
  if (d_tree && (T > TMAC_CACHE_MAX_TREE || (tree_stride != 0 && tree_stride < T))) return TMAC_ERR_SHAPE;
  if (B == 0 || T == 0) return TMAC_OK;
  if (!d_q || !h_q_strides || !d_out) return TMAC_ERR_NULL;
  const int G = n_q_heads / a.c.n_heads;
  const Plan p = plan(a.c, cache->dtype, B, T * G, window, n_persistent);
  if (p.ws && (!d_ws || ws_bytes < p.ws)) return TMAC_ERR_WORKSPACE;
  if (p.ws && !row_aligned16(d_ws)) return TMAC_ERR_ALIGN;
  if (static_cast<int64_t>(p.n_rb) * p.splits > 65535 || static_cast<int64_t>(B) * n_q_heads * T > (1 << 26))
    return TMAC_ERR_SHAPE;
  const int n = cache->dtype == TMAC_F32 ? 4 : 8;
  a.q = static_cast<const uint8_t*>(d_q);
  a.qb = h_q_strides[0], a.qh = h_q_strides[1], a.qt = h_q_strides[2];
  a.tree = d_tree, a.tree_stride = tree_stride;
  a.out = static_cast<uint8_t*>(d_out);
  a.ws = static_cast<float*>(d_ws);
  a.B = B, a.Hq = n_q_heads, a.G = G, a.g_shift = G & (G - 1) ? -1 : __builtin_ctz(G), a.n_rb = p.n_rb, a.splits = p.splits, a.row_cap = p.row_cap;
  constexpr int kMost = 1 << 30;
  a.np = n_persistent < kMost ? n_persistent : kMost;
  a.window = window < kMost ? static_cast<int>(window) : kMost;
  a.scale2 = scale * kLog2e;
  a.q_vec = row_aligned16(d_q) && a.c.d % n == 0 && a.qb % n == 0 && a.qh % n == 0 && a.qt % n == 0;
  a.out_vec = row_aligned16(d_out) && a.c.d % 4 == 0;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (cache->dtype == TMAC_F32)
    by_format<TMAC_F32>(cache->format, a, p, s);
  else if (cache->dtype == TMAC_BF16)
    by_format<TMAC_BF16>(cache->format, a, p, s);
  else
    by_format<TMAC_F16>(cache->format, a, p, s);
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? TMAC_OK : static_cast<int>(err);
}
