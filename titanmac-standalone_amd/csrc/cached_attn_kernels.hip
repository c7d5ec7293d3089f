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
//
// fp32 on codes of 8 bits runs on the 16-bit matrix cores all the same: a code is exact in bfloat16, and an fp32 value is
// the sum of three bfloat16 numbers (8 bits each of its 24), so three products give what an fp32 one gives, in a fifth
// of its time. fp16 probabilities times a value's scale leave fp16's range (a small row's where a large one is also
// held), so those are two bfloat16 numbers, which have fp32's.
template <int DT, int FMT, int DP>
struct Shape {
  static constexpr bool kF32 = DT == TMAC_F32 && FMT == kCacheSame;  // fp32 products
  static constexpr int kType = DT == TMAC_F32 ? TMAC_BF16 : DT;      // of the others
  static constexpr int kParts = DT == TMAC_F32 && FMT != kCacheSame ? 3 : 1;
  static constexpr bool kScaled16 = DT == TMAC_F16 && FMT != kCacheSame;
  static constexpr int kProbType = kScaled16 ? TMAC_BF16 : kType;    // of the second product
  // Probabilities in 16 bit are two numbers, whoever shares the launch: the result's rounding is then the only one of its
  // size. With one, the error over 8192 positions was 0.0023 of the result in bfloat16, with two 0.0017, its rounding's.
  static constexpr int kProbs = kF32 ? 1 : kParts > 1 ? kParts : 2;
  // fp16's least number is 2^-24, and so much is lost of each of a long axis' small probabilities: they are taken times
  // 2^kLift (with kSlack, up to 2^15).
  static constexpr int kLift = DT == TMAC_F16 && FMT == kCacheSame ? 7 : 0;
  static constexpr int kElem = FMT != kCacheSame ? 1 : DT == TMAC_F32 ? 4 : 2;  // bytes of a stored value
  static constexpr int kRun = 16 / kElem;           // values in 16 bytes: a lane's piece of a key
  static constexpr int kPieces = DP / (4 * kRun);   // of each key, per lane; piece c of group g: 4 kRun c + kRun g ..
  static constexpr int kOps = kF32 ? kRun : kRun / 8;  // products per piece
  static constexpr int NJ = DP / 16;                // columns of the values per lane, products per 32 keys
};

// Whether a wave needs more than half of a SIMD's registers: four waves a workgroup then.
constexpr bool wide(int dtype, bool same, int dp, int rt) { return dtype == TMAC_F32 && dp == 128 && (same || rt > 1); }

// x, y as the sum of P pairs of TYPE, each the nearest to what the ones before leave
template <int TYPE, int P>
__device__ __forceinline__ void split2(float x, float y, uint32_t (&w)[P]) {
#pragma unroll
  for (int i = 0; i < P; ++i) {
    w[i] = Mfma<TYPE>::pack2(x, y);
    x -= Mfma<TYPE>::to_f32(static_cast<uint16_t>(w[i]));
    y -= Mfma<TYPE>::to_f32(static_cast<uint16_t>(w[i] >> 16));
  }
}

// Probabilities x, y as the sum of two pairs of TYPE that are both above 0 where x, y are (a number below 0, or 0, times an
// infinite value would be NaN beside the other's infinity): the first is the number below the leading bits of x, so the
// second has one to two of its last places. 2^-15 of x at most are left over in bfloat16, 2^-21 (or half of the least
// number) in fp16.
template <int TYPE>
__device__ __forceinline__ void split_positive2(float x, float y, uint32_t (&w)[2]) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  uint32_t lead;
  if constexpr (TYPE == TMAC_BF16)
    lead = __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);
  else
    lead = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x, y));
  w[0] = __builtin_bit_cast(uint32_t, __builtin_elementwise_sub_sat(__builtin_bit_cast(u16x2, lead), u16x2{1, 1}));
  w[1] = Mfma<TYPE>::pack2(x - Mfma<TYPE>::to_f32(static_cast<uint16_t>(w[0])),
                           y - Mfma<TYPE>::to_f32(static_cast<uint16_t>(w[0] >> 16)));
}

// Probabilities (times the values' scales in 8 bits, which may be of any sign) as the sum of kProbs pairs of kProbType.
template <int DT, int FMT, int DP>
__device__ __forceinline__ void split_probs(float x, float y, uint32_t (&w)[Shape<DT, FMT, DP>::kProbs]) {
  using S = Shape<DT, FMT, DP>;
  if constexpr (FMT == kCacheSame && !S::kF32)
    split_positive2<S::kProbType>(x, y, w);
  else
    split2<S::kProbType, S::kProbs>(x, y, w);
}

// operand e of a key's piece
template <int DT, int FMT, int DP>
__device__ __forceinline__ auto key_operand(const Piece<16>& p, int e) {
  if constexpr (DT == TMAC_F32 && FMT == kCacheSame) {
    return __uint_as_float(p.w[e]);
  } else if constexpr (FMT == kCacheSame) {
    return u32x4{p.w[0], p.w[1], p.w[2], p.w[3]};
  } else {
    constexpr int kType = Shape<DT, FMT, DP>::kType;
    const uint32_t lo = p.w[2 * e], hi = p.w[2 * e + 1];
    return u32x4{code2<kType, FMT, false>(lo), code2<kType, FMT, true>(lo), code2<kType, FMT, false>(hi),
                 code2<kType, FMT, true>(hi)};
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
struct AttnArgs {
  CacheArgs c;
  const uint8_t* q;
  int64_t qb, qh, qt;
  const int64_t* tree;
  int64_t tree_stride;
  uint8_t* out;
  float* ws;
  int B, Hq, G, g_shift, n_rb, splits, np, row_cap, per_xcd, n_blocks;  // g_shift: log2 of G, or -1
  int window;  // up to kNowhere: none
  float scale2, slack, q_sign;  // slack: kSlack / scale2; scale2: |scale| · log2 e (1 for scale 0); the queries are taken times q_sign, the scale's sign
  bool q_vec, out_vec;
};

// A division costs a wave a few dozen instructions, in a kernel that may be done in a few hundred.
__device__ __forceinline__ int by_group(const AttnArgs& a, int r) {
  return a.g_shift >= 0 ? r >> a.g_shift : static_cast<int>(static_cast<unsigned>(r) / static_cast<unsigned>(a.G));
}

// What a row sees: j < np, lo <= j <= lo + span, and drafted rows by bits. (kNowhere: past every position.)
constexpr int kNowhere = 1 << 30;
struct Row {
  int np, lo;
  uint32_t span;
  uint64_t bits;
};
__device__ __forceinline__ Row no_row() { return Row{0, kNowhere, 0, 0}; }

__device__ __forceinline__ bool in_span(int j, int lo, uint32_t span) { return static_cast<uint32_t>(j - lo) <= span; }
__device__ __forceinline__ bool sees(const Row& r, int j, int base) {
  const uint32_t s = static_cast<uint32_t>(j - base);
  return (j < r.np) | in_span(j, r.lo, r.span) | (s < 64u && (r.bits >> (s & 63u) & 1));
}

__device__ __forceinline__ int bits_set(int64_t x) { return static_cast<int>(__popcll(static_cast<uint64_t>(x))); }

// Row t of sequence s. Without a tree position p = base + t.
__device__ __forceinline__ Row row_of(const AttnArgs& a, const Seq& s, int b, int t) {
  Row r = no_row();
  if (t >= s.n) return r;
  const int base = s.len - s.n, np = a.np < s.len ? a.np : s.len;
  if (!a.tree) {
    const int p = base + t, lo = p - a.window > 0 ? p - a.window : 0;
    r.np = np;
    if (p >= a.np) {
      r.lo = lo;
      r.span = p - lo;
    }
    return r;
  }
  const int64_t* const tree = a.tree + b * a.tree_stride;
  const uint64_t have = s.n >= 64 ? ~0ull : (1ull << s.n) - 1;
  const int p = base + bits_set(tree[t]) - 1, lo = p - a.window > 0 ? p - a.window : 0;
  r.np = np < base ? np : base;
  if (lo < base) {
    r.lo = lo;
    r.span = base - 1 - lo;
  }
  r.bits = static_cast<uint64_t>(tree[t]) & have;
  if (a.window < TMAC_CACHE_MAX_TREE) {  // drafted rows may be behind the window: their places differ by up to 64
    for (int u = 0; u < s.n; ++u)
      if (base + bits_set(tree[u]) - 1 < p - a.window && base + u >= a.np) r.bits &= ~(1ull << u);
  }
  return r;
}

// The 32 bits of x from bit s on (s may be negative: zeros below bit 0).
__device__ __forceinline__ uint32_t bits_from(uint64_t x, int s) {
  if (s >= 64 || s <= -32) return 0;
  return static_cast<uint32_t>(s >= 0 ? x >> s : x << -s);
}

// The keys of a block of rows t_lo .. t_hi, as tiles of 2^SH: those with persistent keys, then those of [lo, hi] behind
// them. Every key that a row sees is below np or in [lo, hi]; every row sees the keys below np_all and in
// [lo_all, hi_all].
template <int SH>
struct Keys {
  int np, np_all, lo, hi, lo_all, hi_all, n_a, b0, n_tiles;
  __device__ __forceinline__ int first(int it) const { return (it < n_a ? it : b0 + it - n_a) << SH; }
  __device__ __forceinline__ bool all_see(int key0, int last = (1 << SH) - 1) const {
    return key0 + last < np_all || (key0 >= lo_all && key0 + last <= hi_all);
  }
  __device__ __forceinline__ bool any_sees(int key0, int last) const {
    return key0 < np || (key0 + last >= lo && key0 <= hi);
  }
};

template <int SH = 5>
__device__ __forceinline__ Keys<SH> keys_of(const AttnArgs& a, const Seq& s, int t_lo, int t_hi) {
  Keys<SH> k;
  const int base = s.len - s.n;
  k.np = a.np < s.len ? a.np : s.len;
  k.np_all = k.np;
  if (a.tree) {  // places from base - 1 (a row that sees no drafted row) to base + 63
    k.lo = base - 1 - a.window;
    k.lo_all = base + 63 - a.window;
    k.hi = s.len - 1;
    k.hi_all = base - 1;
    if (base < k.np_all) k.np_all = base;
  } else {
    k.lo = base + t_lo - a.window;
    k.lo_all = base + t_hi - a.window;
    k.hi = base + t_hi;
    k.hi_all = base + t_lo;
    if (k.hi < a.np) k.hi = -1;          // persistent rows only
    if (k.hi_all < a.np) k.hi_all = -1;  // some persistent rows
  }
  if (k.lo < k.np) k.lo = k.np;
  k.n_a = (k.np + (1 << SH) - 1) >> SH;
  k.b0 = k.lo >> SH > k.n_a ? k.lo >> SH : k.n_a;
  const int n_b = k.hi >= k.lo ? (k.hi >> SH) - k.b0 + 1 : 0;
  k.n_tiles = s.ok && t_lo < s.n ? k.n_a + (n_b > 0 ? n_b : 0) : 0;
  return k;
}

// Two 16-bit values, one fp32, or four codes: the top bit of each that is not finite (any bit for fp32), and w with
// zeros in their place.
template <int DT, int FMT>
__device__ __forceinline__ uint32_t not_finite_bits(uint32_t w) {
  if constexpr (FMT == kCacheE4m3) return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
  if constexpr (DT == TMAC_F32) return (w & 0x7f800000u) == 0x7f800000u;
  constexpr uint32_t kExp = DT == TMAC_BF16 ? 0x7f807f80u : 0x7c007c00u, kLow = DT == TMAC_BF16 ? 0x00800080u : 0x04000400u;
  return ((w & kExp) + kLow) & 0x80008000u;
}
template <int DT, int FMT>
__device__ __forceinline__ uint32_t finite_only(uint32_t w) {
  const uint32_t t = not_finite_bits<DT, FMT>(w);
  if constexpr (FMT == kCacheE4m3) return w & ~((t >> 7) * 0xffu);
  if constexpr (DT == TMAC_F32) return t ? 0u : w;
  return w & ~((t >> 15) * 0xffffu);
}

// What finite_only takes from a stored value: the value, if it is not finite, or 0.
template <int DT, int FMT>
__device__ __forceinline__ float not_finite(const uint8_t* p) {
  if constexpr (FMT == kCacheE4m3) return (*p & 0x7f) == 0x7f ? __builtin_nanf("") : 0.f;
  float v[1];
  row_load<DT, 1>(p, v);
  return __builtin_isfinite(v[0]) ? 0.f : v[0];
}

// Bit i: the row sees the i-th of this lane's eight keys kb, kb + 1, .. kb + 3, kb + 16, .. kb + 19.
__device__ __forceinline__ uint32_t row_sees(const Row& r, int kb, int base, bool tree) {
  uint32_t vis = 0;
  if (tree) vis = (bits_from(r.bits, kb - base) & 15u) | (bits_from(r.bits, kb + 16 - base) & 15u) << 4;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int key = kb + 16 * (i >> 2) + (i & 3);
    vis |= ((key < r.np) | in_span(key, r.lo, r.span)) ? 1u << i : 0u;
  }
  return vis;
}

// The running softmax of a row, as the lanes that hold it have it. Exponents are taken relative to mu, which is a score
// times scale2, less LIFT (0 while there is none) and moves only for one that is more than kSlack above it: up to then
// exponentials stay below 2^kSlack, where the sums in fp32 and the probabilities in 16 bit are as good. Moving costs as
// much as a tile's exponentials, and a wave's 16 rows have a new largest score in two of three tiles of 40. lim: that
// bound, not scaled; l: this lane's part of the sum.
constexpr float kSlack = 8.f;
struct Soft {
  float lim, mu, l;
};

// Scores x (−inf where masked) become exponentials times 2^LIFT; what was summed up before moves with mu.
template <int LIFT, int NJ>
__device__ __forceinline__ void soften(Soft& s, float (&x)[8], f32x4 (&acc)[NJ], const AttnArgs& a) {
  float mx = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) mx = fmaxf(mx, x[i]);
  if (__any(mx > s.lim)) {
    mx = fmaxf(mx, lane_xor<16>(mx));
    mx = fmaxf(mx, lane_xor<32>(mx));
    if (mx > s.lim) {  // the same in the row's four lanes
      const float to = fmaf(mx, a.scale2, -static_cast<float>(LIFT)), f = s.lim == -kInf ? 1.f : __builtin_amdgcn_exp2f(s.mu - to);
      s.lim = mx + a.slack;
      s.mu = to;
      s.l *= f;
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[j] *= f;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = __builtin_amdgcn_exp2f(fmaf(x[i], a.scale2, -s.mu));
    s.l += x[i];
  }
}
// The row's sum from its lanes', and what it is relative to: mu, or −inf for a row that saw nothing (one that saw
// nothing but NaN has a sum of NaN).
__device__ __forceinline__ float soft_join(Soft& s) {
  s.l += lane_xor<16>(s.l);
  s.l += lane_xor<32>(s.l);
  return s.lim == -kInf && s.l == s.l ? -kInf : s.mu;
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

// ROWS: the workgroup's waves hold a block of rows each and walk the same keys, for many rows in fp32 (whose products
// take four times as long as their operands' loads); otherwise they hold the same rows and share the keys out.
template <int DT, int FMT, int DP, int RT, int WAVES, bool ROWS>
__global__ __launch_bounds__(64 * WAVES, (wide(DT, FMT == kCacheSame, DP, RT) ? 1 : 2)) void cached_attn_kernel(AttnArgs a) {
  using S = Shape<DT, FMT, DP>;
  constexpr int NJ = S::NJ, kRows = 16 * RT, NB = NJ * S::kElem;
  extern __shared__ float sh[];
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int b, hk, rb, split;
  if constexpr (ROWS) {  // the blocks of a sequence's head, which read the same keys, on one XCD
    int id = xcd_logical_id(a.per_xcd);
    if (id >= a.n_blocks) return;
    rb = id % a.n_rb, id /= a.n_rb;
    split = id % a.splits, id /= a.splits;
    hk = id % a.c.n_heads, b = id / a.c.n_heads;
    rb = rb * WAVES + wave;
  } else {
    b = blockIdx.x, hk = blockIdx.y;
    rb = a.splits == 1 ? blockIdx.z : blockIdx.z / static_cast<unsigned>(a.splits);
    split = blockIdx.z - rb * a.splits;
  }
  const Seq s = seq_of(a.c, b);
  const int rows_all = a.c.T * a.G, row0 = rb * kRows, G = a.G;
  const int t_lo = by_group(a, row0), t_end = by_group(a, row0 + kRows - 1);
  const Keys<5> keys = keys_of(a, s, t_lo, t_end < s.n - 1 ? t_end : s.n - 1);
  const int base = s.len - s.n, len = s.len;
  const bool tree = a.tree != nullptr;
  const bool mixed = a.c.T > 1 || tree;  // some rows may not see all of [lo, hi]
  int tile0 = 0, tile1 = keys.n_tiles;
  if (a.splits > 1) {
    const int per = (keys.n_tiles + a.splits - 1u) / static_cast<unsigned>(a.splits);
    tile0 = per * split < keys.n_tiles ? per * split : keys.n_tiles;
    tile1 = tile0 + per < keys.n_tiles ? tile0 + per : keys.n_tiles;
  }
  constexpr int kStep = ROWS ? 1 : WAVES;
  if (!ROWS) tile0 += wave;

  // The queries of this lane's rows, one of each 16. They are read whatever the sequence's numbers are, which arrive
  // later.
  Row row[RT];
  u32x4 q16[RT][S::kParts][S::kF32 ? 1 : S::kPieces * S::kOps];
  float q32[RT][S::kF32 ? S::kPieces * S::kRun : 1];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = row0 + 16 * rt + n, t = by_group(a, r), gg = r - t * G;
    const bool real = r < rows_all;
    row[rt] = real && keys.n_tiles ? row_of(a, s, b, t) : no_row();
    const uint8_t* const src = a.q + (b * a.qb + (hk * G + gg) * a.qh + t * a.qt) * kRowSize<DT>;
#pragma unroll
    for (int c = 0; c < S::kPieces; ++c) {
      const int i0 = 4 * S::kRun * c + S::kRun * g;
      if (DT != TMAC_F32 && a.q_vec) {
#pragma unroll
        for (int e = 0; e < S::kOps; ++e) {
          u32x4 w{0, 0, 0, 0};
          if (real && i0 + 8 * e < a.c.d) w = *reinterpret_cast<const u32x4*>(src + (i0 + 8 * e) * 2);
          q16[rt][0][S::kF32 ? 0 : c * S::kOps + e] = w;
        }
        continue;
      }
      float x[S::kRun];
#pragma unroll
      for (int u = 0; u < S::kRun; ++u) x[u] = 0.f;
      if (real) {
        if (DT == TMAC_F32 && a.q_vec) {
#pragma unroll
          for (int u = 0; u < S::kRun; u += 4) {
            if (i0 + u >= a.c.d) continue;
            const f32x4 y = *reinterpret_cast<const f32x4*>(src + (i0 + u) * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[u + e] = y[e];
          }
        } else {
#pragma unroll
          for (int u = 0; u < S::kRun; ++u) {
            float y[1] = {0.f};
            if (i0 + u < a.c.d) row_load<DT, 1>(src + (i0 + u) * kRowSize<DT>, y);
            x[u] = y[0] * a.q_sign;
          }
        }
      }
      if constexpr (S::kF32) {
#pragma unroll
        for (int u = 0; u < S::kRun; ++u) q32[rt][c * S::kRun + u] = x[u];
      } else {
#pragma unroll
        for (int e = 0; e < S::kOps; ++e) {
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            uint32_t w[S::kParts];
            split2<S::kType, S::kParts>(x[8 * e + 2 * u], x[8 * e + 2 * u + 1], w);
#pragma unroll
            for (int i = 0; i < S::kParts; ++i) q16[rt][i][c * S::kOps + e][u] = w[i];
          }
        }
      }
    }
  }

  f32x4 acc[RT][NJ];
  Soft soft[RT];

  const int page_mask = (1 << a.c.page_shift) - 1, pitch_b = a.c.pitch * S::kElem;
  const bool narrow = a.c.pitch < DP;
  // Byte offsets of this lane's pieces in a group of 16 keys. Columns past the pitch are read as the row's first: of keys
  // they are cleared, of values they end in results that are not stored.
  int k_off[S::kPieces];
#pragma unroll
  for (int c = 0; c < S::kPieces; ++c) {
    const int col = S::kRun * (4 * c + g);
    k_off[c] = n * pitch_b + (col < a.c.pitch ? col * S::kElem : 0);
  }
  const int v_off = 4 * g * pitch_b + (n * NJ < a.c.pitch ? n * NB : 0);
  const int32_t* const table = a.c.table + b * a.c.table_stride;

  // A tile's pages are looked up two tiles ahead; its keys are asked for when those of the tile before have been
  // multiplied, its values when those have. A tile has two pages where pages are of 16 rows.
  Piece<16> kp[2][S::kPieces];
  Piece<NB> vp[8];
  float ks[8], vs[8];
  const bool halves = a.c.page_shift < 5;
  int page[2], page_next[2] = {0, 0};  // of the tile whose rows were last asked for, and of the one behind it
  int key_next = 0;                    // the first key of the latter
  int64_t at[2];                       // byte offsets of the tile's two groups of 16 keys in the pools
  int64_t at_scale[2];                 // and their rows
  const uint32_t page_rows = static_cast<uint32_t>(a.c.n_heads) << a.c.page_shift, page_bytes = page_rows * pitch_b;
  const uint32_t head_rows = static_cast<uint32_t>(hk) << a.c.page_shift;
  auto look_up = [&](int it) {
    if (it >= tile1) return;
    key_next = keys.first(it);
    page_next[0] = table[key_next >> a.c.page_shift];
    if (halves) page_next[1] = key_next + 16 < len ? table[(key_next + 16) >> a.c.page_shift] : 0;
  };
  auto place = [&]() {
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      if (hf && !halves) {
        page[1] = page[0];
        at[1] = at[0] + 16 * pitch_b;
        at_scale[1] = at_scale[0] + 16;
        continue;
      }
      page[hf] = page_next[hf];
      const uint32_t p = static_cast<uint32_t>(page[hf]) < static_cast<uint32_t>(a.c.n_pages) ? page[hf] : 0;
      const uint32_t r = head_rows + ((key_next + 16 * hf) & page_mask);
      at[hf] = static_cast<int64_t>(static_cast<uint64_t>(p) * page_bytes + r * pitch_b);
      if (FMT != kCacheSame) at_scale[hf] = static_cast<int64_t>(static_cast<uint64_t>(p) * page_rows + r);
    }
  };
  auto load_keys = [&]() {
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const uint8_t* const kb = a.c.k + at[hf];
#pragma unroll
      for (int c = 0; c < S::kPieces; ++c) kp[hf][c].load(kb + k_off[c]);
      if constexpr (FMT != kCacheSame) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(a.c.ks + at_scale[hf] + 4 * g);
#pragma unroll
        for (int i = 0; i < 4; ++i) ks[4 * hf + i] = x[i];
      }
    }
  };
  auto load_values = [&]() {
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const uint8_t* const vb = a.c.v + at[hf];
#pragma unroll
      for (int i = 0; i < 4; ++i) vp[4 * hf + i].load(vb + i * pitch_b + v_off);
      if constexpr (FMT != kCacheSame) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(a.c.vs + at_scale[hf] + 4 * g);
#pragma unroll
        for (int i = 0; i < 4; ++i) vs[4 * hf + i] = x[i];
      }
    }
  };
  bool cleaned = false;
  // This wave's place in LDS: row_cap rows of kPitchO floats, so that 16 rows begin at different banks.
  constexpr int kPitchO = DP + 4;
  const int cap = a.row_cap;
  float* const so = sh + wave * cap * kPitchO;
  int key_now = 0;
  // One tile; `more`: the next one's loads are issued on the way. The last tile is code of its own: as a condition in one loop
  // the loads' registers were copied at its end, which waited for them there.
  auto one_tile = [&](int it, auto more) {
    const int key0 = key_now;
    bool bad[2];
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) bad[hf] = static_cast<unsigned>(page[hf]) >= static_cast<unsigned>(a.c.n_pages);
    // every row sees the whole tile (rows that are none see it too: their results are not used)
    const bool full = !bad[0] && !bad[1] && keys.all_see(key0);

    if (narrow) {
#pragma unroll
      for (int c = 0; c < S::kPieces; ++c)
        if (S::kRun * (4 * c + g) >= a.c.pitch) kp[0][c].clear(), kp[1][c].clear();
    }
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
            if constexpr (S::kF32) {
              sc[rt][hf] = __builtin_amdgcn_mfma_f32_16x16x4f32(key, q32[rt][c * S::kRun + e], sc[rt][hf], 0, 0, 0);
            } else {
#pragma unroll
              for (int i = 0; i < S::kParts; ++i)
                sc[rt][hf] = mfma16<S::kType>(key, q16[rt][i][c * S::kOps + e], sc[rt][hf]);
            }
          }
        }
    }
    float x[RT][8];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[rt][i] = sc[rt][i >> 2][i & 3];
        if constexpr (FMT != kCacheSame) x[rt][i] *= ks[i];
      }
    if constexpr (decltype(more)::value) {
      key_now = key_next;
      place();
      load_keys();
      look_up(it + 2 * kStep);
    }

    uint32_t vis[RT];  // bit i: the row sees key i of this lane's eight
    if (!full) {
      const int kb = key0 + 4 * g;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        vis[rt] = row_sees(row[rt], kb, base, tree);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (!(vis[rt] >> i & 1)) x[rt][i] = -kInf;
        if (bad[0] || bad[1]) {  // a page that is none: NaN for the rows that see it
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (bad[i >> 2] && (vis[rt] >> i & 1)) x[rt][i] = __builtin_nanf("");
        }
      }
      // Values of keys that no row sees may be anything: zeros in their place. So may be those that some rows see
      // and others do not (0 times infinity): zeros here, added after the loop for the rows that see them.
      const uint32_t span = keys.hi >= keys.lo ? keys.hi - keys.lo : 0;
      const int lo = keys.hi >= keys.lo ? keys.lo : kNowhere;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int key = kb + 16 * (i >> 2) + (i & 3);
        const uint32_t on = (((key < keys.np) | in_span(key, lo, span)) & !bad[i >> 2]) ? ~0u : 0u;
#pragma unroll
        for (int w = 0; w < NB / 4; ++w) vp[i].w[w] &= on;
        if constexpr (FMT != kCacheSame) vs[i] = on ? vs[i] : 0.f;
      }
      if (FMT != kCacheInt8 && mixed) {
        uint32_t found = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int w = 0; w < NB / 4; ++w) found |= not_finite_bits<DT, FMT>(vp[i].w[w]);
        if (__any(found != 0)) {
          cleaned = true;
#pragma unroll
          for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int w = 0; w < NB / 4; ++w) vp[i].w[w] = finite_only<DT, FMT>(vp[i].w[w]);
        }
      }
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      soften<S::kLift>(soft[rt], x[rt], acc[rt], a);
      if constexpr (FMT != kCacheSame) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[rt][i] *= vs[i];
        if (!full && mixed) {  // 0 times a scale of NaN
#pragma unroll
          for (int i = 0; i < 8; ++i) x[rt][i] = vis[rt] >> i & 1 ? x[rt][i] : 0.f;
        }
      }
    }
    u32x4 pw[RT][S::kProbs];
    if constexpr (!S::kF32) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          uint32_t w[S::kProbs];
          split_probs<DT, FMT, DP>(x[rt][2 * u], x[rt][2 * u + 1], w);
#pragma unroll
          for (int i = 0; i < S::kProbs; ++i) pw[rt][i][u] = w[i];
        }
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      if constexpr (S::kF32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float v = __uint_as_float(vp[i].w[j]);
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
            acc[rt][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, x[rt][i], acc[rt][j], 0, 0, 0);
        }
      } else {
        const u32x4 v = value_operand<S::kProbType, FMT, NB>(vp, j);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int i = 0; i < S::kProbs; ++i) acc[rt][j] = mfma16<S::kProbType>(v, pw[rt][i], acc[rt][j]);
      }
    }
    if constexpr (decltype(more)::value) load_values();
  };
  if (tile0 < tile1) {
    look_up(tile0);
    key_now = key_next;
    place();
    load_keys();
    load_values();
    look_up(tile0 + kStep);
  }
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    soft[rt] = Soft{-kInf, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[rt][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  if (tile0 < tile1) {
    int it = tile0;
    for (; it + kStep < tile1; it += kStep) one_tile(it, std::true_type{});
    one_tile(it, std::false_type{});
  }
  if (FMT != kCacheInt8 && cleaned) {
    // What was taken for zeros and is not finite, to the rows that see it.
    for (int it = tile0; it < tile1; it += kStep) {
      const int key0 = keys.first(it);
      if (keys.all_see(key0)) continue;
      for (int key = key0; key < key0 + 32 && key < len; ++key) {
        const int64_t r = cache_row(a.c, b, key, hk);
        if (r < 0) continue;
        const uint8_t* const vb = a.c.v + r * pitch_b;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < NJ; ++j) {
            const int col = (4 * g + i) * NJ + j;
            const float v = col < a.c.d ? not_finite<DT, FMT>(vb + col * S::kElem) : 0.f;
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
              if (v != 0.f && sees(row[rt], key, base)) acc[rt][j][i] += v;
          }
      }
    }
  }
  float m[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) m[rt] = soft_join(soft[rt]);

  if constexpr (ROWS) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int r = row0 + 16 * rt + n;
      if (r >= rows_all) continue;
      const int t = by_group(a, r), gg = r - t * G;
      if (a.splits > 1) {
        const int64_t to = ((static_cast<int64_t>(b) * a.c.n_heads + hk) * a.splits + split) * rows_all + r;
        float* const po = a.ws + to * (DP + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < NJ; j += 4)
            *reinterpret_cast<f32x4*>(po + (4 * g + i) * NJ + j) =
                f32x4{acc[rt][j][i], acc[rt][j + 1][i], acc[rt][j + 2][i], acc[rt][j + 3][i]};
        if (g == 0) {
          po[DP] = m[rt];
          po[DP + 1] = soft[rt].l;
        }
        continue;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < NJ; j += 4) {
          float o[4] = {acc[rt][j][i], acc[rt][j + 1][i], acc[rt][j + 2][i], acc[rt][j + 3][i]};
          row_finish(s, t, soft[rt].l, o);
          row_out<DT>(a, b, t, hk * G + gg, (4 * g + i) * NJ + j, o);
        }
    }
    return;
  }

  // The waves' results are joined in LDS: first the rows' references and sums, by which every wave scales what it has, then
  // the scaled results, summed in the waves' order.
  float2* const sm = reinterpret_cast<float2*>(sh + WAVES * cap * kPitchO);  // [WAVES][cap]
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = 16 * rt + n;
    if (r < cap && g == 0) sm[wave * cap + r] = float2{m[rt], soft[rt].l};
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
      const float2 y = sm[w * cap + r];
      sum += y.y * (y.x == top ? 1.f : __builtin_amdgcn_exp2f(y.x - top));
      const f32x4 z = *reinterpret_cast<const f32x4*>(sh + (w * cap + r) * kPitchO + i0);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += z[e];
    }
    if (a.splits > 1) {
      const int64_t to = ((static_cast<int64_t>(b) * a.c.n_heads + hk) * a.splits + split) * rows_all + row0 + r;
      float* const po = a.ws + to * (DP + 4);
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

// Many rows (16 bit): a workgroup of four waves takes 128 rows, each wave 32 of them, and all walk the same keys, 64 at a time,
// through LDS. Its threads read whole rows of the cache (a lane's own operand of a key, 16 bytes of each of 16 rows, costs
// the first-level cache an access per lane: 54 of the 66 us of a chunk of 1024 rows that read its operands so),
// 8-bit codes become 16-bit values once for all waves, and the values' operand is a transposed read. Two stages: the next
// one is stored while this one is worked on, and the one behind it is on its way to registers.
template <int DT, int FMT, int DP>
__global__ __launch_bounds__(256, 2) void cached_attn_rows_kernel(AttnArgs a) {
  constexpr int RT = 2, kWaves = 4, kRows = 16 * RT, NJ = DP / 16, kPieces = DP / 32, kHalves = DP / 64;
  using S = Shape<DT, FMT, DP>;
  constexpr int kProbType = S::kProbType, kProbs = S::kProbs;
  constexpr int kKeys = 64, kHalfTile = kKeys * 64, kTile = kHalves * kHalfTile;  // of 16-bit values
  // a thread's share of a stage: kLoads pieces of 16 bytes of keys and as many of values
  constexpr int kElem = FMT == kCacheSame ? 2 : 1, kChunks = DP * kElem / 16, kLoads = kKeys * kChunks / 256;
  static_assert(kLoads >= 1, "a stage gives every thread a piece");
  __shared__ __attribute__((aligned(16))) uint16_t sk[2][kTile], sv[2][kTile];
  __shared__ float s_ks[2][kKeys], s_vs[2][kKeys];
  __shared__ int s_cleaned;
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int id = xcd_logical_id(a.per_xcd);  // the blocks of a sequence's head, which read the same keys, on one XCD
  if (id >= a.n_blocks) return;
  const int rb = id % a.n_rb;
  id /= a.n_rb;
  const int split = id % a.splits;
  id /= a.splits;
  const int hk = id % a.c.n_heads, b = id / a.c.n_heads;
  const Seq s = seq_of(a.c, b);
  const int rows_all = a.c.T * a.G, first_row = rb * kWaves * kRows, row0 = first_row + wave * kRows, G = a.G;
  const int base = s.len - s.n, len = s.len;
  const bool tree = a.tree != nullptr;
  auto rows_keys = [&](int r0, int r1, auto sh) {
    const int t_lo = by_group(a, r0), t_end = by_group(a, r1);
    return keys_of<decltype(sh)::value>(a, s, t_lo, t_end < s.n - 1 ? t_end : s.n - 1);
  };
  // of the workgroup, in stages, and of this wave
  const Keys<6> keys = rows_keys(first_row, first_row + kWaves * kRows - 1, std::integral_constant<int, 6>{});
  const Keys<5> mine = rows_keys(row0, row0 + kRows - 1, std::integral_constant<int, 5>{});
  int tile0 = 0, tile1 = keys.n_tiles;
  if (a.splits > 1) {
    const int per = (keys.n_tiles + a.splits - 1u) / static_cast<unsigned>(a.splits);
    tile0 = per * split < keys.n_tiles ? per * split : keys.n_tiles;
    tile1 = tile0 + per < keys.n_tiles ? tile0 + per : keys.n_tiles;
  }

  // This thread's rows of a stage and its piece of them: threads in a row read a row's pieces one after the other. A
  // wave's rows of each load lie in one group of 16, so in one page: its place is the wave's to work out.
  const int piece = threadIdx.x % kChunks, my_row = threadIdx.x / kChunks;
  constexpr int kRowStep = 256 / kChunks;
  static_assert(kRowStep % 16 == 0 && 64 / kChunks <= 16, "rows of a wave's load lie in one group of 16");
  const int col = piece * (16 / kElem), pitch_b = a.c.pitch * kElem, page_mask = (1 << a.c.page_shift) - 1;
  const int my_off = (my_row & 15) * pitch_b + (col < a.c.pitch ? piece * 16 : 0);
  const bool narrow = a.c.pitch < DP;
  const uint32_t page_rows = static_cast<uint32_t>(a.c.n_heads) << a.c.page_shift, page_bytes = page_rows * pitch_b;
  const uint32_t head_rows = static_cast<uint32_t>(hk) << a.c.page_shift;
  const int32_t* const table = a.c.table + b * a.c.table_stride;
  const uint32_t span = keys.hi >= keys.lo ? keys.hi - keys.lo : 0;
  const int span_lo = keys.hi >= keys.lo ? keys.lo : kNowhere;
  u32x4 rk[kLoads], rv[kLoads];
  float r_ks = 0.f, r_vs = 0.f;
  int page[kLoads], scale_page = 0;
  bool bad[kLoads];  // of what is in registers: a page that is none
  auto group_key = [&](int it, int u) {
    return keys.first(it) + ((wave * (64 / kChunks) + u * kRowStep) & ~15);
  };
  auto look_up = [&](int it) {
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const int key = group_key(it, u);
      page[u] = key < len ? table[key >> a.c.page_shift] : 0;
    }
    if (FMT != kCacheSame && threadIdx.x < kKeys) {
      const int key = keys.first(it) + static_cast<int>(threadIdx.x);
      scale_page = key < len ? table[key >> a.c.page_shift] : -1;
    }
  };
  auto load = [&](int it) {
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      bad[u] = static_cast<uint32_t>(page[u]) >= static_cast<uint32_t>(a.c.n_pages);
      const uint32_t p = bad[u] ? 0 : page[u];  // rows past the end are those of some page: no row sees them
      const int64_t off = static_cast<int64_t>(static_cast<uint64_t>(p) * page_bytes +
                                               (head_rows + (group_key(it, u) & page_mask)) * pitch_b);
      rk[u] = *reinterpret_cast<const u32x4*>(a.c.k + off + my_off);
      rv[u] = *reinterpret_cast<const u32x4*>(a.c.v + off + my_off);
    }
    if (FMT != kCacheSame && threadIdx.x < kKeys) {
      const int key = keys.first(it) + static_cast<int>(threadIdx.x);
      r_ks = r_vs = 0.f;
      if (static_cast<uint32_t>(scale_page) < static_cast<uint32_t>(a.c.n_pages) && key < len) {
        const int64_t r = static_cast<int64_t>(scale_page) * page_rows + head_rows + (key & page_mask);
        r_ks = a.c.ks[r];
        if ((key < keys.np) | in_span(key, span_lo, span)) r_vs = a.c.vs[r];
      } else if (key < len) {
        r_ks = 1.f;  // NaN in the keys
      }
    }
  };
  auto store = [&](int it, int st) {
    const int stage0 = keys.first(it);
    const bool part = !keys.all_see(stage0);
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const int r = my_row + u * kRowStep;
      if (narrow && col >= a.c.pitch) rk[u] = u32x4{0, 0, 0, 0};
      if (part) {
        // values that no row sees may be anything: zeros
        const int key = stage0 + r;
        const uint32_t on = ((key < keys.np) | in_span(key, span_lo, span)) ? ~0u : 0u;
#pragma unroll
        for (int w = 0; w < 4; ++w) rv[u][w] &= on;
        if constexpr (FMT != kCacheInt8) {  // rows that do not see a value must not meet what is not finite: see below
          uint32_t found = 0;
#pragma unroll
          for (int w = 0; w < 4; ++w) found |= not_finite_bits<DT, FMT>(rv[u][w]);
          if (found) {
            s_cleaned = 1;
#pragma unroll
            for (int w = 0; w < 4; ++w) rv[u][w] = finite_only<DT, FMT>(rv[u][w]);
          }
        }
      }
      constexpr uint32_t kNan2 = 0x7fff7fffu;
      if constexpr (FMT == kCacheSame) {
        if (bad[u]) rk[u] = u32x4{kNan2, kNan2, kNan2, kNan2};
        const int to = (piece >> 3) * kHalfTile + swz64(r, piece & 7);
        sts16(&sk[st][to], rk[u]);
        sts16(&sv[st][to], rv[u]);
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // 8 of the piece's 16 values
          u32x4 x, y;
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            x[2 * w] = code2<DT, FMT, false>(rk[u][2 * h + w]);
            x[2 * w + 1] = code2<DT, FMT, true>(rk[u][2 * h + w]);
            y[2 * w] = code2<kProbType, FMT, false>(rv[u][2 * h + w]);
            y[2 * w + 1] = code2<kProbType, FMT, true>(rv[u][2 * h + w]);
          }
          if (bad[u]) x = u32x4{kNan2, kNan2, kNan2, kNan2};
          const int chunk = 2 * piece + h, to = (chunk >> 3) * kHalfTile + swz64(r, chunk & 7);
          sts16(&sk[st][to], x);
          sts16(&sv[st][to], y);
        }
      }
    }
    if (FMT != kCacheSame && threadIdx.x < kKeys) {
      s_ks[st][threadIdx.x] = r_ks;
      s_vs[st][threadIdx.x] = r_vs;
    }
  };

  // the queries of this lane's rows, one of each 16: values 32 c + 8 g .. of piece c
  Row row[RT];
  u32x4 q[RT][kPieces];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = row0 + 16 * rt + n, t = by_group(a, r), gg = r - t * G;
    const bool real = r < rows_all;
    row[rt] = real && keys.n_tiles ? row_of(a, s, b, t) : no_row();
    const uint8_t* const src = a.q + (b * a.qb + (hk * G + gg) * a.qh + t * a.qt) * 2;
#pragma unroll
    for (int c = 0; c < kPieces; ++c) {
      const int i0 = 32 * c + 8 * g;
      u32x4 w{0, 0, 0, 0};
      if (a.q_vec) {
        if (real && i0 < a.c.d) w = *reinterpret_cast<const u32x4*>(src + i0 * 2);
      } else if (real) {
        float x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          float y[1] = {0.f};
          if (i0 + u < a.c.d) row_load<DT, 1>(src + (i0 + u) * 2, y);
          x[u] = y[0] * a.q_sign;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) w[u] = Mfma<DT>::pack2(x[2 * u], x[2 * u + 1]);
      }
      q[rt][c] = w;
      // in registers before the loop: a wait for them inside would be one for the stages on their way
      asm volatile("" : "+v"(q[rt][c]));
    }
  }
  f32x4 acc[RT][NJ];
  Soft soft[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    soft[rt] = Soft{-kInf, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[rt][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  if (threadIdx.x == 0) s_cleaned = 0;
  __syncthreads();
  if (tile0 < tile1) {
    look_up(tile0);
    load(tile0);
    if (tile0 + 1 < tile1) look_up(tile0 + 1);
    store(tile0, 0);
    if (tile0 + 1 < tile1) {
      load(tile0 + 1);
      if (tile0 + 2 < tile1) look_up(tile0 + 2);
    }
    __syncthreads();
  }
  for (int it = tile0; it < tile1; ++it) {
    const int st = (it - tile0) & 1;
    if (it + 1 < tile1) {
      store(it + 1, st ^ 1);
      if (it + 2 < tile1) {
        load(it + 2);
        if (it + 3 < tile1) look_up(it + 3);
      }
    }
    const int stage0 = keys.first(it);
#pragma unroll 1
    for (int sub = 0; sub < kKeys; sub += 32) {
      const int key0 = stage0 + sub;
      if (!mine.any_sees(key0, 31)) continue;
      float x[RT][8];
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        f32x4 sc[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) sc[rt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < kPieces; ++c) {
          const u32x4 key = lds16(&sk[st][(c >> 1) * kHalfTile + swz64(sub + 16 * hf + n, (4 * c + g) & 7)]);
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) sc[rt] = mfma16<DT>(key, q[rt][c], sc[rt]);
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int i = 0; i < 4; ++i) x[rt][4 * hf + i] = sc[rt][i];
      }
      float vs[8];
      if constexpr (FMT != kCacheSame) {
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const f32x4 y = *reinterpret_cast<const f32x4*>(&s_ks[st][sub + 16 * hf + 4 * g]);
          const f32x4 z = *reinterpret_cast<const f32x4*>(&s_vs[st][sub + 16 * hf + 4 * g]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            vs[4 * hf + i] = z[i];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) x[rt][4 * hf + i] *= y[i];
          }
        }
      }
      const bool full = mine.all_see(key0);
      uint32_t vis[RT];
      if (!full) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          vis[rt] = row_sees(row[rt], key0 + 4 * g, base, tree);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (!(vis[rt] >> i & 1)) x[rt][i] = -kInf;
        }
      }
      u32x4 pw[RT][kProbs];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        soften<S::kLift>(soft[rt], x[rt], acc[rt], a);
        if constexpr (FMT != kCacheSame) {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[rt][i] *= vs[i];
          if (!full) {  // 0 times a scale of NaN
#pragma unroll
            for (int i = 0; i < 8; ++i) x[rt][i] = vis[rt] >> i & 1 ? x[rt][i] : 0.f;
          }
        }
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t y[kProbs];
          split_probs<DT, FMT, DP>(x[rt][2 * w], x[rt][2 * w + 1], y);
#pragma unroll
          for (int i = 0; i < kProbs; ++i) pw[rt][i][w] = y[i];
        }
      }
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const u32x4 v = lds_read_tr4x2_swz64(&sv[st][(j >> 2) * kHalfTile], sub + 4 * g, sub + 16 + 4 * g, 16 * (j & 3), lane);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int i = 0; i < kProbs; ++i) acc[rt][j] = mfma16<kProbType>(v, pw[rt][i], acc[rt][j]);
      }
    }
    __syncthreads();
  }
  if (FMT != kCacheInt8 && s_cleaned) {
    // What was taken for zeros and is not finite, to the rows that see it.
    for (int it = tile0; it < tile1; ++it) {
      const int key0 = keys.first(it);
      if (keys.all_see(key0)) continue;
      for (int key = key0; key < key0 + kKeys && key < len; ++key) {
        if (!((key < keys.np) | in_span(key, span_lo, span))) continue;
        const int64_t r = cache_row(a.c, b, key, hk);
        if (r < 0) continue;
        const uint8_t* const vb = a.c.v + r * pitch_b;
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int c = 16 * j + 4 * g + i;
            const float v = c < a.c.d ? not_finite<DT, FMT>(vb + c * kElem) : 0.f;
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
              if (v != 0.f && sees(row[rt], key, base)) acc[rt][j][i] += v;
          }
      }
    }
  }
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const float m = soft_join(soft[rt]);
    const int r = row0 + 16 * rt + n;
    if (r >= rows_all) continue;
    const int t = by_group(a, r), gg = r - t * G;
    const int64_t to = ((static_cast<int64_t>(b) * a.c.n_heads + hk) * a.splits + split) * rows_all + r;
    float* const po = a.ws + to * (DP + 4);
    if (a.splits > 1 && g == 0) {
      po[DP] = m;
      po[DP + 1] = soft[rt].l;
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      float o[4] = {acc[rt][j][0], acc[rt][j][1], acc[rt][j][2], acc[rt][j][3]};
      if (a.splits > 1) {
        *reinterpret_cast<f32x4*>(po + 16 * j + 4 * g) = f32x4{o[0], o[1], o[2], o[3]};
      } else {
        row_finish(s, t, soft[rt].l, o);
        row_out<DT>(a, b, t, hk * G + gg, 16 * j + 4 * g, o);
      }
    }
  }
}

// The parts of a row, joined in their order. Up to kFewParts of them: DP / 4 threads a row, four parts' loads in flight.
constexpr int kFewParts = 8, kMostParts = 64;

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
  float m[kFewParts], l[kFewParts];
  f32x4 x[kFewParts];
#pragma unroll
  for (int w = 0; w < kFewParts; ++w) {
    const int64_t at = w < a.splits ? w * step : 0;
    m[w] = p0[at + DP];
    l[w] = w < a.splits ? p0[at + DP + 1] : 0.f;
    x[w] = *reinterpret_cast<const f32x4*>(p0 + at + i0);
  }
  float top = m[0], sum = 0.f, o[N] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int w = 1; w < kFewParts; ++w) top = fmaxf(top, m[w]);
#pragma unroll
  for (int w = 0; w < kFewParts; ++w) {
    if (w >= a.splits) break;
    const float f = m[w] == top ? 1.f : __builtin_amdgcn_exp2f(m[w] - top);
    sum += l[w] * f;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += x[w][e] * f;
  }
  const int t = by_group(a, r), gg = r - t * a.G;
  row_finish(seq_of(a.c, b), t, sum, o);
  row_out<DT>(a, b, t, hk * a.G + gg, i0, o);
}

// More parts: a workgroup a row. Lane w of each wave holds part w's statistics; every DP / 4 threads sum up each
// 1024 / DP-th part, and those sums meet in LDS.
template <int DT, int DP>
__global__ __launch_bounds__(256) void cached_attn_join_many_kernel(AttnArgs a) {
  constexpr int L = DP / 4, kGroups = 256 / L, kEach = kMostParts / kGroups;
  __shared__ __attribute__((aligned(16))) f32x4 part[kGroups][L];
  __shared__ float factor[kMostParts];
  const int rows_all = a.c.T * a.G, lane = threadIdx.x & 63;
  const int64_t bh = static_cast<int64_t>(blockIdx.x) / rows_all;
  const int r = static_cast<int>(blockIdx.x % rows_all);
  const int b = static_cast<int>(bh / a.c.n_heads), hk = static_cast<int>(bh % a.c.n_heads);
  const float* const p0 = a.ws + (bh * a.splits * rows_all + r) * (DP + 4);
  const int64_t step = static_cast<int64_t>(rows_all) * (DP + 4);
  const int group = threadIdx.x / L, i0 = threadIdx.x % L * 4;
  f32x4 x[kEach];
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int w = group + k * kGroups;
    x[k] = *reinterpret_cast<const f32x4*>(p0 + (w < a.splits ? w * step : 0) + i0);
  }
  const bool have = lane < a.splits;
  const float m = have ? p0[lane * step + DP] : -kInf, l = have ? p0[lane * step + DP + 1] : 0.f;
  const float top = lanes_max(m), f = m == top ? 1.f : __builtin_amdgcn_exp2f(m - top);
  const float sum = lanes_sum(l * f);
  if (threadIdx.x < kMostParts) factor[threadIdx.x] = f;
  __syncthreads();
  f32x4 y{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int w = group + k * kGroups;
    if (w >= a.splits) break;
    const float g = factor[w];
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] += x[k][e] * g;
  }
  part[group][threadIdx.x % L] = y;
  __syncthreads();
  if (group || i0 >= a.c.d) return;
  float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < kGroups; ++k) {
    const f32x4 z = part[k][threadIdx.x];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += z[e];
  }
  const int t = by_group(a, r), gg = r - t * a.G;
  row_finish(seq_of(a.c, b), t, sum, o);
  row_out<DT>(a, b, t, hk * a.G + gg, i0, o);
}

struct Plan {
  int rt, waves, n_rb, splits, row_cap;
  bool rows;
  size_t ws;
};

// How the rows (G·T of each key head and sequence) and the keys are shared out. Times in us, 16-bit unless said.
Plan plan(const CacheArgs& c, int dtype, int B, int rows, int64_t window, int np) {
  Plan p{};
  const bool same = !c.ks;
  const int dp = c.pitch <= 64 ? 64 : 128;
  const int64_t len = static_cast<int64_t>(c.max_pages) << c.page_shift;
  int64_t keys = (window < kNowhere ? window : kNowhere) + c.T + np;
  if (keys > len) keys = len;
  const int64_t tiles = keys / 32 + 2, heads = static_cast<int64_t>(B) * c.n_heads, n16 = heads * ((rows + 15) / 16);
  // Waves with rows of their own, where there are many: 1280 tiles of 16 rows on 162 of keys 68, with the keys shared
  // out 79; 15680 on 10 49 and 76; 1024 on 130 82 and 97; 780 on 36 26.0 and 15.2; 160 on 66 18.9 and 15.5.
  p.rows = rows > 64 && n16 >= 1000;
  // 32 rows a workgroup, 16 where those are few and the keys as well: 640 tiles of rows on 20 of keys 14.4 with 16, 16.2
  // with 32; 320 on 8 7.8 and 9.3; 108 on 29 10.4 and 13.9; 1280 on 20 22.3 and 21.4; 2560 63 and 40; 128 on 130 30 and
  // 24. Wide fp32 rows: 690 on 49 192 and 165.
  p.rt = rows <= 16 || (tiles <= 48 && n16 <= (wide(dtype, same, dp, 1) ? 256 : 704)) ? 1 : 2;
  const int cap = 16 * p.rt;
  int64_t s = 1;
  if (p.rows) {
    p.rt = 2;
    p.waves = 4;
    p.n_rb = (rows + 127) / 128;
    // two workgroups for every CU, each with 8 tiles at least: 160 blocks of 162 tiles 115 whole, 65-68 in three parts
    const int64_t blocks = heads * p.n_rb;
    s = 512 / blocks;
    if (s > tiles / 8) s = tiles / 8;
  } else {
    p.n_rb = (rows + cap - 1) / cap;
    p.row_cap = rows < cap ? rows : cap;
    const int64_t blocks = heads * p.n_rb;
    // Four waves a workgroup instead of eight where the tiles are few, or the workgroups many: eight waves with 32 rows
    // fill a CU's registers alone (320 blocks of 20 tiles 21.1, with four waves 16.3; 20 blocks 10.4 and 10.9); with 16
    // rows 640 blocks of 18 tiles 15.9 and 13.8, 480 13.8 and 13.7, 160 9.1 and 9.8, 640 of 34 36.8 and 37.4.
    p.waves = tiles <= 8 || wide(dtype, same, dp, p.rt) || (blocks > 256 && (p.rt == 2 || tiles <= 24)) ? 4 : 8;
    // Few blocks with long axes in parts, until each CU has a workgroup of four waves (two in 8 bits, whose tiles are
    // half as large). 10 blocks of 512 tiles 87 whole, 14 in 25 parts; 80 of 130 tiles 27.3 and 19.3 in three; 96 of 130
    // with d = 128 55 and 41 in two; 160 33-38 and 36 in three; in 8 bits 40 of 130 22.2 and 11.9 in 12, 160 23.9 and 22.7
    // in three, 240 30 and 34 in two. Shorter axes gain less than the second launch costs the host (10 blocks of 34 tiles
    // 9.5 and 7.9).
    if (tiles > 48) {
      s = same ? 256 / blocks : 512 / blocks >= 3 ? 512 / blocks : 1;
      if (s > tiles / 4) s = tiles / 4;
      if (s > 1) p.waves = 4;
    }
  }
  if (s > kMostParts) s = kMostParts;
  p.splits = s < 1 ? 1 : static_cast<int>(s);
  p.ws = p.splits > 1 ? static_cast<size_t>(heads) * p.splits * rows * (dp + 4) * 4 : 0;
  return p;
}

int check(const tmac_cache* cache, int B, int T, int Hq, int64_t window, int np, CacheArgs& c) {
  const int st = cache_args(cache, B, T, c);
  if (st != TMAC_OK) return st;
  if (Hq <= 0 || Hq > 65535 || Hq % c.n_heads || static_cast<int64_t>(T) * Hq > (1 << 26)) return TMAC_ERR_SHAPE;
  if (static_cast<int64_t>(B) * Hq * T > (1 << 26)) return TMAC_ERR_SHAPE;
  if (window < 0 || np < 0) return TMAC_ERR_VALUE;
  return TMAC_OK;
}

template <int DT, int FMT, int DP>
void launch(const AttnArgs& a, const Plan& p, hipStream_t s) {
  const size_t lds = static_cast<size_t>(p.waves) * p.row_cap * (DP + 4 + 2) * 4;
  const dim3 grid(a.B, a.c.n_heads, p.n_rb * p.splits);
  if (p.rows) {
    if constexpr (DT == TMAC_F32)
      cached_attn_kernel<DT, FMT, DP, 2, 4, true><<<8 * a.per_xcd, 256, 0, s>>>(a);
    else
      cached_attn_rows_kernel<DT, FMT, DP><<<8 * a.per_xcd, 256, 0, s>>>(a);
  } else if (p.rt == 2) {
    if constexpr (!wide(DT, FMT == kCacheSame, DP, 2)) {
      if (p.waves == 8) cached_attn_kernel<DT, FMT, DP, 2, 8, false><<<grid, 64 * 8, lds, s>>>(a);
    }
    if (p.waves == 4) cached_attn_kernel<DT, FMT, DP, 2, 4, false><<<grid, 64 * 4, lds, s>>>(a);
  } else if (p.waves == 4) {
    cached_attn_kernel<DT, FMT, DP, 1, 4, false><<<grid, 64 * 4, lds, s>>>(a);
  } else if constexpr (!wide(DT, FMT == kCacheSame, DP, 1)) {
    cached_attn_kernel<DT, FMT, DP, 1, 8, false><<<grid, 64 * 8, lds, s>>>(a);
  }
  const int64_t rows = static_cast<int64_t>(a.B) * a.c.n_heads * a.c.T * a.G;
  if (p.splits > kFewParts)  // at most 512 blocks of up to 128 rows are parted, so these are few
    cached_attn_join_many_kernel<DT, DP><<<static_cast<unsigned>(rows), 256, 0, s>>>(a);
  else if (p.splits > 1)
    cached_attn_join_kernel<DT, DP><<<static_cast<unsigned>((rows * (DP / 4) + 255) / 256), 256, 0, s>>>(a);
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
  const int64_t blocks = static_cast<int64_t>(B) * a.c.n_heads * p.n_rb * p.splits;  // below 2^27 by check()
  const int n = cache->dtype == TMAC_F32 ? 4 : 8;
  a.q = static_cast<const uint8_t*>(d_q);
  a.qb = h_q_strides[0], a.qh = h_q_strides[1], a.qt = h_q_strides[2];
  a.tree = d_tree, a.tree_stride = tree_stride;
  a.out = static_cast<uint8_t*>(d_out);
  a.ws = static_cast<float*>(d_ws);
  a.B = B, a.Hq = n_q_heads, a.G = G, a.g_shift = G & (G - 1) ? -1 : __builtin_ctz(G), a.n_rb = p.n_rb;
  a.splits = p.splits, a.row_cap = p.row_cap, a.n_blocks = static_cast<int>(blocks), a.per_xcd = (a.n_blocks + 7) / 8;
  a.np = n_persistent < kNowhere ? n_persistent : kNowhere;
  a.window = window < kNowhere ? static_cast<int>(window) : kNowhere;
  a.scale2 = scale == 0.f ? 1.f : fabsf(scale) * kLog2e;
  a.slack = kSlack / a.scale2;
  a.q_sign = scale > 0.f ? 1.f : scale < 0.f ? -1.f : scale;
  a.q_vec = a.q_sign == 1.f && row_aligned16(d_q) && a.c.d % n == 0 && a.qb % n == 0 && a.qh % n == 0 && a.qt % n == 0;
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
