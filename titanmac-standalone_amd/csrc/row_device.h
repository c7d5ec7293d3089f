// Rows of values in global memory, shared by the kernels that stream them: N values at once as one
// 16-byte access (N = kRowVec<DT>) or a single value (N = 1, rows that are not 16-byte aligned),
// converted to and from fp32; and the running statistics of a row's softmax.
#pragma once

#include "tmac_device.h"

namespace tmac {

template <int DT>
constexpr int kRowVec = DT == TMAC_F32 ? 4 : 8;
template <int DT>
constexpr int kRowSize = DT == TMAC_F32 ? 4 : 2;

template <int DT, int N>
__device__ __forceinline__ void row_load(const void* __restrict__ p, float (&v)[N]) {
  if constexpr (N == 1) {
    if constexpr (DT == TMAC_F32)
      v[0] = *static_cast<const float*>(p);
    else
      v[0] = Mfma<DT>::to_f32(*static_cast<const uint16_t*>(p));
  } else if constexpr (DT == TMAC_F32) {
    static_assert(N == 4, "one 16-byte access");
    const f32x4 x = *static_cast<const f32x4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = x[i];
  } else {
    static_assert(N == 8, "one 16-byte access");
    const u32x4 x = *static_cast<const u32x4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = Mfma<DT>::to_f32(static_cast<uint16_t>(x[i] & 0xffff));
      v[2 * i + 1] = Mfma<DT>::to_f32(static_cast<uint16_t>(x[i] >> 16));
    }
  }
}

template <int DT, int N>
__device__ __forceinline__ void row_store(void* __restrict__ p, const float (&v)[N]) {
  if constexpr (N == 1) {
    if constexpr (DT == TMAC_F32)
      *static_cast<float*>(p) = v[0];
    else
      *static_cast<uint16_t*>(p) = Mfma<DT>::from_f32(v[0]);
  } else if constexpr (DT == TMAC_F32) {
    *static_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
  } else {
    u32x4 x;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = Mfma<DT>::pack2(v[2 * i], v[2 * i + 1]);
    *static_cast<u32x4*>(p) = x;
  }
}

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kFar = -1e4f;  // differences are cut here in products with an exponential that is then 0

__device__ __forceinline__ float exp_d(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }

// Running softmax statistics: m the maximum, s = Σ e^{z − m}, h = Σ e^{z − m} (z − m). mu is m, or 0 while nothing
// above −inf was seen (so that −inf − mu is −inf and not NaN); a NaN, or +inf (whose z − mu is NaN), makes s NaN.
struct Stat {
  float m, mu, s, h;
};
__device__ __forceinline__ Stat stat_none() { return Stat{-__builtin_inff(), 0.f, 0.f, 0.f}; }

__device__ __forceinline__ void stat_raise(Stat& a, float m) {
  if (m > a.m) {
    const float d = fmaxf(a.m - m, kFar), f = exp_d(d);  // f = 0 for the first m
    a.h = f * fmaf(a.s, d, a.h);
    a.s *= f;
    a.m = a.mu = m;
  }
}
template <bool ENT>
__device__ __forceinline__ void stat_add(Stat& a, float z) {
  const float d = z - a.mu, e = exp_d(d);
  a.s += e;
  if (ENT) a.h = fmaf(e, fmaxf(d, kFar), a.h);
}
// The value of lane (lane ^ J), on the vector ALU: quad permutes and mirrors of 8 and 16 lanes, whose
// compositions are the exchanges by 4 and 8, and the swaps of rows and halves, which return a lane's
// own value and the other's in an order that depends on the lane.
template <int CTRL>
__device__ __forceinline__ uint32_t lane_dpp(uint32_t x) {
  return __builtin_amdgcn_update_dpp(0u, x, CTRL, 0xf, 0xf, true);
}
template <int J>
__device__ __forceinline__ uint32_t lane_xor(uint32_t x) {
  constexpr int kMirror = 0x140, kHalfMirror = 0x141, kReverse4 = 0x1b;
  if constexpr (J == 1) {
    return lane_dpp<0xb1>(x);  // 1, 0, 3, 2
  } else if constexpr (J == 2) {
    return lane_dpp<0x4e>(x);  // 2, 3, 0, 1
  } else if constexpr (J == 4) {
    return lane_dpp<kReverse4>(lane_dpp<kHalfMirror>(x));
  } else if constexpr (J == 8) {
    return lane_dpp<kHalfMirror>(lane_dpp<kMirror>(x));
  } else if constexpr (J == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return r[0] ^ r[1] ^ x;
  } else {
    static_assert(J == 32, "a power of two below 64");
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return r[0] ^ r[1] ^ x;
  }
}
template <int J>
__device__ __forceinline__ float lane_xor(float x) {
  return __uint_as_float(lane_xor<J>(__float_as_uint(x)));
}
template <int J>
__device__ __forceinline__ uint64_t lane_xor(uint64_t x) {
  return static_cast<uint64_t>(lane_xor<J>(static_cast<uint32_t>(x >> 32))) << 32 |
         lane_xor<J>(static_cast<uint32_t>(x));
}
__device__ __forceinline__ float lanes_max(float x) {
  x = fmaxf(x, lane_xor<1>(x));
  x = fmaxf(x, lane_xor<2>(x));
  x = fmaxf(x, lane_xor<4>(x));
  x = fmaxf(x, lane_xor<8>(x));
  x = fmaxf(x, lane_xor<16>(x));
  return fmaxf(x, lane_xor<32>(x));
}
__device__ __forceinline__ float lanes_sum(float x) {
  x += lane_xor<1>(x);
  x += lane_xor<2>(x);
  x += lane_xor<4>(x);
  x += lane_xor<8>(x);
  x += lane_xor<16>(x);
  return x + lane_xor<32>(x);
}

// a's sums moved to the maximum m >= a.m; where a has no term above −inf they are 0 (or NaN)
__device__ __forceinline__ void stat_rescale(Stat& a, float m) {
  const float d = a.m == -__builtin_inff() ? 0.f : fmaxf(a.m - m, kFar), f = exp_d(d);
  a.h = f * fmaf(a.s, d, a.h);
  a.s *= f;
  a.m = m;
  a.mu = m == -__builtin_inff() ? 0.f : m;
}
__device__ __forceinline__ void stat_join(Stat& a, const Stat& b) {
  stat_raise(a, b.m);
  // b's terms at a's maximum; where b has none above −inf it has s = h = 0 (or NaN)
  const float d = b.m == -__builtin_inff() ? 0.f : fmaxf(b.m - a.mu, kFar), f = exp_d(d);
  a.h = fmaf(f, fmaf(b.s, d, b.h), a.h);
  a.s = fmaf(f, b.s, a.s);
}
// the statistics of all 64 lanes, in every lane
__device__ __forceinline__ void stat_wave(Stat& a) {
  stat_rescale(a, lanes_max(a.m));
  a.s = lanes_sum(a.s);
  a.h = lanes_sum(a.h);
}
// and of the workgroup's waves, in every thread; sh: one entry per wave, read when this returns
template <int WAVES>
__device__ __forceinline__ void stat_block(Stat& a, Stat* sh) {
  stat_wave(a);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = a;
  __syncthreads();
  float m = sh[0].m;
#pragma unroll
  for (int w = 1; w < WAVES; ++w) m = fmaxf(m, sh[w].m);
  a = Stat{m, m == -__builtin_inff() ? 0.f : m, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    Stat b = sh[w];
    stat_rescale(b, m);
    a.s += b.s;
    a.h += b.h;
  }
}

inline bool row_aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace tmac
