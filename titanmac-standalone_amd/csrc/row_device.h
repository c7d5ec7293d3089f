// Rows of values in global memory, shared by the kernels that stream them: N values at once as one
// 16-byte access (N = kRowVec<DT>) or a single value (N = 1, rows that are not 16-byte aligned),
// converted to and from fp32.
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

inline bool row_aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace tmac
