// The key/value cache's rows: written from the new tokens' keys and values, read back, moved.
//
// A row (page, head, place) is d values. A group of `lanes` lanes (a power of two) holds one row, each a chunk of
// kRowVec values: one 16-byte access in the model's type. All three kernels move bytes once and are bound by
// memory or, for a decoded token, by their launch.

#include "cache_device.h"

namespace {
using namespace tmac;

// x[0..N) = the row's values from chunk i on, zeros behind d
template <int DT, bool VEC, int N>
__device__ __forceinline__ void load_chunk(const uint8_t* row, int i, int d, float (&x)[N]) {
  if (VEC) {
    if (i < d) {
      row_load<DT, N>(row + static_cast<int64_t>(i) * kRowSize<DT>, x);
      return;
    }
  } else {
#pragma unroll
    for (int u = 0; u < N; ++u) {
      float one[1] = {0.f};
      if (i + u < d) row_load<DT, 1>(row + static_cast<int64_t>(i + u) * kRowSize<DT>, one);
      x[u] = one[0];
    }
    return;
  }
#pragma unroll
  for (int u = 0; u < N; ++u) x[u] = 0.f;
}

struct Strides {
  int64_t b, h, t;
};

// a chunk of a row into a pool, from chunk i on; all 64 lanes take part
template <int DT, int FMT, int N>
__device__ __forceinline__ void put_chunk(uint8_t* pool, float* scales, int64_t row, int pitch, int i, int lanes_log2,
                                          const float (&x)[N]) {
  const bool mine = row >= 0 && i < pitch;
  if constexpr (FMT == kCacheSame) {
    if (mine) row_store<DT, N>(pool + (row * pitch + i) * kRowSize<DT>, x);
  } else {
    uint32_t m = 0;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const uint32_t w = __float_as_uint(x[u]) & 0x7fffffffu;
      m = w > m ? w : m;
    }
    for (int o = 1; o < 1 << lanes_log2; o <<= 1) {
      const uint32_t w = __shfl_xor(m, o);
      m = w > m ? w : m;
    }
    const float scale = code_scale<FMT>(m);
    if (!mine) return;
    uint8_t* const to = pool + row * pitch + i;
    if constexpr (N == 4) {
      *reinterpret_cast<uint32_t*>(to) = to_code4<FMT>(x[0], x[1], x[2], x[3], scale);
    } else {
      *reinterpret_cast<u32x2*>(to) = u32x2{to_code4<FMT>(x[0], x[1], x[2], x[3], scale),
                                            to_code4<FMT>(x[4], x[5], x[6], x[7], scale)};
    }
    if (i == 0) scales[row] = scale;
  }
}

// lanes_log2: log2 of the lanes of a row. grid.x: rows (t, h) of a sequence, grid.y: sequences. A row's key and value by
// the same lanes: one look at the table, two loads in flight (8 prompts of 2047 rows of 10 heads
// of 64 bf16 18.2 us, 4.6 TB/s; with a row's key and value apart 21.4). The order of the rows makes no difference.
template <int DT, int FMT, bool VEC>
__global__ __launch_bounds__(256) void cache_write_kernel(CacheArgs a, const uint8_t* __restrict__ k, Strides ks,
                                                          const uint8_t* __restrict__ v, Strides vs, int B,
                                                          int lanes_log2) {
  constexpr int N = kRowVec<DT>;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const uint32_t r = static_cast<uint32_t>(at >> lanes_log2);
  const int i = static_cast<int>(at & ((1 << lanes_log2) - 1)) * N;
  // heads fastest: the heads of a token lie together in a projection's output
  const int t = static_cast<int>(r / static_cast<uint32_t>(a.n_heads)), h = static_cast<int>(r - t * a.n_heads);
  for (int b = blockIdx.y; b < B; b += gridDim.y) {
    const Seq s = seq_of(a, b);
    int64_t row = -1;
    float x[N], y[N];
#pragma unroll
    for (int u = 0; u < N; ++u) x[u] = y[u] = 0.f;
    if (s.ok && t < s.n) {
      load_chunk<DT, VEC, N>(k + (b * ks.b + h * ks.h + t * ks.t) * kRowSize<DT>, i, a.d, x);
      load_chunk<DT, VEC, N>(v + (b * vs.b + h * vs.h + t * vs.t) * kRowSize<DT>, i, a.d, y);
      row = cache_row(a, b, s.len - s.n + t, h);
    }
    put_chunk<DT, FMT, N>(a.k, a.ks, row, a.pitch, i, lanes_log2, x);
    put_chunk<DT, FMT, N>(a.v, a.vs, row, a.pitch, i, lanes_log2, y);
  }
}

// N values of a pool's row from chunk i on, as fp32
template <int DT, int FMT, int N>
__device__ __forceinline__ void pool_load(const uint8_t* pool, const float* scales, int64_t row, int pitch, int i,
                                          float (&x)[N]) {
  if constexpr (FMT == kCacheSame) {
    row_load<DT, N>(pool + (row * pitch + i) * kRowSize<DT>, x);
  } else {
    const float s = scales[row];
#pragma unroll
    for (int u = 0; u < N; u += 4) {
      const f32x4 c = code4<FMT>(*reinterpret_cast<const uint32_t*>(pool + row * pitch + i + u));
#pragma unroll
      for (int j = 0; j < 4; ++j) x[u + j] = c[j] * s;
    }
  }
}

// Rows (h, t), t fastest: those of a page are together on both sides. Key and value by the same lanes.
template <int DT, int FMT, bool VEC>
__global__ __launch_bounds__(256) void cache_read_kernel(CacheArgs a, uint8_t* __restrict__ k, uint8_t* __restrict__ v,
                                                         int B, int T, int lanes_log2) {
  constexpr int N = kRowVec<DT>;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const uint32_t r = static_cast<uint32_t>(at >> lanes_log2);
  const int i = static_cast<int>(at & ((1 << lanes_log2) - 1)) * N;
  const int h = static_cast<int>(r / static_cast<uint32_t>(T)), t = static_cast<int>(r - h * static_cast<uint32_t>(T));
  if (h >= a.n_heads || i >= a.d) return;
  for (int b = blockIdx.y; b < B; b += gridDim.y) {
    const int len = a.lengths[b];
    const bool ok = len >= 0 && len <= (static_cast<int64_t>(a.max_pages) << a.page_shift);
    float x[N], y[N];
    const int64_t row = ok && t < len ? cache_row(a, b, t, h) : -1;
    if (row >= 0) {
      pool_load<DT, FMT, N>(a.k, a.ks, row, a.pitch, i, x);
      pool_load<DT, FMT, N>(a.v, a.vs, row, a.pitch, i, y);
    } else {
      const float fill = ok && t >= len ? 0.f : __builtin_nanf("");
#pragma unroll
      for (int u = 0; u < N; ++u) x[u] = y[u] = fill;
    }
    const int64_t to = (((static_cast<int64_t>(b) * a.n_heads + h) * T + t) * a.d + i) * kRowSize<DT>;
    if (VEC) {
      row_store<DT, N>(k + to, x);
      row_store<DT, N>(v + to, y);
    } else {
#pragma unroll
      for (int u = 0; u < N; ++u) {
        if (i + u >= a.d) continue;
        const float one[1] = {x[u]}, two[1] = {y[u]};
        row_store<DT, 1>(k + to + u * kRowSize<DT>, one);
        row_store<DT, 1>(v + to + u * kRowSize<DT>, two);
      }
    }
  }
}

// One workgroup moves the rows of one sequence, head and pool: up to 64 rows of up to 512 bytes, all loaded before the
// first is stored, so places may be read and written in any order.
__global__ __launch_bounds__(256) void cache_keep_kernel(CacheArgs a, const int32_t* __restrict__ path,
                                                         int64_t path_stride, int A, int bytes_log2, int row_bytes) {
  const int h = blockIdx.x, y = blockIdx.y, b = y >> 1;
  const bool is_v = y & 1;
  const Seq s = seq_of(a, b);
  if (!s.ok || s.n == 0) return;
  uint8_t* const pool = is_v ? a.v : a.k;
  float* const scales = is_v ? a.vs : a.ks;
  const int base = s.len - s.n;
  // thread: 16-byte chunk c of rows r0, r0 + 256 / chunks, ...
  const int chunks_log2 = bytes_log2 - 4, c = threadIdx.x & ((1 << chunks_log2) - 1), r0 = threadIdx.x >> chunks_log2;
  const int step = 256 >> chunks_log2;
  u32x4 x[8];
  float sc[8];
  int64_t to[8];
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const int r = r0 + u * step;
    to[u] = -1;
    if (r >= A || r >= s.n || c * 16 >= row_bytes) continue;
    const int from = path[b * path_stride + r];
    if (from < 0 || from >= s.n || from == r) continue;
    const int64_t src = cache_row(a, b, base + from, h);
    to[u] = cache_row(a, b, base + r, h);
    if (src < 0) to[u] = -1;
    if (to[u] < 0) continue;
    x[u] = *reinterpret_cast<const u32x4*>(pool + src * row_bytes + c * 16);
    if (scales && c == 0) sc[u] = scales[src];
  }
  __syncthreads();  // waits for the loads too
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    if (to[u] < 0) continue;
    *reinterpret_cast<u32x4*>(pool + to[u] * row_bytes + c * 16) = x[u];
    if (scales && c == 0) scales[to[u]] = sc[u];
  }
}

int log2_up(int n) {
  int l = 0;
  while ((1 << l) < n) ++l;
  return l;
}

Strides strides_of(const int64_t* s) { return Strides{s[0], s[1], s[2]}; }

// whether every row starts at a 16-byte boundary and is a whole number of 16-byte accesses
bool rows_align16(const void* p, const int64_t* s, int d, int dtype) {
  const int n = dtype == TMAC_F32 ? 4 : 8;
  return row_aligned16(p) && d % n == 0 && (!s || (s[0] % n == 0 && s[1] % n == 0 && s[2] % n == 0));
}

template <class F>
void by_types(int dtype, int format, bool vec, F f) {
  auto by_vec = [&](auto dt, auto fmt) {
    if (vec)
      f(dt, fmt, std::true_type{});
    else
      f(dt, fmt, std::false_type{});
  };
  auto by_format = [&](auto dt) {
    if (format == TMAC_CACHE_SAME)
      by_vec(dt, std::integral_constant<int, kCacheSame>{});
    else if (format == TMAC_CACHE_INT8)
      by_vec(dt, std::integral_constant<int, kCacheInt8>{});
    else
      by_vec(dt, std::integral_constant<int, kCacheE4m3>{});
  };
  if (dtype == TMAC_F32)
    by_format(std::integral_constant<int, TMAC_F32>{});
  else if (dtype == TMAC_BF16)
    by_format(std::integral_constant<int, TMAC_BF16>{});
  else
    by_format(std::integral_constant<int, TMAC_F16>{});
}

constexpr int kMaxGridY = 65535;
int grid_y(int B) { return B < kMaxGridY ? B : kMaxGridY; }

}  // namespace

extern "C" int tmac_cache_write(const tmac_cache* cache, const void* d_new_k, const int64_t* h_k_strides,
                                const void* d_new_v, const int64_t* h_v_strides, int B, int T, void* stream) {
  CacheArgs a;
  const int st = cache_args(cache, B, T, a);
  if (st != TMAC_OK) return st;
  if (B == 0 || T == 0) return TMAC_OK;
  if (!d_new_k || !d_new_v || !h_k_strides || !h_v_strides) return TMAC_ERR_NULL;
  const bool vec = rows_align16(d_new_k, h_k_strides, a.d, cache->dtype) &&
                   rows_align16(d_new_v, h_v_strides, a.d, cache->dtype);
  const int l2 = log2_up((a.pitch + (cache->dtype == TMAC_F32 ? 3 : 7)) / (cache->dtype == TMAC_F32 ? 4 : 8));
  const int64_t threads = (static_cast<int64_t>(T) * a.n_heads) << l2;
  const dim3 grid(static_cast<unsigned>((threads + 255) / 256), grid_y(B));
  by_types(cache->dtype, cache->format, vec, [&](auto dt, auto fmt, auto w) {
    cache_write_kernel<decltype(dt)::value, decltype(fmt)::value, decltype(w)::value>
        <<<grid, 256, 0, static_cast<hipStream_t>(stream)>>>(
            a, static_cast<const uint8_t*>(d_new_k), strides_of(h_k_strides), static_cast<const uint8_t*>(d_new_v),
            strides_of(h_v_strides), B, l2);
  });
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? TMAC_OK : static_cast<int>(err);
}

extern "C" int tmac_cache_read(const tmac_cache* cache, void* d_out_k, void* d_out_v, int B, int T, void* stream) {
  CacheArgs a;
  const int st = cache_args(cache, B, T, a);
  if (st != TMAC_OK) return st;
  if (B == 0 || T == 0) return TMAC_OK;
  if (!d_out_k || !d_out_v) return TMAC_ERR_NULL;
  const bool vec = rows_align16(d_out_k, nullptr, a.d, cache->dtype) && rows_align16(d_out_v, nullptr, a.d, cache->dtype);
  const int l2 = log2_up((a.d + (cache->dtype == TMAC_F32 ? 3 : 7)) / (cache->dtype == TMAC_F32 ? 4 : 8));
  const int64_t threads = (static_cast<int64_t>(T) * a.n_heads) << l2;
  const dim3 grid(static_cast<unsigned>((threads + 255) / 256), grid_y(B));
  by_types(cache->dtype, cache->format, vec, [&](auto dt, auto fmt, auto w) {
    cache_read_kernel<decltype(dt)::value, decltype(fmt)::value, decltype(w)::value>
        <<<grid, 256, 0, static_cast<hipStream_t>(stream)>>>(a, static_cast<uint8_t*>(d_out_k),
                                                             static_cast<uint8_t*>(d_out_v), B, T, l2);
  });
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? TMAC_OK : static_cast<int>(err);
}

extern "C" int tmac_cache_keep(const tmac_cache* cache, const int32_t* d_path, int64_t path_stride, int A, int B, int T,
                               void* stream) {
  CacheArgs a;
  const int st = cache_args(cache, B, T, a);
  if (st != TMAC_OK) return st;
  if (T > TMAC_CACHE_MAX_TREE || A < 0 || A > T || path_stride < 0 || (B > 1 && path_stride < A)) return TMAC_ERR_SHAPE;
  if (B == 0 || A == 0) return TMAC_OK;
  if (!d_path) return TMAC_ERR_NULL;
  if (B > kMaxGridY / 2) return TMAC_ERR_SHAPE;
  const int row_bytes = a.pitch * (cache->format != TMAC_CACHE_SAME ? 1 : cache->dtype == TMAC_F32 ? 4 : 2);
  cache_keep_kernel<<<dim3(a.n_heads, 2 * B), 256, 0, static_cast<hipStream_t>(stream)>>>(
      a, d_path, path_stride, A, log2_up(row_bytes), row_bytes);
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? TMAC_OK : static_cast<int>(err);
}
