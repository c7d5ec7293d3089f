// Log probabilities of given tokens under stored logits, with entropy and top alternatives, and the
// gradient of the logits, for gfx950.
//
//   lp = z_t − lse(z),   H = −Σ_j p_j ln p_j,   the k largest p_j (ties to the lower index)
//   dz_j = g_lp (δ_jt − p_j) − g_H p_j (ln p_j + H)
//
// (models/titanmac.py:666-680: F.cross_entropy of the shifted logits, whose row terms are −lp.) Rows are
// a vocabulary long, so everything is bound by reading them: one pass forward, one read and one write
// backward.
//
// Forward: each thread keeps a running maximum m, s = Σ e^{z − m} and h = Σ e^{z − m} (z − m) over its
// 16-byte groups (the workgroup's threads interleaved), rescaled when m grows; H = ln s − h / s, in which
// nothing cancels. Rows whose base is not 16-byte aligned begin with a partial group. Few rows are split
// over the vocabulary and a second kernel joins the parts.
//
// Alternatives, without a second pass over the row: beside m each thread keeps the group where it first
// saw it. Order the threads by (m, earlier group): the k best values lie with the first k threads, since
// any other thread's best, and so all it has, comes after k threads' bests. Their groups, k of 1024th of
// the row, are read again, and those not below the k-th thread's best are sorted: at most a few dozen
// for ordinary rows, any number of them in rounds that keep the best 64.
//
// m and s are kept for the backward, p = e^{z − m} / s: through lse the rounding of a sum near 12 would
// go into every p.

#include "row_device.h"

using namespace tmac;

namespace {

constexpr int kMaxTop = 64;
constexpr int kUnroll = 4;

// (value, index) as one whole number: larger value first, then lower index; 0 is no entry.
__device__ __forceinline__ uint64_t top_key(float z, int idx) {
  const uint32_t b = __float_as_uint(z + 0.f);  // −0 counts as 0
  const uint32_t o = b & 0x80000000u ? ~b : b | 0x80000000u;
  return static_cast<uint64_t>(o) << 32 | static_cast<uint32_t>(~idx);
}
__device__ __forceinline__ int key_index(uint64_t k) { return static_cast<int>(~static_cast<uint32_t>(k)); }
__device__ __forceinline__ float key_value(uint64_t k) {
  const uint32_t o = static_cast<uint32_t>(k >> 32);
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int x) {
  const uint32_t lo = __shfl_xor(static_cast<uint32_t>(v), x);
  const uint32_t hi = __shfl_xor(static_cast<uint32_t>(v >> 32), x);
  return static_cast<uint64_t>(hi) << 32 | lo;
}
// lanes i and i ^ j exchange so that the larger value is at the lower lane (desc) or the higher
__device__ __forceinline__ uint64_t exchange(uint64_t v, int lane, int j, bool desc) {
  const uint64_t o = shfl_xor64(v, j);
  const bool low = (lane & j) == 0;
  return (v > o) == (low == desc) ? v : o;
}
// bitonic sort of a wave's 64 keys, descending
__device__ __forceinline__ uint64_t wave_sort(uint64_t v, int lane) {
#pragma unroll
  for (int k = 2; k <= 64; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) v = exchange(v, lane, j, (lane & k) == 0);
  return v;
}
// the 64 largest of two descending lists, descending; b is given reversed
__device__ __forceinline__ uint64_t wave_merge(uint64_t a, uint64_t b_rev, int lane) {
  uint64_t v = a > b_rev ? a : b_rev;
#pragma unroll
  for (int j = 32; j > 0; j >>= 1) v = exchange(v, lane, j, true);
  return v;
}

// buf[0 .. n) -> its 64 largest in buf[0 .. 64), descending, 0 where there are fewer; n <= NT, by all of
// the workgroup's NT threads.
template <int NT>
__device__ void block_top(uint64_t* buf, int n) {
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  uint64_t v = tid < n ? buf[tid] : 0;
  const int waves = (n + 63) / 64;
  if (wave < waves) v = wave_sort(v, lane);
  for (int half = 1; half < waves; half *= 2) {
    __syncthreads();
    buf[tid] = v;
    __syncthreads();
    if (wave % (2 * half) == 0 && wave + half < waves) v = wave_merge(v, buf[64 * (wave + half) + 63 - lane], lane);
  }
  __syncthreads();
  if (wave == 0) buf[lane] = v;
  __syncthreads();
}

// A row of V values seen as groups of N that are 16-byte aligned: group q holds elements q N − o ..
// q N − o + N − 1, the first and the last possibly in part.
struct Groups {
  int o, n;        // offset, number of groups
  int full0, full1;  // groups [full0, full1) are whole
};
template <int DT>
__device__ __forceinline__ Groups row_groups(const uint8_t* row, int V) {
  constexpr int N = kRowVec<DT>, E = kRowSize<DT>;
  Groups g;
  g.o = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / E);
  g.n = static_cast<int>((static_cast<int64_t>(V) + g.o + N - 1) / N);
  g.full0 = g.o > 0;
  g.full1 = static_cast<int>((static_cast<int64_t>(V) + g.o) / N);
  return g;
}

constexpr int kTopBuf = 64;  // entries kept between rounds

template <int NT>
struct TopShared {
  uint64_t buf[NT + kTopBuf];
  int count;
};

// The workgroup's k best entries of its groups [q0, q1) of a row, into buf[0 .. k), given each thread's best
// value `m` and the group `arg` of its first one (arg < 0: the thread saw none).
template <int DT, int NT>
__device__ void block_row_top(TopShared<NT>& sh, const uint8_t* row, int V, const Groups& g, int q0, int q1, int k,
                              float m, int arg) {
  constexpr int N = kRowVec<DT>, E = kRowSize<DT>;
  const int tid = threadIdx.x;
  // thread bests by their group's number; unique, since groups are
  sh.buf[tid] = arg >= 0 ? top_key(m, arg) : 0;
  __syncthreads();
  block_top<NT>(sh.buf, NT);
  // the group of the k-th thread's best, or of the last if there are fewer threads with entries
  uint64_t kth = sh.buf[k - 1];
  int n_thr = k;
  if (!kth) {
    n_thr = 0;
    while (sh.buf[n_thr]) ++n_thr;
  }
  // an entry of the k best is not below the k-th best's value, nor, at that value, behind its group
  const uint64_t floor_key = kth ? (kth & ~0xffffffffull) |
                                       static_cast<uint32_t>(~((key_index(kth) + 1) * N - 1 - g.o))
                                 : 1;
  __shared__ int s_thr[kMaxTop];
  if (tid < n_thr) s_thr[tid] = (key_index(sh.buf[tid]) - q0) % NT;
  if (tid == 0) sh.count = 0;
  __syncthreads();
  const int per = (q1 - q0 + NT - 1) / NT;  // groups a thread has, at most
  int n = 0;                                // entries in buf, the same in every thread
  for (int64_t i0 = 0; i0 < static_cast<int64_t>(n_thr) * per; i0 += NT) {
    const int64_t i = i0 + tid;
    uint64_t key[N];
    int mine = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) key[e] = 0;
    if (i < static_cast<int64_t>(n_thr) * per) {
      const int64_t q = q0 + s_thr[i / per] + static_cast<int64_t>(i % per) * NT;
      if (q < q1) {
        const int first = static_cast<int>(q * N - g.o);
        for (int e = 0; e < N; ++e) {
          const int idx = first + e;
          if (idx < 0 || idx >= V) continue;
          float z[1];
          row_load<DT, 1>(row + static_cast<int64_t>(idx) * E, z);
          const uint64_t kk = top_key(z[0], idx);
          if (kk >= floor_key) {
            key[e] = kk;
            ++mine;
          }
        }
      }
    }
    if (mine) atomicAdd(&sh.count, mine);
    __syncthreads();
    const int total = sh.count;
    __syncthreads();
    if (n + total <= NT) {
      if (tid == 0) sh.count = n;
      __syncthreads();
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (key[e]) sh.buf[atomicAdd(&sh.count, 1)] = key[e];
      n += total;
      __syncthreads();
      if (tid == 0) sh.count = 0;
      __syncthreads();
      continue;
    }
    // too many at once: half of the threads' e-th values at a time beside the best 64 so far
    for (int e = 0; e < N; ++e) {
      for (int half = 0; half < 2; ++half) {
        if (n > 64) {
          block_top<NT>(sh.buf, n);
          n = 64;
        }
        if (tid == 0) sh.count = n;
        __syncthreads();
        uint64_t kk = 0;
#pragma unroll
        for (int u = 0; u < N; ++u)
          if (u == e) kk = key[u];
        if (kk && (tid & 1) == half) sh.buf[atomicAdd(&sh.count, 1)] = kk;
        __syncthreads();
        n = sh.count;
        __syncthreads();
      }
    }
    if (tid == 0) sh.count = 0;
    __syncthreads();
  }
  block_top<NT>(sh.buf, n);
}

struct Row2 {
  int64_t sb, st;  // strides of [B, T, V] rows, elements
  int T;
};
__device__ __forceinline__ int64_t row_offset(const Row2& r, int row) {
  const int b = row / r.T;
  return b * r.sb + (row - b * r.T) * r.st;
}

struct Out {
  float* lp;
  float* ent;        // nullable
  int64_t* top_ids;  // nullable, [rows, k]
  float* top_lp;
  float* stats;      // [rows, 2]: m (0 for a row of −inf), s
};

// What a row's outputs are made of, by one thread (and, for the alternatives, the threads of top()).
template <int DT>
__device__ __forceinline__ void write_row(const Out& o, int row, const Stat& a, const uint8_t* z_row, int64_t target,
                                          int64_t ignore, int V) {
  const float log_s = __builtin_amdgcn_logf(a.s) * kLn2;
  float lp = __builtin_nanf("");
  if (target == ignore) {
    lp = 0.f;
  } else if (target >= 0 && target < V) {
    float z[1];
    row_load<DT, 1>(z_row + target * kRowSize<DT>, z);
    lp = (z[0] - a.mu) - log_s;
  }
  o.lp[row] = lp;
  if (o.ent) o.ent[row] = log_s - a.h / a.s;
  o.stats[2 * static_cast<int64_t>(row)] = a.mu;
  o.stats[2 * static_cast<int64_t>(row) + 1] = a.s;
}
__device__ __forceinline__ void write_top(const Out& o, int row, int i, int k, const Stat& a, uint64_t key) {
  const int64_t at = static_cast<int64_t>(row) * k + i;
  // a row without a distribution (a NaN, +inf, nothing but −inf) has no alternatives
  const bool ok = a.s > 0.f && a.s < __builtin_inff();
  o.top_ids[at] = ok ? key_index(key) : -1;
  o.top_lp[at] = ok ? (key_value(key) - a.mu) - __builtin_amdgcn_logf(a.s) * kLn2 : __builtin_nanf("");
}

// One (row, part of the row) per workgroup and turn. One part: it writes the row's outputs; more: its
// statistics and best entries go to ws_stat [rows, parts] and ws_top [rows, parts, k].
template <int DT, bool ENT, bool TOP, int NT>
__device__ __forceinline__ void logprob_part(const uint8_t* __restrict__ z, const Row2& zr,
                                             const int64_t* __restrict__ targets, int64_t ignore, int V, int k,
                                             int parts, const Out& out, Stat* __restrict__ ws_stat,
                                             uint64_t* __restrict__ ws_top, int block) {
  constexpr int N = kRowVec<DT>, E = kRowSize<DT>, U = kUnroll;
  const int row = block / parts, part = block - row * parts;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int64_t target = targets[row];
  const uint8_t* const zp = z + row_offset(zr, row) * E;
  if (!ENT && !TOP && target == ignore) {  // nothing of this row is asked
    if (parts == 1 && tid == 0) {
      out.lp[row] = 0.f;
      out.stats[2 * static_cast<int64_t>(row)] = 0.f;
      out.stats[2 * static_cast<int64_t>(row) + 1] = 1.f;
    }
    return;
  }
  const Groups g = row_groups<DT>(zp, V);
  const int per = (g.n + parts - 1) / parts;
  const int q0 = min(part * per, g.n), q1 = min(q0 + per, g.n);
  Stat a = stat_none();
  int arg = -1;

  auto take = [&](int q) {  // a group that is not whole, value by value
    const int first = q * N - g.o;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int idx = first + e;
      if (idx < 0 || idx >= V) continue;
      float x[1];
      row_load<DT, 1>(zp + static_cast<int64_t>(idx) * E, x);
      if (TOP && (arg < 0 || x[0] > a.m)) arg = q;
      stat_raise(a, x[0]);
      stat_add<ENT>(a, x[0]);
    }
  };
  int q = q0 + tid;
  if (q < q1 && q < g.full0) {
    take(q);
    q += NT;
  }
  const int w1 = min(q1, g.full1);
  const uint8_t* const base = zp - static_cast<int64_t>(g.o) * E;
  for (; q + (U - 1) * NT < w1; q += U * NT) {
    float v[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u) row_load<DT, N>(base + static_cast<int64_t>(q + u * NT) * 16, v[u]);
    float gm[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      gm[u] = v[u][0];
#pragma unroll
      for (int e = 1; e < N; ++e) gm[u] = fmaxf(gm[u], v[u][e]);
    }
    float m = gm[0];
#pragma unroll
    for (int u = 1; u < U; ++u) m = fmaxf(m, gm[u]);
    if (TOP && (arg < 0 || m > a.m)) {
      int first = 0;
#pragma unroll
      for (int u = U - 1; u >= 0; --u)
        if (gm[u] == m) first = u;
      arg = q + first * NT;
    }
    stat_raise(a, m);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < N; ++e) stat_add<ENT>(a, v[u][e]);
  }
  for (; q < w1; q += NT) {
    float v[N];
    row_load<DT, N>(base + static_cast<int64_t>(q) * 16, v);
    float m = v[0];
#pragma unroll
    for (int e = 1; e < N; ++e) m = fmaxf(m, v[e]);
    if (TOP && (arg < 0 || m > a.m)) arg = q;
    stat_raise(a, m);
#pragma unroll
    for (int e = 0; e < N; ++e) stat_add<ENT>(a, v[e]);
  }
  if (q < q1) take(q);

  __shared__ Stat s_stat[NT / 64];
  const float best = a.m;
  for (int o = 32; o > 0; o >>= 1) stat_join(a, stat_shfl(a, o));
  if (lane == 0) s_stat[wave] = a;
  __syncthreads();
  a = s_stat[0];
#pragma unroll
  for (int w = 1; w < NT / 64; ++w) stat_join(a, s_stat[w]);

  if (parts == 1) {
    if (tid == 0) write_row<DT>(out, row, a, zp, target, ignore, V);
  } else if (tid == 0) {
    ws_stat[block] = a;
  }
  if constexpr (TOP) {
    __shared__ TopShared<NT> sh;
    const bool ok = a.s > 0.f && a.s < __builtin_inff();
    // a part may hold nothing but −inf of a row that has a distribution (s = 0)
    if (parts > 1 ? a.s < __builtin_inff() : ok) {
      block_row_top<DT, NT>(sh, zp, V, g, q0, q1, k, best, arg);
    } else {
      sh.buf[tid] = 0;
      __syncthreads();
    }
    if (tid < k) {
      if (parts == 1)
        write_top(out, row, tid, k, a, sh.buf[tid]);
      else
        ws_top[static_cast<int64_t>(block) * k + tid] = sh.buf[tid];
    }
  }
}

template <int DT, bool ENT, bool TOP, int NT>
__global__ __launch_bounds__(NT) void logprob_kernel(const uint8_t* __restrict__ z, Row2 zr,
                                                     const int64_t* __restrict__ targets, int64_t ignore, int V,
                                                     int k, int parts, Out out, Stat* __restrict__ ws_stat,
                                                     uint64_t* __restrict__ ws_top, int blocks) {
  for (int b = blockIdx.x; b < blocks; b += gridDim.x) {
    logprob_part<DT, ENT, TOP, NT>(z, zr, targets, ignore, V, k, parts, out, ws_stat, ws_top, b);
    __syncthreads();  // the shared sums are read before the next row's are written
  }
}

// Joins the parts of a row: one workgroup per row.
template <int DT, int NT>
__global__ __launch_bounds__(NT) void logprob_join_kernel(const uint8_t* __restrict__ z, Row2 zr,
                                                          const int64_t* __restrict__ targets, int64_t ignore, int V,
                                                          int k, int parts, bool skip, Out out,
                                                          const Stat* __restrict__ ws_stat,
                                                          const uint64_t* __restrict__ ws_top) {
  const int row = blockIdx.x, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int64_t target = targets[row];
  if (skip && target == ignore) {
    if (tid == 0) {
      out.lp[row] = 0.f;
      out.stats[2 * static_cast<int64_t>(row)] = 0.f;
      out.stats[2 * static_cast<int64_t>(row) + 1] = 1.f;
    }
    return;
  }
  __shared__ Stat s_stat[NT / 64];
  Stat a = stat_none();
  for (int p = tid; p < parts; p += NT) stat_join(a, ws_stat[static_cast<int64_t>(row) * parts + p]);
  for (int o = 32; o > 0; o >>= 1) stat_join(a, stat_shfl(a, o));
  if (lane == 0) s_stat[wave] = a;
  __syncthreads();
  a = s_stat[0];
#pragma unroll
  for (int w = 1; w < NT / 64; ++w) stat_join(a, s_stat[w]);
  if (tid == 0)
    write_row<DT>(out, row, a, z + row_offset(zr, row) * kRowSize<DT>, target, ignore, V);
  if (k) {
    __shared__ uint64_t buf[NT];
    // 64 kept, NT - 64 new ones a round
    const int total = parts * k;
    const uint64_t* const from = ws_top + static_cast<int64_t>(row) * total;
    buf[tid] = 0;
    __syncthreads();
    for (int i0 = 0; i0 < total; i0 += NT - 64) {
      const int i = i0 + tid - 64;
      if (tid >= 64) buf[tid] = i < total ? from[i] : 0;
      __syncthreads();
      block_top<NT>(buf, NT);
    }
    if (tid < k) write_top(out, row, tid, k, a, buf[tid]);
  }
}

// Gradient: workgroup (row, chunk of kChunk groups of the output row).
constexpr int kGradThreads = 256, kGradGroups = 1024;

template <int DT, bool ENT>
__device__ __forceinline__ void logprob_grad_chunk(
    const uint8_t* __restrict__ z, Row2 zr, const int64_t* __restrict__ targets, int64_t ignore,
    const float* __restrict__ stats, const float* __restrict__ ent, const float* __restrict__ g_lp, int64_t g_lp_st,
    const float* __restrict__ g_ent, int64_t g_ent_st, uint8_t* __restrict__ dz, int V, int chunks, int64_t block) {
  constexpr int N = kRowVec<DT>, E = kRowSize<DT>;
  const int row = static_cast<int>(block / chunks);
  const int chunk = static_cast<int>(block - static_cast<int64_t>(row) * chunks);
  const int64_t target = targets[row];
  const bool given = target != ignore;
  const float gl = given && g_lp ? g_lp[row * g_lp_st] : 0.f;
  const float ge = ENT ? g_ent[row * g_ent_st] : 0.f;
  const float mu = stats[2 * static_cast<int64_t>(row)], s = stats[2 * static_cast<int64_t>(row) + 1];
  const float inv = 1.f / s, log_s = __builtin_amdgcn_logf(s) * kLn2;
  // dz_j = g_lp δ_jt − p_j (g_lp + g_H (ln p_j + H))
  const float H = ENT ? ent[row] : 0.f;
  const float c0 = ENT ? fmaf(ge, H - log_s, gl) : gl;
  const bool bad = given && (target < 0 || target >= V);  // its lp is NaN
  const bool zero = !given && !(ENT && ge != 0.f);         // nothing of the row was asked
  const uint8_t* const zp = z + row_offset(zr, row) * E;
  uint8_t* const dp = dz + static_cast<int64_t>(row) * V * E;
  const Groups g = row_groups<DT>(dp, V);
  const bool same = ((reinterpret_cast<uintptr_t>(zp) ^ reinterpret_cast<uintptr_t>(dp)) & 15) == 0;
  const int t = given && !bad ? static_cast<int>(target) : -1;
  auto value = [&](float x, int idx) {
    const float d = x - mu, p = exp_d(d) * inv;
    float r = ENT ? -p * fmaf(ge, fmaxf(d, kFar), c0) : -p * c0;
    if (idx == t) r += gl;
    return bad ? __builtin_nanf("") : r;
  };
  const int q_end = min((chunk + 1) * kGradGroups, g.n);
  for (int q = chunk * kGradGroups + threadIdx.x; q < q_end; q += kGradThreads) {
    const int first = q * N - g.o;
    const int64_t at = static_cast<int64_t>(first) * E;
    if (q >= g.full0 && q < g.full1) {
      float v[N];
      if (zero) {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = 0.f;
      } else {
        if (same) {
          row_load<DT, N>(zp + at, v);
        } else {
#pragma unroll
          for (int e = 0; e < N; ++e) {
            float x[1];
            row_load<DT, 1>(zp + at + e * E, x);
            v[e] = x[0];
          }
        }
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = value(v[e], first + e);
      }
      row_store<DT, N>(dp + at, v);
    } else {
      for (int e = 0; e < N; ++e) {
        const int idx = first + e;
        if (idx < 0 || idx >= V) continue;
        float x[1] = {0.f};
        if (!zero) {
          row_load<DT, 1>(zp + static_cast<int64_t>(idx) * E, x);
          x[0] = value(x[0], idx);
        }
        row_store<DT, 1>(dp + static_cast<int64_t>(idx) * E, x);
      }
    }
  }
}

template <int DT, bool ENT>
__global__ __launch_bounds__(kGradThreads) void logprob_grad_kernel(
    const uint8_t* __restrict__ z, Row2 zr, const int64_t* __restrict__ targets, int64_t ignore,
    const float* __restrict__ stats, const float* __restrict__ ent, const float* __restrict__ g_lp, int64_t g_lp_st,
    const float* __restrict__ g_ent, int64_t g_ent_st, uint8_t* __restrict__ dz, int V, int chunks, int64_t blocks) {
  for (int64_t b = blockIdx.x; b < blocks; b += gridDim.x)
    logprob_grad_chunk<DT, ENT>(z, zr, targets, ignore, stats, ent, g_lp, g_lp_st, g_ent, g_ent_st, dz, V, chunks, b);
}

// The mean of −lp over the rows that are not ignored (NaN where there are none), and −1 / their number for
// the backward: one workgroup, sums in a fixed order.
template <int DT>
__global__ __launch_bounds__(1024) void logprob_mean_kernel(const float* __restrict__ lp,
                                                            const int64_t* __restrict__ targets, int64_t ignore,
                                                            int rows, void* __restrict__ loss,
                                                            float* __restrict__ neg_inv) {
  __shared__ float s_sum[16];
  __shared__ int s_n[16];
  float sum = 0.f;
  int n = 0;
  for (int i = threadIdx.x; i < rows; i += 1024) {
    sum += lp[i];
    n += targets[i] != ignore;
  }
  for (int o = 32; o > 0; o >>= 1) {
    sum += __shfl_xor(sum, o);
    n += __shfl_xor(n, o);
  }
  if ((threadIdx.x & 63) == 0) {
    s_sum[threadIdx.x >> 6] = sum;
    s_n[threadIdx.x >> 6] = n;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0.f;
    n = 0;
    for (int w = 0; w < 16; ++w) {
      sum += s_sum[w];
      n += s_n[w];
    }
    const float v[1] = {-sum / static_cast<float>(n)};
    row_store<DT, 1>(loss, v);
    *neg_inv = -1.f / static_cast<float>(n);
  }
}

// ------------------------------------------------------------------ host

constexpr int64_t kMaxRows = 1 << 30, kMaxV = 1 << 28;
constexpr int kMaxGrid = 1 << 21;    // workgroups of a launch; they take turns beyond that
constexpr int kShortRow = 32 << 10;  // bytes of a row below which 256 threads take it

int check(int B, int T, int64_t V, int64_t st, int64_t sb, int dtype) {
  if (dtype != TMAC_F32 && dtype != TMAC_BF16 && dtype != TMAC_F16) return TMAC_ERR_DTYPE;
  if (B < 0 || T < 0 || V <= 0 || V > kMaxV || static_cast<int64_t>(B) * T > kMaxRows) return TMAC_ERR_SHAPE;
  if ((T > 1 && st < 0) || (B > 1 && sb < 0)) return TMAC_ERR_SHAPE;
  return TMAC_OK;
}

int launch_status() {
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? TMAC_OK : static_cast<int>(err);
}

// Workgroups per row: enough of them for the chip, of at least 2048 groups (32 KB) of the row each.
int row_parts(int rows, int64_t V, int dtype) {
  const int64_t groups = (V + (dtype == TMAC_F32 ? 3 : 7)) / (dtype == TMAC_F32 ? 4 : 8);
  int64_t parts = 512 / (rows > 0 ? rows : 1);
  const int64_t most = groups / 512;
  if (parts > most) parts = most;
  return static_cast<int>(parts < 1 ? 1 : parts);
}

template <typename F>
void by_type(int dtype, F&& f) {
  using std::integral_constant;
  if (dtype == TMAC_F32)
    f(integral_constant<int, TMAC_F32>{});
  else if (dtype == TMAC_BF16)
    f(integral_constant<int, TMAC_BF16>{});
  else
    f(integral_constant<int, TMAC_F16>{});
}
template <typename F>
void by_flag(bool on, F&& f) {
  if (on)
    f(std::true_type{});
  else
    f(std::false_type{});
}

size_t stat_bytes(int rows, int parts) { return parts > 1 ? sizeof(Stat) * static_cast<size_t>(rows) * parts : 0; }

}  // namespace

extern "C" int tmac_logprob_workspace(int B, int T, int64_t V, int top_k, int dtype, size_t* ws_bytes) {
  if (!ws_bytes) return TMAC_ERR_NULL;
  const int st = check(B, T, V, 0, 0, dtype);
  if (st != TMAC_OK) return st;
  if (top_k < 0 || top_k > kMaxTop || top_k > V) return TMAC_ERR_VALUE;
  const int parts = row_parts(B * T, V, dtype);
  *ws_bytes = stat_bytes(B * T, parts) + (parts > 1 ? 8 * static_cast<size_t>(B * T) * parts * top_k : 0);
  return TMAC_OK;
}

extern "C" int tmac_logprob_fwd(const void* d_z, int64_t stride_b, int64_t stride_t, const int64_t* d_targets,
                                int64_t ignore_index, float* d_lp, float* d_entropy, int top_k, int64_t* d_top_ids,
                                float* d_top_lp, float* d_stats, void* d_ws, size_t ws_bytes, int B, int T, int64_t V,
                                int dtype, void* stream) {
  const int st = check(B, T, V, stride_t, stride_b, dtype);
  if (st != TMAC_OK) return st;
  size_t need = 0;
  const int wst = tmac_logprob_workspace(B, T, V, top_k, dtype, &need);
  if (wst != TMAC_OK) return wst;
  const int rows = B * T;
  if (rows == 0) return TMAC_OK;
  if (!d_z || !d_targets || !d_lp || !d_stats || (top_k && (!d_top_ids || !d_top_lp))) return TMAC_ERR_NULL;
  if (reinterpret_cast<uintptr_t>(d_z) % (dtype == TMAC_F32 ? 4 : 2)) return TMAC_ERR_ALIGN;
  if (need && (!d_ws || ws_bytes < need)) return TMAC_ERR_WORKSPACE;
  if (need && !row_aligned16(d_ws)) return TMAC_ERR_ALIGN;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int parts = row_parts(rows, V, dtype), v = static_cast<int>(V);
  const int E = dtype == TMAC_F32 ? 4 : 2;
  const Row2 zr{stride_b, stride_t, T};
  const Out out{d_lp, d_entropy, d_top_ids, d_top_lp, d_stats};
  Stat* const ws_stat = static_cast<Stat*>(d_ws);
  uint64_t* const ws_top = reinterpret_cast<uint64_t*>(static_cast<uint8_t*>(d_ws) + stat_bytes(rows, parts));
  const uint8_t* const z = static_cast<const uint8_t*>(d_z);
  by_type(dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    by_flag(d_entropy != nullptr, [&](auto e) {
      by_flag(top_k > 0, [&](auto t) {
        constexpr bool ENT = decltype(e)::value, TOP = decltype(t)::value;
        const int blocks = rows * parts, grid = blocks < kMaxGrid ? blocks : kMaxGrid;
        if (parts > 1 || V * E < kShortRow)
          logprob_kernel<DT, ENT, TOP, 256><<<grid, 256, 0, s>>>(z, zr, d_targets, ignore_index, v, top_k, parts, out,
                                                                 ws_stat, ws_top, blocks);
        else
          logprob_kernel<DT, ENT, TOP, 1024><<<grid, 1024, 0, s>>>(z, zr, d_targets, ignore_index, v, top_k, 1, out,
                                                                   ws_stat, ws_top, blocks);
      });
    });
    if (parts > 1)
      logprob_join_kernel<DT, 256><<<rows, 256, 0, s>>>(z, zr, d_targets, ignore_index, v, top_k, parts,
                                                        !d_entropy && !top_k, out, ws_stat, ws_top);
  });
  return launch_status();
}

extern "C" int tmac_logprob_bwd(const void* d_z, int64_t stride_b, int64_t stride_t, const int64_t* d_targets,
                                int64_t ignore_index, const float* d_stats, const float* d_entropy,
                                const float* d_g_lp, int64_t g_lp_stride, const float* d_g_entropy,
                                int64_t g_entropy_stride, void* d_dz, int B, int T, int64_t V, int dtype,
                                void* stream) {
  const int st = check(B, T, V, stride_t, stride_b, dtype);
  if (st != TMAC_OK) return st;
  const int rows = B * T;
  if (rows == 0) return TMAC_OK;
  if (!d_z || !d_targets || !d_stats || !d_dz || (d_g_entropy && !d_entropy)) return TMAC_ERR_NULL;
  const int E = dtype == TMAC_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(d_z) % E || reinterpret_cast<uintptr_t>(d_dz) % E) return TMAC_ERR_ALIGN;
  const int64_t groups = (V + 16 / E - 2) / (16 / E) + 1;  // of a row at any alignment
  const int64_t chunks = (groups + kGradGroups - 1) / kGradGroups;
  const int64_t blocks = chunks * rows;
  by_type(dtype, [&](auto dt) {
    by_flag(d_g_entropy != nullptr, [&](auto e) {
      logprob_grad_kernel<decltype(dt)::value, decltype(e)::value>
          <<<static_cast<unsigned>(blocks < (1 << 23) ? blocks : 1 << 23), kGradThreads, 0, static_cast<hipStream_t>(stream)>>>(
              static_cast<const uint8_t*>(d_z), Row2{stride_b, stride_t, T}, d_targets, ignore_index, d_stats,
              d_entropy, d_g_lp, g_lp_stride, d_g_entropy, g_entropy_stride, static_cast<uint8_t*>(d_dz),
              static_cast<int>(V), static_cast<int>(chunks), blocks);
    });
  });
  return launch_status();
}

extern "C" int tmac_logprob_mean(const float* d_lp, const int64_t* d_targets, int64_t ignore_index, int rows,
                                 void* d_loss, int dtype, float* d_neg_inv, void* stream) {
  if (dtype != TMAC_F32 && dtype != TMAC_BF16 && dtype != TMAC_F16) return TMAC_ERR_DTYPE;
  if (rows < 0) return TMAC_ERR_SHAPE;
  if (!d_loss || !d_neg_inv || (rows && (!d_lp || !d_targets))) return TMAC_ERR_NULL;
  by_type(dtype, [&](auto dt) {
    logprob_mean_kernel<decltype(dt)::value><<<1, 1024, 0, static_cast<hipStream_t>(stream)>>>(
        d_lp, d_targets, ignore_index, rows, d_loss, d_neg_inv);
  });
  return launch_status();
}
