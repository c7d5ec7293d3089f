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
// saw it, and the best value of its other groups. Order the threads by (m, earlier group), and take any
// place in that order that k threads reach: the k best values lie with the threads up to it, since all that
// another one has comes after k threads' bests. The place is the k-th of 64 that the waves publish (an
// equal share each: for k up to 8 the k-th of all). Of those threads the best group is read again, 16 bytes
// of a line each, and the others only where their best reaches the bound too (a thread's groups are
// strewn over the row, so that reading all of them costs k / 512 of the row's groups but an eighth of its
// lines for k = 8). What reaches the bound is sorted: a few dozen entries for ordinary rows, any number
// in rounds that keep the best 64.
//
// m and s are kept for the backward, p = e^{z − m} / s: through lse the rounding of a sum near 12 would
// go into every p.

#include "row_device.h"

using namespace tmac;

namespace {

constexpr int kMaxTop = 64;
constexpr int kUnroll = 2;

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

// lanes i and i ^ J exchange so that the larger value is at the lower lane (desc) or the higher
template <int J>
__device__ __forceinline__ uint64_t exchange(uint64_t v, int lane, bool desc) {
  const uint64_t o = lane_xor<J>(v);
  const bool low = (lane & J) == 0;
  return (v > o) == (low == desc) ? v : o;
}
template <int J>
__device__ __forceinline__ uint64_t exchanges(uint64_t v, int lane, bool desc) {
  v = exchange<J>(v, lane, desc);
  if constexpr (J > 1) v = exchanges<J / 2>(v, lane, desc);
  return v;
}
// bitonic sort of a wave's 64 keys, descending
__device__ __forceinline__ uint64_t wave_sort(uint64_t v, int lane) {
  v = exchanges<1>(v, lane, (lane & 2) == 0);
  v = exchanges<2>(v, lane, (lane & 4) == 0);
  v = exchanges<4>(v, lane, (lane & 8) == 0);
  v = exchanges<8>(v, lane, (lane & 16) == 0);
  v = exchanges<16>(v, lane, (lane & 32) == 0);
  return exchanges<32>(v, lane, true);
}
// the 64 largest of two descending lists, descending; b is given reversed
__device__ __forceinline__ uint64_t wave_merge(uint64_t a, uint64_t b_rev, int lane) {
  return exchanges<32>(a > b_rev ? a : b_rev, lane, true);
}

// The 64 largest of buf[0 .. n), n <= NT, in descending order in the lanes of wave 0 (0 where there are fewer);
// by all of the workgroup's NT threads, which have written buf before a barrier.
template <int NT>
__device__ uint64_t block_top(uint64_t* buf, int n) {
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
  return v;
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

// What a thread saw of its groups: the best value, the first group that has it (−1: no entry), and the best
// value of its other groups.
struct Best {
  float m, second;
  int group;
};
__device__ __forceinline__ void best_add(Best& a, float m, int group) {
  a.second = __builtin_amdgcn_fmed3f(a.m, a.second, m);  // second <= m of a
  if (a.group < 0 || m > a.m) a.group = group;
  a.m = fmaxf(a.m, m);
}

template <int NT>
struct TopShared {
  uint64_t buf[NT];
  uint64_t bests[64];   // the waves' highest threads' bests, an equal number of each wave's
  int group[NT];        // every thread's best group
  uint16_t thread[NT];  // the threads whose best is among what may be the k best
  uint16_t again[NT];   // those of them whose other groups have to be looked at too
  int threads, agains, count;
};

// First part of the alternatives, before a barrier.
template <int NT>
__device__ __forceinline__ void top_publish(TopShared<NT>& sh, const Best& best) {
  constexpr int kShare = 64 * 64 / NT;
  const int tid = threadIdx.x, lane = tid & 63;
  const uint64_t v = wave_sort(best.group >= 0 ? top_key(best.m, best.group) : 0, lane);
  if (lane < kShare) sh.bests[(tid >> 6) * kShare + lane] = v;
  sh.group[tid] = best.group;
  if (tid == 0) sh.threads = sh.agains = sh.count = 0;
}

// Second part, after it: the k best entries of the workgroup's groups [q0, q1) of a row, in wave 0's lanes.
template <int DT, int NT>
__device__ uint64_t top_entries(TopShared<NT>& sh, const uint8_t* row, int V, const Groups& g, int q0, int q1, int k,
                                const Best& best) {
  constexpr int N = kRowVec<DT>, E = kRowSize<DT>;
  const int tid = threadIdx.x, lane = tid & 63;
  // the k-th of the published bests is reached by k threads: every other thread's entries come after those
  const uint64_t sorted = wave_sort(sh.bests[lane], lane);
  const uint64_t bound = static_cast<uint64_t>(__builtin_amdgcn_readlane(static_cast<uint32_t>(sorted >> 32), k - 1)) << 32 |
                         static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<uint32_t>(sorted), k - 1));
  // nor is an entry of the k best below its value, or, at that value, behind its group; with no bound every
  // entry may be among them
  const uint32_t last = bound ? static_cast<uint32_t>((key_index(bound) + 1) * N - 1 - g.o) : ~0u;
  const uint64_t floor_key = bound ? (bound & ~0xffffffffull) | static_cast<uint32_t>(~last) : 1;
  const float floor_value = bound ? key_value(bound) : -__builtin_inff();
  if (best.group >= 0 && top_key(best.m, best.group) >= bound) {
    sh.thread[atomicAdd(&sh.threads, 1)] = static_cast<uint16_t>(tid);
    if (best.second >= floor_value) sh.again[atomicAdd(&sh.agains, 1)] = static_cast<uint16_t>(tid);
  }
  __syncthreads();
  // item i: a group that those threads saw, their best one first (−1 and less: none)
  const int per = (q1 - q0 + NT - 1) / NT, n_thr = sh.threads;  // groups a thread has, at most
  const int items = n_thr + sh.agains * per;
  auto group = [&](int i) {
    if (i < n_thr) return sh.group[sh.thread[i]];
    i -= n_thr;
    const int t = i / per, q = q0 + sh.again[t] + (i - t * per) * NT;
    return q < q1 && q != sh.group[sh.again[t]] ? q : -1;
  };
  auto add = [&](float z, int idx) {
    if (z >= floor_value) {
      const uint64_t kk = top_key(z, idx);
      if (kk >= floor_key) {
        const int at = atomicAdd(&sh.count, 1);
        if (at < NT) sh.buf[at] = kk;
      }
    }
  };
  for (int i = tid; i < items; i += NT) {
    const int q = group(i);
    if (q < 0) continue;
    const int first = q * N - g.o;
    const uint8_t* const at = row + static_cast<int64_t>(first) * E;
    if (q >= g.full0 && q < g.full1) {
      float z[N];
      row_load<DT, N>(at, z);
#pragma unroll
      for (int e = 0; e < N; ++e) add(z[e], first + e);
    } else {
      for (int e = max(0, -first); e < N && first + e < V; ++e) {
        float z[1];
        row_load<DT, 1>(at + e * E, z);
        add(z[0], first + e);
      }
    }
  }
  __syncthreads();
  const int total = sh.count;
  if (total <= NT) return block_top<NT>(sh.buf, total);
  // too many: again, the e-th values of half of the threads at a time beside the best 64 so far
  __syncthreads();
  if (tid == 0) sh.count = 0;
  for (int i0 = 0; i0 < items; i0 += NT) {
    const int q = i0 + tid < items ? group(i0 + tid) : -1;
#pragma unroll 1
    for (int round = 0; round < 2 * N; ++round) {
      const int idx = q * N - g.o + (round >> 1);
      __syncthreads();
      if (q >= 0 && (tid & 1) == (round & 1) && idx >= 0 && idx < V) {
        float z[1];
        row_load<DT, 1>(row + static_cast<int64_t>(idx) * E, z);
        add(z[0], idx);
      }
      __syncthreads();
      const int n = sh.count;
      if (n <= 64) continue;
      const uint64_t v = block_top<NT>(sh.buf, n);
      __syncthreads();
      if (tid < 64) sh.buf[tid] = v;
      if (tid == 0) sh.count = 64;
    }
  }
  __syncthreads();
  return block_top<NT>(sh.buf, sh.count);
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
  const int tid = threadIdx.x;
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
  Best best{-__builtin_inff(), -__builtin_inff(), -1};

  auto take = [&](int q) {  // a group that is not whole, value by value
    const int first = q * N - g.o;
    float m = -__builtin_inff();
    for (int e = max(0, -first); e < N && first + e < V; ++e) {
      float x[1];
      row_load<DT, 1>(zp + static_cast<int64_t>(first + e) * E, x);
      m = fmaxf(m, x[0]);
      stat_raise(a, x[0]);
      stat_add<ENT>(a, x[0]);
    }
    if (TOP) best_add(best, m, q);
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
    if (TOP) {
#pragma unroll
      for (int u = 0; u < U; ++u) best_add(best, gm[u], q + u * NT);
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
    if (TOP) best_add(best, m, q);
    stat_raise(a, m);
#pragma unroll
    for (int e = 0; e < N; ++e) stat_add<ENT>(a, v[e]);
  }
  if (q < q1) take(q);

  __shared__ Stat s_stat[NT / 64];
  if constexpr (TOP) {
    __shared__ TopShared<NT> sh;
    top_publish<NT>(sh, best);
    stat_block<NT / 64>(a, s_stat);
    // a part may hold nothing but −inf of a row that has a distribution (s = 0)
    uint64_t v = 0;
    if (a.s < __builtin_inff() && (parts > 1 || a.s > 0.f)) v = top_entries<DT, NT>(sh, zp, V, g, q0, q1, k, best);
    if (tid < k) {
      if (parts == 1)
        write_top(out, row, tid, k, a, v);
      else
        ws_top[static_cast<int64_t>(block) * k + tid] = v;
    }
  } else {
    stat_block<NT / 64>(a, s_stat);
  }
  if (tid == 0) {
    if (parts == 1)
      write_row<DT>(out, row, a, zp, target, ignore, V);
    else
      ws_stat[block] = a;
  }
}

template <int DT, bool ENT, bool TOP, int NT>
__global__ __launch_bounds__(NT, 8) void logprob_kernel(const uint8_t* __restrict__ z, Row2 zr,
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
  stat_block<NT / 64>(a, s_stat);
  if (tid == 0)
    write_row<DT>(out, row, a, z + row_offset(zr, row) * kRowSize<DT>, target, ignore, V);
  if (k) {
    // each wave merges its parts' descending lists, then the waves' lists
    __shared__ uint64_t buf[NT];
    uint64_t v = 0;
    for (int p = wave; p < parts; p += NT / 64) {
      const uint64_t* const from = ws_top + (static_cast<int64_t>(row) * parts + p) * k;
      v = wave_merge(v, 63 - lane < k ? from[63 - lane] : 0, lane);
    }
    for (int half = 1; half < NT / 64; half *= 2) {
      buf[tid] = v;
      __syncthreads();
      if (wave % (2 * half) == 0) v = wave_merge(v, buf[64 * (wave + half) + 63 - lane], lane);
      __syncthreads();
    }
    if (tid < k) write_top(out, row, tid, k, a, v);
  }
}

// Gradient: workgroup (row, chunk of kChunk groups of the output row).
constexpr int kGradGroups = 1024;

// A factor of g_lp, one value of a type in memory: read as two halves, without a branch and before anything else, so
// that nothing waits for it before the row's own values are on their way (8192 x 128000 bf16 702 us, read where it is
// used 718, without a factor 690).
struct Factor {
  const uint16_t *low, *high;  // the same for 16 bit
  int dtype;
  struct Bits {
    uint16_t low, high;
    int dtype;
    __device__ __forceinline__ float value() const {
      const float f16 = Mfma<TMAC_F16>::to_f32(high);
      return dtype == TMAC_F16 ? f16 : __uint_as_float(static_cast<uint32_t>(high) << 16 | (dtype == TMAC_F32 ? low : 0));
    }
  };
  __device__ __forceinline__ Bits load() const { return Bits{*low, *high, dtype}; }
};
struct NoFactor {
  struct Bits {
    __device__ __forceinline__ float value() const { return 1.f; }
  };
  __device__ __forceinline__ Bits load() const { return Bits{}; }
};

template <int DT, bool ENT, int NT, typename Bits>
__device__ __forceinline__ void logprob_grad_chunk(
    const uint8_t* __restrict__ z, Row2 zr, const int64_t* __restrict__ targets, int64_t ignore,
    const float* __restrict__ stats, const float* __restrict__ ent, const float* __restrict__ g_lp, int64_t g_lp_st,
    const Bits& factor, const float* __restrict__ g_ent, int64_t g_ent_st, uint8_t* __restrict__ dz, int V, int chunks,
    int64_t block) {
  constexpr int N = kRowVec<DT>, E = kRowSize<DT>;
  const int row = static_cast<int>(block / chunks);
  const int chunk = static_cast<int>(block - static_cast<int64_t>(row) * chunks);
  const int64_t target = targets[row];
  const bool given = g_lp && target != ignore;
  const float gl = given ? g_lp[row * g_lp_st] * factor.value() : 0.f;
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
  for (int q = chunk * kGradGroups + threadIdx.x; q < q_end; q += NT) {
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

template <int DT, bool ENT, int NT, typename F>
__global__ __launch_bounds__(NT) void logprob_grad_kernel(
    const uint8_t* __restrict__ z, Row2 zr, const int64_t* __restrict__ targets, int64_t ignore,
    const float* __restrict__ stats, const float* __restrict__ ent, const float* __restrict__ g_lp, int64_t g_lp_st,
    F factor, const float* __restrict__ g_ent, int64_t g_ent_st, uint8_t* __restrict__ dz, int V, int chunks,
    int64_t blocks) {
  const typename F::Bits bits = factor.load();
  for (int64_t b = blockIdx.x; b < blocks; b += gridDim.x)
    logprob_grad_chunk<DT, ENT, NT>(z, zr, targets, ignore, stats, ent, g_lp, g_lp_st, bits, g_ent, g_ent_st, dz, V,
                                    chunks, b);
}

// The mean of −lp over the rows that are not ignored (NaN where there are none), and −1 / their number for
// the backward: one workgroup, sums in a fixed order. Eight rows in flight a thread: 2^18 rows 41 us, one after the other
// about 87.
template <int DT>
__global__ __launch_bounds__(1024) void logprob_mean_kernel(const float* __restrict__ lp,
                                                            const int64_t* __restrict__ targets, int64_t ignore,
                                                            int rows, void* __restrict__ loss,
                                                            float* __restrict__ neg_inv) {
  __shared__ float s_sum[16];
  __shared__ int s_n[16];
  float sum = 0.f;
  int n = 0;
  constexpr int U = 8;
  for (int i = threadIdx.x; i < rows; i += U * 1024) {
    float x[U];
    int64_t t[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = i + 1024 * u < rows;
      x[u] = in ? lp[i + 1024 * u] : 0.f;
      t[u] = in ? targets[i + 1024 * u] : ignore;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      sum += x[u];
      n += t[u] != ignore;
    }
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
constexpr int kMaxGrid = 1 << 21;  // workgroups of a launch; they take turns beyond that
// Groups of a row up to which one wave takes it, forward (without alternatives) and backward: rows this short cost what
// starting their waves does. us with one wave, and with the widths below: 2^20 rows of 32 bf16 forward 376 / 690, backward
// 447 / 1070, 2^18 rows of 256 97 / 175 and 116 / 270.
constexpr int kWaveGroups = 64;
// Threads of a row otherwise: 128 below 32 KB (us, 128 / 256 / 512 threads: 20000 rows of 1000 bf16 18 / 28 / 50, 8000 of
// 8000 24 / 24 / 31), then 512 (8192 of 128000: 382 / 351 / 344), with alternatives 256 (4096 of 128000: five of
// them 201 / 197 / 214, twenty 209 / 200 / 218, 64 568 / 243 / 230).
constexpr int kShortRow = 32 << 10;
// Whole rows with alternatives up to which 512 threads take one (16 rows: 12.4 us, with 256 threads 14.7).
constexpr int kFewRows = 1024;

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

// 16-byte groups of a row at any alignment
int64_t max_groups(int64_t V, int dtype) {
  const int n = dtype == TMAC_F32 ? 4 : 8;
  return (V + n - 2) / n + 1;
}

// Workgroups per row: one below 8192 groups (128 KB), whose second launch costs more than it gains (16 rows of 50000
// bf16 with twenty alternatives: 12.4 us, in six parts 13.5; 200 rows 11.9 against 17.4), else about 1024 in all,
// of at least 1024 groups each (16 rows of 128000 bf16: 13.5 us, of 4096 groups 15.7, whole rows 18.6; one row of
// 128000 fp32 with 64 alternatives 13.4, of 256 groups 18.6: more lists to join).
int row_parts(int rows, int64_t V, int dtype) {
  const int64_t groups = (V + (dtype == TMAC_F32 ? 3 : 7)) / (dtype == TMAC_F32 ? 4 : 8);
  if (groups < 8192) return 1;
  int64_t parts = 1024 / (rows > 0 ? rows : 1);
  const int64_t most = groups / 1024;
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

template <typename F>
int launch_grad(const void* d_z, int64_t stride_b, int64_t stride_t, const int64_t* d_targets, int64_t ignore_index,
                const float* d_stats, const float* d_entropy, const float* d_g_lp, int64_t g_lp_stride, F factor,
                const float* d_g_entropy, int64_t g_entropy_stride, void* d_dz, int B, int T, int64_t V, int dtype,
                void* stream) {
  const int st = check(B, T, V, stride_t, stride_b, dtype);
  if (st != TMAC_OK) return st;
  const int rows = B * T;
  if (rows == 0) return TMAC_OK;
  if (!d_z || !d_targets || !d_stats || !d_dz || (d_g_entropy && !d_entropy)) return TMAC_ERR_NULL;
  const int E = dtype == TMAC_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(d_z) % E || reinterpret_cast<uintptr_t>(d_dz) % E) return TMAC_ERR_ALIGN;
  const int64_t groups = max_groups(V, dtype), chunks = (groups + kGradGroups - 1) / kGradGroups, blocks = chunks * rows;
  by_type(dtype, [&](auto dt) {
    auto with = [&](auto e) {
      auto launch = [&](auto nt) {
        constexpr int NT = decltype(nt)::value;
        logprob_grad_kernel<decltype(dt)::value, decltype(e)::value, NT, F>
            <<<static_cast<unsigned>(blocks < (1 << 23) ? blocks : 1 << 23), NT, 0, static_cast<hipStream_t>(stream)>>>(
                static_cast<const uint8_t*>(d_z), Row2{stride_b, stride_t, T}, d_targets, ignore_index, d_stats,
                d_entropy, d_g_lp, g_lp_stride, factor, d_g_entropy, g_entropy_stride, static_cast<uint8_t*>(d_dz),
                static_cast<int>(V), static_cast<int>(chunks), blocks);
      };
      if (groups <= kWaveGroups)
        launch(std::integral_constant<int, 64>{});
      else
        launch(std::integral_constant<int, 256>{});
    };
    if constexpr (std::is_same<F, NoFactor>::value)
      by_flag(d_g_entropy != nullptr, with);
    else  // the loss has no entropies
      with(std::false_type{});
  });
  return launch_status();
}

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
        auto launch = [&](auto nt) {
          constexpr int NT = decltype(nt)::value;
          logprob_kernel<DT, ENT, TOP, NT><<<grid, NT, 0, s>>>(z, zr, d_targets, ignore_index, v, top_k, parts, out,
                                                               ws_stat, ws_top, blocks);
        };
        if constexpr (!TOP) {
          if (max_groups(V, dtype) <= kWaveGroups) {
            launch(std::integral_constant<int, 64>{});
            return;
          }
        }
        if (parts == 1 && V * E < kShortRow)
          launch(std::integral_constant<int, 128>{});
        else if (TOP && (parts > 1 || rows > kFewRows))
          launch(std::integral_constant<int, 256>{});
        else
          launch(std::integral_constant<int, 512>{});
      });
    });
    if (parts > 1)
      logprob_join_kernel<DT, 512><<<rows, 512, 0, s>>>(z, zr, d_targets, ignore_index, v, top_k, parts,
                                                        !d_entropy && !top_k, out, ws_stat, ws_top);
  });
  return launch_status();
}

extern "C" int tmac_logprob_bwd(const void* d_z, int64_t stride_b, int64_t stride_t, const int64_t* d_targets,
                                int64_t ignore_index, const float* d_stats, const float* d_entropy,
                                const float* d_g_lp, int64_t g_lp_stride, const float* d_g_entropy,
                                int64_t g_entropy_stride, void* d_dz, int B, int T, int64_t V, int dtype,
                                void* stream) {
  return launch_grad(d_z, stride_b, stride_t, d_targets, ignore_index, d_stats, d_entropy, d_g_lp, g_lp_stride,
                     NoFactor{}, d_g_entropy, g_entropy_stride, d_dz, B, T, V, dtype, stream);
}

extern "C" int tmac_logprob_mean_bwd(const void* d_z, int64_t stride_b, int64_t stride_t, const int64_t* d_targets,
                                     int64_t ignore_index, const float* d_stats, const float* d_neg_inv,
                                     const void* d_g_loss, int g_dtype, void* d_dz, int B, int T, int64_t V, int dtype,
                                     void* stream) {
  if (g_dtype != TMAC_F32 && g_dtype != TMAC_BF16 && g_dtype != TMAC_F16) return TMAC_ERR_DTYPE;
  if (!d_neg_inv || !d_g_loss) return TMAC_ERR_NULL;
  const uint16_t* const g = static_cast<const uint16_t*>(d_g_loss);
  return launch_grad(d_z, stride_b, stride_t, d_targets, ignore_index, d_stats, nullptr, d_neg_inv, 0,
                     Factor{g, g + (g_dtype == TMAC_F32), g_dtype}, nullptr, 0, d_dz, B, T, V, dtype, stream);
}

extern "C" int tmac_logprob_mean(const float* d_lp, const int64_t* d_targets, int64_t ignore_index, int rows,
                                 void* d_loss, int dtype, float* d_neg_inv, void* stream) {
  if (dtype != TMAC_F32 && dtype != TMAC_BF16 && dtype != TMAC_F16) return TMAC_ERR_DTYPE;
  if (rows < 0 || rows > kMaxRows) return TMAC_ERR_SHAPE;
  if (!d_loss || !d_neg_inv || (rows && (!d_lp || !d_targets))) return TMAC_ERR_NULL;
  by_type(dtype, [&](auto dt) {
    logprob_mean_kernel<decltype(dt)::value><<<1, 1024, 0, static_cast<hipStream_t>(stream)>>>(
        d_lp, d_targets, ignore_index, rows, d_loss, d_neg_inv);
  });
  return launch_status();
}
