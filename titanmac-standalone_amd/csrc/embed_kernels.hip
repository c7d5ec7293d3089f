// Token embedding in front of the blocks and the gradients of its tables, for gfx950.
//
//   out[b, p]      = prefix[p]                                  p < n_prefix (the persistent tokens)
//   out[b, Np + t] = scale · W[ids[b, t]] + P[pos(b, t)]        pos = t, or given
//   dW[v] = scale · Σ_{ids[b, t] = v} g[b, Np + t],   dP, dprefix likewise
//
// (models/titanmac.py:183-190: two nn.Embedding lookups, their sum and the concatenation behind the
// expanded persistent tokens; autograd's gradients of them.) All of it moves memory: one pass writes out
// once, and the gradient, dense as nn.Embedding's, is written once, rows without a token as zeros.
//
// The gradient sums each row's tokens in ascending order of position (deterministic): a sort gives every
// row of W its list of tokens; a list of up to 64 is summed where its row is written; longer ones (the
// frequent tokens: a text's first hundred ids are half of it) are summed 64 tokens a workgroup into fp32
// partial rows that a third kernel adds in order, so one frequent token does not hold one workgroup.

#include "row_device.h"

using namespace tmac;

namespace {

constexpr int kThreads = 256;

// Rows per workgroup: about `per` pieces (cpr of them a row) for each thread, more where the grid would
// pass 2^22 workgroups.
int rows_per_block(int64_t rows, int cpr, int per) {
  int64_t rpb = kThreads * per > cpr ? kThreads * per / cpr : 1;
  while ((rows + rpb - 1) / rpb > (1 << 22)) rpb *= 2;
  return static_cast<int>(rpb);
}

template <int DT, int N>
__global__ __launch_bounds__(kThreads) void embed_fwd_kernel(
    const int64_t* __restrict__ ids, const int64_t* __restrict__ pos, const uint8_t* __restrict__ W,
    int64_t ldw, const uint8_t* __restrict__ P, int64_t ldp, const uint8_t* __restrict__ prefix, int64_t ldpre,
    uint8_t* __restrict__ out, int rows, int T, int Np, int d, int64_t V, int64_t n_pos, float scale, int cpr,
    int rpb) {
  constexpr int E = kRowSize<DT>;
  const int row0 = blockIdx.x * rpb;
  const int n = min(rpb, rows - row0) * cpr;
  const int S = Np + T;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int r = i / cpr, c = (i - r * cpr) * N;
    const int row = row0 + r;
    const int b = row / S, s = row - b * S;
    float v[N];
    if (s < Np) {
      row_load<DT, N>(prefix + (static_cast<int64_t>(s) * ldpre + c) * E, v);
    } else {
      const int64_t tok = static_cast<int64_t>(b) * T + (s - Np);
      const int64_t id = ids[tok];
      const int64_t p = pos ? pos[tok] : s - Np;
      // an index outside its table reads nothing and gives a row of NaN
      const bool ok = id >= 0 && id < V && (!P || (p >= 0 && p < n_pos));
      if (ok) {
        row_load<DT, N>(W + (id * ldw + c) * E, v);
        float q[N];
        if (P) row_load<DT, N>(P + (p * ldp + c) * E, q);
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = P ? fmaf(scale, v[e], q[e]) : scale * v[e];
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = __builtin_nanf("");
      }
    }
    row_store<DT, N>(out + (static_cast<int64_t>(row) * d + c) * E, v);
  }
}

// ------------------------------------------------------------------ the sort

constexpr int kSortWaves = 16;
constexpr int kMaxRange = 512;  // rows of W per workgroup of the sort

__device__ __forceinline__ int wave_scan(int v, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(v, o);
    if (lane >= o) v += u;
  }
  return v;
}

// Stable counting sort of the tokens by id, without passes over digits: workgroup w owns the ids
// [w R, (w + 1) R) and reads all of them twice (they stay in L2). The first time it counts, per wave, how
// often each of its ids comes and how many ids come before its range, which is where its part of the list
// begins; the second time each wave places its tokens behind those of the waves before it.
// row_start[v]: where id v's tokens begin (row_start[V] their number); perm: the row of g of each, in
// ascending order; key: its id. An id outside [0, V) is in no list.
__global__ __launch_bounds__(64 * kSortWaves) void embed_sort_kernel(
    const int64_t* __restrict__ ids, int n_tok, int T, int Np, int V, int R, int32_t* __restrict__ row_start,
    int32_t* __restrict__ perm, int32_t* __restrict__ key) {
  __shared__ int hist[kSortWaves * kMaxRange];
  __shared__ int s_tot[kSortWaves], s_below[kSortWaves];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int lo = blockIdx.x * R, hi = min(lo + R, V);
  const int per = (n_tok + 64 * kSortWaves - 1) / (64 * kSortWaves) * 64;
  const int begin = wave * per, end = min(begin + per, n_tok);
  int* const mine = hist + wave * R;
  for (int i = tid; i < kSortWaves * R; i += 64 * kSortWaves) hist[i] = 0;
  __syncthreads();
  int below = 0;
  for (int n = begin + lane; n < end; n += 64) {
    const int64_t id = ids[n];
    if (id >= 0 && id < lo) ++below;
    if (id >= lo && id < hi) atomicAdd(mine + static_cast<int>(id - lo), 1);
  }
  below = wave_scan(below, lane);
  if (lane == 63) s_below[wave] = below;
  __syncthreads();
  int tot = 0;
  if (tid < R)
    for (int w = 0; w < kSortWaves; ++w) tot += hist[w * R + tid];
  const int inc = wave_scan(tot, lane);
  if (lane == 63) s_tot[wave] = inc;
  __syncthreads();
  int run = inc - tot;
  for (int w = 0; w < kSortWaves; ++w) run += s_below[w] + (w < wave ? s_tot[w] : 0);
  if (tid < R && lo + tid < V) {
    row_start[lo + tid] = run;
    for (int w = 0; w < kSortWaves; ++w) {
      const int c = hist[w * R + tid];
      hist[w * R + tid] = run;
      run += c;
    }
    if (lo + tid == V - 1) row_start[V] = run;
  }
  __syncthreads();
  for (int n0 = begin; n0 < end; n0 += 64) {
    const int n = n0 + lane;
    const int64_t id = n < end ? ids[n] : -1;
    const int rel = id >= lo && id < hi ? static_cast<int>(id - lo) : -1;
    // the tokens of one id at a time, in the order of the lanes
    for (uint64_t todo = __ballot(rel >= 0); todo;) {
      const int r = __builtin_amdgcn_readlane(rel, __builtin_ctzll(todo));
      const uint64_t same = __ballot(rel == r);
      int at = 0;
      if (lane == 0) at = atomicAdd(mine + r, __popcll(same));
      at = __builtin_amdgcn_readfirstlane(at);
      if (rel == r) {
        const int slot = at + __popcll(same & ((1ull << lane) - 1));
        perm[slot] = n + (n / T + 1) * Np;
        key[slot] = static_cast<int>(id);
      }
      todo &= ~same;
    }
  }
}

// ------------------------------------------------------------------ the sums

constexpr int kList = 64;  // longest list that is summed in one piece; tokens per partial row

// v += the rows perm[a .. b) of g at column c, in order
template <int DT, int N>
__device__ __forceinline__ void sum_rows(const uint8_t* __restrict__ g, int64_t ldg,
                                         const int32_t* __restrict__ perm, int a, int b, int c, float (&v)[N]) {
  constexpr int E = kRowSize<DT>, U = 4;
  for (; a + U <= b; a += U) {
    float x[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u) row_load<DT, N>(g + (perm[a + u] * ldg + c) * E, x[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] += x[u][e];
  }
  for (; a < b; ++a) {
    float x[N];
    row_load<DT, N>(g + (perm[a] * ldg + c) * E, x);
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] += x[e];
  }
}

// Workgroups [0, n_chunks): the part of each long list that lies in sorted tokens [64 j, 64 j + 64), into
// part[j][0] (the list of the first of them) and part[j][1] (of the last, if another). Long lists have more
// than 64 tokens, so no third one reaches into the chunk. The other workgroups: rpb rows of dW each.
template <int DT, int N>
__global__ __launch_bounds__(kThreads) void embed_grad_kernel(
    const uint8_t* __restrict__ g, int64_t ldg, const int32_t* __restrict__ row_start,
    const int32_t* __restrict__ perm, const int32_t* __restrict__ key, float* __restrict__ part,
    uint8_t* __restrict__ dW, int V, int d, float scale, int cpr, int rpb, int n_chunks) {
  constexpr int E = kRowSize<DT>;
  if (static_cast<int>(blockIdx.x) < n_chunks) {
    const int j = blockIdx.x, n_valid = row_start[V];
    const int a0 = kList * j, b0 = min(a0 + kList, n_valid);
    if (a0 >= b0) return;
    const int k0 = key[a0], k1 = key[b0 - 1];
    for (int which = 0; which < (k0 == k1 ? 1 : 2); ++which) {
      const int k = which ? k1 : k0;
      const int s = row_start[k], e = row_start[k + 1];
      if (e - s <= kList) continue;
      const int a = max(a0, s), b = min(b0, e);
      for (int c = threadIdx.x; c < cpr; c += kThreads) {
        float v[N] = {};
        sum_rows<DT, N>(g, ldg, perm, a, b, c * N, v);
        float* const to = part + (static_cast<int64_t>(2 * j + which) * d + c * N);
#pragma unroll
        for (int q = 0; q < N; ++q) to[q] = v[q];
      }
    }
    return;
  }
  const int row0 = (blockIdx.x - n_chunks) * rpb;
  const int n = min(rpb, V - row0) * cpr;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int r = i / cpr, c = (i - r * cpr) * N;
    const int a = row_start[row0 + r], b = row_start[row0 + r + 1];
    if (b - a > kList) continue;
    float v[N] = {};
    sum_rows<DT, N>(g, ldg, perm, a, b, c, v);
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] *= scale;
    row_store<DT, N>(dW + (static_cast<int64_t>(row0 + r) * d + c) * E, v);
  }
}

// The long list that begins in chunk j, if one does (it reaches the chunk's end, so at most one): its
// partial rows, added in order by eight groups of threads and those groups' sums in order.
template <int DT, int N>
__global__ __launch_bounds__(1024) void embed_grad_long_kernel(
    const int32_t* __restrict__ row_start, const int32_t* __restrict__ key, const float* __restrict__ part,
    uint8_t* __restrict__ dW, int V, int d, float scale, int cpr) {
  constexpr int E = kRowSize<DT>, kGroups = 8, kWide = 1024 / kGroups;
  __shared__ float sums[kGroups][kWide][N];
  const int j = blockIdx.x, n_valid = row_start[V];
  const int last = kList * j + kList - 1;  // a long list that begins here covers it
  if (last >= n_valid) return;
  const int k = key[last];
  const int s = row_start[k], e = row_start[k + 1];
  if (e - s <= kList || s < kList * j) return;
  // chunks j .. j1 hold it: in chunk j it is the last list, in the others the first
  const int j1 = (e - 1) / kList, n = j1 - j + 1, per = (n + kGroups - 1) / kGroups;
  const int grp = threadIdx.x / kWide, t = threadIdx.x % kWide;
  const int first = s == kList * j ? 0 : 1;
  for (int c0 = 0; c0 < cpr; c0 += kWide) {
    const int c = c0 + t;
    float v[N] = {};
    if (c < cpr) {
      const int end = min(n, (grp + 1) * per);
#pragma unroll 8
      for (int i = grp * per; i < end; ++i) {
        const float* from = part + (static_cast<int64_t>(2 * (j + i) + (i ? 0 : first)) * d + c * N);
#pragma unroll
        for (int q = 0; q < N; ++q) v[q] += from[q];
      }
    }
#pragma unroll
    for (int q = 0; q < N; ++q) sums[grp][t][q] = v[q];
    __syncthreads();
    if (grp == 0 && c < cpr) {
      for (int o = 1; o < kGroups; ++o)
#pragma unroll
        for (int q = 0; q < N; ++q) v[q] += sums[o][t][q];
#pragma unroll
      for (int q = 0; q < N; ++q) v[q] *= scale;
      row_store<DT, N>(dW + (static_cast<int64_t>(k) * d + c * N) * E, v);
    }
    __syncthreads();
  }
}

// Row s of [prefix | positions]: the sum over the sequences of g[b, s], zeros behind the last position.
template <int DT, int N>
__global__ __launch_bounds__(kThreads) void embed_pos_grad_kernel(
    const uint8_t* __restrict__ g, int64_t ldg, uint8_t* __restrict__ dprefix, uint8_t* __restrict__ dP, int B,
    int T, int Np, int d, int row_first, int rows, int cpr, int rpb) {
  constexpr int E = kRowSize<DT>;
  const int S = Np + T;
  const int row0 = row_first + blockIdx.x * rpb;
  const int n = min(rpb, rows - row0) * cpr;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int r = i / cpr, c = (i - r * cpr) * N;
    const int s = row0 + r;
    float v[N] = {};
    if (s < S) {
#pragma unroll 4
      for (int b = 0; b < B; ++b) {
        float x[N];
        row_load<DT, N>(g + ((static_cast<int64_t>(b) * S + s) * ldg + c) * E, x);
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] += x[e];
      }
    }
    uint8_t* const to = s < Np ? dprefix + (static_cast<int64_t>(s) * d + c) * E
                               : dP + (static_cast<int64_t>(s - Np) * d + c) * E;
    row_store<DT, N>(to, v);
  }
}

// ------------------------------------------------------------------ host

constexpr int64_t kMaxRows = 1 << 30;
constexpr int kMaxD = 1 << 20;

int check_sizes(int B, int T, int Np, int d, int dtype) {
  if (dtype != TMAC_F32 && dtype != TMAC_BF16 && dtype != TMAC_F16) return TMAC_ERR_DTYPE;
  if (B < 0 || T < 0 || Np < 0 || d <= 0 || d > kMaxD) return TMAC_ERR_SHAPE;
  if (static_cast<int64_t>(B) * (static_cast<int64_t>(Np) + T) > kMaxRows) return TMAC_ERR_SHAPE;
  return TMAC_OK;
}

int launch_status() {
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? TMAC_OK : static_cast<int>(err);
}

// f(DT, N): the type and whether 16-byte accesses apply
template <typename F>
void dispatch(int dtype, bool wide, F&& f) {
  using std::integral_constant;
  auto with = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (wide)
      f(dt, integral_constant<int, kRowVec<DT>>{});
    else
      f(dt, integral_constant<int, 1>{});
  };
  if (dtype == TMAC_F32)
    with(integral_constant<int, TMAC_F32>{});
  else if (dtype == TMAC_BF16)
    with(integral_constant<int, TMAC_BF16>{});
  else
    with(integral_constant<int, TMAC_F16>{});
}

bool wide_rows(const void* p, int64_t ld, int dtype) {
  return !p || (row_aligned16(p) && ld % (dtype == TMAC_F32 ? 4 : 8) == 0);
}

size_t up16(size_t n) { return (n + 15) & ~static_cast<size_t>(15); }

struct GradWs {
  size_t perm, key, part, total;
};
GradWs grad_ws(int64_t n_tok, int64_t V, int d) {
  GradWs w;
  w.perm = up16(4 * static_cast<size_t>(V + 1));
  w.key = w.perm + up16(4 * static_cast<size_t>(n_tok));
  w.part = w.key + up16(4 * static_cast<size_t>(n_tok));
  const size_t chunks = n_tok > kList ? static_cast<size_t>((n_tok + kList - 1) / kList) : 0;
  w.total = w.part + 8 * chunks * static_cast<size_t>(d);
  return w;
}

}  // namespace

extern "C" int tmac_embed_fwd(const int64_t* d_ids, const int64_t* d_pos, const void* d_W, int64_t ldw,
                              const void* d_P, int64_t ldp, const void* d_prefix, int64_t ldpre, void* d_out,
                              int B, int T, int n_prefix, int d, int64_t V, int64_t n_pos, float scale, int dtype,
                              void* stream) {
  const int st = check_sizes(B, T, n_prefix, d, dtype);
  if (st != TMAC_OK) return st;
  if (V <= 0 || V > kMaxRows || ldw < d) return TMAC_ERR_SHAPE;
  if (d_P && (n_pos <= 0 || n_pos > kMaxRows || ldp < d || (!d_pos && n_pos < T))) return TMAC_ERR_SHAPE;
  if (n_prefix && ldpre < d) return TMAC_ERR_SHAPE;
  const int rows = B * (n_prefix + T);
  if (rows == 0) return TMAC_OK;
  if (!d_W || !d_out || (T > 0 && !d_ids) || (n_prefix && !d_prefix)) return TMAC_ERR_NULL;
  const bool wide = d % (dtype == TMAC_F32 ? 4 : 8) == 0 && row_aligned16(d_out) && wide_rows(d_W, ldw, dtype) &&
                    wide_rows(d_P, ldp, dtype) && (!n_prefix || wide_rows(d_prefix, ldpre, dtype));
  dispatch(dtype, wide, [&](auto dt, auto n) {
    constexpr int DT = decltype(dt)::value, N = decltype(n)::value;
    const int cpr = d / N, rpb = rows_per_block(rows, cpr, 1);
    embed_fwd_kernel<DT, N><<<(rows + rpb - 1) / rpb, kThreads, 0, static_cast<hipStream_t>(stream)>>>(
        d_ids, d_pos, static_cast<const uint8_t*>(d_W), ldw, static_cast<const uint8_t*>(d_P), ldp,
        static_cast<const uint8_t*>(d_prefix), ldpre, static_cast<uint8_t*>(d_out), rows, T, n_prefix, d, V, n_pos,
        scale, cpr, rpb);
  });
  return launch_status();
}

extern "C" int tmac_embed_grad_workspace(int64_t n_tokens, int64_t V, int d, size_t* ws_bytes) {
  if (!ws_bytes) return TMAC_ERR_NULL;
  if (n_tokens < 0 || n_tokens > kMaxRows || V <= 0 || V > kMaxRows || d <= 0 || d > kMaxD) return TMAC_ERR_SHAPE;
  *ws_bytes = grad_ws(n_tokens, V, d).total;
  return TMAC_OK;
}

extern "C" int tmac_embed_grad(const int64_t* d_ids, const void* d_g, int64_t ldg, void* d_dW, void* d_ws,
                               size_t ws_bytes, int B, int T, int n_prefix, int d, int64_t V, float scale,
                               int dtype, void* stream) {
  const int st = check_sizes(B, T, n_prefix, d, dtype);
  if (st != TMAC_OK) return st;
  if (V <= 0 || V > kMaxRows || ldg < d) return TMAC_ERR_SHAPE;
  const int n_tok = B * T;
  if (!d_dW || (n_tok > 0 && (!d_ids || !d_g))) return TMAC_ERR_NULL;
  const GradWs w = grad_ws(n_tok, V, d);
  if (!d_ws || ws_bytes < w.total) return TMAC_ERR_WORKSPACE;
  if (!row_aligned16(d_ws)) return TMAC_ERR_ALIGN;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  uint8_t* const ws = static_cast<uint8_t*>(d_ws);
  int32_t* const row_start = reinterpret_cast<int32_t*>(ws);
  int32_t* const perm = reinterpret_cast<int32_t*>(ws + w.perm);
  int32_t* const key = reinterpret_cast<int32_t*>(ws + w.key);
  float* const part = reinterpret_cast<float*>(ws + w.part);
  const int n_v = static_cast<int>(V);
  const int R = max(1, min(kMaxRange, (n_v + 511) / 512));
  embed_sort_kernel<<<(n_v + R - 1) / R, 64 * kSortWaves, 0, s>>>(d_ids, n_tok, T, n_prefix, n_v, R, row_start,
                                                                  perm, key);
  const bool wide = d % (dtype == TMAC_F32 ? 4 : 8) == 0 && row_aligned16(d_dW) && wide_rows(d_g, ldg, dtype);
  dispatch(dtype, wide, [&](auto dt, auto n) {
    constexpr int DT = decltype(dt)::value, N = decltype(n)::value;
    const int cpr = d / N, rpb = rows_per_block(V, cpr, 4);
    const int chunks = n_tok > kList ? (n_tok + kList - 1) / kList : 0;
    embed_grad_kernel<DT, N><<<chunks + (n_v + rpb - 1) / rpb, kThreads, 0, s>>>(
        static_cast<const uint8_t*>(d_g), ldg, row_start, perm, key, part, static_cast<uint8_t*>(d_dW), n_v, d,
        scale, cpr, rpb, chunks);
    if (chunks)
      embed_grad_long_kernel<DT, N><<<chunks, 1024, 0, s>>>(row_start, key, part, static_cast<uint8_t*>(d_dW), n_v,
                                                           d, scale, cpr);
  });
  return launch_status();
}

extern "C" int tmac_embed_pos_grad(const void* d_g, int64_t ldg, void* d_dprefix, void* d_dP, int B, int T,
                                   int n_prefix, int d, int64_t n_pos, int dtype, void* stream) {
  const int st = check_sizes(B, T, n_prefix, d, dtype);
  if (st != TMAC_OK) return st;
  if (n_pos < 0 || n_pos > kMaxRows || ldg < d || (d_dP && n_pos < T)) return TMAC_ERR_SHAPE;
  // rows [first, last) of [prefix | positions]
  const int first = d_dprefix ? 0 : n_prefix, last = n_prefix + (d_dP ? static_cast<int>(n_pos) : 0);
  if (first >= last) return TMAC_OK;
  if (B > 0 && !d_g) return TMAC_ERR_NULL;
  const bool wide = d % (dtype == TMAC_F32 ? 4 : 8) == 0 && row_aligned16(d_dprefix) && row_aligned16(d_dP) &&
                    wide_rows(d_g, ldg, dtype);
  dispatch(dtype, wide, [&](auto dt, auto n) {
    constexpr int DT = decltype(dt)::value, N = decltype(n)::value;
    const int cpr = d / N, rpb = rows_per_block(last - first, cpr, 1);
    embed_pos_grad_kernel<DT, N><<<(last - first + rpb - 1) / rpb, kThreads, 0, static_cast<hipStream_t>(stream)>>>(
        static_cast<const uint8_t*>(d_g), ldg, static_cast<uint8_t*>(d_dprefix), static_cast<uint8_t*>(d_dP), B, T,
        n_prefix, d, first, last, cpr, rpb);
  });
  return launch_status();
}
