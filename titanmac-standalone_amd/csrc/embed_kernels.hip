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
// row of W its list of tokens; a list of up to 16 is summed where its row is written; longer ones (the
// frequent tokens: with ids that fall off as 1 / (rank + 1) over 128000, the first hundred are 39 % of a text) are
// summed 16 tokens a workgroup into fp32 partial rows that a third kernel adds in order, so one frequent token does
// not hold one workgroup. With lists of up to 64 tokens in one thread's chain of loads the sums take 54 us instead
// of 37 for 32768 tokens of 640 bf16, V = 128000.

#include "row_device.h"

using namespace tmac;

namespace {

constexpr int kThreads = 256;
constexpr int kMaxRowsPerBlock = 4 * kThreads;
constexpr int64_t kMaxItems = 1 << 30;  // threads of a launch (one takes less than 2^32); workgroups take turns beyond

// Rows per workgroup and turn: about `per` (at most 4) pieces, cpr of them a row, for each thread.
int rows_per_block(int cpr, int per) { return kThreads * per > cpr ? kThreads * per / cpr : 1; }
int grid(int64_t blocks, int threads) {
  return static_cast<int>(blocks < kMaxItems / threads ? blocks : kMaxItems / threads);
}

struct Lookup {
  const int64_t *ids, *pos;
  const uint8_t *W, *P, *prefix;
  int64_t ldw, ldp, ldpre;
  uint8_t* out;
  int rows, T, Np, d;
  int64_t V, n_pos;
  float scale;
  int cpr, rpb;
};

// One piece per thread and turn: two or four in flight measured 10 and 25 % slower (9.9 us against 10.9 and 12.8
// for 4 x 4112 rows of 640 bf16: the registers cost more waves than the loads gain).
template <int DT, int N, int NT>
__device__ __forceinline__ void lookup_rows(const Lookup& a, int64_t first, int64_t step) {
  constexpr int E = kRowSize<DT>;
  const int S = a.Np + a.T;
  for (int64_t row0 = first * a.rpb; row0 < a.rows; row0 += step * a.rpb) {
    const int n = static_cast<int>(min(static_cast<int64_t>(a.rpb), a.rows - row0)) * a.cpr;
    for (int i = threadIdx.x; i < n; i += NT) {
      const int r = i / a.cpr, c = (i - r * a.cpr) * N;
      const int row = static_cast<int>(row0) + r;
      const int b = row / S, s = row - b * S;
      float v[N];
      if (s < a.Np) {
        row_load<DT, N>(a.prefix + (s * a.ldpre + c) * E, v);
      } else {
        const int64_t tok = static_cast<int64_t>(b) * a.T + (s - a.Np);
        const int64_t id = a.ids[tok];
        const int64_t p = a.pos ? a.pos[tok] : s - a.Np;
        // an index outside its table reads nothing and gives a row of NaN
        if (id >= 0 && id < a.V && (!a.P || (p >= 0 && p < a.n_pos))) {
          float q[N];
          row_load<DT, N>(a.W + (id * a.ldw + c) * E, v);
          if (a.P) row_load<DT, N>(a.P + (p * a.ldp + c) * E, q);
#pragma unroll
          for (int e = 0; e < N; ++e) v[e] = a.P ? fmaf(a.scale, v[e], q[e]) : a.scale * v[e];
        } else {
#pragma unroll
          for (int e = 0; e < N; ++e) v[e] = __builtin_nanf("");
        }
      }
      row_store<DT, N>(a.out + (static_cast<int64_t>(row) * a.d + c) * E, v);
    }
  }
}

template <int DT, int N>
__global__ __launch_bounds__(kThreads) void embed_fwd_kernel(Lookup a) {
  lookup_rows<DT, N, kThreads>(a, blockIdx.x, gridDim.x);
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

// The ids of a workgroup of the sort: [0, 8), then eight ranges to an octave up to 8192, then 512 each.
// A narrow range is cheap where every batch of ids has some in it: the ids' bits are what the placing below counts
// instructions by. The narrow ones lie low because tables made by frequency have their frequent ids there; where they
// lie elsewhere it costs time only (8 x 4096 tokens of 640 bf16, V = 128000, the ids permuted: lookup and lists 42 us
// for 36, sums 44 for 37).
struct IdRange {
  int lo, n;
};
__host__ __device__ inline IdRange id_range(int block) {
  if (block == 0) return IdRange{0, 8};
  const int o = (block - 1) >> 3, i = (block - 1) & 7;
  if (o <= 9) return IdRange{(8 + i) << o, 1 << o};
  return IdRange{(1 << 13) + (block - 81) * kMaxRange, kMaxRange};
}
int n_ranges(int64_t V) {
  if (V > (1 << 13)) return static_cast<int>(81 + (V - (1 << 13) + kMaxRange - 1) / kMaxRange);
  int n = 1;
  while (id_range(n).lo < V) ++n;
  return n;
}

// Stable counting sort of the tokens by id, without passes over digits: each workgroup owns a range of
// ids and reads all of them twice (they stay in L2). The first time it counts, per wave, how
// often each of its ids comes and how many ids come before its range, which is where its part of the list
// begins; the second time each wave places its tokens behind those of the waves before it.
// row_start[v]: where id v's tokens begin (row_start[V] their number); perm: the row of g of each, in
// ascending order; key: its id. An id outside [0, V) is in no list.
struct Lists {
  int32_t *row_start, *perm, *key;
};
struct Tokens {
  const int64_t* ids;
  int n;
  int T;
  uint32_t T_inv;  // 2^32 / T
  int Np, V;
};

// HELD: batches of 64 ids that a wave keeps in registers between the two readings (all it has), or 0.
template <int HELD>
__device__ __forceinline__ void sort_range(const Tokens& a, const Lists& to, int block) {
  const int64_t* const __restrict__ ids = a.ids;
  const int n_tok = a.n, T = a.T, Np = a.Np, V = a.V;
  const uint32_t T_inv = a.T_inv;
  int32_t *const row_start = to.row_start, *const perm = to.perm, *const key = to.key;
  __shared__ int hist[kSortWaves * kMaxRange];
  __shared__ int s_tot[kSortWaves], s_below[kSortWaves];
  constexpr int kAhead = HELD ? HELD : 8, kLoads = kAhead < 8 ? kAhead : 8;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const IdRange range = id_range(block);
  const int lo = range.lo, R = min(range.n, V - lo);  // lo < V
  const int per = (n_tok + 64 * kSortWaves - 1) / (64 * kSortWaves) * 64;
  const int begin = wave * per, end = min(begin + per, n_tok);
  int* const mine = hist + wave * R;
  for (int i = tid; i < kSortWaves * R; i += 64 * kSortWaves) hist[i] = 0;
  // this lane's part of kAhead batches of ids from n0 on, relative to the range: −1 outside it
  int below = 0;
  int rel[kAhead];
  auto load = [&](int n0, bool count) {
#pragma unroll
    for (int u0 = 0; u0 < kAhead; u0 += kLoads) {
      int64_t id[kLoads];
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        const int n = n0 + 64 * (u0 + u) + lane;
        id[u] = n < end ? ids[n] : -1;
      }
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        // ids of 2^32 and more, and negative ones, to the largest unsigned value
        const uint32_t x = static_cast<uint64_t>(id[u]) >> 32 ? ~0u : static_cast<uint32_t>(id[u]);
        if (count) below += x < static_cast<uint32_t>(lo);
        const uint32_t r = x - static_cast<uint32_t>(lo);
        rel[u0 + u] = x != ~0u && r < static_cast<uint32_t>(R) ? static_cast<int>(r) : -1;
      }
    }
  };
  __syncthreads();
  for (int n0 = begin; n0 < end; n0 += 64 * kAhead) {
    load(n0, true);
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (rel[u] >= 0) atomicAdd(mine + rel[u], 1);
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
  if (tid < R) {
    row_start[lo + tid] = run;
    for (int w = 0; w < kSortWaves; ++w) {
      const int c = hist[w * R + tid];
      hist[w * R + tid] = run;
      run += c;
    }
    if (lo + tid == V - 1) row_start[V] = run;
  }
  __syncthreads();
  const int bits = 32 - __builtin_clz(R);
  for (int n0 = begin; n0 < end; n0 += 64 * kAhead) {
    if (!HELD) load(n0, false);  // HELD: there is one turn, and they are still here
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const bool in = rel[u] >= 0;
      uint64_t same = __ballot(in);
      if (!same) continue;
      // the lanes with this lane's id; the first of them takes the places for all
      uint32_t lo32 = static_cast<uint32_t>(same), hi32 = static_cast<uint32_t>(same >> 32);
      for (int b = 0; b < bits; ++b) {
        const uint32_t bit = rel[u] >> b & 1;
        const uint64_t set = __ballot(bit);
        lo32 &= ~(static_cast<uint32_t>(set) ^ (0u - bit));
        hi32 &= ~(static_cast<uint32_t>(set >> 32) ^ (0u - bit));
      }
      same = static_cast<uint64_t>(hi32) << 32 | lo32;
      const int n = n0 + 64 * u + lane, lead = in ? __builtin_ctzll(same) : lane;
      int at = 0;
      if (in && lane == lead) at = atomicAdd(mine + rel[u], __popcll(same));
      at = __shfl(at, lead);
      if (in) {
        const int slot = at + __popcll(same & ((1ull << lane) - 1));
        int b = T > 1 ? static_cast<int>(__umulhi(static_cast<uint32_t>(n), T_inv)) : n;  // n / T, or one less
        if (T > 1 && n - b * T >= T) ++b;
        perm[slot] = n + (b + 1) * Np;
        key[slot] = lo + rel[u];
      }
    }
  }
}

template <int HELD>
__global__ __launch_bounds__(64 * kSortWaves, 8) void embed_sort_kernel(Tokens t, Lists to) {
  sort_range<HELD>(t, to, blockIdx.x);
}

// The lookup of a training step and its tokens' lists in one launch: the sort waits for LDS and L2 most of its
// time, the lookup for memory.
template <int DT, int N, int HELD>
__global__ __launch_bounds__(64 * kSortWaves, 8) void embed_fwd_lists_kernel(Lookup a, Tokens t, Lists to,
                                                                            int sort_blocks) {
  const int b = blockIdx.x;
  if (b < sort_blocks)
    sort_range<HELD>(t, to, b);
  else
    lookup_rows<DT, N, 64 * kSortWaves>(a, b - sort_blocks, gridDim.x - sort_blocks);
}

// ------------------------------------------------------------------ the sums

constexpr int kList = 16;  // longest list that is summed in one piece; tokens per partial row

// v += the rows perm[a .. b) of g at column c, in order
template <int DT, int N>
__device__ __forceinline__ void sum_rows(const uint8_t* __restrict__ g, int64_t ldg,
                                         const int32_t* __restrict__ perm, int a, int b, int c, float (&v)[N]) {
  constexpr int E = kRowSize<DT>, U = 8;
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

// What one launch of the gradients covers.
struct Grad {
  const uint8_t* g;  // rows of pitch ldg
  int64_t ldg;
  const int32_t *row_start, *perm, *key;  // the sorted lists
  float* part;
  uint8_t* dW;  // [V, d] by sorted tokens
  int V, rpb, chunks, row_blocks;
  float scale;
  uint8_t *dprefix, *dP;  // rows [first, last) of [prefix | positions] by sums over the sequences
  int B, T, Np;
  uint32_t first, last;  // up to 2^31
  int pos_blocks, pos_rpb;
  int runs, run_first, run_pieces, run_blocks;  // and the pieces of rows [run_first, first) by runs of the sequences
  int d, cpr;
};

// The part of each long list that lies in sorted tokens [16 j, 16 j + 16), into part[j][0] (the list of the
// first of them) and part[j][1] (of the last, if another). Long lists have more than 16 tokens, so no third
// one reaches into the chunk.
template <int DT, int N>
__device__ __forceinline__ void grad_chunk(const Grad& a, int j) {
  const int n_valid = a.row_start[a.V];
  const int a0 = kList * j, b0 = min(a0 + kList, n_valid);
  if (a0 >= b0) return;
  const int k0 = a.key[a0], k1 = a.key[b0 - 1];
  for (int which = 0; which < (k0 == k1 ? 1 : 2); ++which) {
    const int k = which ? k1 : k0;
    const int s = a.row_start[k], e = a.row_start[k + 1];
    if (e - s <= kList) continue;
    for (int c = threadIdx.x; c < a.cpr; c += kThreads) {
      float v[N] = {};
      sum_rows<DT, N>(a.g, a.ldg, a.perm, max(a0, s), min(b0, e), c * N, v);
      float* const to = a.part + (static_cast<int64_t>(2 * j + which) * a.d + c * N);
#pragma unroll
      for (int q = 0; q < N; ++q) to[q] = v[q];
    }
  }
}

// rpb rows of dW: their lists' ends first, so that the rows without a token (most of a large table) are
// stores and nothing else.
template <int DT, int N>
__device__ __forceinline__ void grad_rows(const Grad& a, int block) {
  constexpr int E = kRowSize<DT>;
  __shared__ int s_start[kMaxRowsPerBlock + 1];
  const int row0 = block * a.rpb, rows = min(a.rpb, a.V - row0), n = rows * a.cpr;
  for (int i = threadIdx.x; i <= rows; i += kThreads) s_start[i] = a.row_start[row0 + i];
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int r = i / a.cpr, c = (i - r * a.cpr) * N;
    const int p = s_start[r], q = s_start[r + 1];
    if (q - p > kList) continue;
    float v[N] = {};
    sum_rows<DT, N>(a.g, a.ldg, a.perm, p, q, c, v);
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] *= a.scale;
    row_store<DT, N>(a.dW + (static_cast<int64_t>(row0 + r) * a.d + c) * E, v);
  }
  __syncthreads();
}

// Rows s of [prefix | positions]: the sum over the sequences of g[b, s], one thread a piece, zeros behind the last
// position.
template <int DT, int N>
__device__ __forceinline__ void grad_positions(const Grad& a, int block) {
  constexpr int E = kRowSize<DT>;
  const uint32_t S = a.Np + a.T, row0 = a.first + static_cast<uint32_t>(block) * a.pos_rpb;
  const int n = static_cast<int>(min(static_cast<uint32_t>(a.pos_rpb), a.last - row0)) * a.cpr;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int r = i / a.cpr, c = (i - r * a.cpr) * N;
    const uint32_t s = row0 + r;
    float v[N] = {};
    if (s < S) {
#pragma unroll 4
      for (int b = 0; b < a.B; ++b) {
        float x[N];
        row_load<DT, N>(a.g + ((static_cast<int64_t>(b) * S + s) * a.ldg + c) * E, x);
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] += x[e];
      }
    }
    row_store<DT, N>(s < static_cast<uint32_t>(a.Np) ? a.dprefix + (static_cast<int64_t>(s) * a.d + c) * E
                                                     : a.dP + (static_cast<int64_t>(s - a.Np) * a.d + c) * E,
                     v);
  }
}

// The same for pieces of rows that are too few to fill the card with one thread each, of many sequences: a.runs
// threads sum equal runs of the sequences, and their sums are added in pairs (a fixed order). Training passes in us,
// against one thread for all sequences, whose loads wait for one another: 5000 x 3 tokens and 4 prefix rows of 640 bf16
// 92 (562), 4096 x 16 and 16 of 640 245 (774), 20000 x 1 of 64 66 (1185), with 4 prefix rows 75 (1888).
template <int DT, int N>
__device__ __forceinline__ void grad_runs(const Grad& a, int block) {
  constexpr int E = kRowSize<DT>, U = 8;
  __shared__ float sums[N][kThreads];
  const int S = a.Np + a.T, wide = kThreads / a.runs, tid = threadIdx.x;
  const int run = tid / wide, piece = block * wide + (tid - run * wide);
  const bool in = piece < a.run_pieces;
  const int r = piece / a.cpr, c = (piece - r * a.cpr) * N, s = a.run_first + r;
  float v[N] = {};
  if (in) {
    const int per = (a.B + a.runs - 1) / a.runs, end = min(a.B, (run + 1) * per);
    auto row = [&](int b) { return a.g + ((static_cast<int64_t>(b) * S + s) * a.ldg + c) * E; };
    int b = run * per;
    for (; b + U <= end; b += U) {
      float x[U][N];
#pragma unroll
      for (int u = 0; u < U; ++u) row_load<DT, N>(row(b + u), x[u]);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] += x[u][e];
    }
    for (; b < end; ++b) {
      float x[N];
      row_load<DT, N>(row(b), x);
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] += x[e];
    }
  }
  for (int o = a.runs / 2; o > 0; o /= 2) {
#pragma unroll
    for (int e = 0; e < N; ++e) sums[e][tid] = v[e];
    __syncthreads();
    if (run < o) {
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] += sums[e][tid + o * wide];
    }
    __syncthreads();
  }
  if (in && run == 0)
    row_store<DT, N>(s < a.Np ? a.dprefix + (static_cast<int64_t>(s) * a.d + c) * E
                              : a.dP + (static_cast<int64_t>(s - a.Np) * a.d + c) * E,
                     v);
}

// The chunks of long lists first, whose sums the next launch waits for. RUNS: whether a.run_blocks is not 0, which
// takes registers and LDS that every other launch is better without (8 x 4096 tokens of 640 bf16 36.7 us, 40.6 with).
template <int DT, int N, bool RUNS>
__global__ __launch_bounds__(kThreads) void embed_grad_kernel(Grad a) {
  // up to 2^26, 2^19, 2^31 and 2^30
  const uint32_t chunks = a.chunks, runs = chunks + (RUNS ? a.run_blocks : 0), sums = runs + a.pos_blocks;
  const uint32_t blocks = sums + a.row_blocks;
  for (uint32_t b = blockIdx.x; b < blocks; b += gridDim.x) {
    if (b < chunks) {
      grad_chunk<DT, N>(a, static_cast<int>(b));
      continue;
    }
    if constexpr (RUNS) {
      if (b < runs) {
        grad_runs<DT, N>(a, static_cast<int>(b - chunks));
        continue;
      }
    }
    if (b < sums)
      grad_positions<DT, N>(a, static_cast<int>(b - runs));
    else
      grad_rows<DT, N>(a, static_cast<int>(b - sums));
  }
}

// The long lists that begin in this workgroup's chunks (one reaches its chunk's end, so there is at most one a
// chunk): their partial rows, added in order by eight groups of threads and those groups' sums in order.
constexpr int kLongChunks = 8;

template <int DT, int N>
__global__ __launch_bounds__(1024) void embed_grad_long_kernel(Grad a) {
  constexpr int E = kRowSize<DT>, kGroups = 8, kWide = 1024 / kGroups;
  __shared__ float sums[kGroups][kWide][N];
  __shared__ int s_key[kLongChunks];
  for (int base = blockIdx.x * kLongChunks; base < a.chunks; base += gridDim.x * kLongChunks) {
    if (threadIdx.x < kLongChunks) {
      const int j = base + threadIdx.x, last = kList * j + kList - 1;  // the entry that such a list covers
      int k = -1;
      if (last < a.row_start[a.V]) {
        k = a.key[last];
        const int s = a.row_start[k], e = a.row_start[k + 1];
        if (e - s <= kList || s < kList * j) k = -1;
      }
      s_key[threadIdx.x] = k;
    }
    __syncthreads();
    for (int i0 = 0; i0 < kLongChunks; ++i0) {
      const int j = base + i0, k = s_key[i0];
      if (k < 0) continue;
      // chunks j .. j1 hold it: in chunk j it is the last list, in the others the first
      const int s = a.row_start[k], e = a.row_start[k + 1];
      const int j1 = (e - 1) / kList, n = j1 - j + 1, per = (n + kGroups - 1) / kGroups;
      const int grp = threadIdx.x / kWide, t = threadIdx.x % kWide;
      const int first = s == kList * j ? 0 : 1;
      for (int c0 = 0; c0 < a.cpr; c0 += kWide) {
        const int c = c0 + t;
        float v[N] = {};
        if (c < a.cpr) {
          const int end = min(n, (grp + 1) * per);
#pragma unroll 8
          for (int i = grp * per; i < end; ++i) {
            const float* from = a.part + (static_cast<int64_t>(2 * (j + i) + (i ? 0 : first)) * a.d + c * N);
#pragma unroll
            for (int q = 0; q < N; ++q) v[q] += from[q];
          }
        }
#pragma unroll
        for (int q = 0; q < N; ++q) sums[grp][t][q] = v[q];
        __syncthreads();
        if (grp == 0 && c < a.cpr) {
          for (int o = 1; o < kGroups; ++o)
#pragma unroll
            for (int q = 0; q < N; ++q) v[q] += sums[o][t][q];
#pragma unroll
          for (int q = 0; q < N; ++q) v[q] *= a.scale;
          row_store<DT, N>(a.dW + (static_cast<int64_t>(k) * a.d + c * N) * E, v);
        }
        __syncthreads();
      }
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------ host

constexpr int64_t kMaxRows = 1 << 30;
constexpr int kMaxD = 1 << 20;

int check_sizes(int B, int T, int Np, int d, int dtype) {
  if (dtype != TMAC_F32 && dtype != TMAC_BF16 && dtype != TMAC_F16) return TMAC_ERR_DTYPE;
  if (B < 0 || T < 0 || Np < 0 || Np > kMaxRows || d <= 0 || d > kMaxD) return TMAC_ERR_SHAPE;
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

// Runs of B sequences that `pieces` pieces of rows are summed in: a power of two, no more than fill the card (2^19
// threads) and of at least 8 sequences, one turn of loads; 1: one thread a piece, whose sums hide beside the other
// table's up to some sequences. us of the gradients with one thread and with runs: 128 x 128 tokens of 640 bf16 29 / 33,
// 128 x 16 of 256 16.2 / 16.3, 256 x 64 of 640 41 / 34, 512 x 128 81 / 57, 2000 x 64 270 / 137.
constexpr int kManySequences = 256;
int n_runs(int B, int64_t pieces) {
  int n = 1;
  if (B < kManySequences) return n;
  while (2 * n <= kThreads && 2 * n * pieces <= 1 << 19 && B / (2 * n) >= 8) n *= 2;
  return n;
}

bool wide_rows(const void* p, int64_t ld, int dtype) {
  return !p || (row_aligned16(p) && ld % (dtype == TMAC_F32 ? 4 : 8) == 0);
}

size_t up16(size_t n) { return (n + 15) & ~static_cast<size_t>(15); }

struct ListsAt {
  size_t perm, key, total;
};
ListsAt lists_at(int64_t n_tok, int64_t V) {
  ListsAt w;
  w.perm = up16(4 * static_cast<size_t>(V + 1));
  w.key = w.perm + up16(4 * static_cast<size_t>(n_tok));
  w.total = w.key + up16(4 * static_cast<size_t>(n_tok));
  return w;
}
Lists lists(void* at, int64_t n_tok, int64_t V) {
  const ListsAt w = lists_at(n_tok, V);
  uint8_t* const p = static_cast<uint8_t*>(at);
  return Lists{reinterpret_cast<int32_t*>(p), reinterpret_cast<int32_t*>(p + w.perm),
               reinterpret_cast<int32_t*>(p + w.key)};
}
size_t part_bytes(int64_t n_tok, int d) {
  return n_tok > kList ? 8 * static_cast<size_t>((n_tok + kList - 1) / kList) * static_cast<size_t>(d) : 0;
}
Tokens tokens(const int64_t* ids, int n_tok, int T, int n_prefix, int64_t V) {
  return Tokens{ids, n_tok, T, T > 1 ? static_cast<uint32_t>((1ull << 32) / static_cast<uint32_t>(T)) : 0, n_prefix,
                static_cast<int>(V)};
}
constexpr int kHeld = 4;  // batches that the sort of few tokens keeps in registers
bool held(int n_tok) { return n_tok <= kHeld * 64 * kSortWaves; }

}  // namespace

extern "C" int tmac_embed_lists_bytes(int64_t n_tokens, int64_t V, size_t* bytes) {
  if (!bytes) return TMAC_ERR_NULL;
  if (n_tokens < 0 || n_tokens > kMaxRows || V <= 0 || V > kMaxRows) return TMAC_ERR_SHAPE;
  *bytes = lists_at(n_tokens, V).total;
  return TMAC_OK;
}

extern "C" int tmac_embed_fwd(const int64_t* d_ids, const int64_t* d_pos, const void* d_W, int64_t ldw,
                              const void* d_P, int64_t ldp, const void* d_prefix, int64_t ldpre, void* d_out,
                              void* d_lists, size_t lists_bytes, int B, int T, int n_prefix, int d, int64_t V,
                              int64_t n_pos, float scale, int dtype, void* stream) {
  const int st = check_sizes(B, T, n_prefix, d, dtype);
  if (st != TMAC_OK) return st;
  if (V <= 0 || V > kMaxRows || ldw < d) return TMAC_ERR_SHAPE;
  if (d_P && (n_pos <= 0 || n_pos > kMaxRows || ldp < d || (!d_pos && n_pos < T))) return TMAC_ERR_SHAPE;
  if (n_prefix && ldpre < d) return TMAC_ERR_SHAPE;
  const int rows = B * (n_prefix + T), n_tok = B * T;
  if (d_lists && lists_bytes < lists_at(n_tok, V).total) return TMAC_ERR_WORKSPACE;
  if (d_lists && !row_aligned16(d_lists)) return TMAC_ERR_ALIGN;
  if (rows == 0 && !d_lists) return TMAC_OK;
  if ((rows && (!d_W || !d_out)) || (n_tok > 0 && !d_ids) || (B > 0 && n_prefix && !d_prefix)) return TMAC_ERR_NULL;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const bool wide = d % (dtype == TMAC_F32 ? 4 : 8) == 0 && row_aligned16(d_out) && wide_rows(d_W, ldw, dtype) &&
                    wide_rows(d_P, ldp, dtype) && (!n_prefix || wide_rows(d_prefix, ldpre, dtype));
  dispatch(dtype, wide, [&](auto dt, auto n) {
    constexpr int DT = decltype(dt)::value, N = decltype(n)::value;
    Lookup a{d_ids, d_pos, static_cast<const uint8_t*>(d_W), static_cast<const uint8_t*>(d_P),
             static_cast<const uint8_t*>(d_prefix), ldw, ldp, ldpre, static_cast<uint8_t*>(d_out), rows, T, n_prefix, d,
             V, n_pos, scale, d / N, 1};
    if (!d_lists) {
      a.rpb = rows_per_block(a.cpr, 1);
      embed_fwd_kernel<DT, N><<<grid((rows + a.rpb - 1) / a.rpb, kThreads), kThreads, 0, s>>>(a);
      return;
    }
    a.rpb = rows_per_block(a.cpr, 64 * kSortWaves / kThreads);
    const Tokens t = tokens(d_ids, n_tok, T, n_prefix, V);
    const Lists to = lists(d_lists, n_tok, V);
    const int sort_blocks = n_ranges(V);  // up to 2^21: with the others' 2^20, 3 · 2^30 threads
    const int blocks = sort_blocks + grid((rows + a.rpb - 1) / a.rpb, 64 * kSortWaves);
    if (held(n_tok))
      embed_fwd_lists_kernel<DT, N, kHeld><<<blocks, 64 * kSortWaves, 0, s>>>(a, t, to, sort_blocks);
    else
      embed_fwd_lists_kernel<DT, N, 0><<<blocks, 64 * kSortWaves, 0, s>>>(a, t, to, sort_blocks);
  });
  return launch_status();
}

extern "C" int tmac_embed_bwd_workspace(int64_t n_tokens, int64_t V, int64_t n_pos, int d, size_t* ws_bytes) {
  if (!ws_bytes) return TMAC_ERR_NULL;
  if (n_tokens < 0 || n_tokens > kMaxRows || V < 0 || V > kMaxRows || n_pos < 0 || n_pos > kMaxRows || d <= 0 ||
      d > kMaxD)
    return TMAC_ERR_SHAPE;
  // one list at a time: the two sorts take turns
  *ws_bytes = lists_at(n_tokens, V > n_pos ? V : n_pos).total + part_bytes(n_tokens, d);
  return TMAC_OK;
}

extern "C" int tmac_embed_bwd(const int64_t* d_ids, const int64_t* d_pos, const void* d_lists, const void* d_g,
                              int64_t ldg, void* d_dW, void* d_dP, void* d_dprefix, void* d_ws, size_t ws_bytes, int B,
                              int T, int n_prefix, int d, int64_t V, int64_t n_pos, float scale, int dtype,
                              void* stream) {
  const int st = check_sizes(B, T, n_prefix, d, dtype);
  if (st != TMAC_OK) return st;
  const bool sums = d_dP && !d_pos;  // positions 0 .. T - 1: plain sums, no sort
  if (ldg < d || (d_dW && (V <= 0 || V > kMaxRows)) || (d_dP && (n_pos <= 0 || n_pos > kMaxRows)) ||
      (sums && n_pos < T) || (d_dprefix && !n_prefix))
    return TMAC_ERR_SHAPE;
  const int n_tok = B * T;
  if ((n_tok > 0 || (B > 0 && d_dprefix)) && !d_g) return TMAC_ERR_NULL;
  if (d_dW && n_tok > 0 && !d_ids && !d_lists) return TMAC_ERR_NULL;
  if (d_lists && !row_aligned16(d_lists)) return TMAC_ERR_ALIGN;
  const int64_t v_sort = d_dW && !d_lists ? V : 0, p_sort = d_dP && d_pos ? n_pos : 0;
  size_t need = 0;
  if (d_dW || p_sort) tmac_embed_bwd_workspace(n_tok, v_sort, p_sort, d, &need);
  if (need && (!d_ws || ws_bytes < need)) return TMAC_ERR_WORKSPACE;
  if (need && !row_aligned16(d_ws)) return TMAC_ERR_ALIGN;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const bool wide = d % (dtype == TMAC_F32 ? 4 : 8) == 0 && row_aligned16(d_dW) && row_aligned16(d_dP) &&
                    row_aligned16(d_dprefix) && wide_rows(d_g, ldg, dtype);
  const size_t part_at = lists_at(n_tok, v_sort > p_sort ? v_sort : p_sort).total;

  // the gradient `out` of a table by sorted tokens (its lists given, or made of `index`), the sums beside it
  auto part = [&](const int64_t* index, const void* given, void* out, int64_t n_rows, float factor, bool with_sums) {
    Grad a{};
    a.g = static_cast<const uint8_t*>(d_g);
    a.ldg = ldg;
    a.d = d;
    a.B = B;
    a.T = T;
    a.Np = n_prefix;
    if (with_sums) {
      a.dprefix = static_cast<uint8_t*>(d_dprefix);
      a.dP = sums ? static_cast<uint8_t*>(d_dP) : nullptr;
      a.first = d_dprefix ? 0 : n_prefix;
      a.last = static_cast<uint32_t>(n_prefix) + static_cast<uint32_t>(sums ? n_pos : 0);
    }
    if (out) {
      const Lists to = lists(given ? const_cast<void*>(given) : d_ws, n_tok, n_rows);
      a.row_start = to.row_start;
      a.perm = to.perm;
      a.key = to.key;
      a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(d_ws) + part_at);
      a.dW = static_cast<uint8_t*>(out);
      a.V = static_cast<int>(n_rows);
      a.scale = factor;
      a.chunks = n_tok > kList ? (n_tok + kList - 1) / kList : 0;
      if (!given) {
        const Tokens t = tokens(index, n_tok, T, n_prefix, n_rows);
        if (held(n_tok))
          embed_sort_kernel<kHeld><<<n_ranges(n_rows), 64 * kSortWaves, 0, s>>>(t, to);
        else
          embed_sort_kernel<0><<<n_ranges(n_rows), 64 * kSortWaves, 0, s>>>(t, to);
      }
    }
    dispatch(dtype, wide, [&](auto dt, auto n) {
      constexpr int DT = decltype(dt)::value, N = decltype(n)::value;
      a.cpr = d / N;
      a.rpb = rows_per_block(a.cpr, 4);
      a.pos_rpb = rows_per_block(a.cpr, 1);
      a.row_blocks = (a.V + a.rpb - 1) / a.rpb;
      // the rows that have a sum; behind them only the positions' rows of zeros
      const int64_t S = static_cast<int64_t>(n_prefix) + T, summed = (a.last < S ? a.last : S) - a.first;
      a.runs = summed > 0 ? n_runs(B, summed * a.cpr) : 1;
      if (a.runs > 1) {
        a.run_first = static_cast<int>(a.first);
        a.run_pieces = static_cast<int>(summed * a.cpr);
        a.run_blocks = (a.run_pieces + kThreads / a.runs - 1) / (kThreads / a.runs);
        a.first += static_cast<uint32_t>(summed);
      }
      a.pos_blocks = static_cast<int>((static_cast<int64_t>(a.last) - a.first + a.pos_rpb - 1) / a.pos_rpb);
      const int64_t blocks = static_cast<int64_t>(a.chunks) + a.run_blocks + a.pos_blocks + a.row_blocks;
      if (!blocks) return;
      if (a.run_blocks)
        embed_grad_kernel<DT, N, true><<<grid(blocks, kThreads), kThreads, 0, s>>>(a);
      else
        embed_grad_kernel<DT, N, false><<<grid(blocks, kThreads), kThreads, 0, s>>>(a);
      if (a.chunks)
        embed_grad_long_kernel<DT, N><<<grid((a.chunks + kLongChunks - 1) / kLongChunks, 1024), 1024, 0, s>>>(a);
    });
  };
  const bool any_sums = sums || d_dprefix;
  if (d_dW)
    part(d_ids, d_lists, d_dW, V, scale, any_sums);
  else if (any_sums)
    part(nullptr, nullptr, nullptr, 0, 1.f, true);
  if (p_sort) part(d_pos, nullptr, d_dP, n_pos, 1.f, false);
  return launch_status();
}
