// Log probabilities of given tokens straight from the hidden states, for gfx950: the language model head
// (models/titanmac.py:126-128, nn.Linear without bias) and the softmax over its vocabulary in one pass that
// never stores the logits. 16-bit inputs, MFMA with fp32 accumulation, fp32 statistics.
//
//   z = X · Wᵀ,   lp = z_t − lse(z),   H = −Σ p ln p          X [M, K], W [V, K]
//
// A workgroup owns a tile of rows and walks a strip of the vocabulary. In the accumulators' layout (the
// weight as operand A, the rows as B) a lane holds 16 entries of one row, so the running maximum and sums
// (row_device.h) stay in the lane; halves and waves are joined at the strip's end, strips by a second kernel.

#include "row_device.h"

using namespace tmac;

namespace {

// 128-byte LDS rows (64 16-bit values), 16-byte chunk c of row r at c ^ ((r >> 1) & 7): the
// 16-byte operand reads of 16 consecutive rows cover the 64 banks once.
__device__ __forceinline__ int xswz(int row, int chunk) {
  return row * 64 + ((chunk ^ ((row >> 1) & 7)) << 3);
}

constexpr int kCols = 128;  // vocabulary entries per tile

struct Part {  // a strip's statistics of one row
  float m, s, h;
};

template <int DT, bool ENT, int MI>
__global__ __launch_bounds__(256, 2) void head_kernel(
    const uint16_t* __restrict__ X, int64_t ldx, const uint16_t* __restrict__ W, int64_t ldw,
    const int64_t* __restrict__ targets, int M, int V, int n_steps, int n_mt, int n_nt, int n_strips, int per_strip,
    Part* __restrict__ parts, float* __restrict__ zt, int per_xcd) {
  constexpr int kRows = 64 * MI;
  constexpr int kX = kRows * 64, kStage = kX + kCols * 64;
  __shared__ __attribute__((aligned(16))) uint16_t smem[2 * kStage];

  const int logical = xcd_logical_id(per_xcd);
  if (logical >= n_mt * n_strips) return;
  const int strip = logical / n_mt;
  const int m0 = (logical - strip * n_mt) * kRows;
  const int t0 = strip * per_strip, t1 = min(t0 + per_strip, n_nt);  // t0 < n_nt

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int l32 = lane & 31, h = lane >> 5;
  const int wm = wave & 1, wn = wave >> 1;
  const int drow = lane >> 3, dpos = lane & 7;

  // Lane L of a copy covering rows R..R+7 fills chunk position L & 7 of row R + L / 8 and fetches the
  // chunk the swizzle stores there. Rows past M and entries past V read the last valid one.
  uint32_t xoff[2 * MI];
#pragma unroll
  for (int j = 0; j < 2 * MI; ++j) {
    const int row = 16 * MI * wave + 8 * j + drow;
    xoff[j] = static_cast<uint32_t>(min(row, M - 1 - m0)) * static_cast<uint32_t>(2 * ldx) +
              16u * static_cast<uint32_t>(dpos ^ ((row >> 1) & 7));
  }
  const uint32_t lds0 = lds_offset(smem);
  const uint16_t* const xb = X + static_cast<int64_t>(m0) * ldx;
  auto issue = [&](int tile, int k, int stage) {
    const uint32_t st = lds0 + static_cast<uint32_t>(stage * kStage * 2);
    const uint16_t* const xs = xb + 64 * k;
    const uint16_t* const ws = W + static_cast<int64_t>(tile) * kCols * ldw + 64 * k;
    const int last = V - 1 - tile * kCols;
#pragma unroll
    for (int j = 0; j < 2 * MI; ++j) dma_lds16(xs, xoff[j], st + (16 * MI * wave + 8 * j) * 128);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = 32 * wave + 8 * j + drow;
      const uint32_t off = static_cast<uint32_t>(min(row, last)) * static_cast<uint32_t>(2 * ldw) +
                           16u * static_cast<uint32_t>(dpos ^ ((row >> 1) & 7));
      dma_lds16(ws, off, st + kX * 2 + (32 * wave + 8 * j) * 128);
    }
  };

  f32x16 acc[MI][2];
  Stat stat[MI];
  int target[MI];  // −1: no entry of this row is asked for
#pragma unroll
  for (int mi = 0; mi < MI; ++mi) {
    stat[mi] = stat_none();
    const int row = m0 + 32 * MI * wm + 32 * mi + l32;
    const int64_t t = targets[min(row, M - 1)];
    target[mi] = row < M && t >= 0 && t < V ? static_cast<int>(t) : -1;
#pragma unroll
    for (int ni = 0; ni < 2; ++ni) acc[mi][ni] = f32x16{};
  }

  auto read_ops = [&](u32x4(&xa)[MI], u32x4(&wf)[2], const uint16_t* st, int kk) {
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) xa[mi] = lds16(st + xswz(32 * MI * wm + 32 * mi + l32, 2 * kk + h));
#pragma unroll
    for (int ni = 0; ni < 2; ++ni) wf[ni] = lds16(st + kX + xswz(64 * wn + 32 * ni + l32, 2 * kk + h));
  };
  auto compute = [&](const uint16_t* st) {
    u32x4 xa[2][MI], wf[2][2];
    read_ops(xa[0], wf[0], st, 0);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      if (kk + 1 < 4) read_ops(xa[(kk + 1) & 1], wf[(kk + 1) & 1], st, kk + 1);
#pragma unroll
      for (int mi = 0; mi < MI; ++mi)
#pragma unroll
        for (int ni = 0; ni < 2; ++ni)
          acc[mi][ni] = Mfma<DT>::run(wf[kk & 1][ni], xa[kk & 1][mi], acc[mi][ni]);
    }
  };
  // the tile's logits into the statistics: value j of acc[mi][ni] is entry col0 + 32 ni + 8 (j / 4) + 4 h + j % 4
  auto finish = [&](int tile) {
    const int col0 = tile * kCols + 64 * wn;
    if (col0 + 64 > V) {
#pragma unroll
      for (int mi = 0; mi < MI; ++mi)
#pragma unroll
        for (int ni = 0; ni < 2; ++ni)
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (col0 + 32 * ni + 8 * (j >> 2) + 4 * h + (j & 3) >= V) acc[mi][ni][j] = -__builtin_inff();
    }
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) {
      if (__ballot(target[mi] >= col0 && target[mi] < col0 + 64)) {
#pragma unroll
        for (int ni = 0; ni < 2; ++ni)
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (col0 + 32 * ni + 8 * (j >> 2) + 4 * h + (j & 3) == target[mi])
              zt[m0 + 32 * MI * wm + 32 * mi + l32] = acc[mi][ni][j];
      }
      float m = acc[mi][0][0];
#pragma unroll
      for (int ni = 0; ni < 2; ++ni)
#pragma unroll
        for (int j = 0; j < 16; ++j) m = fmaxf(m, acc[mi][ni][j]);
      stat_raise(stat[mi], m);
#pragma unroll
      for (int ni = 0; ni < 2; ++ni) {
#pragma unroll
        for (int j = 0; j < 16; ++j) stat_add<ENT>(stat[mi], acc[mi][ni][j]);
        acc[mi][ni] = f32x16{};
      }
    }
  };

  // the steps of all the strip's tiles in one sequence, so that a tile's first copies fly during the
  // previous one's statistics
  int tile = t0, k = 0, next_tile = t0, next_k = 0, i = 0;
  auto advance = [&](int& t, int& kk) {
    if (++kk == n_steps) {
      kk = 0;
      ++t;
    }
  };
  issue(next_tile, next_k, 0);
  advance(next_tile, next_k);
  while (tile < t1) {
    // every wave's copies of this step are in LDS, and every wave is done with the step before (its reads
    // have returned), whose stage the next copies overwrite
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    ring_barrier();
    if (next_tile < t1) {
      issue(next_tile, next_k, (i + 1) & 1);
      advance(next_tile, next_k);
    }
    compute(smem + (i & 1) * kStage);
    ++i;
    if (k == n_steps - 1) finish(tile);
    advance(tile, k);
  }

  // the lane halves, then the two waves that share rows, hold parts of the same rows
  __syncthreads();
  Stat* const sh = reinterpret_cast<Stat*>(smem);
#pragma unroll
  for (int mi = 0; mi < MI; ++mi) {
    const Stat& a = stat[mi];
    stat_join(stat[mi], Stat{lane_xor<32>(a.m), lane_xor<32>(a.mu), lane_xor<32>(a.s), lane_xor<32>(a.h)});
    if (wn == 1 && h == 0) sh[32 * MI * wm + 32 * mi + l32] = stat[mi];
  }
  __syncthreads();
  if (wn == 0 && h == 0) {
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) {
      const int r = 32 * MI * wm + 32 * mi + l32;
      stat_join(stat[mi], sh[r]);
      if (m0 + r < M) parts[static_cast<int64_t>(strip) * M + m0 + r] = Part{stat[mi].m, stat[mi].s, stat[mi].h};
    }
  }
}

// One wave per row: its strips' statistics joined, and the row's results.
__global__ __launch_bounds__(256) void head_join_kernel(const Part* __restrict__ parts, const float* __restrict__ zt,
                                                        const int64_t* __restrict__ targets, int64_t ignore,
                                                        float* __restrict__ lp, float* __restrict__ ent, int M, int V,
                                                        int n_strips) {
  const int row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (row >= M) return;
  Stat a = stat_none();
  for (int p = lane; p < n_strips; p += 64) {
    const Part q = parts[static_cast<int64_t>(p) * M + row];
    stat_join(a, Stat{q.m, q.m == -__builtin_inff() ? 0.f : q.m, q.s, q.h});
  }
  stat_wave(a);
  if (lane) return;
  const float log_s = __builtin_amdgcn_logf(a.s) * kLn2;
  const int64_t t = targets[row];
  float r = __builtin_nanf("");
  if (t == ignore)
    r = 0.f;
  else if (t >= 0 && t < V)
    r = (zt[row] - a.mu) - log_s;
  lp[row] = r;
  if (ent) ent[row] = log_s - a.h / a.s;
}

// ------------------------------------------------------------------ host

struct Plan {
  int mi, n_mt, n_nt, n_strips, per_strip;
};

// Row tiles of 192, or of 64 where that leaves out empty thirds; strips so that the workgroups fill whole
// rounds of the 512 that run at once, with as few tiles in a row as that allows.
Plan plan(int M, int V) {
  Plan p;
  p.mi = M <= 64 ? 1 : 3;
  p.n_mt = (M + 64 * p.mi - 1) / (64 * p.mi);
  p.n_nt = (V + kCols - 1) / kCols;
  const int room = (1 << 22) / p.n_mt;  // workgroups of a launch
  const int most = p.n_nt < 512 ? p.n_nt < room ? p.n_nt : room : 512 < room ? 512 : room;
  int64_t best = -1;
  p.n_strips = p.per_strip = 1;
  for (int s = 1; s <= most || s == 1; ++s) {
    const int per = (p.n_nt + s - 1) / s, strips = (p.n_nt + per - 1) / per;
    const int64_t rounds = (static_cast<int64_t>(p.n_mt) * strips + 511) / 512;
    const int64_t cost = rounds * (per + 1);  // a tile's worth for a strip's start and end
    if (best < 0 || cost < best) {
      best = cost;
      p.n_strips = strips;
      p.per_strip = per;
    }
  }
  return p;
}

constexpr int64_t kMaxRows = 1 << 30, kMaxV = 1 << 28, kMaxPitch = 1 << 22;

int check(int M, int64_t V, int K, int dtype) {
  if (dtype != TMAC_BF16 && dtype != TMAC_F16) return TMAC_ERR_DTYPE;
  if (M < 0 || M > kMaxRows || V <= 0 || V > kMaxV || K <= 0 || K % 64 || K > kMaxPitch) return TMAC_ERR_SHAPE;
  return TMAC_OK;
}

size_t zt_offset(int M, const Plan& p) {
  return (sizeof(Part) * static_cast<size_t>(p.n_strips) * M + 15) & ~static_cast<size_t>(15);
}

}  // namespace

extern "C" int tmac_head_logprob_workspace(int M, int64_t V, int K, size_t* ws_bytes) {
  if (!ws_bytes) return TMAC_ERR_NULL;
  const int st = check(M, V, K, TMAC_BF16);
  if (st != TMAC_OK) return st;
  *ws_bytes = M ? zt_offset(M, plan(M, static_cast<int>(V))) + 4 * static_cast<size_t>(M) : 0;
  return TMAC_OK;
}

extern "C" int tmac_head_logprob(const void* d_X, int64_t ldx, const void* d_W, int64_t ldw, const int64_t* d_targets,
                                 int64_t ignore_index, float* d_lp, float* d_entropy, int M, int64_t V, int K,
                                 void* d_ws, size_t ws_bytes, int dtype, void* stream) {
  const int st = check(M, V, K, dtype);
  if (st != TMAC_OK) return st;
  if (M == 0) return TMAC_OK;
  if (!d_X || !d_W || !d_targets || !d_lp) return TMAC_ERR_NULL;
  if (ldx < K || ldw < K || ldx > kMaxPitch || ldw > kMaxPitch) return TMAC_ERR_SHAPE;
  if (ldx % 8 || ldw % 8 || !row_aligned16(d_X) || !row_aligned16(d_W)) return TMAC_ERR_ALIGN;
  size_t need = 0;
  tmac_head_logprob_workspace(M, V, K, &need);
  if (!d_ws || ws_bytes < need) return TMAC_ERR_WORKSPACE;
  if (!row_aligned16(d_ws)) return TMAC_ERR_ALIGN;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int v = static_cast<int>(V);
  const Plan p = plan(M, v);
  Part* const parts = static_cast<Part*>(d_ws);
  float* const zt = reinterpret_cast<float*>(static_cast<uint8_t*>(d_ws) + zt_offset(M, p));
  const int per_xcd = (p.n_mt * p.n_strips + 7) / 8;
  auto launch = [&](auto dt, auto e, auto mi) {
    head_kernel<decltype(dt)::value, decltype(e)::value, decltype(mi)::value><<<8 * per_xcd, 256, 0, s>>>(
        static_cast<const uint16_t*>(d_X), ldx, static_cast<const uint16_t*>(d_W), ldw, d_targets, M, v, K / 64,
        p.n_mt, p.n_nt, p.n_strips, p.per_strip, parts, zt, per_xcd);
  };
  auto by_rows = [&](auto dt, auto e) {
    if (p.mi == 1)
      launch(dt, e, std::integral_constant<int, 1>{});
    else
      launch(dt, e, std::integral_constant<int, 3>{});
  };
  auto by_entropy = [&](auto dt) {
    if (d_entropy)
      by_rows(dt, std::true_type{});
    else
      by_rows(dt, std::false_type{});
  };
  if (dtype == TMAC_BF16)
    by_entropy(std::integral_constant<int, TMAC_BF16>{});
  else
    by_entropy(std::integral_constant<int, TMAC_F16>{});
  head_join_kernel<<<(M + 3) / 4, 256, 0, s>>>(parts, zt, d_targets, ignore_index, d_lp, d_entropy, M, v, p.n_strips);
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? TMAC_OK : static_cast<int>(err);
}
