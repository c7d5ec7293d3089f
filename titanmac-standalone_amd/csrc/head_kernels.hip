// Log probabilities of given tokens straight from the hidden states, for gfx950: the language model head
// (models/titanmac.py:126-128, nn.Linear without bias) and the softmax over its vocabulary in one pass that
// never stores the logits. 16-bit inputs, MFMA with fp32 accumulation, fp32 statistics.
//
//   z = X · Wᵀ,   lp = z_t − lse(z),   H = −Σ p ln p          X [M, K], W [V, K]
//
// A workgroup owns a tile of rows and walks a strip of the vocabulary. In the accumulators' layout (the
// weight as operand A, the rows as B) a lane holds 16 entries of one row, so the running maximum and sums
// (row_device.h) stay in the lane; halves and waves are joined at the strip's end, strips by a second kernel.
//
// head_kernel takes any K and any rows: 192 x 128 tiles (64 x 128 for up to 64 rows) of both operands through
// two LDS stages of 64-wide steps, two workgroups per CU. Few rows are bound by reading W: 16 rows of 640 x 128000
// 25 us (6.5 TB/s). Many are bound by the copies into LDS, 53 bytes per clock and CU of about 54: 0.99 PFLOP/s at
// 1503 x 1024 x 50001. head_rows_kernel keeps the rows in registers instead.

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

// The same for rows enough to fill its tiles and K = 64 KS of up to 640: a wave keeps its 64 rows of X in registers
// as MFMA operands for the whole strip (2 K / 4 of them), so only the weight passes through LDS: 32 entries at a
// time, each 1 KB operand read feeding two MFMAs. Per CU that is 64 bytes per clock of LDS reads and 16 of copies
// at the full MFMA rate, where the kernel above needs 107 of 128 and 53 of 54. One wave per SIMD, so the statistics
// of one tile (a third of its MFMAs' time on the vector ALU) run beside the MFMAs of the next, a few instructions
// after each, and so do the copies. Four LDS stages; copies are two tiles ahead; the barrier that hands a stage
// over stands in the middle of the tile before, away from the first use.
// SPLIT = 2, for K = 128 KS of 768 and 1024: two waves share 64 rows, each with half of K in its registers, and
// exchange products through LDS so that each finishes 32 of the rows; a tile comes in two units, of half of both
// halves. 1503 x 1024 x 50001 fp16 with entropy 154 us, 159 with 32 rows of all of K a wave (an operand read for
// each MFMA: 128 bytes per clock of LDS); 8192 x 1024 x 32000 454 and 468.
// 8192 x 640 x 128000 bf16: 1047 us (1.28 PFLOP/s; the library's product of large squares 1.37), 1434 with the
// kernel above; with all copies at once after the barrier 1076; with the statistics left to the compiler's
// schedule, which puts them behind the MFMAs, 1119.
constexpr int kTile = 32, kStages = 4;
constexpr int kAhead = 2;  // k-steps that a weight operand is read ahead of its MFMAs (of 4 registers' turns)

template <int DT, bool ENT, int KS, int SPLIT>
__global__ __launch_bounds__(256, 1) void head_rows_kernel(
    const uint16_t* __restrict__ X, int64_t ldx, const uint16_t* __restrict__ W, int64_t ldw,
    const int64_t* __restrict__ targets, int M, int V, int n_mt, int n_nt, int n_strips, int per_strip,
    Part* __restrict__ parts, float* __restrict__ zt, int per_xcd) {
  // a wave's k-steps of 16 of a unit and of a tile; elements of a 64-wide slab and of a unit
  constexpr int kK = 4 * KS / SPLIT, kAll = 4 * KS, kSlab = kTile * 64, kStage = KS * kSlab;
  constexpr int kOwn = 2 / SPLIT;  // of the wave's two blocks of 32 rows, those whose statistics it keeps
  constexpr int kGive = SPLIT == 2 ? 4 * 1024 : 0;  // values of the halves' exchange
  __shared__ __attribute__((aligned(16))) uint16_t smem[kStages * kStage + 2 * kGive];

  const int logical = xcd_logical_id(per_xcd);
  if (logical >= n_mt * n_strips) return;
  const int strip = logical / n_mt;
  const int t0 = strip * per_strip, n_tiles = min(per_strip, n_nt - t0);  // t0 < n_nt

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int l32 = lane & 31, h = lane >> 5;
  const int half = SPLIT == 2 ? wave & 1 : 0;  // of K
  const int m0 = (logical - strip * n_mt) * (256 / SPLIT) + 64 * (wave / SPLIT);
  const int row0[2] = {m0 + 32 * half, m0 + 32 * (1 - half)};  // the wave's own block of rows first

  // Each wave copies entries 8 wave .. 8 wave + 7 of every slab of a unit (xswz in each slab; entries past V
  // read the last one).
  const int crow = 8 * wave + (lane >> 3);
  const uint32_t cchunk = 16u * static_cast<uint32_t>((lane & 7) ^ ((crow >> 1) & 7));
  const uint32_t lds0 = lds_offset(smem) + static_cast<uint32_t>(wave * 1024);
  auto issue = [&](int i, int part, int stage, int s) {  // slab s of a unit of tile i (past the strip: its last)
    constexpr int kOf = KS / SPLIT;  // slabs of a unit that lie in one half of K
    const int slab = s / kOf * KS + part * kOf + s % kOf;
    const int e0 = (t0 + min(i, n_tiles - 1)) * kTile;
    const uint32_t off = static_cast<uint32_t>(min(crow, V - 1 - e0)) * static_cast<uint32_t>(2 * ldw) + cchunk;
    dma_lds16(W + static_cast<int64_t>(e0) * ldw + 64 * slab, off,
              lds0 + static_cast<uint32_t>((stage * kStage + s * kSlab) * 2));
  };

  u32x4 x[2][kAll];
  int target[kOwn];  // −1: no entry of this row is asked for
#pragma unroll
  for (int mi = 0; mi < 2; ++mi) {
    const int row = min(row0[mi] + l32, M - 1);
    const uint16_t* const p = X + static_cast<int64_t>(row) * ldx + 64 * KS * half + 8 * h;
#pragma unroll
    for (int kk = 0; kk < kAll; ++kk) {
      x[mi][kk] = ldg16(p + 16 * kk);
      // the first 28 operands in vector registers, the others in accumulation registers, which MFMAs read as
      // well: left to itself the compiler copies four registers per MFMA (1183 us for 1119)
      if (mi * kAll + kk >= 28) asm volatile("" : "+a"(x[mi][kk]));
    }
    if (mi < kOwn) {
      const int64_t t = targets[row];
      target[mi] = row0[mi] + l32 < M && t >= 0 && t < V ? static_cast<int>(t) : -1;
    }
  }
  // this lane's operand of k-step kk lies at chunk 2 (kk % 4) + h of its row in slab kk / 4 (of its half)
  int lane_off[4];
#pragma unroll
  for (int k4 = 0; k4 < 4; ++k4) lane_off[k4] = half * (KS / 2) * kSlab + xswz(l32, 2 * k4 + h);
  auto read = [&](int stage, int kk) {  // k-step kk of the unit in that stage
    return lds16(smem + stage * kStage + (kk >> 2) * kSlab + lane_off[kk & 3]);
  };

  Stat stat[kOwn];
#pragma unroll
  for (int mi = 0; mi < kOwn; ++mi) stat[mi] = stat_none();
  // value j of acc[mi] is entry 32 tile + 8 (j / 4) + 4 h + j % 4: what is rare, in branches
  auto mask = [&](f32x16(&acc)[2], int i) {
    const int e0 = (t0 + i) * kTile;
    if (e0 + kTile > V) {
#pragma unroll
      for (int mi = 0; mi < kOwn; ++mi)
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (e0 + 8 * (j >> 2) + 4 * h + (j & 3) >= V) acc[mi][j] = -__builtin_inff();
    }
  };
  auto pick = [&](const f32x16(&acc)[2], int i) {
    const int e0 = (t0 + i) * kTile;
#pragma unroll
    for (int mi = 0; mi < kOwn; ++mi) {
      if (__ballot(target[mi] >= e0 && target[mi] < e0 + kTile)) {
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (e0 + 8 * (j >> 2) + 4 * h + (j & 3) == target[mi]) zt[row0[mi] + l32] = acc[mi][j];
      }
    }
  };
  // quarter q of the other half's products: given to that wave, and taken from it behind a barrier
  float* const xch = reinterpret_cast<float*>(smem + kStages * kStage) + 4 * lane;
  auto give = [&](const f32x16(&acc)[2], int q) {
    *reinterpret_cast<f32x4*>(xch + 1024 * wave + 256 * q) =
        f32x4{acc[1][4 * q], acc[1][4 * q + 1], acc[1][4 * q + 2], acc[1][4 * q + 3]};
  };
  auto taken = [&](int q) { return *reinterpret_cast<const f32x4*>(xch + 1024 * (wave ^ 1) + 256 * q); };
  auto add = [&](const f32x16(&acc)[2]) {
#pragma unroll
    for (int mi = 0; mi < kOwn; ++mi) {
      float m = stat[mi].m;
#pragma unroll
      for (int j = 0; j < 16; ++j) m = fmaxf(m, acc[mi][j]);
      stat_rescale(stat[mi], m);
#pragma unroll
      for (int j = 0; j < 16; ++j) stat_add<ENT>(stat[mi], acc[mi][j]);
    }
  };

  f32x16 acc[2][2];
#pragma unroll
  for (int mi = 0; mi < 2; ++mi)
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[1][mi][j] = -__builtin_inff();  // no tile before the first
  u32x4 w[4];
  // Tile i: its MFMAs into acc[i % 2], the statistics of tile i − 1 beside them: from k-step kSum on its maximum in
  // four, then the sums moved to it, its values over the others. With K in halves the products are exchanged before:
  // given in the first four k-steps, taken behind the first unit's barrier. The scheduling barriers keep that order.
  constexpr int kSum = SPLIT == 2 ? kK / 2 + 2 : 0, kScale = kSum + 4;
  auto body = [&](int i, f32x16(&cur)[2], f32x16(&old)[2]) {
    if (i > 0) {
      mask(old, i - 1);
      if (SPLIT == 1) pick(old, i - 1);
    }
    constexpr int kVals = 16 * kOwn;
    f32x4 other[4];
    float m[kOwn];
#pragma unroll
    for (int mi = 0; mi < kOwn; ++mi) m[mi] = stat[mi].m;
#pragma unroll
    for (int kk = 0; kk < kAll; ++kk) {
      const int part = kk / kK, ku = kk % kK, unit = i * SPLIT + part;
      if (ku == kK / 2) {
        // the next unit has landed (the one after it may be on its way), and every wave is done with the unit
        // before this one (its reads have returned), whose stage the next copies overwrite
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(KS) : "memory");
        ring_barrier();
      }
      w[(kk + kAhead) & 3] = ku + kAhead < kK ? read(unit % kStages, ku + kAhead)
                                              : read((unit + 1) % kStages, ku + kAhead - kK);
#pragma unroll
      for (int mi = 0; mi < 2; ++mi)
        cur[mi] = Mfma<DT>::run(w[kk & 3], x[mi][kk], kk ? cur[mi] : f32x16{});
      if (ku >= kK / 2 && ku < kK / 2 + KS)
        issue(i + (part + 3) / SPLIT, (part + 3) % SPLIT, (unit + 3) % kStages, ku - kK / 2);
      if (SPLIT == 2 && kk < 4) give(old, kk);
      if (SPLIT == 2 && kk == kK / 2) {
#pragma unroll
        for (int q = 0; q < 4; ++q) other[q] = taken(q);
      }
      if (kk >= kSum && kk < kScale) {
#pragma unroll
        for (int v = kVals / 4 * (kk - kSum); v < kVals / 4 * (kk - kSum + 1); ++v) {
          if (SPLIT == 2) old[0][v] += other[v >> 2][v & 3];
          m[v >> 4] = fmaxf(m[v >> 4], old[v >> 4][v & 15]);
        }
      } else if (kk == kScale) {
        if (SPLIT == 2 && i > 0) pick(old, i - 1);
#pragma unroll
        for (int mi = 0; mi < kOwn; ++mi) stat_rescale(stat[mi], m[mi]);
      } else if (kk > kScale) {
        constexpr int kRest = kAll - kScale - 1;
#pragma unroll
        for (int v = kVals * (kk - kScale - 1) / kRest; v < kVals * (kk - kScale) / kRest; ++v)
          stat_add<ENT>(stat[v >> 4], old[v >> 4][v & 15]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
#pragma unroll
  for (int u = 0; u < 3; ++u)
#pragma unroll
    for (int s = 0; s < KS; ++s) issue(u / SPLIT, u % SPLIT, u, s);
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * KS) : "memory");
  ring_barrier();
#pragma unroll
  for (int kk = 0; kk < kAhead; ++kk) w[kk] = read(0, kk);
  for (int i = 0; i < n_tiles; i += 2) {
    body(i, acc[0], acc[1]);
    if (i + 1 < n_tiles) body(i + 1, acc[1], acc[0]);
  }
  auto last = [&](f32x16(&acc)[2]) {
    if constexpr (SPLIT == 2) {
#pragma unroll
      for (int q = 0; q < 4; ++q) give(acc, q);
      ring_barrier();
#pragma unroll
      for (int j = 0; j < 16; ++j) acc[0][j] += taken(j >> 2)[j & 3];
    }
    mask(acc, n_tiles - 1);
    pick(acc, n_tiles - 1);
    add(acc);
  };
  if (n_tiles & 1)
    last(acc[0]);
  else
    last(acc[1]);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no copy outlives the workgroup
  // the lane halves hold parts of the same rows
#pragma unroll
  for (int mi = 0; mi < kOwn; ++mi) {
    const Stat& a = stat[mi];
    stat_join(stat[mi], Stat{lane_xor<32>(a.m), lane_xor<32>(a.mu), lane_xor<32>(a.s), lane_xor<32>(a.h)});
    const int row = row0[mi] + l32;
    if (h == 0 && row < M) parts[static_cast<int64_t>(strip) * M + row] = Part{a.m, a.s, a.h};
  }
}

// One wave per row and turn: its strips' statistics joined, and the row's results.
__global__ __launch_bounds__(256) void head_join_kernel(const Part* __restrict__ parts, const float* __restrict__ zt,
                                                        const int64_t* __restrict__ targets, int64_t ignore,
                                                        float* __restrict__ lp, float* __restrict__ ent, int M, int V,
                                                        int n_strips) {
  const int lane = threadIdx.x & 63;
  for (int row = blockIdx.x * 4 + (threadIdx.x >> 6); row < M; row += gridDim.x * 4) {
    Stat a = stat_none();
    for (int p = lane; p < n_strips; p += 64) {
      const Part q = parts[static_cast<int64_t>(p) * M + row];
      stat_join(a, Stat{q.m, q.m == -__builtin_inff() ? 0.f : q.m, q.s, q.h});
    }
    stat_wave(a);
    if (lane) continue;
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
}

// ------------------------------------------------------------------ host

// Whether head_rows_kernel takes the call: enough work for its start (its rows are loaded before anything else),
// and row tiles of 256 (128 where K > 640) that are not emptier than those of 192. us, with it / without, bf16:
// 256 rows of 640 x 128000 55 / 64, 300 rows 79 / 65, 600 rows 110 / 117, 5000 rows 647 / 851; 512 x 32000: 768 rows
// 36 / 31, 1000 rows 41.5 / 42.8, 5000 rows 150 / 175; 256 x 50000: 1000 rows 36 / 41; 640 x 5000: 3000 rows 36 / 33;
// 1024 x 50001: 192 rows 40 / 33, 256 rows 40 / 50, 1503 rows 152 / 165; 1024 x 8000: 1503 rows 37 / 33, x 11000
// 45 / 48; 768: 384 rows x 32000 30 / 27, x 45000 37 / 39, 1000 rows x 16000 35 / 38.
bool rows_applies(int M, int V, int K) {
  const bool wide = K == 768 || K == 1024;
  if (!wide && (K % 128 || K < 256 || K > 640)) return false;
  const int tile = wide ? 128 : 256;
  const int64_t own = (M + tile - 1) / tile * static_cast<int64_t>(tile), other = (M + 191) / 192 * 192ll;
  return static_cast<int64_t>(M) * V >= (wide ? 12500000 : 25000000) && 100 * own <= 107 * other;
}

struct Plan {
  int ks;  // K / 64 for head_rows_kernel, 0 for head_kernel
  int mi, n_mt, n_nt, n_strips, per_strip;
};

// Strips of the n_nt tiles so that the workgroups fill whole rounds of the `slots` that run at once, with as
// few tiles in a row (`start` tiles' worth for a strip's start and end) as that allows.
void plan_strips(Plan& p, int slots, int start, int longest) {
  const int room = (1 << 22) / p.n_mt;  // workgroups of a launch
  int most = p.n_nt < slots ? p.n_nt : slots;
  if (most > room) most = room;
  int64_t best = -1;
  p.n_strips = p.per_strip = 1;
  int first = (p.n_nt + longest - 1) / longest;
  if (first > most) first = most;
  if (first < 1) first = 1;
  for (int s = first; s <= most || s == first; ++s) {
    const int per = (p.n_nt + s - 1) / s, strips = (p.n_nt + per - 1) / per;
    const int64_t rounds = (static_cast<int64_t>(p.n_mt) * strips + slots - 1) / slots;
    const int64_t cost = rounds * (per + start);
    if (best < 0 || cost < best) {
      best = cost;
      p.n_strips = strips;
      p.per_strip = per;
    }
  }
}

Plan plan(int M, int V, int K) {
  Plan p{};
  if (rows_applies(M, V, K)) {
    p.ks = K / 64;
    p.n_mt = K > 640 ? (M + 127) / 128 : (M + 255) / 256;
    p.n_nt = (V + kTile - 1) / kTile;
    // strips of more than 256 tiles run at the pace of the slowest CU: 8192 x 128000 in one round 1090 us, two 1047
    plan_strips(p, 256, 8, 256);
    return p;
  }
  // row tiles of 192, or of 64 where one covers all rows
  p.mi = M <= 64 ? 1 : 3;
  p.n_mt = (M + 64 * p.mi - 1) / (64 * p.mi);
  p.n_nt = (V + kCols - 1) / kCols;
  plan_strips(p, 512, 1, 1 << 30);
  return p;
}

constexpr int64_t kMaxRows = 1 << 30, kMaxV = 1 << 28, kMaxPitch = 1 << 22;
constexpr int kMaxJoin = 1 << 20;  // workgroups of the join (a launch has less than 2^32 threads)

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
  *ws_bytes = M ? zt_offset(M, plan(M, static_cast<int>(V), K)) + 4 * static_cast<size_t>(M) : 0;
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
  const Plan p = plan(M, v, K);
  Part* const parts = static_cast<Part*>(d_ws);
  float* const zt = reinterpret_cast<float*>(static_cast<uint8_t*>(d_ws) + zt_offset(M, p));
  const int per_xcd = (p.n_mt * p.n_strips + 7) / 8;
  auto launch = [&](auto dt, auto e, auto mi) {
    head_kernel<decltype(dt)::value, decltype(e)::value, decltype(mi)::value><<<8 * per_xcd, 256, 0, s>>>(
        static_cast<const uint16_t*>(d_X), ldx, static_cast<const uint16_t*>(d_W), ldw, d_targets, M, v, K / 64,
        p.n_mt, p.n_nt, p.n_strips, p.per_strip, parts, zt, per_xcd);
  };
  auto launch_rows = [&](auto dt, auto e, auto ks, auto split) {
    head_rows_kernel<decltype(dt)::value, decltype(e)::value, decltype(ks)::value, decltype(split)::value>
        <<<8 * per_xcd, 256, 0, s>>>(
        static_cast<const uint16_t*>(d_X), ldx, static_cast<const uint16_t*>(d_W), ldw, d_targets, M, v, p.n_mt,
        p.n_nt, p.n_strips, p.per_strip, parts, zt, per_xcd);
  };
  auto by_rows = [&](auto dt, auto e) {
    const std::integral_constant<int, 1> one{};
    const std::integral_constant<int, 2> two{};
    if (p.ks == 4)
      launch_rows(dt, e, std::integral_constant<int, 4>{}, one);
    else if (p.ks == 6)
      launch_rows(dt, e, std::integral_constant<int, 6>{}, one);
    else if (p.ks == 8)
      launch_rows(dt, e, std::integral_constant<int, 8>{}, one);
    else if (p.ks == 10)
      launch_rows(dt, e, std::integral_constant<int, 10>{}, one);
    else if (p.ks == 12)
      launch_rows(dt, e, std::integral_constant<int, 6>{}, two);
    else if (p.ks == 16)
      launch_rows(dt, e, std::integral_constant<int, 8>{}, two);
    else if (p.mi == 1)
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
  const int join = (M + 3) / 4;
  head_join_kernel<<<join < kMaxJoin ? join : kMaxJoin, 256, 0, s>>>(parts, zt, d_targets, ignore_index, d_lp, d_entropy,
                                                                     M, v, p.n_strips);
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? TMAC_OK : static_cast<int>(err);
}
