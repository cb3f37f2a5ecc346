// W4A16 GEMM with a fused epilogue, over one weight or over the experts of a
// routed batch (tcgen05, TMEM).
//
//   dense:    C = epilogue(A x dequant(B))
//   experts:  row p of C = epilogue(A[src(p)] x dequant(B_e)),
//             offsets[e] <= p < offsets[e + 1]
//
// Mathematics and accuracy are those of gemm_tc.cu: swap-AB (MMA-M = 128
// weight columns from TMEM, MMA-N = TILE_M activation rows from 128B-swizzled
// shared memory), weights dequantised to the exact half(q * s), FP32
// accumulation with a promotion every promote_blocks. Different here:
//
// * The epilogue (epilogue.cuh) runs on the FP32 sums in registers. A thread
//   holds one weight column; of a gated pair the two columns sit 8 lanes
//   apart, so the pair swaps halves of its rows with one shuffle per row and
//   each lane finishes half of them: no activation is computed twice.
// * Work is over (expert, m-tile, n-tile). How many rows an expert has is only
//   known on the device, so each CTA first sums the experts' tile counts into
//   a table in shared memory and everything else (which tile, which split)
//   follows from that by arithmetic: no extra launch, nothing read back.
// * Gathered activations of few rows come straight from the tokens' rows, four
//   rows per TMA gather; where the gathers would cost more than a copy, they are
//   copied into row order first (copy_rows_first).
// * Small tiles (16, 32, 64 rows) for few rows per weight. There the weights
//   bound it: 4 KB of codes per 64-k block and SM at HBM rate is a block every
//   ~95 ns, and one dequant warp per SMSP needs several times that, so three
//   groups of four dequant warps take the blocks in turn, and the packed ring
//   is as deep as shared memory allows to cover HBM latency.
//
// Registers are what the block's warps leave: 96 a thread at 16 and 32 rows,
// 80 at 64 and 128, 72 before the split at 256. The epilogue spills a little
// (bytes of spill stores): 0 to 16 at 16 rows, 68 to 82 at 32, 56 to 72 at 64, 40
// to 68 at 128, 96 to 176 at 256.
#pragma once

#include "gemm_epi.h"
#include "ptx.cuh"
#include "tc_common.cuh"

#include <algorithm>
#include <climits>

namespace i4g {
namespace epi {

using tc::load_sum16;
using tc::promote_chunk16;
using tc::rotate_down2;
using tc::tile_coords;

constexpr int TILE_N = 128;
constexpr int BK = 64;
constexpr int T_COLS = 32;                     // TMEM columns per weight stage
constexpr int TMEM_COLS = 512;
constexpr int WBLOCK_BYTES = TILE_N * BK / 2;  // 4096
// Blocks after which the accumulator is promoted: 2048 k, as gemm_tc.cu, where
// the result is rounded to FP16; 512 k (256 in small tiles, where that costs a
// few per cent) for FP32 results, which would show the tensor core's drift.
// M = 300, N = 4096, K = 8192 in FP32, off by (2-norm, relative): 2.5e-6 at
// 2048 k (31 us), 6.7e-7 at 512 k (43 us), 6.0e-7 a product with FP32
// multiply-adds.
template <int TILE_M>
__host__ __device__ constexpr int promote_blocks(bool fp32_out) {
  return fp32_out ? (TILE_M <= 64 ? 4 : 8) : 32;
}
constexpr int kTableInts = kMaxExperts + 1 + 32;

template <int TILE_M>
struct Cfg {
  static constexpr int DEQ = TILE_M <= 128 ? 3 : 2;  // dequant groups
  // At 256 rows 28 warps share the registers: launched with 72 each, the warps
  // that only issue copies and MMAs hand theirs to the epilogue, which holds 64
  // sums a thread (a scheduler's seven warps: 40 + 2 x 64 + 4 x 80 <= 7 x 72).
  // With one group, 23 warps and no such split, M = 160, K = 4096, N = 14336
  // took 28.6 us instead of 23.9, M = 4096, N = 28672 740 instead of 720; three
  // groups were no faster.
  static constexpr bool SPLIT_REGS = TILE_M == 256;
  static constexpr int FIRST_DEQ_WARP = SPLIT_REGS ? 4 : 3;  // a split is by whole warpgroups
  static constexpr int PARTS = TILE_M <= 32 ? 1 : (TILE_M <= 128 ? 2 : 4);
  static constexpr int EPI_WARPS = 4 * PARTS;
  static constexpr int COLS = TILE_M / PARTS;  // accumulator columns per epilogue thread
  static constexpr int FIRST_EPI_WARP = FIRST_DEQ_WARP + 4 * DEQ;
  static constexpr int THREADS = 32 * (FIRST_EPI_WARP + EPI_WARPS);
  static constexpr int ACC = TILE_M <= 128 ? 2 : 1;
  // A stage is BS 64-k blocks: their activation boxes in shared memory and
  // their 32 TMEM columns each of dequantised weights, sharing one pair of
  // barriers. While three dequant warps keep a scheduler's half-rate pipes
  // busy, every instruction of the warps that only issue copies and MMAs takes
  // about 18 cycles, so a barrier round per block would bound the kernel;
  // K = 65536, N = 18944, 16 rows: 185 us with two blocks a stage, 148 with four.
  static constexpr int BS = TILE_M <= 64 ? 4 : (TILE_M <= 128 ? 2 : 1);
  static constexpr int BOX_BYTES = TILE_M * BK * 2;
  static constexpr int ACT_BYTES = BS * BOX_BYTES;
  static constexpr int T_STAGE = BS * T_COLS;
  static constexpr int STAGES = TILE_M <= 64 ? 3 : (TILE_M <= 128 ? 4 : 5);
  static constexpr int ACC_COL = TILE_M <= 128 ? STAGES * T_STAGE : 256;
  static constexpr int W_SLOT = BS * (WBLOCK_BYTES + 512);  // + up to two groups of scales a block
  static constexpr int ACT_OFF = 0;
  static constexpr int W_OFF = ACT_OFF + STAGES * ACT_BYTES;
  static constexpr int SPACE = 232448 - 1024 - 1024 - W_OFF - kTableInts * 4 - 1024;
  static constexpr int W_FIT = SPACE / W_SLOT;
  static constexpr int W_STAGES = W_FIT > 32 / BS ? 32 / BS : W_FIT;
  static constexpr int TABLE_OFF = W_OFF + W_STAGES * W_SLOT;
  static constexpr int BAR_OFF = (TABLE_OFF + kTableInts * 4 + 15) / 16 * 16;
  static constexpr int NUM_BARS = 2 * STAGES + 2 * W_STAGES + 2 * ACC + 1;
  static constexpr int MISC_OFF = BAR_OFF + NUM_BARS * 8;
  static constexpr int DYN_BYTES = MISC_OFF + 32 + 1024;
  static_assert(COLS % 16 == 0, "the epilogue works in 16-column chunks");
  static_assert(BOX_BYTES % 1024 == 0, "activation stages keep 1024-byte alignment");
  static_assert(STAGES * T_STAGE <= ACC_COL && ACC_COL + ACC * TILE_M <= TMEM_COLS, "TMEM");
  static_assert(DYN_BYTES <= 232448, "shared memory");
  // A group that stored unit i knows that the MMAs of unit i - STAGES are done;
  // its next unit waits, by parity, for those of unit i + DEQ - STAGES, which
  // is the right phase only if the one two phases before it is known to be over.
  static_assert(DEQ <= STAGES && DEQ <= W_STAGES, "phases that parity can tell apart");
  static_assert(W_STAGES * BS >= 8, "packed weights in flight");
};

// K is walked in units of a stage (BS blocks; the last one may be shorter).
// The cost of a split tail against a whole one, in 64-k blocks: publishing a
// partial tile, the ticket and the last arriver's sums. Measured, split against
// whole, us: 16 rows, N = 28672: K = 4096 (28 blocks less on the longest CTA)
// 21.2 / 19.7, K = 8192 (60 less) 32.0 / 33.6; N = K = 4096 (48) 13.2 / 11.0;
// K = 14336, N = 4096 (172) 16.3 / 28.6. 64 rows: N = 28672, K = 8192 (60) 42.7 /
// 41.2, N = K = 8192 (72) 21.8 / 22.4. 128 rows: N = 28672, K = 8192 (62) 68 / 61,
// N = K = 8192 (72) 30.0 / 32.3. 256 rows, M = 1024: N = 20480, K = 4096 (43)
// 129 / 127, N = 28672, K = 8192 (120) 300 / 320.
template <int TILE_M>
constexpr int split_overhead_blocks() {
  return TILE_M <= 32 ? 50 : (TILE_M <= 128 ? 70 : 48);
}
constexpr int kMinChunkBlocks = 8;
constexpr int kMaxShares = 8;  // shares per tail tile on average

__host__ __device__ inline Sched make_sched(int tiles, int kunits, int bs, int ctas, bool split,
                                            int overhead) {
  Sched s{tiles, 0, 0};
  const int rem = tiles % ctas;
  if (!split || rem == 0) return s;
  const int run = rem * kunits;
  int chunks = run * bs / kMinChunkBlocks;
  if (chunks > ctas) chunks = ctas;
  if (chunks > rem * kMaxShares) chunks = rem * kMaxShares;
  if (chunks <= rem || ((run + chunks - 1) / chunks) * bs + overhead >= kunits * bs) return s;
  s.full_tiles = tiles - rem;
  s.tail_tiles = rem;
  s.chunks = chunks;
  return s;
}

// One CTA's share of a launch's work, and its items in order.
struct Walk {
  Sched s;
  int b, ctas, kunits, num_n;
  int whole;   // whole tiles of this CTA
  int c0, c1;  // its run of the tail's units
  const int* table;  // first m-tile of each expert (shared memory), [E + 1]
  const int* offsets;
  int E, M, num_m;   // num_m: m-tiles of the one weight (dense)

  __device__ __forceinline__ void start() {
    whole = b < s.full_tiles ? (s.full_tiles - 1 - b) / ctas + 1 : 0;
    c0 = c1 = 0;
    if (b < s.chunks) {
      const int run = s.tail_tiles * kunits;
      c0 = static_cast<int>(static_cast<long long>(b) * run / s.chunks);
      c1 = static_cast<int>(static_cast<long long>(b + 1) * run / s.chunks);
    }
  }
  __device__ __forceinline__ int units() const { return whole * kunits + (c1 - c0); }
};

struct Item {
  int e, nt, u0, u1;  // units [u0, u1)
  int row0, rows;  // first row of C (sorted row), rows of this tile (1 .. TILE_M)
  int rem;         // tail tile, or -1: a whole tile
  int slot, base_slot, nparts;
};

// The units [u0, u1) of this CTA's j-th item (item_at without its place).
__device__ __forceinline__ bool span_at(const Walk& w, int j, int& u0, int& u1) {
  u0 = 0;
  u1 = w.kunits;
  if (j < w.whole) return true;
  if (w.c1 <= w.c0) return false;
  const int t = w.c0 / w.kunits + (j - w.whole);
  if (t > (w.c1 - 1) / w.kunits) return false;
  u0 = max(w.c0 - t * w.kunits, 0);
  u1 = min(w.c1 - t * w.kunits, w.kunits);
  return true;
}

template <int TILE_M>
__device__ __forceinline__ bool item_at(const Walk& w, int j, Item& r) {
  int tile;
  if (!span_at(w, j, r.u0, r.u1)) return false;
  r.rem = -1;
  if (j < w.whole) {
    tile = w.b + j * w.ctas;
  } else {
    const int t = w.c0 / w.kunits + (j - w.whole);
    tile = w.s.full_tiles + t;
    // the shares of tile t: owner(v) is the last share starting at or before unit v
    const long long run = static_cast<long long>(w.s.tail_tiles) * w.kunits;
    const long long v0 = static_cast<long long>(t) * w.kunits;
    const int p0 = static_cast<int>(((v0 + 1) * w.s.chunks - 1) / run);
    const int p1 = static_cast<int>(((v0 + w.kunits) * w.s.chunks - 1) / run);
    if (p0 != p1) {
      r.rem = t;
      r.slot = t + w.b;  // unique: tiles and shares both only advance
      r.base_slot = t + p0;
      r.nparts = p1 - p0 + 1;
    }
  }
  // expert: the last one whose first tile is at or before `tile`
  int e = 0;
  if (w.E > 1) {
    int lo = 0, hi = w.E;  // table[lo] * num_n <= tile < table[hi] * num_n
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (w.table[mid] * w.num_n <= tile) lo = mid; else hi = mid;
    }
    e = lo;
  }
  const int first = w.offsets ? w.table[e] : 0;
  const int num_m = w.offsets ? w.table[e + 1] - first : w.num_m;
  int mt = 0;
  r.nt = tile - first * w.num_n;
  if (num_m > 1) tile_coords(r.nt, num_m, w.num_n, mt, r.nt);
  r.e = e;
  int begin = 0, end = w.M;
  if (w.offsets) {
    begin = min(max(w.offsets[e], 0), w.M);
    end = min(max(w.offsets[e + 1], begin), w.M);
  }
  r.row0 = begin + mt * TILE_M;
  r.rows = min(TILE_M, end - r.row0);
  return true;
}

// Where one epilogue thread's values go and what is added to them.
struct Sink {
  void* C;
  int ldc, fp32_out;
  const __half* residual;  // at (row 0 of the tile, this thread's output column), or null
  size_t ldr;
  size_t c0;               // element of C at (row 0 of the tile, output column)
  float bias;
  int activation;
  int rows;
};

// Finishes 16 rows (m .. m + 15 of the tile) of a thread's column in place:
// bias, activation, gate, residual. Gated: the values kept are the first 8 of
// v, rows m + i (gate lanes) or m + 8 + i (up lanes).
template <bool GATED>
__device__ __forceinline__ void finish16(const Sink& k, int m, bool up, float (&v)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] += k.bias;
  if constexpr (!GATED) {
    activate(k.activation, v);
    if (k.residual) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (m + i < k.rows)
          v[i] += __half2float(k.residual[static_cast<size_t>(m + i) * k.ldr]);
    }
  } else {
    float g[8], u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float other = __shfl_xor_sync(0xffffffffu, up ? v[i] : v[8 + i], 8);
      g[i] = up ? other : v[i];
      u[i] = up ? v[8 + i] : other;
    }
    activate(k.activation, g);
    const int mm = m + (up ? 8 : 0);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[i] = g[i] * u[i];
      if (k.residual && mm + i < k.rows)
        v[i] += __half2float(k.residual[static_cast<size_t>(mm + i) * k.ldr]);
    }
  }
}

template <bool GATED>
__device__ __forceinline__ void store16(const Sink& k, int m, bool up, const float (&v)[16]) {
  const int mm = GATED && up ? m + 8 : m;
#pragma unroll
  for (int i = 0; i < (GATED ? 8 : 16); ++i) {
    if (mm + i < k.rows) {
      const size_t at = k.c0 + static_cast<size_t>(mm + i) * k.ldc;
      if (k.fp32_out) static_cast<float*>(k.C)[at] = v[i];
      else static_cast<__half*>(k.C)[at] = __float2half_rn(v[i]);
    }
  }
}

__device__ __forceinline__ void tma_gather4(uint32_t dst, const void* map, uint32_t bar, int x,
                                            int y0, int y1, int y2, int y3) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(dst),
      "l"(map), "r"(bar), "r"(x), "r"(y0), "r"(y1), "r"(y2), "r"(y3)
      : "memory");
}

template <int TILE_M, int GROUP, bool GATED>
__global__ void __launch_bounds__(Cfg<TILE_M>::THREADS, 1)
    gemm_epi_kernel(const __grid_constant__ CUtensorMap act_map, const __grid_constant__ Args a) {
  using L = Cfg<TILE_M>;
  constexpr int STAGES = L::STAGES;
  constexpr int W_STAGES = L::W_STAGES;
  constexpr int ACC = L::ACC;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t act_base = smem_u32(smem + L::ACT_OFF);
  const uint32_t w_base = smem_u32(smem + L::W_OFF);
  const uint32_t bar_base = smem_u32(smem + L::BAR_OFF);
  int* table = reinterpret_cast<int*>(smem + L::TABLE_OFF);  // [E + 1], then warp totals
  // full: a block's activations landed and its weights are in TMEM; empty:
  // the MMAs that read them completed
  auto full = [&](int i) { return bar_base + 8u * i; };
  auto empty = [&](int i) { return bar_base + 8u * (STAGES + i); };
  auto wfull = [&](int i) { return bar_base + 8u * (2 * STAGES + i); };
  auto wempty = [&](int i) { return bar_base + 8u * (2 * STAGES + W_STAGES + i); };
  auto dfull = [&](int i) { return bar_base + 8u * (2 * STAGES + 2 * W_STAGES + i); };
  auto dempty = [&](int i) { return bar_base + 8u * (2 * STAGES + 2 * W_STAGES + ACC + i); };
  const uint32_t drain_bar = bar_base + 8u * (L::NUM_BARS - 1);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::MISC_OFF);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::MISC_OFF + 4);
  volatile uint32_t* ticket_slot = reinterpret_cast<volatile uint32_t*>(smem + L::MISC_OFF + 8);
  volatile int* never = reinterpret_cast<volatile int*>(smem + L::MISC_OFF + 12);

  const int warp = static_cast<int>(uniform(threadIdx.x >> 5));
  const int lane = threadIdx.x & 31;
  const int kblocks = a.K / BK;
  const int kunits = (kblocks + L::BS - 1) / L::BS;
  const int groups = a.K / GROUP;
  const int num_n = a.N / TILE_N;
  const int seg = promote_blocks<TILE_M>(a.fp32_out) / L::BS;  // units between promotions

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(full(i), 1 + 4);  // the activation copy and four dequant warps
      mbar_init(empty(i), 1);
    }
    for (int i = 0; i < W_STAGES; ++i) {
      mbar_init(wfull(i), 1);
      mbar_init(wempty(i), 4);  // the four warps of the group that reads it
    }
    for (int i = 0; i < ACC; ++i) {
      mbar_init(dfull(i), 1);
      mbar_init(dempty(i), L::EPI_WARPS);
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    *never = 0;
    fence_mbarrier_init();
    fence_proxy_async_smem();
  }
  if (warp == 0 && lane == 0) prefetch_tensormap(&act_map);
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = uniform(*tmem_slot);

  Walk walk;
  walk.ctas = gridDim.x;
  walk.b = blockIdx.x;
  walk.kunits = kunits;
  walk.num_n = num_n;
  walk.table = table;
  walk.offsets = a.offsets;
  walk.E = a.offsets ? a.E : 1;
  walk.M = a.M;
  walk.num_m = (a.M + TILE_M - 1) / TILE_M;
  // Launched as a programmatic dependent, this CTA may come this far while the
  // kernel before it still runs; A, C, the weights, the routing and the
  // workspace are touched only after the wait. Before it the dense product,
  // whose first weights are known, warms L2 with one ring of them (a prefetch
  // cannot return stale data); the experts' tiles follow from the routing.
  if (!a.offsets) {
    walk.s = make_sched(walk.num_m * num_n, kunits, L::BS, gridDim.x, a.tickets != nullptr,
                        split_overhead_blocks<TILE_M>());
    walk.start();
    if (warp == 2) {
      Item w;
      if (item_at<TILE_M>(walk, 0, w) && lane == 0) {
        const int kb = w.u0 * L::BS;
        const int nb = min(min(w.u1 * L::BS, kblocks) - kb, W_STAGES * L::BS);
        const uint8_t* src = a.tiles + (static_cast<size_t>(w.nt) * kblocks + kb) * WBLOCK_BYTES;
        for (int b = 0; b < nb; b += 16)
          bulk_prefetch_l2(src + b * WBLOCK_BYTES, min(16, nb - b) * WBLOCK_BYTES);
      }
      __syncwarp();
    }
  }
  grid_dependency_wait();
  if (threadIdx.x == 0) launch_dependents();
  if (a.offsets) {
    // m-tiles before each expert. Offsets that fall would let rows belong to
    // several experts, and so make more tiles than the grid and the workspace
    // are for (16 experts, 64 rows, offsets 0 64 0 64 ...: 11 partial tiles
    // behind the workspace's end); such a table has no tiles at all.
    const int e = threadIdx.x;
    int sum = 0;
    bool falls = false;
    if (e < a.E) {
      const int lo = min(max(a.offsets[e], 0), a.M);
      const int hi = min(max(a.offsets[e + 1], 0), a.M);
      falls = hi < lo;
      sum = (hi - lo + TILE_M - 1) / TILE_M;
    }
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += o;
    }
    if (lane == 31) table[kMaxExperts + 1 + warp] = sum;
    const bool ascending = !__syncthreads_or(falls);
    for (int i = 0; i < warp; ++i) sum += table[kMaxExperts + 1 + i];
    if (e < a.E) table[e + 1] = sum;
    if (e == 0) table[0] = 0;
    __syncthreads();
    walk.s = make_sched(ascending ? table[a.E] * num_n : 0, kunits, L::BS, gridDim.x,
                        a.tickets != nullptr, split_overhead_blocks<TILE_M>());
    walk.start();
  }

  if (warp < L::FIRST_DEQ_WARP) {
    if constexpr (L::SPLIT_REGS) regs_dec<40>();
    if (warp == 0) {
      // ------------------------------------------------- activation producer
      // Gathered rows: lane l fetches rows 4 l .. 4 l + 3 of the tile (and 128
      // further where the tile has them) while there are any; the last fetch may
      // repeat the tile's last row. Rows that are not fetched keep what the
      // stage held: each belongs to one accumulator column, which is not stored.
      constexpr int PER_LANE = (TILE_M / 4 + 31) / 32;
      uint32_t it = 0, s = 0, ph = 0;
      bool ok = true;
      Item w;
      for (int j = 0; ok && __any_sync(0xffffffffu, item_at<TILE_M>(walk, j, w)); ++j) {
        int src[PER_LANE][4];
        if (a.rows) {
  #pragma unroll
          for (int q = 0; q < PER_LANE; ++q)
  #pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int r = min((lane + 32 * q) * 4 + i, w.rows - 1);
              // a negative row becomes -1: the division alone would round to row 0
              const int pair = a.rows[w.row0 + r];
              src[q][i] = (pair / a.row_div) | (pair >> 31);
            }
        }
        const int u0 = static_cast<int>(uniform(w.u0)), u1 = static_cast<int>(uniform(w.u1));
        const int row0 = static_cast<int>(uniform(w.row0));
        const int quads = static_cast<int>(uniform((w.rows + 3) / 4));
        for (int u = u0; u < u1; ++u) {
          ok = mbar_wait_warp(empty(s), ph ^ 1u, abort_flag, a.status, a.wait_limit_ns);
          if (!ok) break;
          const uint32_t dst = act_base + s * L::ACT_BYTES;
          if (!a.rows) {
            // a box past the last block (in the last unit, if K / 64 is not a
            // multiple of BS) reads zeros and counts its bytes like any other
            if (elect_one()) {
              mbar_arrive_expect_tx(full(s), L::ACT_BYTES);
              tma_load_3d(dst, &act_map, full(s), 0, row0, u * L::BS);
            }
          } else {
            const int nb = min(L::BS, kblocks - u * L::BS);
            if (elect_one()) mbar_arrive_expect_tx(full(s), nb * quads * 512);
            __syncwarp();
            for (int b = 0; b < nb; ++b)
  #pragma unroll
              for (int q = 0; q < PER_LANE; ++q)
                if (lane + 32 * q < quads)
                  tma_gather4(dst + b * L::BOX_BYTES + (lane + 32 * q) * 512, &act_map, full(s),
                              (u * L::BS + b) * BK, src[q][0], src[q][1], src[q][2], src[q][3]);
          }
          ++it;
          if (++s == static_cast<uint32_t>(STAGES)) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
      if (!ok && lane == 0) {  // let every copy already issued land
        for (uint32_t i = it > STAGES ? it - STAGES : 0; i < it; ++i)
          mbar_wait(full(i % STAGES), (i / STAGES) & 1u, never, nullptr, 100000000ull);
      }
    } else if (warp == 2) {
      // ----------------------------------------------------- weight producer
      uint32_t s = 0, ph = 0, issued = 0;
      bool ok = true;
      Item w;
      for (int j = 0; ok && __any_sync(0xffffffffu, item_at<TILE_M>(walk, j, w)); ++j) {
        const size_t col = uniform(static_cast<uint32_t>(w.e * num_n + w.nt));  // 128-column run
        const int u0 = static_cast<int>(uniform(w.u0)), u1 = static_cast<int>(uniform(w.u1));
        const int kb0 = u0 * L::BS;
        const uint8_t* wsrc = a.tiles + (col * kblocks + kb0) * WBLOCK_BYTES;
        const __half* ssrc = a.scales + (col * groups + kb0 * BK / GROUP) * TILE_N;
        for (int u = u0; u < u1; ++u) {
          ok = mbar_wait_warp(wempty(s), ph ^ 1u, abort_flag, a.status, a.wait_limit_ns);
          if (!ok) break;
          // a whole unit's sizes are constants; one that starts inside a group
          // of 128 (one block a unit) still needs that group
          constexpr uint32_t kGroupsFull = (L::BS * BK + GROUP - 1) / GROUP;
          uint32_t wbytes = L::BS * WBLOCK_BYTES, sbytes = kGroupsFull * TILE_N * 2;
          if (L::BS > 1 && u == kunits - 1) {
            const uint32_t nb = kblocks - u * L::BS;
            wbytes = nb * WBLOCK_BYTES;
            sbytes = (nb * BK + GROUP - 1) / GROUP * TILE_N * 2;
          }
          if (elect_one()) {
            const uint32_t dst = w_base + s * L::W_SLOT;
            mbar_arrive_expect_tx(wfull(s), wbytes + sbytes);
            bulk_load(dst, wsrc, wbytes, wfull(s));
            bulk_load(dst + L::BS * WBLOCK_BYTES, ssrc, sbytes, wfull(s));
          }
          wsrc += L::BS * WBLOCK_BYTES;
          if (L::BS * BK >= GROUP || (u & 1)) ssrc += kGroupsFull * TILE_N;
          ++issued;
          if (++s == static_cast<uint32_t>(W_STAGES)) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
      if (!ok && lane == 0) {  // let every copy already issued land
        for (uint32_t i = issued > W_STAGES ? issued - W_STAGES : 0; i < issued; ++i)
          mbar_wait(wfull(i % W_STAGES), (i / W_STAGES) & 1u, never, nullptr, 100000000ull);
      }
    } else if (warp == 1) {
      // ------------------------------------------------------------- MMA issue
      // Every loop bound is warp-uniform (see elect_one, uniform). The MMAs of a
      // tall tile are as wide as its rows (rounded up to 16); below 64 rows the
      // width costs no time and finding the rows would.
      const uint64_t b_desc0 = smem_desc_sw128(act_base);
      uint32_t s = 0, ph = 0;
      uint32_t used[2] = {0, 0};  // segments committed per accumulator
      int acc = 0;
      bool ok = true;
      Item w;
      for (int j = 0; ok; ++j) {
        uint32_t idesc = idesc_f16_f32(TILE_N, TILE_M);
        if constexpr (TILE_M > 64) {
          if (!__any_sync(0xffffffffu, item_at<TILE_M>(walk, j, w))) break;
          idesc = idesc_f16_f32(TILE_N, static_cast<int>(uniform((w.rows + 15) & ~15)));
        } else {
          if (!__any_sync(0xffffffffu, span_at(walk, j, w.u0, w.u1))) break;
        }
        const int u1 = static_cast<int>(uniform(w.u1));
        int u = static_cast<int>(uniform(w.u0));
        const uint32_t d_tmem = tmem_base + L::ACC_COL + acc * TILE_M;
        uint32_t accumulate = 0;  // the item's first MMA starts the sum
        while (true) {
          // one segment of at most promote_blocks, once the accumulator
          // is free: the last item drained it, or the epilogue promoted it
          const uint32_t n = acc == 0 ? used[0]++ : used[1]++;
          ok = mbar_wait_warp(dempty(acc), (n & 1u) ^ 1u, abort_flag, a.status, a.wait_limit_ns);
          if (!ok) break;
          tc_fence_after();
          const int end = min(u1, u + seg);
          for (; u < end; ++u) {
            ok = mbar_wait_warp(full(s), ph, abort_flag, a.status, a.wait_limit_ns);
            if (!ok) break;
            tc_fence_after();
            const uint64_t b_desc = b_desc0 + ((s * L::ACT_BYTES) >> 4);
            const uint32_t a_tmem = tmem_base + s * L::T_STAGE;
            if (u * L::BS + L::BS <= kblocks) {
              if constexpr (L::BS == 4)
                mma_f16_ts_blocks4(d_tmem, a_tmem, b_desc, idesc, accumulate, L::BOX_BYTES >> 4,
                                   empty(s));
              else if constexpr (L::BS == 2)
                mma_f16_ts_blocks2(d_tmem, a_tmem, b_desc, idesc, accumulate, L::BOX_BYTES >> 4,
                                   empty(s));
              else
                mma_f16_ts_blocks1(d_tmem, a_tmem, b_desc, idesc, accumulate, empty(s));
            } else {
              // the last unit's blocks
              for (int b = 0; u * L::BS + b < kblocks; ++b)
                mma_f16_ts_block(d_tmem, a_tmem + b * T_COLS, b_desc + ((b * L::BOX_BYTES) >> 4),
                                 idesc, b == 0 ? accumulate : 1u);
              if (elect_one()) tc_commit(empty(s));
            }
            accumulate = 1;
            if (++s == static_cast<uint32_t>(STAGES)) {
              s = 0;
              ph ^= 1u;
            }
          }
          if (!ok) break;
          if (elect_one()) tc_commit(dfull(acc));
          if (u == u1) break;
        }
        if (ACC == 2) acc ^= 1;
      }
      if (elect_one()) tc_commit(drain_bar);  // TMEM is freed only after every MMA completed
      mbar_wait_warp(drain_bar, 0, never, nullptr, 100000000ull);
    }
  } else if (warp < L::FIRST_EPI_WARP) {
    // ---------------------------------------------------------------- dequant
    if constexpr (L::SPLIT_REGS) regs_dec<64>();
    const uint32_t dgroup = static_cast<uint32_t>(warp - L::FIRST_DEQ_WARP) >> 2;
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;  // weight column inside the tile
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    const NibbleMask nibble;
    // this group's units: dgroup, dgroup + DEQ, ... of the CTA's
    const int total = static_cast<int>(uniform(walk.units()));
    const int whole_units = walk.whole * kunits;
    uint32_t ws = dgroup % W_STAGES, wph = (dgroup / W_STAGES) & 1u;
    uint32_t ts = dgroup % STAGES, tph = (dgroup / STAGES) & 1u;
    bool ok = true;
    for (int it = static_cast<int>(dgroup); it < total; it += L::DEQ) {
      int nb = L::BS;
      if (L::BS > 1 && kblocks % L::BS != 0) {
        const int at = it < whole_units ? it : it - whole_units + walk.c0;
        nb = min(nb, kblocks - static_cast<int>(uniform(at % kunits)) * L::BS);
      }
      ok = mbar_wait_warp(wfull(ws), wph, abort_flag, a.status, a.wait_limit_ns);
      if (!ok) break;
      const uint32_t slot = w_base + ws * L::W_SLOT;
#pragma unroll
      for (int b = 0; b < L::BS; ++b) {
        if (b > 0 && b >= nb) break;
        const uint32_t wsrc = slot + b * WBLOCK_BYTES + row * 16;
        uint4 c0, c1;
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(c0.x), "=r"(c0.y), "=r"(c0.z), "=r"(c0.w)
                     : "r"(wsrc));
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(c1.x), "=r"(c1.y), "=r"(c1.z), "=r"(c1.w)
                     : "r"(wsrc + 2048));
        uint16_t sb0, sb1;
        // the block's first scale group inside the unit
        const uint32_t ssrc = slot + L::BS * WBLOCK_BYTES +
                              (b * BK / GROUP) * (TILE_N * 2) + row * 2;
        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(sb0) : "r"(ssrc));
        if (GROUP == 32)
          asm volatile("ld.shared.u16 %0, [%1];" : "=h"(sb1) : "r"(ssrc + TILE_N * 2));
        else
          sb1 = sb0;
        const uint32_t s0 = half_bits_x2(sb0), s1 = half_bits_x2(sb1);
        uint32_t r[32];
        const uint32_t wv[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
        if (__all_sync(0xffffffffu, fast_scale(sb0) && (GROUP != 32 || fast_scale(sb1)))) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            decode_word(wv[i], (i < 4 ? s0 : s1) + kTimes2p20, (i < 4 ? s0 : s1) + kTimesMinus8,
                        nibble, &r[4 * i]);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint32_t sc = i < 4 ? s0 : s1;
            r[4 * i + 0] = decode_pair<0>(wv[i], sc);
            r[4 * i + 1] = decode_pair<1>(wv[i], sc);
            r[4 * i + 2] = decode_pair<2>(wv[i], sc);
            r[4 * i + 3] = decode_pair<3>(wv[i], sc);
          }
        }
        if (b == 0) {
          ok = mbar_wait_warp(empty(ts), tph ^ 1u, abort_flag, a.status, a.wait_limit_ns);
          if (!ok) break;
          tc_fence_after();
        }
        tmem_st_32x32b_x32(tmem_base + lane_addr + ts * L::T_STAGE + b * T_COLS, r);
      }
      if (!ok) break;
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(full(ts));
        // The packed slot is given back only now: the TMEM store has consumed
        // what was loaded from it. An arrival right after the loads can
        // overtake them (they queue behind the epilogue's global stores, the
        // arrival does not), and the next copy into the slot then overtakes
        // the loads: one 64-k block of some columns was wrong in every second
        // launch of M = 1024, N = 2048, K = 12288, where partial tiles are
        // stored while the pipeline runs.
        mbar_arrive(wempty(ws));
      }
      ws += L::DEQ;
      if (ws >= static_cast<uint32_t>(W_STAGES)) {
        ws -= W_STAGES;
        wph ^= 1u;
      }
      ts += L::DEQ;
      while (ts >= static_cast<uint32_t>(STAGES)) {
        ts -= STAGES;
        tph ^= 1u;
      }
    }
  } else {
    // --------------------------------------------------------------- epilogue
    if constexpr (L::SPLIT_REGS) regs_inc<80>();
    constexpr int COLS = L::COLS;
    constexpr int EPI_THREADS = L::EPI_WARPS * 32;
    const int part = (warp - L::FIRST_EPI_WARP) >> 2;  // which accumulator columns
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;  // weight column inside the tile
    const bool up = GATED && (row & 8);
    const int col = GATED ? (row >> 4) * 8 + (row & 7) : row;  // output column inside the tile
    constexpr int OUT_N = GATED ? TILE_N / 2 : TILE_N;
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    const int m0 = part * COLS;  // first tile row of this thread
    Sink sink;
    sink.C = a.C;
    sink.ldc = GATED ? a.N / 2 : a.N;
    sink.fp32_out = a.fp32_out;
    sink.ldr = static_cast<size_t>(a.epilogue.ldr);
    sink.activation = a.epilogue.activation;
    uint32_t uses[2] = {0, 0};  // segments drained per accumulator
    int acc = 0;
    bool failed = false;
    Item w;
    for (int j = 0; item_at<TILE_M>(walk, j, w); ++j) {
      uint32_t used = acc == 0 ? uses[0] : uses[1];
      const uint32_t col0 = tmem_base + lane_addr + L::ACC_COL + acc * TILE_M + m0;
      const int out_col = w.nt * OUT_N + col;
      sink.rows = w.rows;
      sink.c0 = static_cast<size_t>(w.row0) * sink.ldc + out_col;
      sink.residual = a.epilogue.residual
                          ? a.epilogue.residual + static_cast<size_t>(w.row0) * sink.ldr + out_col
                          : nullptr;
      sink.bias = a.epilogue.bias
                      ? __half2float(a.epilogue.bias[static_cast<size_t>(w.e) * a.N +
                                                     w.nt * TILE_N + row])
                      : 0.0f;
      const int nseg = (w.u1 - w.u0 + seg - 1) / seg;
      uint32_t hb[COLS / 4];  // the running sum's high parts (e5m2 x4)
#pragma unroll
      for (int q = 0; q < COLS / 4; ++q) hb[q] = 0u;
      for (int sg = 0; sg + 1 < nseg; ++sg, ++used) {
        if (!failed && mbar_wait(dfull(acc), used & 1u, abort_flag, a.status, a.wait_limit_ns)) {
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < COLS / 16; ++c) {
            promote_chunk16(col0 + c * 16, hb);
            rotate_down2(hb);
            rotate_down2(hb);
          }
          tmem_st_wait();
        } else {
          failed = true;
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(dempty(acc));
      }
      // the shuffles of a gated pair need whole warps, so the outcome of the
      // wait is made the warp's
      const bool ok = __all_sync(0xffffffffu, !failed && mbar_wait(dfull(acc), used & 1u,
                                                                   abort_flag, a.status,
                                                                   a.wait_limit_ns));
      ++used;
      if (acc == 0) uses[0] = used; else uses[1] = used;
      const uint32_t release_bar = dempty(acc);
      if (ACC == 2) acc ^= 1;
      if (!ok) failed = true;
      if (w.rem < 0) {
        // ------------------------------------------------ whole tile -> C
        if (!ok) continue;
        tc_fence_after();
        if constexpr (TILE_M <= 64) {
          // Small tiles run this tens of times a CTA: unrolled, and a chunk's
          // rows are not looked at (7 rows each 64 us so, 66 rolled).
          if (a.fp32_out) {
#pragma unroll
            for (int c = 0; c < COLS / 16; ++c) {
              uint32_t v[16];
              load_sum16(col0 + c * 16, &hb[c * 4], v);
              float f[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) f[i] = __uint_as_float(v[i]);
              finish16<GATED>(sink, m0 + c * 16, up, f);
              store16<GATED>(sink, m0 + c * 16, up, f);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(release_bar);
          } else {
            // rounded to FP16 pairs in registers, the accumulator released,
            // then stored
            constexpr int KEEP = GATED ? 8 : 16;  // values of a chunk this thread keeps
            __half2 hv[COLS / 16 * KEEP / 2];
#pragma unroll
            for (int c = 0; c < COLS / 16; ++c) {
              uint32_t v[16];
              load_sum16(col0 + c * 16, &hb[c * 4], v);
              float f[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) f[i] = __uint_as_float(v[i]);
              finish16<GATED>(sink, m0 + c * 16, up, f);
#pragma unroll
              for (int i = 0; i < KEEP / 2; ++i)
                hv[c * (KEEP / 2) + i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(release_bar);
            __half* const cp = static_cast<__half*>(a.C) + sink.c0;
#pragma unroll
            for (int c = 0; c < COLS / 16; ++c)
#pragma unroll
              for (int i = 0; i < KEEP; ++i) {
                const int m = m0 + c * 16 + i + (up ? 8 : 0);
                const __half2 h = hv[c * (KEEP / 2) + i / 2];
                if (m < w.rows)
                  cp[static_cast<size_t>(m) * sink.ldc] = (i & 1) ? __high2half(h) : __low2half(h);
              }
          }
          continue;
        }
        // In tall tiles the loops over 16-row chunks stay rolled and end at
        // the tile's last row: a CTA runs them a few times, and fetching
        // unrolled code costs more than the branches (M = 203, K = 4096,
        // N = 14336 with GELU 36.5 us unrolled, 32.6 so; 64 experts of
        // 2048 x 4096 with 44 rows each, 128-row tiles, 120 / 94).
        if (TILE_M == 128 || a.fp32_out) {
#pragma unroll 1
          for (int c = 0; c < COLS / 16; ++c) {
            if (m0 + c * 16 >= w.rows) break;
            uint32_t v[16];
            load_sum16(col0 + c * 16, &hb[0], v);
            rotate_down2(hb);
            rotate_down2(hb);
            float f[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) f[i] = __uint_as_float(v[i]);
            finish16<GATED>(sink, m0 + c * 16, up, f);
            store16<GATED>(sink, m0 + c * 16, up, f);
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(release_bar);
        } else {
          // Values are rounded to FP16 pairs in registers, the accumulator
          // released (at 256 rows the MMAs wait for it), then stored. The pairs
          // move down a chunk a step, so that register indices are fixed.
          constexpr int PAIRS = GATED ? 4 : 8;  // of a chunk that this thread keeps
          constexpr int KEPT = COLS / 16 * PAIRS;
          __half2 hv[KEPT];
#pragma unroll
          for (int q = 0; q < KEPT; ++q) hv[q] = __half2();
#pragma unroll 1
          for (int c = 0; c < COLS / 16; ++c) {
#pragma unroll
            for (int q = 0; q + PAIRS < KEPT; ++q) hv[q] = hv[q + PAIRS];
            if (m0 + c * 16 < w.rows) {
              uint32_t v[16];
              load_sum16(col0 + c * 16, &hb[0], v);
              rotate_down2(hb);
              rotate_down2(hb);
              float f[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) f[i] = __uint_as_float(v[i]);
              finish16<GATED>(sink, m0 + c * 16, up, f);
#pragma unroll
              for (int i = 0; i < PAIRS; ++i)
                hv[KEPT - PAIRS + i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(release_bar);
          __half* const cp = static_cast<__half*>(a.C) + sink.c0;
#pragma unroll 1
          for (int c = 0; c < COLS / 16; ++c) {
            if (m0 + c * 16 >= w.rows) break;
#pragma unroll
            for (int i = 0; i < 2 * PAIRS; ++i) {
              const int m = m0 + c * 16 + i + (up ? 8 : 0);
              if (m < w.rows)
                cp[static_cast<size_t>(m) * sink.ldc] =
                    (i & 1) ? __high2half(hv[i / 2]) : __low2half(hv[i / 2]);
            }
#pragma unroll
            for (int q = 0; q + PAIRS < KEPT; ++q) hv[q] = hv[q + PAIRS];
          }
        }
        continue;
      }
      // ------------------------------------------------ split tile -> partial
      // Every epilogue thread takes the barriers below whatever happened. A
      // partial is stored as float4 quads [m / 4][column][m % 4].
      constexpr size_t SLOT4 = static_cast<size_t>(TILE_M / 4) * TILE_N;
      float4* mine4 = reinterpret_cast<float4*>(a.partials) + w.slot * SLOT4;
      if (ok) {
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < COLS / 16; ++c) {
          uint32_t v[16];
          load_sum16(col0 + c * 16, &hb[c * 4], v);
          const int q0 = (m0 + c * 16) / 4;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            __stcg(mine4 + static_cast<size_t>(q0 + i) * TILE_N + row,
                   make_float4(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]),
                               __uint_as_float(v[4 * i + 2]), __uint_as_float(v[4 * i + 3])));
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(release_bar);
        __threadfence();
      }
      if (!epi_bar_and(EPI_THREADS, ok)) {
        failed = true;
        continue;
      }
      if (warp == L::FIRST_EPI_WARP && lane == 0) {
        __threadfence();
        *ticket_slot = atomicAdd(&a.tickets[w.rem], 1u);
      }
      epi_bar_sync(EPI_THREADS);
      const bool last = *ticket_slot == static_cast<uint32_t>(w.nparts - 1);
      if (last) {
        // the tile's last arriver adds the partials in share order (whichever
        // CTA it is, the sum is the same) and finishes the tile
        __threadfence();
        const float4* base = reinterpret_cast<const float4*>(a.partials) + w.base_slot * SLOT4 +
                             static_cast<size_t>(m0 / 4) * TILE_N + row;
#pragma unroll 1
        for (int c = 0; c < COLS / 16; ++c) {
          if (m0 + c * 16 >= w.rows) break;  // the same for the whole warp
          float f[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) f[i] = 0.0f;
          const float4* at = base + static_cast<size_t>(c * 4) * TILE_N;
#pragma unroll 2
          for (int p = 0; p < w.nparts; ++p) {
            float4 t[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              t[i] = __ldcg(at + p * SLOT4 + static_cast<size_t>(i) * TILE_N);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              f[4 * i] += t[i].x;
              f[4 * i + 1] += t[i].y;
              f[4 * i + 2] += t[i].z;
              f[4 * i + 3] += t[i].w;
            }
          }
          finish16<GATED>(sink, m0 + c * 16, up, f);
          store16<GATED>(sink, m0 + c * 16, up, f);
        }
      }
      epi_bar_sync(EPI_THREADS);  // the ticket slot is read by all before it changes
      if (last && warp == L::FIRST_EPI_WARP && lane == 0) a.tickets[w.rem] = 0u;
    }
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

template <int TILE_M, int GROUP, bool GATED>
cudaError_t launch_impl(const CUtensorMap& act_map, const Args& args, int grid,
                        cudaStream_t stream) {
  auto kernel = gemm_epi_kernel<TILE_M, GROUP, GATED>;
  static std::atomic<uint64_t> configured{0};
  cudaError_t e = ensure_dynamic_smem(kernel, Cfg<TILE_M>::DYN_BYTES, configured);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(Cfg<TILE_M>::THREADS);
  cfg.dynamicSmemBytes = Cfg<TILE_M>::DYN_BYTES;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, act_map, args);
}

template <int TILE_M>
cudaError_t launch_tile(const CUtensorMap& act_map, bool gated, int group, const Args& args,
                        int grid, cudaStream_t stream) {
#define I4G_EPI_CASE(G)                                                             \
  if (group == G)                                                                   \
    return gated ? launch_impl<TILE_M, G, true>(act_map, args, grid, stream)        \
                 : launch_impl<TILE_M, G, false>(act_map, args, grid, stream);
  I4G_EPI_CASE(32)
  I4G_EPI_CASE(64)
  I4G_EPI_CASE(128)
#undef I4G_EPI_CASE
  return cudaErrorInvalidValue;
}

}  // namespace epi
}  // namespace i4g
