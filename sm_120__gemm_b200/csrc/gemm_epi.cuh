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
// accumulation with a promotion every kPromoteBlocks blocks. Different here:
//
// * The epilogue (epilogue.cuh) runs on the FP32 sums in registers. A thread
//   holds one weight column; of a gated pair the two columns sit 8 lanes
//   apart, so the pair swaps halves of its rows with one shuffle per row and
//   each lane finishes half of them: no activation is computed twice.
// * Work is over (expert, m-tile, n-tile). How many rows an expert has is only
//   known on the device, so each CTA first sums the experts' tile counts into
//   a table in shared memory and everything else (which tile, which split)
//   follows from that by arithmetic: no extra launch, nothing read back.
// * Gathered activations come straight from the tokens' rows, four rows per
//   TMA gather, so no permuted copy of A is written.
// * Small tiles (16, 32, 64 rows) for few rows per weight. There the weights
//   bound it: 4 KB of codes per 64-k block and SM at HBM rate is a block every
//   ~95 ns, and one dequant warp per SMSP needs several times that, so three
//   groups of four dequant warps take the blocks in turn, and the packed ring
//   is as deep as shared memory allows to cover HBM latency.
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
constexpr int W_SLOT = WBLOCK_BYTES + 512;     // + up to two groups of scales
constexpr int FIRST_DEQ_WARP = 3;
constexpr int kPromoteBlocks = 32;             // 2048 k, as gemm_tc.cu
constexpr int kTableInts = kMaxExperts + 1 + 32;

template <int TILE_M>
struct Cfg {
  static constexpr int DEQ = TILE_M <= 64 ? 3 : (TILE_M <= 128 ? 2 : 1);  // dequant groups
  static constexpr int PARTS = TILE_M <= 32 ? 1 : (TILE_M <= 128 ? 2 : 4);
  static constexpr int EPI_WARPS = 4 * PARTS;
  static constexpr int COLS = TILE_M / PARTS;  // accumulator columns per epilogue thread
  static constexpr int FIRST_EPI_WARP = FIRST_DEQ_WARP + 4 * DEQ;
  static constexpr int THREADS = 32 * (FIRST_EPI_WARP + EPI_WARPS);
  static constexpr int ACC = TILE_M <= 128 ? 2 : 1;
  static constexpr int ACT_BYTES = TILE_M * BK * 2;
  // a stage is one 64-k block: its activation box in shared memory and its
  // 32 TMEM columns of dequantised weights, sharing one pair of barriers
  static constexpr int STAGES = TILE_M <= 64 ? 9 : (TILE_M <= 128 ? 8 : 5);
  static constexpr int ACC_COL = TILE_M <= 128 ? STAGES * T_COLS : 256;
  static constexpr int ACT_OFF = 0;
  static constexpr int W_OFF = ACT_OFF + STAGES * ACT_BYTES;
  static constexpr int SPACE = 232448 - 1024 - W_OFF - kTableInts * 4 - 1024;
  static constexpr int W_FIT = SPACE / W_SLOT;
  static constexpr int W_STAGES = W_FIT > 36 ? 36 : W_FIT;
  static constexpr int TABLE_OFF = W_OFF + W_STAGES * W_SLOT;
  static constexpr int BAR_OFF = (TABLE_OFF + kTableInts * 4 + 15) / 16 * 16;
  static constexpr int NUM_BARS = 2 * STAGES + 2 * W_STAGES + 2 * ACC + 1;
  static constexpr int MISC_OFF = BAR_OFF + NUM_BARS * 8;
  static constexpr int DYN_BYTES = MISC_OFF + 32 + 1024;
  static_assert(COLS % 16 == 0, "the epilogue works in 16-column chunks");
  static_assert(ACT_BYTES % 1024 == 0, "activation stages keep 1024-byte alignment");
  static_assert(STAGES * T_COLS <= ACC_COL && ACC_COL + ACC * TILE_M <= TMEM_COLS, "TMEM");
  static_assert(DYN_BYTES <= 232448, "shared memory");
  static_assert(W_STAGES >= 8, "packed weights in flight");
};

// The cost of a split tail against a whole one, in 64-k blocks of a CTA's
// time: publishing a partial tile, the ticket and the last arriver's sums.
template <int TILE_M>
constexpr int split_overhead_blocks() {
  return TILE_M <= 64 ? 24 : 36;
}
constexpr int kMinChunkBlocks = 8;
constexpr int kMaxShares = 8;  // shares per tail tile on average

__host__ __device__ inline Sched make_sched(int tiles, int kblocks, int units, bool split,
                                            int overhead) {
  Sched s{tiles, 0, 0};
  const int rem = tiles % units;
  if (!split || rem == 0) return s;
  const int run = rem * kblocks;
  int chunks = run / kMinChunkBlocks;
  if (chunks > units) chunks = units;
  if (chunks > rem * kMaxShares) chunks = rem * kMaxShares;
  if (chunks <= rem || (run + chunks - 1) / chunks + overhead >= kblocks) return s;
  s.full_tiles = tiles - rem;
  s.tail_tiles = rem;
  s.chunks = chunks;
  return s;
}

// One CTA's share of a launch's work, and its items in order.
struct Walk {
  Sched s;
  int b, units, kblocks, num_n;
  int whole;   // whole tiles of this CTA
  int c0, c1;  // its run of the tail's blocks
  const int* table;  // first m-tile of each expert (shared memory), [E + 1]
  const int* offsets;
  int E, M, tile_m;

  __device__ __forceinline__ void start() {
    whole = b < s.full_tiles ? (s.full_tiles - 1 - b) / units + 1 : 0;
    c0 = c1 = 0;
    if (b < s.chunks) {
      const int run = s.tail_tiles * kblocks;
      c0 = static_cast<int>(static_cast<long long>(b) * run / s.chunks);
      c1 = static_cast<int>(static_cast<long long>(b + 1) * run / s.chunks);
    }
  }
  __device__ __forceinline__ int blocks() const { return whole * kblocks + (c1 - c0); }
};

struct Item {
  int e, nt, kb0, kb1;
  int row0, rows;  // first row of C (sorted row), rows of this tile (1 .. TILE_M)
  int rem;         // tail tile, or -1: a whole tile
  int slot, base_slot, nparts;
};

template <int TILE_M>
__device__ __forceinline__ bool item_at(const Walk& w, int j, Item& r) {
  int tile;
  r.kb0 = 0;
  r.kb1 = w.kblocks;
  r.rem = -1;
  if (j < w.whole) {
    tile = w.b + j * w.units;
  } else {
    if (w.c1 <= w.c0) return false;
    const int t = w.c0 / w.kblocks + (j - w.whole);
    if (t > (w.c1 - 1) / w.kblocks) return false;
    r.kb0 = max(w.c0 - t * w.kblocks, 0);
    r.kb1 = min(w.c1 - t * w.kblocks, w.kblocks);
    tile = w.s.full_tiles + t;
    // the shares of tile t: owner(v) is the last share starting at or before block v
    const long long run = static_cast<long long>(w.s.tail_tiles) * w.kblocks;
    const long long v0 = static_cast<long long>(t) * w.kblocks;
    const int p0 = static_cast<int>(((v0 + 1) * w.s.chunks - 1) / run);
    const int p1 = static_cast<int>(((v0 + w.kblocks) * w.s.chunks - 1) / run);
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
  const int first = w.table[e], num_m = w.table[e + 1] - first;
  int mt;
  tile_coords(tile - first * w.num_n, num_m, w.num_n, mt, r.nt);
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

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int kblocks = a.K / BK;
  const int groups = a.K / GROUP;
  const int num_n = a.N / TILE_N;

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(full(i), 1 + 4 * 32);  // the activation copy and 128 dequant threads
      mbar_init(empty(i), 1);
    }
    for (int i = 0; i < W_STAGES; ++i) {
      mbar_init(wfull(i), 1);
      mbar_init(wempty(i), 4);  // the four warps of the group that reads it
    }
    for (int i = 0; i < ACC; ++i) {
      mbar_init(dfull(i), 1);
      mbar_init(dempty(i), L::EPI_WARPS * 32);
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
  // Only set-up precedes the wait for the kernel before this one (programmatic
  // dependent launch): offsets, rows, A, C and the workspace come after it.
  grid_dependency_wait();
  if (threadIdx.x == 0) launch_dependents();
  // m-tiles before each expert
  int mine = 0;
  if (a.offsets) {
    const int e = threadIdx.x;
    if (e < a.E) {
      const int lo = min(max(a.offsets[e], 0), a.M);
      const int hi = min(max(a.offsets[e + 1], lo), a.M);
      mine = (hi - lo + TILE_M - 1) / TILE_M;
    }
    int sum = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += o;
    }
    mine = sum;  // inclusive, within the warp
    if (lane == 31) table[kMaxExperts + 1 + warp] = sum;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  if (a.offsets) {
    int before = 0;
    for (int i = 0; i < warp; ++i) before += table[kMaxExperts + 1 + i];
    if (threadIdx.x < a.E) table[threadIdx.x + 1] = before + mine;
    if (threadIdx.x == 0) table[0] = 0;
  } else if (threadIdx.x == 0) {
    table[0] = 0;
    table[1] = (a.M + TILE_M - 1) / TILE_M;
  }
  __syncthreads();

  Walk walk;
  walk.units = gridDim.x;
  walk.b = blockIdx.x;
  walk.kblocks = kblocks;
  walk.num_n = num_n;
  walk.table = table;
  walk.offsets = a.offsets;
  walk.E = a.offsets ? a.E : 1;
  walk.M = a.M;
  walk.s = make_sched(table[walk.E] * num_n, kblocks, gridDim.x, a.tickets != nullptr,
                      split_overhead_blocks<TILE_M>());
  walk.start();

  if (warp == 0) {
    // ------------------------------------------------- activation producer
    // Gathered rows: lane l fetches rows 4 l .. 4 l + 3 of the tile (and 128
    // further where the tile has them); rows past the tile's last repeat its
    // last one and are never stored.
    constexpr int GATHERS = TILE_M / 4;
    constexpr int PER_LANE = (GATHERS + 31) / 32;
    uint32_t it = 0;
    bool ok = true;
    Item w;
    for (int j = 0; ok && item_at<TILE_M>(walk, j, w); ++j) {
      int src[PER_LANE][4];
      if (a.rows) {
#pragma unroll
        for (int q = 0; q < PER_LANE; ++q)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = min((lane + 32 * q) * 4 + i, w.rows - 1);
            src[q][i] = a.rows[w.row0 + r] / a.row_div;
          }
      }
      for (int kb = w.kb0; kb < w.kb1; ++kb, ++it) {
        const int s = it % STAGES;
        const uint32_t ph = (it / STAGES) & 1u;
        ok = mbar_wait(empty(s), ph ^ 1u, abort_flag, a.status, a.wait_limit_ns);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(full(s), L::ACT_BYTES);
        __syncwarp();
        const uint32_t dst = act_base + s * L::ACT_BYTES;
        if (a.rows) {
#pragma unroll
          for (int q = 0; q < PER_LANE; ++q)
            if (GATHERS >= 32 || lane < GATHERS)
              tma_gather4(dst + (lane + 32 * q) * 512, &act_map, full(s), kb * BK, src[q][0],
                          src[q][1], src[q][2], src[q][3]);
        } else if (lane == 0) {
          tma_load_2d(dst, &act_map, full(s), kb * BK, w.row0);
        }
      }
    }
    if (!ok && lane == 0) {  // let every copy already issued land
      for (uint32_t i = it > STAGES ? it - STAGES : 0; i < it; ++i)
        mbar_wait(full(i % STAGES), (i / STAGES) & 1u, never, nullptr, 100000000ull);
    }
  } else if (warp == 2) {
    // ----------------------------------------------------- weight producer
    if (lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      Item w;
      for (int j = 0; ok && item_at<TILE_M>(walk, j, w); ++j) {
        const size_t col = static_cast<size_t>(w.e) * num_n + w.nt;  // 128-column run
        const uint8_t* wblk = a.tiles + col * kblocks * WBLOCK_BYTES;
        const __half* sblk = a.scales + col * groups * TILE_N;
        for (int kb = w.kb0; kb < w.kb1; ++kb, ++it) {
          const int s = it % W_STAGES;
          const uint32_t ph = (it / W_STAGES) & 1u;
          if (!mbar_wait(wempty(s), ph ^ 1u, abort_flag, a.status, a.wait_limit_ns)) {
            ok = false;
            break;
          }
          const int g0 = GROUP == 32 ? 2 * kb : (GROUP == 64 ? kb : kb >> 1);
          constexpr uint32_t sbytes = GROUP == 32 ? 512 : 256;
          mbar_arrive_expect_tx(wfull(s), WBLOCK_BYTES + sbytes);
          bulk_load(w_base + s * W_SLOT, wblk + static_cast<size_t>(kb) * WBLOCK_BYTES,
                    WBLOCK_BYTES, wfull(s));
          bulk_load(w_base + s * W_SLOT + WBLOCK_BYTES, sblk + static_cast<size_t>(g0) * TILE_N,
                    sbytes, wfull(s));
        }
      }
      if (!ok) {
        for (uint32_t i = it > W_STAGES ? it - W_STAGES : 0; i < it; ++i)
          mbar_wait(wfull(i % W_STAGES), (i / W_STAGES) & 1u, never, nullptr, 100000000ull);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------- MMA issue
    if (lane == 0) {
      constexpr uint32_t IDESC = idesc_f16_f32(TILE_N, TILE_M);
      const uint64_t b_desc0 = smem_desc_sw128(act_base);
      uint32_t s = 0, ph = 0;
      uint32_t uses[2] = {0, 0};  // segments committed per accumulator
      int acc = 0;
      bool ok = true;
      Item w;
      for (int j = 0; ok && item_at<TILE_M>(walk, j, w); ++j) {
        uint32_t used = acc == 0 ? uses[0] : uses[1];
        if (!mbar_wait_lean(dempty(acc), (used & 1u) ^ 1u, abort_flag, a.status,
                            a.wait_limit_ns)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + L::ACC_COL + acc * TILE_M;
        int left = kPromoteBlocks;
        for (int kb = w.kb0; kb < w.kb1; ++kb) {
          if (left == 0) {
            // segment boundary: the epilogue promotes, then the MMAs go on
            tc_commit(dfull(acc));
            ++used;
            if (!mbar_wait_lean(dempty(acc), (used & 1u) ^ 1u, abort_flag, a.status,
                                a.wait_limit_ns)) {
              ok = false;
              break;
            }
            tc_fence_after();
            left = kPromoteBlocks;
          }
          --left;
          if (!mbar_wait_lean(full(s), ph, abort_flag, a.status, a.wait_limit_ns)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t b_desc = b_desc0 + ((s * L::ACT_BYTES) >> 4);
          const uint32_t a_tmem = tmem_base + s * T_COLS;
          const uint32_t first = kb != w.kb0;
#pragma unroll
          for (int k16 = 0; k16 < BK / 16; ++k16)
            mma_f16_ts(d_tmem, a_tmem + 8 * k16, b_desc + 2 * k16, IDESC, k16 == 0 ? first : 1u);
          tc_commit(empty(s));
          if (++s == static_cast<uint32_t>(STAGES)) {
            s = 0;
            ph ^= 1u;
          }
        }
        if (!ok) break;
        tc_commit(dfull(acc));
        ++used;
        if (acc == 0) uses[0] = used; else uses[1] = used;
        if (ACC == 2) acc ^= 1;
      }
      tc_commit(drain_bar);  // TMEM is freed only after every MMA completed
      mbar_wait(drain_bar, 0, never, nullptr, 100000000ull);
    }
  } else if (warp < L::FIRST_EPI_WARP) {
    // ---------------------------------------------------------------- dequant
    const uint32_t dgroup = static_cast<uint32_t>(warp - FIRST_DEQ_WARP) >> 2;
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;  // weight column inside the tile
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t total = static_cast<uint32_t>(walk.blocks());
    for (uint32_t it = dgroup; it < total; it += L::DEQ) {
      const int s = it % W_STAGES;
      const int ts = it % STAGES;
      const bool landed = mbar_wait(wfull(s), (it / W_STAGES) & 1u, abort_flag, a.status,
                                    a.wait_limit_ns);
      if (!__all_sync(0xffffffffu, landed)) break;  // a warp leaves as a whole
      const uint32_t wsrc = w_base + s * W_SLOT + row * 16;
      uint4 c0, c1;
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(c0.x), "=r"(c0.y), "=r"(c0.z), "=r"(c0.w)
                   : "r"(wsrc));
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(c1.x), "=r"(c1.y), "=r"(c1.z), "=r"(c1.w)
                   : "r"(wsrc + 2048));
      uint16_t sb0, sb1;
      const uint32_t ssrc = w_base + s * W_SLOT + WBLOCK_BYTES + row * 2;
      asm volatile("ld.shared.u16 %0, [%1];" : "=h"(sb0) : "r"(ssrc));
      if (GROUP == 32)
        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(sb1) : "r"(ssrc + TILE_N * 2));
      else
        sb1 = sb0;
      const uint32_t s0 = half_bits_x2(sb0), s1 = half_bits_x2(sb1);
      uint32_t r[32];
      const uint32_t wv[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t sc = i < 4 ? s0 : s1;
        r[4 * i + 0] = decode_pair<0>(wv[i], sc);
        r[4 * i + 1] = decode_pair<1>(wv[i], sc);
        r[4 * i + 2] = decode_pair<2>(wv[i], sc);
        r[4 * i + 3] = decode_pair<3>(wv[i], sc);
      }
      const bool free = mbar_wait(empty(ts), ((it / STAGES) & 1u) ^ 1u, abort_flag, a.status,
                                  a.wait_limit_ns);
      if (!__all_sync(0xffffffffu, free)) break;
      tc_fence_after();
      tmem_st_32x32b_x32(tmem_base + lane_addr + ts * T_COLS, r);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(full(ts));
      // The packed slot is given back only now: the TMEM store has consumed
      // what was loaded from it. An arrival right after the loads can overtake
      // them (they queue behind the epilogue's global stores, the arrival does
      // not), and the next copy into the slot then overtakes the loads: one
      // 64-k block of some columns was wrong in every second launch of
      // M = 1024, N = 2048, K = 12288, where partial tiles are stored while
      // the pipeline runs.
      __syncwarp();
      if (lane == 0) mbar_arrive(wempty(s));
    }
  } else {
    // --------------------------------------------------------------- epilogue
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
      const int nseg = (w.kb1 - w.kb0 + kPromoteBlocks - 1) / kPromoteBlocks;
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
        mbar_arrive(dempty(acc));
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
          mbar_arrive(release_bar);
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
          mbar_arrive(release_bar);
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
        mbar_arrive(release_bar);
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
