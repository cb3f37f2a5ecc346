// Host side of the epilogue / experts GEMM kernel: tile height, workspace, grid.
#include "gemm_epi.cuh"

#include <cmath>

namespace i4g {
namespace epi {

// The kernels are built one tile height a file (gemm_epi_<rows>.cu).
#define I4G_EPI_EXTERN(TM)                                                                  \
  extern template cudaError_t launch_tile<TM>(const CUtensorMap&, bool, int, const Args&, int, \
                                              cudaStream_t);
I4G_EPI_EXTERN(16)
I4G_EPI_EXTERN(32)
I4G_EPI_EXTERN(64)
I4G_EPI_EXTERN(128)
I4G_EPI_EXTERN(256)
#undef I4G_EPI_EXTERN

namespace {

// m-tiles of `tile` rows that M rows over E weights make: exact for one weight;
// for experts, what a routing that spreads them at random makes (an expert's
// rows are about normal with the mean as variance).
double m_tiles(int tile, int M, int E) {
  if (E == 1) return (M + tile - 1) / tile;
  const int active = std::min(E, M);
  const double mean = static_cast<double>(M) / active;
  double each = 1.0;
  if (mean > 2.0 * tile) each = mean / tile + 0.5;
  else
    for (int j = 1; j <= 4 && j * tile < mean + 6.0 * std::sqrt(mean); ++j)
      each += 0.5 * std::erfc((j * tile + 0.5 - mean) / std::sqrt(2.0 * mean));
  return active * each;
}

// 64-k blocks that the busiest of `sm_count` CTAs goes through, the tiles they
// are in, and whether the last wave is split along K.
struct Load {
  double blocks, tiles;
  bool split;
};
template <int TILE_M>
Load load_of(double mt, int N, int K, int sm_count) {
  constexpr int BS = Cfg<TILE_M>::BS;
  const int kblocks = K / BK, kunits = (kblocks + BS - 1) / BS;
  const int tiles = static_cast<int>(mt * (N / TILE_N) + 0.5);
  const Sched s = make_sched(tiles, kunits, BS, sm_count, kblocks >= 2 * kMinChunkBlocks,
                             split_overhead_blocks<TILE_M>());
  if (!s.chunks) {
    const int rounds = (tiles + sm_count - 1) / sm_count;
    return {static_cast<double>(rounds) * kblocks, static_cast<double>(rounds), false};
  }
  const int rounds = s.full_tiles / sm_count;
  const int share = (s.tail_tiles * kunits + s.chunks - 1) / s.chunks;
  return {static_cast<double>(rounds) * kblocks + share * BS, rounds + 1.0, true};
}
Load load_of(int tile, double mt, int N, int K, int sm_count) {
  switch (tile) {
    case 16: return load_of<16>(mt, N, K, sm_count);
    case 32: return load_of<32>(mt, N, K, sm_count);
    case 64: return load_of<64>(mt, N, K, sm_count);
    case 128: return load_of<128>(mt, N, K, sm_count);
    default: return load_of<256>(mt, N, K, sm_count);
  }
}

}  // namespace

// A tile height's time in us is a line in the blocks of the busiest CTA: what a
// block costs (more in tall tiles the fuller they are: what L2 delivers to an SM
// bounds those, about 95 KB a us), a split tail and what a tile's end leaves
// uncovered. Fitted to 250 measurements on B200 (dense products of 17 to 1024
// rows, experts of 0.5 to 500 rows each, K 768 to 14336, N 1024 to 28672, back
// to back); the heights it picks are 0.4 % (dense) and 1.2 % (experts) from the
// best of all five in the mean, where the smallest tile that holds the rows is
// 18 % from it. N = K = 4096, 16 / 32 / 64 / 128 / 256 rows a tile: 100 rows
// 19.6 / 14.6 / 14.5 / 19.0 / 27.8 us, 512 rows - / 38.5 / 25.1 / 22.5 / 29.3.
int choose_tile(int M, int E, int N, int K, int sm_count) {
  struct Line {
    int tile;
    double base, block, full_block, split, end;
  };
  static constexpr Line kLines[] = {
      {16, 4.5, 0.106, 0.0, 4.4, 0.8},     {32, 5.7, 0.114, 0.0, 6.2, 1.7},
      {64, 5.7, 0.128, 0.0, 8.6, 1.9},     {128, 6.0, 0.120, 0.088, 13.5, 2.2},
      {256, 6.5, 0.179, 0.203, 15.2, 4.0},
  };
  int best = 256;
  double least = 0.0;
  for (const Line& l : kLines) {
    const double mt = m_tiles(l.tile, M, E);
    const Load w = load_of(l.tile, mt, N, K, sm_count);
    const double full = std::min(1.0, M / (mt * l.tile));  // of a tile's rows
    const double us = l.base + w.blocks * (l.block + l.full_block * full) +
                      (w.split ? l.split : 0.0) + l.end * (w.tiles - 1.0);
    if (l.tile == 16 || us < least) {
      least = us;
      best = l.tile;
    }
  }
  return best;
}

// Inside the product a gather of four rows of 128 bytes holds its copy unit for
// 0.03 us, a block of a tile as many times as its rows need; the copy ahead
// costs a launch and the bytes. Over rows that lie in order already, us more
// inside / ahead: 64 experts of 2048 x 4096, 3 rows each 14.8 / 4.2, 12 rows
// each 48 / 4.3; 8 experts of 4096 x 4096, half a row each 1.1 / 1.6.
bool copy_rows_first(int tile_m, int M, int E, int N, int K, int sm_count) {
  const double mt = m_tiles(tile_m, M, E);
  const double quads = std::max(1.0, 0.25 * M / mt + 0.5);
  const double inside = 0.03 * quads * load_of(tile_m, mt, N, K, sm_count).blocks;
  return inside > 3.5 + 4.0 * M * K / 9e6;
}

// Both kernels' times in us, as lines through measurements on B200 (back-to-back
// calls, g128): each in the 64-k blocks of its busiest SM. Decode / this kernel
// at M = 8: N = K = 4096 5.5 / 11.0; K = 14336, N = 4096 11.2 / 16.3; K = 4096,
// N = 14336 11.4 / 13.4, N = 28672 19.2 / 19.5; K = 8192, N = 28672 35 / 32. At
// M = 16 the decode kernel's second row of fragments costs it a quarter more
// (K = 4096, N = 14336 13.8 / 13.4, N = 28672 24 / 19.5).
bool decode_is_faster(int M, int N, int K, int sm_count) {
  if (M > dec::MAX_M) return false;
  const int kblocks = K / BK;
  const long tiles = N / TILE_N;
  const int cluster = dec::choose_cluster(N, K, sm_count);
  const long ctas = (tiles * cluster + sm_count - 1) / sm_count;  // of the busiest SM
  const long blocks = ctas * ((kblocks + cluster - 1) / cluster);
  const double decode = M <= 8 ? 3.9 + 0.1185 * blocks : 4.2 + 0.15 * blocks;
  using L = Cfg<16>;
  const int kunits = (kblocks + L::BS - 1) / L::BS;
  const Sched s = make_sched(static_cast<int>(tiles), kunits, L::BS, sm_count, true,
                             split_overhead_blocks<16>());
  const long whole = (s.full_tiles + sm_count - 1) / sm_count * kblocks;
  const long share = s.chunks ? (static_cast<long>(s.tail_tiles) * kblocks + s.chunks - 1) / s.chunks
                              : 0;
  return decode < 8.0 + 0.09 * (whole + share) + (s.chunks ? 6.0 : 0.0);
}

int box_blocks(int tile_m) {
  switch (tile_m) {
    case 16: return Cfg<16>::BS;
    case 32: return Cfg<32>::BS;
    case 64: return Cfg<64>::BS;
    case 128: return Cfg<128>::BS;
    default: return Cfg<256>::BS;
  }
}

namespace {

// A warp copies 2 KB of a row, four 16-byte loads a lane in flight.
constexpr int kGatherThreads = 256;
constexpr int kGatherPiece = 1024;  // halves

__global__ void __launch_bounds__(kGatherThreads)
    gather_rows_kernel(const __half* __restrict__ A, int a_rows, const int* __restrict__ offsets,
                       const int* __restrict__ rows, int row_div, __half* __restrict__ out, int M,
                       int E, int K) {
  grid_dependency_wait();
  if (threadIdx.x == 0) launch_dependents();
  const int lane = threadIdx.x & 31;
  const int pieces = (K + kGatherPiece - 1) / kGatherPiece;
  const long long end = static_cast<long long>(min(max(offsets[E], 0), M)) * pieces;
  const int warps = gridDim.x * (kGatherThreads / 32);
  for (long long i = blockIdx.x * (kGatherThreads / 32) + (threadIdx.x >> 5); i < end;
       i += warps) {
    const int p = static_cast<int>(i / pieces);
    const int k0 = static_cast<int>(i - static_cast<long long>(p) * pieces) * kGatherPiece;
    const int r = rows[p] / row_div;
    const bool has = rows[p] >= 0 && r < a_rows;  // rows outside A read as zeros
    const uint4* src =
        reinterpret_cast<const uint4*>(A + static_cast<size_t>(has ? r : 0) * K + k0);
    uint4* dst = reinterpret_cast<uint4*>(out + static_cast<size_t>(p) * K + k0);
    const int n = min(kGatherPiece, K - k0) / 8;
    uint4 v[kGatherPiece / 256];
#pragma unroll
    for (int q = 0; q < kGatherPiece / 256; ++q)
      v[q] = has && lane + 32 * q < n ? src[lane + 32 * q] : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int q = 0; q < kGatherPiece / 256; ++q)
      if (lane + 32 * q < n) dst[lane + 32 * q] = v[q];
  }
}

}  // namespace

cudaError_t gather_rows(const __half* A, int a_rows, const int* offsets, const int* rows,
                        int row_div, __half* out, int M, int E, int K, int sm_count,
                        cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  const long long pieces = static_cast<long long>(M) * ((K + kGatherPiece - 1) / kGatherPiece);
  constexpr int kWarps = kGatherThreads / 32;
  cfg.gridDim = dim3(
      static_cast<unsigned>(std::min<long long>(sm_count * 8, (pieces + kWarps - 1) / kWarps)));
  cfg.blockDim = dim3(kGatherThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, gather_rows_kernel, A, a_rows, offsets, rows, row_div, out, M, E,
                            K);
}

long tiles_bound(int tile_m, int M, int E, int N) {
  // each expert's last tile may be partial, and no more experts than rows have any
  const long extra = std::min(E, M);
  const long m_tiles = E == 1 ? (M + tile_m - 1) / tile_m : M / tile_m + extra;
  return m_tiles * (N / TILE_N);
}

size_t workspace_bytes(int tile_m, long tiles, int K, int sm_count) {
  const int kblocks = K / BK;
  if (kblocks < 2 * kMinChunkBlocks) return 0;  // too short to cut
  // at most sm_count - 1 tail tiles and sm_count shares, or a tail of all
  // `tiles` and kMaxShares shares of each
  const long tail = std::min<long>(tiles, sm_count - 1);
  const long shares = std::min<long>(sm_count, tail * kMaxShares);
  return tc::kTicketBytes +
         static_cast<size_t>(tail + shares) * static_cast<size_t>(tile_m) * TILE_N * 4;
}

int grid_for(int tile_m, long tiles, int K, int sm_count, bool split) {
  const long most = split ? tiles * std::max(1, std::min(kMaxShares, K / BK / kMinChunkBlocks))
                          : tiles;
  return static_cast<int>(std::max<long>(1, std::min<long>(most, sm_count)));
}

Sched schedule(int tile_m, long tiles, long tiles_most, int K, int sm_count) {
  const bool split = workspace_bytes(tile_m, tiles_most, K, sm_count) > 0;
  const int grid = grid_for(tile_m, tiles_most, K, sm_count, split);
  const int bs = box_blocks(tile_m), kunits = (K / BK + bs - 1) / bs;
  const int overhead = tile_m == 256   ? split_overhead_blocks<256>()
                       : tile_m >= 64  ? split_overhead_blocks<64>()
                                       : split_overhead_blocks<16>();
  return make_sched(static_cast<int>(tiles), kunits, bs, grid, split, overhead);
}

cudaError_t launch(const CUtensorMap& act_map, int tile_m, bool gated, int group, const Args& args,
                   int grid, cudaStream_t stream) {
  switch (tile_m) {
    case 16: return launch_tile<16>(act_map, gated, group, args, grid, stream);
    case 32: return launch_tile<32>(act_map, gated, group, args, grid, stream);
    case 64: return launch_tile<64>(act_map, gated, group, args, grid, stream);
    case 128: return launch_tile<128>(act_map, gated, group, args, grid, stream);
    case 256: return launch_tile<256>(act_map, gated, group, args, grid, stream);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace epi
}  // namespace i4g
