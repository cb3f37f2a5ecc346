// Host side of the epilogue / experts GEMM kernel: tile height, workspace, grid.
#include "gemm_epi.cuh"

namespace i4g {
namespace epi {

// Smallest tile that holds the rows of one weight: below 256 rows the time is
// the weights' (read and dequantised once per m-tile), not the MMAs'.
int choose_tile(int rows) {
  for (int t = 16; t < 256; t *= 2)
    if (rows <= t) return t;
  return 256;
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

// One row per warp, 16 bytes a lane: bound by the bytes it writes. The row
// gather inside the product costs about 70 cycles of the copy unit for four
// rows of 128 bytes, which for 64 rows a tile is more than the block's MMAs.
constexpr int kGatherThreads = 256;

__global__ void __launch_bounds__(kGatherThreads)
    gather_rows_kernel(const __half* __restrict__ A, int a_rows, const int* __restrict__ offsets,
                       const int* __restrict__ rows, int row_div, __half* __restrict__ out, int M,
                       int E, int K) {
  grid_dependency_wait();
  if (threadIdx.x == 0) launch_dependents();
  const int lane = threadIdx.x & 31;
  const int end = min(max(offsets[E], 0), M);
  const int warps = gridDim.x * (kGatherThreads / 32);
  for (int p = blockIdx.x * (kGatherThreads / 32) + (threadIdx.x >> 5); p < end; p += warps) {
    const int r = rows[p] / row_div;
    const bool has = rows[p] >= 0 && r < a_rows;  // rows outside A read as zeros
    const uint4* src = reinterpret_cast<const uint4*>(A + static_cast<size_t>(has ? r : 0) * K);
    uint4* dst = reinterpret_cast<uint4*>(out + static_cast<size_t>(p) * K);
#pragma unroll 8
    for (int c = lane; c < K / 8; c += 32) dst[c] = has ? src[c] : make_uint4(0, 0, 0, 0);
  }
}

}  // namespace

cudaError_t gather_rows(const __half* A, int a_rows, const int* offsets, const int* rows,
                        int row_div, __half* out, int M, int E, int K, int sm_count,
                        cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(std::min(sm_count * 8, (M + kGatherThreads / 32 - 1) / (kGatherThreads / 32)));
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
