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
