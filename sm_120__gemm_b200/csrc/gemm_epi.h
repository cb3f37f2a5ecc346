// Host-side interface of the epilogue / experts GEMM kernel (gemm_epi.cuh).
#pragma once

#include "epilogue.cuh"
#include "gemm_tc.h"

namespace i4g {
namespace epi {

constexpr int kMaxExperts = 512;

// One launch: a dense product (offsets == nullptr: M rows of A, one weight) or
// the products of sorted rows with their experts' weights (rows offsets[e] ..
// offsets[e + 1] - 1 of C belong to expert e; M bounds them).
struct Args {
  const uint8_t* tiles;    // [E] weights in the tile layout
  const __half* scales;    // [E] scales in the 128-column layout
  void* C;                 // [M][N], gated: [M][N / 2]; half or float
  const int* offsets;      // [E + 1] or null
  const int* rows;         // pair of each sorted row (its row of A is
                           // rows[p] / row_div), or null: row p of A
  int row_div;
  int E, M, N, K;
  int fp32_out;
  Epilogue epilogue;
  uint32_t* tickets;       // split tail (null: whole tiles only)
  float* partials;
  int* status;
  unsigned long long wait_limit_ns;
};

// How the tiles of a launch are shared out over `units` CTAs: whole tiles,
// round robin, then the tail_tiles tiles of the last, partial wave cut along K
// into `chunks` equal runs of 64-k blocks, one per CTA.
struct Sched {
  int full_tiles, tail_tiles, chunks;
};

// Activation rows per tile (16, 32, 64, 128, 256) for M rows, of one weight or
// spread over E experts.
int choose_tile(int M, int E, int N, int K, int sm_count);
// Whether the decode kernel's cluster schedule serves a dense product faster.
bool decode_is_faster(int M, int N, int K, int sm_count);
// Whether gathered activations are first copied into row order by a kernel of
// their own (gather_rows) instead of four rows per copy instruction inside the
// product.
bool copy_rows_first(int tile_m, int M, int E, int N, int K, int sm_count);
// 64-k blocks of the activation box of a tile height.
int box_blocks(int tile_m);
// out[p] = A[rows[p] / row_div] for p < offsets[E]; K halves a row.
cudaError_t gather_rows(const __half* A, int a_rows, const int* offsets, const int* rows,
                        int row_div, __half* out, int M, int E, int K, int sm_count,
                        cudaStream_t stream);
// Most tiles a launch can have (rows spread over E weights in the worst way).
long tiles_bound(int tile_m, int M, int E, int N);
// Workspace of the split tail for any number of tiles (0: nothing to split).
size_t workspace_bytes(int tile_m, long tiles, int K, int sm_count);
int grid_for(int tile_m, long tiles, int K, int sm_count, bool split);
// The schedule a launch of `tiles` tiles finds when its grid and workspace are
// for `tiles_most`.
Sched schedule(int tile_m, long tiles, long tiles_most, int K, int sm_count);
cudaError_t launch(const CUtensorMap& act_map, int tile_m, bool gated, int group, const Args& args,
                   int grid, cudaStream_t stream);
// The instances of one tile height (one translation unit each).
template <int TILE_M>
cudaError_t launch_tile(const CUtensorMap& act_map, bool gated, int group, const Args& args,
                        int grid, cudaStream_t stream);

}  // namespace epi
}  // namespace i4g
