#include "gemm_epi.cuh"

template cudaError_t i4g::epi::launch_tile<16>(const CUtensorMap&, bool, int, const Args&, int,
                                                cudaStream_t);
