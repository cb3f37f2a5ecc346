// Host-side interface of expert routing and combination (route.cu).
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstddef>

namespace i4g {
namespace route {

constexpr int kMaxExperts = 512;
constexpr int kMaxTopK = 32;
constexpr int kMaxGroups = 32;

struct Args {
  const void* logits;  // [T][ld], float or half
  size_t ld;
  const float* bias;   // [E], added to the scores for the choice only, or null
  int T, E, top_k;
  int sigmoid;         // else softmax
  int n_group, topk_group, top2;
  int renormalize;
  float scale;
  int* ids;            // [T][top_k]
  float* weights;      // [T][top_k]
  int* offsets;        // [E + 1]
  int* rows;           // [T * top_k]
  int* slots;          // [T][top_k]
};

size_t workspace_bytes(int T, int E, int sm_count);
cudaError_t launch(const Args& a, bool fp32_logits, int sm_count, void* workspace,
                   cudaStream_t stream);
cudaError_t combine(const __half* y, int y_rows, const int* slots, const float* weights,
                    const __half* residual, __half* out, int T, int top_k, int N,
                    cudaStream_t stream);

}  // namespace route
}  // namespace i4g
