// The fused epilogue: what happens to a sum of the GEMM before it is rounded.
//
//   y = act(x + bias)                  plain
//   y = act(g + bias_g) * (u + bias_u)  gated: g and u are columns 8 apart in
//                                      a group of 16 (8 gates, their 8 ups)
//   C = round(y + residual)
//
// All of it runs in FP32 on the FP32 sums; the one rounding is the store to C.
#pragma once

#include <cuda_fp16.h>
#include <cstdint>

namespace i4g {

// Values of i4g_activation (i4g.h).
constexpr int kActNone = 0, kActRelu = 1, kActSilu = 2, kActGelu = 3, kActGeluTanh = 4;
constexpr int kNumActivations = 5;

struct Epilogue {
  const __half* bias;      // [N] (per expert: [E][N]), or null
  const __half* residual;  // [M][ldr] at the output's columns, or null
  int ldr;
  int activation;
};

// x * sigmoid(x (c0 + c1 x^2)): SiLU is c0 = 1, c1 = 0; tanh-GELU, whose
// 0.5 (1 + tanh(u / 2)) is sigmoid(u), is c0 = sqrt(8/pi), c1 = 0.044715 c0.
// 1 + exp(-u) overflows to infinity for very negative u and the quotient is
// then the limit, -0. The fast exp and divide are each within a few FP32
// units in the last place here, far below the rounding to FP16.
__device__ __forceinline__ float sigmoid_gate(float x, float c0, float c1) {
  const float u = x * fmaf(c1 * x, x, c0);
  return __fdividef(x, 1.0f + __expf(-u));
}

// Applies the activation to N values; the kind is the same for every thread,
// so the branch is taken once for all of them.
template <int N>
__device__ __forceinline__ void activate(int kind, float (&x)[N]) {
  if (kind == kActNone) return;
  if (kind == kActRelu) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = x[i] < 0.0f ? 0.0f : x[i];  // keeps a NaN
  } else if (kind == kActGelu) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = 0.5f * x[i] * erfcf(x[i] * -0.70710678f);
  } else {
    const float c0 = kind == kActSilu ? 1.0f : 1.59576912f;
    const float c1 = kind == kActSilu ? 0.0f : 0.07135482f;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = sigmoid_gate(x[i], c0, c1);
  }
}

}  // namespace i4g
