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

// Where the decode kernel puts the results: one contiguous matrix.
struct EpilogueOut {
  void* C;       // [M][ldc], half or float
  int ldc, fp32_out, gated;
  Epilogue epilogue;
};

// The hardware's 2^x and 1/x: the steps themselves are within a few FP32 units
// in the last place; subnormals count as zeros. The argument of 2^x is rounded
// to FP32 first, so the relative error of an activation grows with its exponent
// on the negative side, where the value falls towards 0. These steps with an
// exact 2^x and 1/x, largest relative error: SiLU 3.5e-7 down to -5, 1e-6 to
// -20, 3.8e-6 to -86; tanh-GELU 1.1e-6 to -3, 2.8e-6 to -5, 8.5e-6 to -8; GELU
// 6.6e-7 to -3, 1.2e-6 to -5, 7.7e-6 to -13. FP16's rounding is 4.9e-4; only FP32
// results can show it.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kLog2e = 1.44269504f;

// x * sigmoid(x (c0 + c1 x^2)): SiLU is c0 = 1, c1 = 0; tanh-GELU, whose
// 0.5 (1 + tanh(u / 2)) is sigmoid(u), is c0 = sqrt(8/pi), c1 = 0.044715 c0.
// x^2 is capped so that c1 = 0 takes it out for infinite x too (0 times
// infinity is a NaN); tanh-GELU's u is beyond every exponent there anyway.
// +infinity gives +infinity; 1 + exp(-u) overflows to infinity for very
// negative finite x and the product is then the limit, -0.
__device__ __forceinline__ float sigmoid_gate(float x, float c0, float c1) {
  const float u = x * fmaf(c1, fminf(x * x, 1e30f), c0);
  return x * rcp_fast(1.0f + exp2_fast(-kLog2e * u));
}

// GELU x Phi(x) = max(x, 0) - |x| erfc(z) / 2 with z = |x| / sqrt 2: no
// cancellation on the negative side. erfc(z) exp(z^2) is a polynomial of degree
// 8 in t = 1 / (1 + z / 2) (the substitution of Press et al., Numerical Recipes),
// times t, fitted by weighted least squares for the least largest relative error
// (4e-8; 3.3e-7 evaluated in FP32, before the exponential's, see above): 20
// instructions, 5.4 us less than the library's erfc in a product of M = 203,
// K = 4096, N = 14336, whose one wave of tiles hides no epilogue.
__device__ __forceinline__ float gelu_erf(float x) {
  const float a = fminf(fabsf(x), 40.0f);  // exp(-800) is 0: infinities keep their limits
  const float t = rcp_fast(fmaf(a, 0.35355339f, 1.0f));
  float p = -0.05889091f;
  p = fmaf(p, t, 0.28370258f);
  p = fmaf(p, t, -0.48538491f);
  p = fmaf(p, t, 0.27597940f);
  p = fmaf(p, t, -0.02517844f);
  p = fmaf(p, t, 0.20207012f);
  p = fmaf(p, t, 0.24326095f);
  p = fmaf(p, t, 0.28235349f);
  p = fmaf(p, t, 0.28208768f);
  const float h = 0.5f * a * (p * t) * exp2_fast((-0.5f * kLog2e) * a * a);
  return x < 0.0f ? -h : x - h;
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
    for (int i = 0; i < N; ++i) x[i] = gelu_erf(x[i]);
  } else {
    const float c0 = kind == kActSilu ? 1.0f : 1.59576912f;
    const float c1 = kind == kActSilu ? 0.0f : 0.07135482f;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = sigmoid_gate(x[i], c0, c1);
  }
}

}  // namespace i4g
