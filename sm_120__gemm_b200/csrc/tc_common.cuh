// Device pieces shared by the tcgen05 GEMM kernels: tile order, TMEM loads and
// the promotion of an accumulator into a running FP32 sum.
#pragma once

#include "ptx.cuh"

#include <cuda_fp8.h>

namespace i4g {
namespace tc {

constexpr int GROUP_M = 8;                     // rasterisation band (m-tiles)

__device__ __forceinline__ void tile_coords(int tile, int num_m, int num_n, int& mt, int& nt) {
  // Bands of GROUP_M m-tiles, walked n-major inside a band, so that the
  // activation rows of a band and a run of weight blocks stay in L2.
  const int band_tiles = GROUP_M * num_n;
  const int band = tile / band_tiles;
  const int first_m = band * GROUP_M;
  const int band_m = min(GROUP_M, num_m - first_m);
  const int within = tile - band * band_tiles;
  mt = first_m + within % band_m;
  nt = within / band_m;
}

__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
        "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

__device__ __forceinline__ void tmem_ld_wait16(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                 "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

// Running sum of promotion. Its high part H is kept coarse, in FP8 (e5m2,
// saturating), four values per 32-bit register: any H leaves the remainder
// S - H exact in FP32 (S has 24 significant bits, H 3 at the same or the next
// exponent), and a coarse H costs the epilogue warps few registers.
__device__ __forceinline__ float2 e5m2x2_to_float2(uint32_t pair) {
  const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(pair),
                                                   __NV_E5M2);
  __half2 h;
  memcpy(&h, &r, sizeof(h));
  return __half22float2(h);
}

__device__ __forceinline__ uint32_t float2_to_e5m2x2(float lo, float hi) {
  return static_cast<uint32_t>(
      __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E5M2));
}

// H of accumulator columns 4q .. 4q+3 of one lane, from word q of hb.
__device__ __forceinline__ void high_parts(uint32_t w, float (&h)[4]) {
  const float2 a = e5m2x2_to_float2(w & 0xFFFFu), b = e5m2x2_to_float2(w >> 16);
  h[0] = a.x;
  h[1] = a.y;
  h[2] = b.x;
  h[3] = b.y;
}

// Promotes 16 accumulator columns at taddr (hb words 0..3), read with one
// load wait: S = H + D (one FP32 rounding per value), H <- e5m2(S),
// D <- S - H (exact), stored back.
__device__ __forceinline__ void promote_chunk16(uint32_t taddr, uint32_t* hb) {
  uint32_t v[16];
  tmem_ld_32x32b_x16(taddr, v);
  tmem_ld_wait16(v);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float h[4], sum[4];
    high_parts(hb[q], h);
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] = h[i] + __uint_as_float(v[4 * q + i]);
    hb[q] = float2_to_e5m2x2(sum[0], sum[1]) | (float2_to_e5m2x2(sum[2], sum[3]) << 16);
    high_parts(hb[q], h);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[4 * q + i] = __float_as_uint(sum[i] - h[i]);
  }
  uint32_t a[8], b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    a[i] = v[i];
    b[i] = v[8 + i];
  }
  tmem_st_32x32b_x8(taddr, a);
  tmem_st_32x32b_x8(taddr + 8, b);
}

// Final read of 16 accumulator columns (hb words 0..3): v = H + D in FP32.
__device__ __forceinline__ void load_sum16(uint32_t taddr, const uint32_t* hb, uint32_t (&v)[16]) {
  tmem_ld_32x32b_x16(taddr, v);
  tmem_ld_wait16(v);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float h[4];
    high_parts(hb[q], h);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[4 * q + i] = __float_as_uint(h[i] + __uint_as_float(v[4 * q + i]));
  }
}

// Moves words 4.. of a running-sum array down by four, so that a rolled loop
// over 16-column chunks always reads words 0..3 (static register indices).
template <int NW>
__device__ __forceinline__ void shift_down4(uint32_t (&hb)[NW]) {
#pragma unroll
  for (int q = 0; q + 4 < NW; ++q) hb[q] = hb[q + 4];
}

// Rotates a running-sum array down by two words (the first two move to the
// end), so that a rolled loop over 8-column chunks always updates words 0, 1
// and a full pass leaves the array in its original order.
template <int NW>
__device__ __forceinline__ void rotate_down2(uint32_t (&hb)[NW]) {
  const uint32_t w0 = hb[0], w1 = hb[1];
#pragma unroll
  for (int q = 0; q + 2 < NW; ++q) hb[q] = hb[q + 2];
  hb[NW - 2] = w0;
  hb[NW - 1] = w1;
}

}  // namespace tc
}  // namespace i4g
