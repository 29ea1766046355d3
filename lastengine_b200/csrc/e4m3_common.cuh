// What the kernels of 8-bit numbers (e4m3: sign, four bits of exponent, three of fraction, largest 448) share.
//
// A row of 8-bit numbers q comes with a float scale s and stands for s q.  A product of such rows is
//   z[m, n] = (sum_k qx[m, k] qw[n, k]) sx[m] sw[n]
// with the sum in float: products of two such numbers have at most eight significant bits and are exact.
#pragma once
#include <cuda_fp8.h>

#include "common.cuh"

#define E4M3_TOP 448.0f
#define E4M3_LEAST 7.888609052210118e-31f      // 2^-100: what a row's largest number counts as at least

__device__ __forceinline__ float e4m3_to_f32(uint8_t v) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)v, __NV_E4M3)));
}
__device__ __forceinline__ uint8_t f32_to_e4m3(float v) { return (uint8_t)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3); }
__device__ __forceinline__ uint32_t f32x4_to_e4m3(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

// act(gate) * up of n values each, into the gates.  The activation is looked at once: looked at for every value it kept the values' chains of
// instructions apart, one behind the other (pairs of SMs, 8,191 rows x 21,504 x 2,048: 280 us).
template <typename TC, int N>
__device__ __forceinline__ void gate_all(float* g, const float* u, int act) {
  if (act == 0) {
#pragma unroll
    for (int i = 0; i < N; i++) g[i] = gate_mul<TC>(g[i], u[i], 0);
  } else if (act == 1) {
#pragma unroll
    for (int i = 0; i < N; i++) g[i] = gate_mul<TC>(g[i], u[i], 1);
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) g[i] = gate_mul<TC>(g[i], u[i], (act & ~255) | 2);
  }
}

// What an entry point of the products checks of its epilogue (0 store, 1 add into float C, 2 gated over rows of W interleaved in
// blocks of 16; an activation above it as in the bfloat16 products); returns the message or null.
static inline const char* e4m3_epilogue_fault(int act, int epilogue, int c_dtype, int N) {
  if (c_dtype != LEB_F32 && c_dtype != LEB_BF16) return "unknown type of C";
  if (epilogue < 0 || epilogue > 2 || !(LEB_GATE_ACT_OK(act, epilogue) || (LEB_PLAIN_ACT_OK(act, epilogue) && c_dtype == LEB_BF16)))
    return "unknown epilogue, or an activation that does not go with it";
  if (epilogue == 1 && c_dtype != LEB_F32) return "adding needs a float C";
  if (epilogue == 2 && N % 32 != 0) return "the gated epilogue needs rows of W in blocks of 32";
  return nullptr;
}
