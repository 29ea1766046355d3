// Rows of 8-bit numbers with a scale each, out of float or bfloat16 rows as they are (quantize) or out of the residual stream
// through its RMSNorm (norm):
//   quantize  a = max(max |x|, 2^-100), q = round(448 x / a), s = a / 448
//   norm      x += y, g = x w, r = 1 / sqrt(mean(x^2) + eps), a = max(max |g|, 2^-100), q = round(448 g / a), s = r a / 448
// The norm's factor r is the same for the whole row, so it goes into the scale and the numbers are rounded without it: the sum of
// squares and the largest |g| are one pass, and the row is read once.  A row that holds a number that is not finite (or whose
// squares' sum is not) gets a scale and numbers that are NaN.
//
// Bound by memory: a float row is read and a quarter of its bytes written.  The largest |g| is taken over the bits (for numbers
// without a sign they order as the numbers do, infinity and NaN on top).
#include "e4m3_common.cuh"

namespace {

struct RowSums {
  float squares;
  uint32_t top;      // bits of the largest |g|
};

// Over a block of up to 1024 threads; every thread gets the result, added up in the same order.
__device__ __forceinline__ RowSums block_sums(float squares, uint32_t top, float* red_s, uint32_t* red_t) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = (blockDim.x + 31) >> 5;
  squares = warp_sum(squares);
  top = __reduce_max_sync(0xffffffffu, top);
  if (lane == 0) red_s[warp] = squares, red_t[warp] = top;
  __syncthreads();
  RowSums r{0.f, 0u};
  for (int w = 0; w < nw; w++) r.squares += red_s[w], r.top = max(r.top, red_t[w]);
  return r;
}

// The factor on a row's numbers before they are rounded, and the scale that takes it back (without the norm's r).
__device__ __forceinline__ void row_factor(RowSums t, float& inv, float& scale) {
  if (t.top >= 0x7f800000u || !isfinite(t.squares)) {
    inv = scale = __int_as_float(0x7fffffff);
    return;
  }
  const float a = fmaxf(__uint_as_float(t.top), E4M3_LEAST);
  inv = E4M3_TOP / a;
  scale = a / E4M3_TOP;
}

// The row of x that row p of the result is made of; -1 where `rows` names none.
__device__ __forceinline__ long long source_row(const int* rows, int p, int div, int M) {
  if (!rows) return p;
  const int at = rows[p];
  return at >= 0 && at / div < M ? at / div : -1;
}

// Any width, any alignment: a block per row, the row read twice.
template <typename TX>
__global__ void __launch_bounds__(256) quantize_any_kernel(uint8_t* __restrict__ q, float* __restrict__ scale, const TX* __restrict__ x,
                                                           const int* __restrict__ rows, const float* __restrict__ weights, int div, int M, int D,
                                                           long long ldx, long long ldq) {
  __shared__ float red_s[8];
  __shared__ uint32_t red_t[8];
  pdl_wait();
  const int p = blockIdx.x;
  const long long m = source_row(rows, p, div, M);
  const TX* xi = x + (m < 0 ? 0 : m) * ldx;
  uint32_t top = m < 0 ? 0x7fffffffu : 0u;
  if (m >= 0)
    for (int i = threadIdx.x; i < D; i += 256) top = max(top, __float_as_uint(to_f32(xi[i])) & 0x7fffffffu);
  float inv, s;
  row_factor(block_sums(0.f, top, red_s, red_t), inv, s);
  if (threadIdx.x == 0) scale[p] = weights && m >= 0 ? s * weights[rows[p]] : s;
  uint8_t* o = q + p * ldq;
  for (int i = threadIdx.x; i < D; i += 256) o[i] = f32_to_e4m3(m < 0 ? inv : to_f32(xi[i]) * inv);
}

template <typename TY, typename TH>
__global__ void __launch_bounds__(256) rmsnorm_e4m3_any_kernel(uint8_t* __restrict__ q, float* __restrict__ scale, float* __restrict__ x,
                                                               const float* __restrict__ w, const TY* __restrict__ y, TH* __restrict__ h, int D,
                                                               float eps, long long ldq) {
  __shared__ float red_s[8];
  __shared__ uint32_t red_t[8];
  pdl_wait();
  const size_t at = (size_t)blockIdx.x * D;
  float squares = 0.f;
  uint32_t top = 0u;
  for (int i = threadIdx.x; i < D; i += 256) {
    float v = x[at + i];
    if (y) x[at + i] = v = v + to_f32(y[at + i]);
    squares += v * v;
    top = max(top, __float_as_uint(v * w[i]) & 0x7fffffffu);
  }
  const RowSums t = block_sums(squares, top, red_s, red_t);
  const float r = 1.0f / sqrtf(t.squares / (float)D + eps);
  float inv, s;
  row_factor(t, inv, s);
  if (threadIdx.x == 0) scale[blockIdx.x] = s * r;
  uint8_t* o = q + blockIdx.x * ldq;
  for (int i = threadIdx.x; i < D; i += 256) {
    const float g = x[at + i] * w[i];
    o[i] = f32_to_e4m3(g * inv);
    if (h) h[at + i] = from_f32<TH>(g * r);
  }
}

}  // namespace

// q [P, D] 8-bit (rows ldq apart), scale [P]; x [M, D] (rows ldx apart); rows [P] or null (then P = M): row p is x[rows[p] / div], its
// scale times weights[rows[p]] where they are given.
LEB_API int leb_quantize_e4m3(void* q, float* scale, const void* x, int x_dtype, const int* rows, const float* weights, int div, int P, int M, int D,
                              long long ldx, long long ldq, cudaStream_t st) {
  if (P <= 0) return 0;
  LEB_REQUIRE(D > 0 && div > 0, "leb_quantize_e4m3: rows of %d numbers, %d places to a row", D, div);
  LEB_REQUIRE(rows || (P == M && !weights), "leb_quantize_e4m3: %d rows out of %d need a list of them", P, M);
  if (x_dtype == LEB_F32)
    leb_launch(quantize_any_kernel<float>, dim3(P), dim3(256), 0, st, (uint8_t*)q, scale, (const float*)x, rows, weights, div, M, D, ldx, ldq);
  else if (x_dtype == LEB_BF16)
    leb_launch(quantize_any_kernel<bf16>, dim3(P), dim3(256), 0, st, (uint8_t*)q, scale, (const bf16*)x, rows, weights, div, M, D, ldx, ldq);
  else
    return leb_fail("leb_quantize_e4m3: unknown type of x %d", x_dtype);
  LEB_CHECK_LAUNCH("leb_quantize_e4m3");
  return 0;
}

// q [M, D] 8-bit (rows ldq apart), scale [M], x [M, D] float (x += y first where y is given), h [M, D] or null: the normed rows.
LEB_API int leb_rmsnorm_e4m3(void* q, float* scale, float* x, const float* w, const void* y, int y_dtype, void* h, int h_dtype, int M, int D,
                             float eps, long long ldq, cudaStream_t st) {
  if (M <= 0) return 0;
  LEB_REQUIRE(D > 0, "leb_rmsnorm_e4m3: rows of %d numbers", D);
  LEB_REQUIRE((y_dtype == LEB_F32 || y_dtype == LEB_BF16) && (h_dtype == LEB_F32 || h_dtype == LEB_BF16), "leb_rmsnorm_e4m3: unknown type of y (%d) or h (%d)", y_dtype, h_dtype);
#define GO(TY, TH) leb_launch(rmsnorm_e4m3_any_kernel<TY, TH>, dim3(M), dim3(256), 0, st, (uint8_t*)q, scale, x, w, (const TY*)y, (TH*)h, D, eps, ldq)
  if (y_dtype == LEB_F32) {
    if (h_dtype == LEB_F32) GO(float, float); else GO(float, bf16);
  } else {
    if (h_dtype == LEB_F32) GO(bf16, float); else GO(bf16, bf16);
  }
#undef GO
  LEB_CHECK_LAUNCH("leb_rmsnorm_e4m3");
  return 0;
}
