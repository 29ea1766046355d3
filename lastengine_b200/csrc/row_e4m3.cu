// Rows of 8-bit numbers with a scale each, out of float or bfloat16 rows as they are (quantize) or out of the residual stream
// through its RMSNorm (norm):
//   quantize  a = max(max |x|, 2^-100), q = round(448 x / a), s = a / 448
//   norm      x += y, g = x w, r = 1 / sqrt(mean(x^2) + eps), a = max(max |g|, 2^-100), q = round(448 g / a), s = r a / 448
// The norm's factor r is the same for the whole row, so it goes into the scale and the numbers are rounded without it: the sum of
// squares and the largest |g| are one pass, and the row is read once.  A row that holds a number that is not finite (or whose
// squares' sum is not) gets a scale and numbers that are NaN.
//
// Bound by memory: a float row is read and a quarter of its bytes written.  A thread keeps its numbers in registers between the sums and the
// rounding, so a row is read once, with all loads out before the first is used: eight neighbours at a time where rows begin on 16 bytes
// (a warp a row up to 1,024 numbers, a block above), single numbers otherwise; rows of more than 16,384 are read twice.  The largest
// |g| is taken over the bits (for numbers without a sign they order as the numbers do, infinity and NaN on top).
#include "e4m3_common.cuh"

namespace {

struct RowSums {
  float squares;
  uint32_t top;      // bits of the largest |g|
};

// Over the threads of a row: a warp, or the block (up to 1,024 threads); every thread gets the result, added up in the same order.
template <bool WARP>
__device__ __forceinline__ RowSums row_sums(float squares, uint32_t top) {
  squares = warp_sum(squares);
  top = __reduce_max_sync(0xffffffffu, top);
  RowSums r{squares, top};
  if (!WARP) {
    __shared__ float red_s[32];
    __shared__ uint32_t red_t[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = (blockDim.x + 31) >> 5;
    if (lane == 0) red_s[warp] = squares, red_t[warp] = top;
    __syncthreads();
    r = RowSums{0.f, 0u};
    for (int w = 0; w < nw; w++) r.squares += red_s[w], r.top = max(r.top, red_t[w]);
  }
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
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// The row of x that row p of the result is made of; -1 where `rows` names none.
__device__ __forceinline__ long long source_row(const int* rows, int p, int div, int M) {
  if (!rows) return p;
  const int at = rows[p];
  return at >= 0 && at / div < M ? at / div : -1;
}

// V neighbours, of which `n` are there (the others read as zero and are not written); V = 8 at full 16 bytes
template <int V, typename T>
__device__ __forceinline__ void load_some(const T* p, int n, float (&v)[V]) {
  if (V == 8 && n >= V) {
    const float4 a = load4(p), b = load4(p + 4);
    v[0] = a.x, v[1 % V] = a.y, v[2 % V] = a.z, v[3 % V] = a.w, v[4 % V] = b.x, v[5 % V] = b.y, v[6 % V] = b.z, v[7 % V] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < V; i++) v[i] = i < n ? to_f32(p[i]) : 0.f;
  }
}
template <>
__device__ __forceinline__ void load_some<8, bf16>(const bf16* p, int n, float (&v)[8]) {
  if (n >= 8) {
    const uint4 r = *reinterpret_cast<const uint4*>(p);
    const uint32_t u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; i++) v[2 * i] = __uint_as_float(u[i] << 16), v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = i < n ? to_f32(p[i]) : 0.f;
  }
}
template <int V, typename T>
__device__ __forceinline__ void store_some(T* p, int n, const float (&v)[V]) {
  if (V == 8 && n >= V) {
    store4(p, make_float4(v[0], v[1 % V], v[2 % V], v[3 % V]));
    store4(p + 4, make_float4(v[4 % V], v[5 % V], v[6 % V], v[7 % V]));
  } else {
#pragma unroll
    for (int i = 0; i < V; i++)
      if (i < n) p[i] = from_f32<T>(v[i]);
  }
}
template <int V>
__device__ __forceinline__ void store_eight(uint8_t* p, int n, const float (&v)[V], float f) {
  if (V == 8 && n >= V) {
    *reinterpret_cast<uint2*>(p) = make_uint2(f32x4_to_e4m3(v[0] * f, v[1 % V] * f, v[2 % V] * f, v[3 % V] * f),
                                              f32x4_to_e4m3(v[4 % V] * f, v[5 % V] * f, v[6 % V] * f, v[7 % V] * f));
  } else {
#pragma unroll
    for (int i = 0; i < V; i++)
      if (i < n) p[i] = f32_to_e4m3(v[i] * f);
  }
}

// CH pieces of V numbers a thread; ROWS > 1: a warp a row, that many rows a block.  CH = 0: any width, the row read twice.
template <typename TX, int V, int CH, int ROWS>
__global__ void __launch_bounds__(512) quantize_kernel(uint8_t* __restrict__ q, float* __restrict__ scale, const TX* __restrict__ x, const int* __restrict__ rows,
                                const float* __restrict__ weights, int div, int P, int M, int D, long long ldx, long long ldq) {
  const int tid = ROWS > 1 ? threadIdx.x & 31 : threadIdx.x, T = ROWS > 1 ? 32 : blockDim.x;
  const int p = ROWS > 1 ? blockIdx.x * ROWS + (threadIdx.x >> 5) : blockIdx.x;
  pdl_wait();
  if (p >= P) return;
  const long long m = source_row(rows, p, div, M);
  const TX* xi = x + (m < 0 ? 0 : m) * ldx;
  const int width = m < 0 ? 0 : D;      // (a row that is not there: nothing is read)
  float v[CH > 0 ? CH : 1][V];
  uint32_t top = m < 0 ? 0x7fffffffu : 0u;
  if (CH > 0) {
#pragma unroll
    for (int c = 0; c < CH; c++) load_some<V>(xi + (tid + c * T) * V, width - (tid + c * T) * V, v[c]);
#pragma unroll
    for (int c = 0; c < CH; c++)
#pragma unroll
      for (int i = 0; i < V; i++) top = max(top, magnitude(v[c][i]));
  } else {
    for (int i = tid; i < width; i += T) top = max(top, magnitude(to_f32(xi[i])));
  }
  float inv, s;
  row_factor(row_sums<(ROWS > 1)>(0.f, top), inv, s);
  if (tid == 0) scale[p] = weights && m >= 0 ? s * weights[rows[p]] : s;
  uint8_t* o = q + p * ldq;
  if (CH > 0) {
#pragma unroll
    for (int c = 0; c < CH; c++) store_eight<V>(o + (tid + c * T) * V, D - (tid + c * T) * V, v[c], inv);
  } else {
    for (int i = tid; i < D; i += T) o[i] = f32_to_e4m3(m < 0 ? inv : to_f32(xi[i]) * inv);
  }
}

template <int V, int CH, int ROWS>
__global__ void __launch_bounds__(512) rmsnorm_e4m3_kernel(uint8_t* __restrict__ q, float* __restrict__ scale, float* __restrict__ x, const float* __restrict__ w,
                                    const void* __restrict__ y, int y_dtype, void* __restrict__ h, int h_dtype, int M, int D, float eps, long long ldq) {
  const int tid = ROWS > 1 ? threadIdx.x & 31 : threadIdx.x, T = ROWS > 1 ? 32 : blockDim.x;
  const int m = ROWS > 1 ? blockIdx.x * ROWS + (threadIdx.x >> 5) : blockIdx.x;
  pdl_wait();
  if (m >= M) return;
  const size_t at = (size_t)m * D;
  float v[CH > 0 ? CH : 1][V], g[CH > 0 ? CH : 1][V];
  float squares = 0.f;
  uint32_t top = 0u;
  if (CH > 0) {
#pragma unroll
    for (int c = 0; c < CH; c++) load_some<V>(x + at + (tid + c * T) * V, D - (tid + c * T) * V, v[c]);
    if (y) {
      if (y_dtype == LEB_F32) {
#pragma unroll
        for (int c = 0; c < CH; c++) load_some<V>((const float*)y + at + (tid + c * T) * V, D - (tid + c * T) * V, g[c]);
      } else {
#pragma unroll
        for (int c = 0; c < CH; c++) load_some<V>((const bf16*)y + at + (tid + c * T) * V, D - (tid + c * T) * V, g[c]);
      }
#pragma unroll
      for (int c = 0; c < CH; c++) {
#pragma unroll
        for (int i = 0; i < V; i++) v[c][i] += g[c][i];
        store_some<V>(x + at + (tid + c * T) * V, D - (tid + c * T) * V, v[c]);
      }
    }
#pragma unroll
    for (int c = 0; c < CH; c++) load_some<V>(w + (tid + c * T) * V, D - (tid + c * T) * V, g[c]);
#pragma unroll
    for (int c = 0; c < CH; c++)
#pragma unroll
      for (int i = 0; i < V; i++) {
        squares += v[c][i] * v[c][i];
        g[c][i] *= v[c][i];
        top = max(top, magnitude(g[c][i]));
      }
  } else {
    for (int i = tid; i < D; i += T) {
      float a = x[at + i];
      if (y) x[at + i] = a = a + (y_dtype == LEB_F32 ? ((const float*)y)[at + i] : to_f32(((const bf16*)y)[at + i]));
      squares += a * a;
      top = max(top, magnitude(a * w[i]));
    }
  }
  const RowSums t = row_sums<(ROWS > 1)>(squares, top);
  const float r = 1.0f / sqrtf(t.squares / (float)D + eps);
  float inv, s;
  row_factor(t, inv, s);
  if (tid == 0) scale[m] = s * r;
  uint8_t* o = q + m * ldq;
  if (CH > 0) {
#pragma unroll
    for (int c = 0; c < CH; c++) {
      const int i = (tid + c * T) * V;
      store_eight<V>(o + i, D - i, g[c], inv);
      if (h) {
#pragma unroll
        for (int k = 0; k < V; k++) v[c][k] = g[c][k] * r;
        if (h_dtype == LEB_F32) store_some<V>((float*)h + at + i, D - i, v[c]);
        else store_some<V>((bf16*)h + at + i, D - i, v[c]);
      }
    }
  } else {
    for (int i = tid; i < D; i += T) {
      const float a = x[at + i] * w[i];
      o[i] = f32_to_e4m3(a * inv);
      if (h && h_dtype == LEB_F32) ((float*)h)[at + i] = a * r;
      else if (h) ((bf16*)h)[at + i] = from_f32<bf16>(a * r);
    }
  }
}

// How a row of D numbers is shared out: GO(V, CH, ROWS, blocks of rows, threads).
#define ROW_SHAPES(wide, D, rows)                                       \
  if (wide) {                                                           \
    if (D <= 256) GO(8, 1, 8, ceil_div(rows, 8), 256);                  \
    else if (D <= 512) GO(8, 2, 8, ceil_div(rows, 8), 256);             \
    else if (D <= 1024) GO(8, 4, 4, ceil_div(rows, 4), 128);            \
    else if (D <= 2048) GO(8, 1, 1, rows, 256);                         \
    else if (D <= 4096) GO(8, 2, 1, rows, 256);                         \
    else if (D <= 8192) GO(8, 4, 1, rows, 256);                         \
    else if (D <= 16384) GO(8, 4, 1, rows, 512);                        \
    else GO(1, 0, 1, rows, 512);                                        \
  } else {                                                              \
    if (D <= 128) GO(1, 4, 8, ceil_div(rows, 8), 256);                  \
    else if (D <= 1024) GO(1, 8, 1, rows, 128);                         \
    else if (D <= 2048) GO(1, 8, 1, rows, 256);                         \
    else if (D <= 4096) GO(1, 8, 1, rows, 512);                         \
    else if (D <= 8192) GO(1, 16, 1, rows, 512);                        \
    else if (D <= 16384) GO(1, 32, 1, rows, 512);                       \
    else GO(1, 0, 1, rows, 512);                                        \
  }

template <typename TX>
void launch_quantize(bool wide, uint8_t* q, float* scale, const TX* x, const int* rows, const float* weights, int div, int P, int M, int D, long long ldx,
                     long long ldq, cudaStream_t st) {
#define GO(V, CH, ROWS, blocks, threads) \
  leb_launch(quantize_kernel<TX, V, CH, ROWS>, dim3(blocks), dim3(threads), 0, st, q, scale, x, rows, weights, div, P, M, D, ldx, ldq)
  ROW_SHAPES(wide, D, P)
#undef GO
}

// What the entry points take: one packed argument each, numbers of 64 bits in this order (seventeen converted arguments cost a caller in Python
// as much as a small kernel takes).
struct QuantizeArgs {
  long long q, scale, x, x_dtype, rows, weights, div, P, M, D, ldx, ldq;
};
struct NormArgs {
  long long q, scale, x, w, y, y_dtype, h, h_dtype, M, D, ldq;
  double eps;
};
constexpr long long MOST = (1LL << 31) - 65536;      // rows, and numbers of a row

}  // namespace

// q [P, D] 8-bit (rows ldq apart), scale [P]; x [M, D] (rows ldx apart); rows [P] or null (then P = M): row p is x[rows[p] / div], its
// scale times weights[rows[p]] where they are given.
LEB_API int leb_quantize_e4m3(const void* packed, cudaStream_t st) {
  const QuantizeArgs& a = *(const QuantizeArgs*)packed;
  if (a.P <= 0) return 0;
  LEB_REQUIRE(a.D > 0 && a.D < MOST && a.P < MOST && a.M < MOST && a.div > 0 && a.div < MOST, "leb_quantize_e4m3: %lld rows out of %lld of %lld numbers, %lld places to a row", a.P, a.M, a.D, a.div);
  LEB_REQUIRE(a.rows || (a.P == a.M && !a.weights), "leb_quantize_e4m3: %lld rows out of %lld need a list of them", a.P, a.M);
  LEB_REQUIRE(a.x_dtype == LEB_F32 || a.x_dtype == LEB_BF16, "leb_quantize_e4m3: unknown type of x %lld", a.x_dtype);
  const bool wide = (a.x & 15) == 0 && a.ldx % (a.x_dtype == LEB_F32 ? 4 : 8) == 0 && (a.q & 7) == 0 && a.ldq % 8 == 0;
  if (a.x_dtype == LEB_F32)
    launch_quantize(wide, (uint8_t*)a.q, (float*)a.scale, (const float*)a.x, (const int*)a.rows, (const float*)a.weights, (int)a.div, (int)a.P, (int)a.M, (int)a.D, a.ldx, a.ldq, st);
  else
    launch_quantize(wide, (uint8_t*)a.q, (float*)a.scale, (const bf16*)a.x, (const int*)a.rows, (const float*)a.weights, (int)a.div, (int)a.P, (int)a.M, (int)a.D, a.ldx, a.ldq, st);
  LEB_CHECK_LAUNCH("leb_quantize_e4m3");
  return 0;
}

// q [M, D] 8-bit (rows ldq apart), scale [M], x [M, D] float (x += y first where y is given), h [M, D] or null: the normed rows.
LEB_API int leb_rmsnorm_e4m3(const void* packed, cudaStream_t st) {
  const NormArgs& a = *(const NormArgs*)packed;
  if (a.M <= 0) return 0;
  LEB_REQUIRE(a.D > 0 && a.D < MOST && a.M < MOST, "leb_rmsnorm_e4m3: %lld rows of %lld numbers", a.M, a.D);
  LEB_REQUIRE((a.y_dtype == LEB_F32 || a.y_dtype == LEB_BF16) && (a.h_dtype == LEB_F32 || a.h_dtype == LEB_BF16), "leb_rmsnorm_e4m3: unknown type of y (%lld) or h (%lld)", a.y_dtype, a.h_dtype);
  const bool wide = a.D % 8 == 0 && ((a.x | a.w | a.y | a.h) & 15) == 0 && (a.q & 7) == 0 && a.ldq % 8 == 0;
  const int D = (int)a.D;
#define GO(V, CH, ROWS, blocks, threads)                                                                                                                         \
  leb_launch(rmsnorm_e4m3_kernel<V, CH, ROWS>, dim3(blocks), dim3(threads), 0, st, (uint8_t*)a.q, (float*)a.scale, (float*)a.x, (const float*)a.w, (const void*)a.y, \
             (int)a.y_dtype, (void*)a.h, (int)a.h_dtype, (int)a.M, D, (float)a.eps, a.ldq)
  ROW_SHAPES(wide, D, (int)a.M)
#undef GO
  LEB_CHECK_LAUNCH("leb_rmsnorm_e4m3");
  return 0;
}
