// Rows of 8-bit numbers with a scale each, out of float or bfloat16 rows as they are (quantize) or out of the residual stream
// through its RMSNorm (norm):
//   quantize  a = max(max |x|, 2^-100), q = round(448 x / a), s = a / 448
//   norm      x += y, g = x w, r = 1 / sqrt(mean(x^2) + eps), a = max(max |g|, 2^-100), q = round(448 g / a), s = r a / 448
// The norm's factor r is the same for the whole row, so it goes into the scale and the numbers are rounded without it: the sum of
// squares and the largest |g| are one pass, and the row is read once.  A row that holds a number that is not finite (or whose
// squares' sum is not) gets a scale and numbers that are NaN.
//
// Bound by memory: a float row is read and a quarter of its bytes written.  A thread keeps its numbers in registers between the sums and the
// rounding, so a row is read once, with all loads out before the first is used: eight neighbours at a time where rows begin on 16 bytes,
// single numbers (four of a thread side by side, so that they are written as one word) otherwise; rows of more than 16,384 are read twice, a number
// at a time (2,048 bfloat16 rows of 28,672: 151 us, 27 by their bytes).  The largest
// |g| is taken over the bits (for numbers without a sign they order as the numbers do, infinity and NaN on top).
#include "e4m3_common.cuh"

namespace {

struct RowSums {
  float squares;
  uint32_t top;      // bits of the largest |g|
};

// Over the threads of a row: a warp, or the block (up to 512 threads); every thread gets the result, added up in the same order.
template <bool WARP>
__device__ __forceinline__ RowSums row_sums(float squares, uint32_t top) {
  squares = warp_sum(squares);
  top = __reduce_max_sync(0xffffffffu, top);
  RowSums r{squares, top};
  if (!WARP) {
    __shared__ float red_s[16];
    __shared__ uint32_t red_t[16];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = (blockDim.x + 31) >> 5;
    if (nw == 1) return r;
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

// V neighbours of a row as they lie in memory, of which `n` are there (the others read as zero and are not written).
template <typename T, int V>
struct Some {
  T v[V];
  __device__ __forceinline__ void load(const T* p, int n, bool = false) {
#pragma unroll
    for (int i = 0; i < V; i++) v[i] = i < n ? p[i] : from_f32<T>(0.f);
  }
  __device__ __forceinline__ uint32_t top() const {
    uint32_t t = 0u;
#pragma unroll
    for (int i = 0; i < V; i++) t = max(t, magnitude(to_f32(v[i])));
    return t;
  }
  __device__ __forceinline__ float at(int i) const { return to_f32(v[i]); }
};
// Sixteen bytes that nobody reads again, past L1.
__device__ __forceinline__ float4 load4_once(const float* p) {
  float4 v;
  asm volatile("ld.global.L1::no_allocate.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p) : "memory");
  return v;
}
template <>
struct Some<float, 8> {
  float v[8];
  __device__ __forceinline__ void load(const float* p, int n, bool once = false) {
    if (n >= 8) {
      const float4 a = once ? load4_once(p) : load4(p), b = once ? load4_once(p + 4) : load4(p + 4);
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = i < n ? p[i] : 0.f;
    }
  }
  __device__ __forceinline__ uint32_t top() const {
    uint32_t t = 0u;
#pragma unroll
    for (int i = 0; i < 8; i++) t = max(t, magnitude(v[i]));
    return t;
  }
  __device__ __forceinline__ float at(int i) const { return v[i]; }
};
template <>
struct Some<bf16, 8> {      // two numbers a word
  uint32_t u[4];
  __device__ __forceinline__ void load(const bf16* p, int n, bool = false) {
    if (n >= 8) {
      const uint4 r = *reinterpret_cast<const uint4*>(p);
      u[0] = r.x, u[1] = r.y, u[2] = r.z, u[3] = r.w;
    } else {
      const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
      for (int i = 0; i < 4; i++) u[i] = (2 * i < n ? (uint32_t)h[2 * i] : 0u) | (2 * i + 1 < n ? (uint32_t)h[2 * i + 1] << 16 : 0u);
    }
  }
  __device__ __forceinline__ uint32_t top() const {
    uint32_t t = 0u;
#pragma unroll
    for (int i = 0; i < 4; i++) t = __vmaxu2(t, u[i] & 0x7fff7fffu);
    return max(t << 16, t & 0xffff0000u);
  }
  __device__ __forceinline__ float at(int i) const { return __uint_as_float(i & 1 ? u[i >> 1] & 0xffff0000u : u[i >> 1] << 16); }
};
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
__device__ __forceinline__ void store_eight(uint8_t* p, int n, const float (&v)[V]) {
  if (V == 8 && n >= V) {
    *reinterpret_cast<uint2*>(p) = make_uint2(f32x4_to_e4m3(v[0], v[1 % V], v[2 % V], v[3 % V]), f32x4_to_e4m3(v[4 % V], v[5 % V], v[6 % V], v[7 % V]));
  } else if (V == 4 && n >= V) {
    *reinterpret_cast<uint32_t*>(p) = f32x4_to_e4m3(v[0], v[1 % V], v[2 % V], v[3 % V]);
  } else {
#pragma unroll
    for (int i = 0; i < V; i++)
      if (i < n) p[i] = f32_to_e4m3(v[i]);
  }
}

// CH pieces of V numbers a thread; ROWS > 1: a warp a row, that many rows a block.  CH = 0: any width, the row read twice.
template <typename TX, int V, int CH, int ROWS>
__global__ void __launch_bounds__(512) quantize_kernel(uint8_t* __restrict__ q, float* __restrict__ scale, const TX* __restrict__ x, const int* __restrict__ rows,
                                                       const float* __restrict__ weights, int div, int P, int M, int D, long long ldx, long long ldq) {
  constexpr bool WARP = ROWS > 1;
  constexpr int C = CH > 0 ? CH : 1;
  const int tid = WARP ? threadIdx.x & 31 : threadIdx.x, T = WARP ? 32 : blockDim.x;
  const int p = WARP ? blockIdx.x * ROWS + (threadIdx.x >> 5) : blockIdx.x;
  pdl_wait();
  if (p >= P) return;
  const long long m = source_row(rows, p, div, M);
  const TX* xi = x + (m < 0 ? 0 : m) * ldx;
  const int width = m < 0 ? 0 : D;      // (a row that is not there: nothing is read)
  uint32_t top = m < 0 ? 0x7fffffffu : 0u;
  Some<TX, V> v[C];
  if (CH > 0) {
#pragma unroll
    for (int c = 0; c < C; c++) v[c].load(xi + (tid + c * T) * V, width - (tid + c * T) * V, true);
#pragma unroll
    for (int c = 0; c < C; c++) top = max(top, v[c].top());
  } else {
    for (int i = tid; i < width; i += T) top = max(top, magnitude(to_f32(xi[i])));
  }
  float inv, s;
  row_factor(row_sums<WARP>(0.f, top), inv, s);
  if (tid == 0) scale[p] = weights && m >= 0 ? s * weights[rows[p]] : s;
  uint8_t* o = q + p * ldq;
  if (CH > 0) {
#pragma unroll
    for (int c = 0; c < C; c++) {
      float z[V];
#pragma unroll
      for (int i = 0; i < V; i++) z[i] = v[c].at(i) * inv;
      store_eight<V>(o + (tid + c * T) * V, D - (tid + c * T) * V, z);
    }
  } else {
    for (int i = tid; i < D; i += T) o[i] = f32_to_e4m3(m < 0 ? inv : to_f32(xi[i]) * inv);
  }
}

template <typename TY, int V, int CH, int ROWS>
__global__ void __launch_bounds__(512) rmsnorm_e4m3_kernel(uint8_t* __restrict__ q, float* __restrict__ scale, float* __restrict__ x, const float* __restrict__ w,
                                                           const TY* __restrict__ y, void* __restrict__ h, int h_dtype, int M, int D, float eps, long long ldq) {
  constexpr bool WARP = ROWS > 1;
  constexpr int C = CH > 0 ? CH : 1;
  const int tid = WARP ? threadIdx.x & 31 : threadIdx.x, T = WARP ? 32 : blockDim.x;
  const int m = WARP ? blockIdx.x * ROWS + (threadIdx.x >> 5) : blockIdx.x;
  pdl_wait();
  if (m >= M) return;
  const size_t at = (size_t)m * D;
  float squares = 0.f;
  uint32_t top = 0u;
  Some<float, V> v[C];
  if (CH > 0) {
#pragma unroll
    for (int c = 0; c < C; c++) v[c].load(x + at + (tid + c * T) * V, D - (tid + c * T) * V);
    if (y) {
      Some<TY, V> b[C];
#pragma unroll
      for (int c = 0; c < C; c++) b[c].load(y + at + (tid + c * T) * V, D - (tid + c * T) * V);
#pragma unroll
      for (int c = 0; c < C; c++) {
#pragma unroll
        for (int i = 0; i < V; i++) v[c].v[i] += b[c].at(i);
        store_some<V>(x + at + (tid + c * T) * V, D - (tid + c * T) * V, v[c].v);
      }
    }
#pragma unroll
    for (int c = 0; c < C; c++) {
      Some<float, V> f;
      f.load(w + (tid + c * T) * V, D - (tid + c * T) * V);
#pragma unroll
      for (int i = 0; i < V; i++) {
        squares += v[c].v[i] * v[c].v[i];
        v[c].v[i] *= f.v[i];
      }
      top = max(top, v[c].top());
    }
  } else {
    for (int i = tid; i < D; i += T) {
      float a = x[at + i];
      if (y) x[at + i] = a = a + to_f32(y[at + i]);
      squares += a * a;
      top = max(top, magnitude(a * w[i]));
    }
  }
  const RowSums t = row_sums<WARP>(squares, top);
  const float r = 1.0f / sqrtf(t.squares / (float)D + eps);
  float inv, s;
  row_factor(t, inv, s);
  if (tid == 0) scale[m] = s * r;
  uint8_t* o = q + m * ldq;
  if (CH > 0) {
#pragma unroll
    for (int c = 0; c < C; c++) {
      const int i = (tid + c * T) * V;
      float z[V];
#pragma unroll
      for (int k = 0; k < V; k++) z[k] = v[c].v[k] * inv;
      store_eight<V>(o + i, D - i, z);
      if (h) {
#pragma unroll
        for (int k = 0; k < V; k++) z[k] = v[c].v[k] * r;
        if (h_dtype == LEB_F32) store_some<V>((float*)h + at + i, D - i, z);
        else store_some<V>((bf16*)h + at + i, D - i, z);
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

// How rows of D numbers are shared out: GO(V, CH, ROWS, blocks, threads).  Few rows: many threads a row, whose loads are one trip to memory.
// Many rows: few threads a row with many loads each, so that threads seldom wait for one another (8,191 bfloat16 rows of 8,192:
// 512 threads with two pieces 54 us, 128 with eight 32).
#define MANY_ROWS 1024
#define FEW_ROW_SHAPES(wide, fours, D, rows)                                               \
  if (wide && D <= 1024) GO(8, 1, 1, rows, 128);                                           \
  else if (wide && D <= 2048) GO(8, 1, 1, rows, 256);                                      \
  else if (wide && D <= 4096) GO(8, 1, 1, rows, 512);                                      \
  else if (wide && D <= 8192) GO(8, 2, 1, rows, 512);                                      \
  else if (wide && D <= 16384) GO(8, 4, 1, rows, 512);                                     \
  else if (fours && D <= 512) GO(4, 1, 1, rows, 128);                                      \
  else if (fours && D <= 1024) GO(4, 1, 1, rows, 256);                                     \
  else if (fours && D <= 2048) GO(4, 1, 1, rows, 512);                                     \
  else if (fours && D <= 4096) GO(4, 2, 1, rows, 512);                                     \
  else if (fours && D <= 8192) GO(4, 4, 1, rows, 512);                                     \
  else if (fours && D <= 16384) GO(4, 8, 1, rows, 512);                                    \
  else if (D <= 4096) GO(1, 8, 1, rows, 512);                                              \
  else GO(1, 0, 1, rows, 512);
#define QUANTIZE_SHAPES(wide, fours, D, rows)                                              \
  if (wide && D <= 256) GO(8, 1, 8, ceil_div(rows, 8), 256);                               \
  else if (wide && D <= 512) GO(8, 2, 8, ceil_div(rows, 8), 256);                          \
  else if (rows < MANY_ROWS) { FEW_ROW_SHAPES(wide, fours, D, rows) }                      \
  else if (wide && D <= 1024) GO(8, 4, 8, ceil_div(rows, 8), 256);                         \
  else if (wide && D <= 2048) GO(8, 8, 8, ceil_div(rows, 8), 256);                         \
  else if (wide && D <= 4096) GO(8, 8, 1, rows, 64);                                       \
  else if (wide && D <= 8192) GO(8, 8, 1, rows, 128);                                      \
  else if (wide && D <= 16384) GO(8, 8, 1, rows, 256);                                     \
  else if (!wide && fours && D <= 512) GO(4, 4, 8, ceil_div(rows, 8), 256);                \
  else if (!wide && fours && D <= 1024) GO(4, 8, 8, ceil_div(rows, 8), 256);               \
  else if (!wide && fours && D <= 2048) GO(4, 8, 1, rows, 64);                             \
  else if (!wide && fours && D <= 4096) GO(4, 8, 1, rows, 128);                            \
  else if (!wide && fours && D <= 8192) GO(4, 8, 1, rows, 256);                            \
  else { FEW_ROW_SHAPES(wide, fours, D, rows) }
// The norm holds its weights beside the row, and what is added: two pieces a thread (2,048 rows of 2,048 with a bfloat16 addition: four pieces
// 13.3 us, two 10.7; 16,000 rows 59.3 and 56.1, without the addition 31.3 and 29.5; 2,048 rows of 1,001 with it: a warp a row 12.2, four 7.5).
// Short rows without an addition have little to load: a warp takes one (16,000 rows of 1,024: 15.6 us, two warps 18.9; with the addition
// 31.8 and 30.0).  Chosen with the addition; without it two sizes lose to twice as many pieces a thread: 16,000 x 1,001 22.5 us (20.0),
// 8,191 x 4,096 33.7 (32.4).  Wider rows off 16 bytes have no other shape to compare with: 8,191 x 6,001 87 us, 4,096 x 12,001 109 (38 either by their bytes).
#define NORM_SHAPES(wide, fours, adds, D, rows)                                            \
  if (wide && D <= 256) GO(8, 1, 8, ceil_div(rows, 8), 256);                               \
  else if (wide && D <= 512) GO(8, 2, 8, ceil_div(rows, 8), 256);                          \
  else if (rows < MANY_ROWS) { FEW_ROW_SHAPES(wide, fours, D, rows) }                      \
  else if (wide && D <= 1024 && !adds) GO(8, 4, 8, ceil_div(rows, 8), 256);                \
  else if (wide && D <= 1024) GO(8, 2, 1, rows, 64);                                       \
  else if (wide && D <= 2048) GO(8, 2, 1, rows, 128);                                      \
  else if (wide && D <= 4096) GO(8, 2, 1, rows, 256);                                      \
  else if (!wide && fours && D <= 512 && !adds) GO(4, 4, 8, ceil_div(rows, 8), 256);       \
  else if (!wide && fours && D <= 512) GO(4, 1, 1, rows, 128);                             \
  else if (!wide && fours && D <= 1024 && !adds) GO(4, 4, 1, rows, 64);                    \
  else if (!wide && fours && D <= 1024) GO(4, 2, 1, rows, 128);                            \
  else if (!wide && fours && D <= 2048 && !adds) GO(4, 4, 1, rows, 128);                   \
  else if (!wide && fours && D <= 2048) GO(4, 2, 1, rows, 256);                            \
  else if (!wide && fours && D <= 4096) GO(4, 4, 1, rows, 256);                            \
  else if (!wide && fours && D <= 8192) GO(4, 8, 1, rows, 256);                            \
  else { FEW_ROW_SHAPES(wide, fours, D, rows) }

template <typename TX>
void launch_quantize(bool wide, bool fours, uint8_t* q, float* scale, const TX* x, const int* rows, const float* weights, int div, int P, int M, int D,
                     long long ldx, long long ldq, cudaStream_t st) {
#define GO(V, CH, ROWS, blocks, threads) \
  leb_launch(quantize_kernel<TX, V, CH, ROWS>, dim3(blocks), dim3(threads), 0, st, q, scale, x, rows, weights, div, P, M, D, ldx, ldq)
  QUANTIZE_SHAPES(wide, fours, D, P)
#undef GO
}
template <typename TY>
void launch_norm(bool wide, bool fours, uint8_t* q, float* scale, float* x, const float* w, const TY* y, void* h, int h_dtype, int M, int D, float eps, long long ldq, cudaStream_t st) {
#define GO(V, CH, ROWS, blocks, threads) \
  leb_launch(rmsnorm_e4m3_kernel<TY, V, CH, ROWS>, dim3(blocks), dim3(threads), 0, st, q, scale, x, w, y, h, h_dtype, M, D, eps, ldq)
  const bool adds = y != nullptr;
  NORM_SHAPES(wide, fours, adds, D, M)
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
  const bool wide = (a.x & 15) == 0 && a.ldx % (a.x_dtype == LEB_F32 ? 4 : 8) == 0 && (a.q & 7) == 0 && a.ldq % 8 == 0, fours = (a.q & 3) == 0 && a.ldq % 4 == 0;
  if (a.x_dtype == LEB_F32)
    launch_quantize(wide, fours, (uint8_t*)a.q, (float*)a.scale, (const float*)a.x, (const int*)a.rows, (const float*)a.weights, (int)a.div, (int)a.P, (int)a.M, (int)a.D, a.ldx, a.ldq, st);
  else
    launch_quantize(wide, fours, (uint8_t*)a.q, (float*)a.scale, (const bf16*)a.x, (const int*)a.rows, (const float*)a.weights, (int)a.div, (int)a.P, (int)a.M, (int)a.D, a.ldx, a.ldq, st);
  LEB_CHECK_LAUNCH("leb_quantize_e4m3");
  return 0;
}

// q [M, D] 8-bit (rows ldq apart), scale [M], x [M, D] float (x += y first where y is given), h [M, D] or null: the normed rows.
LEB_API int leb_rmsnorm_e4m3(const void* packed, cudaStream_t st) {
  const NormArgs& a = *(const NormArgs*)packed;
  if (a.M <= 0) return 0;
  LEB_REQUIRE(a.D > 0 && a.D < MOST && a.M < MOST, "leb_rmsnorm_e4m3: %lld rows of %lld numbers", a.M, a.D);
  LEB_REQUIRE((a.y_dtype == LEB_F32 || a.y_dtype == LEB_BF16) && (a.h_dtype == LEB_F32 || a.h_dtype == LEB_BF16), "leb_rmsnorm_e4m3: unknown type of y (%lld) or h (%lld)", a.y_dtype, a.h_dtype);
  const bool wide = a.D % 8 == 0 && ((a.x | a.w | a.y | a.h) & 15) == 0 && (a.q & 7) == 0 && a.ldq % 8 == 0, fours = (a.q & 3) == 0 && a.ldq % 4 == 0;
  if (a.y_dtype == LEB_F32)
    launch_norm(wide, fours, (uint8_t*)a.q, (float*)a.scale, (float*)a.x, (const float*)a.w, (const float*)a.y, (void*)a.h, (int)a.h_dtype, (int)a.M, (int)a.D, (float)a.eps, a.ldq, st);
  else
    launch_norm(wide, fours, (uint8_t*)a.q, (float*)a.scale, (float*)a.x, (const float*)a.w, (const bf16*)a.y, (void*)a.h, (int)a.h_dtype, (int)a.M, (int)a.D, (float)a.eps, a.ldq, st);
  LEB_CHECK_LAUNCH("leb_rmsnorm_e4m3");
  return 0;
}
