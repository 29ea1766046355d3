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
// (a warp a row up to 512 numbers, a block above), single numbers otherwise; rows of more than 16,384 (8,192) are read twice.  The largest
// |g| is taken over the bits (for numbers without a sign they order as the numbers do, infinity and NaN on top).
#include "e4m3_common.cuh"

namespace {

struct RowSums {
  float squares;
  uint32_t top;      // bits of the largest |g|
};

// Over the threads of a row: a warp, or the block (up to 512 threads); every thread gets the result, added up in the same order.
// turn: 0 and 1 in turn from row to row (a thread may be a row ahead of the others, never two).
template <bool WARP>
__device__ __forceinline__ RowSums row_sums(float squares, uint32_t top, int turn) {
  squares = warp_sum(squares);
  top = __reduce_max_sync(0xffffffffu, top);
  RowSums r{squares, top};
  if (!WARP) {
    __shared__ float red_s[2][16];
    __shared__ uint32_t red_t[2][16];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = (blockDim.x + 31) >> 5;
    if (lane == 0) red_s[turn][warp] = squares, red_t[turn][warp] = top;
    __syncthreads();
    r = RowSums{0.f, 0u};
    for (int w = 0; w < nw; w++) r.squares += red_s[turn][w], r.top = max(r.top, red_t[turn][w]);
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
  __device__ __forceinline__ void load(const T* p, int n) {
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
template <>
struct Some<float, 8> {
  float v[8];
  __device__ __forceinline__ void load(const float* p, int n) {
    if (n >= 8) {
      const float4 a = load4(p), b = load4(p + 4);
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
  __device__ __forceinline__ void load(const bf16* p, int n) {
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
  } else {
#pragma unroll
    for (int i = 0; i < V; i++)
      if (i < n) p[i] = f32_to_e4m3(v[i]);
  }
}

// CH pieces of V numbers a thread; ROWS > 1: a warp a row, that many rows at a time.  CH = 0: any width, the row read twice.
// The blocks walk the rows; a row's loads go out before the row before it is rounded, so that memory is read while threads meet.
template <typename TX, int V, int CH, int ROWS>
__global__ void __launch_bounds__(512) quantize_kernel(uint8_t* __restrict__ q, float* __restrict__ scale, const TX* __restrict__ x, const int* __restrict__ rows,
                                const float* __restrict__ weights, int div, int P, int M, int D, long long ldx, long long ldq) {
  constexpr bool WARP = ROWS > 1;
  const int tid = WARP ? threadIdx.x & 31 : threadIdx.x, T = WARP ? 32 : blockDim.x;
  const int step = gridDim.x * ROWS;
  int p = WARP ? blockIdx.x * ROWS + (threadIdx.x >> 5) : blockIdx.x;
  pdl_wait();
  if (CH == 0) {
    for (int turn = 0; p < P; p += step, turn ^= 1) {
      const long long m = source_row(rows, p, div, M);
      const TX* xi = x + (m < 0 ? 0 : m) * ldx;
      uint32_t top = m < 0 ? 0x7fffffffu : 0u;
      for (int i = tid; i < (m < 0 ? 0 : D); i += T) top = max(top, magnitude(to_f32(xi[i])));
      float inv, s;
      row_factor(row_sums<WARP>(0.f, top, turn), inv, s);
      if (tid == 0) scale[p] = weights && m >= 0 ? s * weights[rows[p]] : s;
      uint8_t* o = q + p * ldq;
      for (int i = tid; i < D; i += T) o[i] = f32_to_e4m3(m < 0 ? inv : to_f32(xi[i]) * inv);
    }
    return;
  }
  constexpr int C = CH > 0 ? CH : 1;
  Some<TX, V> next[C];
  long long m_next = -1;
  auto fetch = [&](int row) {
    m_next = source_row(rows, row, div, M);
    const TX* xi = x + (m_next < 0 ? 0 : m_next) * ldx;
    const int width = m_next < 0 ? 0 : D;      // (a row that is not there: nothing is read)
#pragma unroll
    for (int c = 0; c < C; c++) next[c].load(xi + (tid + c * T) * V, width - (tid + c * T) * V);
  };
  if (p < P) fetch(p);
  for (int turn = 0; p < P; p += step, turn ^= 1) {
    Some<TX, V> now[C];
    const long long m = m_next;
#pragma unroll
    for (int c = 0; c < C; c++) now[c] = next[c];
    if (p + step < P) fetch(p + step);
    uint32_t top = m < 0 ? 0x7fffffffu : 0u;
#pragma unroll
    for (int c = 0; c < C; c++) top = max(top, now[c].top());
    float inv, s;
    row_factor(row_sums<WARP>(0.f, top, turn), inv, s);
    if (tid == 0) scale[p] = weights && m >= 0 ? s * weights[rows[p]] : s;
    uint8_t* o = q + p * ldq;
#pragma unroll
    for (int c = 0; c < C; c++) {
      float v[V];
#pragma unroll
      for (int i = 0; i < V; i++) v[i] = now[c].at(i) * inv;
      store_eight<V>(o + (tid + c * T) * V, D - (tid + c * T) * V, v);
    }
  }
}

template <typename TY, int V, int CH, int ROWS>
__global__ void __launch_bounds__(512) rmsnorm_e4m3_kernel(uint8_t* __restrict__ q, float* __restrict__ scale, float* __restrict__ x, const float* __restrict__ w,
                                    const TY* __restrict__ y, void* __restrict__ h, int h_dtype, int M, int D, float eps, long long ldq) {
  constexpr bool WARP = ROWS > 1;
  const int tid = WARP ? threadIdx.x & 31 : threadIdx.x, T = WARP ? 32 : blockDim.x;
  const int step = gridDim.x * ROWS;
  int m = WARP ? blockIdx.x * ROWS + (threadIdx.x >> 5) : blockIdx.x;
  pdl_wait();
  auto finish = [&](RowSums t, float& inv, float& r) {
    float s;
    r = 1.0f / sqrtf(t.squares / (float)D + eps);
    row_factor(t, inv, s);
    if (tid == 0) scale[m] = s * r;
  };
  if (CH == 0) {
    for (int turn = 0; m < M; m += step, turn ^= 1) {
      const size_t at = (size_t)m * D;
      float squares = 0.f, inv, r;
      uint32_t top = 0u;
      for (int i = tid; i < D; i += T) {
        float a = x[at + i];
        if (y) x[at + i] = a = a + to_f32(y[at + i]);
        squares += a * a;
        top = max(top, magnitude(a * w[i]));
      }
      finish(row_sums<WARP>(squares, top, turn), inv, r);
      uint8_t* o = q + m * ldq;
      for (int i = tid; i < D; i += T) {
        const float a = x[at + i] * w[i];
        o[i] = f32_to_e4m3(a * inv);
        if (h && h_dtype == LEB_F32) ((float*)h)[at + i] = a * r;
        else if (h) ((bf16*)h)[at + i] = from_f32<bf16>(a * r);
      }
    }
    return;
  }
  constexpr int C = CH > 0 ? CH : 1;
  Some<float, V> next[C];
  Some<TY, V> next_y[C];
  auto fetch = [&](int row) {
    const size_t at = (size_t)row * D;
#pragma unroll
    for (int c = 0; c < C; c++) next[c].load(x + at + (tid + c * T) * V, D - (tid + c * T) * V);
    if (y)
#pragma unroll
      for (int c = 0; c < C; c++) next_y[c].load(y + at + (tid + c * T) * V, D - (tid + c * T) * V);
  };
  if (m < M) fetch(m);
  for (int turn = 0; m < M; m += step, turn ^= 1) {
    const size_t at = (size_t)m * D;
    float v[C][V];
#pragma unroll
    for (int c = 0; c < C; c++) {
#pragma unroll
      for (int i = 0; i < V; i++) v[c][i] = y ? next[c].at(i) + next_y[c].at(i) : next[c].at(i);
      if (y) store_some<V>(x + at + (tid + c * T) * V, D - (tid + c * T) * V, v[c]);
    }
    if (m + step < M) fetch(m + step);
    float squares = 0.f, inv, r;
    uint32_t top = 0u;
#pragma unroll
    for (int c = 0; c < C; c++) {
      Some<float, V> f;
      f.load(w + (tid + c * T) * V, D - (tid + c * T) * V);
#pragma unroll
      for (int i = 0; i < V; i++) {
        squares += v[c][i] * v[c][i];
        v[c][i] *= f.at(i);
        top = max(top, magnitude(v[c][i]));
      }
    }
    finish(row_sums<WARP>(squares, top, turn), inv, r);
    uint8_t* o = q + m * ldq;
#pragma unroll
    for (int c = 0; c < C; c++) {
      const int i = (tid + c * T) * V;
      float z[V];
#pragma unroll
      for (int k = 0; k < V; k++) z[k] = v[c][k] * inv;
      store_eight<V>(o + i, D - i, z);
      if (h) {
#pragma unroll
        for (int k = 0; k < V; k++) z[k] = v[c][k] * r;
        if (h_dtype == LEB_F32) store_some<V>((float*)h + at + i, D - i, z);
        else store_some<V>((bf16*)h + at + i, D - i, z);
      }
    }
  }
}

// How a row of D numbers is shared out: GO(V, CH, ROWS, threads).
#define ROW_SHAPES(wide, D)                \
  if (wide) {                              \
    if (D <= 256) GO(8, 1, 8, 256);        \
    else if (D <= 512) GO(8, 2, 8, 256);   \
    else if (D <= 1024) GO(8, 1, 1, 128);  \
    else if (D <= 2048) GO(8, 1, 1, 256);  \
    else if (D <= 4096) GO(8, 2, 1, 256);  \
    else if (D <= 8192) GO(8, 2, 1, 512);  \
    else if (D <= 16384) GO(8, 4, 1, 512); \
    else GO(1, 0, 1, 512);                 \
  } else {                                 \
    if (D <= 128) GO(1, 4, 8, 256);        \
    else if (D <= 1024) GO(1, 8, 1, 128);  \
    else if (D <= 2048) GO(1, 8, 1, 256);  \
    else if (D <= 4096) GO(1, 8, 1, 512);  \
    else if (D <= 8192) GO(1, 16, 1, 512); \
    else GO(1, 0, 1, 512);                 \
  }

// As many blocks as fit the SMs at once, or as there are rows for.
template <typename... KArgs, typename... Args>
int launch_rows(void (*kern)(KArgs...), int& resident, int at_a_time, int threads, int rows, cudaStream_t st, Args... args) {
  if (resident == 0) {      // (the same for every caller, whoever is first)
    int n = 0;
    resident = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, threads, 0) == cudaSuccess && n > 0 ? n : 1;
  }
  const int blocks = ceil_div(rows, at_a_time), most = resident * sm_count();
  return leb_launch(kern, dim3(blocks < most ? blocks : most), dim3(threads), 0, st, args...) == cudaSuccess ? 0 : 1;
}

template <typename TX>
void launch_quantize(bool wide, uint8_t* q, float* scale, const TX* x, const int* rows, const float* weights, int div, int P, int M, int D, long long ldx,
                     long long ldq, cudaStream_t st) {
#define GO(V, CH, ROWS, threads)                                                                                                                     \
  do {                                                                                                                                               \
    static int resident = 0;                                                                                                                         \
    launch_rows(quantize_kernel<TX, V, CH, ROWS>, resident, ROWS, threads, P, st, q, scale, x, rows, weights, div, P, M, D, ldx, ldq);              \
  } while (0)
  ROW_SHAPES(wide, D)
#undef GO
}
template <typename TY>
void launch_norm(bool wide, uint8_t* q, float* scale, float* x, const float* w, const TY* y, void* h, int h_dtype, int M, int D, float eps, long long ldq, cudaStream_t st) {
#define GO(V, CH, ROWS, threads)                                                                                                                     \
  do {                                                                                                                                               \
    static int resident = 0;                                                                                                                         \
    launch_rows(rmsnorm_e4m3_kernel<TY, V, CH, ROWS>, resident, ROWS, threads, M, st, q, scale, x, w, y, h, h_dtype, M, D, eps, ldq);               \
  } while (0)
  ROW_SHAPES(wide, D)
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
  if (a.y_dtype == LEB_F32)
    launch_norm(wide, (uint8_t*)a.q, (float*)a.scale, (float*)a.x, (const float*)a.w, (const float*)a.y, (void*)a.h, (int)a.h_dtype, (int)a.M, (int)a.D, (float)a.eps, a.ldq, st);
  else
    launch_norm(wide, (uint8_t*)a.q, (float*)a.scale, (float*)a.x, (const float*)a.w, (const bf16*)a.y, (void*)a.h, (int)a.h_dtype, (int)a.M, (int)a.D, (float)a.eps, a.ldq, st);
  LEB_CHECK_LAUNCH("leb_rmsnorm_e4m3");
  return 0;
}
