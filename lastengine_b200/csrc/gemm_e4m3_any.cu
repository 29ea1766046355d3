// 8-bit matrix product for operands of any sizes and strides: C[m, n] (+)= (sum_k A[m, k] W[n, k]) sa[m] sw[n].
// 64 x 64 results per block, four by four a thread, k in chunks of 32 through shared memory as floats, summed in order: a row's
// result does not depend on the other rows.  It is the way for rows that are not 16 bytes apart to run at all; the tensor-core
// kernels take the others.  Bound by the FMA pipes and their loads from shared memory: 2,048 rows x 4,096 x 2,048 1,064 us (32 TFLOP/s; the
// tensor cores 15.7), 1 row x 16,384 x 2,048 222 (7.1), of whose 64 rows of results a block has one.
#include "e4m3_tc.cuh"

namespace {

template <typename TC>
__global__ void __launch_bounds__(256) gemm_e4m3_any_kernel(TC* __restrict__ C, const uint8_t* __restrict__ A, const float* __restrict__ sa,
                                                            const uint8_t* __restrict__ W, const float* __restrict__ sw, int M, int N, int K,
                                                            long long lda, long long ldw, long long ldc, int epilogue, const int* __restrict__ offsets,
                                                            int m_tiles, long long w_group_stride) {
  __shared__ float as[64][33], ws[64][33];
  const int act = epilogue >> 8;
  epilogue &= 255;
  pdl_wait();
  int lo = 0, hi = M;
  if (offsets) {      // rows [offsets[e], offsets[e + 1]) go with expert e's weights, from where the experts before have ended on (whatever the offsets hold)
    const int e = blockIdx.x / m_tiles;
    __shared__ int ends[8];
    int last = 0;
    for (int i = threadIdx.x + 1; i <= e; i += 256) last = max(last, min(offsets[i], M));
    last = __reduce_max_sync(0xffffffffu, last);
    if ((threadIdx.x & 31) == 0) ends[threadIdx.x >> 5] = last;
    __syncthreads();
    for (int i = 0; i < 8; i++) last = max(last, ends[i]);
    lo = max(min(offsets[e], M), last);
    hi = min(offsets[e + 1], M);
    W += e * w_group_stride;
    sw += (size_t)e * N;
  }
  const long long at = lo + (long long)(blockIdx.x % m_tiles) * 64;      // (an expert has blocks for all rows: beyond 2^31 where there are many)
  if (at >= hi) return;
  const int m0 = (int)at, n0 = blockIdx.y * 64;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, kk = threadIdx.x & 31, row8 = threadIdx.x >> 5;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < K; k0 += 32) {
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int r = row8 + 8 * j, m = m0 + r, n = n0 + r, k = k0 + kk;
      as[r][kk] = m < hi && k < K ? e4m3_to_f32(A[m * lda + k]) : 0.f;
      ws[r][kk] = n < N && k < K ? e4m3_to_f32(W[n * ldw + k]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 32; k++)
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] += as[ty * 4 + i][k] * ws[tx + 16 * j][k];
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int m = m0 + ty * 4 + i;
    if (m >= hi) continue;
    float z[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int n = n0 + tx + 16 * j;
      z[j] = n < N ? acc[i][j] * sa[m] * sw[n] : 0.f;
    }
    TC* c = C + m * ldc;
    if (epilogue == 2) {
#pragma unroll
      for (int j = 0; j < 4; j += 2)
        if (n0 + 16 * j < N) c[n0 / 2 + 8 * j + tx] = from_f32<TC>(gate_mul<float>(z[j], z[j + 1], act));
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int n = n0 + tx + 16 * j;
        if (n >= N) continue;
        float v = z[j];
        if (epilogue == 1) v += to_f32(c[n]);
        else if (LEB_PLAIN_ACT_OK(act, epilogue)) v = plain_act(v, act);
        c[n] = from_f32<TC>(v);
      }
    }
  }
}

}  // namespace

int leb_gemm_e4m3_any(const E8Product& p, cudaStream_t st) {
  const int m_tiles = ceil_div(p.M, 64);
  const long long xs = (long long)m_tiles * (p.offsets ? p.n_groups : 1);
  LEB_REQUIRE(xs < (1LL << 31) && ceil_div(p.N, 64) <= 65535, "leb_linear_e4m3: %d rows in %d groups and %d columns in one launch", p.M, p.n_groups, p.N);
  const dim3 grid((unsigned)xs, ceil_div(p.N, 64));
  if (p.c_dtype == LEB_F32)
    leb_launch(gemm_e4m3_any_kernel<float>, grid, dim3(256), 0, st, (float*)p.C, (const uint8_t*)p.A, p.sa, (const uint8_t*)p.W, p.sw, p.M, p.N, p.K, p.lda, p.ldw, p.ldc, p.epilogue, p.offsets, m_tiles, p.w_group_stride);
  else
    leb_launch(gemm_e4m3_any_kernel<bf16>, grid, dim3(256), 0, st, (bf16*)p.C, (const uint8_t*)p.A, p.sa, (const uint8_t*)p.W, p.sw, p.M, p.N, p.K, p.lda, p.ldw, p.ldc, p.epilogue, p.offsets, m_tiles, p.w_group_stride);
  LEB_CHECK_LAUNCH("leb_linear_e4m3");
  return 0;
}
