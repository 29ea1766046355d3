// The entry point of the products of 8-bit rows, and which kernel a product goes to.
#include "e4m3_tc.cuh"

// C [M, N] (or [M, N / 2] gated; rows ldc apart) (+)= the product of A [M, K] with scales sa [M] and W [N, K] with scales sw [N]; with offsets
// [n_groups + 1] (on the device) rows [offsets[e], offsets[e + 1]) with W[e], sw[e], experts w_group_stride apart, and rows beyond the last
// offset left as they are.  epilogue: 0 store, 1 add into float C, 2 gated, an activation above it as in the bfloat16 products.
// status: device int, set non-zero by a block whose bounded wait gave up.
LEB_API int leb_linear_e4m3(void* C, int c_dtype, const void* A, const float* sa, const void* W, const float* sw, int M, int N, int K, long long lda,
                            long long ldw, long long ldc, int epilogue, const int* offsets, int n_groups, long long w_group_stride, int* status,
                            cudaStream_t st) {
  if (M <= 0 || N <= 0) return 0;
  if (const char* fault = e4m3_epilogue_fault(epilogue >> 8, epilogue & 255, c_dtype, N)) return leb_fail("leb_linear_e4m3: %s (epilogue %d, N %d)", fault, epilogue, N);
  LEB_REQUIRE(K > 0 && status != nullptr && (!offsets || n_groups > 0), "leb_linear_e4m3: an inner size of %d, %d groups", K, n_groups);
  const E8Product p{C, c_dtype, A, sa, W, sw, M, N, K, lda, ldw, ldc, epilogue, offsets, n_groups, w_group_stride, status};
  // TMA fetches rows that begin on 16 bytes and lie a multiple of that apart (and not on one another); experts are read as one stack
  const long long rows_w = (long long)N * (offsets ? n_groups : 1);
  const bool tma = lda % 16 == 0 && lda >= K && ldw % 16 == 0 && ldw >= K && ((uintptr_t)A & 15) == 0 && ((uintptr_t)W & 15) == 0 &&
                   (!offsets || n_groups == 1 || w_group_stride == N * ldw) && n_groups <= E8_MAX_GROUPS && rows_w < (1LL << 31) - 256 && M < (1LL << 31) - 256;
  if (!tma) return leb_gemm_e4m3_any(p, st);
  const int groups = offsets ? min(n_groups, M) : 1, rows = ceil_div(M, groups);      // of a group, about
  if (rows >= 512) return leb_gemm_e4m3_pairs(p, st);
  const int mp = rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : 128;
  const long long tiles = (long long)ceil_div(N, 128) * (offsets ? max(groups, M / mp) : ceil_div(M, mp));
  const int nk = ceil_div(K, E8_BK);
  int n_slices = 1;
  while (n_slices < 8 && tiles * n_slices <= sm_count() && nk >= n_slices * 2 * 2) n_slices *= 2;
  return leb_gemm_e4m3_few(p, mp, n_slices, st);
}
