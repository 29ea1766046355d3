// The entry point of the products of 8-bit rows, and which kernel a product goes to.
#include "e4m3_tc.cuh"

// One packed argument, numbers of 64 bits in this order (see row_e4m3.cu).
struct LinearArgs {
  long long C, c_dtype, A, sa, W, sw, M, N, K, lda, ldw, ldc, epilogue, offsets, n_groups, w_group_stride, status;
};

// C [M, N] (or [M, N / 2] gated; rows ldc apart) (+)= the product of A [M, K] with scales sa [M] and W [N, K] with scales sw [N]; with offsets
// [n_groups + 1] (on the device) rows [offsets[e], offsets[e + 1]) with W[e], sw[e], experts w_group_stride apart, and rows beyond the last
// offset left as they are.  epilogue: 0 store, 1 add into float C, 2 gated, an activation above it as in the bfloat16 products.
// status: device int, set non-zero by a block whose bounded wait gave up.
LEB_API int leb_linear_e4m3(const void* packed, cudaStream_t st) {
  const LinearArgs& a = *(const LinearArgs*)packed;
  if (a.M <= 0 || a.N <= 0) return 0;
  constexpr long long MOST = (1LL << 31) - 65536;
  LEB_REQUIRE(a.K > 0 && a.M < MOST && a.N < MOST && a.K < MOST && a.status && (!a.offsets || (a.n_groups > 0 && a.n_groups < MOST)),
              "leb_linear_e4m3: %lld rows, %lld columns, an inner size of %lld, %lld groups", a.M, a.N, a.K, a.n_groups);
  if (const char* fault = e4m3_epilogue_fault((int)(a.epilogue >> 8), (int)(a.epilogue & 255), (int)a.c_dtype, (int)a.N))
    return leb_fail("leb_linear_e4m3: %s (epilogue %lld, N %lld)", fault, a.epilogue, a.N);
  const E8Product p{(void*)a.C, (int)a.c_dtype, (const void*)a.A, (const float*)a.sa, (const void*)a.W, (const float*)a.sw, (int)a.M, (int)a.N, (int)a.K, a.lda, a.ldw, a.ldc,
                    (int)a.epilogue, (const int*)a.offsets, (int)a.n_groups, a.w_group_stride, (int*)a.status};
  const int M = p.M, N = p.N, K = p.K;
  // TMA fetches rows that begin on 16 bytes and lie a multiple of that apart (and not on one another); experts are read as one stack
  const bool tma = p.lda % 16 == 0 && p.lda >= K && p.ldw % 16 == 0 && p.ldw >= K && ((a.A | a.W) & 15) == 0 &&
                   (!p.offsets || ((p.n_groups == 1 || p.w_group_stride == N * p.ldw) && p.n_groups <= E8_MAX_GROUPS && a.N * a.n_groups < MOST));
  if (!tma) return leb_gemm_e4m3_any(p, st);
  const int groups = p.offsets ? min(p.n_groups, M) : 1, rows = ceil_div(M, groups);      // of a group, about
  if (rows >= 512) return leb_gemm_e4m3_pairs(p, st);
  const int mp = rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : 128;
  const long long tiles = (long long)ceil_div(N, 128) * (p.offsets ? max(groups, M / mp) : ceil_div(M, mp));
  const int nk = ceil_div(K, E8_BK);
  int n_slices = 1;
  while (n_slices < 8 && tiles * n_slices <= sm_count() && nk >= n_slices * 2 * 2) n_slices *= 2;
  return leb_gemm_e4m3_few(p, mp, n_slices, st);
}
