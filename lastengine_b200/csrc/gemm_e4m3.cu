// The entry point of the products of 8-bit rows, and which kernel a product goes to.
#include "e4m3_tc.cuh"

namespace {

// Which kernel takes a product of `groups` times about `rows` rows.
//
// The weights-first kernel takes them in tiles of 128 columns by the fewest rows (16 to 128) with which there are at most four tiles of
// rows and at most two tiles an SM (else as many rows as there are, up to 128), and cuts K over up to eight blocks while that
// leaves no SM with more than two, or with more than 4/3 eighths.  The pairs of SMs take 256 x 256.  Which is ahead goes by what either takes:
//   weights first  2.7 + c (b (0.2 + 0.0014 rows) + 0.055 rows') us (+ 1.5 for a cluster): c the blocks an SM goes through, b its stages
//                  of 128 numbers of k, rows' those a block finishes
//   pairs          2.8 + w (0.31 b + 3) us: w the tiles a pair goes through
// Fitted to 90 products of 40 to 3,000 rows, 64 to 24,000 columns and K of 128 to 12,000; over these, 117 more and 103 grouped ones (2 to
// 128 experts, 0.1 to 512 rows each) the choice takes 1.5% more time than the best form of each.  Where it turns: 96 rows x
// 2,048 x 2,048 weights first 6.1 us, pairs 10.4; 512 rows x 16,384 x 2,048 36.8 and 17.4.
struct Form {
  bool pairs;
  int rows, slices;      // of the weights-first kernel
};

Form form_of(int groups, int rows, int N, int K) {
  const int sms = sm_count(), nk = ceil_div(K, E8_BK), n_tiles = ceil_div(N, 128);
  Form f{false, 16, 1};
  for (; f.rows <= 128; f.rows *= 2)
    if (ceil_div(rows, f.rows) <= 4 && (long long)groups * ceil_div(rows, f.rows) * n_tiles <= 2 * sms) break;
  if (f.rows > 128)
    for (f.rows = 16; f.rows < 128 && f.rows < rows; f.rows *= 2) {}
  const long long tiles = (long long)groups * ceil_div(rows, f.rows) * n_tiles;
  while (f.slices < 8 && tiles * f.slices * 2 <= (f.slices < 4 ? 2 * sms : sms * 4 / 3) && nk >= 4 * f.slices) f.slices *= 2;
  if (rows < 48) return f;
  const double each = (double)tiles * f.slices / sms, finished = rows < f.rows ? rows : f.rows;
  const double few = 2.7 + (each > 1 ? each : 1) * (ceil_div(nk, f.slices) * (0.2 + 0.0014 * f.rows) + 0.055 * finished * (f.slices == 1 ? 1 : 1.0 / f.slices + 0.2)) + (f.slices > 1 ? 1.5 : 0);
  const long long turns = ((long long)groups * ceil_div(rows, 256) * ceil_div(N, 256) + sms / 2 - 1) / (sms / 2);
  f.pairs = 2.8 + turns * (0.31 * nk + 3) < few;
  return f;
}

// One packed argument, numbers of 64 bits in this order (see row_e4m3.cu).
struct LinearArgs {
  long long C, c_dtype, A, sa, W, sw, M, N, K, lda, ldw, ldc, epilogue, offsets, n_groups, w_group_stride, status;
};

}  // namespace

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
  const int groups = p.offsets ? min(p.n_groups, M) : 1;
  const Form f = form_of(groups, ceil_div(M, groups), N, K);
  return f.pairs ? leb_gemm_e4m3_pairs(p, st) : leb_gemm_e4m3_few(p, f.rows, f.slices, st);
}
