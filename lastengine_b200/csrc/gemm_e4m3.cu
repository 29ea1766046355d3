// The entry point of the products of 8-bit rows, and which kernel a product goes to.
#include "e4m3_tc.cuh"

namespace {

// Which kernel takes a product of `groups` times about `rows` rows: the one that is through first, by what either takes (us).
//
// weights first (tiles of 128 columns by 16 to 128 rows; s blocks share a tile's K, all of them on the SMs at once, clusters of eight only
// where no part of the chip has to take more of them than fit), c blocks an SM, b stages of 128 numbers of k a block, `held` of them on
// their way at a time:
//   2.4 + b max((0.8 + 1.4 min(c, 2)) / held, 0.18 + 0.0004 rows, c (0.25 + 0.0005 rows) where c > 1)
//       + max(c, 1) rows' (0.016 / s + 0.024 in a cluster) + 0.38 for a cluster      (rows' those of a tile that there are)
// pairs of SMs (tiles of 256 x 256), w of them a pair:
//   2.9 + w (0.34 b + 2.6)
// Fitted to 203 products of 1 to 2,500 rows, 64 to 24,000 columns and K of 128 to 12,000, each in every form that it has; over these and 58
// grouped ones (2 to 128 experts of 0.5 to 400 rows) the choice takes 2.5% more time than the best form of each.  Where it turns: 61 rows
// x 2,048 x 2,048 weights first 5.8 us, pairs 10.3; 512 rows x 16,384 x 2,048 23 and 16.2.
struct Form {
  bool pairs;
  int rows, slices;      // of the weights-first kernel
};

Form form_of(int groups, int rows, int N, int K, int sms) {
  const int nk = ceil_div(K, E8_BK);
  Form best{false, 16, 1};
  double least = 1e30;
  for (int mp = 16; mp <= 128; mp *= 2) {
    if ((mp > 16 && mp >= 2 * rows) || (mp == 16 && rows > 128) || (mp == 32 && rows > 768)) continue;
    const long long tiles = (long long)groups * ceil_div(rows, mp) * ceil_div(N, 128);
    const double there = rows < mp ? rows : mp;
    for (int s = 1; s <= 8; s *= 2) {
      if (s > 1 && (mp == 128 || tiles * s > (s == 8 ? sms * 13 / 8 : 2 * sms) || nk < 2 * s)) break;
      const double c = (double)tiles * s / sms, alone = (0.8 + 1.4 * (c < 2 ? c : 2)) / few_stages(mp, s > 1, tiles <= sms);
      double stage = 0.18 + 0.0004 * mp;
      if (alone > stage) stage = alone;
      if (c > 1 && c * (0.25 + 0.0005 * mp) > stage) stage = c * (0.25 + 0.0005 * mp);
      const double us = 2.4 + ceil_div(nk, s) * stage + (c > 1 ? c : 1) * there * (0.016 / s + (s > 1 ? 0.024 : 0)) + (s > 1 ? 0.38 : 0);
      if (us < least) least = us, best = Form{false, mp, s};
    }
  }
  if (rows < 40) return best;
  const int pairs = sms / 2 > 0 ? sms / 2 : 1;
  const long long turns = ((long long)groups * ceil_div(rows, 256) * ceil_div(N, 256) + pairs - 1) / pairs;
  best.pairs = 2.9 + turns * (0.34 * nk + 2.6) < least;
  return best;
}

// One packed argument, numbers of 64 bits in this order (see row_e4m3.cu).
struct LinearArgs {
  long long C, c_dtype, A, sa, W, sw, M, N, K, lda, ldw, ldc, epilogue, offsets, n_groups, w_group_stride, status;
};

}  // namespace

// The form that takes a product of so many groups of about so many rows on a device of `sms` SMs: 0 pairs, else rows of a tile | slices of K << 16.
LEB_API int leb_linear_e4m3_form(int groups, int rows, int N, int K, int sms) {
  const Form f = form_of(groups, rows, N, K, sms);
  return f.pairs ? 0 : f.rows | f.slices << 16;
}

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
  const Form f = form_of(groups, ceil_div(M, groups), N, K, sm_count());
  return f.pairs ? leb_gemm_e4m3_pairs(p, st) : leb_gemm_e4m3_few(p, f.rows, f.slices, st);
}
