// Chunks with first positions for 32-bit caches, and for bfloat16 caches of heads and pages that no tensor-core kernel takes: any width of
// key and value heads up to 256, up to 64 query heads a kv head.
//
// A block owns 64 rows (positions times the query heads of one kv head, so that a tile's keys serve them all) and walks the tiles of 32
// positions that any of its rows sees, the first positions' before the window's (first_tiles in common.cuh).  The arithmetic is the FMA
// pipes', in tiles that stay in registers: of the 64 x 32 scores a thread has four rows by four keys, of the 64 x vd results the same four
// rows by an eighth of the dimensions, so that eight lanes share a row from the scores to its sum.  Operands lie in shared memory, keys and
// queries an odd number of 16-byte pieces apart, values as they lie in the cache ([dimension][position]): four numbers a load, no two lanes of
// a quarter at one bank.  The next tile is on its way while a tile is worked on (32-bit: asynchronous copies; bfloat16 becomes float on the way).
// Scores, weights, maxima and sums are float; scores carry log2(e), exponentials are exp2f.
//
// A row's weights of positions it does not see are zero, and where a tile has such positions a zero weight takes its value for zero: an
// infinity that one row sees stays out of the others.
//
// Bound by shared memory's loads (224 of 16 bytes a lane for a tile's 2,048 multiplications, 1.9 us of an SM) and, with few blocks, by their latency: 2,000
// rows, window 1,024, 32 heads of 64 over 8 take 550 us (34% of the FMA pipes' rate; a row by itself, attention_stream_any.cu, 1,063), 700 rows 281 (474),
// with heads of 128, 16 over 2, 372 (655).  Few rows or short windows are the other kernel's: 32 rows 51 us and 47.
#include "common.cuh"

#define ASR_NEG (-1e30f)
#define ASR_ROWS 64
#define ASR_KEYS 32
#define ASR_PITCH (ASR_KEYS + 4)      // numbers from a row of weights, or a dimension of values, to the next

__device__ __forceinline__ void asr_cp16(float* dst, const float* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void asr_cp4(float* dst, const float* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void asr_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ float asr_remote(const float* p, int rank) {
  uint32_t a;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float asr_dot(float4 a, float4 b, float s) {
  return fmaf(a.w, b.w, fmaf(a.z, b.z, fmaf(a.y, b.y, fmaf(a.x, b.x, s))));
}
// Numbers from a query or key to the next.
__host__ __device__ __forceinline__ int asr_pitch(int hd) { return 4 * ((hd + 3) / 4 | 1); }

// T: the cache's numbers; D: value heads of up to D numbers.
template <typename T, int D>
__global__ void __launch_bounds__(128, D <= 64 ? 3 : D <= 128 ? 2 : 1)
attention_stream_rows_kernel(T* __restrict__ out, const T* __restrict__ q, const T* __restrict__ k_pool, const T* __restrict__ v_pool,
                             const int* __restrict__ block_table, int bt_width, const int* __restrict__ seq_slot,
                             const int* __restrict__ seq_pos0, const int* __restrict__ seq_qstart, const int* __restrict__ seq_qlen,
                             const T* __restrict__ gate, int gate_stride, int gate_elem, int M, int nh, int nkv, int hd, int vd, int page_size,
                             int window, int chunk, int first, float scale, const float* __restrict__ slopes, const float* __restrict__ sinks, int n_splits) {
  constexpr int ND = D / 8;
  extern __shared__ __align__(128) float asr_smem[];
  const int G = nh / nkv, TP = ASR_ROWS / G, pitch = asr_pitch(hd);
  const int v_rows = (vd + 7) & ~7, stage = ASR_KEYS * pitch + v_rows * ASR_PITCH;
  float* q_s = asr_smem;                          // [64][pitch]
  float* p_s = q_s + ASR_ROWS * pitch;            // [64][ASR_PITCH]
  float* stages = p_s + ASR_ROWS * ASR_PITCH;     // two of: keys [32][pitch], values [v_rows][ASR_PITCH]
  pdl_wait();
  // kv heads vary fastest; of a sequence's tiles the ones with the longest key range come first
  const int kvh = blockIdx.x, b = blockIdx.y, split = blockIdx.z % n_splits;
  const int row0 = (int)(gridDim.z / n_splits - 1 - blockIdx.z / n_splits) * TP;
  const int qlen = seq_qlen[b], start = seq_qstart[b];
  if (row0 >= qlen || start < 0 || start + qlen > M) return;
  const int np = min(TP, qlen - row0), rows = np * G, h0 = kvh * G;
  const size_t m_base = (size_t)start + row0;
  if (seq_slot[b] < 0) {      // a padding sequence: its rows are zero
    for (int idx = split * 128 + threadIdx.x; idx < rows * vd; idx += n_splits * 128) {
      const int r = idx / vd;
      out[((m_base + r / G) * nh + h0 + r % G) * vd + idx % vd] = from_f32<T>(0.f);
    }
    return;
  }
  const int q_lo = seq_pos0[b] + row0, q_hi = q_lo + np - 1;
  const int key_lo = first_key(q_lo, window, chunk), key_last = first_key(q_hi, window, chunk);
  const int nf = first_tiles(first, key_lo, ASR_KEYS), jb0 = key_lo / ASR_KEYS, n_all = nf + q_hi / ASR_KEYS - jb0 + 1;
  // this block's share of the tiles (none for the last ones where they do not go round)
  const int per_split = (n_all + n_splits - 1) / n_splits, t_lo = min(n_all, split * per_split), t_hi = min(n_all, t_lo + per_split);
  const int* table = block_table + (size_t)b * bt_width;
  auto key_of = [&](int t) { return (t < nf ? t : jb0 + t - nf) * ASR_KEYS; };

  // numbers behind a head's width are zero, of queries and of keys
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll 4
  for (int r = warp; r < ASR_ROWS; r += 4) {
    const T* mine = q + ((m_base + r / G) * nh + h0 + r % G) * (size_t)hd;
    for (int d = lane; d < pitch; d += 32) q_s[r * pitch + d] = r < rows && d < hd ? to_f32(mine[d]) : 0.f;
  }
  for (int idx = threadIdx.x; idx < 2 * ASR_KEYS * (pitch - hd); idx += 128) {
    const int k = idx / (pitch - hd), d = hd + idx % (pitch - hd);
    stages[(k / ASR_KEYS) * stage + (k % ASR_KEYS) * pitch + d] = 0.f;
  }
  // a thread's pieces of a tile of keys (numbers where a key is no number of pieces): the first one's key and place, the steps to the next
  const bool vec = hd % 4 == 0;
  const int per_key = vec ? hd / 4 : hd, k_r0 = threadIdx.x / per_key, k_c0 = threadIdx.x % per_key, k_rs = 128 / per_key, k_cs = 128 % per_key;
  auto pieces = [&](auto f) {
    int r = k_r0, c = k_c0;
    for (int i = threadIdx.x; i < ASR_KEYS * per_key; i += 128) {
      f(i, r, c);
      r += k_rs;
      c += k_cs;
      if (c >= per_key) c -= per_key, r++;
    }
  };
  auto page_of = [&](int t) { return t < t_hi ? max(table[key_of(t) / page_size], 0) : 0; };
  int page = page_of(t_lo);      // of the next tile: asked for a tile ahead
  auto issue = [&](int t) {
    if (t < t_hi) {
      const int off = key_of(t) % page_size;
      float* ks = stages + (t & 1) * stage;
      float* vs = ks + ASR_KEYS * pitch;
      const T* k_src = k_pool + (((size_t)page * nkv + kvh) * page_size + off) * hd;
      const T* v_src = v_pool + ((size_t)page * nkv + kvh) * vd * page_size + off;
      page = page_of(t + 1);
      if constexpr (sizeof(T) == 4) {
        if (vec) pieces([&](int i, int r, int c) { asr_cp16(ks + r * pitch + 4 * c, k_src + 4 * i); });
        else pieces([&](int i, int r, int c) { asr_cp4(ks + r * pitch + c, k_src + i); });
        for (int i = threadIdx.x; i < vd * 8; i += 128) asr_cp16(vs + (i >> 3) * ASR_PITCH + 4 * (i & 7), v_src + (size_t)(i >> 3) * page_size + 4 * (i & 7));
      } else {
        if (vec) pieces([&](int i, int r, int c) { *reinterpret_cast<float4*>(ks + r * pitch + 4 * c) = load4(k_src + 4 * i); });
        else pieces([&](int i, int r, int c) { ks[r * pitch + c] = to_f32(k_src[i]); });
        for (int i = threadIdx.x; i < vd * 8; i += 128)
          *reinterpret_cast<float4*>(vs + (i >> 3) * ASR_PITCH + 4 * (i & 7)) = load4(v_src + (size_t)(i >> 3) * page_size + 4 * (i & 7));
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  const int kg = threadIdx.x & 7, rg = threadIdx.x >> 3;      // keys and dimensions kg + 8 j, rows rg + 16 i
  const float scale2 = scale * 1.4426950408889634f;
  float mx[4], l[4], slope2[4], acc[4][ND];
  int pos[4], lo[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int r = rg + 16 * i;
    pos[i] = r < rows ? q_lo + r / G : -1;      // (a row that is none sees nothing)
    lo[i] = first_key(pos[i], window, chunk);
    slope2[i] = slopes && r < rows ? slopes[h0 + r % G] * 1.4426950408889634f : 0.f;
    mx[i] = ASR_NEG;
    l[i] = 0.f;
#pragma unroll
    for (int n = 0; n < ND; n++) acc[i][n] = 0.f;
  }

  issue(t_lo);
  for (int t = t_lo; t < t_hi; t++) {
    const int key0 = key_of(t);
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();      // this tile is there for all, and all are done with the one before
    issue(t + 1);
    const float* ks = stages + (t & 1) * stage;
    const float* vs = ks + ASR_KEYS * pitch;
    float s[4][4];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int j = 0; j < 4; j++) s[i][j] = 0.f;
#pragma unroll 2
    for (int d = 0; d < hd; d += 4) {
      float4 kk[4];
#pragma unroll
      for (int j = 0; j < 4; j++) kk[j] = load4(ks + (kg + 8 * j) * pitch + d);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float4 qq = load4(q_s + (rg + 16 * i) * pitch + d);
#pragma unroll
        for (int j = 0; j < 4; j++) s[i][j] = asr_dot(qq, kk[j], s[i][j]);
      }
    }
    // whether every row of the block sees all of the tile (places of rows that are none are not stored)
    const bool whole = key0 + ASR_KEYS - 1 <= q_lo && (key0 >= key_last || key0 + ASR_KEYS <= first);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      float top = mx[i];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int key = key0 + kg + 8 * j;
        s[i][j] = s[i][j] * scale2 - slope2[i] * (float)(pos[i] - key);
        if (!whole && (key > pos[i] || (key < lo[i] && key >= first))) s[i][j] = ASR_NEG;
        top = fmaxf(top, s[i][j]);
      }
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float corr = exp2f(mx[i] - top);
      mx[i] = top;
      l[i] *= corr;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float p = s[i][j] == ASR_NEG ? 0.f : exp2f(s[i][j] - top);
        l[i] += p;
        p_s[(rg + 16 * i) * ASR_PITCH + kg + 8 * j] = p;
      }
#pragma unroll
      for (int n = 0; n < ND; n++) acc[i][n] *= corr;
    }
    __syncwarp();      // (a row's eight lanes are of one warp)
    auto product = [&](auto masked) {
#pragma unroll 1
      for (int k = 0; k < ASR_KEYS; k += 4) {
        float4 p[4];
#pragma unroll
        for (int i = 0; i < 4; i++) p[i] = load4(p_s + (rg + 16 * i) * ASR_PITCH + k);
#pragma unroll
        for (int n = 0; n < ND; n++) {
          if (8 * n >= vd) break;
          const float4 v = load4(vs + (kg + 8 * n) * ASR_PITCH + k);
#pragma unroll
          for (int i = 0; i < 4; i++) {
            float4 w = v;
            if (decltype(masked)::value) {
              w.x = p[i].x == 0.f ? 0.f : v.x, w.y = p[i].y == 0.f ? 0.f : v.y;
              w.z = p[i].z == 0.f ? 0.f : v.z, w.w = p[i].w == 0.f ? 0.f : v.w;
            }
            acc[i][n] = asr_dot(p[i], w, acc[i][n]);
          }
        }
      }
    };
    if (whole) product(std::false_type{});
    else product(std::true_type{});
    __syncwarp();      // the weights may be written again
  }
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], o);
  auto quotient = [&](float m, float sum, int h) { return sinks ? sink_quotient(m * 0.6931471805599453f, sum, sinks[h]) : (sum > 0.f ? 1.0f / sum : 0.f); };
  auto store = [&](int r, int d, float x) {
    const size_t m = m_base + r / G;
    const int h = h0 + r % G;
    out[(m * nh + h) * (size_t)vd + d] = from_f32<T>(x * (gate ? head_gate(gate, m, gate_stride, h, d, vd, gate_elem) : 1.f));
  };
  if (n_splits == 1) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int r = rg + 16 * i;
      if (r >= rows) continue;
      const float inv = quotient(mx[i], l[i], h0 + r % G);
#pragma unroll
      for (int n = 0; n < ND; n++)
        if (kg + 8 * n < vd) store(r, kg + 8 * n, acc[i][n] * inv);
    }
    return;
  }
  // The blocks of a cluster join: each has its rows, their maxima and sums in shared memory (the tiles are done with), and adds up its share of
  // the rows over all blocks, in the blocks' order.
  __syncthreads();
  float* o_s = stages;                       // [64][vd]
  float* m_s = p_s;                          // maxima, sums, then factors [row of the share][block]
  float* l_s = m_s + ASR_ROWS;
  float* f_s = l_s + ASR_ROWS;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int r = rg + 16 * i;
    if (kg == 0) m_s[r] = mx[i], l_s[r] = l[i];
#pragma unroll
    for (int n = 0; n < ND; n++)
      if (kg + 8 * n < vd) o_s[r * vd + kg + 8 * n] = acc[i][n];
  }
  asr_cluster_sync();
  const int share = (rows + n_splits - 1) / n_splits, r0 = split * share, n_rows = min(share, rows - r0);
  for (int i = threadIdx.x; i < n_rows; i += 128) {
    float top = ASR_NEG, sum = 0.f;
    for (int j = 0; j < n_splits; j++) top = fmaxf(top, asr_remote(m_s + r0 + i, j));
    for (int j = 0; j < n_splits; j++) sum += asr_remote(l_s + r0 + i, j) * exp2f(asr_remote(m_s + r0 + i, j) - top);
    const float inv = quotient(top, sum, h0 + (r0 + i) % G);
    for (int j = 0; j < n_splits; j++) f_s[i * n_splits + j] = inv * exp2f(asr_remote(m_s + r0 + i, j) - top);
  }
  __syncthreads();
  for (int idx = threadIdx.x; idx < n_rows * vd; idx += 128) {
    const int i = idx / vd;
    float x = 0.f;
#pragma unroll
    for (int j = 0; j < 8; j++)      // (asked for together; a cluster has eight blocks at most)
      if (j < n_splits) x += f_s[i * n_splits + j] * asr_remote(o_s + r0 * vd + idx, j);
    store(r0 + i, idx - i * vd, x);
  }
  asr_cluster_sync();      // no block ends while others read its memory
}

static size_t asr_smem_bytes(int hd, int vd) {
  return sizeof(float) * ((size_t)ASR_ROWS * (asr_pitch(hd) + ASR_PITCH) + 2 * ((size_t)ASR_KEYS * asr_pitch(hd) + (size_t)((vd + 7) & ~7) * ASR_PITCH));
}

// Returns 1 when the sizes are ones this kernel takes.
LEB_API int leb_attention_stream_rows_supported(int nh, int nkv, int hd, int vd, int page_size) {
  return nkv > 0 && nh % nkv == 0 && nh / nkv <= ASR_ROWS && hd >= 1 && hd <= 256 && vd >= 1 && vd <= 256 && page_size > 0 && page_size % 32 == 0;
}

// Prompt attention of the step's rows over the paged cache (which already holds their keys and values).  q [M][nh*hd], out [M][nh*vd], pools
// [page][nkv][page_size][hd] and [page][nkv][vd][page_size] on 16-byte boundaries, all of `dtype`.  max_kvlen: the most positions a sequence holds; blocks: of a cluster
// that shares a tile's keys (0: as many as suit the step).
LEB_API int leb_attention_stream_rows(void* out, const void* q, const void* k_pool, const void* v_pool, int dtype, const int* block_table,
                                      int bt_width, const int* seq_slot, const int* seq_pos0, const int* seq_qstart, const int* seq_qlen,
                                      const void* gate, int gate_stride, int gate_elem, int M, int B, int nh, int nkv, int hd, int vd, int page_size,
                                      int window, int chunk, int first, float scale, const float* slopes, const float* sinks, int max_qlen,
                                      int max_kvlen, int blocks, cudaStream_t st) {
  if (B <= 0 || M <= 0 || max_qlen <= 0) return 0;
  LEB_REQUIRE(leb_attention_stream_rows_supported(nh, nkv, hd, vd, page_size),
              "leb_attention_stream_rows: sizes not taken (heads %d, kv heads %d, widths %d and %d, page %d)", nh, nkv, hd, vd, page_size);
  LEB_REQUIRE((((uintptr_t)k_pool | (uintptr_t)v_pool) & 15) == 0, "leb_attention_stream_rows: pools must be 16-byte aligned");
  const size_t smem = asr_smem_bytes(hd, vd);
  // blocks of a cluster that shares a tile's keys: as many as nine tenths of the places take (with all of them some clusters wait for a second
  // wave: 700 rows, 8 heads of 80 and 48, five blocks 145 us, four 106), two where the tiles are fewer than two waves, with two tiles of keys or more for each.
  // us of 1, 2, 4, 8 blocks, window 1,024, 32 heads of 64 over 8: 64 rows 173, 99, 79, 66, 256 rows 231, 159, 163, 178 (three: 123), 700 rows 291, 280,
  // 345, 439; 2,000 rows 550, 607, 708, 1,001
  const int TP = ASR_ROWS / (nh / nkv);
  const long long per_head = (long long)ceil_div(max_qlen, TP) * B, by_rows = (long long)M / TP + B, held = vd <= 64 ? 3 : vd <= 128 ? 2 : 1,
                  by_smem = 227 * 1024 / (long long)(smem + 1024), places = (long long)sm_count() * (by_smem < held ? by_smem : held);
  const long long tiles = (per_head < by_rows ? per_head : by_rows) * nkv, fits = places * 9 / (10 * tiles), room = fits < 2 && tiles < 2 * places ? 2 : fits;
  long long keys = window > 0 ? window : max_kvlen;
  if (chunk > 0 && chunk < keys) keys = chunk;
  keys += (long long)first + (TP < max_qlen ? TP : max_qlen);
  if (keys > max_kvlen) keys = max_kvlen;
  const long long most = keys / (2 * ASR_KEYS), want = blocks > 0 ? blocks : room < most ? room : most;
  const int n_splits = want >= 8 ? 8 : want < 1 ? 1 : (int)want;
  dim3 grid(nkv, B, ceil_div(max_qlen, TP) * n_splits);
  LEB_REQUIRE(grid.y <= 65535 && grid.z <= 65535, "leb_attention_stream_rows: grid too large (%u, %u)", grid.y, grid.z);
#define LEB_ASR(T, D)                                                                                                                        \
  {                                                                                                                                          \
    constexpr auto kern = attention_stream_rows_kernel<T, D>;                                                                                \
    const cudaError_t e = leb_allow_smem<kern>();                                                                                            \
    if (e != cudaSuccess) return leb_fail("leb_attention_stream_rows: shared memory %zu: %s", smem, cudaGetErrorString(e));                  \
    leb_launch_cluster(n_splits, kern, grid, dim3(128), smem, st, (T*)out, (const T*)q, (const T*)k_pool, (const T*)v_pool, block_table, bt_width, seq_slot,   \
               seq_pos0, seq_qstart, seq_qlen, (const T*)gate, gate_stride, gate_elem, M, nh, nkv, hd, vd, page_size, window, chunk, first,  \
               scale, slopes, sinks, n_splits);                                                                                                  \
  }
#define LEB_ASR_T(T)                       \
  {                                        \
    if (vd <= 64) LEB_ASR(T, 64)           \
    else if (vd <= 128) LEB_ASR(T, 128)    \
    else LEB_ASR(T, 256)                   \
  }
  if (dtype == LEB_F32) LEB_ASR_T(float)
  else if (dtype == LEB_BF16) LEB_ASR_T(bf16)
  else return leb_fail("leb_attention_stream_rows: unknown dtype %d", dtype);
#undef LEB_ASR_T
#undef LEB_ASR
  LEB_CHECK_LAUNCH("leb_attention_stream_rows");
  return 0;
}
