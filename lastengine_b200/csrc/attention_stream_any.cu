// Decode attention with first positions for 32-bit caches, and for bfloat16 caches of heads that the tensor-core kernel does not take: one
// new token per sequence against its window and its sequence's first positions (first_tiles in common.cuh), any width of key and value
// heads up to 256.
//
// A decode step reads every visible key and value once, so the kernel is built around that stream, as the bfloat16 one is
// (attention_decode.cu): a block owns one sequence, up to HC query heads of one kv head and one share of the keys; its warps take tiles of
// 32 positions in turn, brought in by asynchronous copies into a place of the warp's own (the next keys while the weights are made, the
// next values when these are done with: more warps hide the trip better than a second place would), each with its own running
// (max, sum, acc) per head.  The arithmetic is the FMA pipes':
//  * scores: a lane owns a key and goes through its numbers in pieces of 16 bytes, the queries of the HC heads coming from shared memory
//    for all lanes at once (key rows are an odd number of pieces apart: no two lanes of a quarter meet a bank);
//  * weights: a lane makes those of its key, which then lie in shared memory for the values' lanes;
//  * values, stored [dim][position]: a lane multiplies four positions of a dimension with their weights for all HC heads; the eight
//    lanes' sums are added up once, at the end.
// Warps join through shared memory, the blocks that share a sequence's keys as a cluster.  Everything is float; exponentials are expf.
//
// Bound by the instructions of a tile (some 900 a warp with four heads of 64, 2.4 us with the SM's twelve warps), not by memory: 32 streams
// of 100 to 3,000 positions, window 1,024, 32 heads of 64 over 8: 34 us (68 MB, 2.0 TB/s; the general kernel 155), 64 streams with heads of
// 128, one query head each: 55 us (270 MB, 4.9 TB/s).  Measured beside it: eight lanes a key and sums by exchange 51 and 53 us, with two
// tiles' places a warp and four warps an SM 70.
// bfloat16, 32 streams, window 1,024: 16 heads of 80 over 8 54 us (84 MB, 1.6 TB/s), 8 of 256 over 4 58 us (135 MB, 2.3), 16 of 192 over 8 81 us (203 MB, 2.5).
#include "common.cuh"

#define ASF_NEG (-1e30f)

__device__ __forceinline__ void asf_cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void asf_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ float asf_remote(const float* p, int rank) {
  uint32_t a;
  float v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}

// Sums over the eight lanes that differ in the lowest three bits.  x[HC]: afterwards x[0] is the sum of x[asf_head(lane)] (all of
// them where HC is 1): halves of the heads change sides while there are several, what is left is added up.
template <int HC>
__device__ __forceinline__ void asf_sum8(float (&x)[HC], int lane) {
  int n = HC;
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    if (n > 1) {
      const bool upper = lane & o;
      n >>= 1;
#pragma unroll
      for (int h = 0; h < HC / 2; h++) {
        if (h < n) {
          const float give = upper ? x[h] : x[h + n], keep = upper ? x[h + n] : x[h];
          x[h] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
      }
    } else {
      x[0] += __shfl_xor_sync(0xffffffffu, x[0], o);
    }
  }
}
template <int HC>
__device__ __forceinline__ int asf_head(int lane) {
  return HC == 4 ? ((lane & 1) << 1 | (lane >> 1 & 1)) : HC == 2 ? (lane & 1) : 0;
}

__device__ __forceinline__ float asf_max(float v) {      // over the warp
  float m;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
}

// T: the cache's numbers; D: heads of up to D numbers; HC: query heads of a block (1, 2 or 4); VEC: a key is a number of 16-byte pieces.
template <typename T, int D, int HC, bool VEC>
__global__ void __launch_bounds__(128, D <= 64 ? 3 : D <= 128 ? 2 : 1)
attention_stream_any_kernel(T* __restrict__ out, const T* __restrict__ q, const T* __restrict__ k_pool,
                            const T* __restrict__ v_pool, const int* __restrict__ block_table, int bt_width,
                            const int* __restrict__ seq_slot, const int* __restrict__ seq_pos0, const int* __restrict__ seq_qstart,
                            const int* __restrict__ row_seq, const int* __restrict__ row_pos, const T* __restrict__ gate, int gate_stride, int gate_elem, int nh, int nkv, int hd, int vd, int page_size,
                            int window, int chunk, int first, float scale, const float* __restrict__ slopes,
                            const float* __restrict__ sinks, int n_splits) {
  constexpr int NV = D / 4, E = 16 / sizeof(T), VP = 32 / E;      // numbers of a 16-byte piece, pieces of a dimension's 32 values
  extern __shared__ __align__(128) float asf_smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int c = lane & 7, g = lane >> 3;
  const int G = nh / nkv, n_hc = (G + HC - 1) / HC;
  const int kvh = blockIdx.x / n_hc, hc = blockIdx.x % n_hc, b = blockIdx.y, split = blockIdx.z;
  const int h0 = kvh * G + hc * HC, heads = min(HC, G - hc * HC);
  pdl_wait();
  // a block's row: that of sequence b, or (row_seq) row b, of any sequence
  const int seq = row_seq ? row_seq[b] : b, slot = seq_slot[seq];
  const size_t m_row = row_seq ? b : seq_qstart[b];
  // (as in the bfloat16 kernel: out has one row per sequence of the launch; the same for all blocks of a cluster)
  if (m_row >= gridDim.y) return;
  if (slot < 0) {  // padding sequence
    for (int idx = split * blockDim.x + threadIdx.x; idx < heads * vd; idx += n_splits * blockDim.x)
      out[(m_row * nh + h0 + idx / vd) * vd + idx % vd] = from_f32<T>(0.f);
    return;
  }
  const int qpos = row_seq ? row_pos[b] : seq_pos0[b], kv_len = qpos + 1;
  const int key_lo = first_key(qpos, window, chunk);
  const int n_first = first_tiles(first, key_lo, 32), shift = key_lo / 32 - n_first;
  const int n_tiles = (kv_len - 1) / 32 - shift + 1, per_split = (n_tiles + n_splits - 1) / n_splits;
  const int t_lo = split * per_split, t_hi = min(n_tiles, t_lo + per_split);
  const int* table = block_table + (size_t)seq * bt_width;
  const int pieces = hd / E, row = VEC ? E * (pieces | 1) : hd;         // numbers from a key to the next
  const int k_numbers = 32 * row, stage = k_numbers + 32 * vd;         // of a tile: keys [32][row], values [vd][32]
  T* ks = reinterpret_cast<T*>(asf_smem) + (size_t)warp * stage;
  T* vs = ks + k_numbers;
  float* weight_s = reinterpret_cast<float*>(reinterpret_cast<T*>(asf_smem) + (size_t)warps * stage) + warp * HC * 32;      // [HC][32]
  float* q_s = weight_s + (warps - warp) * HC * 32;                      // [HC][q_row]
  const int q_row = (hd + 3) & ~3;

  auto key_of = [&](int tile) { return (tile >= n_first ? tile + shift : tile) * 32; };
  const uint32_t k_to = (uint32_t)__cvta_generic_to_shared(ks), v_to = (uint32_t)__cvta_generic_to_shared(vs) + 16 * lane;
  const int v_step = 32 / VP * page_size;      // a warp's pass copies 32 / VP dimensions
  auto page_of = [&](int tile) { return max(table[key_of(tile) / page_size], 0); };
  // a lane's pieces of a tile of keys: the first one's key and place, the steps to the next
  const int k_r0 = VEC ? lane / pieces : 0, k_c0 = VEC ? lane % pieces : 0, k_rs = VEC ? 32 / pieces : 0, k_cs = VEC ? 32 % pieces : 0;
  auto issue_k = [&](int tile, int page) {      // (in the cache a tile's keys lie together)
    if (tile < t_hi) {
      const T* src = k_pool + (((size_t)page * nkv + kvh) * page_size + key_of(tile) % page_size) * hd + E * lane;
      if (VEC) {
        int r = k_r0, c4 = k_c0;
#pragma unroll 4
        for (int i = lane, n = 0; i < 32 * pieces; i += 32, n++) {
          asf_cp16(k_to + sizeof(T) * (r * row + E * c4), src + 32 * E * n);
          r += k_rs;
          c4 += k_cs;
          if (c4 >= pieces) c4 -= pieces, r++;
        }
      } else {
        for (int i = lane, n = 0; i < 2 * hd * (int)sizeof(T); i += 32, n++) asf_cp16(k_to + 16 * i, src + 32 * E * n);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto issue_v = [&](int tile, int page) {
    if (tile < t_hi) {
      const T* src = v_pool + (((size_t)page * nkv + kvh) * vd + lane / VP) * page_size + key_of(tile) % page_size + E * (lane % VP);
#pragma unroll 4
      for (int i = lane, n = 0; i < VP * vd; i += 32, n++) asf_cp16(v_to + 512 * n, src + (size_t)v_step * n);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  int page = t_lo + warp < t_hi ? page_of(t_lo + warp) : 0;
  issue_k(t_lo + warp, page);
  issue_v(t_lo + warp, page);

  for (int i = threadIdx.x; i < HC * hd; i += blockDim.x) {
    const int h = i / hd, d = i - h * hd;
    q_s[h * q_row + d] = h < heads ? to_f32(q[(m_row * nh + h0 + h) * hd + d]) * scale : 0.f;
  }
  __syncthreads();
  float slope[HC];
#pragma unroll
  for (int h = 0; h < HC; h++) slope[h] = slopes && h < heads ? slopes[h0 + h] : 0.f;

  float mx[HC], l[HC], acc[NV][HC];
#pragma unroll
  for (int h = 0; h < HC; h++) {
    mx[h] = ASF_NEG;
    l[h] = 0.f;
#pragma unroll
    for (int i = 0; i < NV; i++) acc[i][h] = 0.f;
  }
  for (int tile = t_lo + warp; tile < t_hi; tile += warps) {
    page = tile + warps < t_hi ? page_of(tile + warps) : 0;
    asm volatile("cp.async.wait_group 1;" ::: "memory");      // the keys (their values may be on their way)
    __syncwarp();
    const int key0 = key_of(tile);
    float x[HC];
#pragma unroll
    for (int h = 0; h < HC; h++) x[h] = 0.f;
    const T* mine = ks + lane * row;
    if (VEC) {
#pragma unroll 4
      for (int d = 0; d < hd; d += 4) {
        const float4 kk = load4(mine + d);
#pragma unroll
        for (int h = 0; h < HC; h++) {
          const float4 qq = load4(q_s + h * q_row + d);
          x[h] = fmaf(kk.x, qq.x, x[h]);
          x[h] = fmaf(kk.y, qq.y, x[h]);
          x[h] = fmaf(kk.z, qq.z, x[h]);
          x[h] = fmaf(kk.w, qq.w, x[h]);
        }
      }
    } else {
      for (int d = 0; d < hd; d++) {
        const float kk = to_f32(mine[d]);
#pragma unroll
        for (int h = 0; h < HC; h++) x[h] = fmaf(kk, q_s[h * q_row + d], x[h]);
      }
    }
    __syncwarp();      // everyone is done with the keys
    issue_k(tile + warps, page);
    const bool partial = (key0 < key_lo && key0 + 32 > first) || key0 + 32 > kv_len;
    const int kp = key0 + lane;
    const bool read = kp < kv_len && (kp >= key_lo || kp < first);
    bool moved = false;
    float corr[HC];
#pragma unroll
    for (int h = 0; h < HC; h++) {
      if (slopes) x[h] -= slope[h] * (float)(qpos - kp);
      const float mn = fmaxf(mx[h], asf_max(read ? x[h] : ASF_NEG));
      corr[h] = expf(mx[h] - mn);
      moved |= mn != mx[h];
      mx[h] = mn;
      const float w = read ? expf(x[h] - mn) : 0.f;
      l[h] = l[h] * corr[h] + w;      // of this lane's keys
      weight_s[h * 32 + lane] = w;
    }
    __syncwarp();
    float p[HC][4];
#pragma unroll
    for (int h = 0; h < HC; h++) {
      const float4 w = load4(weight_s + h * 32 + 4 * c);
      p[h][0] = w.x, p[h][1] = w.y, p[h][2] = w.z, p[h][3] = w.w;
    }
    if (moved) {      // (the same for all lanes: maxima are)
#pragma unroll
      for (int i = 0; i < NV; i++)
#pragma unroll
        for (int h = 0; h < HC; h++) acc[i][h] *= corr[h];
    }
    asm volatile("cp.async.wait_group 1;" ::: "memory");      // the values (the next keys may be on their way)
    __syncwarp();
    if (partial) {
      const uint32_t seen = __ballot_sync(0xffffffffu, read) >> (4 * c);
#pragma unroll
      for (int i = 0; i < NV; i++) {
        if (4 * i + g < vd) {
          float4 v4 = load4(vs + (4 * i + g) * 32 + 4 * c);      // zero times whatever lies where nothing is read would not be zero
          v4.x = seen & 1 ? v4.x : 0.f, v4.y = seen & 2 ? v4.y : 0.f, v4.z = seen & 4 ? v4.z : 0.f, v4.w = seen & 8 ? v4.w : 0.f;
#pragma unroll
          for (int h = 0; h < HC; h++) acc[i][h] += v4.x * p[h][0] + v4.y * p[h][1] + v4.z * p[h][2] + v4.w * p[h][3];
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < NV; i++) {
        if (4 * i + g < vd) {
          const float4 v4 = load4(vs + (4 * i + g) * 32 + 4 * c);
#pragma unroll
          for (int h = 0; h < HC; h++) acc[i][h] += v4.x * p[h][0] + v4.y * p[h][1] + v4.z * p[h][2] + v4.w * p[h][3];
        }
      }
    }
    __syncwarp();      // everyone is done with the values and the scores
    issue_v(tile + warps, page);
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();     // the rings are done with: their memory takes the results
  float* o_s = asf_smem;                                // [warp][HC][vd]
  float* m_s = o_s + warps * HC * vd;                   // [warp][HC]
  float* l_s = m_s + warps * HC;
  float* mine = l_s + warps * HC;                       // this block's rows, for the cluster's blocks to read: [HC][vd], maxima, sums
#pragma unroll
  for (int h = 0; h < HC; h++) l[h] = warp_sum(l[h]);
  const int head = asf_head<HC>(lane);
#pragma unroll
  for (int i = 0; i < NV; i++) {
    if (4 * i >= vd) break;
    asf_sum8<HC>(acc[i], lane);
    if (c < HC && 4 * i + g < vd) o_s[(warp * HC + head) * vd + 4 * i + g] = acc[i][0];
  }
  if (g == 0 && c < HC) {
    float top = mx[0], sum = l[0];
#pragma unroll
    for (int h = 1; h < HC; h++) top = head == h ? mx[h] : top, sum = head == h ? l[h] : sum;
    m_s[warp * HC + head] = top;
    l_s[warp * HC + head] = sum;
  }
  __syncthreads();
  auto finish = [&](int idx, float M, float L, float a) {
    const int h = h0 + idx / vd, d = idx % vd;
    const float inv = sinks ? sink_quotient(M, L, sinks[h]) : (L > 0.f ? 1.0f / L : 0.f);
    out[(m_row * nh + h) * vd + d] = from_f32<T>(a * inv * (gate ? head_gate(gate, m_row, gate_stride, h, d, vd, gate_elem) : 1.f));
  };
  for (int idx = threadIdx.x; idx < heads * vd; idx += blockDim.x) {
    const int h = idx / vd;
    float M = ASF_NEG, L = 0.f, a = 0.f;
    for (int w = 0; w < warps; w++) M = fmaxf(M, m_s[w * HC + h]);
    for (int w = 0; w < warps; w++) {
      const float f = expf(m_s[w * HC + h] - M);
      L += l_s[w * HC + h] * f;
      a += o_s[w * HC * vd + idx] * f;
    }
    if (n_splits == 1) {
      finish(idx, M, L, a);
    } else {
      mine[idx] = a;
      if (idx % vd == 0) mine[HC * vd + h] = M, mine[HC * vd + HC + h] = L;
    }
  }
  if (n_splits > 1) {
    asf_cluster_sync();
    for (int idx = split * blockDim.x + threadIdx.x; idx < heads * vd; idx += n_splits * blockDim.x) {
      const int h = idx / vd;
      float ms[8], ls[8], as[8];      // a cluster has eight blocks at most; all are asked for together
      float M = ASF_NEG, L = 0.f, a = 0.f;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const int rank = min(j, n_splits - 1);
        ms[j] = asf_remote(mine + HC * vd + h, rank);
        ls[j] = asf_remote(mine + HC * vd + HC + h, rank);
        as[j] = asf_remote(mine + idx, rank);
      }
#pragma unroll
      for (int j = 0; j < 8; j++) M = fmaxf(M, ms[j]);
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float f = j < n_splits ? expf(ms[j] - M) : 0.f;
        L += ls[j] * f;
        a += as[j] * f;
      }
      finish(idx, M, L, a);
    }
    asf_cluster_sync();      // no block ends while others read its memory
  }
}

// Returns 1 when the sizes are ones this kernel takes.
LEB_API int leb_attention_stream_any_supported(int nh, int nkv, int hd, int vd, int page_size) {
  return nkv > 0 && nh % nkv == 0 && hd >= 1 && hd <= 256 && vd >= 1 && vd <= 256 && page_size > 0 && page_size % 32 == 0;
}

template <typename T>
static int launch_attention_stream_any(T* out, const T* q, const T* k_pool, const T* v_pool, const int* block_table, int bt_width,
                                       const int* seq_slot, const int* seq_pos0, const int* seq_qstart, const int* row_seq, const int* row_pos,
                                       const T* gate, int gate_stride,
                                       int gate_elem, int B, int nh, int nkv, int hd, int vd, int page_size, int window, int chunk, int first,
                                       float scale, const float* slopes, const float* sinks, int max_kvlen, int blocks, cudaStream_t st) {
  constexpr int E = 16 / sizeof(T);
  const int G = nh / nkv, widest = hd > vd ? hd : vd;
  const int HC = G == 1 ? 1 : widest > 128 ? 2 : 4, n_hc = ceil_div(G, HC);
  const bool vec = hd % E == 0;
  const int row = vec ? E * (hd / E | 1) : hd;
  const size_t stage = (size_t)32 * (row + vd) * sizeof(T);
  const int warps = stage <= 17 * 1024 ? 4 : 3;      // three blocks an SM; with wider 32-bit heads two or one
  const size_t rings = warps * (stage + HC * 32 * sizeof(float)) + HC * ((hd + 3) & ~3) * sizeof(float);
  const size_t results = ((size_t)(warps + 1) * HC * (vd + 2)) * sizeof(float), smem = rings > results ? rings : results;
  // blocks of a cluster: as many as run at once (to the nearest), with a tile a warp or more for each.  us of 1, 2, 4, 8 blocks: one stream of
  // 1,000 positions 25.1, 15.9, 11.0, 8.5; 32 streams of 100 to 3,000, window 1,024, 256 blocks where 444 fit, 38.9, 33.9, 41.4, 61.6; 64
  // streams with heads of 128, 256 where 296 fit, 55.0, 58.6, 72.4, 109.9
  long long keys = window > 0 ? window : max_kvlen;
  if (chunk > 0 && chunk < keys) keys = chunk;
  keys = keys + first < max_kvlen ? keys + first : max_kvlen;
  const long long per = (long long)B * nkv * n_hc, fit = 220 * 1024 / (long long)(smem + 2048);
  const long long room = (long long)sm_count() * (fit < 1 ? 1 : fit > 3 ? 3 : fit), most = keys / (32 * warps);
  long long n = (2 * room + per) / (2 * per);
  n = n < most ? n : most;
  if (blocks > 0) n = blocks;
  const int n_splits = (int)(n < 1 ? 1 : n > 8 ? 8 : n);
  dim3 grid(nkv * n_hc, B, n_splits);
  LEB_REQUIRE(grid.y <= 65535, "leb_attention_stream_any: grid too large");
#define LEB_ASF_K(D_, HC_, VEC_)                                                                                                      \
  {                                                                                                                                   \
    constexpr auto kern = attention_stream_any_kernel<T, D_, HC_, VEC_>;                                                              \
    const cudaError_t e = leb_allow_smem<kern>();                                                                                     \
    if (e != cudaSuccess) return leb_fail("leb_attention_stream_any: shared memory %zu: %s", smem, cudaGetErrorString(e));            \
    leb_launch_cluster(n_splits, kern, grid, dim3(32 * warps), smem, st, out, q, k_pool, v_pool, block_table, bt_width, seq_slot, seq_pos0, \
                       seq_qstart, row_seq, row_pos, gate, gate_stride, gate_elem, nh, nkv, hd, vd, page_size, window, chunk, first, scale, slopes, sinks, n_splits); \
  }
#define LEB_ASF(D_, HC_)               \
  {                                    \
    if (vec) LEB_ASF_K(D_, HC_, true) else LEB_ASF_K(D_, HC_, false) \
  }
  if (widest <= 64) {
    if (HC == 1) LEB_ASF(64, 1) else LEB_ASF(64, 4)
  } else if (widest <= 128) {
    if (HC == 1) LEB_ASF(128, 1) else LEB_ASF(128, 4)
  } else {
    if (HC == 1) LEB_ASF(256, 1) else LEB_ASF(256, 2)
  }
#undef LEB_ASF
#undef LEB_ASF_K
  LEB_CHECK_LAUNCH("leb_attention_stream_any");
  return 0;
}

// A decode step: every sequence brings one row; or, with row_seq and row_pos [B], B rows of any sequences (each then reads its keys by
// itself: for chunks of few rows).  q [B][nh*hd], out [B][nh*vd], pools [page][nkv][page_size][hd] and
// [page][nkv][vd][page_size] on 16-byte boundaries, all of `dtype`.  max_kvlen: the most positions a sequence holds; blocks: of a cluster
// that shares a sequence's keys (0: as many as suit the step).
LEB_API int leb_attention_stream_any(void* out, const void* q, const void* k_pool, const void* v_pool, int dtype, const int* block_table,
                                     int bt_width, const int* seq_slot, const int* seq_pos0, const int* seq_qstart, const int* row_seq,
                                     const int* row_pos, const void* gate, int gate_stride, int gate_elem, int B, int nh, int nkv, int hd, int vd, int page_size, int window, int chunk,
                                     int first, float scale, const float* slopes, const float* sinks, int max_kvlen, int blocks, cudaStream_t st) {
  if (B <= 0) return 0;
  LEB_REQUIRE(leb_attention_stream_any_supported(nh, nkv, hd, vd, page_size),
              "leb_attention_stream_any: sizes not taken (heads %d, kv heads %d, widths %d and %d, page %d)", nh, nkv, hd, vd, page_size);
  LEB_REQUIRE((row_seq == nullptr) == (row_pos == nullptr), "leb_attention_stream_any: rows come with their sequences and positions");
  LEB_REQUIRE((((uintptr_t)k_pool | (uintptr_t)v_pool) & 15) == 0, "leb_attention_stream_any: pools must be 16-byte aligned");
#define LEB_ASF_T(T)                                                                                                                    \
  launch_attention_stream_any((T*)out, (const T*)q, (const T*)k_pool, (const T*)v_pool, block_table, bt_width, seq_slot, seq_pos0, seq_qstart, \
                              row_seq, row_pos, (const T*)gate, gate_stride, gate_elem, B, nh, nkv, hd, vd, page_size, window, chunk, first, scale, slopes, \
                              sinks, max_kvlen, blocks, st)
  if (dtype == LEB_F32) return LEB_ASF_T(float);
  if (dtype == LEB_BF16) return LEB_ASF_T(bf16);
#undef LEB_ASF_T
  return leb_fail("leb_attention_stream_any: unknown dtype %d", dtype);
}
