// Decode attention of 32-bit caches with first positions: one new token per sequence against its window and its sequence's first
// positions (first_tiles in common.cuh), any width of key and value heads up to 256.
//
// A decode step reads every visible key and value once, so the kernel is built around that stream, as the bfloat16 one is
// (attention_decode.cu): a block owns one sequence, up to HC query heads of one kv head and one share of the keys; its warps take tiles of
// 32 positions in turn, brought in by asynchronous copies a tile ahead (a warp's own two stages: no warp waits for another), each with its
// own running (max, sum, acc) per head.  The arithmetic is the FMA pipes':
//  * scores: eight lanes share a key (its 16-byte pieces), four keys at a time; the eight partial sums of HC heads are added up by
//    exchanging halves of the heads, so that each lane ends up with one head's score;
//  * weights: a lane takes four neighbouring positions (eight lanes a tile, four times over);
//  * values, stored [dim][position]: a lane multiplies four positions of a dimension with their weights for all HC heads; the eight
//    lanes' sums are added up once, at the end.
// Warps join through shared memory, the blocks that share a sequence's keys as a cluster.  Everything is float; exponentials are expf.
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

// D: heads of up to D numbers; HC: query heads of a block (1, 2 or 4); VEC: keys are read in pieces of 16 bytes (hd a multiple of 4).
template <int D, int HC, bool VEC>
__global__ void __launch_bounds__(128)
attention_stream_f32_kernel(float* __restrict__ out, const float* __restrict__ q, const float* __restrict__ k_pool,
                            const float* __restrict__ v_pool, const int* __restrict__ block_table, int bt_width,
                            const int* __restrict__ seq_slot, const int* __restrict__ seq_pos0, const int* __restrict__ seq_qstart,
                            const float* __restrict__ gate, int gate_stride, int gate_elem, int nh, int nkv, int hd, int vd, int page_size,
                            int window, int chunk, int first, float scale, const float* __restrict__ slopes,
                            const float* __restrict__ sinks, int n_splits) {
  constexpr int NK = D / 32, NV = D / 4;
  extern __shared__ __align__(128) float asf_smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int c = lane & 7, g = lane >> 3;
  const int G = nh / nkv, n_hc = (G + HC - 1) / HC;
  const int kvh = blockIdx.x / n_hc, hc = blockIdx.x % n_hc, b = blockIdx.y, split = blockIdx.z;
  const int h0 = kvh * G + hc * HC, heads = min(HC, G - hc * HC);
  pdl_wait();
  const int slot = seq_slot[b];
  const size_t m_row = seq_qstart[b];
  // (as in the bfloat16 kernel: out has one row per sequence of the launch; the same for all blocks of a cluster)
  if (m_row >= gridDim.y) return;
  if (slot < 0) {  // padding sequence
    for (int idx = split * blockDim.x + threadIdx.x; idx < heads * vd; idx += n_splits * blockDim.x)
      out[(m_row * nh + h0 + idx / vd) * vd + idx % vd] = 0.f;
    return;
  }
  const int qpos = seq_pos0[b], kv_len = qpos + 1;
  const int key_lo = first_key(qpos, window, chunk);
  const int n_first = first_tiles(first, key_lo, 32), shift = key_lo / 32 - n_first;
  const int n_tiles = (kv_len - 1) / 32 - shift + 1, per_split = (n_tiles + n_splits - 1) / n_splits;
  const int t_lo = split * per_split, t_hi = min(n_tiles, t_lo + per_split);
  const int* table = block_table + (size_t)b * bt_width;
  const int k_floats = 32 * hd, stage = k_floats + 32 * vd;      // of a tile: keys [32][hd], values [vd][32]
  float* ring = asf_smem + (size_t)warp * 2 * stage;
  float* score_s = asf_smem + (size_t)warps * 2 * stage + warp * HC * 32;      // [HC][32]

  auto key_of = [&](int tile) { return (tile >= n_first ? tile + shift : tile) * 32; };
  auto issue = [&](int tile, int s) {
    if (tile < t_hi) {
      const int key0 = key_of(tile), page = max(table[key0 / page_size], 0), off = key0 % page_size;
      const float* ks = k_pool + (((size_t)page * nkv + kvh) * page_size + off) * hd;      // the tile's keys lie together
      const float* vs = v_pool + ((size_t)page * nkv + kvh) * vd * page_size + off;
      const uint32_t to = (uint32_t)__cvta_generic_to_shared(ring + s * stage);
      for (int i = lane; i < 8 * hd; i += 32) asf_cp16(to + 16 * i, ks + 4 * i);
      for (int i = lane; i < 8 * vd; i += 32) asf_cp16(to + 4 * k_floats + 16 * i, vs + (size_t)(i >> 3) * page_size + 4 * (i & 7));
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  issue(t_lo + warp, 0);

  // the query's numbers that meet this lane's pieces of a key, already scaled
  float qv[HC][4 * NK];
#pragma unroll
  for (int h = 0; h < HC; h++)
#pragma unroll
    for (int i = 0; i < 4 * NK; i++) {
      const int d = VEC ? 4 * (c + 8 * (i >> 2)) + (i & 3) : c + 8 * i;
      qv[h][i] = h < heads && d < hd ? q[(m_row * nh + h0 + h) * hd + d] * scale : 0.f;
    }
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
  int s = 0;
  for (int tile = t_lo + warp; tile < t_hi; tile += warps, s ^= 1) {
    issue(tile + warps, s ^ 1);
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncwarp();      // every lane's pieces of this stage have landed
    const float* ks = ring + s * stage;
    const float* vs = ks + k_floats;
    const int key0 = key_of(tile);
#pragma unroll 2
    for (int t = 0; t < 8; t++) {      // key 4t + g
      const float* row = ks + (4 * t + g) * hd;
      float x[HC];
#pragma unroll
      for (int h = 0; h < HC; h++) x[h] = 0.f;
#pragma unroll
      for (int i = 0; i < NK; i++) {
        if (VEC) {
          if (4 * (c + 8 * i) < hd) {
            const float4 kk = load4(row + 4 * (c + 8 * i));
#pragma unroll
            for (int h = 0; h < HC; h++)
              x[h] += kk.x * qv[h][4 * i] + kk.y * qv[h][4 * i + 1] + kk.z * qv[h][4 * i + 2] + kk.w * qv[h][4 * i + 3];
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int d = c + 8 * (4 * i + e);
            if (d < hd) {
              const float kk = row[d];
#pragma unroll
              for (int h = 0; h < HC; h++) x[h] += kk * qv[h][4 * i + e];
            }
          }
        }
      }
      asf_sum8<HC>(x, lane);
      if (c < HC) score_s[asf_head<HC>(lane) * 32 + 4 * t + g] = x[0];
    }
    __syncwarp();
    const bool partial = (key0 < key_lo && key0 + 32 > first) || key0 + 32 > kv_len;
    float p[HC][4];
    bool read[4], moved = false;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int kp = key0 + 4 * c + e;
      read[e] = kp < kv_len && (kp >= key_lo || kp < first);
    }
    float corr[HC];
#pragma unroll
    for (int h = 0; h < HC; h++) {
      const float4 v4 = load4(score_s + h * 32 + 4 * c);
      p[h][0] = v4.x, p[h][1] = v4.y, p[h][2] = v4.z, p[h][3] = v4.w;
      float top = ASF_NEG;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        if (slopes) p[h][e] -= slope[h] * (float)(qpos - key0 - 4 * c - e);
        p[h][e] = read[e] ? p[h][e] : ASF_NEG;
        top = fmaxf(top, p[h][e]);
      }
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float mn = fmaxf(mx[h], top);
      corr[h] = expf(mx[h] - mn);
      moved |= mn != mx[h];
      mx[h] = mn;
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        p[h][e] = read[e] ? expf(p[h][e] - mn) : 0.f;
        sum += p[h][e];
      }
      l[h] = l[h] * corr[h] + sum;      // of this lane's positions
    }
    if (moved) {      // (the same for all lanes: maxima are)
#pragma unroll
      for (int i = 0; i < NV; i++)
#pragma unroll
        for (int h = 0; h < HC; h++) acc[i][h] *= corr[h];
    }
    if (partial) {
#pragma unroll
      for (int i = 0; i < NV; i++) {
        if (4 * i + g < vd) {
          float4 v4 = load4(vs + (4 * i + g) * 32 + 4 * c);      // zero times whatever lies where nothing is read would not be zero
          v4.x = read[0] ? v4.x : 0.f, v4.y = read[1] ? v4.y : 0.f, v4.z = read[2] ? v4.z : 0.f, v4.w = read[3] ? v4.w : 0.f;
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
    __syncwarp();      // everyone is done with the stage and the scores
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();     // the rings are done with: their memory takes the results
  float* o_s = asf_smem;                                // [warp][HC][vd]
  float* m_s = o_s + warps * HC * vd;                   // [warp][HC]
  float* l_s = m_s + warps * HC;
  float* mine = l_s + warps * HC;                       // this block's rows, for the cluster's blocks to read: [HC][vd], maxima, sums
  asf_sum8<HC>(l, lane);
  const int head = asf_head<HC>(lane);
#pragma unroll
  for (int i = 0; i < NV; i++) {
    asf_sum8<HC>(acc[i], lane);
    if (c < HC && 4 * i + g < vd) o_s[(warp * HC + head) * vd + 4 * i + g] = acc[i][0];
  }
  if (g == 0 && c < HC) {
    float top = mx[0];
#pragma unroll
    for (int h = 1; h < HC; h++) top = head == h ? mx[h] : top;
    m_s[warp * HC + head] = top;
    l_s[warp * HC + head] = l[0];
  }
  __syncthreads();
  auto finish = [&](int idx, float M, float L, float a) {
    const int h = h0 + idx / vd, d = idx % vd;
    const float inv = sinks ? sink_quotient(M, L, sinks[h]) : (L > 0.f ? 1.0f / L : 0.f);
    out[(m_row * nh + h) * vd + d] = a * inv * (gate ? head_gate(gate, m_row, gate_stride, h, d, vd, gate_elem) : 1.f);
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
LEB_API int leb_attention_stream_f32_supported(int nh, int nkv, int hd, int vd, int page_size) {
  return nkv > 0 && nh % nkv == 0 && hd >= 1 && hd <= 256 && vd >= 1 && vd <= 256 && page_size > 0 && page_size % 32 == 0;
}

// A decode step over a 32-bit cache: every sequence brings one row.  q [B][nh*hd], out [B][nh*vd], pools [page][nkv][page_size][hd] and
// [page][nkv][vd][page_size] on 16-byte boundaries.  max_kvlen: the most positions a sequence holds; blocks: of a cluster that shares a
// sequence's keys (0: as many as suit the step).
LEB_API int leb_attention_stream_f32(float* out, const float* q, const float* k_pool, const float* v_pool, const int* block_table, int bt_width,
                                     const int* seq_slot, const int* seq_pos0, const int* seq_qstart, const float* gate, int gate_stride,
                                     int gate_elem, int B, int nh, int nkv, int hd, int vd, int page_size, int window, int chunk, int first,
                                     float scale, const float* slopes, const float* sinks, int max_kvlen, int blocks, cudaStream_t st) {
  if (B <= 0) return 0;
  LEB_REQUIRE(leb_attention_stream_f32_supported(nh, nkv, hd, vd, page_size),
              "leb_attention_stream_f32: sizes not taken (heads %d, kv heads %d, widths %d and %d, page %d)", nh, nkv, hd, vd, page_size);
  LEB_REQUIRE((((uintptr_t)k_pool | (uintptr_t)v_pool) & 15) == 0, "leb_attention_stream_f32: pools must be 16-byte aligned");
  const int G = nh / nkv, widest = hd > vd ? hd : vd;
  const int HC = G == 1 ? 1 : widest > 128 ? 2 : 4, n_hc = ceil_div(G, HC);
  const size_t stage = (size_t)32 * (hd + vd) * sizeof(float);
  int warps = (int)(200 * 1024 / (2 * stage));
  warps = warps < 1 ? 1 : warps > 4 ? 4 : warps;
  const size_t rings = warps * (2 * stage + HC * 32 * sizeof(float)), results = ((size_t)(warps + 1) * HC * (vd + 2)) * sizeof(float);
  const size_t smem = rings > results ? rings : results;
  // blocks of a cluster: as many as run at once, with two tiles a warp or more for each
  long long keys = window > 0 ? window : max_kvlen;
  if (chunk > 0 && chunk < keys) keys = chunk;
  keys = keys + first < max_kvlen ? keys + first : max_kvlen;
  const long long per = (long long)B * nkv * n_hc, fit = 220 * 1024 / (long long)(smem + 2048);
  long long n = (long long)sm_count() * (fit < 1 ? 1 : fit > 4 ? 4 : fit) / per, most = keys / (64 * warps);
  n = n < most ? n : most;
  if (blocks > 0) n = blocks;
  const int n_splits = (int)(n < 1 ? 1 : n > 8 ? 8 : n);
  dim3 grid(nkv * n_hc, B, n_splits);
  LEB_REQUIRE(grid.y <= 65535, "leb_attention_stream_f32: grid too large");
#define LEB_ASF_K(D_, HC_, VEC_)                                                                                                      \
  {                                                                                                                                   \
    constexpr auto kern = attention_stream_f32_kernel<D_, HC_, VEC_>;                                                                 \
    const cudaError_t e = leb_allow_smem<kern>();                                                                                     \
    if (e != cudaSuccess) return leb_fail("leb_attention_stream_f32: shared memory %zu: %s", smem, cudaGetErrorString(e));            \
    leb_launch_cluster(n_splits, kern, grid, dim3(32 * warps), smem, st, out, q, k_pool, v_pool, block_table, bt_width, seq_slot, seq_pos0, \
                       seq_qstart, gate, gate_stride, gate_elem, nh, nkv, hd, vd, page_size, window, chunk, first, scale, slopes, sinks, n_splits); \
  }
#define LEB_ASF(D_, HC_)               \
  {                                    \
    if (hd % 4 == 0) LEB_ASF_K(D_, HC_, true) else LEB_ASF_K(D_, HC_, false) \
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
  LEB_CHECK_LAUNCH("leb_attention_stream_f32");
  return 0;
}
