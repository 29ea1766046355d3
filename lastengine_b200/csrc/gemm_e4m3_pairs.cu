// 8-bit matrix product for many rows on pairs of SMs (tcgen05 with cta_group::2): C[m, n] (+)= (sum_k A[m, k] W[n, k]) sa[m] sw[n], dense
// or with rows grouped by expert.
//
// A cluster of two blocks shares a tile of 256 rows of A by 256 rows of W: block r loads rows [128 r, 128 r + 128) of either, 32 KB a
// stage of 128 numbers of k, one elected lane of the first block issues the products, which read both blocks' shared memory, and each
// block holds its 128 rows of the sums in its tensor memory.  Two accumulators (all 512 columns): the epilogue of a tile runs under the
// products of the next.  A product of 8-bit numbers takes half the time of one of bfloat16 and leaves as many sums, so eight
// warps share the epilogue (four more than the bfloat16 product has): each takes 32 rows by 128 columns, scales them, and turns them in
// shared memory in lines of 64 bytes, so that a store covers whole sectors.
//
// Roles: warp 0 asks for tiles, warp 1 issues products, warps 2-9 are the epilogue.  Tiles are dealt in bands of PAIRS_BAND row
// tiles, down a band's rows first, so that the blocks that run together share few slabs of operands in L2.
// Every wait is bounded: a role that gives up sets the status word and all leave; both blocks stay until the copies that either asked for
// have landed and the products are done.
#include "e4m3_tc.cuh"

#define PAIRS_THREADS 320
#define PAIRS_STAGES 6
#define PAIRS_BAND 8

namespace {

// a TMA load whose bytes are counted on a barrier that may lie in the pair's other block
__device__ __forceinline__ void pair_load_2d(void* dst, const CUtensorMap* map, uint32_t bar_cluster_addr, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(smem_u32(dst)), "l"((uint64_t)map), "r"(bar_cluster_addr), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void pair_umma_e4m3(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// arrives on the barrier at this address in both blocks once the products issued so far are complete
__device__ __forceinline__ void pair_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
               ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar_cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar_cluster_addr) : "memory");
}
__device__ __forceinline__ int remote_int(uint32_t cluster_addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(cluster_addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}

template <typename TC, bool GROUPED>
__global__ void __launch_bounds__(PAIRS_THREADS, 1)
gemm_e4m3_pairs_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w,
                       const __grid_constant__ CUtensorMap map_c, int tma_c, TC* __restrict__ C,
                       const float* __restrict__ sa, const float* __restrict__ sw, int M, int N, int K, long long ldc, int epilogue,
                       const int* __restrict__ offsets, int n_groups, int* __restrict__ status) {
  constexpr int STAGES = PAIRS_STAGES, HALF = 128 * E8_BK;      // bytes of a block's half of a stage of either operand
  constexpr int PER = 16 / sizeof(TC);                          // results in 16 bytes
  const int act = epilogue >> 8;
  epilogue &= 255;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t *s_a = smem, *s_w = smem + STAGES * HALF, *s_lines = s_w + STAGES * HALF;      // lines: 2 KB a warp
  __shared__ uint64_t full[STAGES], empty[STAGES], acc_full[2], acc_empty[2], drained;   // full, acc_empty: used in the first block
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_s, sent_s;
  __shared__ __align__(16) float sw_s[2][256];
  __shared__ E8Groups groups;
  volatile int* abort_flag = &abort_s;

  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = e8_cluster_rank();      // 0: the block that issues the products
  const int pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;
  const int nk = (K + E8_BK - 1) / E8_BK;
  const int m_tiles = (M + 255) / 256, n_tiles = (N + 255) / 256;
  int num_tiles = m_tiles * n_tiles;

  if (threadIdx.x == 64) {
    tma_prefetch_map(&map_a);
    tma_prefetch_map(&map_w);
    if (tma_c) tma_prefetch_map(&map_c);
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; s++) {
      mbar_init(&full[s], 1);      // the first block announces the bytes of both
      mbar_init(&empty[s], 1);     // the commit to both
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 16);      // eight epilogue warps in each block
    }
    mbar_init(&drained, 1);
    abort_s = sent_s = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  e8_cluster_sync();      // both blocks' barriers exist before anything is sent to them
  tc_fence_after();
  const uint32_t tmem_acc = tmem_slot;
  pdl_trigger();      // (not before tensor memory is this block's)
  pdl_wait();
  if (GROUPED) {
    e8_count_groups(groups, offsets, n_groups, M, 256, n_tiles);
    num_tiles = groups.cum[n_groups];
  }
  // this block's first row of A and C, the row its rows end at, first column of C, the expert
  auto place = [&](int tile, int& m0, int& m_end, int& n0, int& e) {
    int mt, nt;
    if (GROUPED) {
      e = e8_group_of(groups, n_groups, tile);
      const int local = tile - groups.cum[e], rows = (groups.end[e] - groups.off[e] + 255) / 256;
      mt = local % rows;
      nt = local / rows;
      m0 = groups.off[e] + mt * 256 + 128 * (int)rank;
      m_end = groups.end[e];
    } else {
      const int band = tile / (PAIRS_BAND * n_tiles), r = tile - band * (PAIRS_BAND * n_tiles), rows = min(PAIRS_BAND, m_tiles - band * PAIRS_BAND);
      nt = r / rows;
      mt = band * PAIRS_BAND + r - nt * rows;
      e = 0;
      m0 = mt * 256 + 128 * (int)rank;
      m_end = M;
    }
    n0 = nt * 256;
  };

  // a role that gives up says so to both blocks, whose roles then leave at their next wait
  auto gives_up = [&](int code) {
    if (lane == 0) {
      atomicExch(status, code);
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(e8_map_to_rank(smem_u32(&abort_s), rank ^ 1)), "r"(1) : "memory");
    }
  };

  if (warp == 0) {
    const uint32_t full0 = e8_map_to_rank(smem_u32(&full[0]), 0);
    uint32_t s = 0, ph = 1;
    int sent = 0;
    bool ok = true;
    for (int tile = pair; tile < num_tiles && ok; tile += n_pairs) {
      int m0, m_end, n0, e;
      place(tile, m0, m_end, n0, e);
      const int w0 = e * N + n0 + 128 * (int)rank;
      int kk = n0 / 256 * 5 % nk;      // tiles that share rows of A start at different k
      for (int kb = 0; kb < nk; kb++) {
        if (!e8_wait(&empty[s], ph, abort_flag)) { ok = false; break; }
        if (elect_lane()) {
          if (rank == 0) mbar_expect_tx(&full[s], 4 * HALF);
          pair_load_2d(s_a + s * HALF, &map_a, full0 + s * 8, kk * E8_BK, m0);
          pair_load_2d(s_w + s * HALF, &map_w, full0 + s * 8, kk * E8_BK, w0);
        }
        __syncwarp();
        sent++;
        if (++kk == nk) kk = 0;
        if (++s == STAGES) s = 0, ph ^= 1;
      }
    }
    if (lane == 0) sent_s = sent;
    if (!ok) gives_up(61);
  } else if (warp == 1) {
    if (rank == 0) {
      const uint64_t a_desc = make_desc(smem_u32(s_a)), w_desc = make_desc(smem_u32(s_w));
      uint32_t s = 0, ph = 0, t = 0;
      int gave_up = 0;
      for (int tile = pair; tile < num_tiles && !gave_up; tile += n_pairs, t++) {
        const uint32_t buf = t & 1;
        if (!e8_wait(&acc_empty[buf], ((t >> 1) & 1) ^ 1, abort_flag)) { gave_up = 64; break; }
        tc_fence_after();
        const uint32_t d_tmem = tmem_acc + buf * 256;
        for (int kb = 0; kb < nk; kb++) {
          if (!e8_wait(&full[s], ph, abort_flag)) { gave_up = 62; break; }
          tc_fence_after();
          if (elect_lane()) {
            const uint64_t da = a_desc + (uint64_t)(s * (HALF / 16)), dw = w_desc + (uint64_t)(s * (HALF / 16));
#pragma unroll
            for (int k = 0; k < E8_BK / 32; k++) pair_umma_e4m3(d_tmem, da + (uint64_t)(k * 2), dw + (uint64_t)(k * 2), e8_idesc(256, 256), (kb | k) != 0);
            pair_commit(&empty[s]);
            if (kb + 1 == nk) pair_commit(&acc_full[buf]);
          }
          __syncwarp();
          if (++s == STAGES) s = 0, ph ^= 1;
        }
      }
      if (gave_up) gives_up(gave_up);
    }
  } else {
    const int quad = warp & 3, half = (warp - 2) >> 2;      // rows 32 quad, columns 128 half
    uint8_t* lines = s_lines + (warp - 2) * 2048;
    const uint32_t acc_empty0 = e8_map_to_rank(smem_u32(&acc_empty[0]), 0);
    const int n_out = epilogue == 2 ? N / 2 : N;
    const bool vec = ldc % PER == 0 && ((uintptr_t)C & 15) == 0;
    const int r4 = lane >> 2, u4 = lane & 3;      // in a line's stores: rows r4 + 8 j, 16 bytes u4
    uint32_t t = 0;
    bool gave_up = false, pending = false;
    const bool adds = sizeof(TC) == 4 && epilogue == 1;
    for (int tile = pair; tile < num_tiles; tile += n_pairs, t++) {
      int m0, m_end, n0, e;
      place(tile, m0, m_end, n0, e);
      const uint32_t buf = t & 1;
      const int row0 = m0 + quad * 32, c_base = half * 128;
      {
        const int i = threadIdx.x - 64;
        sw_s[buf][i] = n0 + i < N ? sw[(size_t)e * N + n0 + i] : 0.f;
      }
      const float sam = row0 + lane < m_end ? sa[row0 + lane] : 0.f;
      // (the other buffer may still be read: a tile has one barrier, so nobody is two tiles ahead; the warps leave together)
      if (!e8_all<256>(!gave_up)) break;
      const bool ok = e8_wait(&acc_full[buf], (t >> 1) & 1, abort_flag);
      if (!ok) {
        gives_up(63);
        gave_up = true;
        continue;
      }
      tc_fence_after();
      // Four times 16 bytes of this lane's row (columns from `col` on) go out by lines of 64 bytes.  Whole groups of 32 rows are stored, or
      // added, by a TMA copy (what lies beyond C is left out), an expert's last ones and results that TMA does not take by the lanes.
      const bool copies = tma_c && row0 < m_end && (!GROUPED || row0 + 32 <= m_end);
      auto put = [&](const uint4* u, int col) {
        if (pending) {      // the line before has left shared memory
          if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
          __syncwarp();
        }
#pragma unroll
        for (int i = 0; i < 4; i++) *reinterpret_cast<uint4*>(lines + lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4)) = u[i];
        if (copies) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (copies) {
          if (lane == 0) {
            if (adds)
              asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3}], [%1];"
                           ::"l"((uint64_t)&map_c), "r"(smem_u32(lines)), "r"(col), "r"(row0) : "memory");
            else
              asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];"
                           ::"l"((uint64_t)&map_c), "r"(smem_u32(lines)), "r"(col), "r"(row0) : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
          pending = true;
          return;
        }
        pending = false;
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int r = r4 + 8 * j, row = row0 + r, c = col + u4 * PER;
          const uint4 x = *reinterpret_cast<const uint4*>(lines + r * 64 + ((u4 ^ ((r >> 1) & 3)) << 4));
          if (row < m_end && c < n_out) {
            TC* o = C + row * ldc + c;
            if (vec && !adds && c + PER <= n_out) *reinterpret_cast<uint4*>(o) = x;
            else {
              const TC* f = reinterpret_cast<const TC*>(&x);
#pragma unroll
              for (int i = 0; i < PER; i++)
                if (c + i < n_out) o[i] = adds ? from_f32<TC>(to_f32(f[i]) + to_f32(o[i])) : f[i];
            }
          }
        }
        __syncwarp();
      };
      uint4 kept[2];      // of a gated bfloat16 result: the first half of a line
      const uint32_t tm = tmem_acc + ((uint32_t)(quad * 32) << 16) + buf * 256 + (uint32_t)c_base;
      const int c_end = min(128, N - n0 - c_base);      // (may be negative: nothing of this half)
      uint32_t vs[5][32];      // unrolled, so that no copy of a piece's registers is made while its load is on its way
      tmem_ld32(tm, vs[0]);
#pragma unroll
      for (int c = 0; c < 128; c += 32) {
        uint32_t* const v = vs[c / 32];
        tmem_ld_wait();
        float z[32];
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          const float4 f = *reinterpret_cast<const float4*>(&sw_s[buf][c_base + c + i]);
          z[i] = __uint_as_float(v[i]) * sam * f.x;
          z[i + 1] = __uint_as_float(v[i + 1]) * sam * f.y;
          z[i + 2] = __uint_as_float(v[i + 2]) * sam * f.z;
          z[i + 3] = __uint_as_float(v[i + 3]) * sam * f.w;
        }
        if (c + 32 < 128) tmem_ld32(tm + (uint32_t)(c + 32), vs[c / 32 + 1]);      // on its way while these are finished
        if (c >= c_end) continue;
        const int col = n0 + c_base + c;
        if (epilogue == 2) {
          gate_all<TC, 16>(z, z + 16, act);
        } else if (sizeof(TC) == 2 && LEB_PLAIN_ACT_OK(act, epilogue)) {
#pragma unroll
          for (int i = 0; i < 32; i++) z[i] = plain_act(z[i], act);
        }
        uint4 u[4];
        if (sizeof(TC) == 4) {
#pragma unroll
          for (int l = 0; l < 2; l++) {
            if (l == 1 && (epilogue == 2 || col + 16 >= N)) break;
#pragma unroll
            for (int i = 0; i < 4; i++)
              u[i] = make_uint4(__float_as_uint(z[16 * l + 4 * i]), __float_as_uint(z[16 * l + 4 * i + 1]), __float_as_uint(z[16 * l + 4 * i + 2]), __float_as_uint(z[16 * l + 4 * i + 3]));
            put(u, epilogue == 2 ? col / 2 : col + 16 * l);
          }
        } else if (epilogue == 2) {
          uint4 h[2];
#pragma unroll
          for (int i = 0; i < 2; i++)
            h[i] = make_uint4(pack2(z[8 * i], z[8 * i + 1]), pack2(z[8 * i + 2], z[8 * i + 3]), pack2(z[8 * i + 4], z[8 * i + 5]), pack2(z[8 * i + 6], z[8 * i + 7]));
          if (c & 32) {
            u[0] = kept[0], u[1] = kept[1], u[2] = h[0], u[3] = h[1];
            put(u, (col - 32) / 2);
          } else if (col + 32 >= N) {      // nothing follows
            u[0] = h[0], u[1] = h[1], u[2] = u[3] = make_uint4(0, 0, 0, 0);
            put(u, col / 2);
          } else {
            kept[0] = h[0], kept[1] = h[1];
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; i++)
            u[i] = make_uint4(pack2(z[8 * i], z[8 * i + 1]), pack2(z[8 * i + 2], z[8 * i + 3]), pack2(z[8 * i + 4], z[8 * i + 5]), pack2(z[8 * i + 6], z[8 * i + 7]));
          put(u, col);
        }
      }
      // this warp has read its sums: tell the block that issues the products
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_cluster(acc_empty0 + buf * 8);
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  e8_cluster_sync();      // both blocks are through: nobody frees tensor memory or leaves while the other may still use it
  const bool left = abort_s | remote_int(e8_map_to_rank(smem_u32(&abort_s), rank ^ 1));
  if (left) {      // the copies asked for land and the products end first (else every one has been waited for)
    if (rank == 0 && threadIdx.x == 0) {
      const int theirs = remote_int(e8_map_to_rank(smem_u32(&sent_s), 1));
      const int begin = e8_first_out(sent_s, theirs, STAGES), end = max(sent_s, theirs);
      for (int i = begin; i < end; i++) {
        const int owed = e8_owed(i, sent_s, theirs, 2 * HALF);
        if (owed > 0) mbar_expect_tx(&full[i % STAGES], (uint32_t)owed);
        if (owed < 0) mbar_complete_tx(&full[i % STAGES], (uint32_t)-owed);
      }
      for (int i = begin; i < end; i++) e8_passed(&full[i % STAGES], i / STAGES);
    } else if (warp == 1) {
      if (elect_lane()) {
        if (rank == 0) pair_commit(&drained);
        e8_passed(&drained, 0);
      }
      __syncwarp();
    }
    __syncthreads();
  }
  e8_cluster_sync();      // (what was read of the other's memory has been, and in a pair that gave up the copies into either's have landed)
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_acc), "r"(512u));
  }
}

template <typename TC, bool GROUPED>
int launch_pairs(const E8Product& p, cudaStream_t st) {
  constexpr size_t smem = (size_t)PAIRS_STAGES * 2 * 128 * E8_BK + 8 * 2048 + 1024;
  auto kern = gemm_e4m3_pairs_kernel<TC, GROUPED>;
  cudaError_t e = leb_allow_smem<gemm_e4m3_pairs_kernel<TC, GROUPED>, (int)smem>();
  if (e != cudaSuccess) return leb_fail("leb_linear_e4m3: shared memory %zu: %s", smem, cudaGetErrorString(e));
  CUtensorMap ma, mw;
  if (e8_tensor_map(&ma, p.A, p.M, p.K, p.lda, 128)) return 1;
  if (e8_tensor_map(&mw, p.W, (long long)p.N * (p.offsets ? p.n_groups : 1), p.K, p.ldw, 128)) return 1;
  // results as the copies of the epilogue see them: 32 rows by 64 bytes, turned as the lanes leave them.  (A copy leaves out what lies beyond C in
  // steps of 16 bytes: rows that end inside such a step are the lanes' to store.)
  const int n_out = (p.epilogue & 255) == 2 ? p.N / 2 : p.N, size = sizeof(TC);
  const int tma_c = (long long)n_out * size % 16 == 0 && p.ldc * size % 16 == 0 && ((uintptr_t)p.C & 15) == 0 && p.ldc >= n_out;
  CUtensorMap mc = ma;
  if (tma_c) {
    cuuint64_t dims[2] = {(cuuint64_t)n_out, (cuuint64_t)p.M}, strides[1] = {(cuuint64_t)p.ldc * size};
    cuuint32_t box[2] = {(cuuint32_t)(64 / size), 32}, estr[2] = {1, 1};
    CUresult r = encode_fn()(&mc, size == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, p.C, dims, strides, box, estr,
                             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return leb_fail("leb_linear_e4m3: cuTensorMapEncodeTiled failed (%d) for the results [%d,%d] rows %lld apart", (int)r, p.M, n_out, p.ldc);
  }
  const long long m_tiles = p.M / 256 + (GROUPED ? min(p.n_groups, p.M) : (p.M % 256 != 0)), tiles = m_tiles * ceil_div(p.N, 256);
  if (tiles >= 1LL << 30) return leb_fail("leb_linear_e4m3: %lld tiles", tiles);
  const long long pairs = tiles < sm_count() / 2 ? tiles : sm_count() / 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * pairs));
  cfg.blockDim = dim3(PAIRS_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = g_leb_pdl ? 2 : 1;
  e = cudaLaunchKernelEx(&cfg, kern, ma, mw, mc, tma_c, (TC*)p.C, p.sa, p.sw, p.M, p.N, p.K, p.ldc, p.epilogue, p.offsets, p.n_groups, p.status);
  if (e != cudaSuccess) return leb_fail("leb_linear_e4m3: %s", cudaGetErrorString(e));
  LEB_CHECK_LAUNCH("leb_linear_e4m3");
  return 0;
}

}  // namespace

int leb_gemm_e4m3_pairs(const E8Product& p, cudaStream_t st) {
  if (p.c_dtype == LEB_F32) return p.offsets ? launch_pairs<float, true>(p, st) : launch_pairs<float, false>(p, st);
  return p.offsets ? launch_pairs<bf16, true>(p, st) : launch_pairs<bf16, false>(p, st);
}
