// 8-bit matrix product on tcgen05 with the weights as the 128-row operand: C[m, n] (+)= (sum_k A[m, k] W[n, k]) sa[m] sw[n], dense or
// with rows grouped by expert.
//
// With few rows the product is bound by reading W, so a tile is 128 rows of W by MP rows of A (16 to 128) and the accumulator in
// tensor memory is the transposed tile.  Where there are fewer tiles than SMs a cluster of up to eight blocks shares a tile: each
// takes a part of K, sends its sums of every row to the block that finishes the row (st.async into its shared memory, counted there on a
// barrier), and finishes its share of the rows, adding up in the blocks' order.  (With the sums left where they were made, read by
// the finishing blocks between two cluster barriers, the way from the last tile of W to the results took 1.8 us, 0.9 without a cluster.)
// Otherwise the blocks walk the tiles, with two accumulators, so that loads go on under the epilogue.
//
// Roles: warp 0 asks for the tiles of W and A (TMA, 128 numbers of k a stage), warp 1 issues the products, warps 2-5 take the sums out of
// tensor memory, where a lane has a row of W, and apply the epilogue: a warp stores 32 neighbouring columns of a row of A.  (Turned in
// shared memory first, 16 rows at a time between two barriers, so that a lane has four columns, 128 rows x 16,384 x 2,048 took 17.0 us and not 12.8.)  The epilogue is
// looked at once for 32 rows: looked at for each, the unrolled code was more than the time.
//
// Every wait is bounded: a role that gives up sets the status word and all leave; the block stays until the copies asked for have
// landed and its products are done.
#include <type_traits>

#include "e4m3_tc.cuh"

#define FEW_THREADS 192
// Stages of W that a block asks L2 for ahead of its wait for the kernel before.  One row x 16,384 x 2,048: 8.9 us with none, 8.2 with 3,
// 8.5 with 5, 9.6 with all 16, which are in the way of what the kernel before still loads; x 4,096 x 4,096: 6.5, 6.4, 6.1, 6.2.
#define FEW_AHEAD 5

template <typename TC, int MP, int STAGES, int PER_SM, bool GROUPED, bool CLUSTER>
__global__ void __launch_bounds__(FEW_THREADS, PER_SM)
gemm_e4m3_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_a, TC* __restrict__ C,
                     const float* __restrict__ sa, const float* __restrict__ sw, int M, int N, int K, long long ldc, int epilogue, int n_slices,
                     const int* __restrict__ offsets, int n_groups, int* __restrict__ status) {
  constexpr int W_BYTES = 128 * E8_BK, A_BYTES = MP * E8_BK;
  constexpr uint32_t TMEM_COLS = 2 * MP < 32 ? 32 : 2 * MP;
  const int act = epilogue >> 8;
  epilogue &= 255;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t *s_w = smem, *s_a = smem + STAGES * W_BYTES, *s_part = s_a + STAGES * A_BYTES;      // part: the sums that a cluster's blocks have sent
  __shared__ uint64_t full[STAGES], empty[STAGES], acc_full[2], acc_empty[2], parts_full, drained;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_s, sent_s, parts_s;
  __shared__ float sa_s[2][MP];      // (rows beyond a tile's last: anything, not used)
  __shared__ E8Groups groups;
  volatile int* abort_flag = &abort_s;

  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int nk = (K + E8_BK - 1) / E8_BK, per = (nk + n_slices - 1) / n_slices;
  const int slice = CLUSTER ? (int)e8_cluster_rank() : 0;
  const int kb_lo = slice * per, my_nk = max(0, min(nk, kb_lo + per) - kb_lo);
  const int first = blockIdx.x / n_slices, step = gridDim.x / n_slices;
  const int m_tiles = (M + MP - 1) / MP, n_tiles = (N + 127) / 128;
  int num_tiles = m_tiles * n_tiles;

  if (threadIdx.x == 64) {
    tma_prefetch_map(&map_w);
    tma_prefetch_map(&map_a);
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; s++) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 4);
    }
    mbar_init(&parts_full, 1);
    mbar_init(&drained, 1);
    abort_s = sent_s = parts_s = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_acc = tmem_slot;
  if (CLUSTER) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");      // this block's barriers exist (waited for before sums are sent)
  pdl_trigger();      // (not before tensor memory is this block's: the next kernel's blocks may hold theirs while they wait for this one)
  if (!GROUPED && warp == 0 && first < num_tiles && elect_lane())      // the first tile's weights, on their way to L2 while the kernel before ends
    for (int i = 0; i < min(my_nk, FEW_AHEAD); i++) tma_prefetch_2d(&map_w, (kb_lo + i) * E8_BK, first / m_tiles * 128);
  __syncwarp();
  pdl_wait();
  if (GROUPED) {
    e8_count_groups(groups, offsets, n_groups, M, MP, n_tiles);
    num_tiles = groups.cum[n_groups];
  }
  if (CLUSTER) num_tiles = min(num_tiles, step);      // (a cluster has one tile at most, whatever the offsets hold)
  // first row of A and C, the row its rows end at, first column of C, the expert
  auto place = [&](int tile, int& m0, int& m_end, int& n0, int& e) {
    if (GROUPED) {
      e = e8_group_of(groups, n_groups, tile);
      const int local = tile - groups.cum[e], mt = (groups.end[e] - groups.off[e] + MP - 1) / MP;
      n0 = local / mt * 128;
      m0 = groups.off[e] + local % mt * MP;
      m_end = groups.end[e];
    } else {
      e = 0;
      n0 = tile / m_tiles * 128;
      m0 = tile % m_tiles * MP;
      m_end = M;
    }
  };
  // In a cluster: V of the rows that this block finishes from its row r on (`there` of them are there; c0: the first in C), this lane's column: the
  // sums of all `used` slices, scaled, through the epilogue.  All lanes of a warp call.
  const int share = CLUSTER ? MP / n_slices : 1, units = share / 4, used = (nk + per - 1) / per;
  // where four rows (unit u) of column n lie: columns side by side
  auto place_of = [&](int k, int n, int u) { return ((k * units + u) * 128 + n) * 4; };
  auto finish = [&](auto rows_at_a_time, int r, int there, int n_loc, int n, float swn, const float* sa_t, TC* c0) {
    constexpr int V = decltype(rows_at_a_time)::value;
    const float* part = reinterpret_cast<const float*>(s_part);
    float z[V], old[V];
    TC* const c = c0 + r * ldc;
#pragma unroll
    for (int i = 0; i < V; i++) z[i] = 0.f, old[i] = epilogue == 1 && n < N && r + i < there ? to_f32(c[i * ldc + n]) : 0.f;
#pragma unroll
    for (int k = 0; k < 8; k++)
      if (k < used) {
        if (V == 4) {
          const float4 f = *reinterpret_cast<const float4*>(part + place_of(k, n_loc, r >> 2));
          z[0] += f.x, z[1] += f.y, z[2 % V] += f.z, z[3 % V] += f.w;
        } else {
          const float2 f = *reinterpret_cast<const float2*>(part + (k * 128 + n_loc) * share);
          z[0] += f.x, z[1] += f.y;
        }
      }
#pragma unroll
    for (int i = 0; i < V; i++) z[i] = z[i] * sa_t[r + i] * swn + old[i];
    if (epilogue == 2) {      // lanes 0-15 hold 16 gate columns, lanes 16-31 their up columns
      float up[V];
#pragma unroll
      for (int i = 0; i < V; i++) up[i] = __shfl_down_sync(0xffffffffu, z[i], 16);
      gate_all<TC, V>(z, up, act);
      if (lane < 16 && n < N)
#pragma unroll
        for (int i = 0; i < V; i++)
          if (r + i < there) c[i * ldc + 16 * (n >> 5) + lane] = from_f32<TC>(z[i]);
    } else {
      if (sizeof(TC) == 2 && epilogue == 0 && LEB_PLAIN_ACT_OK(act, epilogue)) {
#pragma unroll
        for (int i = 0; i < V; i++) z[i] = plain_act(z[i], act);
      }
      if (n < N)
#pragma unroll
        for (int i = 0; i < V; i++)
          if (r + i < there) c[i * ldc + n] = from_f32<TC>(z[i]);
    }
  };

  bool gave_up = false, met = false;
  if (warp == 0) {
    uint32_t s = 0, ph = 1;
    int sent = 0;
    bool ok = true;
    for (int tile = first; tile < num_tiles && ok; tile += step) {
      int m0, m_end, n0, e;
      place(tile, m0, m_end, n0, e);
      for (int kb = 0; kb < my_nk; kb++) {
        if (!e8_wait(&empty[s], ph, abort_flag)) { ok = false; break; }
        if (elect_lane()) {
          mbar_expect_tx(&full[s], W_BYTES + A_BYTES);
          tma_load_2d(s_w + s * W_BYTES, &map_w, &full[s], (kb_lo + kb) * E8_BK, e * N + n0);
          tma_load_2d(s_a + s * A_BYTES, &map_a, &full[s], (kb_lo + kb) * E8_BK, m0);
        }
        __syncwarp();
        sent++;
        if (++s == STAGES) s = 0, ph ^= 1;
      }
    }
    if (lane == 0) {
      sent_s = sent;
      if (!ok) atomicExch(status, 51);
    }
  } else if (warp == 1) {
    const uint64_t w_desc = make_desc(smem_u32(s_w)), a_desc = make_desc(smem_u32(s_a));
    uint32_t s = 0, ph = 0, t = 0;
    int role = 0;
    for (int tile = first; tile < num_tiles && !role; tile += step, t++) {
      const uint32_t buf = t & 1;
      if (!e8_wait(&acc_empty[buf], ((t >> 1) & 1) ^ 1, abort_flag)) { role = 54; break; }
      tc_fence_after();
      const uint32_t d_tmem = tmem_acc + buf * MP;
      for (int kb = 0; kb < my_nk; kb++) {
        if (!e8_wait(&full[s], ph, abort_flag)) { role = 52; break; }
        tc_fence_after();
        if (elect_lane()) {
          const uint64_t dw = w_desc + (uint64_t)(s * (W_BYTES / 16)), da = a_desc + (uint64_t)(s * (A_BYTES / 16));
#pragma unroll
          for (int k = 0; k < E8_BK / 32; k++) umma_e4m3(d_tmem, dw + (uint64_t)(k * 2), da + (uint64_t)(k * 2), e8_idesc(128, MP), (kb | k) != 0);
          umma_commit(&empty[s]);
          if (kb + 1 == my_nk) umma_commit(&acc_full[buf]);
        }
        __syncwarp();
        if (++s == STAGES) s = 0, ph ^= 1;
      }
    }
    if (role && lane == 0) atomicExch(status, role);
  } else {
    const int quad = warp & 3, n_loc = quad * 32 + lane, tid = threadIdx.x - 64;
    float* const part = reinterpret_cast<float*>(s_part);
    uint32_t t = 0;
    for (int tile = first; tile < num_tiles; tile += step, t++) {
      int m0, m_end, n0, e;
      place(tile, m0, m_end, n0, e);
      const uint32_t buf = t & 1, tm = tmem_acc + ((uint32_t)(quad * 32) << 16) + buf * MP;
      const int rows = min(MP, m_end - m0);
      if (tid < rows) sa_s[buf][tid] = sa[m0 + tid];
      const int n = n0 + n_loc;
      const float swn = n < N ? sw[(size_t)e * N + n] : 0.f;
      // (the other buffer may still be read: a tile has one barrier, so nobody is two tiles ahead; the warps leave together)
      if (!e8_all<128>(!gave_up)) break;
      if (my_nk > 0) {
        const bool ok = e8_wait(&acc_full[buf], (t >> 1) & 1, abort_flag);
        if (!ok) {
          if (lane == 0) atomicExch(status, 53);
          gave_up = true;
        }
        tc_fence_after();
      }
      if (CLUSTER) {      // one tile
        // V rows of a column at a time (those behind the tile's last are sent with them, and not used)
        const int V = share >= 4 ? 4 : 2, shift = __ffs(share) - 1, own = min(share, rows - slice * share);
        if (tid == 0 && own > 0) {
          mbar_expect_tx(&parts_full, (uint32_t)(used * ((own + V - 1) / V * V) * 512));
          parts_s = 1;
        }
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");      // the others' barriers exist
        if (my_nk > 0)
#pragma unroll 1
          for (int c0 = 0; c0 < rows; c0 += 16) {
            uint32_t v[16];
            tmem_ld16(tm + (uint32_t)c0, v);      // (after a wait that gave up: anything; what the others wait for is sent all the same)
            tmem_ld_wait();
            if (V == 4) {
#pragma unroll
              for (int i = 0; i < 16; i += 4) {
                const uint32_t owner = (uint32_t)(c0 + i) >> shift;
                if (c0 + i < rows) e8_send4(e8_map_to_rank(smem_u32(part + place_of(slice, n_loc, ((c0 + i) & (share - 1)) >> 2)), owner), v + i, e8_map_to_rank(smem_u32(&parts_full), owner));
              }
            } else {
#pragma unroll
              for (int i = 0; i < 16; i += 2) {
                const uint32_t owner = (uint32_t)(c0 + i) >> 1;
                if (c0 + i < rows) e8_send2(e8_map_to_rank(smem_u32(part + (slice * 128 + n_loc) * 2), owner), v + i, e8_map_to_rank(smem_u32(&parts_full), owner));
              }
            }
          }
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");      // (waited for before the block leaves)
        met = true;
        if (own > 0) {
          if (!e8_wait(&parts_full, 0, abort_flag) && lane == 0) atomicExch(status, 55);
          const float* const sa_t = sa_s[buf] + slice * share;
          TC* const c0 = C + (m0 + slice * share) * ldc;
          if (V == 4) {
#pragma unroll 2
            for (int r = 0; r < own; r += 4) finish(std::integral_constant<int, 4>{}, r, own, n_loc, n, swn, sa_t, c0);
          } else {
            finish(std::integral_constant<int, 2>{}, 0, own, n_loc, n, swn, sa_t, c0);
          }
        }
        break;
      }
      if (gave_up) continue;
      constexpr int R = MP < 32 ? MP : 32;      // rows at a time
#pragma unroll 1
      for (int c0 = 0; c0 < rows; c0 += R) {
        uint32_t v[32];
        if (R == 32) tmem_ld32(tm + (uint32_t)c0, v);
        else tmem_ld16(tm + (uint32_t)c0, v);
        TC* const c = C + (m0 + c0) * ldc + n;
        float z[R];
        if (epilogue == 1) {
#pragma unroll
          for (int i = 0; i < R; i++) z[i] = n < N && c0 + i < rows ? to_f32(c[i * ldc]) : 0.f;
        }
        tmem_ld_wait();
        if (c0 + R >= rows) {      // all sums are out of tensor memory: the accumulator is free
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&acc_empty[buf]);
        }
        const float* f = sa_s[buf] + c0;
        if (epilogue == 1) {
#pragma unroll
          for (int i = 0; i < R; i++) z[i] += __uint_as_float(v[i]) * f[i] * swn;
        } else {
#pragma unroll
          for (int i = 0; i < R; i++) z[i] = __uint_as_float(v[i]) * f[i] * swn;
        }
        if (epilogue == 2) {      // lanes 0-15 hold 16 gate columns, lanes 16-31 their up columns
          TC* const o = C + (m0 + c0) * ldc + 16 * (n >> 5) + lane;
#pragma unroll
          for (int h = 0; h < R; h += 16) {
            float up[16];
#pragma unroll
            for (int i = 0; i < 16; i++) up[i] = __shfl_down_sync(0xffffffffu, z[h + i], 16);
            gate_all<TC, 16>(z + h, up, act);
          }
          if (lane < 16 && n < N)
#pragma unroll
            for (int i = 0; i < R; i++)
              if (c0 + i < rows) o[i * ldc] = from_f32<TC>(z[i]);
        } else {
          if (sizeof(TC) == 2 && epilogue == 0 && LEB_PLAIN_ACT_OK(act, epilogue)) {
#pragma unroll
            for (int i = 0; i < R; i++) z[i] = plain_act(z[i], act);
          }
          if (n < N)
#pragma unroll
            for (int i = 0; i < R; i++)
              if (c0 + i < rows) c[i * ldc] = from_f32<TC>(z[i]);
        }
      }
    }
  }

  if (CLUSTER) {      // nobody leaves before all sums have been sent
    __syncwarp();
    if (!met) {
      asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
      asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    }
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  if (abort_s) {      // a role gave up: the copies asked for land and the products end before the block does (else every one has been waited for)
    if (threadIdx.x == 0) {
      for (int i = max(sent_s - STAGES, 0); i < sent_s; i++) e8_passed(&full[i % STAGES], i / STAGES);
      if (parts_s) e8_passed(&parts_full, 0);
    } else if (warp == 1) {
      if (elect_lane()) {
        umma_commit(&drained);
        e8_passed(&drained, 0);
      }
      __syncwarp();
    }
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_acc, TMEM_COLS);
  }
}

namespace {

template <typename TC, int MP, int STAGES, int PER_SM, bool GROUPED, bool CLUSTER>
int launch_few(const E8Product& p, int n_slices, cudaStream_t st) {
  constexpr size_t smem = (size_t)STAGES * (128 + MP) * E8_BK + (CLUSTER ? MP * 512 : 0) + 1024;
  auto kern = gemm_e4m3_few_kernel<TC, MP, STAGES, PER_SM, GROUPED, CLUSTER>;
  cudaError_t e = leb_allow_smem<gemm_e4m3_few_kernel<TC, MP, STAGES, PER_SM, GROUPED, CLUSTER>, (int)smem>();
  if (e != cudaSuccess) return leb_fail("leb_linear_e4m3: shared memory %zu: %s", smem, cudaGetErrorString(e));
  CUtensorMap mw, ma;
  if (e8_tensor_map(&mw, p.W, (long long)p.N * (p.offsets ? p.n_groups : 1), p.K, p.ldw, 128)) return 1;
  if (e8_tensor_map(&ma, p.A, p.M, p.K, p.lda, MP)) return 1;
  // grouped: the most tiles the offsets can give (every expert with rows may end with a part tile)
  const long long m_tiles = p.M / MP + (GROUPED ? min(p.n_groups, p.M) : (p.M % MP != 0)), tiles = m_tiles * ceil_div(p.N, 128);
  long long clusters = tiles;
  if (n_slices == 1 && tiles > (long long)sm_count() * PER_SM) clusters = (long long)sm_count() * PER_SM;
  if (tiles >= 1LL << 30 || clusters * n_slices >= 1LL << 31) return leb_fail("leb_linear_e4m3: %lld tiles", tiles);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(clusters * n_slices));
  cfg.blockDim = dim3(FEW_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)n_slices;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = g_leb_pdl ? 2 : 1;
  e = cudaLaunchKernelEx(&cfg, kern, mw, ma, (TC*)p.C, p.sa, p.sw, p.M, p.N, p.K, p.ldc, p.epilogue, n_slices, p.offsets, p.n_groups, p.status);
  if (e != cudaSuccess) return leb_fail("leb_linear_e4m3: %s", cudaGetErrorString(e));
  LEB_CHECK_LAUNCH("leb_linear_e4m3");
  return 0;
}

template <typename TC, int MP, bool GROUPED, bool CLUSTER, bool FEW_TILES>
int launch_few_form(const E8Product& p, int n_slices, cudaStream_t st) {
  return launch_few<TC, MP, few_stages(MP, CLUSTER, FEW_TILES), few_alone(MP, CLUSTER, FEW_TILES) ? 1 : 2, GROUPED, CLUSTER>(p, n_slices, st);
}
template <typename TC, bool GROUPED>
int launch_few_rows(const E8Product& p, int mp, int n_slices, bool few_tiles, cudaStream_t st) {
  if (n_slices > 1) {
    if (mp == 16) return launch_few_form<TC, 16, GROUPED, true, false>(p, n_slices, st);
    if (mp == 32) return launch_few_form<TC, 32, GROUPED, true, false>(p, n_slices, st);
    return launch_few_form<TC, 64, GROUPED, true, false>(p, n_slices, st);
  }
  if (mp == 16) return launch_few_form<TC, 16, GROUPED, false, false>(p, 1, st);
  if (mp == 32) return launch_few_form<TC, 32, GROUPED, false, false>(p, 1, st);
  if (mp == 128) return launch_few_form<TC, 128, GROUPED, false, false>(p, 1, st);
  return few_tiles ? launch_few_form<TC, 64, GROUPED, false, true>(p, 1, st) : launch_few_form<TC, 64, GROUPED, false, false>(p, 1, st);
}

}  // namespace

// mp: 16, 32, 64 or 128 rows of A a tile; n_slices: 1, 2, 4 or 8 blocks that share a tile's K (1 with 128 rows).
int leb_gemm_e4m3_few(const E8Product& p, int mp, int n_slices, cudaStream_t st) {
  const int groups = p.offsets ? min(p.n_groups, p.M) : 1;
  const bool few_tiles = (long long)groups * ceil_div(ceil_div(p.M, groups), mp) * ceil_div(p.N, 128) <= sm_count();
  if (p.c_dtype == LEB_F32) return p.offsets ? launch_few_rows<float, true>(p, mp, n_slices, few_tiles, st) : launch_few_rows<float, false>(p, mp, n_slices, few_tiles, st);
  return p.offsets ? launch_few_rows<bf16, true>(p, mp, n_slices, few_tiles, st) : launch_few_rows<bf16, false>(p, mp, n_slices, few_tiles, st);
}
