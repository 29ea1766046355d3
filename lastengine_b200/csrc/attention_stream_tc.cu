// Prompt attention of streams on the fifth-generation tensor cores: a window and a sequence's first positions, key and value heads of up
// to 128 numbers (multiples of 8; tiles of 64 or 128, filled up with zeros by the copies), pages of 64 positions or a multiple.
//
// A row at position p reads positions j <= p with j >= first_key(p) or j < first.  A block owns a tile of 128 rows: the G query heads
// of one kv head times TP = 128 / G consecutive positions (a multiple of 8; the rows that are left are idle).  It walks a list of
// pages (of larger pages: their parts of 64 positions), those of first positions and then those from its first row's window to its last
// row, two pages (128 keys) at a time:
//
//   S[128, 128] = Q[128, HD] . K[128, HD]^T       operands in shared memory, S in tensor memory
//   P           = exp2(S * scale * log2 e - m)     two threads per row, one a page, P (bfloat16) to tensor memory
//   O[128, HD] += P[128, 128] . V[128, HD]         P from tensor memory, V from shared memory
//
// Warps: eight for the softmax, one that brings Q and pages by TMA, one that issues the products, two that put zeros where a page holds
// values no row of the tile reads (registers move between warpgroups).  Two blocks share an SM, so that one's products run under the other's exponentials, and a
// scheduler has four softmax warps: what bounds the loop is the chain from a row's scores to its weights, not a pipe.
// P is rounded to bfloat16 (l is the sum of the floats): results are 1.26 to 1.28 times as far from 64 bits as results rounded once.  Callers that want
// more ask for weights of two terms or 32 bits (`wide`), and get another kernel.
// Where there are few tiles, a cluster of n_splits blocks shares the pages of one and joins its sums through shared memory.
// With heads of 64, P has columns beside S and the next scores are issued as soon as a row of S is in registers; with heads of 128, O
// takes those columns, P lies over S and the next scores follow the product that reads P.
//
// Bounds: 128 keys of a tile are 1,024 cycles of the SM's special function unit (16 exponentials a cycle) and 512 (heads of 64) or 1,024
// of its tensor cores, 512 or 1,280 of shared memory's 128 bytes a cycle; a tile alone takes some 2,400, two blocks on an SM 1,250 each.
// 8,191 rows, window 4,096, 128 first positions, 32 heads over 8: heads of 64 300 us (701 TFLOP/s; the form with pages of 64 keys and
// three blocks an SM, attention_prefill_tc.cu, 390), heads of 128 403 us (1,045); turns of 3 to 1,500 rows of 12 streams, window 1,024, 53 us
// (83), of 100 to 2,047 rows, 16 heads of 128 over 4, window 2,048, 45 us (mma.sync 190).  A block's fixed part is some 6,000 cycles; zeros
// by the softmax warps, rows stored by their own threads and blocks without a tile cost another 8,000 on the turns (69 and 66 us).
// Measured beside it: one thread a row 311 to 317, two tiles a block (one block an SM) 329, 64 keys at a time with two buffers of S 323 (heads
// of 128: 442), an eighth to a half of the exponentials as polynomials on the multiply-add pipes 304 to 365 (heads of 128: 428 to 515).
//
// Every wait on an mbarrier is bounded; a wait that gives up sets the status word, all roles leave their loops, and the block returns once its copies
// have landed, its products are done and tensor memory is freed.
#include "attention_tc.cuh"

#define AST_NEG (-1e30f)
#define AST_MOST_SPLITS 8      // blocks that share a tile's keys: a portable cluster
#define AST_LISTED 128         // sequences whose tiles a grid may list

template <int HD>
struct AstShape {
  static constexpr int THREADS = 384;
  // registers a thread: at the launch, then of the softmax warps and of the other four (as many in all)
  static constexpr int REGS = 80, REGS_SOFTMAX = 96, REGS_OTHER = 48;
  static_assert(2 * REGS_SOFTMAX + REGS_OTHER <= 3 * REGS, "more registers than the block is launched with");
  static constexpr int STAGES = HD == 64 ? 2 : 1;                     // iterations' keys and values on their way
  static constexpr int Q_BYTES = 128 * HD * 2;
  static constexpr int KV_BYTES = 128 * HD * 2;                       // of an iteration's keys (or values)
  static constexpr int SMEM = 1024 + Q_BYTES + STAGES * 2 * KV_BYTES;
  static constexpr bool OWN_P = HD == 64;                             // P beside S (else over it)
  static constexpr int COLUMNS = 256;                                 // S, P and O
};

// All threads of the cluster's blocks; what they wrote to their shared memory is visible to the others.
__device__ __forceinline__ void ast_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// The number at this address of block `rank`'s shared memory.
__device__ __forceinline__ uint32_t ast_map(const void* p, int rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ float ast_remote(const float* p, int rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(ast_map(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ float4 ast_remote4(const float* p, int rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(ast_map(p, rank)) : "memory");
  return v;
}

// The lowest n bits (none for n <= 0, all from 32 on).
__device__ __forceinline__ uint32_t ast_below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }

// SHARED: a cluster of n_splits blocks shares a tile's keys (else n_splits is 1).  EXACT: heads of HD numbers and pages of 64 positions (the
// same with these as arguments takes some 5 us longer on the turns of 12 streams).
template <int HD, bool SHARED, bool EXACT>
__global__ void __launch_bounds__(AstShape<HD>::THREADS, 2)
attention_stream_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                           const __grid_constant__ CUtensorMap map_v, bf16* __restrict__ out, const int* __restrict__ block_table,
                           int bt_width, const int* __restrict__ seq_slot, const int* __restrict__ seq_pos0,
                           const int* __restrict__ seq_qstart, const int* __restrict__ seq_qlen, const bf16* __restrict__ gate,
                           int gate_stride, int gate_elem, int nh, int nkv, int n_seqs, int G, int TP, int hd_, int vd_, int per_page_, int window, int chunk, int first,
                           float scale, const float* __restrict__ slopes, const float* __restrict__ sinks, int n_blocks, int* __restrict__ status) {
  const int n_splits = SHARED ? n_blocks : 1, hd = EXACT ? HD : hd_, vd = EXACT ? HD : vd_, per_page = EXACT ? 1 : per_page_;
  using Shape = AstShape<HD>;
  constexpr int PAGE = 64, NS = Shape::STAGES, HALVES = HD / 64;
  constexpr int Q_BYTES = Shape::Q_BYTES, KV_BYTES = Shape::KV_BYTES;
  constexpr bool OWN_P = Shape::OWN_P;
  constexpr uint32_t COL_S = 0, COL_P = OWN_P ? 128 : 0, COL_O = OWN_P ? 192 : 128;
  extern __shared__ uint8_t ast_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)ast_raw + 1023) & ~(uintptr_t)1023);   // swizzled tiles want 1024
  uint8_t* sq = smem;                         // [64 dimensions][128 rows][128 bytes]
  uint8_t* sk = sq + Q_BYTES;                 // [stage][64 dimensions][128 keys][128 bytes]
  uint8_t* sv = sk + NS * KV_BYTES;           // [stage][page][dimension][64 positions]
  __shared__ uint64_t q_full, k_full[NS], v_full[NS], k_empty[NS], v_empty[NS], s_full, s_free, p_full, pv_done, zeroed[NS], drained;
  __shared__ float row_s[2][2][128];          // what the two threads of a row tell each other: [iteration's parity][thread][row]
  __shared__ float last_s[2][128], join_s[SHARED ? AST_MOST_SPLITS : 1][SHARED ? 64 : 128];      // maxima and sums of this block's rows; factors of the rows it stores
  __shared__ int place_s[SHARED ? 64 : 128];      // and where those lie in out, from the tile's first row and head on (-1: nowhere)
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_s, sent_s[2];      // sent_s: iterations whose keys and values were asked for
  volatile int* abort_flag = &abort_s;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // kv heads vary fastest; of a sequence's tiles the ones with the longest key range come first
  const int kvh = blockIdx.x, split = blockIdx.z % n_splits;
  int b = blockIdx.y, tile = (int)(gridDim.z / n_splits - 1 - blockIdx.z / n_splits), qlen;
  if (n_seqs > 0) {      // the tiles of up to AST_LISTED sequences one after the other: which is this one (every warp looks for itself)
    const int t = blockIdx.z / n_splits;
    int q[AST_LISTED / 32], n[AST_LISTED / 32], sum = 0;
#pragma unroll
    for (int e = 0; e < AST_LISTED / 32; e++) {
      const int j = lane * (AST_LISTED / 32) + e;
      q[e] = j < n_seqs ? seq_qlen[j] : 0;
      n[e] = (q[e] + TP - 1) / TP;
      sum += n[e];
    }
    int end = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, end, o);
      if (lane >= o) end += up;
    }
    const unsigned past = __ballot_sync(0xffffffffu, end > t);
    const int owner = past ? __ffs(past) - 1 : 31;
    int at = end - sum, found = 0;
    tile = qlen = 0;
#pragma unroll
    for (int e = 0; e < AST_LISTED / 32; e++) {
      if (t >= at && t < at + n[e]) found = lane * (AST_LISTED / 32) + e, tile = at + n[e] - 1 - t, qlen = q[e];
      at += n[e];
    }
    b = __shfl_sync(0xffffffffu, found, owner);
    tile = __shfl_sync(0xffffffffu, tile, owner);
    qlen = __shfl_sync(0xffffffffu, past ? qlen : 0, owner);      // (behind the last tile: nothing to do)
  } else {
    qlen = seq_qlen[b];      // step data: written long before the kernel before this one
  }
  const int row0 = tile * TP;
  if (row0 >= qlen) {
    pdl_wait();   // a kernel counts as complete when its blocks are: none may finish before its predecessor has
    return;
  }
  const int rows = min(TP, qlen - row0);
  const int pos0 = seq_pos0[b];
  const size_t m_base = (size_t)seq_qstart[b] + row0;
  const int h0 = kvh * G;
  const bool live = seq_slot[b] >= 0;
  const int q_lo = pos0 + row0, key_hi = q_lo + rows;      // keys [.., key_hi) exist for the tile
  const int key_lo = first_key(q_lo, window, chunk);
  const int nf = first_tiles(first, key_lo, PAGE), jb0 = key_lo / PAGE;
  const int n_pages = nf + (key_hi - 1) / PAGE - jb0 + 1, n_all = (n_pages + 1) / 2;
  if (!live) {   // a padding sequence: its rows are zero
    pdl_wait();
    for (int idx = split * blockDim.x + threadIdx.x; idx < rows * G * (vd / 8); idx += n_splits * blockDim.x) {
      const int i = idx / (G * (vd / 8)), rest = idx % (G * (vd / 8));
      reinterpret_cast<uint4*>(out + ((m_base + i) * nh + h0) * vd)[rest] = make_uint4(0, 0, 0, 0);
    }
    return;
  }
  // this block's share of the iterations (none for the last ones where they do not go round)
  const int per_split = (n_all + n_splits - 1) / n_splits, it0 = split * per_split, n_it = max(0, min(n_all - it0, per_split));
  const int* table = block_table + (size_t)b * bt_width;

  // where 64 positions lie: their head's page (-1: there are none; a page given back, of which every key is masked: 0) and which 64
  struct At { int page, part; };
  auto at_of = [&](int v) {
    v += 2 * it0;
    if (v >= n_pages) return At{-1, 0};
    const int j = v < nf ? v : jb0 + v - nf;
    return per_page == 1 ? At{max(table[j], 0) * nkv + kvh, 0} : At{max(table[j / per_page], 0) * nkv + kvh, j % per_page};
  };
  At p0{-1, 0}, p1{-1, 0};
  if (threadIdx.x == 32 * 8) {      // the TMA producer: asked for before the wait for the kernel before, as the step's other tables are
    p0 = at_of(0), p1 = at_of(1);
    asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&map_q) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&map_k) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&map_v) : "memory");
  }
  // Whether iteration i brings value columns that no row of the tile reads (between the first positions and the tile's window, or beyond
  // the last row): they become zero before the product reads them, whatever they hold.
  auto key_of = [&](int v) { return (v < nf ? v : jb0 + v - nf) * PAGE; };
  auto unread = [&](int v) {
    const int key0 = key_of(v);
    return v < n_pages && ((key_lo > key0 && first - key0 < min(key_lo - key0, PAGE)) || key_hi < key0 + PAGE);
  };
  if (threadIdx.x == 0) {
    abort_s = 0;
    sent_s[0] = sent_s[1] = n_it;
    mbar_init(&q_full, 1);
    for (int s = 0; s < NS; s++) {
      mbar_init(&k_full[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_empty[s], 1);
      mbar_init(&zeroed[s], 2);
    }
    mbar_init(&s_full, 1);
    mbar_init(&s_free, 8);
    mbar_init(&p_full, 8);
    mbar_init(&pv_done, 1);
    mbar_init(&drained, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) {
    tmem_alloc(&tmem_slot, Shape::COLUMNS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();      // barriers and tensor memory are set up; now q and the cache must be complete
  const uint32_t tmem = tmem_slot;
  // instruction descriptors: float accumulate, bfloat16 operands, both K-major, M = 128; N = 128 keys, N = HD
  constexpr uint32_t IDESC = (1u << 4) | (1u << 7) | (1u << 10) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
  constexpr uint32_t IDESC_PV = (1u << 4) | (1u << 7) | (1u << 10) | (((uint32_t)HD >> 3) << 17) | ((128u >> 4) << 24);
  bool ok = true;
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Shape::REGS_OTHER));
    if (warp == 8) {
      // ---- TMA producer ----
      if (lane == 0) {
        if (n_it > 0) mbar_expect_tx(&q_full, G * HALVES * TP * 128);
        for (int g = 0; g < G && n_it > 0; g++)
          for (int h = 0; h < HALVES; h++)
            if (hd == HD) tma_load_2d(sq + h * (128 * 128) + g * (TP * 128), &map_q, &q_full, (h0 + g) * HD + h * 64, (int)m_base);
            else tma_load_3d(sq + h * (128 * 128) + g * (TP * 128), &map_q, &q_full, h * 64, h0 + g, (int)m_base);
        for (int i = 0; i < n_it; i++) {
          const int s = i % NS;
          const At a = p0, c = p1;
          p0 = at_of(2 * i + 2), p1 = at_of(2 * i + 3);      // asked for before the waits below
          const uint32_t bytes = c.page >= 0 ? KV_BYTES : KV_BYTES / 2;
          if (!mbar_wait(&k_empty[s], ((i / NS) & 1) ^ 1, abort_flag)) { atomicExch(status, 31); sent_s[0] = sent_s[1] = i; break; }
          mbar_expect_tx(&k_full[s], bytes);
          for (int h = 0; h < HALVES; h++) {
            tma_load_2d(sk + s * KV_BYTES + h * (128 * 128), &map_k, &k_full[s], h * 64, (a.page * per_page + a.part) * PAGE);
            if (c.page >= 0) tma_load_2d(sk + s * KV_BYTES + h * (128 * 128) + 64 * 128, &map_k, &k_full[s], h * 64, (c.page * per_page + c.part) * PAGE);
          }
          if (!mbar_wait(&v_empty[s], ((i / NS) & 1) ^ 1, abort_flag)) { atomicExch(status, 32); sent_s[0] = i + 1; sent_s[1] = i; break; }
          mbar_expect_tx(&v_full[s], bytes);
          if (vd == HD) {
            tma_load_2d(sv + s * KV_BYTES, &map_v, &v_full[s], a.part * PAGE, a.page * HD);
            if (c.page >= 0) tma_load_2d(sv + s * KV_BYTES + HD * 128, &map_v, &v_full[s], c.part * PAGE, c.page * HD);
          } else {      // (a head's dimensions end inside the box: zeros behind them)
            tma_load_3d(sv + s * KV_BYTES, &map_v, &v_full[s], a.part * PAGE, 0, a.page);
            if (c.page >= 0) tma_load_3d(sv + s * KV_BYTES + HD * 128, &map_v, &v_full[s], c.part * PAGE, 0, c.page);
          }
        }
      }
    } else if (warp == 9) {
      // ---- MMA issuer: the whole warp walks the loop, one lane issues ----
      const int n = __shfl_sync(0xffffffffu, n_it, 0), odd = __shfl_sync(0xffffffffu, it0 + n_it == n_all ? n_pages & 1 : 0, 0);      // the sequence's last page may be alone
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
      const uint64_t q_desc = make_desc(smem_u32(sq)), k_desc = make_desc(smem_u32(sk)), v_desc = make_desc(smem_u32(sv));
      auto arrived = [&](uint64_t* bar, uint32_t parity, int code) -> bool {
        const bool in = mbar_wait_warp(bar, parity, abort_flag);
        if (!in && lane == 0) atomicExch(status, code);
        return in;
      };
      auto scores = [&](int i) -> bool {
        const int s = i % NS;
        if (!arrived(&k_full[s], (i / NS) & 1, 33)) return false;
        tc_fence_after();
        if (elect_lane()) {
#pragma unroll
          for (int kk = 0; kk < HD / 16; kk++)
            umma_bf16(tm + COL_S, q_desc + (kk >> 2) * 1024 + (kk & 3) * 2, k_desc + s * (KV_BYTES / 16) + (kk >> 2) * 1024 + (kk & 3) * 2, IDESC, kk > 0);
          umma_commit(&k_empty[s]);
          umma_commit(&s_full);
        }
        __syncwarp();
        return true;
      };
      ok = n > 0 && arrived(&q_full, 0, 34) && scores(0);
      for (int i = 0; i < n && ok; i++) {
        const int s = i % NS, steps = i == n - 1 && odd ? 4 : 8;
        // P beside S: the next scores wait until every softmax warp holds its rows of these
        if (OWN_P && i + 1 < n && !(arrived(&s_free, i & 1, 35) && scores(i + 1))) break;
        if (!arrived(&v_full[s], (i / NS) & 1, 36)) break;
        if (!arrived(&zeroed[s], (i / NS) & 1, 42) || !arrived(&p_full, i & 1, 37)) break;
        tc_fence_after();
        if (elect_lane()) {
          for (int kk = 0; kk < steps; kk++)
            umma_bf16_ts(tm + COL_O, tm + COL_P + kk * 8, v_desc + s * (KV_BYTES / 16) + (kk >> 2) * (HD * 128 / 16) + (kk & 3) * 2, IDESC_PV, (i > 0 || kk > 0));
          umma_commit(&v_empty[s]);
          umma_commit(&pv_done);
        }
        __syncwarp();
        // P over S: the tensor pipe runs the product that reads it before the one that overwrites it
        if (!OWN_P && i + 1 < n && !scores(i + 1)) break;
      }
    } else {
      // ---- the other two warps: unread value columns, a page each ----
      const int p = warp - 10;
      for (int i = 0; i < n_it; i++) {
        const int s = i % NS, v = 2 * (it0 + i) + p;
        // (every iteration, so that no phase of a stage's barriers passes these warps by: the product waits for them)
        if (!mbar_wait_warp(&v_full[s], (i / NS) & 1, abort_flag)) { atomicExch(status, 39); break; }
        if (unread(v)) {
          const int key0 = key_of(v);
          for (int r = lane; r < HD; r += 32) {
            uint8_t* vrow = sv + s * KV_BYTES + p * (HD * 128) + r * 128;   // dimension r: 64 positions, 16-byte pieces swizzled by r & 7
#pragma unroll 2
            for (int e = 0; e < 8; e++) {
              const int at = key0 + 8 * e;
              const uint32_t keep = (ast_below(first - at) | ~ast_below(key_lo - at)) & ast_below(key_hi - at) & 255u;
              if (keep == 255u) continue;
              uint4* piece = reinterpret_cast<uint4*>(vrow + ((e ^ (r & 7)) << 4));
              uint4 x = make_uint4(0, 0, 0, 0);
              if (keep) {
                auto pair = [&](uint32_t w, int j) { return w & ((keep >> j & 1 ? 0xffffu : 0u) | (keep >> (j + 1) & 1 ? 0xffff0000u : 0u)); };
                x = *piece;
                x = make_uint4(pair(x.x, 0), pair(x.y, 2), pair(x.z, 4), pair(x.w, 6));
              }
              *piece = x;
            }
          }
          fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&zeroed[s]);
      }
    }
    if (SHARED) {
      ast_cluster_sync();
      ast_cluster_sync();
    }
  } else {
    // ---- softmax: two threads own row r = (head r / TP, position r % TP), `half` 0 the first page of an iteration, 1 the second ----
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Shape::REGS_SOFTMAX));
    const int half = warp >> 2, r = threadIdx.x & 127, g = r / TP, pi = r % TP;
    const int qpos = q_lo + pi;
    const int key_lo_row = first_key(qpos, window, chunk);
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + COL_S + half * 64 + lane_base, t_p = tmem + COL_P + half * 32 + lane_base;
    const uint32_t t_o = tmem + COL_O + half * (HD / 2) + lane_base;      // the half of a row of O that this thread rescales and stores
    const float scale2 = scale * 1.4426950408889634f;
    // With slopes the scores are finished (scaled, less slope (qpos - key), times log2 e) as they come out of tensor memory,
    // and what follows multiplies them by one.
    const float slope2 = slopes && g < G ? slopes[h0 + g] * 1.4426950408889634f : 0.f;
    const float scale_after = slopes ? 1.f : scale2;
    float m_used = AST_NEG, l = 0.f;
    // The two warps of 32 rows meet once an iteration.  One that leaves the loop early has to let the other go.
    auto meet = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp & 3)) : "memory"); };
    // Pages that every row of the tile reads whole need no look at single keys: those that end at or before the tile's first
    // row and begin at or behind the last row's window, or hold first positions only.  (Idle rows read what comes: they are never written.)
    const int lo_last = first_key(key_hi - 1, window, chunk);
    for (int i = 0; i < n_it; i++) {
      const int vp = 2 * (it0 + i) + half, key0 = key_of(vp);
      const bool there = vp < n_pages;
      const bool whole = there && key0 + PAGE - 1 <= q_lo && (key0 >= lo_last || key0 + PAGE <= first);
      if (!mbar_wait_warp(&s_full, i & 1, abort_flag)) { atomicExch(status, 38); ok = false; break; }
      tc_fence_after();
      uint32_t v[PAGE];
      tmem_ld32(t_s, v);
      tmem_ld32(t_s + 32, v + 32);
      tmem_ld_wait();
      if (OWN_P) {      // the next scores may come
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_free);
      }
      if (slopes) {
        const float at0 = slope2 * (float)(key0 - qpos);
#pragma unroll
        for (int c = 0; c < PAGE; c++) v[c] = __float_as_uint(fmaf(__uint_as_float(v[c]), scale2, fmaf(slope2, (float)c, at0)));
      }
      if (!whole) {
        // columns [0, c_first) and [c_lo, c_end) of this page are keys this row reads
        const int c_lo = key_lo_row - key0, c_first = first - key0, c_end = there ? qpos - key0 + 1 : 0;
#pragma unroll
        for (int h = 0; h < PAGE; h += 32) {
          const uint32_t seen = (ast_below(c_first - h) | ~ast_below(c_lo - h)) & ast_below(c_end - h);
#pragma unroll
          for (int c = 0; c < 32; c++)
            if (!(seen & (1u << c))) v[h + c] = __float_as_uint(AST_NEG);
        }
      }
      float rm[2] = {AST_NEG, AST_NEG};
#pragma unroll
      for (int c = 0; c < PAGE; c += 4)
#pragma unroll
        for (int e = 0; e < 2; e++) rm[e] = max3(rm[e], __uint_as_float(v[c + 2 * e]), __uint_as_float(v[c + 2 * e + 1]));
      const float mine = fmaxf(rm[0], rm[1]);
      row_s[i & 1][half][r] = mine;
      meet();      // (with P over S: from here on both have their scores in registers)
      const float top = fmaxf(mine, row_s[i & 1][half ^ 1][r]);
      // maxima are kept times scale * log2(e); a row with no key in these pages keeps what it had
      const float m_new = top > 0.5f * AST_NEG ? fmaxf(m_used, top * scale_after) : m_used;
      bool move = false;
      if (m_used < 0.5f * AST_NEG) m_used = m_new;  // nothing accumulated for this row yet: O's row is zero
      else if (m_new > m_used + 8.f) move = true;   // the reference maximum has to follow
      // P beside S: the last one has to have been read, and O to hold the pages before these; P over S: that product came before these scores
      if (OWN_P && i > 0 && !mbar_wait_warp(&pv_done, (i - 1) & 1, abort_flag)) { atomicExch(status, 40); ok = false; break; }
      if (__any_sync(0xffffffffu, move)) {
        tc_fence_after();
        const float f = move ? ex2(m_used - m_new) : 1.f;
#pragma unroll 1
        for (int hcol = 0; hcol < HD / 2; hcol += 16) {
          uint32_t o[16];
          tmem_ld16(t_o + hcol, o);
          tmem_ld_wait();
#pragma unroll
          for (int c = 0; c < 16; c++) o[c] = __float_as_uint(__uint_as_float(o[c]) * f);
          tmem_st16(t_o + hcol, o);
        }
        l *= f;
        if (move) m_used = m_new;
      }
      const float m_ref = m_used > 0.5f * AST_NEG ? m_used : 0.f;
      const uint64_t scale_pair = f2(scale_after, scale_after), ref_pair = f2(-m_ref, -m_ref);
      uint64_t ps[2] = {f2(0.f, 0.f), f2(0.f, 0.f)};
#pragma unroll
      for (int c0 = 0; c0 < PAGE; c0 += 32) {
        uint32_t pk[16];
#pragma unroll
        for (int c = 0; c < 32; c += 2) {
          // a masked score is -1e30: 2^(that * scale - m_ref) is exactly zero
          const float2 x = halves(fma_f2(f2(__uint_as_float(v[c0 + c]), __uint_as_float(v[c0 + c + 1])), scale_pair, ref_pair));
          const float p0 = ex2(x.x), p1 = ex2(x.y);
          ps[(c >> 1) & 1] = add_f2(ps[(c >> 1) & 1], f2(p0, p1));
          __nv_bfloat162 pp = __floats2bfloat162_rn(p0, p1);
          pk[c >> 1] = *reinterpret_cast<uint32_t*>(&pp);
        }
        tmem_st16(t_p + c0 / 2, pk);
      }
      tmem_st_wait();
      const float2 sums = halves(add_f2(ps[0], ps[1]));
      l += sums.x + sums.y;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full);   // one arrival per softmax warp
    }
    if (ok && n_it > 0 && !mbar_wait_warp(&pv_done, (n_it - 1) & 1, abort_flag)) { atomicExch(status, 41); ok = false; }
    if (!ok) {
      asm volatile("bar.arrive %0, 64;" ::"r"(1 + (warp & 3)) : "memory");
    } else {
      row_s[n_it & 1][half][r] = l;
      meet();
      l += row_s[n_it & 1][half ^ 1][r];
    }
    tc_fence_after();
    if (!SHARED && vd == HD && !(gate && gate_elem)) {
      // Finished rows go to shared memory as bfloat16 (keys are done with) and out from there, whole rows at a time: stored by their own
      // threads every store would touch 32 lines.
      const bool row_valid = ok && g < G && pi < rows;
      float inv = l > 0.f ? 1.0f / l : 0.f;
      if (sinks && row_valid) inv = sink_quotient(m_used * 0.6931471805599453f, l, sinks[h0 + g]);
      if (gate && row_valid) inv *= head_gate(gate, m_base + pi, gate_stride, h0 + g, 0, HD, 0);
      if (half == 0) place_s[r] = row_valid ? pi * nh + g : -1;
      if (ok) {
#pragma unroll
        for (int d0 = 0; d0 < HD / 2; d0 += 32) {
          uint32_t o[32];
          tmem_ld32(t_o + d0, o);
          tmem_ld_wait();
#pragma unroll
          for (int c = 0; c < 32; c += 8) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
              __nv_bfloat162 pp = __floats2bfloat162_rn(__uint_as_float(o[c + 2 * e]) * inv, __uint_as_float(o[c + 2 * e + 1]) * inv);
              w[e] = *reinterpret_cast<uint32_t*>(&pp);
            }
            const int piece = (half * (HD / 2) + d0 + c) / 8;
            *reinterpret_cast<uint4*>(sk + r * (HD * 2) + ((piece ^ (r & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
      asm volatile("bar.sync 9, 256;" ::: "memory");
#pragma unroll
      for (int n = 0; n < 128 * (HD / 8) / 256; n++) {
        const int row = (n * 256 + (int)threadIdx.x) / (HD / 8), piece = threadIdx.x % (HD / 8), place = place_s[row];
        if (place >= 0)
          reinterpret_cast<uint4*>(out + (m_base * nh + h0 + place) * HD)[piece] = *reinterpret_cast<const uint4*>(sk + row * (HD * 2) + ((piece ^ (row & 7)) << 4));
      }
    } else {
      // Rows of O, their maxima and sums go to shared memory (keys and values are done with), from where they are stored row by row.  The
      // blocks that share a tile each join 128 / n_splits of its rows, reading from all of them, in the blocks' order.
      float* so = reinterpret_cast<float*>(sk);      // [row][16-byte pieces moved by row & 7]
      const bool any = ok && n_it > 0;
      if (half == 0) {
        last_s[0][r] = any ? m_used : AST_NEG;
        last_s[1][r] = any ? l : 0.f;
      }
      if (any) {
  #pragma unroll
        for (int d0 = 0; d0 < HD / 2; d0 += 32) {
          uint32_t o[32];
          tmem_ld32(t_o + d0, o);
          tmem_ld_wait();
  #pragma unroll
          for (int c = 0; c < 32; c += 4) {
            const int piece = (half * (HD / 2) + d0 + c) / 4;
            *reinterpret_cast<uint4*>(so + r * HD + ((piece ^ (r & 7)) << 2)) = make_uint4(o[c], o[c + 1], o[c + 2], o[c + 3]);
          }
        }
      }
      if (SHARED) ast_cluster_sync();
      else asm volatile("bar.sync 9, 256;" ::: "memory");
      auto from = [&](const float* p, int rank) { return SHARED ? ast_remote(p, rank) : *p; };
      const int share = (128 + n_splits - 1) / n_splits, r0 = split * share, n_rows = min(share, 128 - r0);
      for (int i = threadIdx.x; i < n_rows; i += 256) {      // a row's factors, one per block
        const int row = r0 + i, gg = row / TP, ii = row % TP;
        float top = AST_NEG, sum = 0.f;
        for (int j = 0; j < n_splits; j++) top = fmaxf(top, from(&last_s[0][row], j));
        for (int j = 0; j < n_splits; j++) sum += from(&last_s[1][row], j) * ex2(from(&last_s[0][row], j) - top);
        float inv = sum > 0.f ? 1.0f / sum : 0.f;
        if (gg < G && ii < rows) {
          if (sinks) inv = sink_quotient(top * 0.6931471805599453f, sum, sinks[h0 + gg]);
          if (gate && !gate_elem) inv *= head_gate(gate, m_base + ii, gate_stride, h0 + gg, 0, vd, 0);
        }
        for (int j = 0; j < n_splits; j++)
          join_s[j][i] = from(&last_s[1][row], j) > 0.f ? inv * ex2(from(&last_s[0][row], j) - top) : 0.f;
        place_s[i] = gg < G && ii < rows ? ii * nh + gg : -1;
      }
      asm volatile("bar.sync 9, 256;" ::: "memory");
      for (int idx = threadIdx.x; idx < n_rows * (HD / 4); idx += 256) {
        const int i = idx / (HD / 4), piece = idx % (HD / 4), row = r0 + i, place = place_s[i];
        if (place < 0 || 4 * piece >= vd) continue;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int j = 0; j < n_splits; j++) {
          const float f = join_s[j][i];
          if (f == 0.f) continue;      // (that block read nothing for this row: its numbers may be anything)
          const float* at = so + row * HD + ((piece ^ (row & 7)) << 2);
          const float4 y = SHARED ? ast_remote4(at, j) : load4(at);
          x.x += f * y.x, x.y += f * y.y, x.z += f * y.z, x.w += f * y.w;
        }
        if (gate && gate_elem) {
          const size_t m = m_base + row % TP;
          const int h = h0 + row / TP;
          x.x *= head_gate(gate, m, gate_stride, h, 4 * piece, vd, 1), x.y *= head_gate(gate, m, gate_stride, h, 4 * piece + 1, vd, 1);
          x.z *= head_gate(gate, m, gate_stride, h, 4 * piece + 2, vd, 1), x.w *= head_gate(gate, m, gate_stride, h, 4 * piece + 3, vd, 1);
        }
        store4(out + (m_base * nh + h0 + place) * vd + 4 * piece, x);
      }
    }
    if (SHARED) ast_cluster_sync();      // no block ends while others read its memory
  }
  tc_fence_before();
  __syncthreads();
  if (abort_s) {      // a role gave up: the block stays until its copies have landed and its products are done (else every one has been waited for)
    auto passed = [](uint64_t* bar, int phase) {
      for (int n = 0; n < 1 << 16 && !mbar_try_wait(bar, phase & 1); n++) {}
    };
    if (threadIdx.x == 32 * 8) {
      if (n_it > 0) passed(&q_full, 0);
      for (int i = max(sent_s[0] - NS, 0); i < sent_s[0]; i++) passed(&k_full[i % NS], i / NS);
      for (int i = max(sent_s[1] - NS, 0); i < sent_s[1]; i++) passed(&v_full[i % NS], i / NS);
    } else if (warp == 9) {
      if (elect_lane()) {
        umma_commit(&drained);
        passed(&drained, 0);
      }
      __syncwarp();
    }
    __syncthreads();
  }
  __syncwarp();
  if (warp == 8) tmem_dealloc(tmem, Shape::COLUMNS);
}

// Positions of a tile: as many as fit 128 rows with all heads of a kv head, in eights (a head's rows start on a group of eight
// rows of the swizzled tile).
static int ast_positions(int G) { return (128 / G) & ~7; }

// Blocks that share a tile's keys: as many as there is room for on the SMs (two each), with two iterations of 128 keys or more for each.
static int ast_splits(int M, int B, int nh, int nkv, int window, int chunk, int first, int max_qlen, int max_kvlen) {
  const int TP = ast_positions(nh / nkv);
  const long long per_head = (long long)ceil_div(max_qlen, TP) * B, by_rows = (long long)M / TP + B;
  const long long tiles = (per_head < by_rows ? per_head : by_rows) * nkv, room = 2ll * sm_count() / tiles;
  long long keys = (long long)(window > 0 ? window : max_kvlen);
  if (chunk > 0 && chunk < keys) keys = chunk;
  keys += first + (TP < max_qlen ? TP : max_qlen);
  if (keys > max_kvlen) keys = max_kvlen;
  const long long most = (keys + 127) / 128 / 2;
  long long n = room < most ? room : most;
  return (int)(n < 1 ? 1 : n > AST_MOST_SPLITS ? AST_MOST_SPLITS : n);
}

// Returns 1 when the sizes are ones this kernel takes.
LEB_API int leb_attention_stream_tc_supported(int nh, int nkv, int hd, int vd, int page_size) {
  return hd > 0 && vd > 0 && hd % 8 == 0 && vd % 8 == 0 && hd <= 128 && vd <= 128 && page_size > 0 && page_size % 64 == 0 && nkv > 0 &&
         nh % nkv == 0 && nh / nkv <= 16;
}

template <int HD, bool SHARED, bool EXACT>
static int launch_attention_stream_tc(void* out, const void* q, int q_stride, int M, const void* k_pool, const void* v_pool, int n_pages,
                                      const int* block_table, int bt_width, const int* seq_slot, const int* seq_pos0,
                                      const int* seq_qstart, const int* seq_qlen, const void* gate, int gate_stride, int gate_elem,
                                      int B, int nh, int nkv, int hd, int vd, int page_size, int window, int chunk, int first, float scale, const float* slopes,
                                      const float* sinks, int max_qlen, int n_splits, int* status, cudaStream_t st) {
  using Shape = AstShape<HD>;
  const int G = nh / nkv, TP = ast_positions(G);
  CUtensorMap mq, mk, mv;
  if (hd == HD ? tensor_map(&mq, q, M, nh * HD, q_stride, TP) : tensor_map3(&mq, "leb_attention_stream_tc", q, hd, nh, M, hd, q_stride, 1, TP)) return 1;
  if (tensor_map(&mk, k_pool, n_pages * nkv * page_size, hd, hd, 64)) return 1;
  if (vd == HD) {
    // the same through a map of two dimensions
    if (tensor_map(&mv, v_pool, n_pages * nkv * HD, page_size, page_size, HD)) return 1;
  } else if (tensor_map3(&mv, "leb_attention_stream_tc", v_pool, page_size, vd, n_pages * nkv, page_size, (long long)vd * page_size, HD, 1)) return 1;
  // Sequences of very different lengths: a list of tiles, so that none of the blocks of a full grid has to come and go for nothing (952 tiles of
  // 12 sequences, 4,512 blocks otherwise).
  dim3 grid(nkv, B, ceil_div(max_qlen, TP) * n_splits);
  const bool listed = B > 1 && B <= AST_LISTED && M / TP + B < ceil_div(max_qlen, TP) * B;
  if (listed) grid = dim3(nkv, 1, (M / TP + B) * n_splits);
  LEB_REQUIRE(grid.y <= 65535 && grid.z <= 65535, "leb_attention_stream_tc: grid too large (%u, %u)", grid.y, grid.z);
  constexpr auto kern = attention_stream_tc_kernel<HD, SHARED, EXACT>;
  // The warpgroups share out the registers of the launch: with fewer than REGS a thread they would wait for ever.
  static std::atomic<int> regs{0};
  if (regs.load(std::memory_order_relaxed) == 0) {
    cudaFuncAttributes a;
    if (cudaFuncGetAttributes(&a, kern) != cudaSuccess) return leb_fail("leb_attention_stream_tc: no attributes of the kernel");
    regs.store(a.numRegs, std::memory_order_relaxed);
  }
  LEB_REQUIRE(regs.load(std::memory_order_relaxed) >= Shape::REGS, "leb_attention_stream_tc: built with %d registers a thread, %d are shared out",
              regs.load(std::memory_order_relaxed), Shape::REGS);
  const cudaError_t e = leb_allow_smem<kern, Shape::SMEM>();
  if (e != cudaSuccess) return leb_fail("leb_attention_stream_tc: shared memory %d: %s", Shape::SMEM, cudaGetErrorString(e));
  leb_launch_cluster(SHARED ? n_splits : 1, kern, grid, dim3(Shape::THREADS), Shape::SMEM, st, mq, mk, mv, (bf16*)out, block_table, bt_width,
                     seq_slot, seq_pos0, seq_qstart, seq_qlen, (const bf16*)gate, gate_stride, gate_elem, nh, nkv, listed ? B : 0, G, TP, hd, vd, page_size / 64, window, chunk, first,
                     scale, slopes, sinks, n_splits, status);
  LEB_CHECK_LAUNCH("leb_attention_stream_tc");
  return 0;
}

// Prompt attention of the step's rows over the paged cache (which already holds their keys and values).  q: [M, nh*hd] with row
// stride q_stride; k_pool [n_pages][nkv][page_size][hd], v_pool [n_pages][nkv][vd][page_size]; out [M, nh*vd].  status: device int, set non-zero by a
// block whose bounded wait gave up.  slopes, sinks [nh] or null as in leb_attention.  scale: 1e-20 or more (masked
// scores are -1e30 before they are scaled).  max_kvlen: the most positions a sequence of the step holds.
// n_splits: blocks that share a tile's keys (0: as many as suit the step).
LEB_API int leb_attention_stream_tc(void* out, const void* q, int q_stride, int M, const void* k_pool, const void* v_pool, int n_pages,
                                    const int* block_table, int bt_width, const int* seq_slot, const int* seq_pos0,
                                    const int* seq_qstart, const int* seq_qlen, const void* gate, int gate_stride, int gate_elem, int B,
                                    int nh, int nkv, int hd, int vd, int page_size, int window, int chunk, int first, float scale,
                                    const float* slopes, const float* sinks, int max_qlen, int max_kvlen, int n_splits,
                                    int* status, cudaStream_t st) {
  if (B <= 0 || max_qlen <= 0 || M <= 0) return 0;
  LEB_REQUIRE(leb_attention_stream_tc_supported(nh, nkv, hd, vd, page_size),
              "leb_attention_stream_tc: sizes not taken (heads %d, kv heads %d, widths %d and %d, page %d)", nh, nkv, hd, vd, page_size);
  LEB_REQUIRE(status != nullptr, "leb_attention_stream_tc: a status word is required");
  LEB_REQUIRE((((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_pool | (uintptr_t)v_pool) & 15) == 0 && q_stride % 8 == 0,
              "leb_attention_stream_tc: q, out and the pools must be 16-byte aligned, q's row stride a multiple of 8");
  LEB_REQUIRE((long long)n_pages * nkv * (page_size > vd ? page_size : vd) < 1ll << 31, "leb_attention_stream_tc: pools of %d pages of %d positions and %d kv heads",
              n_pages, page_size, nkv);
  LEB_REQUIRE(n_splits >= 0 && n_splits <= AST_MOST_SPLITS, "leb_attention_stream_tc: %d blocks for a tile's keys, %d at most", n_splits, AST_MOST_SPLITS);
  if (n_splits == 0) n_splits = ast_splits(M, B, nh, nkv, window, chunk, first, max_qlen, max_kvlen);
#define LEB_AST_ARGS out, q, q_stride, M, k_pool, v_pool, n_pages, block_table, bt_width, seq_slot, seq_pos0, seq_qstart, seq_qlen, gate, \
                     gate_stride, gate_elem, B, nh, nkv, hd, vd, page_size, window, chunk, first, scale, slopes, sinks, max_qlen, n_splits, status, st
  const bool exact = page_size == 64 && hd == vd && (hd == 64 || hd == 128), narrow = hd <= 64 && vd <= 64;
#define LEB_AST(HD_, SHARED_) \
  (exact ? launch_attention_stream_tc<HD_, SHARED_, true>(LEB_AST_ARGS) : launch_attention_stream_tc<HD_, SHARED_, false>(LEB_AST_ARGS))
  if (n_splits > 1) return narrow ? LEB_AST(64, true) : LEB_AST(128, true);
  return narrow ? LEB_AST(64, false) : LEB_AST(128, false);
#undef LEB_AST
#undef LEB_AST_ARGS
}
