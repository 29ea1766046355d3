// What the tcgen05 kernels of 8-bit numbers share beside tc_common.cuh: the products themselves, tensor maps of byte matrices, and the
// walk over tiles of rows grouped by expert.  A block of 128 numbers of k is a row of 128 bytes, as 64 of bfloat16 are, so tiles,
// swizzle and descriptors are the same; an instruction multiplies 32 of them.
#pragma once
#include "e4m3_common.cuh"
#include "tc_common.cuh"

#define E8_BK 128            // numbers of k in a stage
#define E8_MAX_GROUPS 256

// float accumulator, e4m3 A and B, both K-major
__host__ __device__ constexpr uint32_t e8_idesc(int rows, int cols) { return (1u << 4) | ((uint32_t)(cols >> 3) << 17) | ((uint32_t)(rows >> 4) << 24); }

__device__ __forceinline__ void umma_e4m3(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// A tile's way to L2 only.  What L2 holds is current whoever writes it, so weights may be asked for so ahead of the wait for the
// kernel before, even where that kernel makes them.
__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap* map, int x, int y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"((uint64_t)map), "r"(x), "r"(y) : "memory");
}
// A tensor map's own way to the SM, ahead of the first copy that goes by it.
__device__ __forceinline__ void tma_prefetch_map(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)map) : "memory"); }
__device__ __forceinline__ uint32_t e8_cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t e8_map_to_rank(uint32_t smem_addr, uint32_t rank) {   // the same place in another block of the cluster
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_addr), "r"(rank));
  return a;
}
// Values' way to another block's shared memory, their bytes counted on a barrier there.
__device__ __forceinline__ void e8_send4(uint32_t cluster_addr, const uint32_t* v, uint32_t bar_cluster_addr) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];"
               ::"r"(cluster_addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(bar_cluster_addr) : "memory");
}
__device__ __forceinline__ void e8_send2(uint32_t cluster_addr, const uint32_t* v, uint32_t bar_cluster_addr) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.b32 [%0], {%1, %2}, [%3];"
               ::"r"(cluster_addr), "r"(v[0]), "r"(v[1]), "r"(bar_cluster_addr) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr));
}
__device__ __forceinline__ void e8_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
#ifndef E8_PATIENT      // (the tests build kernels whose waits give up now and then, also before their first try)
#define E8_PATIENT 1
#endif
// mbar_wait_warp: a bounded wait of all lanes of a warp together
__device__ __forceinline__ bool e8_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  if (E8_PATIENT) return mbar_wait_warp(bar, parity, abort_flag);
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag)) != 0;
}
// Whether all of the THREADS that share barrier 1 say so: they meet, and go on or leave together.
template <int THREADS>
__device__ __forceinline__ bool e8_all(bool ok) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.and.pred q, 1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"(ok ? 1u : 0u), "n"(THREADS)
      : "memory");
  return all != 0;
}
// A block that gave up stays until copies that it asked for have landed: a phase's end, or some milliseconds (copies land within microseconds).
__device__ __forceinline__ void e8_passed(uint64_t* bar, int phase) {
  for (int n = 0; n < 1 << 14; n++) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(phase & 1)
        : "memory");
    if (ok) return;
    __nanosleep(64);
  }
}
// A pair that gives up stops its two producers anywhere: the first block has announced the bytes of both on its barriers, and asked for its own half, in
// `own` stages, the other block has asked for its half in `theirs`, and either may be ahead by as many stages as there were free ones.  A
// phase ends once its bytes have been announced and have landed, so a stage that only one of them came to is settled by hand: the
// bytes `theirs` is ahead by have yet to be announced, those that it never asked for are taken off.  Then each phase from the
// first that may be open (all before it were consumed, or the stage could not have been asked for again) ends when, and not before, all
// copies asked for in it have landed.
__host__ __device__ inline int e8_first_out(int own, int theirs, int stages) {
  const int most = own > theirs ? own : theirs;
  return most > stages ? most - stages : 0;
}
// Bytes to announce in stage i (negative: to take off); `half`: one block's.
__host__ __device__ inline int e8_owed(int i, int own, int theirs, int half) {
  if (i >= own && i < theirs) return half;
  return i < own && i >= theirs ? -half : 0;
}
// Takes bytes that nobody will send off a barrier's count.
__device__ __forceinline__ void mbar_complete_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Rows grouped by expert: the offsets, and the running count of tiles of `tile_rows` rows.  Offsets are held to the rows that there are, and to
// begin where the experts before have ended: whatever they hold, a row has one expert at most and no tile lies elsewhere.
struct E8Groups {
  int off[E8_MAX_GROUPS + 1];      // first row of every expert
  int end[E8_MAX_GROUPS];          // behind its last
  int cum[E8_MAX_GROUPS + 1];      // tiles of the experts before
};
// All threads of the block; the offsets have been written by now.  Two barriers.
__device__ __forceinline__ void e8_count_groups(E8Groups& g, const int* __restrict__ offsets, int n_groups, int M, int tile_rows, int n_tiles) {
  constexpr int EACH = E8_MAX_GROUPS / 32;      // experts a lane
  for (int e = threadIdx.x; e < n_groups; e += blockDim.x) {
    g.off[e] = min(max(offsets[e], 0), M);
    g.end[e] = min(max(offsets[e + 1], 0), M);
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int last = 0;      // the furthest end of the experts before this lane's
    for (int i = 0; i < EACH; i++)
      if (lane * EACH + i < n_groups) last = max(last, g.end[lane * EACH + i]);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, last, o);
      if (lane >= o) last = max(last, v);
    }
    last = __shfl_up_sync(0xffffffffu, last, 1);
    if (lane == 0) last = 0;
    int n[EACH], sum = 0;
#pragma unroll
    for (int i = 0; i < EACH; i++) {
      const int e = lane * EACH + i;
      n[i] = 0;
      if (e < n_groups) {
        const int lo = max(g.off[e], last), hi = max(g.end[e], lo);
        last = max(last, g.end[e]);
        g.off[e] = lo;
        g.end[e] = hi;
        n[i] = (hi - lo + tile_rows - 1) / tile_rows * n_tiles;
      }
      sum += n[i];
    }
    int before = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += v;
    }
    before -= sum;
#pragma unroll
    for (int i = 0; i < EACH; i++) {
      const int e = lane * EACH + i;
      if (e < n_groups) g.cum[e] = before;
      before += n[i];
      if (e == n_groups - 1) g.cum[n_groups] = before;
    }
  }
  __syncthreads();
}
// The expert of a tile: the last one whose count of tiles before it is not beyond the tile.
__device__ __forceinline__ int e8_group_of(const E8Groups& g, int n_groups, int tile) {
  int lo = 0, hi = n_groups;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (g.cum[mid] <= tile) lo = mid; else hi = mid;
  }
  return lo;
}

// A [rows, cols] byte matrix with rows ld bytes apart, read in boxes of box_rows x 128 under the 128-byte swizzle; what lies outside reads
// as zero.
static inline int e8_tensor_map(CUtensorMap* out, const void* ptr, long long rows, int cols, long long ld, int box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return leb_fail("leb_linear_e4m3: the driver has no cuTensorMapEncodeTiled");
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld};
  cuuint32_t box[2] = {(cuuint32_t)E8_BK, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = fn(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return leb_fail("leb_linear_e4m3: cuTensorMapEncodeTiled failed (%d) for [%lld,%d] rows %lld apart", (int)r, rows, cols, ld);
  return 0;
}

// A product as its kernels take it.
struct E8Product {
  void* C;
  int c_dtype;
  const void* A;
  const float* sa;
  const void* W;
  const float* sw;
  int M, N, K;
  long long lda, ldw, ldc;
  int epilogue;            // with its activation above
  const int* offsets;      // [n_groups + 1] on the device, or null
  int n_groups;
  long long w_group_stride;
  int* status;
};
// Stages of 128 numbers of k that a block of the weights-first kernel holds: what shared memory has room for with two blocks an SM, beside the
// sums that a cluster's blocks send one another.  A block's own pace is its stages by the time memory takes, so where there are no more tiles
// (of 64 rows) than SMs, and for tiles of 128 rows always, one block has an SM: 0.90 of the time of half as many stages over 73 products
// of 60 to 2,500 rows, 0.86 with 128 rows (84 products; 0.92 with more tiles than SMs, where 64 rows gain nothing).
constexpr bool few_alone(int rows, bool cluster, bool few_tiles) { return !cluster && (rows == 128 || (rows == 64 && few_tiles)); }
constexpr int few_stages(int rows, bool cluster, bool few_tiles) {
  if (few_alone(rows, cluster, few_tiles)) return rows == 128 ? 6 : 8;
  return cluster ? (rows == 16 ? 5 : rows == 32 ? 4 : 3) : (rows == 16 ? 6 : rows == 32 ? 5 : 4);
}

int leb_gemm_e4m3_any(const E8Product& p, cudaStream_t st);
int leb_gemm_e4m3_few(const E8Product& p, int mp, int n_slices, cudaStream_t st);
int leb_gemm_e4m3_pairs(const E8Product& p, cudaStream_t st);
