// The paged cache's bookkeeping on the device: page lists, block tables and slot maps of a step from its sequences' lengths,
// without the host.  And keys and values stored where a slot map says.
//
// State, per cache: lens [slots], kept [slots] (the first page of a sequence's list, behind those of its first positions, that
// has not been given back), pages [slots][width] (page list, -1 where nothing is held), free (a stack of page numbers),
// counts {pages on the stack, status of the last step's tables}.
//
//   tables   pos0 = lens[slot]; sequence b, in order, takes ceil((pos0 + qlen) / P) - ceil(pos0 / P) pages off the top of the
//            stack: of all pages a step takes, number t is free[n_free - 1 - t].  Only page lists are written, beyond
//            what they held: lengths and stack stay, so the same step may be laid out again.
//   advance  lens += qlen, the pages taken leave the stack, and those that no later row reads go back on it, in
//            the order of sequences and of pages in a sequence.
//
// A step is laid out whole or not at all: a step that asks for more pages than there are (status: how many are short), that is
// longer than its tables (-1), whose rows are not as many as its lengths say (-2) or that names a slot or a
// length that cannot be (-3) leaves everything as it was, and all its sequences become padding (slot -1, no rows), which no
// kernel reads or writes a cache for.
//
// Kernels of a step read its tables ahead of their own wait for the kernel before them (common.cuh): they count on everything the
// tables were made by being complete when the step's first such kernel starts.  The launches here are plain ones, which start when
// all before them is complete and visible: `advance` behind `tables` gives a step that.
#include "common.cuh"

#define STB_THREADS 256

// Exclusive sums of two numbers per thread over a block, on top of the running totals, which every thread gets back.
__device__ __forceinline__ void stb_scan2(int& a, int& b, int& total_a, int& total_b, int2* warps) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  int ia = a, ib = b;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int ua = __shfl_up_sync(0xffffffffu, ia, o), ub = __shfl_up_sync(0xffffffffu, ib, o);
    if (lane >= o) { ia += ua; ib += ub; }
  }
  if (lane == 31) warps[warp] = make_int2(ia, ib);
  __syncthreads();
  int pa = total_a, pb = total_b;
  for (int w = 0; w < nw; w++) {
    const int2 t = warps[w];
    if (w < warp) { pa += t.x; pb += t.y; }
    total_a += t.x;
    total_b += t.y;
  }
  __syncthreads();
  a = pa + ia - a;
  b = pb + ib - b;
}

// What a step's sequence b asks for; false where it names a slot or a length that cannot be.
struct StbSeq { int slot, qlen, pos0; };
__device__ __forceinline__ StbSeq stb_seq(const int* seq_slot, const int* seq_qlen, const int* lens, int b, int n_slots, int& bad) {
  StbSeq s{seq_slot[b], seq_qlen[b], 0};
  if (s.slot < -1 || s.slot >= n_slots || s.qlen < 0) {
    bad = 1;
    s.slot = -1;
    s.qlen = 0;
  }
  if (s.slot >= 0) s.pos0 = lens[s.slot];
  return s;
}

__global__ void __launch_bounds__(STB_THREADS)
stream_tables_kernel(int* __restrict__ table, int width, int* __restrict__ slot_map, int* __restrict__ row_seq,
                     int* __restrict__ row_pos, int* __restrict__ step_slot, int* __restrict__ step_qlen,
                     int* __restrict__ pos0_out, int* __restrict__ qstart_out, const int* __restrict__ seq_slot,
                     const int* __restrict__ seq_qlen, const int* __restrict__ lens, int n_slots, int* pages, int pages_width,
                     const int* __restrict__ free_pages, int n_pages, int* counts, int M, int B, int page) {
  extern __shared__ int stb_smem[];
  int* qstart = stb_smem;          // [B + 1]
  int* taken = qstart + B + 1;     // [B]
  __shared__ int2 warps[STB_THREADS / 32];
  int rows = 0, need = 0, bad = 0, longer = 0;
  for (int b0 = 0; b0 < B; b0 += STB_THREADS) {
    const int b = b0 + threadIdx.x;
    int q = 0, n = 0;
    if (b < B) {
      const StbSeq s = stb_seq(seq_slot, seq_qlen, lens, b, n_slots, bad);
      q = s.qlen;
      if (s.slot >= 0) {
        const long long end = (long long)s.pos0 + s.qlen;
        if (end > (long long)min(width, pages_width) * page) longer = 1;
        else n = (int)((end + page - 1) / page) - (s.pos0 + page - 1) / page;
      }
    }
    stb_scan2(q, n, rows, need, warps);
    if (b < B) {
      qstart[b] = q;
      taken[b] = n;
    }
  }
  if (threadIdx.x == 0) qstart[B] = rows;
  bad = __syncthreads_or(bad);
  longer = __syncthreads_or(longer);
  const int n_free = min(counts[0], n_pages);
  const int status = bad ? -3 : longer ? -1 : rows != M ? -2 : need > n_free ? need - n_free : 0;
  const bool ok = status == 0;
  const int at = blockIdx.x * STB_THREADS + threadIdx.x, step = gridDim.x * STB_THREADS;
  if (at == 0) counts[1] = status;
  for (int b = at; b < B; b += step) {
    const int slot = seq_slot[b];
    const bool live = ok && slot >= 0;
    step_slot[b] = live ? slot : -1;
    step_qlen[b] = ok ? seq_qlen[b] : 0;
    pos0_out[b] = live ? lens[slot] : 0;
    qstart_out[b] = ok ? qstart[b] : min(b, max(M - 1, 0));
  }
  for (int r = at; r < M; r += step) {
    int b = 0, pos = 0, to = -1;
    if (ok) {      // (rows == M > 0: there is a sequence with rows)
      int lo = 0, hi = B;          // the last sequence that starts at or before this row (one of those that start there is not empty)
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (qstart[mid] <= r) lo = mid;
        else hi = mid;
      }
      b = lo;
      const int slot = seq_slot[b];
      const int pos0 = slot >= 0 ? lens[slot] : 0;
      pos = pos0 + r - qstart[b];
      if (slot >= 0) {
        const int j = pos / page, had = (pos0 + page - 1) / page;
        const int pg = j < had ? pages[(size_t)slot * pages_width + j] : free_pages[n_free - 1 - (taken[b] + j - had)];
        to = pg * page + pos % page;
      }
    }
    row_seq[r] = b;
    row_pos[r] = pos;
    slot_map[r] = to;
  }
  const long long cells = (long long)B * width;
  for (long long i = at; i < cells; i += step) {
    const int b = (int)(i / width), j = (int)(i % width);
    int v = -1;
    const int slot = seq_slot[b];
    if (ok && slot >= 0) {
      const int pos0 = lens[slot], had = (pos0 + page - 1) / page;
      if (j < had) v = pages[(size_t)slot * pages_width + j];
      else if ((long long)j * page < (long long)pos0 + seq_qlen[b]) {
        v = free_pages[n_free - 1 - (taken[b] + j - had)];
        pages[(size_t)slot * pages_width + j] = v;      // (read above only below `had`)
      }
    }
    table[i] = v;
  }
}

// One block.  RELEASE: the sequences end instead, and everything they hold goes back.
#define STB_ADVANCE_THREADS 1024
template <bool RELEASE>
__global__ void __launch_bounds__(STB_ADVANCE_THREADS)
stream_advance_kernel(const int* __restrict__ seq_slot, const int* __restrict__ seq_qlen, int* lens, int n_slots, int* kept,
                      int* pages, int pages_width, int* free_pages, int n_pages, int* counts, int B, int page, int window,
                      int first) {
  __shared__ int2 warps[STB_ADVANCE_THREADS / 32];
  // of each sequence of a round: its slot (-1: none), where on the stack its pages go, how many of the first positions' go
  // back, where the others begin, how many go back in all
  __shared__ int slot_s[STB_ADVANCE_THREADS], to_s[STB_ADVANCE_THREADS], head_s[STB_ADVANCE_THREADS], lo_s[STB_ADVANCE_THREADS], n_s[STB_ADVANCE_THREADS];
  const int fp = (first + page - 1) / page;
  int need = 0, back = 0, bad = 0;
  if (!RELEASE) {      // the pages taken leave the stack before any goes back on it
    for (int b0 = 0; b0 < B; b0 += blockDim.x) {
      const int b = b0 + threadIdx.x;
      int n = 0, zero = 0;
      if (b < B) {
        const StbSeq s = stb_seq(seq_slot, seq_qlen, lens, b, n_slots, bad);
        if (s.slot >= 0) n = (s.pos0 + s.qlen + page - 1) / page - (s.pos0 + page - 1) / page;
      }
      stb_scan2(n, zero, need, back, warps);
    }
  }
  const int top = counts[0] - need;
  for (int b0 = 0; b0 < B; b0 += blockDim.x) {
    const int b = b0 + threadIdx.x;
    StbSeq s{-1, 0, 0};
    int head = 0, lo = 0, hi = 0;
    if (b < B) {
      if (RELEASE) {
        s.slot = seq_slot[b];
        if (s.slot < 0 || s.slot >= n_slots) s.slot = -1;
        else s.pos0 = lens[s.slot];
      } else {
        s = stb_seq(seq_slot, seq_qlen, lens, b, n_slots, bad);
      }
    }
    if (s.slot >= 0) {
      const int len = s.pos0 + s.qlen;
      lo = max(kept[s.slot], fp);
      if (RELEASE) {
        head = min(fp, (len + page - 1) / page);
        hi = max(lo, (len + page - 1) / page);
      } else {      // the next row, at position len, reads back to len + 1 - window
        hi = window > 0 ? max(lo, max(0, len + 1 - window) / page) : lo;
      }
      lens[s.slot] = RELEASE ? 0 : len;
      kept[s.slot] = RELEASE ? fp : hi;
    }
    int to = head + hi - lo, zero = 0, nothing = 0;
    n_s[threadIdx.x] = to;
    stb_scan2(to, zero, back, nothing, warps);
    slot_s[threadIdx.x] = s.slot;
    to_s[threadIdx.x] = top + to;
    head_s[threadIdx.x] = head;
    lo_s[threadIdx.x] = lo;
    __syncthreads();
    for (int i = threadIdx.x >> 5; i < min((int)blockDim.x, B - b0); i += blockDim.x >> 5) {      // a warp per sequence
      if (slot_s[i] < 0) continue;
      int* mine = pages + (size_t)slot_s[i] * pages_width;
      for (int k = threadIdx.x & 31; k < n_s[i]; k += 32) {
        const int j = k < head_s[i] ? k : lo_s[i] + k - head_s[i], at = to_s[i] + k;
        if (j < pages_width && at >= 0 && at < n_pages) {      // (always, unless a slot is named twice)
          free_pages[at] = mine[j];
          mine[j] = -1;
        }
      }
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) counts[0] = min(max(top + back, 0), n_pages);
}

static const int STB_MOST_SEQS = 16384;      // sequences a step may have: two words each in shared memory

LEB_API int leb_stream_tables(int* table, int width, int* slot_map, int* row_seq, int* row_pos, int* step_slot, int* step_qlen,
                              int* pos0, int* qstart, const int* seq_slot, const int* seq_qlen, const int* lens, int n_slots,
                              int* pages, int pages_width, const int* free_pages, int n_pages, int* counts, int M, int B, int page,
                              cudaStream_t st) {
  if (B <= 0) return 0;
  LEB_REQUIRE(B <= STB_MOST_SEQS, "leb_stream_tables: %d sequences in a step, %d at most", B, STB_MOST_SEQS);
  LEB_REQUIRE(page > 0 && width > 0 && pages_width > 0 && n_slots > 0 && M >= 0, "leb_stream_tables: sizes (page %d, width %d, slots %d, rows %d)",
              page, width, n_slots, M);
  constexpr auto kern = stream_tables_kernel;
  const size_t smem = (2 * (size_t)B + 1) * sizeof(int);
  if (smem > 48 * 1024) {
    const cudaError_t e = leb_allow_smem<kern>();
    if (e != cudaSuccess) return leb_fail("leb_stream_tables: shared memory %zu: %s", smem, cudaGetErrorString(e));
  }
  const long long items = (long long)M > (long long)B * width ? M : (long long)B * width;
  const long long most = 4ll * sm_count(), want = (items + STB_THREADS - 1) / STB_THREADS;
  const int blocks = (int)(want < 1 ? 1 : want < most ? want : most);
  kern<<<blocks, STB_THREADS, smem, st>>>(table, width, slot_map, row_seq, row_pos, step_slot, step_qlen, pos0, qstart, seq_slot,
                                          seq_qlen, lens, n_slots, pages, pages_width, free_pages, n_pages, counts, M, B, page);
  LEB_CHECK_LAUNCH("leb_stream_tables");
  return 0;
}

LEB_API int leb_stream_advance(const int* seq_slot, const int* seq_qlen, int* lens, int n_slots, int* kept, int* pages,
                               int pages_width, int* free_pages, int n_pages, int* counts, int B, int page, int window, int first,
                               cudaStream_t st) {
  if (B <= 0) return 0;
  LEB_REQUIRE(page > 0 && window >= 0 && first >= 0, "leb_stream_advance: page %d, window %d, first %d", page, window, first);
  stream_advance_kernel<false><<<1, STB_ADVANCE_THREADS, 0, st>>>(seq_slot, seq_qlen, lens, n_slots, kept, pages, pages_width, free_pages,
                                                                  n_pages, counts, B, page, window, first);
  LEB_CHECK_LAUNCH("leb_stream_advance");
  return 0;
}

LEB_API int leb_stream_release(const int* seq_slot, int* lens, int n_slots, int* kept, int* pages, int pages_width, int* free_pages,
                               int n_pages, int* counts, int B, int page, int first, cudaStream_t st) {
  if (B <= 0) return 0;
  LEB_REQUIRE(page > 0 && first >= 0, "leb_stream_release: page %d, first %d", page, first);
  stream_advance_kernel<true><<<1, STB_ADVANCE_THREADS, 0, st>>>(seq_slot, nullptr, lens, n_slots, kept, pages, pages_width, free_pages,
                                                                 n_pages, counts, B, page, 0, first);
  LEB_CHECK_LAUNCH("leb_stream_release");
  return 0;
}

// Row m of keys and values [M][nkv][dim] goes to position slots[m] % page of page slots[m] / page: the key as a row of its head's
// keys, the value as a column of its head's values.  -1 (and what lies outside the pool): nowhere.
template <typename T>
__global__ void store_rows_kernel(T* __restrict__ k_pool, T* __restrict__ v_pool, const T* __restrict__ k, int k_stride,
                                  const T* __restrict__ v, int v_stride, const int* __restrict__ slots, int n_pages, int M, int nkv,
                                  int hd, int vd, int page) {
  const int m = blockIdx.x;
  const int slot = slots[m];
  const int pg = slot / page, off = slot % page;
  if (slot < 0 || pg >= n_pages) return;
  for (int i = threadIdx.x; i < nkv * hd; i += blockDim.x)
    k_pool[(((size_t)pg * nkv + i / hd) * page + off) * hd + i % hd] = k[(size_t)m * k_stride + i];
  for (int i = threadIdx.x; i < nkv * vd; i += blockDim.x)
    v_pool[((size_t)pg * nkv * vd + i) * page + off] = v[(size_t)m * v_stride + i];
}

LEB_API int leb_store_rows(void* k_pool, void* v_pool, const void* k, int k_stride, const void* v, int v_stride, int dtype,
                           const int* slots, int n_pages, int M, int nkv, int hd, int vd, int page, cudaStream_t st) {
  if (M <= 0) return 0;
  LEB_REQUIRE(n_pages > 0 && nkv > 0 && hd > 0 && vd > 0 && page > 0, "leb_store_rows: sizes (pages %d, kv heads %d, widths %d and %d, page %d)",
              n_pages, nkv, hd, vd, page);
  if (dtype == LEB_F32)
    store_rows_kernel<float><<<M, 256, 0, st>>>((float*)k_pool, (float*)v_pool, (const float*)k, k_stride, (const float*)v, v_stride, slots,
                                                n_pages, M, nkv, hd, vd, page);
  else if (dtype == LEB_BF16)
    store_rows_kernel<bf16><<<M, 256, 0, st>>>((bf16*)k_pool, (bf16*)v_pool, (const bf16*)k, k_stride, (const bf16*)v, v_stride, slots,
                                               n_pages, M, nkv, hd, vd, page);
  else
    return leb_fail("leb_store_rows: unknown dtype %d", dtype);
  LEB_CHECK_LAUNCH("leb_store_rows");
  return 0;
}
