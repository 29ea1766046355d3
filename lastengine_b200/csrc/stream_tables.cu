// The paged cache's bookkeeping on the device: page lists, block tables and slot maps of a step from its sequences' lengths,
// without the host.  And keys and values stored where a slot map says.
//
// State, per cache: lens [slots], kept [slots] (the first page of a sequence's list, behind those of its first positions, that
// has not been given back), pages [slots][width] (page list, -1 where nothing is held), free (a stack of page numbers),
// counts {pages on the stack, status of the last step's tables}, and (or null) refused {steps refused, status of the first of them},
// which the tables only add to: it is for the program to read and clear, however many steps ran in between.
//
//   tables   pos0 = lens[slot]; sequence b, in order, takes ceil((pos0 + qlen) / P) - ceil(pos0 / P) pages off the top of the
//            stack: of all pages a step takes, number t is free[n_free - 1 - t].  Only page lists are written, beyond
//            what they held: lengths and stack stay, so the same step may be laid out again.
//   advance  lens += qlen, the pages taken leave the stack, and those that no later row reads go back on it, in
//            the order of sequences and of pages in a sequence.
//
// A step is laid out whole or not at all: a step that asks for more pages than there are (status: how many are short), that is
// longer than its tables (-1), whose rows are not as many as its lengths say (-2) or that names a slot or a
// length that cannot be (-3) leaves everything as it was, and all its sequences become padding (slot -1), which no kernel reads or writes
// a cache for.  They have no rows, or (`keep_rows`) share the step's rows out among themselves, for which attention then stores zeros.
//
// Kernels of a step read its tables ahead of their own wait for the kernel before them (common.cuh): they count on everything the
// tables were made by being complete when the step's first such kernel starts.  `advance` behind `tables` gives a step that: it waits for
// the tables, and lets nothing behind it start before it has ended.  Decode attention reads what earlier steps stored ahead of its wait in
// the same way; the stores therefore let nothing start before they have ended either.
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
  int2 t = lane < nw ? warps[lane] : make_int2(0, 0);      // every warp sums up the warps' totals
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int ua = __shfl_up_sync(0xffffffffu, t.x, o), ub = __shfl_up_sync(0xffffffffu, t.y, o);
    if (lane >= o) { t.x += ua; t.y += ub; }
  }
  const int pa = __shfl_sync(0xffffffffu, t.x, max(warp - 1, 0)), pb = __shfl_sync(0xffffffffu, t.y, max(warp - 1, 0));
  a = total_a + (warp ? pa : 0) + ia - a;
  b = total_b + (warp ? pb : 0) + ib - b;
  total_a += __shfl_sync(0xffffffffu, t.x, nw - 1);
  total_b += __shfl_sync(0xffffffffu, t.y, nw - 1);
  __syncthreads();      // `warps` may be written again
}

// The launches here may be scheduled under their predecessor and wait for it first thing; unlike pdl_wait() this does not let their own
// successor in before they end (see above).
__device__ __forceinline__ void stb_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

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

// Every block sums up the step's sequences for itself (STB_ITEMS a thread and round, their loads under way together), then takes its
// share of rows and of table lines: no block waits for another, and one launch lays out the step.
#define STB_ITEMS 4
__global__ void __launch_bounds__(STB_THREADS)
stream_tables_kernel(int* __restrict__ table, int width, int* __restrict__ slot_map, int* __restrict__ row_seq,
                     int* __restrict__ row_pos, int* __restrict__ step_slot, int* __restrict__ step_qlen,
                     int* __restrict__ pos0_out, int* __restrict__ qstart_out, const int* __restrict__ seq_slot,
                     const int* __restrict__ seq_qlen, const int* lens, int n_slots, int* pages, int pages_width,
                     const int* free_pages, int n_pages, int* counts, int* refused, int M, int B, int page, int keep_rows) {
  extern __shared__ int stb_smem[];
  int* qstart = stb_smem;          // [B + 1] first row
  int* taken = qstart + B + 1;     // [B] of the step's new pages, those of the sequences before
  int* pos0_s = taken + B;         // [B] positions held before
  int* slot_s = pos0_s + B;        // [B]
  __shared__ int2 warps[STB_THREADS / 32];
  stb_wait();
  const int n_free = min(counts[0], n_pages);
  int rows = 0, need = 0, bad = 0, longer = 0, more = 0;
  const long long longest = min((long long)min(width, pages_width) * page, 0x80000000ll - page);      // positions are counted in 32 bits
  for (int b0 = 0; b0 < B; b0 += STB_THREADS * STB_ITEMS) {
    const int first = b0 + threadIdx.x * STB_ITEMS;
    StbSeq s[STB_ITEMS];
#pragma unroll
    for (int e = 0; e < STB_ITEMS; e++) {
      s[e] = StbSeq{-1, 0, 0};
      if (first + e < B) s[e] = stb_seq(seq_slot, seq_qlen, lens, first + e, n_slots, bad);
    }
    int q = 0, n = 0, nq[STB_ITEMS], nn[STB_ITEMS];
#pragma unroll
    for (int e = 0; e < STB_ITEMS; e++) {
      nq[e] = s[e].qlen;
      nn[e] = 0;
      if (s[e].slot >= 0) {
        const long long end = (long long)s[e].pos0 + s[e].qlen;
        if (end > longest) longer = 1;
        else nn[e] = (int)((end + page - 1) / page) - (s[e].pos0 + page - 1) / page;
      }
      q += nq[e];
      n += nn[e];
    }
    stb_scan2(q, n, rows, need, warps);
#pragma unroll
    for (int e = 0; e < STB_ITEMS; e++) {
      if (first + e < B) {
        qstart[first + e] = q;
        taken[first + e] = n;
        pos0_s[first + e] = s[e].pos0;
        slot_s[first + e] = s[e].slot;
      }
      more |= nq[e] > M || (unsigned)q + (unsigned)nq[e] > (unsigned)M;      // (the first sum above M is exact, later ones may have gone round)
      q += nq[e];
      n += nn[e];
    }
  }
  if (threadIdx.x == 0) qstart[B] = rows;
  bad = __syncthreads_or(bad);
  longer = __syncthreads_or(longer);
  more = __syncthreads_or(more);
  const int status = bad ? -3 : longer ? -1 : more || rows != M ? -2 : need > n_free ? need - n_free : 0;
  const bool ok = status == 0;
  const int at = blockIdx.x * STB_THREADS + threadIdx.x, step = gridDim.x * STB_THREADS;
  if (at == 0) {
    counts[1] = status;
    if (refused && !ok) {
      const int before = refused[0];
      if (before == 0) refused[1] = status;
      if (before < 0x7fffffff) refused[0] = before + 1;
    }
  }
  // of a refused step's rows, where they are kept: the first one of sequence b (as many for each as for the others, to one row: no more than
  // any share of the rows among the sequences gives the longest)
  auto share = [&](int b) { return (int)((long long)b * M / B); };
  for (int b = at; b < B; b += step) {
    const int slot = ok ? slot_s[b] : -1;
    step_slot[b] = slot;
    step_qlen[b] = ok ? qstart[b + 1] - qstart[b] : keep_rows ? share(b + 1) - share(b) : 0;
    pos0_out[b] = slot >= 0 ? pos0_s[b] : 0;
    qstart_out[b] = ok ? qstart[b] : keep_rows ? share(b) : min(b, max(M - 1, 0));
  }
  // Rows, then table lines (a warp takes 128 places of one), shared out over all threads.  The sequence of a row is the last one that starts
  // at or before it (of those that start there, the one with rows).
  const int lane = threadIdx.x & 31, per_line = (width + 127) / 128, row_warps = (M + 31) / 32;
  for (int w = at >> 5; w < row_warps; w += step >> 5) {
    const int r = w * 32 + lane;
    if (r >= M) break;
    int b = 0, pos = 0, to = -1;
    if (ok) {      // (rows == M > 0: there is a sequence with rows)
      int lo = 0, hi = B;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (qstart[mid] <= r) lo = mid;
        else hi = mid;
      }
      b = lo;
      const int slot = slot_s[b], pos0 = slot >= 0 ? pos0_s[b] : 0;
      pos = pos0 + r - qstart[b];
      if (slot >= 0) {
        const int j = pos / page, had = (pos0 + page - 1) / page;
        const int pg = j < had ? pages[(size_t)slot * pages_width + j] : free_pages[n_free - 1 - (taken[b] + j - had)];
        to = pg * page + pos % page;
      }
    } else if (keep_rows) {      // the last sequence whose share begins at or before the row
      b = (int)(((long long)(r + 1) * B - 1) / M);
      pos = r - share(b);
    }
    row_seq[r] = b;
    row_pos[r] = pos;
    slot_map[r] = to;
  }
  const int warps_all = step >> 5, from = (int)(((at >> 5) + warps_all - row_warps % warps_all) % warps_all);      // on from where the rows ended
  for (int w = from; w < B * per_line; w += warps_all) {
    const int b = w / per_line, j0 = (w - b * per_line) * 128;
    const int slot = ok ? slot_s[b] : -1;
    const int pos0 = slot >= 0 ? pos0_s[b] : 0, had = (pos0 + page - 1) / page;
    const int now = slot >= 0 ? (pos0 + (qstart[b + 1] - qstart[b]) + page - 1) / page : 0;
    int* line = table + (size_t)b * width;
    int* mine = pages + (size_t)(slot < 0 ? 0 : slot) * pages_width;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int j = j0 + e * 32 + lane;
      if (j >= width) break;
      int v = -1;
      if (j < now) {
        if (j < had) v = mine[j];
        else mine[j] = v = free_pages[n_free - 1 - (taken[b] + j - had)];      // (read above only below `had`)
      }
      line[j] = v;
    }
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
  // of each sequence of a round: its slot (-1: none), how many pages of those before it go back, how many of the first positions' go
  // back, where the others begin
  __shared__ int slot_s[STB_ADVANCE_THREADS], to_s[STB_ADVANCE_THREADS], head_s[STB_ADVANCE_THREADS], lo_s[STB_ADVANCE_THREADS];
  const int fp = (first + page - 1) / page;
  int need = 0, back = 0, bad = 0;
  stb_wait();
  const int n_free = counts[0];
  const bool rounds = B > (int)blockDim.x;
  if (!RELEASE && rounds) {      // the pages taken leave the stack before any goes back on it
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
  for (int b0 = 0; b0 < B; b0 += blockDim.x) {
    const int b = b0 + threadIdx.x;
    StbSeq s{-1, 0, 0};
    int head = 0, lo = 0, hi = 0, n = 0;
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
      if (!RELEASE && !rounds) n = (len + page - 1) / page - (s.pos0 + page - 1) / page;
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
    int to = head + hi - lo;
    const int before = back;
    stb_scan2(to, n, back, need, warps);      // (over several rounds `need` is known already, and n is 0)
    slot_s[threadIdx.x] = s.slot;
    to_s[threadIdx.x] = to;
    head_s[threadIdx.x] = head;
    lo_s[threadIdx.x] = lo;
    __syncthreads();
    // a thread per page that goes back: that of the last sequence whose pages begin at or before it
    for (int k = before + threadIdx.x; k < back; k += blockDim.x) {
      int i = 0, end = blockDim.x;
      while (end - i > 1) {
        const int mid = (i + end) >> 1;
        if (to_s[mid] <= k) i = mid;
        else end = mid;
      }
      const int own = k - to_s[i], j = own < head_s[i] ? own : lo_s[i] + own - head_s[i], at = n_free - need + k;
      if (slot_s[i] >= 0 && j < pages_width && at >= 0 && at < n_pages) {      // (always, unless a slot is named twice)
        int* mine = pages + (size_t)slot_s[i] * pages_width;
        free_pages[at] = mine[j];
        mine[j] = -1;
      }
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) counts[0] = min(max(n_free - need + back, 0), n_pages);
}

static const int STB_MOST_SEQS = 8192;      // sequences a step may have: four words each in shared memory

LEB_API int leb_stream_tables(int* table, int width, int* slot_map, int* row_seq, int* row_pos, int* step_slot, int* step_qlen,
                              int* pos0, int* qstart, const int* seq_slot, const int* seq_qlen, const int* lens, int n_slots,
                              int* pages, int pages_width, const int* free_pages, int n_pages, int* counts, int* refused, int M, int B,
                              int page, int keep_rows, cudaStream_t st) {
  if (B <= 0) return 0;
  LEB_REQUIRE(B <= STB_MOST_SEQS, "leb_stream_tables: %d sequences in a step, %d at most", B, STB_MOST_SEQS);
  LEB_REQUIRE(page > 0 && width > 0 && pages_width > 0 && n_slots > 0 && M >= 0, "leb_stream_tables: sizes (page %d, width %d, slots %d, rows %d)",
              page, width, n_slots, M);
  constexpr auto kern = stream_tables_kernel;
  const size_t smem = (4 * (size_t)B + 1) * sizeof(int);
  if (smem > 48 * 1024) {
    const cudaError_t e = leb_allow_smem<kern, (4 * STB_MOST_SEQS + 1) * (int)sizeof(int)>();
    if (e != cudaSuccess) return leb_fail("leb_stream_tables: shared memory %zu: %s", smem, cudaGetErrorString(e));
  }
  const long long lines = (long long)B * ((width + 127) / 128) * 32;      // threads that table lines want
  LEB_REQUIRE(lines / 32 <= 0x7fffffffll, "leb_stream_tables: tables of %d x %d places", B, width);
  const long long most = 4ll * sm_count(), want = (lines + (M + 31) / 32 * 32 + STB_THREADS - 1) / STB_THREADS;
  const int blocks = (int)(want < 1 ? 1 : want < most ? want : most);
  leb_launch(kern, dim3(blocks), dim3(STB_THREADS), smem, st, table, width, slot_map, row_seq, row_pos, step_slot, step_qlen, pos0, qstart,
             seq_slot, seq_qlen, lens, n_slots, pages, pages_width, free_pages, n_pages, counts, refused, M, B, page, keep_rows);
  LEB_CHECK_LAUNCH("leb_stream_tables");
  return 0;
}

// Threads of the one block: one per sequence, up to eight warps at least for the pages that go back.
static int advance_threads(int B) { return B <= 256 ? 256 : B <= 512 ? 512 : STB_ADVANCE_THREADS; }

LEB_API int leb_stream_advance(const int* seq_slot, const int* seq_qlen, int* lens, int n_slots, int* kept, int* pages,
                               int pages_width, int* free_pages, int n_pages, int* counts, int B, int page, int window, int first,
                               cudaStream_t st) {
  if (B <= 0) return 0;
  LEB_REQUIRE(page > 0 && window >= 0 && first >= 0, "leb_stream_advance: page %d, window %d, first %d", page, window, first);
  leb_launch(stream_advance_kernel<false>, dim3(1), dim3(advance_threads(B)), 0, st, seq_slot, seq_qlen, lens, n_slots, kept, pages,
             pages_width, free_pages, n_pages, counts, B, page, window, first);
  LEB_CHECK_LAUNCH("leb_stream_advance");
  return 0;
}

LEB_API int leb_stream_release(const int* seq_slot, int* lens, int n_slots, int* kept, int* pages, int pages_width, int* free_pages,
                               int n_pages, int* counts, int B, int page, int first, cudaStream_t st) {
  if (B <= 0) return 0;
  LEB_REQUIRE(page > 0 && first >= 0, "leb_stream_release: page %d, first %d", page, first);
  leb_launch(stream_advance_kernel<true>, dim3(1), dim3(advance_threads(B)), 0, st, seq_slot, nullptr, lens, n_slots, kept, pages,
             pages_width, free_pages, n_pages, counts, B, page, 0, first);
  LEB_CHECK_LAUNCH("leb_stream_release");
  return 0;
}

// Row m of keys and values [M][nkv][dim] goes to position slots[m] % page of page slots[m] / page: the key as a row of its head's
// keys, the value as a column of its head's values.  -1 (and what lies outside the pool): nowhere.
//
// Few rows: a block per row.
template <typename T>
__global__ void __launch_bounds__(256)
store_rows_kernel(T* __restrict__ k_pool, T* __restrict__ v_pool, const T* __restrict__ k, int k_stride, const T* __restrict__ v,
                  int v_stride, const int* __restrict__ slots, int n_pages, int M, int nkv, int hd, int vd, int page) {
  stb_wait();
  const int m = blockIdx.x;
  const int slot = slots[m];
  const int pg = slot / page, off = slot % page;
  if (slot < 0 || pg >= n_pages) return;
  for (int i = threadIdx.x; i < nkv * hd; i += blockDim.x)
    k_pool[(((size_t)pg * nkv + i / hd) * page + off) * hd + i % hd] = k[(size_t)m * k_stride + i];
  for (int i = threadIdx.x; i < nkv * vd; i += blockDim.x)
    v_pool[((size_t)pg * nkv * vd + i) * page + off] = v[(size_t)m * v_stride + i];
}

// Many rows: a block per 64 rows and kv head.  Values are turned in shared memory, DC dimensions at a time: a warp then writes one
// dimension of 64 rows, a line of 128 bytes (bfloat16, two rows a lane) where the rows' places follow one another in a page.
// Where there are few blocks, gridDim.z of them share the keys and the dimensions of a tile.
// VK / VV: keys / values can be loaded (and keys stored) in pieces of 16 bytes.
#define STR_ROWS 64
// From which rows on, us by rows and by tiles (8 kv heads of 64): a prompt of 64, 128, 256, 512 rows 2.59, 2.78, 3.68, 5.26 and 2.29, 2.30,
// 2.30, 2.46; single tokens of as many streams 2.60, 2.59, 3.03, 4.48 and 3.41, 3.40, 3.58, 4.75.  Bound by memory: 16,439 rows (67 MB) 12.8 us,
// 5.2 TB/s (a block per row 77; with the places worked out by divisions for every piece 15.8, 69% of the issue slots).
#define STR_FEW 192
// The pieces (0 .. per - 1) of `rows` rows, shared out over the eight warps of `parts` blocks: calls f(row, piece).  A lane's place in a row is
// worked out once: a warp takes as many rows at a time as it has lanes for, or one.
template <typename F>
__device__ __forceinline__ void str_pieces(int rows, int per, int part, int parts, F f) {
  const int lane = threadIdx.x & 31, warp = part * 8 + (threadIdx.x >> 5), warps = parts * 8;
  if (per <= 32) {
    const int at_once = 32 / per, row = lane / per, c = lane - row * per;
    if (row < at_once) {
#pragma unroll 2
      for (int r = warp * at_once + row; r < rows; r += warps * at_once) f(r, c);
    }
  } else {
    for (int r = warp; r < rows; r += warps)
#pragma unroll 2
      for (int c = lane; c < per; c += 32) f(r, c);
  }
}
template <typename T, bool VK, bool VV, int DC>
__global__ void __launch_bounds__(256)
store_tile_kernel(T* __restrict__ k_pool, T* __restrict__ v_pool, const T* __restrict__ k, int k_stride, const T* __restrict__ v,
                  int v_stride, const int* __restrict__ slots, int n_pages, int M, int nkv, int hd, int vd, int page) {
  constexpr int W = 16 / sizeof(T), STRIDE = DC + 4 / sizeof(T);      // a row of v_s is an odd number of words
  __shared__ int slot_s[STR_ROWS];
  __shared__ long long place_s[STR_ROWS];      // of a row's page and head: the first position's place in a pool of one number a position
  __shared__ __align__(16) T v_s[STR_ROWS * STRIDE];
  stb_wait();
  const int m0 = blockIdx.x * STR_ROWS, head = blockIdx.y, rows = min(STR_ROWS, M - m0);
  if (threadIdx.x < STR_ROWS) {
    int s = (int)threadIdx.x < rows ? slots[m0 + threadIdx.x] : -1;
    const int pg = s / page;
    if (pg >= n_pages) s = -1;
    slot_s[threadIdx.x] = s < 0 ? -1 : s - pg * page;      // from here on a row's place in its page
    place_s[threadIdx.x] = s < 0 ? 0 : ((long long)pg * nkv + head) * page;
  }
  __syncthreads();
  const T* ks = k + (size_t)m0 * k_stride + (size_t)head * hd;
  const T* vs = v + (size_t)m0 * v_stride + (size_t)head * vd;
  str_pieces(rows, VK ? hd / W : hd, blockIdx.z, gridDim.z, [&](int row, int c) {
    const int off = slot_s[row];
    if (off < 0) return;
    T* dst = k_pool + (place_s[row] + off) * hd;
    if (VK) reinterpret_cast<uint4*>(dst)[c] = *reinterpret_cast<const uint4*>(ks + (size_t)row * k_stride + c * W);
    else dst[c] = ks[(size_t)row * k_stride + c];
  });
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int d0 = blockIdx.z * DC; d0 < vd; d0 += DC * gridDim.z) {
    const int n = min(DC, vd - d0);
    if (d0 >= DC * (int)gridDim.z) __syncthreads();
    str_pieces(rows, VV ? n / W : n, 0, 1, [&](int row, int c) {
      if (VV) {
        const uint4 x = *reinterpret_cast<const uint4*>(vs + (size_t)row * v_stride + d0 + c * W);
        uint32_t* to = reinterpret_cast<uint32_t*>(v_s + row * STRIDE + c * W);
        to[0] = x.x, to[1] = x.y, to[2] = x.z, to[3] = x.w;
      } else {
        v_s[row * STRIDE + c] = vs[(size_t)row * v_stride + d0 + c];
      }
    });
    __syncthreads();
    if (sizeof(T) == 2) {
      // two rows a lane, two dimensions a warp's turn
      const int ra = 2 * lane, sa = slot_s[ra], sb = slot_s[ra + 1];
      const bool joined = sa >= 0 && sb == sa + 1 && place_s[ra] == place_s[ra + 1] && ((sa | page) & 1) == 0 &&      // both places in one aligned word
                          ((uintptr_t)v_pool & 3) == 0;
      T* const pa = v_pool + place_s[ra] * vd + max(sa, 0);
      T* const pb = v_pool + place_s[ra + 1] * vd + max(sb, 0);
      for (int d = 2 * warp; d < n; d += 16) {
        const uint32_t a = *reinterpret_cast<const uint32_t*>(v_s + ra * STRIDE + d), c = *reinterpret_cast<const uint32_t*>(v_s + (ra + 1) * STRIDE + d);
        const size_t at = (size_t)(d0 + d) * page;
        const bool second = d + 1 < n;
        if (joined) {
          *reinterpret_cast<uint32_t*>(pa + at) = __byte_perm(a, c, 0x5410);
          if (second) *reinterpret_cast<uint32_t*>(pa + at + page) = __byte_perm(a, c, 0x7632);
        } else {
          const T* ea = reinterpret_cast<const T*>(&a);
          const T* ec = reinterpret_cast<const T*>(&c);
          if (sa >= 0) {
            pa[at] = ea[0];
            if (second) pa[at + page] = ea[1];
          }
          if (sb >= 0) {
            pb[at] = ec[0];
            if (second) pb[at + page] = ec[1];
          }
        }
      }
    } else {
#pragma unroll
      for (int h = 0; h < STR_ROWS; h += 32) {
        const int slot = slot_s[h + lane];
        if (slot < 0) continue;
        T* to = v_pool + place_s[h + lane] * vd + (size_t)d0 * page + slot;
        for (int d = warp; d < n; d += 8) to[(size_t)d * page] = v_s[(h + lane) * STRIDE + d];
      }
    }
  }
}

template <typename T>
static int launch_store_rows(T* k_pool, T* v_pool, const T* k, int k_stride, const T* v, int v_stride, const int* slots, int n_pages,
                             int M, int nkv, int hd, int vd, int page, int many, cudaStream_t st) {
  if (!many) {
    leb_launch(store_rows_kernel<T>, dim3(M), dim3(256), 0, st, k_pool, v_pool, k, k_stride, v, v_stride, slots, n_pages, M, nkv, hd, vd, page);
  } else {
    constexpr int W = 16 / sizeof(T);
    const bool vk = hd % W == 0 && k_stride % W == 0 && (((uintptr_t)k | (uintptr_t)k_pool) & 15) == 0;
    const bool vv = vd % W == 0 && v_stride % W == 0 && ((uintptr_t)v & 15) == 0;
    dim3 grid(ceil_div(M, STR_ROWS), nkv);
    LEB_REQUIRE(grid.y <= 65535, "leb_store_rows: grid too large (%u kv heads)", grid.y);
    const bool few = (long long)grid.x * grid.y < 2ll * sm_count();
    if (few) grid.z = ceil_div(vd, 16);
#define LEB_STR(VK, VV)                                                                                                                     \
  (few ? leb_launch(store_tile_kernel<T, VK, VV, 16>, grid, dim3(256), 0, st, k_pool, v_pool, k, k_stride, v, v_stride, slots, n_pages, M, nkv, hd, vd, page) \
       : leb_launch(store_tile_kernel<T, VK, VV, 64>, grid, dim3(256), 0, st, k_pool, v_pool, k, k_stride, v, v_stride, slots, n_pages, M, nkv, hd, vd, page))
    if (vk && vv) LEB_STR(true, true);
    else if (vk) LEB_STR(true, false);
    else if (vv) LEB_STR(false, true);
    else LEB_STR(false, false);
#undef LEB_STR
  }
  LEB_CHECK_LAUNCH("leb_store_rows");
  return 0;
}

LEB_API int leb_store_rows(void* k_pool, void* v_pool, const void* k, int k_stride, const void* v, int v_stride, int dtype,
                           const int* slots, int n_pages, int M, int nkv, int hd, int vd, int page, cudaStream_t st) {
  if (M <= 0) return 0;
  LEB_REQUIRE(n_pages > 0 && nkv > 0 && hd > 0 && vd > 0 && page > 0, "leb_store_rows: sizes (pages %d, kv heads %d, widths %d and %d, page %d)",
              n_pages, nkv, hd, vd, page);
  const int many = M >= STR_FEW;
  if (dtype == LEB_F32)
    return launch_store_rows((float*)k_pool, (float*)v_pool, (const float*)k, k_stride, (const float*)v, v_stride, slots, n_pages, M, nkv, hd, vd, page, many, st);
  if (dtype == LEB_BF16)
    return launch_store_rows((bf16*)k_pool, (bf16*)v_pool, (const bf16*)k, k_stride, (const bf16*)v, v_stride, slots, n_pages, M, nkv, hd, vd, page, many, st);
  return leb_fail("leb_store_rows: unknown dtype %d", dtype);
}
