// Pages of a KV cache: who has which (a table and reference counts, both on the device), and copying them.
//
// A table (sequences, pages of a sequence) names pages of a pool, -1 where there is none; refs counts the entries that name a page, 0 is
// free.  The book-keeping is a few thousand whole numbers: one cluster of eight CTAs does it in one launch, in phases between
// rendezvous of the cluster, so nothing waits for the host and results do not depend on the order of threads (counters are
// only added to; what is given away is ranked by prefix sums: rows in order, free pages from the lowest on).  What bounds it is latency: a launch, three or four rendezvous
// and a trip to memory between each.  us back to back: resize of 128 rows of 18 pages in a pool of 1315 8.6, 256 of 66 in 11761 10.4, 256 of 512 in 70000 15.4, 1024 of 256 in 300000 30;
// compact of the same 11, 13, 21, 52; fork of 128 rows 2.2.  A row is one warp's, which reads its entries 128 at a time: 64 rows of 4096 entries in 300000 48 (compact 53, fork 11.6).
#pragma once
#include "fp8_append.cuh"

namespace fa4 {
namespace pages {

constexpr int kCluster = 8, kThreads = 1024, kWarps = kThreads / 32;        // (at most so many CTAs)
constexpr int kRows = 4096;                    // of a table: their prefix sums stay in shared memory

enum Site { kTableSite = 123, kLengthSite = 124, kPoolSite = 125, kParentSite = 126, kPairSite = 127, kCopySite = 128 };

struct Book {
  int32_t* table;
  int32_t* refs;
  int B, width, num_pages, page_size;
  int ctas;                          // of the cluster
  FastDiv div_page;
  uint32_t* status;
  uint32_t epoch;
};
// Marks on a page number: a row's page that is copied (inside resize); the page of an entry whose row waits for a copy of it, which was to be written to and found no page.
// The latter is in tables: the calls that read and write caches take it for no page at all, here it is an entry like others.
constexpr int kCopied = 0x40000000, kWaits = (int)0x80000000;
__device__ __forceinline__ int page_in(int entry) { return entry < 0 && (entry & kCopied) == 0 ? entry & ~kWaits : entry; }
// Pages of `tokens`.
__device__ __forceinline__ int pages_of(const Book& p, int tokens) {
  const int whole = fast_div(tokens, p.div_page);
  return whole + (whole * p.page_size < tokens);
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// Rendezvous of the cluster behind which everything that was written before it, global memory included, can be read (by __ldcg).
__device__ __forceinline__ void meet(const Book& p) {
  __threadfence();
  if (p.ctas > 1) cluster_sync();
  else __syncthreads();
}

// Exclusive prefix sum over the CTA's warps of a value of each; `all`: the sum.  s: kWarps + 1 words.
__device__ __forceinline__ int scan_warps(int mine, int* s, int* all) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __syncthreads();
  if (lane == 0) s[warp] = mine;
  __syncthreads();
  if (warp == 0) {
    const int v = s[lane];
    int upto = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int w = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += w;
    }
    s[lane] = upto - v;
    if (lane == 31) s[kWarps] = upto;
  }
  __syncthreads();
  *all = s[kWarps];
  return s[warp];
}

// The part of the pool that a warp of the cluster looks at: [from, to), multiples of 32 from the pool's start.
struct Part {
  int from, to;
};
__device__ __forceinline__ Part part_of(const Book& p) {
  const int warps = p.ctas * kWarps, per = ((p.num_pages + warps - 1) / warps + 31) & ~31;
  const int w = (int)cluster_rank() * kWarps + (threadIdx.x >> 5);
  const int64_t from = (int64_t)w * per;
  return {(int)min(from, (int64_t)p.num_pages), (int)min(from + per, (int64_t)p.num_pages)};
}
// Calls what(page of the lane, mask of the lanes whose page is in use) for 32 pages at a time, up to the end of the part (lanes behind it count as in
// use).  Eight groups are on their way together.
template <class What>
__device__ __forceinline__ void over_pages(const Book& p, Part part, What what) {
  const int lane = threadIdx.x & 31;
#pragma unroll 1
  for (int i0 = part.from; i0 < part.to; i0 += 256) {
    int r[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int i = i0 + 32 * k + lane;
      r[k] = i < part.to ? __ldcg(p.refs + i) : 1;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i0 + 32 * k < part.to) what(i0 + 32 * k + lane, __ballot_sync(0xffffffffu, r[k] > 0));
  }
}
__device__ __forceinline__ uint32_t lanes_below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }

struct ResizeParams {
  Book book;
  const int32_t *held, *wanted;
  int32_t* pairs;                    // (B, 2)
  int32_t* granted;                  // (B,), or null
  int32_t* work;                     // B: page written to or -1 (kCopied: is copied), B: entries that lack a page (of a row with a gap -1 - its place), kCluster, num_pages: the free ones, in order
};
__host__ __device__ constexpr int64_t resize_words(int64_t B, int64_t num_pages) { return 2 * B + kCluster + num_pages; }

// A row's lengths, within the table.
struct Lengths {
  int held, wanted;
};
__device__ __forceinline__ Lengths lengths_of(const ResizeParams& p, int b, bool report) {
  Lengths n = {p.held[b], p.wanted[b]};
  const int most = p.book.width * p.book.page_size;
  if (report && (n.held < 0 || n.held > most || n.wanted < 0 || n.wanted > most)) report_bad_index(p.book.status, p.book.epoch, kLengthSite);
  n.held = n.held < 0 ? 0 : (n.held < most ? n.held : most);
  n.wanted = n.wanted < 0 ? 0 : (n.wanted < most ? n.wanted : most);
  return n;
}

// Rows keep the pages of what they hold (held, at most wanted), give back those behind, and get pages for `wanted` tokens.  A row that is about to write
// into a page which other entries name too gets a copy of it (the last of the call's rows keeps the page, if nobody else has it).  A row that has no page
// for some of what it holds keeps what it has.  So does a row whose copy finds no page, and with it the one that was to keep the original: they go on sharing it and do not grow.
__global__ void __launch_bounds__(kThreads) resize_kernel(const __grid_constant__ ResizeParams p) {
  __shared__ int s_first[kRows], s_scan[kWarps + 1];
  const Book& k = p.book;
  const int rank = (int)cluster_rank(), warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row0 = rank * kWarps + warp, step = k.ctas * kWarps;
  int32_t *writes = p.work, *lacks = writes + k.B, *free_of = lacks + k.B, *free_page = free_of + kCluster;
  pdl_wait();
  // ---- what is given back; what is missing
  for (int b = row0; b < k.B; b += step) {
    const Lengths n = lengths_of(p, b, lane == 0);
    const int keep = pages_of(k, min(n.held, n.wanted)), want = pages_of(k, n.wanted), at = fast_div(n.held, k.div_page);
    int32_t* row = k.table + (int64_t)b * k.width;
    int gap = keep, page = -1;                 // first entry without a page among those that hold tokens
#pragma unroll 1
    for (int j1 = 0; j1 < k.width; j1 += 128) {
      int entry[4];                            // (asked for together)
#pragma unroll
      for (int i = 0; i < 4; ++i) entry[i] = j1 + 32 * i + lane < k.width ? row[j1 + 32 * i + lane] : 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j0 = j1 + 32 * i, j = j0 + lane;
        if (j0 >= k.width) break;
        int e = max(page_in(entry[i]), -1);
        if (e >= k.num_pages) {
          report_bad_index(k.status, k.epoch, kTableSite);
          e = -1;
        }
        const bool gone = j >= keep && j < k.width && e >= 0;
        if (gone) atomicSub(k.refs + e, 1);
        if (gone || (e != entry[i] && j < k.width)) row[j] = gone ? -1 : e;
        const uint32_t none = __ballot_sync(0xffffffffu, j < keep && e < 0);
        if (none != 0u && gap == keep) gap = j0 + __ffs(none) - 1;
        // (a row that grows keeps the page its next token goes to)
        if (j0 <= at && at < j0 + 32) page = __shfl_sync(0xffffffffu, e, at & 31);
      }
    }
    // (no page that could be put in a gap has what the row holds there: such a row gets nothing, and is reported; others may have the page its next token would go to)
    const bool into = n.wanted > n.held && n.held != at * k.page_size && page >= 0;
    if (gap < keep && into && p.granted == nullptr && lane == (at & 31)) row[at] = page | kWaits;
    if (lane == 0) {
      writes[b] = gap == keep && into ? page : -1;
      lacks[b] = gap == keep ? max(want - keep, 0) : -1 - gap;
      if (gap < keep) report_bad_index(k.status, k.epoch, kPoolSite);
    }
  }
  meet(k);
  // ---- who gets a copy: all but the last of a page's entries
  for (int b = row0; b < k.B; b += step) {
    const int page = __ldcg(writes + b);
    if (page < 0) continue;
    const int others = __ldcg(k.refs + page) - 1;
    if (others <= 0) continue;
    int earlier = 0;
    for (int i = lane; i < b; i += 32) earlier += (__ldcg(writes + i) & ~kCopied) == page && __ldcg(writes + i) >= 0;
    earlier = __reduce_add_sync(0xffffffffu, earlier);
    if (lane == 0 && earlier < others) {
      writes[b] = page | kCopied;
      ++lacks[b];
    }
  }
  // ---- the free pages, counted
  const Part part = part_of(k);
  int here, before = 0;
  over_pages(k, part, [&](int, uint32_t used) { before += __popc(~used); });
  before = scan_warps(before, s_scan, &here);
  if (threadIdx.x == 0) free_of[rank] = here;
  meet(k);
  // ---- where a row's new pages lie in the list of all that are wanted
  int total, free_pages = 0;
  {
    int mine[kRows / kThreads], sum = 0;
#pragma unroll
    for (int i = 0; i < kRows / kThreads; ++i) {
      const int b = (int)threadIdx.x * (kRows / kThreads) + i;
      mine[i] = b < k.B ? max(__ldcg(lacks + b), 0) : 0;
      sum += mine[i];
    }
    int upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    int at = scan_warps(__shfl_sync(0xffffffffu, upto, 31), s_scan, &total) + upto - sum;
#pragma unroll
    for (int i = 0; i < kRows / kThreads; ++i) {
      s_first[(int)threadIdx.x * (kRows / kThreads) + i] = at;
      at += mine[i];
    }
  }
  for (int r = 0; r < k.ctas; ++r) {
    if (r < rank) before += __ldcg(free_of + r);
    free_pages += __ldcg(free_of + r);
  }
  if (before < total)
    over_pages(k, part, [&](int page, uint32_t used) {
      const int at = before + __popc(~used & ((1u << lane) - 1u));
      if ((used >> lane & 1u) == 0u && at < total) {
        free_page[at] = page;
        k.refs[page] = 1;
      }
      before += __popc(~used);
    });
  meet(k);
  // ---- the rows are filled
  for (int b = row0; b < k.B; b += step) {
    const int writes_to = __ldcg(writes + b), lack_here = __ldcg(lacks + b);
    const bool copies = writes_to >= 0 && (writes_to & kCopied) != 0;
    const Lengths n = lengths_of(p, b, false);
    int32_t* row = k.table + (int64_t)b * k.width;
    // Entries that lack a page lie side by side, up to that of the last token: there is no gap in front of them, and a page that is copied is the last of those that hold tokens.
    const int lacks_here = max(lack_here, 0), from = pages_of(k, n.wanted) - lacks_here, next = s_first[b];
    int got = min(max(free_pages - next, 0), lacks_here), room = lack_here < 0 ? (-1 - lack_here) * k.page_size : got < lacks_here ? (from + got) * k.page_size : n.wanted;
    // (pages run out for all rows behind one, so if a sharer's copy has none, the row that was to keep the original
    // gets none either; what it would write there belongs to both)
    bool refused = copies && got == 0;
    if (total > free_pages && writes_to >= 0 && !copies) {
      bool waits = false;
      for (int i = lane; i < b; i += 32) waits = waits || (__ldcg(writes + i) == (writes_to | kCopied) && s_first[i] >= free_pages);
      refused = __any_sync(0xffffffffu, waits);
    }
    if (refused) {
      // (whoever is not told by `granted` must not write there either)
      if (lane == 0) {
        report_bad_index(k.status, k.epoch, kPoolSite);
        if (p.granted == nullptr) row[fast_div(n.held, k.div_page)] = (writes_to & ~kCopied) | kWaits;
      }
      room = n.held;
    } else if (got < lacks_here && lane == 0) {
      report_bad_index(k.status, k.epoch, kPoolSite);
    }
    for (int i = lane; i < got; i += 32) row[from + i] = __ldcg(free_page + next + i);
    if (lane == 0) {
      const bool done = copies && !refused;
      const int page = writes_to & ~kCopied;
      if (done) atomicSub(k.refs + page, 1);
      p.pairs[2 * b] = done ? page : -1;
      p.pairs[2 * b + 1] = done ? __ldcg(free_page + next) : -1;
      if (p.granted != nullptr) p.granted[b] = room;
    }
  }
}

struct ForkParams {
  Book book;                         // (of the old table)
  const int32_t *held, *parents;
  int32_t *table, *new_held;         // (rows, width), (rows,)
  int rows;
};
constexpr int kForkThreads = 128;

// CTAs 0 .. rows - 1: a new row each; the others: the references of an old row's pages, which change by its children but one.
__global__ void __launch_bounds__(kForkThreads) fork_kernel(const __grid_constant__ ForkParams p) {
  const Book& k = p.book;
  const int tid = threadIdx.x;
  const int64_t most = (int64_t)k.width * k.page_size;
  pdl_wait();
  if ((int)blockIdx.x < p.rows) {
    const int b = blockIdx.x, a = p.parents[b];
    const bool there = a >= 0 && a < k.B;
    if (tid == 0 && !there && a != -1) report_bad_index(k.status, k.epoch, kParentSite);
    int held = there ? p.held[a] : 0;
    if (tid == 0 && (held < 0 || held > most)) report_bad_index(k.status, k.epoch, kLengthSite);
    held = held < 0 ? 0 : (held < most ? held : (int)most);
    const int keep = pages_of(k, held);
    for (int j = tid; j < k.width; j += kForkThreads) {
      const int e = j < keep ? page_in(k.table[(int64_t)a * k.width + j]) : -1;
      p.table[(int64_t)b * k.width + j] = e >= 0 && e < k.num_pages ? e : -1;
    }
    if (tid == 0) p.new_held[b] = held;
    return;
  }
  const int a = (int)blockIdx.x - p.rows;
  __shared__ int s_children;
  if (tid == 0) s_children = 0;
  __syncthreads();
  int mine = 0;
  for (int b = tid; b < p.rows; b += kForkThreads) mine += p.parents[b] == a;
  mine = __reduce_add_sync(0xffffffffu, mine);
  if ((tid & 31) == 0 && mine != 0) atomicAdd(&s_children, mine);
  __syncthreads();
  int held = p.held[a];
  held = held < 0 ? 0 : (held < most ? held : (int)most);
  const int keep = pages_of(k, held), change = s_children - 1;
  for (int j = tid; j < k.width; j += kForkThreads) {
    const int e = page_in(k.table[(int64_t)a * k.width + j]), by = j < keep ? change : -1;
    if (e >= k.num_pages) report_bad_index(k.status, k.epoch, kTableSite);
    else if (e >= 0 && by != 0) atomicAdd(k.refs + e, by);
  }
}

struct CompactParams {
  Book book;
  int32_t* pairs;                    // (num_pages / 2, 2)
  int32_t* used;
  int32_t* work;                     // 3 kCluster, num_pages: where a page went
};
__host__ __device__ constexpr int64_t compact_words(int64_t num_pages) { return 3 * kCluster + num_pages; }

// With `used` pages in use, the i-th of those at `used` or above moves to the i-th free one below.
__global__ void __launch_bounds__(kThreads) compact_kernel(const __grid_constant__ CompactParams p) {
  __shared__ int s_scan[kWarps + 1];
  const Book& k = p.book;
  const int rank = (int)cluster_rank(), lane = threadIdx.x & 31, all = rank * kThreads + threadIdx.x;
  int32_t *live_of = p.work, *holes_of = live_of + kCluster, *movers_of = holes_of + kCluster, *to = movers_of + kCluster;
  pdl_wait();
  const Part part = part_of(k);
  int here, live = 0;
  over_pages(k, part, [&](int page, uint32_t in_use) { live += __popc(in_use & lanes_below(part.to - (page - lane))); });
  scan_warps(live, s_scan, &here);
  if (threadIdx.x == 0) live_of[rank] = here;
  meet(k);
  int used = 0;
  for (int r = 0; r < k.ctas; ++r) used += __ldcg(live_of + r);
  // lanes of a group whose page is free and below `used`; in use and not below
  auto holes_in = [&](int page0, uint32_t in_use) { return ~in_use & lanes_below(used - page0); };
  auto movers_in = [&](int page0, uint32_t in_use) { return in_use & ~lanes_below(used - page0) & lanes_below(part.to - page0); };
  int hole = 0, mover = 0;
  over_pages(k, part, [&](int page, uint32_t in_use) {
    hole += __popc(holes_in(page - lane, in_use));
    mover += __popc(movers_in(page - lane, in_use));
  });
  hole = scan_warps(hole, s_scan, &here);
  if (threadIdx.x == 0) holes_of[rank] = here;
  mover = scan_warps(mover, s_scan, &here);
  if (threadIdx.x == 0) movers_of[rank] = here;
  meet(k);
  int moved = 0;
  for (int r = 0; r < k.ctas; ++r) {
    if (r < rank) {
      hole += __ldcg(holes_of + r);
      mover += __ldcg(movers_of + r);
    }
    moved += __ldcg(movers_of + r);
  }
  const uint32_t in_front = (1u << lane) - 1u;
  over_pages(k, part, [&](int page, uint32_t in_use) {
    const uint32_t holes = holes_in(page - lane, in_use), movers = movers_in(page - lane, in_use);
    if ((holes >> lane & 1u) != 0u) p.pairs[2 * (hole + __popc(holes & in_front)) + 1] = page;
    if ((movers >> lane & 1u) != 0u) p.pairs[2 * (mover + __popc(movers & in_front))] = page;
    else if (page >= used && page < part.to) to[page] = page;
    hole += __popc(holes);
    mover += __popc(movers);
  });
  for (int i = moved + all; i < k.num_pages / 2; i += k.ctas * kThreads) p.pairs[2 * i] = p.pairs[2 * i + 1] = -1;
  if (all == 0) *p.used = used;
  meet(k);
#pragma unroll 4
  for (int i = all; i < moved; i += k.ctas * kThreads) {
    const int from = __ldcg(p.pairs + 2 * i), at = __ldcg(p.pairs + 2 * i + 1);
    k.refs[at] = __ldcg(k.refs + from);
    k.refs[from] = 0;
    to[from] = at;
  }
  meet(k);
  // the table, eight entries of a thread on their way together
  const int64_t entries = (int64_t)k.B * k.width, step = (int64_t)k.ctas * kThreads;
#pragma unroll 1
  for (int64_t i0 = all; i0 < entries; i0 += 8 * step) {
    int e[8], at[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) e[j] = i0 + j * step < entries ? k.table[i0 + j * step] : -1;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int page = page_in(e[j]);
      if (page >= k.num_pages) report_bad_index(k.status, k.epoch, kTableSite);
      at[j] = page >= used && page < k.num_pages ? __ldcg(to + page) : -1;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (at[j] >= 0) k.table[i0 + j * step] = at[j] | (e[j] & kWaits);
  }
}

// ---- copying ------------------------------------------------------------------------------------------------------

// A tensor with a page in every step of its first dimension, as rows of whole pieces (of 16, 4 or 1 bytes).
struct PagedTensor {
  uint8_t* base;
  int64_t page, inner, outer;        // strides, bytes
  int pieces, log_piece;             // of a page
  FastDiv div_row, div_inner;        // pieces of a row; rows side by side along `inner`
  int row, rows_inner;
};
constexpr int kTensors = 8, kCopyThreads = 256, kCopyPieces = 4;
struct CopyParams {
  const int32_t* pairs;
  int n, num_pages;
  int tensors;
  PagedTensor t[kTensors];
  int first[kTensors + 1];           // tasks of a pair that are a tensor's: kCopyThreads * kCopyPieces pieces, or kBulkBytes, each
  FastDiv div_tasks;
  int64_t tasks;                     // n * first[tensors]
  uint32_t* status;
  uint32_t epoch;
  uint64_t budget_ns;
};

template <class T>
__device__ __forceinline__ void copy_pieces(const PagedTensor& t, int from, int to, int i0) {
  T v[kCopyPieces];
  int64_t at[kCopyPieces];
#pragma unroll
  for (int j = 0; j < kCopyPieces; ++j) {
    const int i = i0 + j * kCopyThreads;
    at[j] = -1;
    if (i < t.pieces) {
      const int r = fast_div(i, t.div_row), o = fast_div(r, t.div_inner);
      at[j] = o * t.outer + (r - o * t.rows_inner) * t.inner + (int64_t)(i - r * t.row) * sizeof(T);
      v[j] = *reinterpret_cast<const T*>(t.base + from * t.page + at[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < kCopyPieces; ++j)
    if (at[j] >= 0) *reinterpret_cast<T*>(t.base + to * t.page + at[j]) = v[j];
}

// CTAs take the parts of all pairs in turn.  A warp looks up the pairs of its next 32 parts at a time, so a list that is mostly empty (one pair of many
// rows, or a long tail) costs a memory latency for 32 of them.  what(page from, page to, tensor, part of it) for each, by the whole warp; false: no more.
template <class What>
__device__ __forceinline__ void over_parts(const CopyParams& p, What what) {
  const int lane = threadIdx.x & 31, per = p.first[p.tensors];
  for (int64_t t0 = blockIdx.x; t0 < p.tasks; t0 += 32 * (int64_t)gridDim.x) {
    const int64_t mine = t0 + lane * (int64_t)gridDim.x;
    int2 pages = make_int2(-1, -1);
    int part = 0;
    if (mine < p.tasks) {
      const int pair = fast_div((int)mine, p.div_tasks);
      part = (int)mine - pair * per;
      pages = make_int2(p.pairs[2 * pair], p.pairs[2 * pair + 1]);
      if (pages.x >= 0 && pages.y >= 0 && (pages.x >= p.num_pages || pages.y >= p.num_pages)) {
        report_bad_index(p.status, p.epoch, kPairSite);
        pages.x = -1;
      }
    }
    for (uint32_t todo = __ballot_sync(0xffffffffu, pages.x >= 0 && pages.y >= 0); todo != 0u; todo &= todo - 1u) {
      const int l = __ffs(todo) - 1;
      const int from = __shfl_sync(0xffffffffu, pages.x, l), to = __shfl_sync(0xffffffffu, pages.y, l), at = __shfl_sync(0xffffffffu, part, l);
      int which = 0;
      while (at >= p.first[which + 1]) ++which;
      if (!what(from, to, p.t[which], at - p.first[which])) return;
    }
  }
}

// Through registers: any strides and piece sizes, little to set up.
__global__ void __launch_bounds__(kCopyThreads) copy_kernel(const __grid_constant__ CopyParams p) {
  pdl_wait();
  over_parts(p, [&](int from, int to, const PagedTensor& t, int part) {
    const int i0 = part * (kCopyThreads * kCopyPieces) + threadIdx.x;
    if (t.log_piece == 4) copy_pieces<uint4>(t, from, to, i0);
    else if (t.log_piece == 2) copy_pieces<uint32_t>(t, from, to, i0);
    else copy_pieces<uint8_t>(t, from, to, i0);
    return true;
  });
}

// Through shared memory by bulk copies, for pages that lie in one piece: a warp with a ring of places, of which half are being loaded and half stored.
// HBM bounds it: 2322 pages of 131 KB (609 MB read and written) by itself 103 us, 5.9 TB/s, 90 % of a measured copy (the kernel above 112), behind other work 108.  Rings of 12 places of 16 KB
// or 6 of 32 KB in one CTA an SM 103, of 24 of 8 KB 110.
constexpr int kBulkBytes = 16384, kBulkPlaces = 6, kBulkCtas = 2;      // (CTAs of an SM)
constexpr uint32_t kBulkRequest = kBulkPlaces * kBulkBytes + 128;
__global__ void __launch_bounds__(32) copy_bulk_kernel(const __grid_constant__ CopyParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t s_bar[kBulkPlaces];
  __shared__ uint8_t* s_to[kBulkPlaces];
  __shared__ uint32_t s_bytes[kBulkPlaces];
  __shared__ uint32_t s_abort;
  const uint32_t ring = (smem_u32(smem_raw) + 127u) & ~127u, bars = smem_u32(s_bar);
  const bool lead = threadIdx.x == 0;
  if (lead) {
    s_abort = 0u;
    for (int i = 0; i < kBulkPlaces; ++i) mbar_init(bars + 8 * i, 1);
    fence_barrier_init();
  }
  __syncwarp();
  const WaitCtx wc = {&s_abort, p.status, p.budget_ns, p.epoch};
  int loaded = 0, stored = 0;               // (of the one lane that copies)
  bool ok = true;
  auto store = [&]() {
    const int at = stored % kBulkPlaces;
    ok = mbar_wait(bars + 8 * at, (stored / kBulkPlaces) & 1, wc, kCopySite);
    if (!ok) return;
    bulk_store(s_to[at], ring + at * kBulkBytes, s_bytes[at]);
    bulk_commit_group();
    ++stored;
  };
  pdl_wait();
  over_parts(p, [&](int from, int to, const PagedTensor& t, int part) {
    if (lead) {
      const int64_t off = (int64_t)part * kBulkBytes, rest = (int64_t)t.pieces * 16 - off;
      const int at = loaded % kBulkPlaces;
      // (what lay there is stored: all groups but the newest of those behind it)
      asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kBulkPlaces / 2 - 1) : "memory");
      s_to[at] = t.base + to * t.page + off;
      s_bytes[at] = (uint32_t)(rest < kBulkBytes ? rest : kBulkBytes);
      mbar_arrive_expect_tx(bars + 8 * at, s_bytes[at]);
      bulk_load(ring + at * kBulkBytes, t.base + from * t.page + off, s_bytes[at], bars + 8 * at);
      ++loaded;
      if (loaded - stored > kBulkPlaces / 2) store();
    }
    return __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
  });
  if (lead) {
    while (ok && stored < loaded) store();
    // (where a wait ran out: what is on its way lands before the memory is given back)
    const uint64_t begun = globaltimer_ns();
    for (; stored < loaded; ++stored)
      while (!mbar_try_wait(bars + 8 * (stored % kBulkPlaces), (stored / kBulkPlaces) & 1) && globaltimer_ns() - begun < 50ull * 1000 * 1000) {}
    bulk_wait_group0();
  }
}

}  // namespace pages
}  // namespace fa4
