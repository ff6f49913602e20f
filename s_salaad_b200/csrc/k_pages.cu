// Book-keeping of a paged key-value cache on the device, so that a decode step
// (also one replayed from a graph) never waits for the host: rows that fork,
// end, roll back and grow; pages shared by reference and copied before they
// are written; live pages moved to the lowest page numbers; new tokens'
// keys and values written into their pages.
//
// All of it is bound by latency (a few thousand integers) except the page
// copies, which are bound by HBM: 16-byte loads and stores, several in flight
// per thread, over all layers' K and V at once.  Every choice is made in row
// and page order, so the state never depends on timing; the only atomics are
// integer sums and minima.
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <type_traits>

#include "internal.hpp"

namespace slr {

__device__ unsigned g_status_pages;

namespace {

constexpr int kHeader = SLR_KV_HEADER_WORDS;
enum : int { kShort = 0, kOver = 1, kCopies = 2, kLive = 3 };

struct PagesK {
  int32_t *head, *lens, *refs, *table;
  int rows, num_pages, max_pages, page_size;
  int32_t *growers, *first, *list, *src, *dst;  // workspace
};

__device__ __forceinline__ int64_t pages_of(int64_t len, int page_size) {
  if (len < (int64_t(1) << 31)) return (uint32_t(len) + uint32_t(page_size) - 1) / uint32_t(page_size);  // short division
  return (len + page_size - 1) / page_size;
}

// Length of a row after a change by n < 0 (before any growth).
__device__ __forceinline__ int kept_length(int len, int64_t n) {
  return int(n < 0 ? (len + n < 0 ? 0 : len + n) : len);
}

// A row's length as the state has it, clipped to the table.
__device__ __forceinline__ int checked_length(const PagesK& p, int r, bool* bad) {
  const int64_t cap = int64_t(p.max_pages) * p.page_size;
  const int len = p.lens[r];
  if (len < 0 || len > cap) {
    *bad = true;
    return int(len < 0 ? 0 : cap);
  }
  return len;
}

// The row that row r becomes a copy of; -1: empty.
__device__ __forceinline__ int checked_parent(const PagesK& p, const int32_t* parents, int r, bool* bad) {
  const int from = parents ? parents[r] : r;
  if (from >= p.rows) *bad = true;
  return from >= p.rows || from < 0 ? -1 : from;
}

// What a selection does, in shared memory.
struct Selection {
  int32_t* old;       // [rows][columns of a step] table entries before
  int32_t* len;       // [rows] lengths before
  int32_t* from;      // [rows] parents
  int32_t* children;  // [rows]
  int32_t* keep;      // [rows] entries of the parent that stay
};
constexpr int kSelectionWords = 4;  // words per row besides `old`
template <int kC> __device__ __forceinline__ Selection selection_at(int32_t* sm, int rows) {
  Selection s;
  s.old = sm;
  s.len = s.old + rows * kC;
  s.from = s.len + rows;
  s.children = s.from + rows;
  s.keep = s.children + rows;
  return s;
}

// Reads lengths and parents and counts children; the greatest length in
// *s_most (0 before).  Ends with a barrier.
__device__ __forceinline__ void read_selection(const PagesK& p, const int32_t* parents, const int32_t* n_new, int n_all,
                                               const Selection& s, int* s_most, bool report) {
  const int tid = threadIdx.x;
  bool bad = false;
  int most = 0;
  for (int r = tid; r < p.rows; r += blockDim.x) {
    s.from[r] = checked_parent(p, parents, r, &bad);
    s.len[r] = checked_length(p, r, &bad);
    s.children[r] = 0;
    s.keep[r] = n_new ? n_new[r] : n_all;  // the change of length, for a moment
    most = max(most, s.len[r]);
  }
  __syncthreads();
  most = __reduce_max_sync(0xffffffffu, most);
  if ((tid & 31) == 0) atomicMax(s_most, most);
  for (int r = tid; r < p.rows; r += blockDim.x) {
    const int f = s.from[r];
    if (f >= 0) atomicAdd(s.children + f, 1);
    s.keep[r] = f < 0 ? 0 : int(pages_of(kept_length(s.len[f], s.keep[r]), p.page_size));
  }
  if (bad && report) atomicOr(&g_status_pages, SLR_BAD_INDEX_BIT);
  __syncthreads();
}

template <int kC> __device__ __forceinline__ int table_entry(const PagesK& p, int c0, int i) {
  const int c = c0 + i % kC;
  return c < p.max_pages ? p.table[int64_t(i / kC) * p.max_pages + c] : -1;
}

// Columns [c0, c0 + kC) of all rows, once `old` holds them: table rows become
// their parents' rows, entries behind the kept length -1.  Columns are
// independent, so this works in place.  refs follow by integer atomics, per
// parent: its pages gain (children - 1) references, nothing where a row merely
// moves, and each child loses those behind its kept length.  Returns this
// thread's change of the number of live pages.
template <int kC>
__device__ __forceinline__ int select_columns(const PagesK& p, const Selection& s, int c0) {
  int live = 0;
  auto refer = [&](int page, int change) {
    if (page < 0) return;
    if (page >= p.num_pages) {
      atomicOr(&g_status_pages, SLR_BAD_INDEX_BIT);
      return;
    }
    // a page is live while its count is above 0: the crossings add up to the net change
    const int was = atomicAdd(p.refs + page, change);
    live += int(was + change > 0) - int(was > 0);
  };
#pragma unroll 4
  for (int i = threadIdx.x; i < p.rows * kC; i += blockDim.x) {
    const int r = i / kC, j = i % kC, c = c0 + j;
    if (c >= p.max_pages) continue;
    const int was = s.old[i], f = s.from[r];
    if (s.children[r] != 1) refer(was, s.children[r] - 1);
    int now = -1;
    if (f >= 0) {
      now = s.old[f * kC + j];
      if (c >= s.keep[r]) {
        refer(now, -1);
        now = -1;
      }
    }
    if (was != now) p.table[int64_t(r) * p.max_pages + c] = now;
  }
  return live;
}

// Adds the threads' changes to the header.
__device__ __forceinline__ void add_live(const PagesK& p, int live, int* s_live) {
  live = __reduce_add_sync(0xffffffffu, live);
  if ((threadIdx.x & 31) == 0 && live) atomicAdd(s_live, live);
  __syncthreads();
  if (threadIdx.x == 0 && *s_live) atomicAdd(p.head + kLive, *s_live);
}

// A selection over a large table: few columns per CTA, all read at once, since
// latency is the bound (250 rows x 120 pages: 32 columns and two atomics per
// entry took 54 us, 4 columns 11).
constexpr int kCols = 4;
constexpr int kEarly = 4;  // entries that a thread reads before the lengths are known
__global__ void __launch_bounds__(256) select_kernel(const PagesK p, const int32_t* parents, const int32_t* n_new,
                                                     int n_all) {
  extern __shared__ int32_t sm[];
  const Selection s = selection_at<kCols>(sm, p.rows);
  __shared__ int s_most, s_live;
  const int tid = threadIdx.x, c0 = blockIdx.x * kCols;
  pdl_wait_primary();
  pdl_launch_dependents();
  int early[kEarly];
#pragma unroll
  for (int k = 0; k < kEarly; ++k) {
    const int i = k * int(blockDim.x) + tid;
    early[k] = i < p.rows * kCols ? table_entry<kCols>(p, c0, i) : -1;
  }
  if (tid == 0) s_most = 0, s_live = 0;
  read_selection(p, parents, n_new, n_all, s, &s_most, blockIdx.x == 0);
  // no row has an entry from here on: there is nothing to move or to drop
  if (c0 >= pages_of(s_most, p.page_size)) return;
#pragma unroll
  for (int k = 0; k < kEarly; ++k) {
    const int i = k * int(blockDim.x) + tid;
    if (i < p.rows * kCols) s.old[i] = early[k];
  }
#pragma unroll 4
  for (int i = kEarly * int(blockDim.x) + tid; i < p.rows * kCols; i += blockDim.x)
    s.old[i] = table_entry<kCols>(p, c0, i);
  __syncthreads();
  add_live(p, select_columns<kCols>(p, s, c0), &s_live);
}

constexpr int kGrowThreads = 1024;
constexpr int kListed = 2048;  // pages given out in one call that are listed in shared memory
constexpr int kPer = 8;  // pages of a thread in one step of a scan over refs

// Exclusive scan over the block; *total: the sum.  `sums`: 32 words of shared
// memory that no other thread still reads.  Ends with a barrier.
template <typename I> __device__ __forceinline__ I block_scan(I v, I* sums, I* total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  I incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const I up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) sums[w] = incl;
  __syncthreads();
  const I mine = sums[lane];
  I all = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const I up = __shfl_up_sync(0xffffffffu, all, o);
    if (lane >= o) all += up;
  }
  *total = __shfl_sync(0xffffffffu, all, 31);
  const I before = __shfl_sync(0xffffffffu, all - mine, w);
  __syncthreads();
  return before + incl - v;
}

// Bit j: page i0 + j is free.
__device__ __forceinline__ unsigned free_mask(const PagesK& p, int64_t i0) {
  unsigned mask = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j)
    if (i0 + j < p.num_pages && __ldcg(p.refs + i0 + j) == 0) mask |= 1u << j;
  return mask;
}

// Growth of every row, by one CTA.  Pages are given out lowest number first in
// row order, a row's copy of a shared last page before its new pages.  Bound
// by the latency of its chain of reads (lens and parents, table, refs).
// before: the selection when it was made in this kernel, else null.  What
// other CTAs of the cluster have written is read past L1.
__device__ __forceinline__ void grow_rows(const PagesK& p, const int32_t* parents, const int32_t* n_new, int n_all,
                                          int32_t* sm, const Selection* before) {
  int32_t* low = sm;              // [rows] kept lengths
  int32_t* start = low + p.rows;  // [rows + 1] pages given to the rows before
  int32_t* copy = start + p.rows + 1;
  __shared__ int64_t sums64[32];
  __shared__ int sums[32];
  __shared__ int s_over, s_list[kListed];
  const int tid = threadIdx.x;
  const unsigned first_free = free_mask(p, int64_t(tid) * kPer);  // read early: most calls need no more
  if (tid == 0) s_over = 0;
  const int64_t cap = int64_t(p.max_pages) * p.page_size;
  bool bad = false;
  auto grow_of = [&](int r) -> int64_t {
    const int64_t n = n_new ? n_new[r] : n_all;
    return n <= 0 || (!n_new && low[r] == 0) ? 0 : n;  // one number for all: rows that hold tokens
  };
  if (!before) {
    // lens and parents are read side by side; start holds the lengths before for a moment
    for (int r = tid; r < p.rows; r += kGrowThreads) {
      copy[r] = checked_parent(p, parents, r, &bad);
      start[r] = checked_length(p, r, &bad);
    }
    __syncthreads();
  }
  const int32_t* from = before ? before->from : copy;
  const int32_t* len = before ? before->len : start;
  for (int r = tid; r < p.rows; r += kGrowThreads)
    low[r] = from[r] < 0 ? 0 : kept_length(len[from[r]], n_new ? n_new[r] : n_all);
  __syncthreads();
  // rows about to write into a shared last page
  auto shared_last = [&](int r) -> int {
    if (grow_of(r) == 0 || low[r] % p.page_size == 0) return -1;
    const int last = __ldcg(p.table + int64_t(r) * p.max_pages + low[r] / p.page_size);
    if (last < 0 || last >= p.num_pages) {
      bad = true;
      return -1;
    }
    return __ldcg(p.refs + last) > 1 ? last : -1;
  };
  bool any = false;
  for (int r = tid; r < p.rows; r += kGrowThreads) {
    const int last = shared_last(r);
    copy[r] = last;
    if (last >= 0) p.growers[last] = 0, p.first[last] = INT_MAX, any = true;
    if (low[r] + grow_of(r) > cap) atomicAdd(&s_over, 1);
  }
  any = __syncthreads_or(any);
  if (any) {
    for (int r = tid; r < p.rows; r += kGrowThreads)
      if (copy[r] >= 0) {
        atomicAdd(p.growers + copy[r], 1);
        atomicMin(p.first + copy[r], r);
      }
    __syncthreads();
  }
  // when every sharer grows, the lowest row keeps the page
  const int chunk = (p.rows + kGrowThreads - 1) / kGrowThreads;
  const int r0 = min(p.rows, tid * chunk), r1 = min(p.rows, r0 + chunk);
  int64_t mine = 0;
  auto need_of = [&](int r) -> int64_t {
    return pages_of(low[r] + grow_of(r), p.page_size) - pages_of(low[r], p.page_size) + (copy[r] >= 0 ? 1 : 0);
  };
  for (int r = r0; r < r1; ++r) {
    if (copy[r] >= 0 && __ldcg(p.growers + copy[r]) == __ldcg(p.refs + copy[r]) && __ldcg(p.first + copy[r]) == r) copy[r] = -1;
    mine += need_of(r);
  }
  int64_t total = 0;
  int64_t at = block_scan(mine, sums64, &total);
  const int over = s_over;
  bool fits = over == 0 && total <= p.num_pages;
  if (fits)
    for (int r = r0; r < r1; ++r) {
      start[r] = int(at);
      at += need_of(r);
    }
  if (tid == 0) start[p.rows] = fits ? int(total) : 0;
  // the lowest `total` free pages
  int64_t found = 0;
  if (total > 0) {
    for (int64_t base = 0; base < p.num_pages && (found < total || !fits); base += kGrowThreads * kPer) {
      const int64_t i0 = base + tid * kPer;
      const unsigned mask = base ? free_mask(p, i0) : first_free;
      int sum = 0;
      int64_t k = found + block_scan(__popc(mask), sums, &sum);
      if (fits && k < total)
        for (int j = 0; j < kPer; ++j)
          if (mask >> j & 1u) {
            if (k < total) (k < kListed ? s_list[k] : p.list[k]) = int32_t(i0 + j);
            ++k;
          }
      found += sum;
    }
  }
  fits = fits && found >= total;
  __syncthreads();
  if (bad) atomicOr(&g_status_pages, SLR_BAD_INDEX_BIT);
  if (fits) {
    for (int k = tid; k < total; k += kGrowThreads) {
      int lo = 0, hi = p.rows - 1;  // the last row that starts at or before k and takes a page
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (start[mid] <= k) lo = mid;
        else hi = mid - 1;
      }
      const int r = lo, page = k < kListed ? s_list[k] : p.list[k];
      int j = k - start[r] - (copy[r] >= 0 ? 1 : 0);
      const int64_t col = pages_of(low[r], p.page_size) + j;  // j == -1: the copied page
      p.table[int64_t(r) * p.max_pages + col] = page;
      p.refs[page] = 1;
    }
    // the copies, in row order
    int copies = 0, n_mine = 0;
    for (int r = r0; r < r1; ++r) n_mine += copy[r] >= 0;
    int c = any ? block_scan(n_mine, sums, &copies) : 0;
    for (int r = r0; r < r1; ++r)
      if (copy[r] >= 0) {
        p.src[c] = copy[r];
        p.dst[c] = start[r] < kListed ? s_list[start[r]] : p.list[start[r]];
        ++c;
        atomicAdd(p.refs + copy[r], -1);  // another row keeps it
      }
    for (int r = tid; r < p.rows; r += kGrowThreads) p.lens[r] = int(low[r] + grow_of(r));
    if (tid == 0) {
      p.head[kShort] = 0;
      p.head[kOver] = 0;
      p.head[kCopies] = copies;
      atomicAdd(p.head + kLive, int(total));
    }
  } else {
    for (int r = tid; r < p.rows; r += kGrowThreads) p.lens[r] = low[r];
    if (tid == 0) {
      p.head[kShort] = int(max(int64_t(0), min(int64_t(INT_MAX), total - found)));
      p.head[kOver] = over;
      p.head[kCopies] = 0;
    }
  }
}

__global__ void __launch_bounds__(kGrowThreads, 1) grow_kernel(const PagesK p, const int32_t* parents,
                                                               const int32_t* n_new, int n_all) {
  extern __shared__ int32_t sm[];
  pdl_wait_primary();
  pdl_launch_dependents();
  grow_rows(p, parents, n_new, n_all, sm, nullptr);
}

// Selection and growth of a small table in one launch: a cluster of CTAs takes
// the columns in turn, kStepCols at a time, then its first one grows the rows.
// A decode step's calls are bound by the host: one launch less makes this call
// 2.3 us shorter there (on the GPU both take the same).
constexpr int kStepCols = 16, kStepCtas = 8;
constexpr int kStepRows = 512, kStepPages = 512;  // at most: four steps of 8 entries per thread
__global__ void __launch_bounds__(kGrowThreads, 1) step_kernel(const PagesK p, const int32_t* parents,
                                                               const int32_t* n_new, int n_all) {
  extern __shared__ int32_t sm[];
  const Selection s = selection_at<kStepCols>(sm, p.rows);
  __shared__ int s_most, s_live;
  const int tid = threadIdx.x;
  pdl_wait_primary();
  pdl_launch_dependents();
  int early[kEarly];  // of this CTA's first columns, read beside the lengths
#pragma unroll
  for (int k = 0; k < kEarly; ++k) {
    const int i = k * kGrowThreads + tid;
    early[k] = i < p.rows * kStepCols ? table_entry<kStepCols>(p, blockIdx.x * kStepCols, i) : -1;
  }
  if (tid == 0) s_most = 0, s_live = 0;
  __syncthreads();
  read_selection(p, parents, n_new, n_all, s, &s_most, blockIdx.x == 0);
  int live = 0;
  const int used = int(pages_of(s_most, p.page_size));
  for (int c0 = blockIdx.x * kStepCols; c0 < used; c0 += kStepCtas * kStepCols) {
    int done = 0;
    if (c0 == int(blockIdx.x) * kStepCols) {
#pragma unroll
      for (int k = 0; k < kEarly; ++k) {
        const int i = k * kGrowThreads + tid;
        if (i < p.rows * kStepCols) s.old[i] = early[k];
      }
      done = kEarly * kGrowThreads;
    }
#pragma unroll 4
    for (int i = done + tid; i < p.rows * kStepCols; i += kGrowThreads) s.old[i] = table_entry<kStepCols>(p, c0, i);
    __syncthreads();
    live += select_columns<kStepCols>(p, s, c0);
    __syncthreads();
  }
  add_live(p, live, &s_live);
  cooperative_groups::this_cluster().sync();
  if (blockIdx.x == 0) grow_rows(p, parents, n_new, n_all, s.old, &s);
}

// Plan of a compaction: one CTA.  Live pages from the live count on go to the
// free numbers below it, both ascending: no page is both read and written.
__global__ void __launch_bounds__(kGrowThreads, 1) compact_plan_kernel(const PagesK p) {
  __shared__ unsigned long long sums[32];
  __shared__ int s_live;
  const int tid = threadIdx.x;
  pdl_wait_primary();
  pdl_launch_dependents();
  if (tid == 0) s_live = 0;
  __syncthreads();
  const unsigned first_free = free_mask(p, int64_t(tid) * kPer);
  int mine = 0;
  for (int64_t i0 = int64_t(tid) * kPer; i0 < p.num_pages; i0 += kGrowThreads * kPer) {
    const unsigned f = i0 == int64_t(tid) * kPer ? first_free : free_mask(p, i0);
    mine += int(min(int64_t(kPer), p.num_pages - i0)) - __popc(f);
  }
  mine = __reduce_add_sync(0xffffffffu, mine);
  if ((tid & 31) == 0) atomicAdd(&s_live, mine);
  __syncthreads();
  const int64_t live = s_live;
  int64_t holes = 0, movers = 0;
  for (int64_t base = 0; base < p.num_pages; base += kGrowThreads * kPer) {
    const int64_t i0 = base + tid * kPer;
    const unsigned f = base ? free_mask(p, i0) : first_free;
    // bits of the pages below the live count, and of those that exist
    const int64_t n_low = live - i0, n_in = p.num_pages - i0;
    const unsigned low = n_low <= 0 ? 0u : n_low >= kPer ? 0xffu : (1u << n_low) - 1;
    const unsigned in = n_in <= 0 ? 0u : n_in >= kPer ? 0xffu : (1u << n_in) - 1;
    const unsigned hole = f & low, mover = ~f & ~low & in;
    for (unsigned rest = ~low & in; rest; rest &= rest - 1) p.first[i0 + __ffs(rest) - 1] = -1;
    // both counts in one scan
    unsigned long long sum = 0;
    const unsigned long long at =
        block_scan(static_cast<unsigned long long>(__popc(hole)) << 32 | __popc(mover), sums, &sum);
    int64_t h = holes + int64_t(at >> 32), m = movers + int64_t(at & 0xffffffffu);
    for (int j = 0; j < kPer; ++j) {
      if (hole >> j & 1u) p.dst[h++] = int32_t(i0 + j);
      if (mover >> j & 1u) p.src[m++] = int32_t(i0 + j);
    }
    holes += int64_t(sum >> 32);
    movers += int64_t(sum & 0xffffffffu);
  }
  __syncthreads();
  for (int64_t i = tid; i < movers; i += kGrowThreads) {
    const int s = p.src[i], d = p.dst[i];
    p.refs[d] = p.refs[s];
    p.refs[s] = 0;
    p.first[s] = d;
  }
  if (tid == 0) {
    p.head[kShort] = 0;
    p.head[kOver] = 0;
    p.head[kCopies] = int(movers);
    p.head[kLive] = int(live);
  }
}

struct CopyK {
  uint8_t *k, *v;
  int64_t layer_bytes, page_stride, page_bytes;
  int planes, num_pages;
  const int32_t *src, *dst;
  const int32_t* count;  // device word, or null: n
  int n;
  bool check;            // pairs from the caller: those that could clash are left out
  int32_t* table;        // compaction: entries to rewrite through `to`, or null
  const int32_t* to;
  const int32_t* live;
  int64_t entries;
};

constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 4;
// CTAs per SM of a copy that is known to be long: dealt by the hardware as SMs
// come free (6000 pages, 3/5 live: 8 per SM, each with a fixed share, 275 us,
// 24: 258, 64: 252).  Copies that are mostly empty keep to one wave of 8.
constexpr int kManyCtas = 64;

// Pages src[i] -> dst[i] of every plane.  An item is a piece of one page of
// one plane; CTAs take the items in turn.
__global__ void __launch_bounds__(kCopyThreads) copy_kernel(const CopyK a) {
  using Vec = uint4;  // a page's bytes are a multiple of 16
  pdl_wait_primary();
  const int tid = threadIdx.x;
  if (a.table) {
    const int live = *a.live;
    for (int64_t i = int64_t(blockIdx.x) * kCopyThreads + tid; i < a.entries; i += int64_t(gridDim.x) * kCopyThreads) {
      const int e = a.table[i];
      if (e < live) continue;
      const int d = e < a.num_pages ? a.to[e] : -1;
      if (d >= 0) a.table[i] = d;
      else atomicOr(&g_status_pages, SLR_BAD_INDEX_BIT);
    }
  }
  const int n = a.count ? *a.count : a.n;
  constexpr int64_t kPiece = int64_t(kCopyThreads) * kCopyUnroll * sizeof(Vec);
  const int64_t pieces = (a.page_bytes + kPiece - 1) / kPiece;
  const int64_t per_pair = pieces * a.planes;
  int last = -1;
  bool ok = true;
  for (int64_t item = blockIdx.x; item < per_pair * n; item += gridDim.x) {
    const int pair = int(item / per_pair);
    const int64_t rest = item % per_pair;
    const int plane = int(rest / pieces);
    const int64_t off = (rest % pieces) * kPiece;
    const int s = a.src[pair], d = a.dst[pair];
    if (a.check && pair != last) {
      last = pair;
      bool clash = uint32_t(s) >= uint32_t(a.num_pages) || uint32_t(d) >= uint32_t(a.num_pages);
      for (int i = tid; i < n; i += kCopyThreads) {
        const int si = a.src[i], di = a.dst[i];
        if (i != pair && si != di && s != d && (di == d || di == s || si == d)) clash = true;
      }
      ok = !__syncthreads_or(clash);
      if (!ok && tid == 0) atomicOr(&g_status_pages, SLR_BAD_INDEX_BIT);
    }
    if (!ok || s == d) continue;
    uint8_t* plane_base = ((plane & 1) ? a.v : a.k) + int64_t(plane >> 1) * a.layer_bytes;
    const uint8_t* from = plane_base + int64_t(s) * a.page_stride + off;
    uint8_t* to = plane_base + int64_t(d) * a.page_stride + off;
    const int64_t left = a.page_bytes - off;
    Vec x[kCopyUnroll];
#pragma unroll
    for (int i = 0; i < kCopyUnroll; ++i) {
      const int64_t at = (int64_t(i) * kCopyThreads + tid) * int64_t(sizeof(Vec));
      if (at < left) x[i] = *reinterpret_cast<const Vec*>(from + at);
    }
#pragma unroll
    for (int i = 0; i < kCopyUnroll; ++i) {
      const int64_t at = (int64_t(i) * kCopyThreads + tid) * int64_t(sizeof(Vec));
      if (at < left) *reinterpret_cast<Vec*>(to + at) = x[i];
    }
  }
}

constexpr int kAppendThreads = 64;  // 48k tokens of 8 heads of 128: 35.9 us, with 128 threads 36.6, with 512 41.5
// New tokens into their pages: one warp per token, 16-byte chunks (V = 16) or
// single elements where the caller's rows are not aligned (V = element size).
template <int V>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const AppendArgs a, int esize) {
  pdl_wait_primary();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t token = int64_t(blockIdx.x) * (kAppendThreads / 32) + (threadIdx.x >> 5);
  if (token >= a.tokens) return;
  int row = int(token);
  int64_t pos;
  if (a.cu) {
    // 32-ary search for the last row that starts at or before the token
    int lo = 0, hi = a.rows;  // cu[lo] <= token < cu[hi] (cu[rows] = all tokens)
    if (token >= a.cu[a.rows] || token < a.cu[0]) return;  // behind the last row
    while (hi - lo > 1) {
      const int step = (hi - lo + 31) / 32;
      const int at = lo + lane * step;
      const unsigned below = __ballot_sync(0xffffffffu, at < hi && a.cu[at] <= token);
      const int k = below ? 31 - __clz(below) : 0;
      const int nlo = lo + k * step;
      hi = min(hi, nlo + step);
      lo = nlo;
    }
    row = lo;
    pos = int64_t(a.lens[row]) - (a.cu[row + 1] - token);
    if (pos < 0) {
      if (lane == 0) atomicOr(&g_status_pages, SLR_BAD_INDEX_BIT);
      return;
    }
  } else {
    pos = int64_t(a.lens[row]) - 1;
    if (pos < 0) return;  // an empty row
  }
  if (pos >= int64_t(a.max_pages) * a.page_size) {
    if (lane == 0) atomicOr(&g_status_pages, SLR_BAD_INDEX_BIT);
    return;
  }
  const int page = a.table[int64_t(row) * a.max_pages + pos / a.page_size];
  if (page < 0 || page >= a.num_pages) {
    if (lane == 0) atomicOr(&g_status_pages, SLR_BAD_INDEX_BIT);
    return;
  }
  const int64_t base = int64_t(page) * a.page_stride + (pos % a.page_size) * a.token_stride;
  const int E = V / esize;
  const int chunks = a.dim / E, all = a.kv_heads * chunks;
  using Vec = std::conditional_t<V == 16, uint4, std::conditional_t<V == 4, uint32_t, unsigned short>>;
  const uint8_t* nk = static_cast<const uint8_t*>(a.new_k);
  const uint8_t* nv = static_cast<const uint8_t*>(a.new_v);
  uint8_t* pk = static_cast<uint8_t*>(a.k);
  uint8_t* pv = static_cast<uint8_t*>(a.v);
#pragma unroll 4
  for (int i = lane; i < all; i += 32) {
    const int h = i / chunks, d = (i - h * chunks) * E;
    const int64_t dst = (base + h * a.head_stride + d) * esize;
    const Vec x = *reinterpret_cast<const Vec*>(nk + (token * a.k_row + h * a.k_head + d) * esize);
    const Vec y = *reinterpret_cast<const Vec*>(nv + (token * a.v_row + h * a.v_head + d) * esize);
    *reinterpret_cast<Vec*>(pk + dst) = x;
    *reinterpret_cast<Vec*>(pv + dst) = y;
  }
}

// A launch that may start while the kernel before it ends; every kernel here
// waits for that one (griddepcontrol.wait) before it reads anything.
template <typename... P, typename... A>
int launch_after(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t s, const A&... args) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(unsigned(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  SLR_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kernel, P(args)...));
  return SLR_OK;
}

// The device's SMs; on the first call for a device also its kernels' limits
// (the same for every caller and size).
int prepare_device(int* sms) {
  constexpr int kDevices = 32;
  static std::atomic<int> known[kDevices];
  int dev = 0;
  SLR_CHECK_CUDA(cudaGetDevice(&dev));
  int n = dev < kDevices ? known[dev].load(std::memory_order_acquire) : 0;
  if (!n) {
    SLR_CHECK_CUDA(cudaFuncSetAttribute(select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        kAttendMaxRows * (kCols + kSelectionWords) * 4));
    SLR_CHECK_CUDA(cudaFuncSetAttribute(step_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        kStepRows * (kStepCols + kSelectionWords) * 4));
    SLR_CHECK_CUDA(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
    if (dev < kDevices) known[dev].store(n, std::memory_order_release);
  }
  *sms = n;
  return SLR_OK;
}

PagesK views(const PagesArgs& p) {
  PagesK k = {};
  k.head = p.state;
  k.lens = k.head + kHeader;
  k.refs = k.lens + p.rows;
  k.table = k.refs + p.num_pages;
  k.rows = p.rows;
  k.num_pages = p.num_pages;
  k.max_pages = p.max_pages;
  k.page_size = p.page_size;
  int32_t* w = static_cast<int32_t*>(p.workspace);
  const int64_t pages = p.num_pages, pairs = std::max(p.rows, p.num_pages);
  k.growers = w;
  k.first = w + pages;
  k.list = w + 2 * pages;
  k.src = w + 3 * pages;
  k.dst = w + 3 * pages + pairs;
  return k;
}

int copy_launch(const PagesArgs& p, CopyK c, int64_t most_pairs, int64_t ctas, cudaStream_t s) {
  c.k = p.k;
  c.v = p.v;
  c.layer_bytes = p.layer_bytes;
  c.page_stride = p.page_stride_bytes;
  c.page_bytes = p.page_bytes;
  c.planes = 2 * p.layers;
  c.num_pages = p.num_pages;
  const int64_t pieces = ceil_div(p.page_bytes, int64_t(kCopyThreads) * kCopyUnroll * int64_t(sizeof(uint4)));
  const int64_t items = std::max<int64_t>(1, pieces * c.planes * most_pairs);
  return launch_after(copy_kernel, dim3(unsigned(std::min(items, ctas))), kCopyThreads, 0, s, c);
}

}  // namespace

size_t kv_pages_workspace_size(int rows, int num_pages) {
  return size_t(4) * (3 * size_t(num_pages) + 2 * size_t(std::max(rows, num_pages)));
}

int launch_kv_advance(const PagesArgs& p, const int32_t* n_new, int n_all, const int32_t* parents, cudaStream_t s) {
  const PagesK k = views(p);
  int sms = 0;
  int rc = prepare_device(&sms);
  if (rc) return rc;
  const bool select = parents || n_new || n_all < 0;
  if (select && p.rows <= kStepRows && p.max_pages <= kStepPages) {
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = kStepCtas;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(kStepCtas);
    cfg.blockDim = dim3(kGrowThreads);
    cfg.dynamicSmemBytes = size_t(p.rows) * (kStepCols + kSelectionWords) * 4;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    SLR_CHECK_CUDA(cudaLaunchKernelEx(&cfg, step_kernel, k, parents, n_new, n_all));
    CopyK c = {};
    c.src = k.src;
    c.dst = k.dst;
    c.count = k.head + kCopies;
    return copy_launch(p, c, p.rows, 8 * sms, s);
  }
  if (select) {
    const size_t smem = size_t(p.rows) * (kCols + kSelectionWords) * 4;
    rc = launch_after(select_kernel, dim3(unsigned(ceil_div(p.max_pages, kCols))), 256, smem, s, k, parents,
                                n_new, n_all);
    if (rc) return rc;
  }
  const size_t smem = (3 * size_t(p.rows) + 1) * 4;
  rc = launch_after(grow_kernel, dim3(1), kGrowThreads, smem, s, k, parents, n_new, n_all);
  if (rc) return rc;
  CopyK c = {};
  c.src = k.src;
  c.dst = k.dst;
  c.count = k.head + kCopies;
  return copy_launch(p, c, p.rows, 8 * sms, s);
}

int launch_kv_compact(const PagesArgs& p, cudaStream_t s) {
  const PagesK k = views(p);
  int sms = 0;
  int rc = prepare_device(&sms);
  if (rc) return rc;
  rc = launch_after(compact_plan_kernel, dim3(1), kGrowThreads, 0, s, k);
  if (rc) return rc;
  CopyK c = {};
  c.src = k.src;
  c.dst = k.dst;
  c.count = k.head + kCopies;
  c.table = k.table;
  c.to = k.first;
  c.live = k.head + kLive;
  c.entries = int64_t(p.rows) * p.max_pages;
  return copy_launch(p, c, std::max<int64_t>(p.num_pages / 2, ceil_div(c.entries, 1024)),
                     kManyCtas * sms, s);
}

int launch_kv_copy(const PagesArgs& p, const int32_t* src, const int32_t* dst, int n, cudaStream_t s) {
  int sms = 0;
  const int rc = prepare_device(&sms);
  if (rc) return rc;
  CopyK c = {};
  c.src = src;
  c.dst = dst;
  c.n = n;
  c.check = true;
  return copy_launch(p, c, n, kManyCtas * sms, s);
}

int launch_kv_append(const AppendArgs& a, cudaStream_t s) {
  const int e = int(dtype_size(a.dtype));
  const auto even = [&](int64_t stride) { return stride * e % 16 == 0; };
  const bool wide = aligned16(a.new_k) && aligned16(a.new_v) && even(a.k_row) && even(a.k_head) && even(a.v_row) &&
                    even(a.v_head) && a.dim * e % 16 == 0;
  const dim3 grid(unsigned(ceil_div(a.tokens, kAppendThreads / 32)));
  if (wide) return launch_after(append_kernel<16>, grid, kAppendThreads, 0, s, a, e);
  if (e == 4) return launch_after(append_kernel<4>, grid, kAppendThreads, 0, s, a, e);
  return launch_after(append_kernel<2>, grid, kAppendThreads, 0, s, a, e);
}

int read_and_clear_status_pages(unsigned* out) {
  unsigned v = 0, zero = 0;
  SLR_CHECK_CUDA(cudaMemcpyFromSymbol(&v, g_status_pages, sizeof(v)));
  if (v) SLR_CHECK_CUDA(cudaMemcpyToSymbol(g_status_pages, &zero, sizeof(zero)));
  *out = v;
  return SLR_OK;
}

}  // namespace slr
