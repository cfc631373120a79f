// The pages of a key-value cache: copying, reserving, forking, freeing and compacting, on the device.
//
// State, all in device memory and without a copy on the host: the block table that the attention reads (-1 behind the pages of a
// row), the lengths of its rows, and per page the number of rows that hold it (0: free).  A call that needs pages takes the free ones
// in ascending order, in the order of its rows or entries, so that the tables are the same whatever the scheduling.
//
// A call is a planning kernel, one CTA that reads the tables (16 KB for 4096 pages: latencies, not bytes, are its time), and where data
// move a copying kernel that is launched with it, sets itself up under it and reads its plan.  The copying kernel is bound by
// memory: every byte is read and written once.
#include <algorithm>

#include "common.h"
#define FA_WAIT_INLINE
#include "ptx.cuh"

namespace fa {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWarps = kPlanThreads / 32;

// A page to copy; bytes: from its beginning
struct PageMove {
  int src, dst;
  int64_t bytes;
};

// Exclusive sum over the threads of the block, and the total
__device__ __forceinline__ int block_scan(int x, int& total) {
  __shared__ int warp_sums[kPlanWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int sum = x;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int other = __shfl_up_sync(0xffffffffu, sum, off);
    if (lane >= off) sum += other;
  }
  __syncthreads();  // the sums of the call before have been read
  if (lane == 31) warp_sums[warp] = sum;
  __syncthreads();
  const int w = warp_sums[lane];  // 32 warps
  int before = lane < warp ? w : 0;
  total = __reduce_add_sync(0xffffffffu, w);
  before = __reduce_add_sync(0xffffffffu, before);
  return before + sum - x;
}
static_assert(kPlanWarps == 32, "a lane per warp");

// The first `want` free pages in ascending order into `list`; how many there were, at most `want` (exact when fewer).
constexpr int kPagesPerThread = 4;
__device__ __forceinline__ int find_free(const int* refs, int num_pages, int want, int* list) {
  int found = 0;
  for (int base = 0; base < num_pages && found < want; base += kPlanThreads * kPagesPerThread) {
    const int first = base + threadIdx.x * kPagesPerThread;
    bool is_free[kPagesPerThread];
    int mine = 0;
#pragma unroll
    for (int i = 0; i < kPagesPerThread; ++i) {
      is_free[i] = first + i < num_pages && refs[first + i] <= 0;
      mine += is_free[i];
    }
    int total, at = block_scan(mine, total);
    at += found;
#pragma unroll
    for (int i = 0; i < kPagesPerThread; ++i) {
      if (!is_free[i]) continue;
      if (at < want) list[at] = first + i;
      ++at;
    }
    found += total;
  }
  __syncthreads();
  return min(found, want);
}

// Pages that a row holds: its leading entries that are not negative.  They are those of its length, mostly, or a few more.
__device__ __forceinline__ int held_pages(const FaPageTables& t, int row, int64_t of_length) {
  const int* entries = t.block_table + row * t.row_stride;
  int n = 0;
  if (of_length >= 1 && of_length <= t.columns && entries[of_length - 1] >= 0) n = static_cast<int>(of_length);
  while (n < t.columns && entries[n] >= 0) ++n;
  return n;
}
__device__ __forceinline__ int64_t pages_of(int64_t tokens, int page_size) { return (tokens + page_size - 1) / page_size; }

// ---------------------------------------------------------------------------------------------
// reserve: pages for the next tokens of every row
// ---------------------------------------------------------------------------------------------
struct ReserveParams {
  FaPageTables t;
  const int* new_tokens;  // (rows), or null: new_tokens_all for each
  int new_tokens_all, page_size;
  uint8_t* granted;
  int *need, *begin, *held, *list;  // scratch: per row, per row, per row, per page; null: shared memory (small tables)
};
constexpr int kSmallRows = 1024, kSmallPages = 4096;

__global__ void __launch_bounds__(kPlanThreads) reserve_kernel(const __grid_constant__ ReserveParams call) {
  __shared__ int rows_scratch[3][kSmallRows], list_scratch[kSmallPages];
  ReserveParams p = call;
  if (p.need == nullptr) p.need = rows_scratch[0], p.begin = rows_scratch[1], p.held = rows_scratch[2], p.list = list_scratch;
  // what each row needs; a row whose columns do not suffice needs nothing and is refused
  int64_t wanted = 0;
  for (int r0 = 0; r0 < p.t.rows; r0 += kPlanThreads) {
    const int r = r0 + threadIdx.x;
    int need = 0;
    if (r < p.t.rows) {
      const int64_t len = max(p.t.cache_seqlens[r], 0);
      const int64_t more = max(p.new_tokens ? p.new_tokens[r] : p.new_tokens_all, 0);
      const int64_t want = pages_of(len + more, p.page_size);
      const int held = held_pages(p.t, r, pages_of(len, p.page_size));
      if (want > p.t.columns) need = -1;
      else need = static_cast<int>(max(want - held, static_cast<int64_t>(0)));
      p.need[r] = need, p.held[r] = held;
    }
    int total;
    const int before = block_scan(max(need, 0), total);
    // more than there are pages is refused, whatever the sum: limited, so that it stays in 32 bits
    if (r < p.t.rows) p.begin[r] = static_cast<int>(min(wanted + before, static_cast<int64_t>(p.t.num_pages) + 1));
    wanted += total;
  }
  const int want = static_cast<int>(min(wanted, static_cast<int64_t>(p.t.num_pages)));
  const int found = want > 0 ? find_free(p.t.page_refs, p.t.num_pages, want, p.list) : 0;
  for (int r = threadIdx.x; r < p.t.rows; r += kPlanThreads) {
    const int need = p.need[r], begin = p.begin[r];
    const bool granted = need == 0 || (need > 0 && static_cast<int64_t>(begin) + need <= found);
    p.granted[r] = granted;
    if (!granted) continue;
    int* entries = p.t.block_table + r * p.t.row_stride + p.held[r];
    for (int c = 0; c < need; ++c) {
      const int page = p.list[begin + c];
      entries[c] = page;
      p.t.page_refs[page] = 1;
    }
  }
}

// ---------------------------------------------------------------------------------------------
// fork: children share the full pages of their parents and get a copy of the last one
// ---------------------------------------------------------------------------------------------
struct ForkParams {
  FaPageTables t;
  const int *parents, *children;
  int n, page_size;
  int64_t token_bytes;
  uint8_t* granted;
  int* first;  // scratch, per row: the first entry with that child
  int* begin;  // per entry: rank among those that need a page; -1 - rank: needs none; kRefused
  int* list;   // per page
  PageMove* moves;
  int* count;
};
constexpr int kRefused = 0x7fffffff;

// Whether a parent's pages can be shared, apart from what its child is and from a hole among them (see fork_row); partial: the last one
// has to be copied
__device__ __forceinline__ bool forkable(const FaPageTables& t, int parent, int page_size, bool& partial) {
  const int64_t len = max(t.cache_seqlens[parent], 0), pages = pages_of(len, page_size);
  const int held = held_pages(t, parent, pages);
  partial = len % page_size != 0;
  return held > 0 && held >= pages && (!partial || t.block_table[parent * t.row_stride + pages - 1] < t.num_pages);
}

// The tables of a child, by a warp; page: for the parent's last tokens, -1: its pages are full.  Whether it was done: not for a parent
// with -1 before its last page.  No function leaves such a row; it is found here, where all entries are read, and the page that was meant
// for the copy stays free.
__device__ __forceinline__ bool fork_row(const FaPageTables& t, int parent, int child, int page_size, int page) {
  const int lane = threadIdx.x & 31;
  const int len = max(t.cache_seqlens[parent], 0), full = len / page_size;
  const int* from = t.block_table + parent * t.row_stride;
  int* to = t.block_table + child * t.row_stride;
  bool whole = true;
  for (int c = lane; c < full; c += 32) whole &= from[c] >= 0;
  if (!__all_sync(0xffffffffu, whole)) return false;
  for (int c = lane; c < full; c += 32) {
    const int shared = from[c];
    to[c] = shared;
    if (shared < t.num_pages) atomicAdd(t.page_refs + shared, 1);
  }
  if (lane == 0) {
    if (page >= 0) {
      to[full] = page;
      t.page_refs[page] = 1;
    }
    t.cache_seqlens[child] = len;
  }
  return true;
}

__global__ void __launch_bounds__(kPlanThreads) fork_kernel(const __grid_constant__ ForkParams p) {
  grid_launch_dependents();
  auto inside = [&](int row) { return row >= 0 && row < p.t.rows; };
  for (int r = threadIdx.x; r < p.t.rows; r += kPlanThreads) p.first[r] = p.n;
  __syncthreads();
  for (int i = threadIdx.x; i < p.n; i += kPlanThreads)
    if (inside(p.parents[i]) && inside(p.children[i])) atomicMin(p.first + p.children[i], i);
  __syncthreads();
  // Everything is looked at before anything is written.  Parents hold pages and children none, so no row is both.
  int wanted = 0;
  for (int i0 = 0; i0 < p.n; i0 += kPlanThreads) {
    const int i = i0 + threadIdx.x;
    bool valid = false, partial = false;
    if (i < p.n) {
      const int parent = p.parents[i], child = p.children[i];
      if (inside(parent) && inside(child) && p.first[child] == i && p.t.block_table[child * p.t.row_stride] < 0)
        valid = forkable(p.t, parent, p.page_size, partial);
    }
    int total;
    const int rank = wanted + block_scan(valid && partial, total);
    if (i < p.n) p.begin[i] = !valid ? kRefused : partial ? rank : -1 - rank;
    wanted += total;
  }
  const int found = wanted > 0 ? find_free(p.t.page_refs, p.t.num_pages, wanted, p.list) : 0;
  if (threadIdx.x == 0) *p.count = found;
  __syncthreads();  // the ranks
  for (int i = threadIdx.x >> 5; i < p.n; i += kPlanWarps) {  // a warp per entry
    const int rank = p.begin[i];
    if (rank >= found) {  // kRefused is, an entry that needs no page is not
      if ((threadIdx.x & 31) == 0) p.granted[i] = false;
      continue;
    }
    const int parent = p.parents[i], page = rank >= 0 ? p.list[rank] : -1;
    if ((threadIdx.x & 31) == 0 && rank >= 0) {
      const int len = max(p.t.cache_seqlens[parent], 0), full = len / p.page_size;
      p.moves[rank] = PageMove{p.t.block_table[parent * p.t.row_stride + full], page, (len - full * p.page_size) * p.token_bytes};
    }
    const bool done = fork_row(p.t, parent, p.children[i], p.page_size, page);
    if ((threadIdx.x & 31) == 0) p.granted[i] = done;
  }
}

// ---------------------------------------------------------------------------------------------
// free: the rows' references to their pages; a warp per row
// ---------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(256) free_kernel(const FaPageTables t, const int* rows, int n) {
  const int lane = threadIdx.x & 31;
  for (int i = blockIdx.x * 8 + (threadIdx.x >> 5); i < n; i += gridDim.x * 8) {
    const int row = rows[i];
    if (row < 0 || row >= t.rows) continue;
    int* entries = t.block_table + row * t.row_stride;
    for (int c = lane; c < t.columns; c += 32) {
      if (entries[c] < 0) continue;
      const int page = atomicExch(entries + c, -1);  // a row that is named twice is freed once
      if (page < 0 || page >= t.num_pages) continue;
      if (atomicSub(t.page_refs + page, 1) <= 0) atomicAdd(t.page_refs + page, 1);
    }
    if (lane == 0) t.cache_seqlens[row] = 0;
  }
}

// ---------------------------------------------------------------------------------------------
// compact: the i-th live page behind the first `live` pages moves to the i-th free one among them
// ---------------------------------------------------------------------------------------------
struct CompactParams {
  FaPageTables t;
  int64_t page_bytes;
  int* num_live;
  int* list;        // scratch, per page: free pages among the first `live`
  PageMove* moves;
  int* count;
  int* to;          // per page: where it went
};

__global__ void __launch_bounds__(kPlanThreads) compact_kernel(const __grid_constant__ CompactParams p) {
  grid_launch_dependents();
  const int* refs = p.t.page_refs;
  int mine = 0;
  for (int i = threadIdx.x; i < p.t.num_pages; i += kPlanThreads) mine += refs[i] > 0;
  int live;
  block_scan(mine, live);
  const int found = find_free(refs, live, live, p.list);  // pages [0, live): as many free ones as there are live ones behind
  int moved = 0;
  for (int base = live; base < p.t.num_pages; base += kPlanThreads) {
    const int page = base + threadIdx.x, count = page < p.t.num_pages ? refs[page] : 0;
    int total;
    const int at = moved + block_scan(count > 0, total);
    if (count <= 0 && page < p.t.num_pages) p.to[page] = page;  // a table should not name it
    if (count > 0) {
      const int dst = p.list[at];
      p.moves[at] = PageMove{page, dst, p.page_bytes};
      p.to[page] = dst;
      p.t.page_refs[dst] = count;
      p.t.page_refs[page] = 0;
    }
    moved += total;
  }
  if (threadIdx.x == 0) *p.num_live = live, *p.count = found;
}

// ---------------------------------------------------------------------------------------------
// copy: given pages; what cannot be copied as if all sources were read first is left out and told
// ---------------------------------------------------------------------------------------------
struct CopyPlanParams {
  const int *src, *dst;
  int n, num_pages;
  int64_t page_bytes;
  uint8_t* done;
  int* last;  // scratch, per page: the last entry that it is the destination of
  PageMove* moves;
  int* count;
};

__global__ void __launch_bounds__(kPlanThreads) copy_plan_kernel(const __grid_constant__ CopyPlanParams p) {
  grid_launch_dependents();
  auto inside = [&](int page) { return page >= 0 && page < p.num_pages; };
  for (int i = threadIdx.x; i < p.n; i += kPlanThreads)
    if (inside(p.dst[i]) && inside(p.src[i])) p.last[p.dst[i]] = p.last[p.src[i]] = -1;
  __syncthreads();
  for (int i = threadIdx.x; i < p.n; i += kPlanThreads)
    if (inside(p.dst[i]) && inside(p.src[i]) && p.dst[i] != p.src[i]) atomicMax(p.last + p.dst[i], i);
  __syncthreads();
  int count = 0;
  for (int i0 = 0; i0 < p.n; i0 += kPlanThreads) {
    const int i = i0 + threadIdx.x;
    bool ok = false, moves = false;
    int src = 0, dst = 0;
    if (i < p.n) {
      src = p.src[i], dst = p.dst[i];
      ok = inside(src) && inside(dst) && p.last[src] < 0 && (src == dst || p.last[dst] == i);
      moves = ok && src != dst;
      p.done[i] = ok;
    }
    int total;
    const int at = count + block_scan(moves, total);
    if (moves) p.moves[at] = PageMove{src, dst, p.page_bytes};
    count += total;
  }
  if (threadIdx.x == 0) *p.count = count;
}

// ---------------------------------------------------------------------------------------------
// the copying kernel
// ---------------------------------------------------------------------------------------------
constexpr int kCopyThreads = 256;
constexpr int kMaxCaches = 128;  // of a launch

struct MoveParams {
  uint8_t* base[kMaxCaches];
  int64_t page_stride[kMaxCaches];  // bytes
  int caches;
  int chunks;                       // per page
  const PageMove* moves;
  const int* count;
  // compact: table entries from *num_live on are replaced by to[entry]; null: no table
  FaPageTables t;
  const int* to;
  const int* num_live;
};

// Copies of 805 MB (24 pages of 32 caches) by CTAs that take one chunk each and 1184 that take them in turn: 127 and 137 us (6.4 and 5.9
// TB/s, read and written; torch's copy of one tensor 6.5).  Where the plan says how many there are, 32 CTAs per SM take them in turn.
// Chunks of 12, 16, 24, 64 KB 125, 126, 126, 127 us, with larger moves between other pages 200, 195, 191, 220 (32 KB: 190).
// `bytes` of a page, kUnroll 16-byte units of a thread at a time, of which the first begins at `at`
template <int kUnroll>
__device__ __forceinline__ void copy_chunk(const uint8_t* src, uint8_t* dst, int64_t at, int64_t bytes) {
  uint4 x[kUnroll];
#pragma unroll
  for (int i = 0; i < kUnroll; ++i)
    if (at + i * kCopyThreads * 16 < bytes) x[i] = *reinterpret_cast<const uint4*>(src + at + i * kCopyThreads * 16);
#pragma unroll
  for (int i = 0; i < kUnroll; ++i)
    if (at + i * kCopyThreads * 16 < bytes) *reinterpret_cast<uint4*>(dst + at + i * kCopyThreads * 16) = x[i];
}

// kUnroll 16-byte units of a thread in flight: a chunk is kUnroll * 4 KB of a page of one cache
template <int kUnroll>
__global__ void __launch_bounds__(kCopyThreads) move_kernel(const __grid_constant__ MoveParams p) {
  constexpr int kChunk = kUnroll * kCopyThreads * 16;
  grid_dependency_wait();  // the plan
  const int64_t per_move = static_cast<int64_t>(p.caches) * p.chunks, total = *p.count * per_move;
  for (int64_t item = blockIdx.x; item < total; item += gridDim.x) {
    const int64_t m = item / per_move;
    const int rest = static_cast<int>(item - m * per_move), cache = rest / p.chunks, chunk = rest - cache * p.chunks;
    const PageMove move = p.moves[m];
    copy_chunk<kUnroll>(p.base[cache] + move.src * p.page_stride[cache], p.base[cache] + move.dst * p.page_stride[cache],
                        static_cast<int64_t>(chunk) * kChunk + threadIdx.x * 16, move.bytes);
  }
  if (p.to != nullptr) {
    const int live = *p.num_live, pages = p.t.num_pages;
    const int64_t entries = static_cast<int64_t>(p.t.rows) * p.t.columns;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kCopyThreads + threadIdx.x; i < entries;
         i += static_cast<int64_t>(gridDim.x) * kCopyThreads) {
      const int64_t row = i / p.t.columns;
      int* entry = p.t.block_table + row * p.t.row_stride + (i - row * p.t.columns);
      const int page = *entry;
      if (page >= live && page < pages) *entry = p.to[page];
    }
  }
}

// Few pages (kFewPages at most): the plan of an entry is a look at all entries, which each CTA takes by itself, and no launch or
// scratch memory is needed for it.  3 pages of 4 caches (768 KB) 9.4 -> 6.6 us a call, most of it the host's.
constexpr int kFewPages = 512;
struct FewParams {
  uint8_t* base[kMaxCaches];
  int64_t page_stride[kMaxCaches];
  int64_t page_bytes;
  const int *src, *dst;
  uint8_t* done;
  int caches, chunks, n, num_pages;
};
template <int kUnroll>
__global__ void __launch_bounds__(kCopyThreads) copy_few_kernel(const __grid_constant__ FewParams p) {
  constexpr int kChunk = kUnroll * kCopyThreads * 16;
  const int per_entry = p.caches * p.chunks;
  const int i = blockIdx.x / per_entry, rest = blockIdx.x - i * per_entry, cache = rest / p.chunks, chunk = rest - cache * p.chunks;
  const int src = p.src[i], dst = p.dst[i];
  auto inside = [&](int page) { return page >= 0 && page < p.num_pages; };
  bool bad = !inside(src) || !inside(dst);
  for (int j = threadIdx.x; j < p.n; j += kCopyThreads) {
    const int a = p.src[j], b = p.dst[j];
    if (inside(a) && inside(b) && a != b) bad |= b == src || (src != dst && b == dst && j > i);
  }
  bad = __syncthreads_or(bad);
  if (rest == 0 && threadIdx.x == 0) p.done[i] = !bad;
  if (bad || src == dst) return;
  copy_chunk<kUnroll>(p.base[cache] + src * p.page_stride[cache], p.base[cache] + dst * p.page_stride[cache],
                      static_cast<int64_t>(chunk) * kChunk + threadIdx.x * 16, p.page_bytes);
}

// Few forks (kFewForks at most): each CTA makes the plan for itself and copies chunks of one entry in one cache; the
// last CTA that has made it writes the tables, which nobody reads any more.  One launch and no scratch memory: 8 forks in 4 caches
// take the host 6.0 us where the two kernels took 10.5.  Of 48 entries in
// 16 caches 1536 CTAs would make the plan, 25 us where the two kernels take 11.
constexpr int kFewForks = 32, kFewForkCtas = 4 * 148;
struct FewForkParams {
  uint8_t* base[kMaxCaches];
  int64_t page_stride[kMaxCaches];
  FaPageTables t;
  const int *parents, *children;
  uint8_t* granted;
  int64_t token_bytes;
  int* counter;  // zero before and after
  int caches, ctas, n, page_size;  // ctas: for the chunks of a page of a cache
};
template <int kUnroll>
__global__ void __launch_bounds__(kCopyThreads) fork_few_kernel(const __grid_constant__ FewForkParams p) {
  constexpr int kChunk = kUnroll * kCopyThreads * 16, kWarps = kCopyThreads / 32;
  __shared__ int parents[kFewForks], children[kFewForks], pages[kFewForks], warp_sums[kWarps];
  __shared__ uint64_t valid_mask, partial_mask;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) valid_mask = partial_mask = 0;
  if (tid < p.n) parents[tid] = p.parents[tid], children[tid] = p.children[tid];
  __syncthreads();
  if (tid < p.n) {
    const int parent = parents[tid], child = children[tid];
    auto inside = [&](int row) { return row >= 0 && row < p.t.rows; };
    bool valid = inside(parent) && inside(child), partial = false;
    for (int i = 0; i < tid; ++i) valid &= !(children[i] == child && inside(parents[i]));
    if (valid && p.t.block_table[child * p.t.row_stride] < 0 && forkable(p.t, parent, p.page_size, partial)) {
      atomicOr(reinterpret_cast<unsigned long long*>(&valid_mask), 1ull << tid);
      if (partial) atomicOr(reinterpret_cast<unsigned long long*>(&partial_mask), 1ull << tid);
    }
  }
  __syncthreads();
  const uint64_t valid = valid_mask, copies = valid_mask & partial_mask;
  const int want = __popcll(copies);
  // the first `want` free pages, as find_free()
  int found = 0;
  for (int base = 0; base < p.t.num_pages && found < want; base += kCopyThreads * kPagesPerThread) {
    const int first = base + tid * kPagesPerThread;
    bool is_free[kPagesPerThread];
    int mine = 0;
#pragma unroll
    for (int i = 0; i < kPagesPerThread; ++i) {
      is_free[i] = first + i < p.t.num_pages && p.t.page_refs[first + i] <= 0;
      mine += is_free[i];
    }
    int sum = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, sum, off);
      if (lane >= off) sum += other;
    }
    __syncthreads();  // the sums of the round before have been read
    if (lane == 31) warp_sums[warp] = sum;
    __syncthreads();
    int at = found + sum - mine, total = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      const int w = warp_sums[i];
      if (i < warp) at += w;
      total += w;
    }
#pragma unroll
    for (int i = 0; i < kPagesPerThread; ++i) {
      if (is_free[i] && at < want) pages[at] = first + i;
      at += is_free[i];
    }
    found += total;
  }
  found = min(found, want);
  // whether entry i is done, and the page of its copy (-1: it needs none)
  auto plan = [&](int i, int& page) {
    const int rank = __popcll(copies & ((1ull << i) - 1));
    const bool needs = (copies >> i & 1) != 0;
    page = needs && rank < found ? pages[rank] : -1;
    return (valid >> i & 1) != 0 && (!needs || rank < found);
  };
  const int per_entry = p.caches * p.ctas;
  const int entry = blockIdx.x / per_entry, rest = blockIdx.x - entry * per_entry, cache = rest / p.ctas;
  int src = 0, dst = -1, len = 0;
  __syncthreads();  // the pages
  if (plan(entry, dst) && dst >= 0) {
    len = max(p.t.cache_seqlens[parents[entry]], 0);
    src = p.t.block_table[parents[entry] * p.t.row_stride + len / p.page_size];
  }
  __threadfence();
  __syncthreads();  // all that this CTA reads of the tables has been read
  const bool last = __syncthreads_or(tid == 0 && atomicAdd(p.counter, 1) == static_cast<int>(gridDim.x) - 1);
  const int64_t bytes = len % p.page_size * p.token_bytes;
  if (dst >= 0) {
    for (int64_t at = static_cast<int64_t>(rest - cache * p.ctas) * kChunk; at < bytes; at += static_cast<int64_t>(p.ctas) * kChunk)
      copy_chunk<kUnroll>(p.base[cache] + src * p.page_stride[cache], p.base[cache] + dst * p.page_stride[cache], at + tid * 16, bytes);
  }
  if (!last) return;
  __threadfence();
  if (tid == 0) *p.counter = 0;
  for (int i = warp; i < p.n; i += kWarps) {
    int page;
    const bool done = plan(i, page) && fork_row(p.t, parents[i], children[i], p.page_size, page);
    if (lane == 0) p.granted[i] = done;
  }
}

size_t align256(size_t x) { return (x + 255) / 256 * 256; }

// Carves the workspace up; with base == nullptr only the size is wanted
struct Carver {
  uint8_t* base;
  size_t used = 0;
  template <class T>
  T* take(int64_t n) {
    T* at = reinterpret_cast<T*>(base + used);
    used += align256(static_cast<size_t>(std::max<int64_t>(n, 1)) * sizeof(T));
    return at;
  }
};

int check_tables(const FaPageTables* t, bool lengths, const char* who) {
  FA_CHECK_ARG(t != nullptr && t->block_table && (t->cache_seqlens || !lengths) && t->page_refs, std::string(who) + ": tables must be non-NULL");
  FA_CHECK_ARG(t->rows >= 1 && t->columns >= 1 && t->columns <= (1 << 20) && t->num_pages >= 1 && t->row_stride >= t->columns,
               std::string(who) + ": bad rows, columns, row_stride or num_pages");
  return FA_OK;
}

int check_caches(const FaPageCaches* c, const char* who) {
  FA_CHECK_ARG(c != nullptr && c->base != nullptr && c->page_stride != nullptr && c->count >= 1, std::string(who) + ": no caches");
  FA_CHECK_ARG(c->page_bytes >= 16 && c->page_bytes % 16 == 0 && c->page_bytes < (1ll << 40),
               std::string(who) + ": the bytes of a page must be a multiple of 16");
  for (int i = 0; i < c->count; ++i)
    FA_CHECK_ARG(c->base[i] != nullptr && aligned16(c->base[i]) && c->page_stride[i] % 16 == 0 && c->page_stride[i] >= c->page_bytes,
                 std::string(who) + ": caches must be 16-byte aligned, with page strides that are multiples of 16 bytes and hold a page");
  return FA_OK;
}

int check_workspace(const void* ws, size_t bytes, size_t need, const char* who) {
  if (ws == nullptr || bytes < need) return set_error(FA_ERR_WORKSPACE, std::string(who) + ": workspace smaller than fa_pages_workspace_bytes()");
  FA_CHECK_ARG((reinterpret_cast<uintptr_t>(ws) & 255) == 0, std::string(who) + ": workspace must be 256-byte aligned");
  return FA_OK;
}

// Chunks (16-byte units of a thread) as large as still give every SM some: a thread then has that many loads in flight
int chunk_units(int64_t bytes, int sms) { return bytes >= sms * (8ll << 15) ? 8 : bytes >= sms * (4ll << 13) ? 2 : 1; }

int launch_few(const FaPageCaches* c, int num_pages, const int* src, const int* dst, int n, uint8_t* done, cudaStream_t stream) {
  const int sms = device_sm_count();
  if (sms <= 0) return set_error(FA_ERR_CUDA, "fa_pages_copy: device attributes not available");
  FewParams p = {};
  for (int i = 0; i < c->count; ++i) p.base[i] = static_cast<uint8_t*>(c->base[i]), p.page_stride[i] = c->page_stride[i];
  p.page_bytes = c->page_bytes, p.src = src, p.dst = dst, p.done = done, p.caches = c->count, p.n = n, p.num_pages = num_pages;
  const int units = chunk_units(static_cast<int64_t>(n) * c->count * c->page_bytes, sms);
  const int64_t chunk = units * kCopyThreads * 16;
  p.chunks = static_cast<int>((c->page_bytes + chunk - 1) / chunk);
  const int64_t items = static_cast<int64_t>(n) * c->count * p.chunks;
  const auto kernel = units == 8 ? copy_few_kernel<8> : units == 2 ? copy_few_kernel<2> : copy_few_kernel<1>;
  kernel<<<static_cast<unsigned>(items), kCopyThreads, 0, stream>>>(p);
  FA_CHECK_CUDA(cudaGetLastError());
  return FA_OK;
}

// most: moves that there can be
int launch_moves(const FaPageCaches* c, const PageMove* moves, const int* count, int64_t most, const FaPageTables* t, const int* to,
                 const int* num_live, cudaStream_t stream) {
  const int sms = device_sm_count();
  if (sms <= 0) return set_error(FA_ERR_CUDA, "fa_pages: device attributes not available");
  for (int first = 0; first < c->count; first += kMaxCaches) {
    MoveParams p = {};
    p.caches = std::min(c->count - first, kMaxCaches);
    for (int i = 0; i < p.caches; ++i)
      p.base[i] = static_cast<uint8_t*>(c->base[first + i]), p.page_stride[i] = c->page_stride[first + i];
    p.moves = moves, p.count = count;
    if (first + kMaxCaches >= c->count && t != nullptr) p.t = *t, p.to = to, p.num_live = num_live;  // the last launch
    const int unroll = chunk_units(most * p.caches * c->page_bytes, sms);
    const int64_t chunk = unroll * kCopyThreads * 16;
    p.chunks = static_cast<int>((c->page_bytes + chunk - 1) / chunk);
    const int64_t items = std::max<int64_t>(most * p.caches * p.chunks, 1);
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>(items, sms * 32)));
    const auto kernel = unroll == 8 ? move_kernel<8> : unroll == 2 ? move_kernel<2> : move_kernel<1>;
    if (first == 0) {
      FA_CHECK_CUDA(launch_overlapped(kernel, grid, kCopyThreads, 0, stream, p));
    } else {
      kernel<<<grid, kCopyThreads, 0, stream>>>(p);
      FA_CHECK_CUDA(cudaGetLastError());
    }
  }
  return FA_OK;
}

// CTAs for each cache of an entry: all of them are resident together, and they read 32 MB of counts between them at most
int few_fork_ctas(const FaPageCaches* c, int n, int* units) {
  *units = chunk_units(n * c->count * c->page_bytes, 148);
  const int64_t chunk = *units * kCopyThreads * 16, chunks = (c->page_bytes + chunk - 1) / chunk;
  return static_cast<int>(std::min<int64_t>(chunks, kFewForkCtas / (n * c->count)));
}
bool forks_few(const FaPageTables* t, const FaPageCaches* c, int n) {
  if (n < 1 || n > kFewForks || c->count < 1 || c->count > kMaxCaches || c->page_bytes < 16 || c->page_bytes >= (1 << 30)) return false;
  int units;
  const int64_t ctas = few_fork_ctas(c, n, &units);
  return ctas >= 1 && n * c->count * ctas * t->num_pages <= (8 << 20);
}

int launch_few_forks(const FaPageTables* t, const FaPageCaches* c, const int* parents, const int* children, int n, int page_size,
                     uint8_t* granted, cudaStream_t stream) {
  FewForkParams p = {};
  for (int i = 0; i < c->count; ++i) p.base[i] = static_cast<uint8_t*>(c->base[i]), p.page_stride[i] = c->page_stride[i];
  p.t = *t, p.parents = parents, p.children = children, p.granted = granted, p.caches = c->count, p.n = n, p.page_size = page_size;
  p.token_bytes = c->page_bytes / page_size;
  p.counter = next_sched_slot(stream);
  if (p.counter == nullptr) return set_error(FA_ERR_CUDA, "fa_pages_fork: device attributes not available");
  int units;
  p.ctas = few_fork_ctas(c, n, &units);
  const auto kernel = units == 8 ? fork_few_kernel<8> : units == 2 ? fork_few_kernel<2> : fork_few_kernel<1>;
  kernel<<<n * c->count * p.ctas, kCopyThreads, 0, stream>>>(p);
  FA_CHECK_CUDA(cudaGetLastError());
  return FA_OK;
}

bool copies_few(const FaPageCaches* c, int n) {  // the items are counted in 32 bits
  return n <= kFewPages && c->count <= kMaxCaches && static_cast<int64_t>(n) * c->count * (c->page_bytes / 4096 + 1) < (1 << 30);
}

size_t workspace_bytes(int64_t rows, int64_t pages, int64_t entries) {
  Carver c{nullptr};
  for (int i = 0; i < 3; ++i) c.take<int>(std::max(rows, entries));
  c.take<int>(pages), c.take<int>(pages);
  c.take<PageMove>(std::max(pages, entries));
  c.take<int>(1);
  return c.used;
}

}  // namespace
}  // namespace fa

extern "C" size_t fa_pages_workspace_bytes(int32_t rows, int32_t num_pages, int32_t entries) {
  if (rows < 0 || num_pages < 0 || entries < 0) return 0;
  return fa::workspace_bytes(rows, num_pages, entries);
}

extern "C" size_t fa_pages_copy_workspace_bytes(const FaPageCaches* caches, int32_t num_pages, int32_t n) {
  if (caches == nullptr || num_pages < 0 || n < 0 || fa::copies_few(caches, n)) return 0;
  return fa::workspace_bytes(0, num_pages, n);
}

extern "C" size_t fa_pages_reserve_workspace_bytes(const FaPageTables* t) {
  if (t == nullptr || t->rows < 0 || t->num_pages < 0 || (t->rows <= fa::kSmallRows && t->num_pages <= fa::kSmallPages)) return 0;
  return fa::workspace_bytes(t->rows, t->num_pages, 0);
}

extern "C" size_t fa_pages_fork_workspace_bytes(const FaPageTables* t, const FaPageCaches* caches, int32_t n) {
  if (t == nullptr || caches == nullptr || t->rows < 0 || t->num_pages < 0 || n < 0 || fa::forks_few(t, caches, n)) return 0;
  return fa::workspace_bytes(t->rows, t->num_pages, n);
}

extern "C" int fa_pages_reserve(const FaPageTables* t, const int32_t* new_tokens, int32_t new_tokens_all, int32_t page_size, uint8_t* granted,
                                void* workspace, size_t bytes, fa_stream_t stream) {
  using namespace fa;
  int rc = check_tables(t, true, "fa_pages_reserve");
  if (rc != FA_OK) return rc;
  FA_CHECK_ARG(page_size >= 1 && granted != nullptr, "fa_pages_reserve: bad page_size or granted");
  const bool needs = fa_pages_reserve_workspace_bytes(t) > 0;
  if (needs || workspace != nullptr) rc = check_workspace(workspace, bytes, workspace_bytes(t->rows, t->num_pages, 0), "fa_pages_reserve");
  if (rc != FA_OK) return rc;
  rc = check_device_sm100();
  if (rc != FA_OK) return rc;
  ReserveParams p{*t, new_tokens, new_tokens_all, page_size, granted};
  if (needs) {
    Carver c{static_cast<uint8_t*>(workspace)};
    p.need = c.take<int>(t->rows), p.begin = c.take<int>(t->rows), p.held = c.take<int>(t->rows), p.list = c.take<int>(t->num_pages);
  }
  reserve_kernel<<<1, kPlanThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
  FA_CHECK_CUDA(cudaGetLastError());
  return FA_OK;
}

extern "C" int fa_pages_fork(const FaPageTables* t, const FaPageCaches* caches, const int32_t* parents, const int32_t* children, int32_t n,
                             int32_t page_size, uint8_t* granted, void* workspace, size_t bytes, fa_stream_t stream_) {
  using namespace fa;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  int rc = check_tables(t, true, "fa_pages_fork");
  if (rc == FA_OK) rc = check_caches(caches, "fa_pages_fork");
  if (rc != FA_OK) return rc;
  FA_CHECK_ARG(n >= 0 && page_size >= 1 && caches->page_bytes % page_size == 0 && caches->page_bytes / page_size % 16 == 0,
               "fa_pages_fork: the bytes of a token must be a multiple of 16");
  if (n == 0) return FA_OK;
  FA_CHECK_ARG(parents && children && granted, "fa_pages_fork: parents, children, granted must be non-NULL");
  const bool few = forks_few(t, caches, n);
  if (!few || workspace != nullptr) rc = check_workspace(workspace, bytes, workspace_bytes(t->rows, t->num_pages, n), "fa_pages_fork");
  if (rc == FA_OK) rc = check_device_sm100();
  if (rc != FA_OK) return rc;
  if (few) return launch_few_forks(t, caches, parents, children, n, page_size, granted, stream);
  Carver c{static_cast<uint8_t*>(workspace)};
  ForkParams p{*t, parents, children, n, page_size, caches->page_bytes / page_size, granted};
  p.first = c.take<int>(t->rows), p.begin = c.take<int>(n), p.list = c.take<int>(t->num_pages);
  p.moves = c.take<PageMove>(std::min(n, t->num_pages)), p.count = c.take<int>(1);
  fork_kernel<<<1, kPlanThreads, 0, stream>>>(p);
  FA_CHECK_CUDA(cudaGetLastError());
  return launch_moves(caches, p.moves, p.count, std::min(n, t->num_pages), nullptr, nullptr, nullptr, stream);
}

extern "C" int fa_pages_free(const FaPageTables* t, const int32_t* rows, int32_t n, fa_stream_t stream) {
  using namespace fa;
  int rc = check_tables(t, true, "fa_pages_free");
  if (rc != FA_OK) return rc;
  FA_CHECK_ARG(n >= 0, "fa_pages_free: n is negative");
  if (n == 0) return FA_OK;
  FA_CHECK_ARG(rows != nullptr, "fa_pages_free: rows must be non-NULL");
  rc = check_device_sm100();
  if (rc != FA_OK) return rc;
  free_kernel<<<std::min((n + 7) / 8, 148 * 8), 256, 0, static_cast<cudaStream_t>(stream)>>>(*t, rows, n);
  FA_CHECK_CUDA(cudaGetLastError());
  return FA_OK;
}

extern "C" int fa_pages_compact(const FaPageTables* t, const FaPageCaches* caches, int32_t* num_live, void* workspace, size_t bytes,
                                fa_stream_t stream_) {
  using namespace fa;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  int rc = check_tables(t, false, "fa_pages_compact");
  if (rc == FA_OK) rc = check_caches(caches, "fa_pages_compact");
  if (rc != FA_OK) return rc;
  FA_CHECK_ARG(num_live != nullptr, "fa_pages_compact: num_live must be non-NULL");
  rc = check_workspace(workspace, bytes, workspace_bytes(t->rows, t->num_pages, 0), "fa_pages_compact");
  if (rc == FA_OK) rc = check_device_sm100();
  if (rc != FA_OK) return rc;
  Carver c{static_cast<uint8_t*>(workspace)};
  CompactParams p{*t, caches->page_bytes, num_live};
  p.list = c.take<int>(t->num_pages), p.to = c.take<int>(t->num_pages);
  p.moves = c.take<PageMove>(t->num_pages), p.count = c.take<int>(1);
  compact_kernel<<<1, kPlanThreads, 0, stream>>>(p);
  FA_CHECK_CUDA(cudaGetLastError());
  return launch_moves(caches, p.moves, p.count, t->num_pages / 2, t, p.to, num_live, stream);
}

extern "C" int fa_pages_copy(const FaPageCaches* caches, int32_t num_pages, const int32_t* src, const int32_t* dst, int32_t n, uint8_t* done,
                             void* workspace, size_t bytes, fa_stream_t stream_) {
  using namespace fa;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  int rc = check_caches(caches, "fa_pages_copy");
  if (rc != FA_OK) return rc;
  FA_CHECK_ARG(n >= 0 && num_pages >= 1, "fa_pages_copy: n is negative or num_pages not positive");
  if (n == 0) return FA_OK;
  FA_CHECK_ARG(src && dst && done, "fa_pages_copy: src, dst, done must be non-NULL");
  if (copies_few(caches, n)) {
    rc = check_device_sm100();
    return rc != FA_OK ? rc : launch_few(caches, num_pages, src, dst, n, done, stream);
  }
  rc = check_workspace(workspace, bytes, workspace_bytes(0, num_pages, n), "fa_pages_copy");
  if (rc == FA_OK) rc = check_device_sm100();
  if (rc != FA_OK) return rc;
  Carver c{static_cast<uint8_t*>(workspace)};
  CopyPlanParams p{src, dst, n, num_pages, caches->page_bytes, done};
  p.last = c.take<int>(num_pages), p.moves = c.take<PageMove>(std::min(n, num_pages)), p.count = c.take<int>(1);
  copy_plan_kernel<<<1, kPlanThreads, 0, stream>>>(p);
  FA_CHECK_CUDA(cudaGetLastError());
  return launch_moves(caches, p.moves, p.count, std::min(n, num_pages), nullptr, nullptr, nullptr, stream);
}
