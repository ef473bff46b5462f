// Pages of the paged caches for gfx950: copies of whole pages, forks (a new sequence that shares its parent's full
// pages and copies the last, partial one), releases, and compaction (the live pages moved to the pool's front). The
// state is a use count per page, ref [num_pages]: 0 is free; page 0, the null page, is never counted, given out or
// moved. Integers only and every choice in ascending order (the lowest free pages, the k-th live page past the front to
// the k-th hole), so the results do not depend on the order in which workgroups run.
//
// What bounds them: the copies move bytes at a large copy's rate once there are enough pages (compaction of 12,345
// pages, fork of many sequences); a small fork is its two launches. Every cache of a model takes part in one launch (up
// to PG_CACHES of them: latent rows, their scales, indexer keys, ... of every layer), a page of each cut into 16 KiB
// pieces, one workgroup a piece, so that one page of one sequence already spreads over several CUs. Measured:
// compaction of 12,345 pages of five caches, 320 MB read and written, 6.2 us of planning and 60 of moves at 5.2 TB/s (a
// large copy: 4.8); copies of 1 page of four caches 3.7 us, of 128 4.9, of 5,000 (456 MB) 97, 4.7 TB/s; fork of 8 or 128
// sequences 3.5 + 4 to 6 us, their release 2 to 4.
#include "dsa_pages.h"
#include "dsa_scan.h"

namespace dsa {

constexpr int PG_THREADS = 256;                       // a copying workgroup
constexpr int PG_PIECE = PG_THREADS * 16 * 4;         // bytes: four 16-byte loads a thread, all in flight
constexpr int PG_PLAN_THREADS = 1024;                 // a planning workgroup
constexpr int PG_BLOCK = PG_PLAN_THREADS * 4;         // pages of a planning workgroup (one int4 of counts a thread)
// Blocks up to which each planning workgroup counts all of them, a launch less (300 pages: 3.7 us for 1.6 + 3.3 in two
// launches, 12k pages, 4 blocks, 6.2 for 2.6 + 5.0).
constexpr int PG_OWN = 4;

// One piece of page src of every cache it belongs to -> page dst (the whole workgroup).
__device__ __forceinline__ void copy_piece(const PageCaches& set, int piece, int src, int dst) {
  int lo = 0, hi = set.n - 1;  // the cache whose pieces hold it
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (set.first[mid] <= piece) lo = mid;
    else hi = mid - 1;
  }
  const size_t pb = set.page_bytes[lo], off = (size_t)(piece - set.first[lo]) * PG_PIECE;
  const int n = (int)(pb - off < (size_t)PG_PIECE ? pb - off : (size_t)PG_PIECE);
  char* const base = static_cast<char*>(set.p[lo]);
  const char* s = base + (size_t)src * pb + off;
  char* d = base + (size_t)dst * pb + off;
  const int t = threadIdx.x;
  if (((reinterpret_cast<uintptr_t>(base) | pb) & 15) == 0) {
    u32x4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = 16 * (t + PG_THREADS * i);
      if (at < n) v[i] = *reinterpret_cast<const u32x4*>(s + at);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = 16 * (t + PG_THREADS * i);
      if (at < n) *reinterpret_cast<u32x4*>(d + at) = v[i];
    }
  } else {  // pages of odd sizes or places
    for (int at = t; at < n; at += PG_THREADS) d[at] = s[at];
  }
}

__global__ __launch_bounds__(PG_THREADS) void pages_copy_kernel(PageCaches set, const int* __restrict__ src,
                                                                const int* __restrict__ dst, int num_pages) {
  const int i = blockIdx.x / set.pieces, piece = blockIdx.x % set.pieces;
  const int a = src[i], b = dst[i];
  if ((unsigned)a >= (unsigned)num_pages || (unsigned)b >= (unsigned)num_pages || b == 0 || a == b) return;
  copy_piece(set, piece, a, b);
}

typedef int pg_v4i __attribute__((ext_vector_type(4), aligned(4)));  // (a count array may start at any int)

// Four pages' counts from p on, 0 past the pool.
__device__ __forceinline__ pg_v4i load_refs(const int* __restrict__ ref, int p, int num_pages) {
  pg_v4i r = {0, 0, 0, 0};
  if (p + 3 < num_pages) {
    r = *reinterpret_cast<const pg_v4i*>(ref + p);
  } else {
    if (p < num_pages) r.x = ref[p];
    if (p + 1 < num_pages) r.y = ref[p + 1];
    if (p + 2 < num_pages) r.z = ref[p + 2];
  }
  return r;
}

struct ForkRow {
  int parent;  // -1: not a row of the table
  int full;    // whole pages, shared
  bool part;   // a last page to copy
};

__device__ __forceinline__ ForkRow fork_row(int parent, const int* __restrict__ ctx_len, int B, int max_pages,
                                            int page_size) {
  ForkRow f{-1, 0, false};
  if ((unsigned)parent < (unsigned)B) {
    const long cap = (long)max_pages * page_size;
    const long n = min(max((long)ctx_len[parent], 0L), cap);
    f.parent = parent;
    f.full = (int)(n / page_size);
    f.part = n % page_size != 0;
  }
  return f;
}

// One workgroup: each child's new page (pages[i]: 0 where it needs none, -1 where the pool has none left or the parent
// is no row), the lowest free pages to the children in order. free_list: n ints of scratch.
__global__ __launch_bounds__(PG_PLAN_THREADS) void pages_fork_plan_kernel(
    const int* __restrict__ ref, const int* __restrict__ ctx_len, const int* __restrict__ parents,
    int* __restrict__ pages, int* __restrict__ free_list, int B, int n, int max_pages, int page_size, int num_pages) {
  __shared__ int tot[PG_PLAN_THREADS / WAVE];
  const int t = threadIdx.x;
  int need = 0;
  for (int i0 = 0; i0 < n; i0 += PG_PLAN_THREADS) {
    const int i = i0 + t;
    int part = 0;
    if (i < n) part = fork_row(parents[i], ctx_len, B, max_pages, page_size).part;
    int total;
    group_incl_scan<PG_PLAN_THREADS>(part, tot, total);
    need += total;
  }
  int found = 0;  // free pages so far
  for (int p0 = 0; p0 < num_pages && found < need; p0 += PG_BLOCK) {
    const int p = p0 + 4 * t;
    const pg_v4i r = load_refs(ref, p, num_pages);
    const int f[4] = {r.x <= 0 && p > 0 && p < num_pages, r.y <= 0 && p + 1 < num_pages,
                      r.z <= 0 && p + 2 < num_pages, r.w <= 0 && p + 3 < num_pages};
    const int mine = f[0] + f[1] + f[2] + f[3];
    int total;
    int at = found + group_incl_scan<PG_PLAN_THREADS>(mine, tot, total) - mine;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (f[e]) {
        if (at < need) free_list[at] = p + e;
        ++at;
      }
    found += total;
  }
  __syncthreads();  // the list is written
  int rank0 = 0;
  for (int i0 = 0; i0 < n; i0 += PG_PLAN_THREADS) {
    const int i = i0 + t;
    ForkRow f{-1, 0, false};
    if (i < n) f = fork_row(parents[i], ctx_len, B, max_pages, page_size);
    int total;
    const int rank = rank0 + group_incl_scan<PG_PLAN_THREADS>(f.part, tot, total) - (int)f.part;
    rank0 += total;
    if (i < n) pages[i] = f.parent < 0 ? -1 : !f.part ? 0 : rank < found ? free_list[rank] : -1;
  }
}

// Workgroup 0 of a child writes its table row and counts its pages (with_table), the others copy its last page's
// pieces.
__global__ __launch_bounds__(PG_THREADS) void pages_fork_kernel(
    PageCaches set, int with_table, int* __restrict__ ref, const int* __restrict__ table,
    const int* __restrict__ ctx_len, const int* __restrict__ parents, const int* __restrict__ pages,
    int* __restrict__ child, int B, int max_pages, int page_size, int num_pages) {
  const int per = set.pieces + with_table;
  const int i = blockIdx.x / per, piece = blockIdx.x % per - with_table;
  const int page = pages[i];
  const ForkRow f = fork_row(parents[i], ctx_len, B, max_pages, page_size);
  const int* row = table + (size_t)max(f.parent, 0) * max_pages;
  if (piece >= 0) {
    if (page > 0) copy_piece(set, piece, safe_page(row[f.full], num_pages), page);
    return;
  }
  int* out = child + (size_t)i * max_pages;
  for (int c = threadIdx.x; c < max_pages; c += PG_THREADS) {
    int p = 0;
    if (page >= 0) {
      if (c < f.full) p = safe_page(row[c], num_pages);
      else if (c == f.full && f.part) p = page;
    }
    out[c] = p;
    if (p && c == f.full) ref[p] = 1;  // (the new page is this child's alone, whatever its count was: 0 or less is free)
    else if (p) atomicAdd(ref + p, 1);
  }
}

// A row's pages, one use less each; a count never falls below 0. (A thread that finds no use left puts back what it
// took: a count is then below 0 only until it has, and one that found a use never needs to, so the sum of both does not
// depend on the order.)
__global__ __launch_bounds__(PG_THREADS) void pages_release_kernel(int* __restrict__ ref,
                                                                   const int* __restrict__ table,
                                                                   const int* __restrict__ ctx_len, int max_pages,
                                                                   int page_size, int num_pages) {
  const int i = blockIdx.x;
  const long cap = (long)max_pages * page_size;
  const long len = min(max((long)ctx_len[i], 0L), cap);
  const int n = (int)((len + page_size - 1) / page_size);
  const int* row = table + (size_t)i * max_pages;
  for (int c = threadIdx.x; c < n; c += PG_THREADS) {
    const int p = safe_page(row[c], num_pages);
    if (p && atomicSub(ref + p, 1) <= 0) atomicAdd(ref + p, 1);
  }
}

// -- compaction ---------------------------------------------------------------------------------------------------
// L live pages go to pages 1 .. L: those already there stay; the k-th live page past L moves to the k-th hole up to L.
// Moves read pages past L and write pages up to L, so they are independent of each other.

// Of four pages from p on those in use.
__device__ __forceinline__ int live_of(pg_v4i r, int p) {
  return (int)(r.x > 0 && p > 0) + (r.y > 0) + (r.z > 0) + (r.w > 0);
}

// Live pages of each block of PG_BLOCK.
__global__ __launch_bounds__(PG_PLAN_THREADS) void pages_count_kernel(const int* __restrict__ ref,
                                                                      int* __restrict__ counts, int num_pages) {
  __shared__ int tot[PG_PLAN_THREADS / WAVE];
  const int p = blockIdx.x * PG_BLOCK + 4 * threadIdx.x;
  int total;
  group_incl_scan<PG_PLAN_THREADS>(live_of(load_refs(ref, p, num_pages), p), tot, total);
  if (threadIdx.x == 0) counts[blockIdx.x] = total;
}

// code[p]: p where it stays, -(k + 1) where it is the k-th to move, 0 where it is free; holes[k], movers[k]; moves:
// their number. counts: the live pages of each block, or null where the workgroup counts them itself (up to PG_OWN
// blocks).
__global__ __launch_bounds__(PG_PLAN_THREADS) void pages_plan_kernel(const int* __restrict__ ref,
                                                                     const int* __restrict__ counts, int blocks,
                                                                     int* __restrict__ code, int* __restrict__ holes,
                                                                     int* __restrict__ movers, int* __restrict__ moves,
                                                                     int num_pages) {
  __shared__ int tot[PG_PLAN_THREADS / WAVE];
  __shared__ int own[PG_OWN];
  const int t = threadIdx.x, blk = blockIdx.x;
  int total, before = 0, live = 0, front = 0;
  if (!counts) {
    if (t < PG_OWN) own[t] = 0;
    __syncthreads();
#pragma unroll
    for (int b = 0; b < PG_OWN; ++b) {  // (past the pool: none)
      const pg_v4i r = load_refs(ref, b * PG_BLOCK + 4 * t, num_pages);
      const int n = __popcll(__ballot(r.x > 0 && b + t > 0)) + __popcll(__ballot(r.y > 0)) + __popcll(__ballot(r.z > 0)) +
                    __popcll(__ballot(r.w > 0));
      if ((t & (WAVE - 1)) == 0) atomicAdd(&own[b], n);
    }
    __syncthreads();
#pragma unroll
    for (int b = 0; b < PG_OWN; ++b) {
      live += own[b];
      before += b < blk ? own[b] : 0;
    }
#pragma unroll
    for (int b = 0; b < PG_OWN; ++b) front += b < live / PG_BLOCK ? own[b] : 0;
  } else {
    for (int b0 = 0; b0 < blocks; b0 += PG_PLAN_THREADS) {
      const int c = b0 + t < blocks ? counts[b0 + t] : 0;
      group_incl_scan<PG_PLAN_THREADS>(c, tot, total);
      live += total;
      group_incl_scan<PG_PLAN_THREADS>(b0 + t < blk ? c : 0, tot, total);
      before += total;
    }
    for (int b0 = 0; b0 < live / PG_BLOCK; b0 += PG_PLAN_THREADS) {
      group_incl_scan<PG_PLAN_THREADS>(b0 + t < live / PG_BLOCK ? counts[b0 + t] : 0, tot, total);
      front += total;
    }
  }
  // live pages up to page `live`: whole blocks before its own, so far, and its own up to it
  {
    const int p = live / PG_BLOCK * PG_BLOCK + 4 * t;
    const pg_v4i r = load_refs(ref, p, num_pages);
    const int up_to = (int)(r.x > 0 && p > 0 && p <= live) + (r.y > 0 && p + 1 <= live) + (r.z > 0 && p + 2 <= live) +
                      (r.w > 0 && p + 3 <= live);
    group_incl_scan<PG_PLAN_THREADS>(up_to, tot, total);
    front += total;
  }
  const int p = blk * PG_BLOCK + 4 * t;
  const pg_v4i r = load_refs(ref, p, num_pages);
  const int f[4] = {r.x > 0 && p > 0, r.y > 0, r.z > 0, r.w > 0};
  const int mine = f[0] + f[1] + f[2] + f[3];
  int at = before + group_incl_scan<PG_PLAN_THREADS>(mine, tot, total) - mine;  // live pages before this thread's
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int x = p + e;
    if (x < num_pages) {
      int c = 0;
      if (f[e]) {
        c = x;
        if (x > live) {
          c = -(at - front + 1);
          movers[at - front] = x;
        }
      } else if (x > 0 && x <= live) {
        holes[x - 1 - at] = x;
      }
      code[x] = c;
    }
    at += f[e];
  }
  if (blk == 0 && t == 0) *moves = live - front;
}

// The plan carried out: the tables, counts and map (with_table), and the moved pages of these caches.
__global__ __launch_bounds__(PG_THREADS) void pages_compact_kernel(
    PageCaches set, int with_table, const int* __restrict__ ref, const int* __restrict__ table,
    const int* __restrict__ code, const int* __restrict__ holes, const int* __restrict__ movers,
    const int* __restrict__ moves, int* __restrict__ new_ref, int* __restrict__ new_table, int* __restrict__ remap,
    long table_size, int num_pages) {
  const int n = *moves;
  const long units = (long)n * set.pieces;
  for (long u = blockIdx.x; u < units; u += gridDim.x) {
    const int k = (int)(u / set.pieces);
    copy_piece(set, (int)(u % set.pieces), movers[k], holes[k]);
  }
  if (!with_table) return;
  const long at = (long)blockIdx.x * PG_THREADS + threadIdx.x, step = (long)gridDim.x * PG_THREADS;
  for (long i = at; i < table_size; i += step) {
    const int c = code[safe_page(table[i], num_pages)];
    new_table[i] = c < 0 ? holes[-c - 1] : c;
  }
  for (long i = at; i < num_pages; i += step) {
    const int c = code[i];
    remap[i] = c < 0 ? holes[-c - 1] : c;
    // a free page up to the front's end is a hole, counted by the page that fills it (the holes ascend: the last one
    // bounds them); any other free page stays free
    if (c > 0) new_ref[i] = ref[i];
    else if (c < 0) new_ref[holes[-c - 1]] = ref[i], new_ref[i] = 0;
    else if (i == 0 || n == 0 || i > holes[n - 1]) new_ref[i] = 0;
  }
}

size_t pages_fork_bytes(int n) { return (size_t)n * 4; }

static int compact_blocks(int num_pages) { return (num_pages + PG_BLOCK - 1) / PG_BLOCK; }

size_t pages_compact_bytes(int num_pages) {  // counts, moves, code, holes, movers
  return ((size_t)compact_blocks(num_pages) + 1 + 3 * (size_t)num_pages) * 4;
}

// The caches from `at` on that one launch takes.
static PageCaches page_caches(void* const* caches, const long long* page_bytes, int n_caches, int at) {
  PageCaches s;
  s.n = n_caches - at < PG_CACHES ? n_caches - at : PG_CACHES;
  s.pieces = 0;
  for (int i = 0; i < s.n; ++i) {
    s.p[i] = caches[at + i];
    s.page_bytes[i] = page_bytes[at + i];
    s.first[i] = s.pieces;
    s.pieces += (int)((page_bytes[at + i] + PG_PIECE - 1) / PG_PIECE);
  }
  return s;
}

// Whether n pages' pieces number within a launch's workgroups.
bool pages_units_ok(const long long* page_bytes, int n_caches, long n) {
  long pieces = 1;
  for (int i = 0; i < n_caches; ++i) pieces += (long)((page_bytes[i] + PG_PIECE - 1) / PG_PIECE);
  return pieces <= 0xffffffL && pieces * n <= 0xffffffL;  // (x 256 threads: a launch's 2^32)
}

hipError_t launch_pages_copy(void* const* caches, const long long* page_bytes, int n_caches, const int* src,
                             const int* dst, int n, int num_pages, hipStream_t s) {
  for (int at = 0; at < n_caches; at += PG_CACHES) {
    const PageCaches set = page_caches(caches, page_bytes, n_caches, at);
    const hipError_t e = launch("pages_copy_kernel", pages_copy_kernel, dim3((unsigned)(n * set.pieces)),
                                dim3(PG_THREADS), s, set, src, dst, num_pages);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

hipError_t launch_pages_fork(int* ref, const int* table, const int* ctx_len, const int* parents, int* child,
                             int* pages, void* const* caches, const long long* page_bytes, int n_caches, void* ws,
                             int B, int n, int max_pages, int page_size, int num_pages, hipStream_t s) {
  hipError_t e = launch("pages_fork_plan_kernel", pages_fork_plan_kernel, dim3(1), dim3(PG_PLAN_THREADS), s, ref,
                        ctx_len, parents, pages, static_cast<int*>(ws), B, n, max_pages, page_size, num_pages);
  for (int at = 0; e == hipSuccess && (at == 0 || at < n_caches); at += PG_CACHES) {
    const PageCaches set = page_caches(caches, page_bytes, n_caches, at);
    const int first = at == 0;
    e = launch("pages_fork_kernel", pages_fork_kernel, dim3((unsigned)(n * (set.pieces + first))), dim3(PG_THREADS),
               s, set, first, ref, table, ctx_len, parents, pages, child, B, max_pages, page_size, num_pages);
  }
  return e;
}

hipError_t launch_pages_release(int* ref, const int* table, const int* ctx_len, int n, int max_pages, int page_size,
                                int num_pages, hipStream_t s) {
  return launch("pages_release_kernel", pages_release_kernel, dim3(n), dim3(PG_THREADS), s, ref, table, ctx_len,
                max_pages, page_size, num_pages);
}

hipError_t launch_pages_compact(const int* ref, const int* table, int* new_ref, int* new_table, int* remap,
                                void* const* caches, const long long* page_bytes, int n_caches, void* ws,
                                long table_size, int num_pages, int num_cu, hipStream_t s) {
  const int blocks = compact_blocks(num_pages);
  int* counts = static_cast<int*>(ws);
  int *moves = counts + blocks, *code = moves + 1, *holes = code + num_pages, *movers = holes + num_pages;
  const bool counted = blocks > PG_OWN;
  hipError_t e = hipSuccess;
  if (counted)
    e = launch("pages_count_kernel", pages_count_kernel, dim3(blocks), dim3(PG_PLAN_THREADS), s, ref, counts, num_pages);
  if (e == hipSuccess)
    e = launch("pages_plan_kernel", pages_plan_kernel, dim3(blocks), dim3(PG_PLAN_THREADS), s, ref,
               counted ? counts : nullptr, blocks,
               code, holes, movers, moves, num_pages);
  for (int at = 0; e == hipSuccess && (at == 0 || at < n_caches); at += PG_CACHES) {
    const PageCaches set = page_caches(caches, page_bytes, n_caches, at);
    // Up to 64 workgroups a CU, 8 of them at a time: as they come, what is being copied stays close together (12,345
    // pages: 8 a CU 73.5 us, 32 62.6, 64 60.8). No more than there can be moves, half the pages' (300 pages: 64 a CU
    // would take 6.3 us for 4.7).
    const long moved = (long)(num_pages / 2) * set.pieces;
    const long rows = (max(table_size, (long)num_pages) + PG_THREADS - 1) / PG_THREADS;
    const unsigned groups = (unsigned)min(max(moved, rows), 64L * num_cu);
    e = launch("pages_compact_kernel", pages_compact_kernel, dim3(groups), dim3(PG_THREADS), s, set,
               (int)(at == 0), ref, table, code, holes, movers, moves, new_ref, new_table, remap, table_size,
               num_pages);
  }
  return e;
}

}  // namespace dsa
