// paged_pages.hip — the pages of a paged cache between the steps of a batch:
// requests that go on, more than once or not at all, the pages nobody holds, pages
// moved together, and the copies that follow (gfx950).
#include "kv8.h"

#include <algorithm>

namespace dfattn {
namespace {

using namespace kv8;

constexpr uint32_t kMaxRows = 8192, kMaxPages = 1u << 24, kNone = DFATTN_NO_SLOT;
constexpr int kThreads = 256;

enum Mode { kFork, kFree, kCompact };

struct PagesArgs {
  const uint32_t *table, *lens, *parents, *keep, *ended;
  uint32_t *new_table, *new_lens, *refs, *order, *free_start, *src, *dst, *counts;
  // Workspace: per page the lowest row that writes behind its tokens in it and how many do
  // (compact: the page's move); per block of pages its free ones; the rows that need a page.
  uint32_t *owner, *lasts, *sums, *needers, *n_need;
  uint32_t R, N, W, P, n_pages, per_block, n_blocks, n_pairs, parts;
};

// Row i of the result: its row of the table and its length.
struct Row {
  uint32_t from, len, pages;
};
template <Mode M>
__device__ __forceinline__ Row row_of(const PagesArgs &a, uint32_t i) {
  Row r{M == kFork ? a.parents[i] : i, 0, 0};
  if (r.from < a.R) r.len = min(a.lens[r.from], a.W * a.P);
  if (M == kFork && a.keep != nullptr) r.len = min(r.len, a.keep[i]);
  if (M == kFree && a.ended != nullptr && a.ended[i] != 0) r.len = 0;
  r.pages = r.len / a.P + (r.len % a.P != 0);
  return r;
}
// The page that row i writes to behind its tokens, kNone where it starts a new one.
__device__ __forceinline__ uint32_t open_page(const PagesArgs &a, const Row &r) {
  if (r.len % a.P == 0) return kNone;
  const uint32_t p = a.table[(size_t)r.from * a.W + r.pages - 1];
  return p < a.n_pages ? p : kNone;
}

// The sum of x over the workgroup's threads before this one, and over all.
__device__ __forceinline__ uint32_t scan_block(uint32_t x, uint32_t *lds, uint32_t *total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t s = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t y = __shfl_up(s, o, 64);
    if (lane >= o) s += y;
  }
  __syncthreads();  // (the last call's sums have been read)
  if (lane == 63) lds[wave] = s;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    before += w < wave ? lds[w] : 0;
    all += lds[w];
  }
  *total = all;
  return before + s - x;
}

// Tables and page lists in four launches (five with moves), one dependent step each: 3 to 5 us of latency a launch
// for up to some 10^5 pages. Every sum is over fixed blocks in fixed order, and the atomics are integer ones,
// so results do not depend on the order of the work.

// 1: no references yet.
template <Mode M>
__global__ __launch_bounds__(kThreads) void clear_kernel(PagesArgs a) {
  const uint32_t id = blockIdx.x * kThreads + threadIdx.x, step = gridDim.x * kThreads;
  for (uint32_t p = id; p < a.n_pages; p += step) a.refs[p] = 0;
  for (uint32_t i = id; i < a.N; i += step) {
    if constexpr (M == kFork) {
      const uint32_t p = open_page(a, row_of<M>(a, i));
      if (p != kNone) {
        a.owner[p] = kNone;
        a.lasts[p] = 0;
      }
    }
    if (M == kFree && a.ended != nullptr && a.ended[i] != 0) a.new_lens[i] = 0;
  }
}

// 2: the references, and the new rows. A wave takes one of `parts` parts of a row. Bound by the rate of atomics on
// scattered words (2000 rows of 140 pages each 14.4 us, 20 a ns; counting in LDS would need all pages in one workgroup).
template <Mode M>
__global__ __launch_bounds__(kThreads) void count_kernel(PagesArgs a) {
  const uint32_t item = blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  const uint32_t i = item / a.parts, part = item % a.parts;
  if (i >= a.N) return;
  const Row r = row_of<M>(a, i);
  if (M == kFork && part == 0 && lane == 0) a.new_lens[i] = r.len;
  const uint32_t j0 = (uint32_t)((uint64_t)r.pages * part / a.parts), j1 = (uint32_t)((uint64_t)r.pages * (part + 1) / a.parts);
  const uint32_t *row = a.table + (size_t)r.from * a.W;
  for (uint32_t j = j0 + lane; j < j1; j += 64) {
    const uint32_t p = row[j];
    if constexpr (M == kFork) a.new_table[(size_t)i * a.W + j] = p;
    if (p >= a.n_pages) continue;
    atomicAdd(a.refs + p, 1u);
    if (M == kFork && j + 1 == r.pages && r.len % a.P != 0) {
      atomicMin(a.owner + p, i);
      atomicAdd(a.lasts + p, 1u);
    }
  }
}

// 3: the free pages of each block; the last workgroup finds the rows that need a page of their own, in order.
template <Mode M>
__global__ __launch_bounds__(kThreads) void sum_kernel(PagesArgs a) {
  __shared__ uint32_t lds[kThreads / 64];
  uint32_t n = 0, all;
  if (blockIdx.x < a.n_blocks) {
    const uint32_t p0 = blockIdx.x * a.per_block, p1 = min(a.n_pages, p0 + a.per_block);
    for (uint32_t p = p0 + threadIdx.x; p < p1; p += kThreads) n += a.refs[p] == 0;
    scan_block(n, lds, &all);
    if (threadIdx.x == 0) a.sums[blockIdx.x] = all;
    return;
  }
  uint32_t done = 0;
  for (uint32_t i0 = 0; i0 < a.N; i0 += kThreads) {
    const uint32_t i = i0 + threadIdx.x;
    bool need = false;
    if (i < a.N) {
      const uint32_t p = open_page(a, row_of<M>(a, i));
      if (p != kNone) {
        // (What is taken off here never makes a page free: its owner or a row that has it whole stays.)
        need = a.owner[p] != i || a.refs[p] != a.lasts[p];
      }
    }
    const uint32_t k = done + scan_block(need, lds, &all);
    if (need) a.needers[k] = i;
    done += all;
  }
  if (threadIdx.x == 0) *a.n_need = done;
}

// 4: the pages in the order used, free; the rows that need a page take the first free ones; the pages that move.
template <Mode M>
__global__ __launch_bounds__(kThreads) void place_kernel(PagesArgs a) {
  __shared__ uint32_t lds[kThreads / 64];
  uint32_t before = 0, all = 0;
  for (uint32_t b = threadIdx.x; b < a.n_blocks; b += kThreads) {
    const uint32_t s = a.sums[b];
    before += b < blockIdx.x ? s : 0;
    all += s;
  }
  uint32_t free_before, n_free;
  scan_block(before, lds, &free_before);
  scan_block(all, lds, &n_free);
  const uint32_t used = a.n_pages - n_free;
  const uint32_t p0 = blockIdx.x * a.per_block, p1 = min(a.n_pages, p0 + a.per_block);
  uint32_t need = 0, holes = 0;
  if constexpr (M == kFork) need = *a.n_need;
  if constexpr (M == kCompact) {  // the free pages below `used`
    const uint32_t edge = used / a.per_block;
    uint32_t x = 0;
    for (uint32_t b = threadIdx.x; b < edge; b += kThreads) x += a.sums[b];
    for (uint32_t p = edge * a.per_block + threadIdx.x; p < used; p += kThreads) x += a.refs[p] == 0;
    scan_block(x, lds, &holes);
  }
  uint32_t f = free_before;
  for (uint32_t q = p0; q < p1; q += kThreads) {
    const uint32_t p = q + threadIdx.x;
    const bool in = p < p1, free = in && a.refs[p] == 0;
    uint32_t here;
    const uint32_t k = f + scan_block(free, lds, &here);  // free pages before p
    f += here;
    if (!in) continue;
    if constexpr (M == kCompact) {
      a.order[p] = p;
      if (free && p < used) a.dst[k] = p;
      if (!free && p >= used) {
        const uint32_t m = p - k - (used - holes);
        a.src[m] = p;
        a.owner[p] = m;
      }
    } else {
      a.order[free ? used + k : p - k] = p;
      if (M == kFork && free && k < need) {
        const uint32_t i = a.needers[k];
        const Row r = row_of<M>(a, i);
        const size_t last = (size_t)i * a.W + r.pages - 1;
        const uint32_t old = a.table[(size_t)r.from * a.W + r.pages - 1];
        a.new_table[last] = p;
        a.refs[p] = 1;
        atomicSub(a.refs + old, 1u);
        a.src[k] = old;
        a.dst[k] = p;
      }
    }
  }
  if (blockIdx.x != 0) return;
  const uint32_t pairs = M == kFork ? min(need, n_free) : holes;
  if (threadIdx.x == 0) {
    *a.free_start = used + (M == kFork ? pairs : 0);
    if constexpr (M != kFree) a.counts[0] = pairs;
    if constexpr (M == kFork) a.counts[1] = need - pairs;
  }
  if constexpr (M != kFree)
    for (uint32_t k = pairs + threadIdx.x; k < a.n_pairs; k += kThreads) a.src[k] = a.dst[k] = kNone;
  if constexpr (M == kFork)
    for (uint32_t k = pairs + threadIdx.x; k < need; k += kThreads) {
      const uint32_t i = a.needers[k];
      const Row r = row_of<M>(a, i);
      a.new_lens[i] = r.len / a.P * a.P;
      atomicSub(a.refs + a.table[(size_t)r.from * a.W + r.pages - 1], 1u);
    }
}

// 5 (compact): the tables' ids and the references follow.
__global__ __launch_bounds__(kThreads) void rename_kernel(PagesArgs a) {
  const uint32_t item = blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  const uint32_t used = *a.free_start, moves = *a.counts, step = gridDim.x * kThreads;
  for (uint32_t m = blockIdx.x * kThreads + threadIdx.x; m < moves; m += step) {
    const uint32_t from = a.src[m];
    a.refs[a.dst[m]] = a.refs[from];
    a.refs[from] = 0;
  }
  const uint32_t i = item / a.parts, part = item % a.parts;
  if (i >= a.N) return;
  const Row r = row_of<kCompact>(a, i);
  const uint32_t j0 = (uint32_t)((uint64_t)r.pages * part / a.parts), j1 = (uint32_t)((uint64_t)r.pages * (part + 1) / a.parts);
  for (uint32_t j = j0 + lane; j < j1; j += 64) {
    const uint32_t p = a.table[(size_t)i * a.W + j];
    a.new_table[(size_t)i * a.W + j] = p >= used && p < a.n_pages ? a.dst[a.owner[p]] : p;
  }
}

// ---------------------------------------------------------------- small batches: one workgroup, one launch
constexpr int kSmallThreads = 1024, kSmallWaves = kSmallThreads / 64;
constexpr uint32_t kSmallPages = 8192, kSmallRows = 128, kStrips = kSmallPages / kSmallThreads;  // (kSmallRows: of up to 64 pages)

// The five steps above with everything in LDS between barriers: bound by the latency of one workgroup's steps, where the launches
// above have theirs five times. Replayed from a graph, fork / free / compact, here and above: 8 rows of up to 64 pages of 1500
// 4.4, 3.5, 4.4 us and 10.7, 8.8, 12.1; 128 rows of 8192 pages 8.5, 7.7, 11.9 and 11.0, 9.1, 13.3; 256 rows 15, 13, 24 and
// 11.5, 9.1, 13.
template <Mode M>
__global__ __launch_bounds__(kSmallThreads) void small_kernel(PagesArgs a) {
  // first, last: fork: the lowest row that writes in a page and how many do; compact: the pages that move, and where to.
  __shared__ uint32_t refs[kSmallPages], first[M == kFree ? 1 : kSmallPages], last[M == kFree ? 1 : kSmallPages];
  __shared__ uint32_t from[M == kFork ? kSmallRows : 1], pages[kSmallRows], opened[M == kFork ? kSmallRows : 1];
  __shared__ uint32_t counts[kStrips * kSmallWaves], holes_lds, needs;
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (uint32_t p = tid; p < a.n_pages; p += kSmallThreads) {
    refs[p] = 0;
    if constexpr (M == kFork) {
      first[p] = kNone;
      last[p] = 0;
    }
  }
  if (tid < kStrips * kSmallWaves) counts[tid] = 0;
  if (tid == 0) holes_lds = 0;
  for (uint32_t i = tid; i < a.N; i += kSmallThreads) {
    const Row r = row_of<M>(a, i);
    pages[i] = r.pages;
    if constexpr (M == kFork) {
      from[i] = r.from;
      opened[i] = open_page(a, r);
      a.new_lens[i] = r.len;
    }
    if (M == kFree && a.ended != nullptr && a.ended[i] != 0) a.new_lens[i] = 0;
  }
  __syncthreads();
  // Every entry of every row: 1 to 16 waves side by side on a row, 64 entries each at a time.
  uint32_t side = 1;
  while (side < kSmallWaves && side * 64 < a.W) side *= 2;
  auto entries = [&](auto row, auto use) {
    for (uint32_t i = wave / side; i < a.N; i += kSmallWaves / side) {
      const uint32_t *at = a.table + (size_t)row(i) * a.W;
      for (uint32_t j = wave % side * 64 + lane; j < pages[i]; j += side * 64) use(i, j, at[j]);
    }
  };
  entries([&](uint32_t i) { return M == kFork ? from[i] : i; }, [&](uint32_t i, uint32_t j, uint32_t p) {
    if constexpr (M == kFork) a.new_table[(size_t)i * a.W + j] = p;
    if (p < a.n_pages) atomicAdd(refs + p, 1u);
  });
  if constexpr (M == kFork)
    for (uint32_t i = tid; i < a.N; i += kSmallThreads)
      if (opened[i] != kNone) {
        atomicMin(first + opened[i], i);
        atomicAdd(last + opened[i], 1u);
      }
  __syncthreads();
  // The free pages of each 64.
  for (uint32_t strip = 0; strip * kSmallThreads < a.n_pages; ++strip) {
    const uint32_t p = strip * kSmallThreads + tid;
    const uint64_t free = __ballot(p < a.n_pages && refs[p] == 0);
    if (lane == 0) counts[strip * kSmallWaves + wave] = __popcll(free);
  }
  uint32_t need = 0;
  if constexpr (M == kFork) {
    if (wave == 0) {  // (the rows in order; their places go where their pages were)
      for (uint32_t i0 = 0; i0 < a.N; i0 += 64) {
        const uint32_t i = i0 + lane, p = i < a.N ? opened[i] : kNone;
        const bool takes = p != kNone && (first[p] != i || refs[p] != last[p]);
        const uint64_t who = __ballot(takes);
        if (takes) from[need + __popcll(who & ((1ull << lane) - 1))] = i;  // (`from` has been read)
        need += __popcll(who);
      }
      if (lane == 0) needs = need;
    }
  }
  __syncthreads();
  if constexpr (M == kFork) need = needs;
  if (wave == 0) {  // sums before each 64, over all
    static_assert(kStrips * kSmallWaves == 128, "two a lane");
    const uint32_t x = counts[2 * lane], y = counts[2 * lane + 1];
    uint32_t s = x + y;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t t = __shfl_up(s, o, 64);
      if ((int)lane >= o) s += t;
    }
    counts[2 * lane] = s - x - y;
    counts[2 * lane + 1] = s - y;
    if (lane == 63) holes_lds = s;
  }
  __syncthreads();
  const uint32_t n_free = holes_lds, used = a.n_pages - n_free;
  if constexpr (M == kCompact) {
    __syncthreads();
    for (uint32_t strip = 0; strip * kSmallThreads < a.n_pages; ++strip) {
      const uint32_t p = strip * kSmallThreads + tid;
      const bool free = p < a.n_pages && refs[p] == 0;
      const uint32_t k = counts[strip * kSmallWaves + wave] + __popcll(__ballot(free) & ((1ull << lane) - 1));
      if (p >= a.n_pages) continue;
      a.order[p] = p;
      if (free && p < used) last[k] = p;  // the m-th free page below
      if (p == used) holes_lds = k;
      if (p + 1 == a.n_pages && used == a.n_pages) holes_lds = 0;
    }
    __syncthreads();
    const uint32_t moves = holes_lds;
    for (uint32_t strip = 0; strip * kSmallThreads < a.n_pages; ++strip) {
      const uint32_t p = strip * kSmallThreads + tid;
      const bool free = p < a.n_pages && refs[p] == 0;
      const uint32_t k = counts[strip * kSmallWaves + wave] + __popcll(__ballot(free) & ((1ull << lane) - 1));
      if (p >= a.n_pages) continue;
      if (p < used) {
        if (!free) a.refs[p] = refs[p];
        continue;
      }
      a.refs[p] = 0;
      if (free) continue;
      const uint32_t m = p - k - (used - moves), to = last[m];
      first[p] = to;
      a.src[m] = p;
      a.dst[m] = to;
      a.refs[to] = refs[p];
    }
    for (uint32_t k = moves + tid; k < a.n_pairs; k += kSmallThreads) a.src[k] = a.dst[k] = kNone;
    if (tid == 0) {
      *a.free_start = used;
      a.counts[0] = moves;
    }
    __syncthreads();
    entries([](uint32_t i) { return i; }, [&](uint32_t i, uint32_t j, uint32_t p) {
      a.new_table[(size_t)i * a.W + j] = p >= used && p < a.n_pages ? first[p] : p;
    });
    return;
  }
  const uint32_t pairs = M == kFork ? min(need, n_free) : 0;
  if constexpr (M == kFork)
    for (uint32_t k = tid; k < a.N; k += kSmallThreads) {
      if (k >= pairs) a.src[k] = a.dst[k] = kNone;
      if (k >= need) continue;
      const uint32_t i = from[k];
      atomicSub(refs + opened[i], 1u);  // (never to 0: the page's owner, or a row that has it whole, stays)
      if (k >= pairs) a.new_lens[i] = row_of<M>(a, i).len / a.P * a.P;
    }
  __syncthreads();
  for (uint32_t strip = 0; strip * kSmallThreads < a.n_pages; ++strip) {
    const uint32_t p = strip * kSmallThreads + tid;
    const uint32_t n = p < a.n_pages ? refs[p] : 1;
    const uint32_t k = counts[strip * kSmallWaves + wave] + __popcll(__ballot(n == 0) & ((1ull << lane) - 1));
    if (p >= a.n_pages) continue;
    a.order[n == 0 ? used + k : p - k] = p;
    const bool taken = M == kFork && n == 0 && k < pairs;
    a.refs[p] = taken ? 1 : n;
    if (M == kFork && taken) {
      const uint32_t i = from[k];
      a.new_table[(size_t)i * a.W + pages[i] - 1] = p;
      a.src[k] = opened[i];
      a.dst[k] = p;
    }
  }
  if (tid == 0) {
    *a.free_start = used + pairs;
    if constexpr (M == kFork) {
      a.counts[0] = pairs;
      a.counts[1] = need - pairs;
    }
  }
}

// ---------------------------------------------------------------- copies
struct Pool {
  char *data;
  uint32_t units, log2;  // units of 2^log2 bytes a page
};
constexpr uint32_t kPoolsPerLaunch = 128;
struct CopyArgs {
  const uint32_t *src, *dst, *count;
  uint32_t max_copies, n_pages;
  Pool pools[kPoolsPerLaunch];
};

template <typename T>
__device__ __forceinline__ void copy_pool(const CopyArgs &a, T *data, uint32_t units, uint32_t n) {
  constexpr int kAtOnce = 4;
  const uint64_t total = (uint64_t)n * units;
  for (uint64_t u0 = (uint64_t)blockIdx.x * kThreads * kAtOnce; u0 < total; u0 += (uint64_t)gridDim.x * kThreads * kAtOnce) {
    const uint32_t pair0 = (uint32_t)(u0 / units), at0 = (uint32_t)(u0 % units);
    T x[kAtOnce];
    T *to[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const uint64_t at = (uint64_t)at0 + j * kThreads + threadIdx.x;
      const uint32_t over = (uint32_t)(at / units), rest = (uint32_t)(at % units);
      to[j] = nullptr;
      if (u0 + j * kThreads + threadIdx.x >= total) continue;
      const uint32_t s = a.src[pair0 + over], d = a.dst[pair0 + over];
      if (s >= a.n_pages || d >= a.n_pages) continue;
      to[j] = data + (size_t)d * units + rest;
      x[j] = data[(size_t)s * units + rest];
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j)
      if (to[j] != nullptr) *to[j] = x[j];
  }
}

// Pages of many units: a workgroup copies kPiece of one page at a time. The copies are not
// read again soon, so their stores pass the caches by (80 MB copied 25 us, 27 with plain ones).
constexpr uint32_t kPieceSteps = 4, kPiece = kPieceSteps * kThreads;
__device__ __forceinline__ void copy_pages(const CopyArgs &a, u32x4 *data, uint32_t units, uint32_t n) {
  const uint32_t pieces = (units + kPiece - 1) / kPiece;
  const uint64_t total = (uint64_t)n * pieces;
  for (uint64_t item = blockIdx.x; item < total; item += gridDim.x) {
    const uint32_t pair = (uint32_t)(item / pieces), at = (uint32_t)(item % pieces) * kPiece + threadIdx.x;
    const uint32_t s = a.src[pair], d = a.dst[pair];
    if (s >= a.n_pages || d >= a.n_pages) continue;
    const u32x4 *from = data + (size_t)s * units;
    u32x4 *to = data + (size_t)d * units, x[kPieceSteps];
#pragma unroll
    for (uint32_t j = 0; j < kPieceSteps; ++j)
      if (at + j * kThreads < units) x[j] = from[at + j * kThreads];
#pragma unroll
    for (uint32_t j = 0; j < kPieceSteps; ++j)
      if (at + j * kThreads < units) __builtin_nontemporal_store(x[j], to + at + j * kThreads);
  }
}

__global__ __launch_bounds__(kThreads) void copy_kernel(CopyArgs a) {
  const Pool pool = a.pools[blockIdx.y];
  const uint32_t n = a.count != nullptr ? min(*a.count, a.max_copies) : a.max_copies;
  if (pool.log2 == 4 && pool.units >= kThreads)
    copy_pages(a, reinterpret_cast<u32x4 *>(pool.data), pool.units, n);
  else if (pool.log2 == 4)
    copy_pool(a, reinterpret_cast<u32x4 *>(pool.data), pool.units, n);
  else if (pool.log2 == 2)
    copy_pool(a, reinterpret_cast<uint32_t *>(pool.data), pool.units, n);
  else
    copy_pool(a, reinterpret_cast<unsigned char *>(pool.data), pool.units, n);
}

// ---------------------------------------------------------------- host
struct Span {
  const void *p;
  size_t bytes;
};
bool overlap(const Span &x, const Span &y) {
  const char *a = static_cast<const char *>(x.p), *b = static_cast<const char *>(y.p);
  return x.bytes > 0 && y.bytes > 0 && a != nullptr && b != nullptr && a < b + y.bytes && b < a + x.bytes;
}

int check_pages(const char *fn, uint32_t n_requests, uint32_t n_rows, uint32_t max_pages, uint32_t page_size,
                uint32_t n_pages) {
  if (n_requests == 0 || n_rows == 0 || max_pages == 0 || page_size == 0 || n_pages == 0)
    return record_error(DFATTN_ERR_SHAPE, std::string(fn) + ": the numbers of rows and pages and page_size must be >= 1");
  if (n_requests > kMaxRows || n_rows > kMaxRows || n_pages > kMaxPages || (uint64_t)n_pages * page_size > (1ull << 31) ||
      (uint64_t)max_pages * page_size > (1ull << 31))
    return record_error(DFATTN_ERR_OVERFLOW, std::string(fn) + ": shape is too large");
  return DFATTN_OK;
}

uint32_t pages_per_block(uint32_t n_pages) { return std::max(256u, ((n_pages + 1023) / 1024 + 255) & ~255u); }

size_t workspace_bytes_for(uint32_t n_rows, uint32_t n_pages) {
  return 4 * (2 * (size_t)n_pages + 1024 + n_rows + 1);
}

// Parts of a row to a wave each, so that there are some 4096 waves.
uint32_t row_parts(uint32_t n_rows, uint32_t max_pages) {
  return std::max(1u, std::min((max_pages + 63) / 64, 4096 / n_rows));
}

template <Mode M>
int run_pages(const char *fn, PagesArgs &a, void *workspace, size_t workspace_bytes, hipStream_t stream) {
  if (workspace == nullptr || workspace_bytes < workspace_bytes_for(a.N, a.n_pages))
    return record_error(DFATTN_ERR_WORKSPACE, std::string(fn) + ": the workspace is too small");
  if (!aligned_to(workspace, 4)) return record_error(DFATTN_ERR_MISALIGNED, std::string(fn) + ": misaligned pointer");
  if (a.n_pages <= kSmallPages && (uint64_t)a.N * ((a.W + 63) / 64) <= kSmallRows) {
    hipLaunchKernelGGL(small_kernel<M>, dim3(1), dim3(kSmallThreads), 0, stream, a);
    return launched(fn);
  }
  a.owner = static_cast<uint32_t *>(workspace);
  a.lasts = a.owner + a.n_pages;
  a.sums = a.lasts + a.n_pages;
  a.needers = a.sums + 1024;
  a.n_need = a.needers + a.N;
  a.per_block = pages_per_block(a.n_pages);
  a.n_blocks = (a.n_pages + a.per_block - 1) / a.per_block;
  a.parts = row_parts(a.N, a.W);
  const uint32_t fill = std::min(1024u, (std::max(a.n_pages, a.N) + kThreads - 1) / kThreads);
  const uint32_t rows = (a.N * a.parts + kThreads / 64 - 1) / (kThreads / 64);
  hipLaunchKernelGGL(clear_kernel<M>, dim3(fill), dim3(kThreads), 0, stream, a);
  hipLaunchKernelGGL(count_kernel<M>, dim3(rows), dim3(kThreads), 0, stream, a);
  hipLaunchKernelGGL(sum_kernel<M>, dim3(a.n_blocks + (M == kFork)), dim3(kThreads), 0, stream, a);
  hipLaunchKernelGGL(place_kernel<M>, dim3(a.n_blocks), dim3(kThreads), 0, stream, a);
  if constexpr (M == kCompact) hipLaunchKernelGGL(rename_kernel, dim3(rows), dim3(kThreads), 0, stream, a);
  return launched(fn);
}

// Nothing that is written may overlap what is read, or another output.
int check_spans(const char *fn, const Span *spans, int n_out, int n) {
  for (int i = 0; i < n_out; ++i)
    for (int j = i + 1; j < n; ++j)
      if (overlap(spans[i], spans[j]))
        return record_error(DFATTN_ERR_SHAPE, std::string(fn) + ": outputs must not overlap inputs or each other");
  return DFATTN_OK;
}

}  // namespace
}  // namespace dfattn

using namespace dfattn;
using namespace dfattn::kv8;

extern "C" {

size_t dfattn_paged_workspace_bytes(uint32_t n_rows, uint32_t n_pages) {
  if (n_rows == 0 || n_rows > kMaxRows || n_pages == 0 || n_pages > kMaxPages) return 0;
  return workspace_bytes_for(n_rows, n_pages);
}

int dfattn_paged_fork(const uint32_t *block_table, const uint32_t *seq_lens, const uint32_t *parents,
                      const uint32_t *keep_lens, uint32_t *new_table, uint32_t *new_lens, uint32_t *refs,
                      uint32_t *free_pages, uint32_t *free_start, uint32_t *copy_src, uint32_t *copy_dst,
                      uint32_t *counts, uint32_t n_requests, uint32_t n_children, uint32_t max_pages, uint32_t page_size,
                      uint32_t n_pages, void *workspace, size_t workspace_bytes, void *stream) {
  const char *fn = "dfattn_paged_fork";
  int st = check_pages(fn, n_requests, n_children, max_pages, page_size, n_pages);
  if (st == DFATTN_OK)
    st = check_all(fn, {block_table, seq_lens, parents, new_table, new_lens, refs, free_pages, free_start, copy_src,
                        copy_dst, counts}, 4);
  if (st == DFATTN_OK && keep_lens != nullptr) st = check_all(fn, {keep_lens}, 4);
  if (st != DFATTN_OK) return st;
  const size_t r = 4 * (size_t)n_requests, c = 4 * (size_t)n_children, p = 4 * (size_t)n_pages;
  const Span spans[] = {{new_table, c * max_pages}, {new_lens, c}, {refs, p}, {free_pages, p}, {free_start, 4}, {copy_src, c},
                        {copy_dst, c}, {counts, 8}, {workspace, workspace_bytes_for(n_children, n_pages)},
                        {block_table, r * max_pages}, {seq_lens, r}, {parents, c}, {keep_lens, c}};
  st = check_spans(fn, spans, 9, 13);
  if (st != DFATTN_OK) return st;
  PagesArgs a{};
  a.table = block_table;
  a.lens = seq_lens;
  a.parents = parents;
  a.keep = keep_lens;
  a.new_table = new_table;
  a.new_lens = new_lens;
  a.refs = refs;
  a.order = free_pages;
  a.free_start = free_start;
  a.src = copy_src;
  a.dst = copy_dst;
  a.counts = counts;
  a.R = n_requests;
  a.N = n_children;
  a.W = max_pages;
  a.P = page_size;
  a.n_pages = n_pages;
  a.n_pairs = n_children;
  return run_pages<kFork>(fn, a, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

int dfattn_paged_free(const uint32_t *block_table, uint32_t *seq_lens, const uint32_t *ended, uint32_t *refs,
                      uint32_t *free_pages, uint32_t *free_start, uint32_t n_requests, uint32_t max_pages,
                      uint32_t page_size, uint32_t n_pages, void *workspace, size_t workspace_bytes, void *stream) {
  const char *fn = "dfattn_paged_free";
  int st = check_pages(fn, n_requests, n_requests, max_pages, page_size, n_pages);
  if (st == DFATTN_OK) st = check_all(fn, {block_table, seq_lens, refs, free_pages, free_start}, 4);
  if (st == DFATTN_OK && ended != nullptr) st = check_all(fn, {ended}, 4);
  if (st != DFATTN_OK) return st;
  const size_t r = 4 * (size_t)n_requests, p = 4 * (size_t)n_pages;
  const Span spans[] = {{seq_lens, r}, {refs, p}, {free_pages, p}, {free_start, 4},
                        {workspace, workspace_bytes_for(n_requests, n_pages)}, {block_table, r * max_pages}, {ended, r}};
  st = check_spans(fn, spans, 5, 7);
  if (st != DFATTN_OK) return st;
  PagesArgs a{};
  a.table = block_table;
  a.lens = seq_lens;
  a.ended = ended;
  a.new_lens = seq_lens;
  a.refs = refs;
  a.order = free_pages;
  a.free_start = free_start;
  a.R = a.N = n_requests;
  a.W = max_pages;
  a.P = page_size;
  a.n_pages = n_pages;
  return run_pages<kFree>(fn, a, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

int dfattn_paged_compact(const uint32_t *block_table, const uint32_t *seq_lens, uint32_t *new_table, uint32_t *refs,
                         uint32_t *free_pages, uint32_t *free_start, uint32_t *copy_src, uint32_t *copy_dst,
                         uint32_t *counts, uint32_t n_requests, uint32_t max_pages, uint32_t page_size, uint32_t n_pages,
                         void *workspace, size_t workspace_bytes, void *stream) {
  const char *fn = "dfattn_paged_compact";
  int st = check_pages(fn, n_requests, n_requests, max_pages, page_size, n_pages);
  if (st == DFATTN_OK) st = check_all(fn, {block_table, seq_lens, new_table, refs, free_pages, free_start, counts}, 4);
  if (st == DFATTN_OK && n_pages > 1) st = check_all(fn, {copy_src, copy_dst}, 4);
  if (st != DFATTN_OK) return st;
  const size_t r = 4 * (size_t)n_requests, p = 4 * (size_t)n_pages, m = 4 * (size_t)(n_pages / 2);
  const Span spans[] = {{new_table, r * max_pages}, {refs, p}, {free_pages, p}, {free_start, 4}, {copy_src, m}, {copy_dst, m},
                        {counts, 4}, {workspace, workspace_bytes_for(n_requests, n_pages)}, {seq_lens, r},
                        {new_table == block_table ? nullptr : block_table, r * max_pages}};
  st = check_spans(fn, spans, 8, 10);
  if (st != DFATTN_OK) return st;
  PagesArgs a{};
  a.table = block_table;
  a.lens = seq_lens;
  a.new_table = new_table;
  a.refs = refs;
  a.order = free_pages;
  a.free_start = free_start;
  a.src = copy_src;
  a.dst = copy_dst;
  a.counts = counts;
  a.R = a.N = n_requests;
  a.W = max_pages;
  a.P = page_size;
  a.n_pages = n_pages;
  a.n_pairs = n_pages / 2;
  return run_pages<kCompact>(fn, a, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

int dfattn_paged_copy(const void *pools, uint32_t n_pools, const uint32_t *copy_src, const uint32_t *copy_dst,
                      const uint32_t *n_copies, uint32_t max_copies, uint32_t n_pages, void *stream) {
  const char *fn = "dfattn_paged_copy";
  if (n_pages == 0) return record_error(DFATTN_ERR_SHAPE, std::string(fn) + ": n_pages must be >= 1");
  if (n_pages > kMaxPages || n_pools > 65535u || max_copies > kMaxPages)
    return record_error(DFATTN_ERR_OVERFLOW, std::string(fn) + ": shape is too large");
  if (n_pools == 0 || max_copies == 0) return DFATTN_OK;
  int st = check_all(fn, {pools}, alignof(dfattn_page_pool));
  if (st == DFATTN_OK) st = check_all(fn, {copy_src, copy_dst}, 4);
  if (st == DFATTN_OK && n_copies != nullptr) st = check_all(fn, {n_copies}, 4);
  if (st != DFATTN_OK) return st;
  const dfattn_page_pool *given = static_cast<const dfattn_page_pool *>(pools);
  for (uint32_t i = 0; i < n_pools; ++i) {
    if (given[i].data == nullptr) return record_error(DFATTN_ERR_NULL_POINTER, std::string(fn) + ": null pointer");
    if (given[i].page_bytes == 0)
      return record_error(DFATTN_ERR_SHAPE, std::string(fn) + ": a page must have at least one byte");
    if (given[i].page_bytes > (1ull << 30))
      return record_error(DFATTN_ERR_OVERFLOW, std::string(fn) + ": a page has more than 2^30 bytes");
  }
  CopyArgs a{};
  a.src = copy_src;
  a.dst = copy_dst;
  a.count = n_copies;
  a.max_copies = max_copies;
  a.n_pages = n_pages;
  for (uint32_t i0 = 0; i0 < n_pools; i0 += kPoolsPerLaunch) {
    const uint32_t n = std::min(kPoolsPerLaunch, n_pools - i0);
    uint64_t most = 0;
    for (uint32_t i = 0; i < n; ++i) {
      const dfattn_page_pool &p = given[i0 + i];
      const bool four = aligned_to(p.data, 4) && p.page_bytes % 4 == 0;
      const uint32_t log2 = aligned_to(p.data, 16) && p.page_bytes % 16 == 0 ? 4 : four ? 2 : 0;
      a.pools[i] = {static_cast<char *>(p.data), (uint32_t)(p.page_bytes >> log2), log2};
      most = std::max(most, (uint64_t)max_copies * a.pools[i].units);
    }
    // Up to 4096 workgroups in all (1.2 GB of 32 KB pages 254 us, with 2048 266, with 8192 249; but 300 a us start, also
    // where *n_copies turns out to be small).
    const uint32_t each = std::max(1u, 4096 / n);
    const uint32_t groups = (uint32_t)std::min<uint64_t>(each, (most + 4 * kThreads - 1) / (4 * kThreads));
    hipLaunchKernelGGL(copy_kernel, dim3(groups, n), dim3(kThreads), 0, static_cast<hipStream_t>(stream), a);
  }
  return launched(fn);
}

}  // extern "C"
