// Pages of a paged key/value cache as a pool with reference counts: hi_cache_fork makes every row of a page table the
// continuation of another (beams after a selection, several answers to one prompt, new and ended sequences), hi_cache_compact
// moves the pages in use to the front of the pool.
//
// Both are a plan by one block and a launch that carries it out on the whole GPU. What a plan has to find is small (which pages are
// free, in order) but global: 4 bytes a page, read by 1024 threads, 16 pages each at a time. Everything is found on the device, so
// both can be captured; results do not depend on the order of blocks: pages are handed out in ascending order to rows in ascending
// order, and the only atomics are sums and minima of integers.
#include <climits>

#include "hi_common.h"
#include "row_overlap.h"

namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPerThread = 16;      // pages that a thread of a plan looks at in one step
constexpr int kMaxPages = 1 << 30;  // of a pool
constexpr int kMaxRows = 8192;      // rows of a table: a fork's plan keeps 8 bytes of each old row and of each new one in LDS
constexpr int kSetMax = 128;        // cache tensors of one launch: their addresses are kernel arguments (3 KB)
constexpr int kPart = 4096;         // bytes of a page that a wave copies at a time: 4 loads of 16 bytes a lane
constexpr int kSmall = 64;          // pages of at most so many bytes are copied by a lane
constexpr int kListed = 4096;       // free pages that a fork's plan keeps there
constexpr size_t fork_lds(int S, int N) { return (2 * (size_t)S + 2 * (size_t)N + kListed) * 4; }
static_assert(fork_lds(kMaxRows, kMaxRows) + kPlanThreads / 64 * 8 <= 160 * 1024, "a fork's plan and its sums fit a CU's LDS");

// One cache tensor: pages `stride` bytes apart. A page's `bytes` are `runs` runs of one value per position, or with runs 0
// belong to the page as a whole.
struct CacheDesc {
  char* p;
  int64_t stride;
  uint32_t bytes;
  uint32_t runs_unit;  // runs << 5 | bytes of an access (16, 4 or 1)
};
struct CacheSet {
  CacheDesc d[kSetMax];  // those with pages of over kSmall bytes first
  int n, large, parts;   // tensors, the large ones, and parts of kPart bytes that the largest page has
};

// A copy of page src to page dst, of the first `rows` positions (a whole page: `page` of them).
struct Move {
  int src, dst, rows;
};

// The front of a work buffer, filled by a plan.
struct PlanHead {
  int free;   // free pages that were found (fork: at most as many as asked for)
  int moves;  // copies, in `moves`
  int used;   // pages in use (compact)
  int pad;
};

struct WorkLayout {
  size_t count, first, base, list, moves, bytes;
  __host__ __device__ WorkLayout(int S, int N, int pages) {
    const auto up = [](size_t v) { return (v + 15) & ~(size_t)15; };
    count = sizeof(PlanHead);
    first = up(count + (size_t)S * 4);
    base = up(first + (size_t)S * 4);
    list = up(base + (size_t)N * 4);
    moves = up(list + (size_t)pages * 4);
    // copies: of a fork at most one a row, of a compaction at most half of the pages
    bytes = up(moves + (size_t)(N > pages / 2 ? N : pages / 2) * sizeof(Move));
  }
};

// Exclusive sum over the block of v, and the total; sh: one number per wave.
template <typename T>
__device__ __forceinline__ T block_scan(T v, int64_t* sh, T& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  T x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const T y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  __syncthreads();  // the sums of the last call have been read
  if (lane == 63) sh[wave] = x;
  __syncthreads();
  T before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 64; w++) {
    const T s = (T)sh[w];
    if (w < wave) before += s;
    total += s;
  }
  return before + x - v;
}

// The counts of 16 pages from p0 on (used: 1, counts as such behind the end).
__device__ __forceinline__ void load_counts(const int* refs, int pages, int p0, bool wide, int (&r)[kPerThread]) {
  if (wide && p0 + kPerThread <= pages) {
#pragma unroll
    for (int k = 0; k < kPerThread / 4; k++) {
      const u32x4 v = *reinterpret_cast<const u32x4*>(refs + p0 + 4 * k);
#pragma unroll
      for (int e = 0; e < 4; e++) r[4 * k + e] = (int)v[e];
    }
  } else {
#pragma unroll
    for (int k = 0; k < kPerThread; k++) r[k] = p0 + k < pages ? refs[p0 + k] : 1;
  }
}

struct ForkArgs {
  const int *table, *lens, *parent, *refs;
  int *table_out, *lens_out, *refs_out, *missing;
  char* work;
  int ldt, ldo, W, S, N, pages, grow, page, shift;

  __device__ __forceinline__ bool has(int id) const { return (unsigned)id < (unsigned)pages; }
  __device__ __forceinline__ int parent_of(int i) const {
    const int p = parent[i];
    return (unsigned)p < (unsigned)S ? p : -1;
  }
  __device__ __forceinline__ int len(int row) const { return min(max(lens[row], 0), W << shift); }
  __device__ __forceinline__ int need(int n) const { return (int)min((int64_t)W, ((int64_t)n + grow + page - 1) >> shift); }
};

// Block 0 plans; the others, where the counts are not updated in place, copy them.
// A row's pages: entries below `full` (whole pages) are its parent's, shared. Of those from there on up to `need`, a parent's first
// child keeps the pages that nobody else holds; every other is a fresh page, noted as -2 - its rank among the row's.
// What bounds it: four loads one after the other (parent, length, entry, count) and the search for free pages: 6.3 to 6.8 us for 4 rows,
// 7.8 to 8.7 for 256, by card.
__global__ void __launch_bounds__(kPlanThreads) fork_plan_kernel(ForkArgs a) {
  extern __shared__ int lds[];
  __shared__ int64_t sh[kPlanThreads / 64];
  const int tid = threadIdx.x;
  if (blockIdx.x > 0) {
    for (int i = (blockIdx.x - 1) * kPlanThreads + tid; i < a.pages; i += (gridDim.x - 1) * kPlanThreads) a.refs_out[i] = a.refs[i];
    return;
  }
  const WorkLayout w(a.S, a.N, a.pages);
  int* const count = lds;            // [S] children
  int* const first = lds + a.S;      // [S] the first of them
  int* const fresh = first + a.S;    // [N] fresh pages
  int* const source = fresh + a.N;   // [N] page to be copied, or -1
  int* const near = source + a.N;    // [kListed] the first free pages
  const bool wide = ((uintptr_t)a.refs & 15) == 0;
  int r[kPerThread];  // (requested ahead of all that comes before their use)
  load_counts(a.refs, a.pages, tid * kPerThread, wide, r);
  for (int r = tid; r < a.S; r += kPlanThreads) {
    count[r] = 0;
    first[r] = INT_MAX;
  }
  __syncthreads();
  for (int i = tid; i < a.N; i += kPlanThreads) {
    const int p = a.parent_of(i);
    if (p >= 0) {
      atomicAdd(&count[p], 1);
      atomicMin(&first[p], i);
    }
  }
  __syncthreads();
  for (int r = tid; r < a.S; r += kPlanThreads) {
    ((int*)(a.work + w.count))[r] = count[r];
    ((int*)(a.work + w.first))[r] = first[r];
  }
  // the rows, `per` lanes each
  int per = 64;
  while (per > 1 && per * a.N > kPlanThreads) per >>= 1;
  const int sub = tid & (per - 1), lane = tid & 63;
  const uint64_t below = ((1ull << lane) - 1) & ~((1ull << (lane - sub)) - 1);  // lanes of the row before this one
  for (int i0 = 0; i0 < a.N; i0 += kPlanThreads / per) {
    const int i = i0 + tid / per;
    const int p = i < a.N ? a.parent_of(i) : -1;
    const int n = p >= 0 ? a.len(p) : 0, full = n >> a.shift, need = p >= 0 ? a.need(n) : 0;
    const bool heir = p >= 0 && first[p] == i;
    const int rows = n & (a.page - 1);
    int rank = 0;
    if (sub == 0 && i < a.N) source[i] = -1;
    for (int j0 = full; __any(j0 < need); j0 += per) {
      const int j = j0 + sub;
      bool take = j < need;
      int keep = -1;
      if (take && (heir || (j == full && rows > 0))) {
        const int e = a.table[(int64_t)p * a.ldt + j];
        if (a.has(e)) {
          if (heir && a.refs[e] == 1) keep = e;
          else if (j == full && rows > 0) source[i] = e;  // (the row's lane 0, as above)
        }
      }
      const uint64_t all = __ballot(take && keep < 0);
      if (take) a.table_out[(int64_t)i * a.ldo + j] = keep >= 0 ? keep : -2 - (rank + __popcll(all & below));
      const uint64_t row = per == 64 ? ~0ull : ((1ull << per) - 1) << (lane - sub);
      rank += __popcll(all & row);
    }
    if (sub == 0 && i < a.N) fresh[i] = rank;
  }
  __syncthreads();
  // ranks among all rows' fresh pages: as far as there are pages (a rank in a row is below 2^30 too)
  int64_t T = 0;
  for (int i0 = 0; i0 < a.N; i0 += kPlanThreads) {
    const int i = i0 + tid;
    const int64_t v = i < a.N ? fresh[i] : 0;
    int64_t total;
    const int64_t at = T + block_scan(v, sh, total);
    if (i < a.N) ((int*)(a.work + w.base))[i] = (int)min(at, (int64_t)kMaxPages);
    T += total;
  }
  // the first T free pages
  int* const list = (int*)(a.work + w.list);
  int found = 0;
  for (int p0 = 0; p0 < a.pages && found < T; p0 += kPlanThreads * kPerThread) {
    const int mine = p0 + tid * kPerThread;
    int free = 0;
    uint32_t which = 0;
#pragma unroll
    for (int k = 0; k < kPerThread; k++)
      if (r[k] == 0) which |= 1u << k;
    free = __popc(which);
    if (p0 + kPlanThreads * kPerThread < a.pages) load_counts(a.refs, a.pages, mine + kPlanThreads * kPerThread, wide, r);
    int total;
    int at = found + block_scan(free, sh, total);
    while (which) {
      const int k = __ffs(which) - 1;
      which &= which - 1;
      if (at < T) {
        list[at] = mine + k;
        if (at < kListed) near[at] = mine + k;
      }
      at++;
    }
    found += total;
  }
  found = (int)min((int64_t)found, T);
  __syncthreads();  // the list is written (a block's own stores, read past the L1 below)
  // part-filled pages to be copied
  Move* const moves = (Move*)(a.work + w.moves);
  int M = 0;
  for (int i0 = 0; i0 < a.N; i0 += kPlanThreads) {
    const int i = i0 + tid;
    Move m{-1, -1, 0};
    if (i < a.N && source[i] >= 0) {  // the row's first fresh page
      const int at = ((int*)(a.work + w.base))[i];
      if (at < found) {
        m.src = source[i];
        m.dst = at < kListed ? near[at] : __hip_atomic_load(list + at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        m.rows = a.len(a.parent_of(i)) & (a.page - 1);
      }
    }
    int total;
    const int at = M + block_scan((int)(m.src >= 0), sh, total);
    if (m.src >= 0) moves[at] = m;
    M += total;
  }
  if (tid == 0) {
    *(PlanHead*)a.work = PlanHead{found, M, 0, 0};
    if (a.missing) *a.missing = (int)min(T - found, (int64_t)INT_MAX);
  }
}

// By a wave: units [lo, hi) of those that a move copies of one tensor, of each run of `run` units the first `take`.
template <typename T>
__device__ __forceinline__ void copy_units(char* dst, const char* src, uint32_t lo, uint32_t hi, uint32_t run, uint32_t take) {
  constexpr int U = 4;
  const uint32_t lane = threadIdx.x & 63, r0 = lo / take, in0 = lo - r0 * take;
  const T* const s = (const T*)src + (size_t)r0 * run;
  T* const d = (T*)dst + (size_t)r0 * run;
  const float inv = 1.0f / (float)take;
  auto place = [&](uint32_t i) {  // unit in0 + i of the runs from r0 on; i < kPart
    const uint32_t at = in0 + i;
    uint32_t q = in0 + kPart < 1u << 22 ? (uint32_t)((float)at * inv) : at / take;  // off by one at most
    if (q * take > at) q--;
    if (at - q * take >= take) q++;
    return q * run + (at - q * take);
  };
  const uint32_t n = hi - lo;
  for (uint32_t i = lane; i < n; i += U * 64) {
    T v[U];
    uint32_t at[U];
#pragma unroll
    for (int u = 0; u < U; u++)
      if (i + u * 64 < n) v[u] = s[at[u] = place(i + u * 64)];
#pragma unroll
    for (int u = 0; u < U; u++)
      if (i + u * 64 < n) d[at[u]] = v[u];
  }
}

// By a wave: part `part` of tensor d's share of a move.
__device__ __forceinline__ void copy_part(const CacheDesc& d, const Move& m, int page, int part) {
  const uint32_t unit = d.runs_unit & 31, runs = d.runs_unit >> 5;
  const bool whole = runs == 0 || m.rows == page;
  // a run of `page` positions holds bytes / runs; of it the first m.rows positions' are copied
  const uint32_t run = whole ? d.bytes : d.bytes / runs, take = whole ? d.bytes : run / page * m.rows;
  const uint32_t total = whole ? d.bytes : take * runs, lo = (uint32_t)part * kPart;
  if (lo >= total) return;
  const uint32_t hi = min(total, lo + kPart);
  const char* const src = d.p + (int64_t)m.src * d.stride;
  char* const dst = d.p + (int64_t)m.dst * d.stride;
  if (unit == 16) copy_units<u32x4>(dst, src, lo / 16, hi / 16, run / 16, take / 16);
  else if (unit == 4) copy_units<uint32_t>(dst, src, lo / 4, hi / 4, run / 4, take / 4);
  else copy_units<uint8_t>(dst, src, lo, hi, run, take);
}

// By a lane: tensor d's share of a move, of kSmall bytes at most.
__device__ __forceinline__ void copy_small(const CacheDesc& d, const Move& m, int page) {
  const uint32_t runs = d.runs_unit >> 5, run = runs ? d.bytes / runs : d.bytes, take = runs ? run / page * m.rows : run;
  const char* const src = d.p + (int64_t)m.src * d.stride;
  char* const dst = d.p + (int64_t)m.dst * d.stride;
  if (take == run && (d.runs_unit & 31) >= 4) {
    for (uint32_t i = 0; i < d.bytes; i += 4) *(uint32_t*)(dst + i) = *(const uint32_t*)(src + i);
    return;
  }
  for (uint32_t r = 0; r < d.bytes; r += run)
    for (uint32_t i = 0; i < take; i++) dst[r + i] = src[r + i];
}

// All tensors' shares of n moves, by `waves` waves of which this is number `wave`. The large ones' parts are a wave's: 4 KB each in
// flight on every wave of the GPU. Some 1480 moves of 28 layers' pages of 2 x 4 KB 146 us, 4.7 TB/s read and written (blocks that
// copy 16 KB at a time 353).
__device__ __forceinline__ void copy_moves(const CacheSet& c, const Move* moves, int n, int page, int wave, int waves) {
  const int each = c.large * c.parts;
  const int64_t items = (int64_t)n * each;
  auto split = [&](int64_t i, int& m) {
    m = items <= INT_MAX ? (int)i / each : (int)(i / each);
    return (int)(i - (int64_t)m * each);
  };
  if (wave < items) {
    int m, rest = split(wave, m);
    Move move = moves[m];
    for (int64_t i = wave;;) {
      const Move now = move;
      const int t = rest / c.parts, part = rest - t * c.parts;
      i += waves;
      const bool more = i < items;
      if (more) {
        rest = split(i, m);
        move = moves[m];
      }
      copy_part(c.d[t], now, page, part);
      if (!more) break;
    }
  }
  const int small = c.n - c.large;
  for (int64_t i = (int64_t)wave * 64 + (threadIdx.x & 63); i < (int64_t)n * small; i += (int64_t)waves * 64) {
    const int m = (int)(i / small);
    copy_small(c.d[c.large + (int)(i - (int64_t)m * small)], moves[m], page);
  }
}

__device__ __forceinline__ int wave_of(int block) { return 4 * block + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// Blocks 0 .. N - 1 write the new rows, the next S account for what the old ones held, the others copy.
__global__ void __launch_bounds__(256, 8) fork_apply_kernel(ForkArgs a, CacheSet c, bool rows) {
  const WorkLayout w(a.S, a.N, a.pages);
  const PlanHead* head = (const PlanHead*)a.work;
  const int tid = threadIdx.x, lead = rows ? a.N + a.S : 0;
  int x = blockIdx.x;
  if (x >= lead) {
    copy_moves(c, (const Move*)(a.work + w.moves), head->moves, a.page, wave_of(x - lead), 4 * (gridDim.x - lead));
    return;
  }
  if (x < a.N) {
    const int p = a.parent_of(x), n = p >= 0 ? a.len(p) : 0, full = n >> a.shift, need = p >= 0 ? a.need(n) : 0;
    const int at = ((const int*)(a.work + w.base))[x], found = head->free;
    const int* list = (const int*)(a.work + w.list);
    if (tid == 0) a.lens_out[x] = n;
    for (int j = tid; j < a.W; j += 256) {
      int* const out = a.table_out + (int64_t)x * a.ldo + j;
      int e = -1;
      if (j < min(full, need)) {
        e = a.table[(int64_t)p * a.ldt + j];
        if (!a.has(e)) e = -1;
      } else if (j < need) {
        e = *out;
        if (e < 0) {
          const int k = at - 2 - e;
          e = k < found ? list[k] : -1;
          if (e >= 0) a.refs_out[e] = 1;
        }
      }
      __hip_atomic_store(out, e, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    return;
  }
  x -= a.N;
  const int children = ((const int*)(a.work + w.count))[x], heir = ((const int*)(a.work + w.first))[x];
  const int n = a.len(x), full = n >> a.shift, need = children ? a.need(n) : 0;
  for (int j = tid; j < a.W; j += 256) {
    const int e = a.table[(int64_t)x * a.ldt + j];
    if (!a.has(e)) continue;
    int change = -1;
    if (j < min(full, need)) change = children - 1;
    // (what the heir keeps stands in its new row since the plan; a fresh page is never one that was held)
    else if (j < need &&
             __hip_atomic_load(a.table_out + (int64_t)heir * a.ldo + j, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == e) change = 0;
    if (change) atomicAdd(a.refs_out + e, change);
  }
}

struct CompactArgs {
  const int *table, *refs;
  int *table_out, *refs_out, *moved, *used;
  char* work;
  int ldt, ldo, W, S, pages, page, shift;
};

// The used pages at or behind the number U of used pages go, in order, to the free ones before it, in order. 500 pages 4.9 us,
// 6000 9.6.
__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(CompactArgs a) {
  __shared__ int64_t sh[kPlanThreads / 64];
  const int tid = threadIdx.x;
  const WorkLayout w(a.S, 0, a.pages);
  Move* const moves = (Move*)(a.work + w.moves);
  const bool wide = ((uintptr_t)a.refs & 15) == 0;
  constexpr int kStep = kPlanThreads * kPerThread;
  int r[kPerThread];
  int used = 0;
  for (int p0 = tid * kPerThread; p0 < a.pages; p0 += kStep) {
    load_counts(a.refs, a.pages, p0, wide, r);
#pragma unroll
    for (int k = 0; k < kPerThread; k++) used += p0 + k < a.pages && r[k] > 0;
  }
  int U;
  block_scan(used, sh, U);
  const bool once = a.pages <= kStep;  // the counts are still there
  int out = 0, in = 0;  // pages to be moved, and places for them
  for (int p0 = 0; p0 < a.pages; p0 += kStep) {
    const int mine = p0 + tid * kPerThread;
    uint32_t moving = 0, hole = 0;
    if (mine < a.pages) {
      if (!once) load_counts(a.refs, a.pages, mine, wide, r);
#pragma unroll
      for (int k = 0; k < kPerThread; k++) {
        const int p = mine + k;
        if (p >= a.pages) continue;
        const bool u = r[k] > 0;
        if (u && p >= U) moving |= 1u << k;
        if (!u && p < U) hole |= 1u << k;
        r[k] = u ? p : -1;  // (of a page that moves: written again below)
      }
      if (((uintptr_t)a.moved & 15) == 0 && mine + kPerThread <= a.pages) {
#pragma unroll
        for (int k = 0; k < kPerThread; k += 4)
          *reinterpret_cast<u32x4*>(a.moved + mine + k) = u32x4{(uint32_t)r[k], (uint32_t)r[k + 1], (uint32_t)r[k + 2], (uint32_t)r[k + 3]};
      } else {
#pragma unroll
        for (int k = 0; k < kPerThread; k++)
          if (mine + k < a.pages) a.moved[mine + k] = r[k];
      }
    }
    int both;  // (at most 2^14 of either in a step)
    const int at = block_scan((int)(__popc(moving) << 16 | __popc(hole)), sh, both), n_out = both >> 16, n_in = both & 0xffff;
    int at_out = out + (at >> 16), at_in = in + (at & 0xffff);
    for (; moving; moving &= moving - 1)
      __hip_atomic_store(&moves[at_out++].src, mine + __ffs(moving) - 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    for (; hole; hole &= hole - 1)
      __hip_atomic_store(&moves[at_in++].dst, mine + __ffs(hole) - 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    out += n_out;
    in += n_in;
  }
  __syncthreads();
  for (int k = tid; k < out; k += kPlanThreads) {
    const int src = __hip_atomic_load(&moves[k].src, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    a.moved[src] = __hip_atomic_load(&moves[k].dst, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    moves[k].rows = a.page;
  }
  if (tid == 0) {
    *(PlanHead*)a.work = PlanHead{0, out, U, 0};
    if (a.used) *a.used = U;
  }
}

// `lead` blocks rename the table's entries and move the counts, the others copy.
__global__ void __launch_bounds__(256, 8) compact_apply_kernel(CompactArgs a, CacheSet c, int lead) {
  const WorkLayout w(a.S, 0, a.pages);
  const PlanHead* head = (const PlanHead*)a.work;
  if ((int)blockIdx.x >= lead) {
    copy_moves(c, (const Move*)(a.work + w.moves), head->moves, a.page, wave_of(blockIdx.x - lead), 4 * (gridDim.x - lead));
    return;
  }
  const int64_t entries = (int64_t)a.S * a.W;
  for (int64_t i = blockIdx.x * 256 + threadIdx.x; i < entries + a.pages; i += lead * 256) {
    if (i < entries) {
      const int s = (int)(i / a.W), j = (int)(i - (int64_t)s * a.W), e = a.table[(int64_t)s * a.ldt + j];
      a.table_out[(int64_t)s * a.ldo + j] = (unsigned)e < (unsigned)a.pages ? a.moved[e] : -1;
    } else {
      // in place too: a count's own thread takes it away, and places get theirs from one thread
      const int p = (int)(i - entries), m = a.moved[p], n = a.refs[p];
      if (m >= 0) a.refs_out[m] = n;
      if (p >= head->used) a.refs_out[p] = 0;
    }
  }
}

// Tensors t0 .. of the set as a kernel argument; -1 with the reason printed.
int cache_set(const char* who, void* const* caches, const long long* strides, const long long* bytes, const int* runs, int n, int page,
              int pages, int t0, CacheSet& c) {
  c.n = min(n - t0, kSetMax);
  c.large = 0;
  c.parts = 1;
  for (int pass = 0, at = 0; pass < 2; pass++)
    for (int k = t0; k < t0 + c.n; k++) {
      const long long b = bytes[k], st = strides[k];
      const int r = runs[k];
      const uintptr_t p = (uintptr_t)caches[k];
      if (!p || b < 1 || b > INT32_MAX || (pages > 1 && st < b) || r < 0 || r >= 1 << 26 || (r && b % ((long long)r * page)))
        HI_FAIL("%s: cache %d: %lld bytes a page, %lld apart, %d runs of %d positions", who, k, b, st, r, page);
      if ((b <= kSmall) != (pass == 1)) continue;
      const long long each = r ? b / ((long long)r * page) : b;  // of a position in one run
      const uint64_t all = p | (uint64_t)(pages > 1 ? st : 0) | (uint64_t)each;
      c.d[at++] = CacheDesc{(char*)p, (int64_t)st, (uint32_t)b, (uint32_t)r << 5 | (all % 16 == 0 ? 16u : all % 4 == 0 ? 4u : 1u)};
      if (pass == 0) c.parts = max(c.parts, (int)((b + kPart - 1) / kPart));
      if (pass == 0) c.large = at;
    }
  return 0;
}

// Checks what both calls have in common; the position shift of a page.
int pool_check(const char* who, void* const* caches, const long long* strides, const long long* bytes, const int* runs, int n, int page,
               const int* table, int ldt, int W, int S, const int* refs, int pages, const int* table_out, int ldo, const int* refs_out,
               const void* work, size_t work_bytes, int N, int& shift) {
  if (page < 1 || page > 1 << 20 || (page & (page - 1))) HI_FAIL("%s: page of %d positions (a power of two)", who, page);
  if (S < 0 || S > kMaxRows || N < 0 || N > kMaxRows || W < 1 || pages < 1 || pages > kMaxPages || n < 0 || ldt < W || ldo < W)
    HI_FAIL("%s: table [%d, %d] with row strides %d and %d, %d new rows (at most %d), %d pages, %d caches", who, S, W, ldt, ldo, N,
            kMaxRows, pages, n);
  if ((int64_t)W * page > (1 << 30)) HI_FAIL("%s: %d pages of %d positions (at most 2^30 positions a sequence)", who, W, page);
  if (!refs || !refs_out || !work || (S && !table) || (n && (!caches || !strides || !bytes || !runs)))
    HI_FAIL("%s: a null pointer", who);
  if (((uintptr_t)table | (uintptr_t)table_out | (uintptr_t)refs | (uintptr_t)refs_out) & 3 || ((uintptr_t)work & 15))
    HI_FAIL("%s: tables and counts must be 4-byte aligned, work 16-byte aligned", who);
  if (work_bytes < WorkLayout(S, N, pages).bytes)
    HI_FAIL("%s: work of %zu bytes (at least %zu)", who, work_bytes, WorkLayout(S, N, pages).bytes);
  if (!in_place_or_apart(refs, 4 * (int64_t)pages, 4 * (int64_t)pages, refs_out, 4 * (int64_t)pages, 4 * (int64_t)pages, 1))
    HI_FAIL("%s: the new counts must be the old ones' memory or apart from it", who);
  shift = 0;
  while ((1 << shift) < page) shift++;
  CacheSet c;
  for (int t0 = 0; t0 < n; t0 += kSetMax)
    if (cache_set(who, caches, strides, bytes, runs, n, page, pages, t0, c)) return -1;
  return 0;
}

// Blocks (of 4 waves) that copy: what the largest number of moves needs, at most 8 a CU.
int copy_blocks(int64_t moves, const CacheSet& c, int cus) {
  return (int)max((int64_t)1, min((moves * c.n * c.parts + 3) / 4, (int64_t)8 * cus));
}

}  // namespace

HI_EXPORT size_t hi_cache_work_bytes(int S, int N, int pages) {
  if (S < 0 || S > kMaxRows || N < 0 || N > kMaxRows || pages < 1 || pages > kMaxPages) return 0;
  return WorkLayout(S, N, pages).bytes;
}

HI_EXPORT int hi_cache_fork(void* const* caches, const long long* strides, const long long* bytes, const int* runs, int n, int page,
                            const int* table, int ldt, int W, int S, const int* lens, const int* parent, int N, const int* refs,
                            int pages, int grow, int* table_out, int ldo, int* lens_out, int* refs_out, int* missing, void* work,
                            size_t work_bytes, void* stream) {
  const char* who = "hi_cache_fork";
  int shift;
  if (pool_check(who, caches, strides, bytes, runs, n, page, table, ldt, W, S, refs, pages, table_out, ldo, refs_out, work,
                 work_bytes, N, shift)) return -1;
  if (grow < 0 || grow > 1 << 30) HI_FAIL("%s: room for %d positions", who, grow);
  if ((S && !lens) || (N && (!parent || !table_out || !lens_out))) HI_FAIL("%s: a null pointer", who);
  if (((uintptr_t)lens | (uintptr_t)parent | (uintptr_t)lens_out | (uintptr_t)missing) & 3)
    HI_FAIL("%s: lens, parent and missing must be 4-byte aligned", who);
  // parent is read in the launch that writes table_out and lens_out, and the rows' blocks run beside each other
  const CallRows rows[] = {{"table", table, 4 * (int64_t)ldt, 4 * (int64_t)W, S, false}, call_flat("lens", lens, 4 * (int64_t)S, false),
                           call_flat("parent", parent, 4 * (int64_t)N, false), call_flat("refs", refs, 4 * (int64_t)pages, false),
                           {"table_out", table_out, 4 * (int64_t)ldo, 4 * (int64_t)W, N, true},
                           call_flat("lens_out", lens_out, 4 * (int64_t)N, true), call_flat("refs_out", refs_out, 4 * (int64_t)pages, true, 3),
                           call_flat("missing", missing, 4, true), call_flat("work", work, (int64_t)WorkLayout(S, N, pages).bytes, true)};
  const char *a0, *a1;
  if (call_rows_meet(rows, a0, a1)) HI_FAIL("%s: %s and %s must be apart", who, a0, a1);
  const HiDevice* d = hi_device();
  if (!d) return -2;
  const hipStream_t s = (hipStream_t)stream;
  const ForkArgs a{table, lens, parent, refs, table_out, lens_out, refs_out, missing, (char*)work, ldt, ldo, W, S, N, pages, grow,
                   page, shift};
  const int copiers = refs == refs_out ? 0 : min(d->cus, (pages + kPlanThreads - 1) / kPlanThreads);
  const size_t lds = fork_lds(S, N);
  if (lds > 48 * 1024 && hi_blocks_per_cu(reinterpret_cast<const void*>(fork_plan_kernel), kPlanThreads, lds) < 1) return -2;
  hipLaunchKernelGGL(fork_plan_kernel, dim3(1 + copiers), dim3(kPlanThreads), lds, s, a);
  HI_TRY(hipGetLastError());
  CacheSet c;
  for (int t0 = 0; t0 == 0 || t0 < n; t0 += kSetMax) {
    cache_set(who, caches, strides, bytes, runs, n, page, pages, t0, c);
    const int blocks = (t0 == 0 ? N + S : 0) + (c.n ? copy_blocks(N, c, d->cus) : 0);
    if (blocks == 0) break;
    hipLaunchKernelGGL(fork_apply_kernel, dim3(blocks), dim3(256), 0, s, a, c, t0 == 0);
    HI_TRY(hipGetLastError());
  }
  return 0;
}

HI_EXPORT int hi_cache_compact(void* const* caches, const long long* strides, const long long* bytes, const int* runs, int n, int page,
                               const int* table, int ldt, int W, int S, const int* refs, int pages, int* table_out, int ldo,
                               int* refs_out, int* moved, int* used, void* work, size_t work_bytes, void* stream) {
  const char* who = "hi_cache_compact";
  int shift;
  if (pool_check(who, caches, strides, bytes, runs, n, page, table, ldt, W, S, refs, pages, table_out, ldo, refs_out, work,
                 work_bytes, 0, shift)) return -1;
  if (!moved || (S && !table_out) || ((uintptr_t)moved | (uintptr_t)used) & 3)
    HI_FAIL("%s: moved and used must be 4-byte aligned, moved and the new table not null", who);
  if (S && !in_place_or_apart(table, 4 * (int64_t)ldt, 4 * (int64_t)W, table_out, 4 * (int64_t)ldo, 4 * (int64_t)W, S))
    HI_FAIL("%s: the new table must be the old one (with its row stride) or apart from it", who);
  // moved is read by the blocks that write the new table and counts beside each other
  const int64_t span = 4 * (int64_t)pages;
  const CallRows rows[] = {{"table", table, 4 * (int64_t)ldt, 4 * (int64_t)W, S, false}, call_flat("refs", refs, span, false),
                           {"table_out", table_out, 4 * (int64_t)ldo, 4 * (int64_t)W, S, true, 0}, call_flat("refs_out", refs_out, span, true, 1),
                           call_flat("moved", moved, span, true), call_flat("used", used, 4, true),
                           call_flat("work", work, (int64_t)WorkLayout(S, 0, pages).bytes, true)};
  const char *a0, *a1;
  if (call_rows_meet(rows, a0, a1)) HI_FAIL("%s: %s and %s must be apart", who, a0, a1);
  const HiDevice* d = hi_device();
  if (!d) return -2;
  const hipStream_t s = (hipStream_t)stream;
  const CompactArgs a{table, refs, table_out, refs_out, moved, used, (char*)work, ldt, ldo, W, S, pages, page, shift};
  hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, a);
  HI_TRY(hipGetLastError());
  CacheSet c;
  for (int t0 = 0; t0 == 0 || t0 < n; t0 += kSetMax) {
    cache_set(who, caches, strides, bytes, runs, n, page, pages, t0, c);
    const int lead = t0 == 0 ? (int)min((int64_t)d->cus, ((int64_t)S * W + pages + 255) / 256) : 0;
    const int blocks = lead + (c.n ? copy_blocks(pages / 2, c, d->cus) : 0);
    if (blocks == 0) break;
    hipLaunchKernelGGL(compact_apply_kernel, dim3(blocks), dim3(256), 0, s, a, c, lead);
    HI_TRY(hipGetLastError());
  }
  return 0;
}
