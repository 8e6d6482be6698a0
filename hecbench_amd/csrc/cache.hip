// The paged key / value cache: tokens into pages, the page tables from one token to the next, live pages to the front.
#include <algorithm>
#include <climits>

#include "hq_internal.h"

namespace {

constexpr int kThreads = 256;

// ---- tokens into pages ------------------------------------------------------------------------------------------------
struct WriteArgs {
  const hq_u4v *k, *v;
  hq_u4v *kp, *vp;
  const int *table, *starts, *cu;
  int64_t ks, vs;  // 16-byte pieces from one token to the next
  int rows, tokens, width, pages, page_log, kv_heads, pieces;  // pieces of one head's row
};

// The first i with bounds[i + 1] > t, n if there is none: a wave halves the range sixty-four-fold a step.
__device__ __forceinline__ int find_row(const int* bounds, int n, int t) {
  const int lane = threadIdx.x & 63;
  int lo = 0;
  while (n > 0) {
    const int step = (n + 63) >> 6;
    const int at = lo + min((lane + 1) * step, n);
    const int below = __popcll(__ballot(bounds[at] <= t));
    if (below == 64) return lo + n;
    lo += below * step;
    n = min(step, n - below * step) - 1;
  }
  return lo;
}

// One wave a token, keys and values.  Bound by the copy; a short call by the launch and three loads one after the other (bounds, start,
// table), of which the token's own first pieces do not wait for any.
__global__ __launch_bounds__(kThreads) void write_kernel(WriteArgs a) {
  const int t = blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (t >= a.tokens) return;
  const int n = a.kv_heads * a.pieces;
  const hq_u4v* const k = a.k + t * a.ks;
  const hq_u4v* const v = a.v + t * a.vs;
  hq_u4v kx[2], vx[2];
  auto load = [&](int i0) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int i = min(i0 + 64 * j + lane, n - 1);
      kx[j] = k[i];
      vx[j] = v[i];
    }
  };
  load(0);
  const int row = find_row(a.cu, a.rows, t);
  if (row >= a.rows || t < a.cu[row]) return;
  const int64_t p = (int64_t)a.starts[row] + (t - a.cu[row]);
  if (p < 0 || p >= (int64_t)a.width << a.page_log) return;
  const int page = a.table[(int64_t)row * a.width + (p >> a.page_log)], at = (int)p & ((1 << a.page_log) - 1);
  if ((unsigned)page >= (unsigned)a.pages) return;
  for (int i0 = 0;;) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int i = i0 + 64 * j + lane, head = i / a.pieces, piece = i % a.pieces;
      if (i >= n) break;
      const int64_t to = ((((int64_t)page * a.kv_heads + head) << a.page_log) + at) * a.pieces + piece;
      hq_store_stream(a.kp + to, kx[j]);  // past the L2: 12,700 tokens of 8 heads of 128, fp16, 16.9 us (6.2 TB/s), plain 22.7
      hq_store_stream(a.vp + to, vx[j]);
    }
    if ((i0 += 128) >= n) return;
    load(i0);
  }
}

// ---- one step of the page tables ----------------------------------------------------------------------------------------
struct StepArgs {
  hq_u4v* pool;
  const int *table, *lengths, *refs, *parent, *add;
  int *table_out, *lengths_out, *refs_out, *starts_out, *missing;
  int *need, *source;    // of each row: pages that it asks for; the half-filled page that it copies, -1 if none
  int *copies, *ncopies; // {source, target} of the pages to be copied
  int* list;             // pages handed out
  int* change;           // of each page's count; zero between calls
  unsigned* arrived;
  int64_t page_pieces;   // 16-byte pieces of a page
  int planes, rows, width, pages, page;
};

__device__ __forceinline__ void put(int* p, int v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ int get(const int* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// Sum over the workgroup of the values of the threads before this one, and of all.
__device__ __forceinline__ int block_scan(int v, int* parts, int* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int sum = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int u = __shfl_up(sum, d);
    if (lane >= d) sum += u;
  }
  __syncthreads();
  if (lane == 63) parts[wave] = sum;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < (int)blockDim.x / 64; ++w) {
    before += w < wave ? parts[w] : 0;
    all += parts[w];
  }
  *total = all;
  return before + sum - v;
}

// Ranks among the marked ones of a stretch of 16 * 256 pages, page i * 256 + thread being marked[i] of its thread: a bit a page, whose
// sums meet once, so that a stretch costs one trip to memory and two barriers (page by page in steps of 256 threads: 16 of each, and
// 16 us for 4096 pages; the step of 48 rows over 768 pages 24.7 us, in stretches 10.6).
constexpr int kEach = 16, kStretch = kEach * kThreads;
template <int THREADS = kThreads, int EACH = kStretch / THREADS>
struct Ranks {
  unsigned long long bits[EACH];
  int before[EACH], all;
  // counts: 64 words of LDS; n: pages of the stretch, which ends there
  __device__ __forceinline__ Ranks(const bool (&marked)[EACH], int n, int* counts) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __syncthreads();
    if (wave == 0) counts[lane] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      bits[i] = 0;
      if (i * THREADS < n) {
        bits[i] = __ballot(marked[i]);
        if (lane == 0) counts[i * (THREADS / 64) + wave] = __popcll(bits[i]);
      }
    }
    __syncthreads();
    static_assert(EACH * THREADS / 64 == 64, "a lane each");
    const int mine = counts[lane];
    int sum = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int u = __shfl_up(sum, d);
      if (lane >= d) sum += u;
    }
    all = __builtin_amdgcn_readlane(sum, 63);
#pragma unroll
    for (int i = 0; i < EACH; ++i)
      if (i * THREADS < n) before[i] = __shfl(sum - mine, i * (THREADS / 64) + wave);
  }
  __device__ __forceinline__ int of(int i) const {
    return before[i] + __popcll(bits[i] & ((1ull << (threadIdx.x & 63)) - 1));
  }
};

constexpr int kListLds = 4096;  // pages handed out that are listed in LDS; the others are in memory
// One workgroup a row: what it inherits, and how the pages' counts change by it; the last one to arrive hands out pages.
__global__ __launch_bounds__(kThreads) void step_kernel(StepArgs a) {
  extern __shared__ int lds[];
  __shared__ int parts[kEach * kThreads / 64], flag;
  const int s = blockIdx.x, tid = threadIdx.x;
  const int cap = a.width * a.page;
  auto length_of = [&](int r) { return min(max(a.lengths[r], 0), cap); };
  auto start_of = [&](int r) {
    const int p = a.parent[r];
    return p >= 0 && p < a.rows ? length_of(p) : 0;
  };
  auto end_of = [&](int r, int start) { return (int)min((int64_t)start + max(a.add[r], 0), (int64_t)cap); };
  if (s < a.rows) {
    const int p = a.parent[s];
    const bool alive = p >= 0 && p < a.rows;
    if (tid == 0) flag = 0;
    __syncthreads();
    if (alive)
      for (int i = tid; i < s; i += kThreads)
        if (a.parent[i] == p) flag = 1;
    __syncthreads();
    const bool keeps = !flag;
    const int start = start_of(s), full = start / a.page, used = (start + a.page - 1) / a.page, end = end_of(s, start);
    const int last = (end + a.page - 1) / a.page, mine = (length_of(s) + a.page - 1) / a.page;
    const int tail = used > full ? a.table[(int64_t)p * a.width + full] : -1;
    const bool copies = alive && used > full && !keeps && (unsigned)tail < (unsigned)a.pages;
    const int from = copies ? full : used;  // the entries from here to `last` are new
    const bool same = p == s && keeps;
    for (int j = tid; j < a.width; j += kThreads) {
      if (!same && j < mine) {
        const int old = a.table[(int64_t)s * a.width + j];
        if ((unsigned)old < (unsigned)a.pages) atomicSub(a.change + old, 1);
      }
      int e = -1;
      if (j < from) {
        e = a.table[(int64_t)p * a.width + j];
        if ((unsigned)e >= (unsigned)a.pages) e = -1;
        else if (!same) atomicAdd(a.change + e, 1);
      }
      if (j < from || j >= max(last, used)) a.table_out[(int64_t)s * a.width + j] = e;
    }
    if (tid == 0) {
      put(a.need + s, max(last, used) - from);
      put(a.source + s, copies ? tail : -1);
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) flag = __hip_atomic_fetch_add(a.arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
  __syncthreads();
  if (!flag) return;

  // where each row's requests begin in the order of all
  int* const off = lds;
  int* const source = lds + a.rows;
  int* const list = source + a.rows;
  int total = 0;
  for (int r0 = 0; r0 < a.rows; r0 += kThreads) {
    const int r = r0 + tid;
    const int n = r < a.rows ? get(a.need + r) : 0, from = r < a.rows ? get(a.source + r) : 0;
    int all;
    const int before = block_scan(n, parts, &all);
    if (r < a.rows) {
      off[r] = total + before;
      source[r] = from;
    }
    total += all;
  }
  // free pages, lowest first, to the requests in their order
  int nfree = 0;
  for (int i0 = 0; i0 < a.pages; i0 += kStretch) {
    int count[kEach], change[kEach];
    bool free[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int p = min(i0 + i * kThreads + tid, a.pages - 1);
      count[i] = 0;
      change[i] = 1;
      if (i0 + i * kThreads < a.pages) {
        count[i] = a.refs[p];
        change[i] = get(a.change + p);
      }
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      count[i] += change[i];
      free[i] = i0 + i * kThreads + tid < a.pages && count[i] <= 0;
    }
    const Ranks<> ranks(free, a.pages - i0, parts);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int p = i0 + i * kThreads + tid, rank = nfree + ranks.of(i);
      if (p >= a.pages) continue;
      if (change[i]) put(a.change + p, 0);
      const bool taken = free[i] && rank < total;
      a.refs_out[p] = taken ? 1 : count[i];
      if (taken) {
        if (rank < kListLds) list[rank] = p;
        else put(a.list + rank, p);
      }
    }
    nfree += ranks.all;
  }
  if (tid == 0) {
    *a.missing = max(total - nfree, 0);
    put((int*)a.arrived, 0);
    flag = 0;
  }
  if (total > kListLds) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  auto page_of = [&](int rank) { return rank >= nfree ? -1 : rank < kListLds ? list[rank] : get(a.list + rank); };
  for (int r = tid; r < a.rows; r += kThreads) {
    const int start = start_of(r), first = off[r], n = (r + 1 < a.rows ? off[r + 1] : total) - first;
    const int from = source[r] >= 0 ? start / a.page : (start + a.page - 1) / a.page;
    int end = end_of(r, start);
    if (first + n > nfree) end = min(end, (from + max(nfree - first, 0)) * a.page);
    a.lengths_out[r] = end;
    a.starts_out[r] = min(start, end);
    if (source[r] >= 0 && first < nfree) {
      const int at = atomicAdd(&flag, 1);
      a.copies[2 * at] = source[r];
      a.copies[2 * at + 1] = page_of(first);
    }
  }
  for (int x = tid; x < total; x += kThreads) {
    int lo = 0, hi = a.rows - 1;  // the last row whose requests begin at x or before
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (off[mid] <= x) lo = mid;
      else hi = mid - 1;
    }
    const int start = start_of(lo), from = source[lo] >= 0 ? start / a.page : (start + a.page - 1) / a.page;
    a.table_out[(int64_t)lo * a.width + from + x - off[lo]] = page_of(x);
  }
  __syncthreads();
  if (tid == 0) *a.ncopies = flag;
}

// Pages {source, target} of every plane, eight 16-byte pieces of a thread on their way at a time, stored past the L2.
// Every 256 threads of a workgroup take a page of their own.
template <int THREADS = kThreads>
__device__ __forceinline__ void copy_pages(hq_u4v* pool, const int* pairs, int n, int planes, int pages, int64_t pieces) {
  constexpr int GROUPS = THREADS / kThreads;
  const int group = threadIdx.x / kThreads, tid = threadIdx.x % kThreads;
  for (int64_t x = blockIdx.x * GROUPS + group; x < (int64_t)n * planes; x += gridDim.x * GROUPS) {
    const int c = x % n;
    const int64_t plane = x / n;
    const hq_u4v* from = pool + (plane * pages + pairs[2 * c]) * pieces;
    hq_u4v* to = pool + (plane * pages + pairs[2 * c + 1]) * pieces;
    for (int64_t i0 = tid; i0 < pieces; i0 += 8 * kThreads) {
      hq_u4v v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = from[min(i0 + i * kThreads, pieces - 1)];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i0 + i * kThreads < pieces) hq_store_stream(to + i0 + i * kThreads, v[i]);
    }
  }
}
__global__ __launch_bounds__(kThreads) void step_copy_kernel(StepArgs a) {
  copy_pages(a.pool, a.copies, *a.ncopies, a.planes, a.pages, a.page_pieces);
}

// Small tables in one launch: every workgroup works out the whole step in LDS, from the tables alone, then writes its part of the rows and
// of the copies; nobody waits for anybody.  A thread has a row, and up to 16 entries of the table, whose loads are under way together
// (48 rows of 128 pages: 10.6 us in two launches, 7.6 in one).
constexpr int kSmallRows = 1024, kSmallEntries = 16 * kSmallRows;
__global__ __launch_bounds__(kSmallRows) void step_small_kernel(StepArgs a) {
  constexpr int THREADS = kSmallRows, EACH = kStretch / THREADS, BATCH = 8;
  __shared__ int parts[64];
  __shared__ int change[kStretch], length[kSmallRows], first[kSmallRows], off[kSmallRows + 1], pairs[2 * kSmallRows];
  __shared__ unsigned short list[kStretch];
  __shared__ unsigned short from[kSmallRows];
  __shared__ short parent[kSmallRows];
  const int tid = threadIdx.x, cap = a.width * a.page, r = tid;
  const bool row = r < a.rows;
  int p = -1, add = 0, count[EACH];
  if (row) {
    p = a.parent[r];
    add = max(a.add[r], 0);
    length[r] = min(max(a.lengths[r], 0), cap);
    if (p < 0 || p >= a.rows) p = -1;
    parent[r] = (short)p;
    first[r] = INT_MAX;
  }
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    count[i] = i * THREADS + tid < a.pages ? a.refs[i * THREADS + tid] : 1;
    change[i * THREADS + tid] = 0;
  }
  __syncthreads();
  if (p >= 0) atomicMin(first + p, r);
  __syncthreads();
  // what the row inherits, from which entry on it asks for pages, and where its requests begin in the order of all
  int start = 0, end = 0, source = -1, need = 0, total;
  if (row) {
    start = p < 0 ? 0 : length[p];
    end = (int)min((int64_t)start + add, (int64_t)cap);
    const int full = start / a.page, used = (start + a.page - 1) / a.page, last = (end + a.page - 1) / a.page;
    if (used > full && first[p] != r) {
      const int tail = a.table[(int64_t)p * a.width + full];
      if ((unsigned)tail < (unsigned)a.pages) source = tail;
    }
    from[r] = (unsigned short)(source >= 0 ? full : used);
    need = max(last, used) - from[r];
  }
  const int before = block_scan(need, parts, &total);
  if (row) off[r] = before;
  if (tid == 0) off[a.rows] = total;
  __syncthreads();
  const int entries = a.rows * a.width;
  const float by_width = 1.f / a.width;
  auto row_of = [=](int x) { return (int)((x + 0.5f) * by_width); };  // exact: entries * 2^-22 is far below a half
  for (int x0 = tid; x0 < entries; x0 += BATCH * THREADS) {
    int old[BATCH], now[BATCH];
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int x = x0 + i * THREADS;
      old[i] = now[i] = -1;
      if (x0 - tid + i * THREADS >= entries || x >= entries) continue;
      const int s = row_of(x), j = x - s * a.width;
      if (parent[s] == s && first[s] == s) continue;  // it goes on as it is
      if (j < (length[s] + a.page - 1) / a.page) old[i] = a.table[x];
      if (j < from[s]) now[i] = a.table[(int64_t)parent[s] * a.width + j];
    }
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      if ((unsigned)old[i] < (unsigned)a.pages) atomicSub(change + old[i], 1);
      if ((unsigned)now[i] < (unsigned)a.pages) atomicAdd(change + now[i], 1);
    }
  }
  __syncthreads();
  bool free[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    count[i] += change[i * THREADS + tid];
    free[i] = i * THREADS + tid < a.pages && count[i] <= 0;
  }
  const Ranks<THREADS> ranks(free, a.pages, parts);
  const int nfree = ranks.all;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int page = i * THREADS + tid;
    if (page >= a.pages) continue;
    const bool taken = free[i] && ranks.of(i) < total;
    if (taken) list[ranks.of(i)] = (unsigned short)page;
    if (blockIdx.x == 0) a.refs_out[page] = taken ? 1 : count[i];
  }
  __syncthreads();
  // the copies, and the rows' lengths
  const bool copy = source >= 0 && before < nfree;
  int copies;
  const int at = block_scan(copy, parts, &copies);
  if (copy) {
    pairs[2 * at] = source;
    pairs[2 * at + 1] = list[before];
  }
  if (blockIdx.x == 0) {
    if (tid == 0) *a.missing = max(total - nfree, 0);
    if (row) {
      if (before + need > nfree) end = min(end, (from[r] + max(nfree - before, 0)) * a.page);
      a.lengths_out[r] = end;
      a.starts_out[r] = min(start, end);
    }
  }
  for (int x = blockIdx.x * THREADS + tid; x < entries; x += gridDim.x * THREADS) {
    const int s = row_of(x), j = x - s * a.width, asked = j - from[s];
    int e = -1;
    if (asked < 0) {
      e = a.table[(int64_t)parent[s] * a.width + j];
      if ((unsigned)e >= (unsigned)a.pages) e = -1;
    } else if (off[s] + asked < min(off[s + 1], nfree)) {
      e = list[off[s] + asked];
    }
    a.table_out[x] = e;
  }
  __syncthreads();
  copy_pages<THREADS>(a.pool, pairs, copies, a.planes, a.pages, a.page_pieces);
}

// ---- live pages to the front ----------------------------------------------------------------------------------------------
struct CompactArgs {
  hq_u4v* pool;
  const int *table, *refs;
  int *table_out, *refs_out, *live;
  int *pairs;            // {source, target}
  int *to;               // of every page that moves: where
  int* nmoves;
  int64_t page_pieces;
  int planes, rows, width, pages;
};

// The i-th page in use behind the first `live` goes to the i-th hole among them.
__global__ __launch_bounds__(kThreads) void compact_plan_kernel(CompactArgs a) {
  __shared__ int parts[kEach * kThreads / 64];
  int n[kEach];
  auto load = [&](int i0) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) n[i] = a.refs[min(i0 + i * kThreads + (int)threadIdx.x, a.pages - 1)];
  };
  int live = 0;
  for (int i0 = 0; i0 < a.pages; i0 += kStretch) {
    load(i0);
    int mine = 0, all;
#pragma unroll
    for (int i = 0; i < kEach; ++i) mine += i0 + i * kThreads + (int)threadIdx.x < a.pages && n[i] > 0;
    block_scan(mine, parts, &all);
    live += all;
  }
  int holes = 0, movers = 0;
  for (int i0 = 0; i0 < a.pages; i0 += kStretch) {
    if (a.pages > kStretch) load(i0);  // else they are still there
    bool hole[kEach], mover[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int p = i0 + i * kThreads + threadIdx.x;
      hole[i] = p < live && n[i] <= 0;
      mover[i] = p < a.pages && p >= live && n[i] > 0;
    }
    const Ranks<> to(hole, a.pages - i0, parts), from(mover, a.pages - i0, parts);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int p = i0 + i * kThreads + threadIdx.x;
      if (hole[i]) put(a.pairs + 2 * (holes + to.of(i)) + 1, p);
      if (mover[i]) put(a.pairs + 2 * (movers + from.of(i)), p);
      if (p < a.pages && !hole[i]) a.refs_out[p] = mover[i] ? 0 : n[i];
    }
    holes += to.all;
    movers += from.all;
  }
  if (threadIdx.x == 0) {
    *a.live = live;
    *a.nmoves = movers;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  for (int r = threadIdx.x; r < movers; r += kThreads) {
    const int from = get(a.pairs + 2 * r), to = get(a.pairs + 2 * r + 1);
    a.refs_out[to] = a.refs[from];
    a.to[from] = to;
  }
}
__global__ __launch_bounds__(kThreads) void compact_move_kernel(CompactArgs a) {
  const int live = *a.live;
  const int64_t n = (int64_t)a.rows * a.width;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kThreads) {
    const int e = a.table[i];
    a.table_out[i] = e >= live && e < a.pages && a.refs[e] > 0 ? a.to[e] : e;
  }
  // One piece a thread, in the order of the grid: what is read and written at a time lies close together (954 MB of 32 KB pages: 149 us
  // with a unit a workgroup, 160 with three or four, 184 with eight pieces of a thread on their way in 1536 workgroups).
  const int moves = *a.nmoves, parts = (int)((a.page_pieces + kThreads - 1) / kThreads);
  const int64_t units = (int64_t)moves * a.planes * parts;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int64_t y = u / parts, plane = y / moves, i = (u - y * parts) * kThreads + threadIdx.x;
    const int m = (int)(y - plane * moves);
    if (i < a.page_pieces) {
      hq_u4v* const pool = a.pool + plane * a.pages * a.page_pieces + i;
      hq_store_stream(pool + a.pairs[2 * m + 1] * a.page_pieces, pool[a.pairs[2 * m] * a.page_pieces]);
    }
  }
}

// The same in one launch where the counts are one stretch: every workgroup makes the plan for itself, in LDS (300 of 512 pages: 9.6 us in
// two launches, 6.4 in one).
__global__ __launch_bounds__(kThreads) void compact_small_kernel(CompactArgs a) {
  __shared__ int parts[kEach * kThreads / 64];
  __shared__ int pairs[kStretch];       // half of the pages at most move
  __shared__ unsigned short to[kStretch];
  int n[kEach], mine = 0, live;
#pragma unroll
  for (int i = 0; i < kEach; ++i) if (i * kThreads < a.pages) n[i] = a.refs[min(i * kThreads + (int)threadIdx.x, a.pages - 1)];
#pragma unroll
  for (int i = 0; i < kEach; ++i) if (i * kThreads < a.pages) mine += i * kThreads + (int)threadIdx.x < a.pages && n[i] > 0;
  block_scan(mine, parts, &live);
  bool hole[kEach], mover[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int p = i * kThreads + threadIdx.x;
    hole[i] = mover[i] = false;
    if (i * kThreads < a.pages) {
      hole[i] = p < live && n[i] <= 0;
      mover[i] = p < a.pages && p >= live && n[i] > 0;
    }
  }
  const Ranks<> holes(hole, a.pages, parts), movers(mover, a.pages, parts);
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int p = i * kThreads + threadIdx.x;
    if (i * kThreads < a.pages) {
      if (hole[i]) pairs[2 * holes.of(i) + 1] = p;
      if (mover[i]) pairs[2 * movers.of(i)] = p;
    }
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    if (threadIdx.x == 0) *a.live = live;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
    const int p = i * kThreads + threadIdx.x;
      if (i * kThreads < a.pages && p < a.pages) a.refs_out[p] = hole[i] ? a.refs[pairs[2 * holes.of(i)]] : mover[i] ? 0 : n[i];
    }
  }
  const int64_t entries = (int64_t)a.rows * a.width;
  if ((int64_t)blockIdx.x * kThreads < entries) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
    const int p = i * kThreads + threadIdx.x;
      if (i * kThreads < a.pages) to[p] = mover[i] ? pairs[2 * movers.of(i) + 1] : p;
    }
    __syncthreads();
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < entries; i += (int64_t)gridDim.x * kThreads) {
      const int e = a.table[i];
      a.table_out[i] = (unsigned)e < (unsigned)a.pages ? to[e] : e;
    }
  }
  copy_pages(a.pool, pairs, movers.all, a.planes, a.pages, a.page_pieces);
}

bool meet(const void* a, int64_t na, const void* b, int64_t nb) {
  const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  return na > 0 && nb > 0 && x < y + nb && y < x + na;
}
bool pool_bad(const void* pool, int planes, int64_t page_bytes) { return planes > 0 && page_bytes > 0 && !pool; }
}  // namespace

extern "C" int hq_cache_write(const void* k, const void* v, void* k_pages, void* v_pages, int dtype, const int32_t* table,
                              const int32_t* starts, const int32_t* cu, int rows, int64_t tokens, int table_width, int num_pages,
                              int page_size, int kv_heads, int head_dim, int64_t k_stride, int64_t v_stride, void* stream) {
  if (rows < 0 || tokens < 0 || table_width < 0 || num_pages < 0 || kv_heads < 1 || head_dim < 8 || head_dim % 8) return HQ_ERR_BAD_SHAPE;
  if (page_size < 1 || page_size > 1024 || (page_size & (page_size - 1))) return HQ_ERR_BAD_SHAPE;
  if (dtype != HQ_DTYPE_F16 && dtype != HQ_DTYPE_BF16) return HQ_ERR_BAD_ENUM;
  if (rows == 0 || tokens == 0 || table_width == 0 || num_pages == 0) return HQ_OK;
  if (!k || !v || !k_pages || !v_pages || !table || !starts || !cu) return HQ_ERR_NULL_POINTER;
  if (k_stride < (int64_t)kv_heads * head_dim || v_stride < (int64_t)kv_heads * head_dim) return HQ_ERR_BAD_SHAPE;
  if ((((uintptr_t)k | (uintptr_t)v | (uintptr_t)k_pages | (uintptr_t)v_pages) & 15) || k_stride % 8 || v_stride % 8 ||
      (((uintptr_t)table | (uintptr_t)starts | (uintptr_t)cu) & 3))
    return HQ_ERR_MISALIGNED;
  if (tokens > INT_MAX - 64 || (int64_t)kv_heads * head_dim > INT_MAX) return HQ_ERR_TOO_LARGE;
  const HqDevice* dev = nullptr;
  const int rc = hq_current_device(&dev);
  if (rc != HQ_OK) return rc;
  const WriteArgs a{(const hq_u4v*)k, (const hq_u4v*)v, (hq_u4v*)k_pages, (hq_u4v*)v_pages, table, starts, cu, k_stride / 8, v_stride / 8, rows,
                    (int)tokens, table_width, num_pages, __builtin_ctz(page_size), kv_heads, head_dim / 8};
  return hq_launch_as_is(write_kernel, dim3((unsigned)((tokens + 3) / 4)), dim3(kThreads), 0, (hipStream_t)stream, a);
}

extern "C" int hq_cache_step(void* pool, int planes, int64_t page_bytes, const int32_t* table, const int32_t* lengths, const int32_t* refs,
                             const int32_t* parent, const int32_t* add, int32_t* table_out, int32_t* lengths_out, int32_t* refs_out,
                             int32_t* starts_out, int32_t* missing, int rows, int table_width, int num_pages, int page_size, void* stream) {
  if (planes < 0 || page_bytes < 0 || page_bytes % 16 || rows < 0 || table_width < 0 || num_pages < 0 || page_size < 1) return HQ_ERR_BAD_SHAPE;
  if (!missing || (num_pages && (!refs || !refs_out)) || (rows && (!lengths || !parent || !add || !lengths_out || !starts_out)) ||
      (rows && table_width && (!table || !table_out)) || (num_pages && pool_bad(pool, planes, page_bytes)))
    return HQ_ERR_NULL_POINTER;
  if (((uintptr_t)pool & 15) || (((uintptr_t)table | (uintptr_t)lengths | (uintptr_t)refs | (uintptr_t)parent | (uintptr_t)add |
                                  (uintptr_t)table_out | (uintptr_t)lengths_out | (uintptr_t)refs_out | (uintptr_t)starts_out | (uintptr_t)missing) & 3))
    return HQ_ERR_MISALIGNED;
  const int64_t entries = (int64_t)rows * table_width;
  // lengths rounded up to whole pages, entries and pages stay in 32 bits, as do the stretches in which pages are gone through
  if (rows > 16384 || ((int64_t)table_width + 1) * page_size > INT_MAX - 1024 || entries > INT_MAX - 1024 || num_pages > INT_MAX / 4) return HQ_ERR_TOO_LARGE;
  const void* ins[] = {table, lengths, refs, parent, add};
  const int64_t nin[] = {4 * entries, 4 * (int64_t)rows, 4 * (int64_t)num_pages, 4 * (int64_t)rows, 4 * (int64_t)rows};
  const void* outs[] = {table_out, lengths_out, refs_out, starts_out, missing};
  const int64_t nout[] = {4 * entries, 4 * (int64_t)rows, 4 * (int64_t)num_pages, 4 * (int64_t)rows, 4};
  for (int i = 0; i < 5; ++i)
    for (int j = 0; j < 5; ++j)
      if (meet(ins[i], nin[i], outs[j], nout[j]) || (i < j && meet(outs[i], nout[i], outs[j], nout[j]))) return HQ_ERR_BAD_SHAPE;
  const HqDevice* dev = nullptr;
  int rc = hq_current_device(&dev);
  if (rc != HQ_OK) return rc;
  StepArgs a{};
  a.pool = (hq_u4v*)pool;
  a.table = table;
  a.lengths = lengths;
  a.refs = refs;
  a.parent = parent;
  a.add = add;
  a.table_out = table_out;
  a.lengths_out = lengths_out;
  a.refs_out = refs_out;
  a.starts_out = starts_out;
  a.missing = missing;
  a.page_pieces = page_bytes / 16;
  a.planes = planes;
  a.rows = rows;
  a.width = table_width;
  a.pages = num_pages;
  a.page = page_size;
  if (rows <= kSmallRows && entries <= kSmallEntries && num_pages <= kStretch) {
    // one workgroup a compute unit, two where there may be a lot to copy
    const int64_t bytes = (int64_t)rows * planes * page_bytes, each = bytes > (int64_t)1 << 26 ? 2 : 1;
    const int64_t most = std::max((entries + kSmallRows - 1) / kSmallRows, page_bytes ? ((int64_t)rows * planes + 3) / 4 : 0);
    return hq_launch_as_is(step_small_kernel, dim3((unsigned)std::max<int64_t>(1, std::min(most, each * dev->cus))), dim3(kSmallRows), 0,
                           (hipStream_t)stream, a);
  }
  HqWorkspace ws;
  const int64_t most = entries < num_pages ? entries : num_pages;
  rc = hq_get_workspace((hipStream_t)stream, (size_t)(4 * (int64_t)rows + 1 + most), (size_t)num_pages + 1, &ws);
  if (rc != HQ_OK) return rc;
  a.need = (int*)ws.partial;
  a.source = a.need + rows;
  a.copies = a.source + rows;
  a.ncopies = a.copies + 2 * (int64_t)rows;
  a.list = a.ncopies + 1;
  a.arrived = ws.counters;
  a.change = (int*)ws.counters + 1;
  const size_t lds = 8 * (size_t)rows + 4 * kListLds;
  static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(&step_kernel), hipFuncAttributeMaxDynamicSharedMemorySize, 8 * 16384 + 4 * kListLds);
  if (attr != hipSuccess) return (int)attr;
  rc = hq_launch_as_is(step_kernel, dim3(rows > 1 ? rows : 1), dim3(kThreads), lds, (hipStream_t)stream, a);
  if (rc != HQ_OK || rows == 0 || planes == 0 || page_bytes == 0 || num_pages == 0) return rc;
  const int64_t items = (int64_t)rows * planes, grid = 16 * (int64_t)dev->cus;
  return hq_launch_as_is(step_copy_kernel, dim3((unsigned)(items < grid ? items : grid)), dim3(kThreads), 0, (hipStream_t)stream, a);
}

extern "C" int hq_cache_compact(void* pool, int planes, int64_t page_bytes, const int32_t* table, const int32_t* refs, int32_t* table_out,
                                int32_t* refs_out, int32_t* live, int rows, int table_width, int num_pages, void* stream) {
  if (planes < 0 || page_bytes < 0 || page_bytes % 16 || rows < 0 || table_width < 0 || num_pages < 0) return HQ_ERR_BAD_SHAPE;
  const int64_t entries = (int64_t)rows * table_width;
  if (!live || (num_pages && (!refs || !refs_out)) || (entries && (!table || !table_out)) || (num_pages && pool_bad(pool, planes, page_bytes)))
    return HQ_ERR_NULL_POINTER;
  if (((uintptr_t)pool & 15) || (((uintptr_t)table | (uintptr_t)refs | (uintptr_t)table_out | (uintptr_t)refs_out | (uintptr_t)live) & 3))
    return HQ_ERR_MISALIGNED;
  if (entries > INT_MAX || num_pages > INT_MAX / 4) return HQ_ERR_TOO_LARGE;
  const void* ins[] = {table, refs};
  const int64_t nin[] = {4 * entries, 4 * (int64_t)num_pages};
  const void* outs[] = {table_out, refs_out, live};
  const int64_t nout[] = {4 * entries, 4 * (int64_t)num_pages, 4};
  for (int i = 0; i < 3; ++i)
    for (int j = 0; j < 3; ++j)
      if ((i < 2 && meet(ins[i], nin[i], outs[j], nout[j])) || (i < j && meet(outs[i], nout[i], outs[j], nout[j]))) return HQ_ERR_BAD_SHAPE;
  const HqDevice* dev = nullptr;
  int rc = hq_current_device(&dev);
  if (rc != HQ_OK) return rc;
  CompactArgs a{};
  a.pool = (hq_u4v*)pool;
  a.table = table;
  a.refs = refs;
  a.table_out = table_out;
  a.refs_out = refs_out;
  a.live = live;
  a.page_pieces = page_bytes / 16;
  a.planes = planes;
  a.rows = rows;
  a.width = table_width;
  a.pages = num_pages;
  // workgroups that can have something to do
  const int64_t most = std::max({(int64_t)1, (entries + kThreads - 1) / kThreads, page_bytes ? (int64_t)(num_pages / 2) * planes : 0});
  // One launch, in which every workgroup makes the plan (no more of them than the pages' bytes are worth), or, for pools from 1 GiB on, a
  // plan and then copies in the order of the grid, which is only worth its second launch and its workgroups without work where much
  // moves (2048 pages, a third of them holes at random; 2 GiB: 191 us and 167, 1 GiB 95 and 90, 512 MiB 46 and 52; 2 GiB of which 100
  // pages move 43 and 54, two pages 12 and 16).
  const int64_t bytes = num_pages * page_bytes * planes, each = bytes > (int64_t)1 << 28 ? 6 : 1;
  if (num_pages <= kStretch && num_pages > 0 && bytes < (int64_t)1 << 30)
    return hq_launch_as_is(compact_small_kernel, dim3((unsigned)std::min<int64_t>(most, each * dev->cus)), dim3(kThreads), 0, (hipStream_t)stream, a);
  HqWorkspace ws;
  rc = hq_get_workspace((hipStream_t)stream, (size_t)(2 * (int64_t)num_pages + 1), 0, &ws);
  if (rc != HQ_OK) return rc;
  a.nmoves = (int*)ws.partial;
  a.to = a.nmoves + 1;
  a.pairs = a.to + num_pages;  // half of the pages at most move
  rc = hq_launch_as_is(compact_plan_kernel, dim3(1), dim3(kThreads), 0, (hipStream_t)stream, a);
  if (rc != HQ_OK || (entries == 0 && (planes == 0 || page_bytes == 0))) return rc;
  return hq_launch_as_is(compact_move_kernel, dim3((unsigned)std::min<int64_t>(most * std::max<int64_t>(1, (page_bytes / 16 + kThreads - 1) / kThreads), 32768)), dim3(kThreads), 0, (hipStream_t)stream, a);
}
