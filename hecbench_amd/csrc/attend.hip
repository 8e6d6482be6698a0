// Attention over whole prompts packed one behind the other, and of one query a request over a paged cache.
#include "attend.h"

namespace {

// ---- prompts -------------------------------------------------------------------------------------------------------
struct PromptArgs {
  const void *q, *k, *v;
  void* out;
  const int *cu_q, *cu_k;
  int64_t qs, ks, vs;  // elements from one token to the next
  float *po, *pm;      // shares of the sums [total_q * heads][shares][D], and {maximum, sum} [total_q * heads][shares]
  int seqs, total_q, total_k, heads, kv_heads, ratio, causal, shares;
  float c;
  int window, sinks;   // of a windowed call
};

// A workgroup's rows and share of the keys.  Many rows: all keys, and the result; few: the keys are divided among `shares` workgroups.
// WINDOW: keys between the first ones and the rows' windows are left out (Skip), and all below counts without them.
template <typename T, int D, bool WINDOW>
__global__ __launch_bounds__(kThreads, D == 64 ? 4 : 2) void prompt_kernel(PromptArgs a) {
  typedef Many<T, D, WINDOW> A;
  typedef typename Kind<T>::V8 V8;
  constexpr int ROWS = 128;
  extern __shared__ __align__(16) char sm[];
  __shared__ int poison;
  uint32_t x = blockIdx.x;
  const int head = x % (uint32_t)a.kv_heads;
  x /= (uint32_t)a.kv_heads;
  int share = 0;
  if (a.shares > 1) {
    share = x % (uint32_t)a.shares;
    x /= (uint32_t)a.shares;
  }
  const uint32_t ratio = a.ratio;
  Sequence s;
  if (!find_tile(a, x, [=](int n) { return (int)((n * ratio + ROWS - 1) / ROWS); }, &s)) return;
  const int q0 = s.q0, nq = s.nq, k0 = s.k0, nk = s.nk, rows = nq * ratio;
  const int tile = (rows + ROWS - 1) / ROWS - 1 - s.tile;  // the tiles with most keys come first
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int first_row = tile * ROWS, last_row = min(first_row + ROWS, rows) - 1;
  const int row = first_row + wave * 32 + (lane & 31), r = min(row, last_row);
  const int token = (uint32_t)r / ratio, h = head * ratio + (r - token * ratio);
  A w;
  w.sm = sm;
  w.poison = &poison;
  set_up(&poison);
  const T* q = (const T*)a.q + (int64_t)(q0 + token) * a.qs + (int64_t)h * D + 8 * (lane >> 5);
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) w.qf[kk] = *reinterpret_cast<const V8*>(q + 16 * kk);
  auto limit = [&](int t) { return a.causal ? min(max(t + 1 + nk - nq, 0), nk) : nk; };
  w.lim = limit(token);
  PackedTiles<T, D, WINDOW> src;
  int lo_whole = 0;
  if (WINDOW) {
    const int first_place = (int)((uint32_t)first_row / ratio) - nq + nk, last_place = (int)((uint32_t)last_row / ratio) - nq + nk;
    src.skip = skip_of(first_place, last_place, a.window, a.sinks);
    w.lim -= src.skip.gap;
    w.lo = window_of(token - nq + nk, a.window) - src.skip.gap;
    w.sinks = a.sinks;
    w.lo_most = __builtin_amdgcn_readlane(w.lo, 31);
    lo_whole = uniform(window_of(last_place, a.window) - src.skip.gap);
  }
  w.all_see = __builtin_amdgcn_readlane(w.lim, 0);  // a later row sees as much or more
  w.any_sees = __builtin_amdgcn_readlane(w.lim, 31);
  src.k = (const T*)a.k + (int64_t)k0 * a.ks + head * D;
  src.v = (const T*)a.v + (int64_t)k0 * a.vs + head * D;
  src.ks = a.ks;
  src.vs = a.vs;
  src.n = nk - src.skip.gap;
  const int end = uniform(limit((uint32_t)last_row / ratio)) - src.skip.gap, all = WINDOW ? end : nk;
  const int each = a.shares == 1 ? all : max(256, ((all + a.shares - 1) / a.shares + A::TILE - 1) & -A::TILE);
  const int first = (int)min((int64_t)share * each, (int64_t)end);
  w.run(src, first, min(end, first + each), uniform(limit((uint32_t)first_row / ratio)) - src.skip.gap, a.c, lo_whole);
  if (row > last_row) return;  // and so does the partner
  if (a.shares == 1) {
    w.put((T*)a.out + ((int64_t)(q0 + token) * a.heads + h) * D, w.lim == 0);
  } else {
    const bool sees = w.lim > first && (!WINDOW || w.lo < first + each || w.sinks > first);
    w.put_share(a.po, a.pm, ((int64_t)(q0 + token) * a.heads + h) * a.shares + share, sees);
  }
}

// ---- one query a request, over pages -----------------------------------------------------------------------------------
struct PagedArgs {
  const void *q, *k, *v;
  void* out;
  const int *table, *lengths, *groups, *shared;
  float *po, *pm;      // a place for each share of each row: its sums [D]; and its {maximum, sum}
  unsigned* arrived;   // not null: nothing is common, and the last of a request's and head's shares to arrive joins them
  int* np;             // said by the kernel: shares that the common keys are divided into, and of each request whether it has any; without
                       // groups, the first of each request's shares, and how many
  int64_t qs;
  int ngroups, batch, width, pages, page_log, heads, kv_heads, ratio;
  int most_np, ns;     // at most; shares of a request's own keys; without groups, 0: by their number
  int per_row, items;  // places from a row's to the next one's; without groups, shares of all requests, at most
  int prefix_items;    // workgroups of the common keys
  int likely;          // shares that the common keys are divided into, if groups are alike
  float c;
};

// The groups of requests, 64 at a time, a lane each: first request, requests, and the tokens that they have in common: those of the first
// one's row that the caller says are, in whole pages (what is behind is in the same page too, but every request reads what it has
// there as its own).  The lengths are the only load that waits for another.
struct Groups {
  int begin, count, shared;
  __device__ __forceinline__ Groups(const PagedArgs& a, int g0) {
    const int g = g0 + (threadIdx.x & 63), at = min(g, a.ngroups - 1);
    const int b = a.groups[at], e = a.groups[at + 1], s = a.shared[at];
    begin = min(max(b, 0), a.batch);
    count = g < a.ngroups ? min(max(e, begin), a.batch) - begin : 0;
    shared = min(min(max(s, 0), max(a.lengths[min(begin, a.batch - 1)], 0)), a.width << a.page_log) & -(1 << a.page_log);
  }
};
// Common tokens of request b's group; -1: it is in none.
__device__ __forceinline__ int shared_of(const PagedArgs& a, int b) {
  for (int g0 = 0; g0 < a.ngroups; g0 += 64) {
    const Groups g(a, g0);
    const unsigned long long here = __ballot(b >= g.begin && b < g.begin + g.count);
    if (here) return __builtin_amdgcn_readlane(g.shared, __ffsll(here) - 1);
  }
  return -1;
}

// Keys of share s of n, as many as make `shares` shares of whole tiles of 128, `least` at least.
__device__ __forceinline__ void share_of(int n, int shares, int least, int s, int* first, int* end) {
  const int each = max(least, ((n + shares - 1) / shares + 127) & ~127);
  *first = (int)min((int64_t)s * each, (int64_t)n);
  *end = min(*first + each, n);
}

// Share x of the requests' keys, all of one size: the smallest multiple of 128 of which there are no more shares than a.items, one a
// request at least.  Lengths differ, and a share is a workgroup's work (32 requests of up to 4000, two equal shares each: 62.0 us, 57.2
// so; 16 of up to 1000: 13.0 and 12.4; but 8 of up to 2000, whose 128s are a few more than the shares, 12.0 and 12.9).  Runs of equal
// length, whoever's the keys are, are better still for such (56.4), but a workgroup that goes on to the next request waits for it (8 of
// up to 2000: 13.7).  A request a lane; one request, and more than 64, in a.ns equal shares each.
constexpr int kUnit = 128;
struct Share {
  int b, first, end, before, count;  // request; keys; shares of the requests before it, and of it
  // false: there is no such share
  __device__ __forceinline__ bool find(const PagedArgs& a, unsigned x, bool says) {
    const int lane = threadIdx.x & 63, cap = a.width << a.page_log;
    if (a.ns) {
      b = x / (uint32_t)a.ns;
      before = b * a.ns;
      count = a.ns;
      share_of(min(max(a.lengths[b], 0), cap), a.ns, kUnit, x - before, &first, &end);
      return true;
    }
    const int n = min(max(a.lengths[min(lane, a.batch - 1)], 0), cap);
    const unsigned units = lane < a.batch ? max((unsigned)(n + kUnit - 1) / kUnit, 1u) : 0, items = a.items;
    unsigned each = 1, own = units, all = wave_sum(units);
    while (all > items) {  // ends where the longest request is one share
      each += max(1u, (unsigned)((float)each * (float)(all - items) / (float)items));
      // as many as hold them all; one too many, and without a key, where the quotient is a whole number but for its rounding
      own = lane < a.batch ? (unsigned)((float)(units - 1) * (__builtin_amdgcn_rcpf((float)each) * 1.000001f)) + 1 : 0;
      all = wave_sum(own);
    }
    if (x >= all) return false;
    const unsigned to = running_sum(own);
    if (says && lane < a.batch) {
      a.np[2 * lane] = to - own;
      a.np[2 * lane + 1] = own;
    }
    b = __ffsll(__ballot(to > x)) - 1;
    const int keys = __builtin_amdgcn_readlane(n, b);
    count = __builtin_amdgcn_readlane(own, b);
    before = __builtin_amdgcn_readlane(to, b) - count;
    first = (int)min((int64_t)(x - before) * each * kUnit, (int64_t)keys);
    end = (int)min((int64_t)(x - before + 1) * each * kUnit, (int64_t)keys);
    return true;
  }
};

template <typename T, int D>
__device__ __forceinline__ Pages<T, D> pages_of(const PagedArgs& a, int request, int head) {
  return Pages<T, D>((const T*)a.k, (const T*)a.v, a.table + (int64_t)request * a.width, head, a.kv_heads, a.page_log, a.pages);
}

// Up to 16 rows (request, head of the group), those of requests b0 ..., all of which see the keys.
template <typename T, int D, bool JOINS>
__device__ __forceinline__ void few_rows(const PagedArgs& a, char* sm, int b0, int nrows, int head, int first, int end, int64_t slot,
                                         int shares, int before, int item) {
  typedef typename Kind<T>::V8 V8;
  const int lane = threadIdx.x & 63, last_row = nrows - 1, r = min(lane & 15, last_row);
  const uint32_t ratio = a.ratio;
  const int b = b0 + (uint32_t)r / ratio, h = head * ratio + (uint32_t)r % ratio;
  Few<T, D> w;
  w.sm = sm;
  const T* q = (const T*)a.q + (int64_t)b * a.qs + (int64_t)h * D + 8 * (lane >> 4);
#pragma unroll
  for (int kk = 0; kk < D / 32; ++kk) w.qf[kk] = *reinterpret_cast<const V8*>(q + 32 * kk);
  w.run(pages_of<T, D>(a, b0, head), first, end, a.c);
  float sum[D / 16], top, total;
  w.join(sum, &top, &total);
  const int mine = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * (D / 16);
  const bool row = mine <= last_row;
  const int64_t at = (int64_t)(b0 + (uint32_t)mine / ratio) * a.heads + head * ratio + (uint32_t)mine % ratio;
  typedef T TD __attribute__((ext_vector_type(D / 16)));
  if (shares == 1) {
    TD v;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) v[i] = (T)(first >= end ? 0.f : result(sum[i], sum[i] / total));
    if (row) *reinterpret_cast<TD*>((T*)a.out + at * D + d0) = v;
    return;
  }
  if (row) {
    const int64_t place = at * a.per_row + slot;
#pragma unroll
    for (int i = 0; i < D / 16; i += 4)
      hq_store_share(reinterpret_cast<hq_f4v*>(a.po + place * D + d0 + i), hq_f4v{sum[i], sum[i + 1], sum[i + 2], sum[i + 3]});
    if (d0 == 0)
      __hip_atomic_store(reinterpret_cast<unsigned long long*>(a.pm) + place, (unsigned long long)__float_as_uint(total) << 32 | __float_as_uint(share_top(top, first < end)),
                         __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (!JOINS || !a.arrived) return;
  // The last share to arrive joins them all, and there is no second launch.  (32 / 8 heads of 128; a request of 333 keys in two launches 9.8 us,
  // in one 8.0; 4 of 8192, 16 shares, 29.6 and 28.7; 2 of 8192, 32 shares, 16.4 and 16.8; one, 64 shares at once, 11.9 and 14.5.)  The trips of the
  // last one grow with the shares, of which a long request among short ones has many: beyond 32, every 16 are joined first, by the last of them
  // (12 / 1 heads, one of 60000 among 16 of a token, 469 shares: 86.6 us at once, 22.1).
  __shared__ unsigned nth;
  int n = shares, unit = 1, index = item - before;  // what there is to be joined, shares of each, and which of them this is
  for (;;) {
    const bool all = n <= kJoin;
    const int team = all ? 0 : index / kTeam, members = all ? n : min(kTeam, n - team * kTeam), first_share = before + team * kTeam * unit;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    unsigned* const count = a.arrived + (int64_t)((all ? a.items + b0 : first_share) * a.kv_heads + head) * kApart;
    if (threadIdx.x == 0) nth = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (nth != (unsigned)members - 1) return;
    if (threadIdx.x == 0) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const int64_t row0 = (int64_t)b0 * a.heads + head * ratio;
    join_here<T, D>(a, sm, nrows, row0, (int64_t)(first_share - b0) * a.heads, (int64_t)unit * a.heads, members, all, [=](int row) { return row0 + row; });
    if (all) return;
    index = team;
    n = (n + kTeam - 1) / kTeam;
    unit *= kTeam;
  }
}

// Up to 128 of them; a row sees keys up to its request's length.
template <typename T, int D>
__device__ __forceinline__ void many_rows(const PagedArgs& a, char* sm, int* poison, int b0, int nrows, int first_row, int head, int first, int end,
                                          int64_t slot, int shares) {
  typedef typename Kind<T>::V8 V8;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int last_row = min(first_row + 128, nrows) - 1, row = first_row + wave * 32 + (lane & 31), r = min(row, last_row);
  const uint32_t ratio = a.ratio;
  const int b = b0 + (uint32_t)r / ratio, h = head * ratio + (uint32_t)r % ratio;
  Many<T, D> w;
  w.sm = sm;
  w.poison = poison;
  set_up(poison);
  const T* q = (const T*)a.q + (int64_t)b * a.qs + (int64_t)h * D + 8 * (lane >> 5);
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) w.qf[kk] = *reinterpret_cast<const V8*>(q + 16 * kk);
  w.lim = min(min(max(a.lengths[b], 0), a.width << a.page_log), end);
  w.all_see = uniform(wave_min(w.lim));
  w.any_sees = first_row + wave * 32 > last_row ? 0 : -uniform(wave_min(-w.lim));  // a wave without rows works on nothing
  __shared__ int seen[kWaves];  // what every row of the workgroup sees
  if (lane == 0) seen[wave] = w.all_see;
  __syncthreads();
  const int whole = min(min(seen[0], seen[1]), min(seen[2], seen[3]));
  PagedTiles<T, D, false, 1, false> src(pages_of<T, D>(a, b0, head), end);
  w.run(src, first, end, uniform(whole), a.c);
  // the row, worked out once more: in the loop there is no register to spare
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
  const int mine = first_row + (tid >> 6) * 32 + (tid & 31);
  if (mine > last_row) return;
  const int64_t at = (int64_t)(b0 + (uint32_t)mine / ratio) * a.heads + head * ratio + (uint32_t)mine % ratio;
  if (shares == 1) w.put((T*)a.out + at * D, w.lim == 0);
  else w.put_share(a.po, a.pm, at * a.per_row + slot, w.lim > first);
}

// Nothing is common: a share a workgroup.
template <typename T, int D, bool FEW>
__global__ __launch_bounds__(kThreads, D == 64 ? 3 : 2) void paged_alone_kernel(PagedArgs a) {
  extern __shared__ __align__(16) char sm[];
  __shared__ int poison;
  const uint32_t x = blockIdx.x, y = x / (uint32_t)a.kv_heads, item = y % (uint32_t)a.items;
  const int head = x % (uint32_t)a.kv_heads, row0 = y / (uint32_t)a.items * 128;
  Share s;
  if (!s.find(a, item, x == 0 && threadIdx.x < 64 && a.np)) return;
  const int64_t place = ((int64_t)item - s.b) * a.heads;
  if (FEW) few_rows<T, D, true>(a, sm, s.b, a.ratio, head, s.first, s.end, place, s.count, s.before, item);
  else many_rows<T, D>(a, sm, &poison, s.b, a.ratio, row0, head, s.first, s.end, place, s.count);
}

template <typename T, int D>
__global__ __launch_bounds__(kThreads, D == 64 ? 3 : 2) void paged_kernel(PagedArgs a) {
  extern __shared__ __align__(16) char sm[];
  __shared__ int poison;
  uint32_t x = blockIdx.x;
  int b0 = 0, nb = 1, row0 = 0, head, first, end, slot;
  bool few = a.ratio <= 16;
  if ((int)x < a.prefix_items) {
    // The common keys: as many shares as there are workgroups for the tiles of rows that there are.
    const int ratio = a.ratio, lane = threadIdx.x & 63;
    auto tiles = [=](const Groups& g) { return (int)(((int64_t)g.count * ratio + 127) / 128); };
    const Groups some(a, 0);
    int all = __builtin_amdgcn_readlane((int)running_sum(tiles(some)), 63);
    for (int g0 = 64; g0 < a.ngroups; g0 += 64) all += __builtin_amdgcn_readlane((int)running_sum(tiles(Groups(a, g0))), 63);
    const int np = all ? min(max(a.prefix_items / (all * a.kv_heads), 1), a.most_np) : 0;
    if (x == 0 && threadIdx.x == 0) *a.np = np;
    if (np == 0) return;
    head = x % (uint32_t)a.kv_heads;
    x /= (uint32_t)a.kv_heads;
    slot = x % (uint32_t)np;
    int tile = x / (uint32_t)np;
    if (tile >= all) return;
    int n = 0;
    nb = 0;
    for (int g0 = 0; nb == 0 && g0 < a.ngroups; g0 += 64) {
      const Groups g = g0 ? Groups(a, g0) : some;
      const int own = tiles(g), sum = (int)running_sum(own), total = __builtin_amdgcn_readlane(sum, 63);
      if (tile < total) {
        const int at = __ffsll(__ballot(sum > tile)) - 1;
        b0 = __builtin_amdgcn_readlane(g.begin, at);
        nb = __builtin_amdgcn_readlane(g.count, at);
        n = __builtin_amdgcn_readlane(g.shared, at);
        tile -= __builtin_amdgcn_readlane(sum - own, at);
      } else {
        tile -= total;
      }
    }
    if (nb == 0) return;  // only where bounds that do not ascend make more tiles than 32 bits count
    share_of(n, np, 256, slot, &first, &end);
    few = nb * ratio <= 16 && !__ballot(lane < nb && a.lengths[b0 + min(lane, nb - 1)] < end);
    row0 = tile * 128;
  } else {
    x -= a.prefix_items;
    head = x % (uint32_t)a.kv_heads;
    x /= (uint32_t)a.kv_heads;
    const int share = x % (uint32_t)a.ns;
    x /= (uint32_t)a.ns;
    const int tiles = few ? 1 : (a.ratio + 127) / 128, tile = few ? 0 : x % (uint32_t)tiles;
    b0 = few ? x : x / (uint32_t)tiles;
    const int n = min(max(a.lengths[b0], 0), a.width << a.page_log), shared = shared_of(a, b0), from = uniform(min(max(shared, 0), n));
    if (head == 0 && share == 0 && tile == 0 && threadIdx.x == 0) a.np[1 + b0] = shared >= 0;
    share_of(n - from, a.ns, 128, share, &first, &end);
    first += from;
    end += from;
    row0 = tile * 128;
    slot = a.most_np + share;
  }
  if (few) few_rows<T, D, false>(a, sm, b0, nb * a.ratio, head, first, end, slot, 0, 0, 0);
  else many_rows<T, D>(a, sm, &poison, b0, nb * a.ratio, row0, head, first, end, slot, 0);
}

template <typename T, int D, int WAVES, int PRE>
__global__ __launch_bounds__(kThreads) void join_paged_kernel(PagedArgs a) {
  const int64_t row = WAVES > 1 ? blockIdx.x : (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (row >= (int64_t)a.batch * a.heads) return;
  const int b = row / a.heads, slots = a.most_np + a.ns;
  if (a.ngroups) {
    const int np = a.np[1 + b] ? a.np[0] : 0;
    join_shares<T, D, WAVES, PRE>(a.po, a.pm, row, row * slots, 1, np, a.most_np, slots, a.likely, (T*)a.out);
  } else {
    const int before = a.ns ? b * a.ns : a.np[2 * b], count = a.ns ? a.ns : a.np[2 * b + 1];
    if (count > 1) join_shares<T, D, WAVES, PRE>(a.po, a.pm, row, row + (int64_t)(before - b) * a.heads, a.heads, count, count, count, count, (T*)a.out);
  }
}

template <typename T, int D, int WAVES, int PRE>
__global__ __launch_bounds__(kThreads) void join_prompt_kernel(PromptArgs a) {
  const int64_t row = WAVES > 1 ? blockIdx.x : (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (row >= (int64_t)a.total_q * a.heads) return;
  const int token = row / a.heads;
  if (token < a.cu_q[0] || token >= a.cu_q[a.seqs]) return;
  join_shares<T, D, WAVES, PRE>(a.po, a.pm, row, row * a.shares, 1, 0, 0, a.shares, 0, (T*)a.out);
}

// Few rows leave compute units idle, and each of their workgroups with all keys: then the keys are divided, 256 a share at least, and the
// shares joined by a second launch.  Into how many parts, an estimate says, of sequences of the average length (lengths are device memory),
// in us: a tile of 64 keys takes a workgroup 1.04 alone (heads of 64: 0.88), a compute unit 0.96 (0.65) where it has more of them, and
// every share of a row is written and read.  40 tokens behind 2900 keys, 32 / 8 heads of 128: 50.9 us, in 12 shares 16.1; 512 behind
// 8000 143.8, in four 90.5; 1000 by themselves 24.0, in two 35.9; 17 sequences of up to 248, 12 / 1 heads, 11.7 and 29.1.  A window
// makes the keys fewer.
template <typename T, int D, bool WINDOW>
int launch_prompt(PromptArgs a, int cus, hipStream_t stream) {
  const int64_t items = ((int64_t)a.total_q * a.ratio / 128 + a.seqs) * a.kv_heads, rows = (int64_t)a.total_q * a.heads;
  const float queries = (float)a.total_q / a.seqs, all_keys = (float)a.total_k / a.seqs;
  const float keys = WINDOW ? std::min(all_keys, (float)a.window + std::min((float)a.sinks, all_keys) + 128.f / a.ratio) : all_keys;
  const float unit = (D == 128 ? 0.96f : 0.65f) / cus * std::max(queries * a.ratio / 128, 1.f) * a.seqs * a.kv_heads;
  const float deepest = keys / 64, mean = (a.causal ? keys - std::min(queries, all_keys) / 2 * (keys / all_keys) : keys) / 64;
  float best = INFINITY;
  for (int s = 1; s <= 64 && (s == 1 || (s * items <= 4 * (int64_t)cus && (s - 1) * 256 < keys)); ++s) {
    const float depth = s == 1 ? deepest : std::max(2 * std::ceil(keys / (128 * s)), 4.f);  // whole 128s
    const float us = std::max(depth * (D == 128 ? 1.04f : 0.88f), mean * unit) + (s == 1 ? 0.f : 4.f + (float)rows * s * (D + 2) * 8 / 4.2e6f);
    if (us < best) {
      best = us;
      a.shares = s;
    }
  }
  const size_t floats = rows * a.shares * (D + 2);
  if (a.shares > 1 && hq_workspace_out_of_reach(stream, floats, 0)) a.shares = 1;  // longer, and no error
  if (items * a.shares > INT_MAX) return HQ_ERR_TOO_LARGE;
  if (a.shares > 1) {
    HqWorkspace ws;
    const int rc = hq_get_workspace(stream, floats, 0, &ws);
    if (rc != HQ_OK) return rc;
    a.po = ws.partial;
    a.pm = ws.partial + rows * a.shares * D;
  }
  const int rc = hq_launch_as_is(prompt_kernel<T, D, WINDOW>, dim3((unsigned)(items * a.shares)), dim3(kThreads), Many<T, D>::LDS, stream, a);
  if (rc != HQ_OK || a.shares == 1) return rc;
  return launch_join(Joins<PromptArgs>{join_prompt_kernel<T, D, 1, 0>, join_prompt_kernel<T, D, kWaves, 0>, join_prompt_kernel<T, D, 1, 8>,
                                       join_prompt_kernel<T, D, kWaves, 8>},
                     rows, a.shares, stream, a);
}

// Common keys: a workgroup a compute unit for them, two for heads of 64, and the requests' own keys divided until they fill as many (64
// requests in 4 groups behind 15000 keys, 32 / 8 heads, own up to 500: heads of 128 72.9 us, with two 78.1; of 64 50.0, with two 43.2).
// Nothing common: two workgroups a compute unit, of shares by length (Share).
template <typename T, int D>
int launch_paged(PagedArgs a, int cus, hipStream_t stream) {
  const int64_t cap = (int64_t)a.width << a.page_log, rows = (int64_t)a.batch * a.heads, tiles = a.ratio <= 16 ? 1 : (a.ratio + 127) / 128;
  const int64_t own = (int64_t)a.batch * a.kv_heads * tiles;
  if (a.ngroups >= a.batch) a.ngroups = 0;  // groups of one, as good as: whoever shares nothing is not asked about it
  int64_t prefix, grid, slots, places, joined;
  size_t floats, counters;
  bool alone, divide = true;
  for (;;) {
    prefix = 0;
    alone = false;
    if (a.ngroups) {
      const int64_t most_tiles = (int64_t)a.batch * a.ratio / 128 + a.ngroups;
      const int64_t common = D == 64 ? 2 * cus : cus;
      prefix = std::max<int64_t>(common, most_tiles * a.kv_heads);
      a.most_np = (int)std::max<int64_t>(1, std::min<int64_t>(common / a.kv_heads, (cap + 255) / 256));
      a.ns = (int)std::max<int64_t>(1, std::min(cus / own, (cap + 127) / 128));
      grid = prefix + own * a.ns;
      slots = a.per_row = a.most_np + a.ns;
      places = rows * slots;
      // The kernel uses as many of them as there are workgroups for the tiles, groups alike these; where rows are many, by them is how the
      // shares are joined (9 of 33: 4096 rows 80.7 -> 78.8 us with the whole call, 2048 rows 72.6 -> 73.4).
      a.likely = (int)std::min<int64_t>(a.most_np, prefix / (a.kv_heads * std::max<int64_t>(a.ngroups, (int64_t)a.batch * a.ratio / 128)));
      joined = (rows >= 4096 ? a.likely : a.most_np) + a.ns;
    } else {
      a.per_row = 1;
      const int64_t most = a.batch * std::max<int64_t>(1, (cap + kUnit - 1) / kUnit), room = divide ? share_room(cus, a.kv_heads * tiles) : 1;
      a.ns = 0;
      if (a.batch == 1 || a.batch > 64 || a.batch >= room || a.batch == most) a.ns = (int)std::max<int64_t>(1, std::min(room, most) / a.batch);
      a.items = (int)(a.ns ? (int64_t)a.ns * a.batch : std::min(room, most));
      grid = (int64_t)a.items * a.kv_heads * tiles;
      places = a.ns == 1 ? 0 : (int64_t)a.items * a.heads;
      slots = joined = a.items / a.batch;
      alone = a.ratio <= 16 && slots <= 32;
    }
    floats = places * (D + 2) + 1 + 2 * (int64_t)a.batch;
    counters = alone ? (a.items + (int64_t)a.batch) * a.kv_heads * kApart : 0;  // a place for every share's team, and one for the request
    // While the stream is captured and has no room for shares: every request by itself, then in one share.  Longer, and no error.
    if (!places || !hq_workspace_out_of_reach(stream, floats, counters)) break;
    if (!a.ngroups) divide = false;
    a.ngroups = 0;
  }
  if (grid > INT_MAX) return HQ_ERR_TOO_LARGE;
  a.prefix_items = (int)prefix;
  if (places) {
    HqWorkspace ws;
    const int rc = hq_get_workspace(stream, floats, counters, &ws);
    if (rc != HQ_OK) return rc;
    a.arrived = alone ? ws.counters : nullptr;
    a.po = ws.partial;
    a.pm = a.po + places * D;
    a.np = alone ? nullptr : reinterpret_cast<int*>(a.pm + 2 * places);
  }
  void (*const kernel)(PagedArgs) = a.ngroups ? paged_kernel<T, D> : tiles == 1 && a.ratio <= 16 ? paged_alone_kernel<T, D, true> : paged_alone_kernel<T, D, false>;
  constexpr int lds = std::max(Many<T, D>::LDS, Few<T, D>::LDS);
  static_assert(lds <= 65536, "no attribute to set");
  const int rc = hq_launch_as_is(kernel, dim3((unsigned)grid), dim3(kThreads), lds, stream, a);
  if (rc != HQ_OK || !places || alone) return rc;
  return launch_join(Joins<PagedArgs>{join_paged_kernel<T, D, 1, 0>, join_paged_kernel<T, D, kWaves, 0>, join_paged_kernel<T, D, 1, 8>,
                                      join_paged_kernel<T, D, kWaves, 8>},
                     rows, joined, stream, a);
}
}  // namespace

// window 0: none.
static int prompt_attention(const void* q, const void* k, const void* v, void* out, int dtype, const int32_t* cu_q, const int32_t* cu_k, int seqs,
                            int64_t total_q, int64_t total_k, int heads, int kv_heads, int head_dim, int64_t q_stride, int64_t k_stride,
                            int64_t v_stride, float scale, int causal, int window, int sinks, void* stream) {
  if (seqs < 0 || total_q < 0 || total_k < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads) return HQ_ERR_BAD_SHAPE;
  if (head_dim != 64 && head_dim != 128) return HQ_ERR_BAD_SHAPE;
  if (dtype != HQ_DTYPE_F16 && dtype != HQ_DTYPE_BF16) return HQ_ERR_BAD_ENUM;
  if (bad_scale(scale)) return HQ_ERR_BAD_SHAPE;
  if (seqs == 0 || total_q == 0) return HQ_OK;
  if (!q || !out || !cu_q || (total_k && (!k || !v)) || (!cu_k && total_k != total_q)) return HQ_ERR_NULL_POINTER;
  if (q_stride < (int64_t)heads * head_dim || (total_k && (k_stride < (int64_t)kv_heads * head_dim || v_stride < (int64_t)kv_heads * head_dim)))
    return HQ_ERR_BAD_SHAPE;
  if (misaligned(q, q_stride) || misaligned(k, k_stride) || misaligned(v, v_stride) || ((uintptr_t)out & 15) ||
      (((uintptr_t)cu_q | (uintptr_t)cu_k) & 3))
    return HQ_ERR_MISALIGNED;
  if (total_q > INT_MAX || total_q * (heads / kv_heads) > INT_MAX - 128 || total_k > kMostKeys || k_stride > 1 << 22 ||
      v_stride > 1 << 22)  // 32-bit offsets in a tile
    return HQ_ERR_TOO_LARGE;
  const HqDevice* dev = nullptr;
  const int rc = hq_current_device(&dev);
  if (rc != HQ_OK) return rc;
  const PromptArgs a{q, k, v, out, cu_q, cu_k ? cu_k : cu_q, q_stride, k_stride, v_stride, nullptr, nullptr, seqs, (int)total_q, (int)total_k, heads, kv_heads,
                     heads / kv_heads, causal != 0, 1, exponent_scale(scale), window, sinks};
  const hipStream_t s = (hipStream_t)stream;
  return by_type(dtype, head_dim, [&](auto f) {
    typedef decltype(f) F;
    if (window && window < total_k) return launch_prompt<typename F::T, F::D, true>(a, dev->cus, s);
    return launch_prompt<typename F::T, F::D, false>(a, dev->cus, s);
  });
}

extern "C" int hq_prompt_attention(const void* q, const void* k, const void* v, void* out, int dtype, const int32_t* cu_q,
                                   const int32_t* cu_k, int seqs, int64_t total_q, int64_t total_k, int heads, int kv_heads,
                                   int head_dim, int64_t q_stride, int64_t k_stride, int64_t v_stride, float scale, int causal,
                                   void* stream) {
  return prompt_attention(q, k, v, out, dtype, cu_q, cu_k, seqs, total_q, total_k, heads, kv_heads, head_dim, q_stride, k_stride, v_stride, scale, causal,
                          0, 0, stream);
}

extern "C" int hq_prompt_attention_window(const void* q, const void* k, const void* v, void* out, int dtype, const int32_t* cu_q,
                                          const int32_t* cu_k, int seqs, int64_t total_q, int64_t total_k, int heads, int kv_heads,
                                          int head_dim, int64_t q_stride, int64_t k_stride, int64_t v_stride, float scale, int window,
                                          int sinks, void* stream) {
  if (window < 1 || sinks < 0) return HQ_ERR_BAD_SHAPE;
  return prompt_attention(q, k, v, out, dtype, cu_q, cu_k, seqs, total_q, total_k, heads, kv_heads, head_dim, q_stride, k_stride, v_stride, scale, 1,
                          window, sinks, stream);
}

extern "C" int hq_paged_attention(const void* q, const void* k_pages, const void* v_pages, void* out, int dtype, const int32_t* table,
                                  const int32_t* lengths, const int32_t* groups, const int32_t* shared, int ngroups, int batch,
                                  int table_width, int num_pages, int page_size, int heads, int kv_heads, int head_dim, int64_t q_stride,
                                  float scale, void* stream) {
  if (batch < 0 || table_width < 0 || num_pages < 0 || ngroups < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads) return HQ_ERR_BAD_SHAPE;
  if (page_size < 8 || page_size > 1024 || (page_size & (page_size - 1))) return HQ_ERR_BAD_SHAPE;
  if (head_dim != 64 && head_dim != 128) return HQ_ERR_BAD_SHAPE;
  if (dtype != HQ_DTYPE_F16 && dtype != HQ_DTYPE_BF16) return HQ_ERR_BAD_ENUM;
  if (bad_scale(scale)) return HQ_ERR_BAD_SHAPE;
  if (batch == 0) return HQ_OK;
  if (!q || !out || !lengths || (table_width && !table) || (table_width && num_pages && (!k_pages || !v_pages)) || (ngroups && (!groups || !shared)))
    return HQ_ERR_NULL_POINTER;
  if (q_stride < (int64_t)heads * head_dim) return HQ_ERR_BAD_SHAPE;
  if (misaligned(q, q_stride) || (((uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)out) & 15) ||
      (((uintptr_t)table | (uintptr_t)lengths | (uintptr_t)groups | (uintptr_t)shared) & 3))
    return HQ_ERR_MISALIGNED;
  if ((int64_t)table_width * page_size > kMostKeys || (int64_t)batch * heads > INT_MAX / 64 ||
      (int64_t)kv_heads * head_dim * 2 * page_size > UINT32_MAX)  // bytes of a page
    return HQ_ERR_TOO_LARGE;
  const HqDevice* dev = nullptr;
  const int rc = hq_current_device(&dev);
  if (rc != HQ_OK) return rc;
  PagedArgs a{};
  a.q = q;
  a.k = k_pages;
  a.v = v_pages;
  a.out = out;
  a.table = table;
  a.lengths = lengths;
  a.groups = groups;
  a.shared = shared;
  a.qs = q_stride;
  a.ngroups = ngroups;
  a.batch = batch;
  a.width = table_width;
  a.pages = num_pages;
  a.page_log = __builtin_ctz(page_size);
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.ratio = heads / kv_heads;
  a.c = exponent_scale(scale);
  return by_type(dtype, head_dim, [&](auto f) { return launch_paged<typename decltype(f)::T, decltype(f)::D>(a, dev->cus, (hipStream_t)stream); });
}
