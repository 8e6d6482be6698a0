// Attention of the next tokens of every request - one, a few, a chunk of a prompt - over the paged cache, through a sliding window and a
// few first tokens that stay visible, or without.
//
// A request's rows are its new tokens, each with the heads of a key / value head's group; token i of n, of a request that has `length`
// tokens with them, is at place length - n + i and sees the keys up to its own (window: see Skip in attend.h).  Up to 16 rows go the way of
// few rows, bound by the keys' way from memory, the others in tiles of 128 the way of many.  The keys of a tile are divided where there
// are fewer tiles than the device has room for, and the shares meet in the launch.
#include "attend.h"

namespace {

struct ChunkArgs {
  const void *q, *k, *v;
  void* out;
  const int *table, *lengths, *cu_q;
  // Places of shares, 16 rows each of few, 128 each of many, the former first: a row's sums [D]; and its {maximum, sum}
  float *po, *pm;
  unsigned* arrived;  // counters of the shares of few rows; null: nothing is divided
  int* said;          // not null: tiles of many rows may be divided; of each request, by the kernel: its first share, and the shares of a tile
  int64_t qs;
  int batch, total_q, width, pages, page_log, heads, kv_heads, ratio;
  int few, many;      // shares of tiles of few and of many rows, at most
  int ns;             // more than 64 requests: shares of every tile; else 0: as many as there is room for
  int cus, room;      // compute units; shares for two workgroups each
  int window, sinks;
  float c;
};

constexpr int kFew = 16, kUnit = 128, kRows = 128;
// Keys that are not divided, in kUnits: of a tile of few rows (147 take a workgroup 7.3 us, two 8.9), of more than 64 (256 tokens with 356 keys, 32 / 8
// heads of 128, beside a joining launch that finds nothing 15.5 us, divided 17.8; 128 with 428 17.0 and 16.0), and of any of many where that saves the
// joining launch (128 with 428 14.8, with 628 18.6 and 16.9).  (In between every 128 keys count: 12 requests of 5 tokens, 16 / 2 heads, up to 698
// keys 15.7, 17.7 with up to 384 undivided.)
constexpr int kShort = 3, kShortOfAll = 4;

// A request: its new tokens and the tokens it has with them.
struct Request {
  int q0, nq, length;
  // false: its bounds do not ascend.
  __device__ __forceinline__ bool get(const ChunkArgs& a, int i) {
    const int qb = a.cu_q[i], qe = a.cu_q[i + 1], n = a.lengths[i];
    q0 = min(max(qb, 0), a.total_q);
    nq = min(max(qe, q0), a.total_q) - q0;
    length = min(max(n, 0), a.width << a.page_log);
    return qb <= qe;
  }
  __device__ __forceinline__ int tiles(int ratio) const {  // nq * ratio is below 2^31 - 128
    const int rows = nq * ratio;
    return rows <= kFew ? rows > 0 : (rows + kRows - 1) / kRows;
  }
  __device__ __forceinline__ int place(int token) const { return token - nq + length; }
};

// A share of a tile's keys.
struct Item {
  int b, tile, share, count, first;  // request, tile of it (the last, which sees most, first), which of how many shares, and the number of the first
  int each;                          // keys of a share; 0: divided evenly
  Request r;

  // Item x of the call.  Those of many rows come first: they are the longest, and one to a compute unit where there are no more.
  template <int D, bool WINDOW>
  __device__ __forceinline__ bool find(const ChunkArgs& a, int x, bool says) {
    const int lane = threadIdx.x & 63;
    if (a.ns) {
      // Many requests: request i has tiles_from(i) ... , as many as its rows may take at most; which one has x, 64 bounds at a time.
      auto tiles_from = [&](int i) { return (int)((int64_t)min(max(a.cu_q[i], 0), a.total_q) * a.ratio / kRows) + i; };
      const int slot = x / a.ns;
      share = x - slot * a.ns;
      int lo = 0, n = a.batch;
      while (n > 1) {
        const int step = (n + 63) >> 6;
        const bool below = lane * step < n && tiles_from(lo + lane * step) <= slot;
        const int at = max(63 - (int)__clzll(__ballot(below) | 1), 0) * step;
        lo += at;
        n = min(step, n - at);
      }
      b = lo;
      r.get(a, b);
      tile = slot - tiles_from(b);
      count = r.nq * a.ratio <= kFew ? a.ns : 1;
      each = 0;
      first = slot * a.ns;
      return tile >= 0 && tile < r.tiles(a.ratio) && share < count;
    }
    Request mine;
    // Bounds that do not ascend may hold a token many times, more tiles than the host counted on: nothing is divided then, so that no share
    // lies behind the room for them, and no counter waits for one that the grid has no workgroup for.
    const bool ascend = !__ballot(!mine.get(a, min(lane, a.batch - 1)));
    if (lane >= a.batch) mine.nq = 0;
    const int tiles = mine.tiles(a.ratio), rows = mine.nq * a.ratio;
    int keys = mine.length;
    if (WINDOW) keys = (int)min((int64_t)keys, (int64_t)min(a.sinks, keys) + a.window + 14 + (rows <= kFew ? mine.nq : kRows / a.ratio + 2));
    const unsigned few = rows <= kFew ? tiles : 0, many = tiles - few;
    const unsigned units = few && keys <= kShort * kUnit ? 1 : max((unsigned)(keys + kUnit - 1) / kUnit, 1u);
    // Tiles of more than 64 rows are divided where three shares each, or more, find room, two workgroups a compute unit; where they do not, what
    // the shares' sums cost, which are written, read and joined, is more than it brings (behind 3500 keys, 32 / 8 heads of 128: 640 tokens 63 us
    // in three shares, 78 undivided; 768 in two 74 and 78, 896 78 and 78, 1024 82 and 78).  A few of them by themselves are as fast with half as
    // many shares (128 tokens 26.2 us, with all 28.2; 384 52.8 and 46.0).  Fewer rows, bound by memory, are divided in any case.
    const unsigned all_many = wave_sum(many), heavy = rows > 64 ? tiles : 0, all_heavy = wave_sum(heavy), groups = all_heavy * a.kv_heads;
    const bool heavy_too = a.said && 3 * groups <= 2u * a.cus;
    const bool divisible = ascend && a.arrived && (rows <= kFew || (a.said && (rows <= 64 || (heavy_too && units > kShort))));
    const unsigned of = divisible ? tiles : 0, all_of = wave_sum(of);
    const bool half = heavy_too && all_of == all_heavy && 8 * groups <= (unsigned)a.cus;
    const unsigned room = half ? (a.room + 1) / 2 : a.room;
    // The keys of a share: the smallest multiple of kUnit (two of them for many rows) of which there are no more shares than there is room for, or
    // what makes one share of every tile.  (Sums stay in 32 bits.)
    unsigned per = all_many ? 2 : 1, own = 1;
    for (;;) {
      own = divisible ? min((units - 1) / per + 1, 64 * room) : 1;
      const unsigned all = wave_sum(of * own);
      if (all <= room || all <= all_of) break;
      per += max(1u, (unsigned)((float)per * (float)(all - room) / (float)room));
    }
    const unsigned all = wave_sum(many * own);
    if (says && lane < a.batch) {
      a.said[2 * lane] = running_sum(many * own) - many * own;
      a.said[2 * lane + 1] = own;
    }
    const bool is_many = x < (int)all;
    if (!is_many) {
      x -= all;
      if ((unsigned)x >= wave_sum(few * own)) return false;
    }
    const unsigned mine_of = (is_many ? many : few) * own;
    const unsigned to = running_sum(mine_of);
    b = __ffsll(__ballot((int)to > x)) - 1;
    r = Request{__builtin_amdgcn_readlane(mine.q0, b), __builtin_amdgcn_readlane(mine.nq, b), __builtin_amdgcn_readlane(mine.length, b)};
    count = __builtin_amdgcn_readlane(own, b);
    const int before = __builtin_amdgcn_readlane(to, b) - __builtin_amdgcn_readlane(mine_of, b);
    tile = (x - before) / count;
    share = x - before - tile * count;
    first = before + tile * count;
    each = per * kUnit;
    return true;
  }
  // Keys of the share, of the n that the tile goes through.
  __device__ __forceinline__ void keys(int n, int* from, int* to) const {
    const int size = each ? each : ((n + count - 1) / count + kUnit - 1) & -kUnit;
    *from = count == 1 ? 0 : (int)min((int64_t)share * size, (int64_t)n);
    *to = count == 1 ? n : (int)min((int64_t)(share + 1) * size, (int64_t)n);
  }
};

// What rows of a tile see, keys that it leaves out not counted.
struct Sight {
  const ChunkArgs& a;
  const Request& r;
  Skip skip;
  bool window;
  __device__ __forceinline__ Sight(const ChunkArgs& args, const Request& request, bool w, int first_token, int last_token) : a(args), r(request), window(w) {
    if (window) skip = skip_of(r.place(first_token), r.place(last_token), a.window, a.sinks);
  }
  __device__ __forceinline__ int limit(int token) const { return max(r.place(token) + 1, 0) - skip.gap; }
  __device__ __forceinline__ int low(int token) const { return window ? window_of(r.place(token), a.window) - skip.gap : 0; }
  // of the keys first ... end - 1, of which there are some, one at least
  __device__ __forceinline__ bool any(int token, int first, int end) const {
    return first < end && limit(token) > first && (!window || low(token) < end || a.sinks > first);
  }
};

template <typename T, int D>
__device__ __forceinline__ Pages<T, D> pages_of(const ChunkArgs& a, int request, int head) {
  return Pages<T, D>((const T*)a.k, (const T*)a.v, a.table + (int64_t)request * a.width, head, a.kv_heads, a.page_log, a.pages);
}

template <typename T, int D, bool WINDOW>
__device__ __forceinline__ void few_rows(const ChunkArgs& a, char* sm, const Item& item, int head) {
  typedef typename Kind<T>::V8 V8;
  const Request& r = item.r;
  const int lane = threadIdx.x & 63, nrows = r.nq * a.ratio;
  const uint32_t ratio = a.ratio;
  const Sight sight(a, r, WINDOW, 0, r.nq - 1);
  int first, end;
  item.keys(uniform(sight.limit(r.nq - 1)), &first, &end);
  const int mine = min(lane & 15, nrows - 1), token = (uint32_t)mine / ratio, h = head * ratio + (uint32_t)mine % ratio;
  Few<T, D, true> w;
  w.sm = sm;
  w.skip = sight.skip;
  w.lim = min(sight.limit(token), end);
  w.lo = sight.low(token);
  w.sinks = WINDOW ? a.sinks : 0;
  w.all_see = uniform(min(sight.limit(0), end));
  w.lo_most = uniform(sight.low(r.nq - 1));
  const T* q = (const T*)a.q + (int64_t)(r.q0 + token) * a.qs + (int64_t)h * D + 8 * (lane >> 4);
#pragma unroll
  for (int kk = 0; kk < D / 32; ++kk) w.qf[kk] = *reinterpret_cast<const V8*>(q + 32 * kk);
  w.run(pages_of<T, D>(a, item.b, head), first, end, a.c);
  float sum[D / 16], top, total;
  w.join(sum, &top, &total);
  const int row = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * (D / 16);
  auto out_row = [=](int i) { return (int64_t)(r.q0 + (uint32_t)i / ratio) * a.heads + head * ratio + (uint32_t)i % ratio; };
  auto place_of = [=](int share) { return ((int64_t)share * a.kv_heads + head) * kFew; };
  const bool sees = sight.any((uint32_t)min(row, nrows - 1) / ratio, first, end);
  if (item.count == 1) {
    typedef T TD __attribute__((ext_vector_type(D / 16)));
    TD v;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) v[j] = (T)(sees ? result(sum[j], sum[j] / total) : 0.f);
    if (row < nrows) *reinterpret_cast<TD*>((T*)a.out + out_row(row) * D + d0) = v;
    return;
  }
  if (row < nrows) {
    const int64_t place = place_of(item.first + item.share) + row;
#pragma unroll
    for (int j = 0; j < D / 16; j += 4)
      hq_store_share(reinterpret_cast<hq_f4v*>(a.po + place * D + d0 + j), hq_f4v{sum[j], sum[j + 1], sum[j + 2], sum[j + 3]});
    if (d0 == 0)
      __hip_atomic_store(reinterpret_cast<unsigned long long*>(a.pm) + place,
                         (unsigned long long)__float_as_uint(total) << 32 | __float_as_uint(share_top(top, sees)), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  // The last share to arrive joins them; of more than 32, every 16 are joined first, by the last of them.
  __shared__ unsigned nth;
  int n = item.count, unit = 1, index = item.share;
  for (;;) {
    const bool all = n <= kJoin;
    const int team = all ? 0 : index / kTeam, members = all ? n : min(kTeam, n - team * kTeam), first_share = item.first + team * kTeam * unit;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    unsigned* const count = a.arrived + (int64_t)((all ? a.few + item.first : first_share) * a.kv_heads + head) * kApart;
    if (threadIdx.x == 0) nth = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (nth != (unsigned)members - 1) return;
    if (threadIdx.x == 0) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    join_here<T, D>(a, sm, nrows, 0, place_of(first_share), (int64_t)unit * a.kv_heads * kFew, members, all, out_row);
    if (all) return;
    index = team;
    n = (n + kTeam - 1) / kTeam;
    unit *= kTeam;
  }
}

__device__ __forceinline__ int64_t many_place(const ChunkArgs& a, int share, int head) {
  return (int64_t)a.few * a.kv_heads * kFew + ((int64_t)share * a.kv_heads + head) * kRows;
}
template <typename T, int D, bool WINDOW, int SIDES>
__device__ __forceinline__ void many_rows(const ChunkArgs& a, char* sm, int* poison, const Item& item, int head) {
  typedef typename Kind<T>::V8 V8;
  const Request& r = item.r;
  const int lane = threadIdx.x & 63, wave = (threadIdx.x >> 6) % kWaves, rows = r.nq * a.ratio;
  const uint32_t ratio = a.ratio;
  const int first_row = ((rows + kRows - 1) / kRows - 1 - item.tile) * kRows, last_row = min(first_row + kRows, rows) - 1;
  const int first_token = (uint32_t)first_row / ratio, last_token = (uint32_t)last_row / ratio;
  const Sight sight(a, r, WINDOW, first_token, last_token);
  int first, end;
  item.keys(uniform(sight.limit(last_token)), &first, &end);
  const int row = first_row + wave * 32 + (lane & 31), mine = min(row, last_row);
  const int token = (uint32_t)mine / ratio, h = head * ratio + (uint32_t)mine % ratio;
  Many<T, D, WINDOW, SIDES> w;
  w.sm = sm;
  w.poison = poison;
  set_up(poison);
  const T* q = (const T*)a.q + (int64_t)(r.q0 + token) * a.qs + (int64_t)h * D + 8 * (lane >> 5);
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) w.qf[kk] = *reinterpret_cast<const V8*>(q + 16 * kk);
  w.lim = min(sight.limit(token), end);
  w.all_see = __builtin_amdgcn_readlane(w.lim, 0);  // a later row sees as much or more
  w.any_sees = first_row + wave * 32 > last_row ? 0 : __builtin_amdgcn_readlane(w.lim, 31);  // a wave without rows works on nothing
  if (WINDOW) {
    w.lo = sight.low(token);
    w.sinks = a.sinks;
    w.lo_most = __builtin_amdgcn_readlane(w.lo, 31);
  }
  PagedTiles<T, D, WINDOW, SIDES> src(pages_of<T, D>(a, item.b, head), end);
  src.skip = sight.skip;
  w.run(src, first, end, uniform(min(sight.limit(first_token), end)), a.c, uniform(sight.low(last_token)));
  if (SIDES == 2) {
    w.meet();
    if (threadIdx.x >= kThreads) return;
  }
  // the row, worked out once more: in the loop there is no register to spare
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
  const int again = first_row + (tid >> 6) * 32 + (tid & 31);
  if (again > last_row) return;
  const int t = (uint32_t)again / ratio;
  const bool sees = sight.any(t, first, end);
  if (item.count == 1) w.put((T*)a.out + ((int64_t)(r.q0 + t) * a.heads + head * ratio + (uint32_t)again % ratio) * D, !sees);
  else w.put_share(a.po, a.pm, many_place(a, item.first + item.share, head) + again - first_row, sees);
}

template <typename T, int D, bool WINDOW, int SIDES>
__global__ __launch_bounds__(SIDES * kThreads, D == 64 && SIDES == 1 ? 3 : 2) void chunk_kernel(ChunkArgs a) {
  extern __shared__ __align__(16) char sm[];
  __shared__ int poison;
  const uint32_t x = blockIdx.x / (uint32_t)a.kv_heads, head = blockIdx.x - x * (uint32_t)a.kv_heads;
  Item item;
  if (!item.find<D, WINDOW>(a, x, blockIdx.x == 0 && threadIdx.x < 64 && a.said)) return;
  if (item.r.nq * a.ratio <= kFew) {
    if (SIDES == 1 || threadIdx.x < kThreads) few_rows<T, D, WINDOW>(a, sm, item, head);  // barriers wait for no wave that has ended
  } else many_rows<T, D, WINDOW, SIDES>(a, sm, &poison, item, head);
}

// The shares of rows of many together, a row a wave (WAVES 1) or a workgroup, from row to row: where nothing was divided, which the host does
// not know, it is the fewer workgroups that matter.
template <typename T, int D, int WAVES, int PRE>
__global__ __launch_bounds__(kThreads) void join_chunk_kernel(ChunkArgs a) {
  const int lane = threadIdx.x & 63;
  const int i = min(lane, a.batch - 1), qb = a.cu_q[i], qe = a.cu_q[i + 1], before = a.said[2 * i], count = a.said[2 * i + 1];
  if (!__ballot(lane < a.batch && count > 1)) return;
  const int64_t rows = (int64_t)a.total_q * a.heads, step = WAVES > 1 ? gridDim.x : (int64_t)gridDim.x * kWaves;
  for (int64_t row = WAVES > 1 ? blockIdx.x : (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6); row < rows; row += step) {
    const int token = uniform((int)(row / a.heads)), h = uniform((int)(row - (int64_t)token * a.heads)), head = h / a.ratio;
    const unsigned long long here = __ballot(lane < a.batch && qb <= token && token < qe);
    if (!here) continue;
    const int b = __ffsll(here) - 1, n = __builtin_amdgcn_readlane(count, b);
    Request r;
    r.get(a, b);
    const int of = r.nq * a.ratio;
    if (of <= kFew || n <= 1) continue;
    const int mine = (token - r.q0) * a.ratio + (h - head * a.ratio), tile = (of + kRows - 1) / kRows - 1 - mine / kRows;
    const int64_t first = __builtin_amdgcn_readlane(before, b) + (int64_t)tile * n;
    if (first < 0 || first + n > a.many) continue;  // bounds that do not ascend
    if (WAVES > 1) __syncthreads();  // the row before has been put together
    join_shares<T, D, WAVES, PRE>(a.po, a.pm, row, many_place(a, (int)first, head) + mine % kRows, a.kv_heads * kRows, n, n, n, n, (T*)a.out);
  }
}

template <typename T, int D, bool WINDOW, int SIDES>
int launch_sides(dim3 workgroups, hipStream_t stream, const ChunkArgs& a) {
  constexpr int lds = std::max(Many<T, D, WINDOW, SIDES>::LDS, Few<T, D>::LDS);
  if (lds > 65536) {
    static const hipError_t attr =
        hipFuncSetAttribute(reinterpret_cast<const void*>(&chunk_kernel<T, D, WINDOW, SIDES>), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (attr != hipSuccess) return (int)attr;
  }
  return hq_launch_as_is(chunk_kernel<T, D, WINDOW, SIDES>, workgroups, dim3(SIDES * kThreads), lds, stream, a);
}

template <typename T, int D, bool WINDOW>
int launch_chunk(ChunkArgs a, int cus, hipStream_t stream) {
  const int64_t cap = (int64_t)a.width << a.page_log, rows = (int64_t)a.total_q * a.ratio, requests = std::min(a.batch, a.total_q);
  const int64_t keys = WINDOW ? std::min(cap, std::min<int64_t>(a.sinks, cap) + a.window + 14 + std::max(kFew, kRows / a.ratio + 2)) : cap;  // of a tile
  const int64_t units = std::max<int64_t>((keys + kUnit - 1) / kUnit, 1), room = share_room(cus, a.kv_heads);
  // Tiles of many rows, at most, each of whose requests has more than kFew of them; how many there are if all but a token a request are theirs; and
  // how many are counted on, all tokens' where one by itself has more than kFew rows (one of 30000 keys, 32 / 1 heads of 128: undivided, as if there
  // were no tile, 552 us, divided 17.3).
  const int64_t tiles = rows / kRows + std::min(requests, rows / (kFew + 1)), slots = rows / kRows + a.batch;
  const int64_t of_chunks = (rows - requests * a.ratio + kRows - 1) / kRows;
  const int64_t likely = a.ratio > kFew ? std::max((rows + kRows - 1) / kRows, requests) : of_chunks;
  // Tiles that a compute unit has one of, at most, and half of them has, or with up to 1024 keys a quarter: undivided and of twice the waves (SIDES
  // in attend.h; 1024 tokens behind 3500, 32 / 8 heads of 128, 93 -> 77 us, 700 86 -> 69, of 64 84 -> 59 and 78 -> 52, behind nothing 28.6 -> 26.5
  // and 23.1 -> 18.1; up to 256 keys 8.6 and 9.6; 640 tokens, which could be divided in three, behind 1000 40 -> 33, 3500 68 and 68, 16000 212 ->
  // 240; 512 behind 500 29.3 -> 23.5, and 256 behind 700 would go 20.5 -> 23.2).  Not beside many requests, which then find no room next to the
  // tiles: 8 of one token beside 900 106 -> 102, 16 of them 111 -> 117, 30 of up to 4000 117 -> 133 (3 of 16000 beside 1000 tokens go 63 -> 77,
  // which the host cannot tell).
  const bool alone = tiles && units > 2 && (units <= 8 ? 4 : 2) * of_chunks * a.kv_heads > cus && ((rows - requests) / kRows + requests) * a.kv_heads <= cus &&
                     4 * requests * a.kv_heads <= cus;
  a.cus = cus;
  a.room = (int)room;
  bool divide = units > kShort, many_divided;
  size_t floats = 0, counters = 0;
  int64_t few, many, places;
  for (;;) {
    a.ns = 0;
    many_divided = false;
    if (a.batch > 64) {
      a.ns = (int)(divide ? std::max<int64_t>(1, std::min(room / slots, units)) : 1);
      divide = a.ns > 1;
      few = slots * a.ns;
      many = 0;
    } else {
      few = divide ? std::min(std::max(room, requests), requests * units) : requests;
      many = tiles;
      // (Where the likely ones are too many to be divided, or their keys too few, nothing asks for room for shares and a launch that joins them.)
      if (divide && units > kShortOfAll && !alone && tiles && tiles < 2 * room && likely && 3 * likely * a.kv_heads <= 2 * cus) {  // more tiles than that fill the device
        many = tiles + std::min(room, tiles * units);  // some as they are, beside shares that fill the room
        many_divided = true;
      }
    }
    if (!divide) break;
    places = (few * kFew + (many_divided ? many * kRows : 0)) * a.kv_heads;
    floats = places * (D + 2) + 2 * a.batch;
    counters = 2 * few * a.kv_heads * kApart;
    // While the stream is captured and has no room for shares: undivided.  Longer, and no error.
    if (!hq_workspace_out_of_reach(stream, floats, counters)) break;
    divide = false;
  }
  // What is divided shares the room, beside what is not.
  const int64_t grid = a.ns ? few : many_divided ? tiles + std::max(room, requests) : tiles + few;
  if (grid * a.kv_heads > UINT32_MAX / kThreads) return HQ_ERR_TOO_LARGE;  // threads are numbered in 32 bits
  a.few = (int)few;
  a.many = (int)many;
  if (divide) {
    HqWorkspace ws;
    const int rc = hq_get_workspace(stream, floats, counters, &ws);
    if (rc != HQ_OK) return rc;
    a.arrived = ws.counters;
    a.po = ws.partial;
    a.pm = a.po + places * D;
    if (many_divided) a.said = reinterpret_cast<int*>(a.pm + 2 * places);
  }
  const dim3 workgroups((unsigned)(grid * a.kv_heads));
  const int rc = alone ? launch_sides<T, D, WINDOW, 2>(workgroups, stream, a) : launch_sides<T, D, WINDOW, 1>(workgroups, stream, a);
  if (rc != HQ_OK || !a.said) return rc;
  const int64_t all = std::min((int64_t)a.total_q * a.heads, likely * kRows * a.kv_heads);
  if (std::min(room / likely, units / 2) <= 2 * kSharesOfAWave)
    return hq_launch_as_is(join_chunk_kernel<T, D, 1, 0>, dim3((unsigned)((all + kWaves - 1) / kWaves)), dim3(kThreads), 0, stream, a);
  return hq_launch_as_is(join_chunk_kernel<T, D, kWaves, 8>, dim3((unsigned)all), dim3(kThreads), 0, stream, a);
}
}  // namespace

extern "C" int hq_chunk_attention(const void* q, const void* k_pages, const void* v_pages, void* out, int dtype, const int32_t* table,
                                  const int32_t* lengths, const int32_t* cu_q, int batch, int64_t total_q, int table_width, int num_pages,
                                  int page_size, int heads, int kv_heads, int head_dim, int64_t q_stride, float scale, int window, int sinks,
                                  void* stream) {
  if (batch < 0 || total_q < 0 || table_width < 0 || num_pages < 0 || window < 0 || sinks < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads)
    return HQ_ERR_BAD_SHAPE;
  if (page_size < 8 || page_size > 1024 || (page_size & (page_size - 1))) return HQ_ERR_BAD_SHAPE;
  if (head_dim != 64 && head_dim != 128) return HQ_ERR_BAD_SHAPE;
  if (dtype != HQ_DTYPE_F16 && dtype != HQ_DTYPE_BF16) return HQ_ERR_BAD_ENUM;
  if (bad_scale(scale)) return HQ_ERR_BAD_SHAPE;
  if (batch == 0 || total_q == 0) return HQ_OK;
  if (!q || !out || !lengths || !cu_q || (table_width && !table) || (table_width && num_pages && (!k_pages || !v_pages))) return HQ_ERR_NULL_POINTER;
  if (q_stride < (int64_t)heads * head_dim) return HQ_ERR_BAD_SHAPE;
  if (misaligned(q, q_stride) || (((uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)out) & 15) ||
      (((uintptr_t)table | (uintptr_t)lengths | (uintptr_t)cu_q) & 3))
    return HQ_ERR_MISALIGNED;
  const int ratio = heads / kv_heads;
  if ((int64_t)table_width * page_size > kMostKeys || total_q > INT_MAX || total_q * ratio > INT_MAX - kRows || total_q * ratio / kRows + batch > INT_MAX / 2 ||
      (int64_t)kv_heads * head_dim * 2 * page_size > UINT32_MAX)  // bytes of a page
    return HQ_ERR_TOO_LARGE;
  const HqDevice* dev = nullptr;
  const int rc = hq_current_device(&dev);
  if (rc != HQ_OK) return rc;
  ChunkArgs a{};
  a.q = q;
  a.k = k_pages;
  a.v = v_pages;
  a.out = out;
  a.table = table;
  a.lengths = lengths;
  a.cu_q = cu_q;
  a.qs = q_stride;
  a.batch = batch;
  a.total_q = (int)total_q;
  a.width = table_width;
  a.pages = num_pages;
  a.page_log = __builtin_ctz(page_size);
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.ratio = ratio;
  a.window = window;
  a.sinks = sinks;
  a.c = exponent_scale(scale);
  const hipStream_t s = (hipStream_t)stream;
  return by_type(dtype, head_dim, [&](auto f) {
    typedef decltype(f) F;
    if (window && window < (int64_t)table_width * page_size) return launch_chunk<typename F::T, F::D, true>(a, dev->cus, s);
    return launch_chunk<typename F::T, F::D, false>(a, dev->cus, s);
  });
}
