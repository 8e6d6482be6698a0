// Attention: what its kernels over packed prompts and over a paged cache have in common.
//
// For a query row q: out = sum_j p_j v_j / sum_j p_j, p_j = 2^(c q.k_j - m), c = scale * log2(e), in one pass over the keys with an m that
// follows the row's maximum; a larger one scales what has been summed so far.
//
// Two ways through the keys.  Many rows (Many): a tile of 64 keys in LDS serves 128 rows, 32 a wave.  Few (Few): 16 rows at most, each
// wave goes through keys of its own, as what bounds it is their way from memory, and the waves' sums come together at the end.
//
// Rows: the R = heads / kv_heads query heads of a key / value head and the tokens (or requests) are one list of rows
// (token, head of the group), so that a tile of keys in LDS serves all of them.  The scores are computed
// transposed, S^T = K Q^T: the matrix core leaves a row's scores in one lane and its partner 32 lanes on, so maximum and sum are
// sums within a lane and one exchange, and the same registers are, rounded, the operand of O^T = V^T P^T without another move: the
// order of the keys in that sum is free, and the transposing LDS read fetches V's rows in the order in which S^T left them.
#pragma once

#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>
#include <type_traits>

#include "hq_internal.h"

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char lds_char;

// The weights on their way into the product with the values, in 16 bits: 2^(c s - m), where m is not the row's maximum itself but kLift octaves
// below it, and stays until the maximum is kMost octaves above.  bf16 has no need of a lift; fp16, whose normal numbers end at 2^-14, has its
// weights where its range ends.  Each is rounded, to the nearest, by 2^-11 (bf16: 2^-8) of itself at most, as much as the result's own rounding;
// fp16's below 2^-25 of the row's largest by 2^-36 of that largest at most (with the largest at 1 a key of 2^-18.5 was 0.6 % off, and
// one of 2^-25 gone).
template <typename T>
struct Kind;
typedef float f32x4 __attribute__((ext_vector_type(4)));
template <>
struct Kind<__bf16> {
  typedef bf16x8 V8;
  static constexpr uint32_t kExp = 0x7f807f80u, kStep = 0x00800080u, kOne = 0x3f803f80u;
  static constexpr float kLift = 0.f, kMost = 8.f;
  static __device__ __forceinline__ f32x16 mfma(V8 a, V8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ f32x4 mfma(V8 a, V8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Kind<_Float16> {
  typedef f16x8 V8;
  static constexpr uint32_t kExp = 0x7c007c00u, kStep = 0x04000400u, kOne = 0x3c003c00u;
  static constexpr float kLift = 11.f, kMost = 15.f;
  static __device__ __forceinline__ f32x16 mfma(V8 a, V8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ f32x4 mfma(V8 a, V8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};

// The larger of a lane's value and its partner's, 32 lanes on.
__device__ __forceinline__ float pair_max(float v) {
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float pair_sum(float v) {
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}
// The same over the four lanes of a row of Few, 16 lanes apart.
__device__ __forceinline__ float quarters_max(float v) {
  const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return pair_max(fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1])));
}
__device__ __forceinline__ float quarters_sum(float v) {
  const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return pair_sum(__uint_as_float(s[0]) + __uint_as_float(s[1]));
}
__device__ __forceinline__ float finite_or_zero(float m) { return m == -INFINITY ? 0.f : m; }
// m of a row whose maximum is `top` now (differences: beyond 2^24 numbers are further apart than the lift).
template <typename T>
__device__ __forceinline__ bool outgrown(float top, float m) { return top - m > Kind<T>::kMost; }
template <typename T>
__device__ __forceinline__ float lifted(float top) {
  const float m = top - Kind<T>::kLift;
  return outgrown<T>(top, m) ? top : m;
}
// Whether m is so far from 0 that c s rounded, as a maximum is, and c s in an exponent, where it is not, may differ by octaves.
__device__ __forceinline__ bool far(float m) { return fabsf(finite_or_zero(m)) > 0x1p20f; }
// Scores become the exponents of their weights, of a row far from 0 (the product rounded) or not, whose bits are then those that they would
// be without.  Kept behind its branch, one register after the other: in front of it, where the compiler moves it, it costs 17 registers too
// many (24 sequences of up to 901 tokens, 32 heads of 64: 74.6 -> 95.7 us).
template <typename S>
__device__ __forceinline__ void exponents(S& s, int n, float c, float m) {
  float before = far(m) ? c : 1.f, then = far(m) ? 1.f : c, ms = finite_or_zero(m);
  asm volatile("" : "+v"(before), "+v"(then), "+v"(ms));
#pragma unroll
  for (int i = 0; i < n; ++i) {
    float x = fmaf(s[i] * before, then, -ms);
    asm volatile("" : "+v"(x));
    s[i] = x;
  }
}
// A result of a sum o of values and what it is to be scaled by.  A sum that is not finite gives NaN: whether an infinite value comes out
// of a sum as an infinity depends on whether its weight, or that of its share, has become 0 (the tiles that not all rows see mark NaN).
__device__ __forceinline__ float result(float o, float scaled) { return fmaf(o, 0.f, scaled); }
// A share's maximum as those who join the shares read it: -infinity means that the row sees no key of the share, which has no sums then; a
// row that has that of all its shares gives zeros.  One that sees keys, all of whose scores are -infinity or NaN, says the lowest number.
__device__ __forceinline__ float share_top(float m, bool sees) { return sees ? fmaxf(m, -FLT_MAX) : -INFINITY; }

// A value that is the same in all lanes, in scalar registers.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
template <typename P>
__device__ __forceinline__ const P* uniform(const P* p) {
  const uint64_t x = (uint64_t)p;
  return (const P*)((uint64_t)(uint32_t)uniform((int)(x >> 32)) << 32 | (uint32_t)uniform((int)x));
}

constexpr int kThreads = 256, kWaves = 4;

__device__ __forceinline__ int wave_min(int v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v = min(v, __shfl_xor(v, d));
  return v;
}

// ---- keys and values in LDS --------------------------------------------------------------------------------------------
// A row's 16-byte pieces are stored in an order that depends on the row, so that the lanes of a read pass meet different banks (0
// conflicts counted): the keys' by all bits of the row, which 16 lanes read piece by piece, the values' by the bits of the four or eight
// rows that transposing reads take together, 64 or 32 bytes of each.
template <int D>
__device__ __forceinline__ int k_piece(int row, int ch) { return D == 128 ? ch ^ (row & 15) : ch ^ ((row >> 1) & 7); }
template <int D>
__device__ __forceinline__ int v_piece(int row, int ch) {
  return (D == 128 ? ch ^ ((row & 3) << 2) : ch ^ (((row >> 1) & 1) << 2)) ^ (((row >> 2) & 1) << 1);
}

// One instruction brings 1 KB from memory into LDS past the registers, the lanes' pieces one behind the other, so it is the lane's
// address that follows the order of the pieces.  (The compiler does not see that it writes LDS; the waits are explicit.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // that m0 is the compiler's own is why it is listed
__device__ __forceinline__ void to_lds(uint32_t lds, const void* from, uint32_t off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(from) : "memory", "m0");
}
__device__ __forceinline__ void to_lds(uint32_t lds, const void* from) {  // a lane's own address
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(from) : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ uint32_t lds_address(const char* p) { return (uint32_t)(uintptr_t)(lds_char*)p; }

// Keys that no row of a workgroup sees, between the first ones of its sequence and its windows, are not gone through: key u of those
// that are is key u of the sequence below `from`, and `gap` more from there on.  Both multiples of 8: eight keys of a page stay eight.
struct Skip {
  int from = 0, gap = 0;
  __device__ __forceinline__ int key(int u) const { return u + (u >= from ? gap : 0); }
  __device__ __forceinline__ bool within(int base, int n) const { return base < from && base + n > from; }
};
// A row at place p of its sequence sees the first `sinks` keys and `window` up to its own: those from here on.  (A negative place sees none.)
__device__ __forceinline__ int window_of(int place, int window) { return max(max(place, 0) - window + 1, 0); }
// What rows at places first ... last leave out.
__device__ __forceinline__ Skip skip_of(int first, int last, int window, int sinks) {
  const int s8 = (min(sinks, max(last + 1, 0)) + 7) & ~7, gap = (window_of(first, window) & ~7) - s8;
  Skip s;
  if (gap > 0) {
    s.from = s8;
    s.gap = gap;
  }
  return s;
}
// The first n of a block's 32 keys, a bit each.
__device__ __forceinline__ int first_bits(int n) { return n >= 32 ? -1 : n <= 0 ? 0 : (int)((1u << n) - 1); }

// The tiles of one sequence's keys, one head, for the four waves of Many.  Rows behind the last one repeat it.
template <typename T, int D, bool WINDOW = false>
struct PackedTiles {
  static constexpr int CH = D / 8, NL = 64 * CH / kThreads;  // pieces of a row; instructions of a wave for the keys of a tile
  const T *k, *v;
  int64_t ks, vs;
  int n, first;
  uint32_t koff[NL], voff[NL];
  Skip skip;  // WINDOW
  // (Of a thread number that the compiler cannot see through where it happens inside the loop, once: nothing of it is then kept in
  // registers all along.)
  template <typename F>
  static __device__ __forceinline__ void offsets(uint32_t (&off)[NL], int stride, int rows, F piece) {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int row = ((tid >> 6) * NL + i) * (64 / CH) + (tid & 63) / CH;
      off[i] = __umul24(min(row, rows - 1), 2 * stride) + piece(row, tid % CH) * 16;
    }
  }
  static __device__ __forceinline__ void load(const T* from, const uint32_t (&off)[NL], char* to) {
    from = uniform(from);
    const uint32_t lds = uniform((int)(lds_address(to) + (threadIdx.x >> 6) * (NL * 1024)));
#pragma unroll
    for (int i = 0; i < NL; ++i) to_lds(lds + i * 1024, from, off[i]);
  }
  __device__ __forceinline__ void start(int f) {
    first = f;
    offsets(koff, (int)ks, n - first, k_piece<D>);
    offsets(voff, (int)vs, n - first, v_piece<D>);
  }
  __device__ __forceinline__ void advance(int) {}
  // Keys of the first two tiles, if there are two, and values of the first one, all at once.
  __device__ __forceinline__ void begin(char* k0, char* k1, char* v0, bool two) {
    load_k(0, k0);
    load_v(0, v0);
    if (two) load_k(1, k1);
  }
  __device__ __forceinline__ void then(char*, bool) const {}
  // A tile on both sides of what is left out: every lane by an address of its own.
  template <typename F>
  __device__ __forceinline__ void load_across(const T* from, int64_t stride, int base, char* to, F piece) const {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const uint32_t lds = uniform((int)(lds_address(to) + (threadIdx.x >> 6) * (NL * 1024)));
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int row = ((tid >> 6) * NL + i) * (64 / CH) + (tid & 63) / CH;
      to_lds(lds + i * 1024, from + skip.key(min(base + row, n - 1)) * stride + piece(row, tid % CH) * 8);
    }
  }
  __device__ __forceinline__ void load_k(int t, char* to) {
    const int base = first + t * 64;
    if (WINDOW && skip.within(base, 64)) return load_across(k, ks, base, to, k_piece<D>);
    if (base + 64 > n) offsets(koff, (int)ks, n - base, k_piece<D>);
    load(k + (WINDOW ? skip.key(base) : base) * ks, koff, to);
  }
  __device__ __forceinline__ void load_v(int t, char* to) {
    const int base = first + t * 64;
    if (WINDOW && skip.within(base, 64)) return load_across(v, vs, base, to, v_piece<D>);
    if (base + 64 > n) offsets(voff, (int)vs, n - base, v_piece<D>);
    load(v + (WINDOW ? skip.key(base) : base) * vs, voff, to);
  }
};

// The pages of one request, one head.  Eight tokens from a multiple of eight on are in one page.
template <typename T, int D>
struct Pages {
  const char *k, *v;    // this head's rows in page 0
  const int* table;     // the request's row
  uint32_t page_bytes;  // of all heads
  int page_log, pages;
  __device__ __forceinline__ Pages(const T* k0, const T* v0, const int* row, int head, int kv_heads, int log, int n)
      : k((const char*)(k0 + ((int64_t)head << log) * D)), v((const char*)(v0 + ((int64_t)head << log) * D)), table(row),
        page_bytes((uint32_t)kv_heads * (D * 2) << log), page_log(log), pages(n) {}
  // The table's entry, as it is: looking at it where it is loaded would be waiting for it, and for all that is asked for in between.
  __device__ __forceinline__ int id(int key) const { return table[key >> page_log]; }
  __device__ __forceinline__ bool none(int id) const { return (unsigned)id >= (unsigned)pages; }  // no page: to be read as zeros
  __device__ __forceinline__ uint64_t at(int page, int key) const {
    return (uint64_t)(uint32_t)page * page_bytes + (uint32_t)(key & ((1 << page_log) - 1)) * (D * 2);
  }
};
__device__ __forceinline__ void zero_lds(char* to) {  // what one to_lds() would write
  reinterpret_cast<hq_u4v*>(to)[threadIdx.x & 63] = hq_u4v{0, 0, 0, 0};
}

// Where the rows of a wave's instructions are: a lane works out an instruction's place, which then costs two moves to scalar registers
// and an addition (worked out by the scalar unit, load after load, 30 instructions each: 0.6 us a tile with nothing under it).
struct Places {
  uint32_t lo, hi;           // of a lane's instruction
  unsigned long long none;   // instructions whose rows are in no page
  template <typename T, int D>
  __device__ __forceinline__ void set(const Pages<T, D>& p, int id, int key) {
    const uint64_t x = p.at(id, key);
    lo = (uint32_t)x;
    hi = (uint32_t)(x >> 32);
    none = __ballot(p.none(id));
  }
  __device__ __forceinline__ const char* of(const char* pool, int lane) const {
    return pool + ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)hi, lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)lo, lane));
  }
  // Instructions first ... first + N - 1, into `to` and on; off: the lane's offset in the first one, from which the others' differ in what
  // k_piece() or v_piece() make of the rows between.  Whether all of them were needed.
  template <int D, bool VALUES, int N>
  __device__ __forceinline__ bool load(const char* pool, int first, uint32_t off0, char* to) const {
    auto off = [=](int i) { return off0 ^ (uint32_t)(VALUES ? (D == 128 ? (i & 1) * 32 : 0) : D == 128 ? (i & 3) * 64 : (i & 1) * 64); };
    const uint32_t lds = uniform((int)lds_address(to));
    if (!(none >> first & ((1ull << N) - 1))) {
#pragma unroll
      for (int i = 0; i < N; ++i) to_lds(lds + i * 1024, of(pool, first + i), off(i));
      return true;
    }
    for (int i = 0; i < N; ++i) {
      if (none >> (first + i) & 1) zero_lds(to + i * 1024);
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (j == i && !(none >> (first + i) & 1)) to_lds(lds + j * 1024, of(pool, first + j), off(j));
    }
    return false;
  }
};

// The same tiles of pages.  Rows behind the last one are whatever its page holds.  AT_ONCE (heads of 128): keys of the first two tiles and values of
// the first are asked for together, behind one trip for their pages, which long tiles gain from (2048 tokens behind 30000 1007 -> 985 us); or one
// behind the other, with which a share of a few tiles has its first keys sooner (32 requests behind 8192 common keys, four tiles a share, 24.2 us, at
// once 25.1).
template <typename T, int D, bool WINDOW = false, int SIDES = 1, bool AT_ONCE = true>
struct PagedTiles {
  static constexpr int CH = D / 8, NL = 64 * CH / kThreads, RG = 64 / CH;  // RG: rows of an instruction, all in one page
  Pages<T, D> p;
  int n, first;
  int ids;          // pages of the wave's instructions' rows, one a lane, of the tile to come
  Places next, now; // of the tile whose keys are loaded next, and (heads of 128, whose keys are a tile ahead) of its predecessor
  uint32_t koff, voff;
  Skip skip;  // WINDOW
  __device__ __forceinline__ int place(int u) const { return WINDOW ? skip.key(u) : u; }
  __device__ PagedTiles(const Pages<T, D>& pages, int end) : p(pages), n(end) {}
  __device__ __forceinline__ int key(int t) const { return first + t * (64 * SIDES) + (int)((threadIdx.x >> 6) * NL + threadIdx.x % NL) * RG; }
  __device__ __forceinline__ void start(int f) {
    first = f;
    const int lane = threadIdx.x & 63, row = lane / CH;  // of a multiple of 16
    koff = row * D * 2 + k_piece<D>(row, lane % CH) * 16;
    voff = row * D * 2 + v_piece<D>(row, lane % CH) * 16;
    ids = p.id(place(min(key(0), n - 1)));
    if (D == 128 && AT_ONCE) {  // the first two tiles' pages by one trip to memory
      const int then = p.id(place(min(key(1), n - 1)));
      now.set(p, ids, place(key(0)));
      next.set(p, then, place(key(1)));
      ids = p.id(place(min(key(2), n - 1)));
    }
  }
  __device__ __forceinline__ void begin(char* k0, char* k1, char* v0, bool two) {
    if (!AT_ONCE) {
      advance(0);
      load_k(0, k0);
      advance(1);
      return load_v(0, v0);
    }
    now.template load<D, false, NL>(p.k, 0, koff, k0 + (threadIdx.x >> 6) * (NL * 1024));
    load_v(0, v0);
    if (two) load_k(1, k1);
  }
  // With the first tile there.
  __device__ __forceinline__ void then(char* k1, bool two) const {
    if (!AT_ONCE && two) load_k(1, k1);
  }
  // Before the first load of tile t: its pages are there, those of the tile behind it are asked for.
  __device__ __forceinline__ void advance(int t) {
    now = next;
    next.set(p, ids, place(key(t)));
    ids = p.id(place(min(key(t + 1), n - 1)));
  }
  __device__ __forceinline__ void load_k(int, char* to) const { next.template load<D, false, NL>(p.k, 0, koff, to + (threadIdx.x >> 6) * (NL * 1024)); }
  __device__ __forceinline__ void load_v(int, char* to) const {
    (D == 128 ? now : next).template load<D, true, NL>(p.v, 0, voff, to + (threadIdx.x >> 6) * (NL * 1024));
  }
};

// ---- many rows -----------------------------------------------------------------------------------------------------------
// 128 rows of a workgroup, 32 a wave.  WINDOW: a row sees its first keys, and those from a key of its own on.  SIDES 2: twice as many waves and
// keys of a tile, of which four go through the first half and four through the other, and their sums meet at the end: one workgroup then
// keeps a compute unit as busy as two do.
template <typename T, int D, bool WINDOW = false, int SIDES = 1>
struct Many {
  typedef typename Kind<T>::V8 V8;
  static constexpr int NB = 2, TILE = 64 * SIDES;   // a wave's blocks of 32 keys, keys of a tile
  static constexpr int THREADS = SIDES * kThreads, CH = D / 8, NL = TILE * CH / THREADS;
  static constexpr int HALF = TILE * D * 2, LDS = 4 * HALF;  // keys or values of a tile; two of each
  static constexpr bool K_AHEAD = D == 128;         // see run()

  char* sm;
  int* poison;  // in LDS: the tile whose values hold something that is not finite
  V8 qf[D / 16];
  f32x16 o[D / 32];
  float m = -INFINITY, l = 0.f;
  bool slow = false;      // there is a row in the wave whose m is far from 0
  int lim;                // keys below this are seen by the lane's row
  int all_see, any_sees;  // below the first by all rows of the wave, below the second by one of them
  // WINDOW: of those, the row sees the ones below `sinks` and those from `lo` on, `lo_most` at most among the wave's rows
  int lo = 0, lo_most = 0, sinks = 0;

  // The first of the wave's keys of a tile.
  static __device__ __forceinline__ int side() { return SIDES == 1 ? 0 : (int)(threadIdx.x / kThreads) * 64; }
  // Whether a tile holds keys that not every row of the wave sees.
  __device__ __forceinline__ bool partial(int base) const {
    return base + TILE > all_see || (WINDOW && base < lo_most && base + TILE > sinks);
  }

  // In a tile that not every row sees whole, a value that is not finite would reach the rows that do not see it (0 times infinity): it
  // becomes zero, and the bits returned say which values were.
  static __device__ __forceinline__ void clean(char* values, uint32_t& bad) {
    hq_u4v* vs = reinterpret_cast<hq_u4v*>(values) + threadIdx.x;
    hq_u4v v[NL];
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < NL; ++i) v[i] = vs[i * THREADS];
#pragma unroll
    for (int i = 0; i < NL; ++i)
#pragma unroll
      for (int w = 0; w < 4; ++w) any |= (v[i][w] & Kind<T>::kExp) + Kind<T>::kStep;
    bad = 0;
    if (!(any & 0x80008000u)) return;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t e = ((v[i][w] & Kind<T>::kExp) + Kind<T>::kStep) & 0x80008000u;
        bad |= ((e >> 15 & 1u) | (e >> 30 & 2u)) << (8 * i + 2 * w);
        v[i][w] &= ~((e >> 15) * 0xffffu);
      }
      vs[i * THREADS] = v[i];
    }
  }

  // The same places again, one for each value that was not finite and zero for the others.
  static __device__ __forceinline__ void store_bad(char* values, uint32_t bad) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      hq_u4v w;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t b = bad >> (8 * i + 2 * j);
        w[j] = (b & 1 ? Kind<T>::kOne & 0xffffu : 0u) | (b & 2 ? Kind<T>::kOne & 0xffff0000u : 0u);
      }
      reinterpret_cast<hq_u4v*>(values)[threadIdx.x + i * THREADS] = w;
    }
  }

  // V^T of 32 elements of the head (block d) and 16 keys (block b, half t) as the matrix core takes it: the keys in the order in which
  // the scores' registers hold them.
  static __device__ __forceinline__ V8 v_operand(const char* values, int b, int t, int d) {
    const int lane = threadIdx.x & 63;
    const int row = side() + 32 * b + 16 * t + 4 * (lane >> 5) + ((lane >> 2) & 3);
    const int ch = 4 * d + 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
    lds_char* vs = (lds_char*)values + (lane & 1) * 8;
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    union {
      s16x4 h[2];
      V8 v;
    } u;
    u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(vs + row * D * 2 + v_piece<D>(row, ch) * 16));
    u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(vs + (row + 8) * D * 2 + v_piece<D>(row + 8, ch) * 16));
    return u.v;
  }

  // The wave's part of a tile, step by step.  Scores of its rows and the tile's keys:
  __device__ __forceinline__ void scores(f32x16 (&s)[NB], const char* keys) const {
    const int lane = threadIdx.x & 63, half = lane >> 5;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[b][r] = 0.f;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const int row = side() + 32 * b + (lane & 31);
        const V8 a = *reinterpret_cast<const V8*>(keys + row * D * 2 + k_piece<D>(row, 2 * kk + half) * 16);
        s[b] = Kind<T>::mfma(a, qf[kk], s[b]);
      }
    }
  }
  // Which of the lane's registers are keys that the row sees; at: the wave's first key of the tile, 4 more in the upper lanes.
  __device__ __forceinline__ void mask(f32x16 (&s)[NB], int at) const {
    const int left = lim - at;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      // bit i: key i of the block is seen; a bit field of a sign and a bitwise select cost two instructions a score and no scalar register
      const int n = left - 32 * b;
      int seen = first_bits(n);
      if (WINDOW) seen &= ~first_bits(lo - at - 32 * b) | first_bits(sinks - at - 32 * b);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const uint32_t keep = (uint32_t)__builtin_amdgcn_sbfe(seen, 8 * (r / 4) + r % 4, 1);
        s[b][r] = __uint_as_float((__float_as_uint(s[b][r]) & keep) | (~keep & 0xff800000u));
      }
    }
  }
  static __device__ __forceinline__ float top_of(const f32x16 (&s)[NB]) {
    float top = s[0][0];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[b][r]);
    return pair_max(top);
  }
  // Before a tile's weights, its largest scores known.  Whether the scores are exponents now: in a wave with a row far from 0.
  __device__ __forceinline__ bool raise(f32x16 (&s)[NB], float top, float c) {
    scale_sums(top * c);
    if (__builtin_expect(slow, 0))
#pragma unroll
      for (int b = 0; b < NB; ++b) exponents(s[b], 16, c, m);
    return slow;
  }
  // m stays where the maximum has grown by some octaves only: neither fp32 sums nor the 16-bit weights mind larger weights, and the sums
  // need no scaling.  The scaling of 64 registers a tile was a fifth of the vector instructions.
  __device__ __forceinline__ void scale_sums(float top) {
    if (!__builtin_amdgcn_ballot_w64(outgrown<T>(top, m))) return;
    const float mn = outgrown<T>(top, m) ? lifted<T>(top) : m;  // each row by its own scores: its bits do not depend on its neighbours
    const float f = mn == m ? 1.f : __builtin_amdgcn_exp2f(m - mn);
    m = mn;
    slow = __builtin_amdgcn_ballot_w64(far(m)) != 0;
    l *= f;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] *= f;
  }
  // The weights 2^(c s - ms).
  __device__ __forceinline__ void weights(V8 (&p)[NB][2], const f32x16 (&s)[NB], float c, float ms) {
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float e = __builtin_amdgcn_exp2f(fmaf(s[b][8 * t + i], c, -ms));
          sum[i & 1] += e;
          p[b][t][i] = (T)e;
        }
    l += sum[0] + sum[1];
  }
  __device__ __forceinline__ void values(const V8 (&p)[NB][2], const char* values) {
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int t = 0; t < 2; ++t) o[d] = Kind<T>::mfma(v_operand(values, b, t, d), p[b][t], o[d]);
  }
  // scores() of the next tile and weights() of this one, an instruction of the matrix core and its share of the others in turn: left
  // alone, the compiler moves the reads of all operands to the front and runs out of registers.
  __device__ __forceinline__ void scores_and_weights(f32x16 (&n)[NB], const char* keys, V8 (&p)[NB][2], const f32x16 (&s)[NB], float c, float ms) {
    const int lane = threadIdx.x & 63, half = lane >> 5;
    constexpr int STEPS = NB * D / 16, EACH = NB * 16 / STEPS, AHEAD = 4;
    auto operand = [&](int j) {
      const int row = side() + 32 * (j / (D / 16)) + (lane & 31);
      return *reinterpret_cast<const V8*>(keys + row * D * 2 + k_piece<D>(row, 2 * (j % (D / 16)) + half) * 16);
    };
    float sum[2] = {0.f, 0.f};
    V8 a[AHEAD];
    hq_u4v w[NB][2];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) a[j] = operand(j);
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) n[b][r] = 0.f;
#pragma unroll
    for (int j = 0; j < STEPS; ++j) {
      n[j / (D / 16)] = Kind<T>::mfma(a[j % AHEAD], qf[j % (D / 16)], n[j / (D / 16)]);
      if (j + AHEAD < STEPS) a[j % AHEAD] = operand(j + AHEAD);
#pragma unroll
      for (int i = j * EACH; i < (j + 1) * EACH; i += 2) {
        const float e0 = __builtin_amdgcn_exp2f(fmaf(s[i / 16][i % 16], c, -ms)), e1 = __builtin_amdgcn_exp2f(fmaf(s[i / 16][i % 16 + 1], c, -ms));
        sum[0] += e0;
        sum[1] += e1;
        typedef T T2 __attribute__((ext_vector_type(2)));
        uint32_t two = __builtin_bit_cast(uint32_t, T2{(T)e0, (T)e1});
        asm volatile("" : "+v"(two), "+v"(sum[0]), "+v"(sum[1]));  // here and now
        w[i / 16][i / 8 % 2][i % 8 / 2] = two;
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int h = 0; h < 2; ++h) p[b][h] = __builtin_bit_cast(V8, w[b][h]);
    l += sum[0] + sum[1];
  }
  // values() of this tile, and the maximum of the next one's scores.
  __device__ __forceinline__ float values_and_top(const V8 (&p)[NB][2], const char* vs, const f32x16 (&n)[NB]) {
    constexpr int STEPS = D / 32 * NB * 2, EACH = NB * 16 / STEPS, AHEAD = 4;
    auto operand = [&](int j) { return v_operand(vs, j / 2 % NB, j % 2, j / (2 * NB)); };
    V8 a[AHEAD];
    float top = n[0][0];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) a[j] = operand(j);
#pragma unroll
    for (int j = 0; j < STEPS; ++j) {
      o[j / (2 * NB)] = Kind<T>::mfma(a[j % AHEAD], p[j / 2 % NB][j % 2], o[j / (2 * NB)]);
      if (j + AHEAD < STEPS) a[j % AHEAD] = operand(j + AHEAD);
#pragma unroll
      for (int i = j * EACH; i < (j + 1) * EACH; ++i) top = fmaxf(top, n[i / 16][i % 16]);
      asm volatile("" : "+v"(top));
      __builtin_amdgcn_sched_barrier(0);
    }
    return pair_max(top);
  }
  // Rows that see a value that is not finite.
  __device__ __forceinline__ void spoil(char* values, int at, uint32_t bad) {
    const int left = lim - at, low = lo - at, always = sinks - at;
    __syncthreads();
    store_bad(values, bad);
    __syncthreads();
#pragma unroll
    for (int d = 0; d < D / 32; ++d) {
      f32x16 n;
#pragma unroll
      for (int r = 0; r < 16; ++r) n[r] = 0.f;
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          V8 seen;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int key = 32 * b + 16 * t + 8 * (i / 4) + i % 4;
            seen[i] = key < left && (!WINDOW || key >= low || key < always) ? (T)1.f : (T)0.f;
          }
          n = Kind<T>::mfma(v_operand(values, b, t, d), seen, n);
        }
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] = n[r] > 0.f ? NAN : o[d][r];
    }
  }
  __device__ __forceinline__ bool spoiled(int tileno) const { return *(volatile __attribute__((address_space(3))) int*)poison == tileno; }
  __device__ __forceinline__ void note(uint32_t bad, int tileno) {
    if (bad) *poison = tileno;
  }

  // The row's sums as one of several shares; sees: one of the share's keys at least.
  __device__ __forceinline__ void put_share(float* po, float* pm, int64_t at, bool sees) const {
    const int half = (threadIdx.x >> 5) & 1;
    if (sees)
#pragma unroll
      for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<hq_f4v*>(po + at * D + 32 * d + 8 * g + 4 * half) = hq_f4v{o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
    if (half == 0) *reinterpret_cast<float2*>(pm + 2 * at) = float2{share_top(m, sees), l};
  }

  // Keys [first, end) of src; whole: keys below it are seen by every row of the workgroup (WINDOW: of those from lo_whole on).  A tile is on its way from memory while the one
  // before it is worked on, with one barrier a tile.  Heads of 128: the scores of the next tile are in the matrix core while the vector
  // unit makes this one's weights of its own, and the next scores' maximum is taken under this tile's product with the values; the
  // keys so run a tile ahead.  Heads of 64, where the vector unit is the busier of the two and the registers saved are two waves more: one step after
  // the other (16384 tokens, heads of 128: 2186 us one after the other, 2116 so; 8192 tokens, heads of 64: 359 and 376).
  template <typename SRC>
  __device__ __forceinline__ void run(SRC& src, int first, int end, int whole, float c, int lo_whole = 0) {
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
    if (first >= end) return;
    const int nt = (end - first + TILE - 1) / TILE, half4 = side() + 4 * ((threadIdx.x >> 5) & 1);
    f32x16 s0[NB], s1[NB];
    float top = 0.f;
    src.start(first);
    if (K_AHEAD) {
      src.begin(sm, sm + HALF, sm + 2 * HALF, nt > 1);
    } else {
      src.advance(0);
      src.load_k(0, sm);
      src.load_v(0, sm + 2 * HALF);
    }
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) asm volatile("" : "+v"(qf[kk]));  // here, not at every tile: the loads in flight then are the next tile's
    if (K_AHEAD) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      src.then(sm + HALF, nt > 1);
      scores(s0, sm);
      if (partial(first)) mask(s0, first + half4);
      top = top_of(s0);
    }
    // One tile.  K_AHEAD: its scores in s, the next one's go to n (behind the last tile they are of no tile, and not used: one way
    // through the step, as two ways that both sum into o cost the compiler a second set of its registers).
    auto step = [&](int t, auto SLOT, f32x16(&s)[NB], f32x16(&n)[NB]) __attribute__((always_inline)) {
      const int base = first + t * TILE;
      const bool partly = base + TILE > whole || (WINDOW && base < lo_whole && base + TILE > sinks);
      char* const vs = sm + (2 + SLOT) * HALF;
      uint32_t bad = 0;
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (t + 1 < nt) {
        src.advance(t + 1 + K_AHEAD);
        if (t + 1 + K_AHEAD < nt) src.load_k(t + 1 + K_AHEAD, sm + (SLOT + 1 + K_AHEAD) % 2 * HALF);
        src.load_v(t + 1, sm + (3 - SLOT) * HALF);
      }
      if (partly) {
        clean(vs, bad);
        note(bad, t);
        __syncthreads();
      }
      if (base < any_sees) {
        V8 p[NB][2];
        if (K_AHEAD) {
          const bool done = raise(s, top, c);
          scores_and_weights(n, sm + (1 - SLOT) * HALF, p, s, done ? 1.f : c, done ? 0.f : finite_or_zero(m));
          if (partial(base + TILE)) mask(n, base + TILE + half4);
          top = values_and_top(p, vs, n);
        } else {
          scores(s, sm + SLOT * HALF);
          if (partial(base)) mask(s, base + half4);
          const bool done = raise(s, top_of(s), c);
          weights(p, s, done ? 1.f : c, done ? 0.f : finite_or_zero(m));
          values(p, vs);
        }
      }
      if (partly && spoiled(t)) spoil(vs, base + half4, bad);
    };
    if constexpr (K_AHEAD) {
      int t = 0;
      for (; t + 1 < nt; t += 2) {
        step(t, std::integral_constant<int, 0>(), s0, s1);
        step(t + 1, std::integral_constant<int, 1>(), s1, s0);
      }
      if (t < nt) step(t, std::integral_constant<int, 0>(), s0, s1);
    } else {
      for (int t = 0; t < nt; ++t) step(t, t & 1, s0, s1);
    }
    l = pair_sum(l);
  }

  // SIDES 2: the first four waves' sums become those of both sides, by way of LDS, where nothing is needed any more.
  __device__ __forceinline__ void meet() {
    static_assert(D / 2 * kThreads * 4 <= LDS, "the sums of a side");
    __shared__ float2 other[kThreads];
    float* const sums = reinterpret_cast<float*>(sm) + threadIdx.x % kThreads;
    __syncthreads();
    if (threadIdx.x >= kThreads) {
      other[threadIdx.x % kThreads] = float2{m, l};
#pragma unroll
      for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) sums[(16 * d + r) * kThreads] = o[d][r];
    }
    __syncthreads();
    if (threadIdx.x >= kThreads) return;
    const float2 of = other[threadIdx.x];
    const float top = fmaxf(m, of.x), f = __builtin_amdgcn_exp2f(m - finite_or_zero(top)), g = __builtin_amdgcn_exp2f(of.x - finite_or_zero(top));
    m = top;
    l = l * f + of.y * g;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] = o[d][r] * f + sums[(16 * d + r) * kThreads] * g;
  }

  // The row's result.  A lane and its partner hold every other four elements of their row; two exchanges a pair of fours make them eights,
  // half the stores (24 sequences of up to 901 tokens, 32 heads of 64: 71.5 -> 70 us; by way of LDS, in whole rows, no faster).
  __device__ __forceinline__ void put(T* out, bool none) const {
    const float inv = none ? 0.f : 1.f / l;  // and the sums are zero
    auto of = [=](float x) { return result(x, x * inv); };
    typedef T T2 __attribute__((ext_vector_type(2)));
    hq_u4v* to = reinterpret_cast<hq_u4v*>(out) + ((threadIdx.x >> 5) & 1);
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int g = 0; g < 4; g += 2) {
        hq_u4v v;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = 4 * g + 2 * i;
          const auto s = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, T2{(T)of(o[d][r]), (T)of(o[d][r + 1])}),
                                                          __builtin_bit_cast(uint32_t, T2{(T)of(o[d][r + 4]), (T)of(o[d][r + 5])}), false, false);
          v[i] = s[0];
          v[2 + i] = s[1];
        }
        to[4 * d + g] = v;
      }
  }
};

// ---- few rows ------------------------------------------------------------------------------------------------------------
// Up to 16 rows that all see the same keys.  The workgroup's keys are dealt out to its waves in blocks of 32; a wave's block is on its
// way into LDS of its own while the wave works on what it has: the keys' half is free, and filled again, once the scores are made, the values'
// once they are summed, and no wave waits for another.  A row's scores are in four lanes, 16 apart (16x16 tiles: with 32 rows a
// tile half of the vector unit's work would be for rows that are not there).  Bound by memory.  MASKED: rows that see different keys.
template <typename T, int D, bool MASKED = false>
struct Few {
  typedef typename Kind<T>::V8 V8;
  static constexpr int CH = D / 8, RG = 64 / CH, G = 32 / RG;  // pieces of a row; rows of an instruction; instructions of a block's keys
  static constexpr int HALF = 32 * D * 2, LDS = kWaves * 2 * HALF, STRIDE = D + 4;
  static_assert(kWaves * 16 * STRIDE * 4 <= LDS, "the waves' sums");

  char* sm;
  V8 qf[D / 32];
  f32x4 o[D / 16];
  float m = -INFINITY, l = 0.f;
  bool slow = false;  // as in Many
  // MASKED: the lane's row sees keys below lim, of those the ones below `sinks` and from `lo` on; every row the ones below all_see, from lo_most on
  int lim, lo, sinks, all_see, lo_most;
  Skip skip;
  __device__ __forceinline__ int place(int u) const { return MASKED ? skip.key(u) : u; }
  __device__ __forceinline__ bool sees(int u) const { return u < lim && (u >= lo || u < sinks); }

  // As clean() and store_bad() of Many, of the wave's own block.  Whether there was anything that is not finite.
  static __device__ __forceinline__ bool clean(char* values, uint32_t (&bad)[G / 4]) {
    hq_u4v* vs = reinterpret_cast<hq_u4v*>(values) + (threadIdx.x & 63);
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const hq_u4v v = vs[i * 64];
#pragma unroll
      for (int w = 0; w < 4; ++w) any |= (v[w] & Kind<T>::kExp) + Kind<T>::kStep;
    }
    if (!__ballot((any & 0x80008000u) != 0)) return false;
#pragma unroll
    for (int j = 0; j < G / 4; ++j) {
      bad[j] = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        hq_u4v v = vs[(4 * j + i) * 64];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t e = ((v[w] & Kind<T>::kExp) + Kind<T>::kStep) & 0x80008000u;
          bad[j] |= ((e >> 15 & 1u) | (e >> 30 & 2u)) << (8 * i + 2 * w);
          v[w] &= ~((e >> 15) * 0xffffu);
        }
        vs[(4 * j + i) * 64] = v;
      }
    }
    return true;
  }
  static __device__ __forceinline__ void store_bad(char* values, const uint32_t (&bad)[G / 4]) {
#pragma unroll
    for (int i = 0; i < G; ++i) {
      hq_u4v w;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t b = bad[i / 4] >> (8 * (i % 4) + 2 * j);
        w[j] = (b & 1 ? Kind<T>::kOne & 0xffffu : 0u) | (b & 2 ? Kind<T>::kOne & 0xffff0000u : 0u);
      }
      reinterpret_cast<hq_u4v*>(values)[(threadIdx.x & 63) + i * 64] = w;
    }
  }
  // V^T of 16 elements of the head (block d) and the block's 32 keys.
  static __device__ __forceinline__ V8 v_operand(const char* values, int d) {
    const int lane = threadIdx.x & 63;
    const int row = 4 * (lane >> 4) + ((lane >> 2) & 3), ch = 2 * d + ((lane >> 1) & 1);
    lds_char* at = (lds_char*)values + (lane & 1) * 8;
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    union {
      s16x4 h[2];
      V8 v;
    } u;
    u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + row * D * 2 + v_piece<D>(row, ch) * 16));
    u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + (row + 16) * D * 2 + v_piece<D>(row + 16, ch) * 16));
    return u.v;
  }

  __device__ __forceinline__ void run(const Pages<T, D>& p, int first, int end, float c) {
    const int lane = threadIdx.x & 63, wave = uniform((int)(threadIdx.x >> 6)), quarter = lane >> 4;
#pragma unroll
    for (int d = 0; d < D / 16; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int blocks = (end - first + 31) / 32;
    if (wave >= blocks) return;
    char* const ks = sm + wave * 2 * HALF;
    char* const vs = ks + HALF;
    const uint32_t koff = (lane / CH) * D * 2 + k_piece<D>(lane / CH, lane % CH) * 16, voff = (lane / CH) * D * 2 + v_piece<D>(lane / CH, lane % CH) * 16;
    // pages of 64 / G blocks, a lane for each instruction of each
    constexpr int SET = 64 / G;
    auto ids_of = [&](int set) { return p.id(place(min(first + (wave + kWaves * (set * SET + lane / G)) * 32 + lane % G * RG, end - 1))); };
    Places here;
    auto places_of = [&](int set, int id) {
      Places x;
      x.set(p, id, place(first + (wave + kWaves * (set * SET + lane / G)) * 32 + lane % G * RG));
      return x;
    };
    int ids = ids_of(0), ids_next = 0;
    here = places_of(0, ids);
    // Whether all G instructions were needed: what the waits count.
    auto load = [&](const char* pool, int block, const Places& places, int set_ids, char* to, auto values) {
      const int base = first + block * 32, at = block / kWaves % SET * G;
      // (MASKED: rows behind the last one are whatever their page holds, unseen)
      if (MASKED || base + 32 <= end) return places.template load<D, values, G>(pool, at, values ? voff : koff, to);
      // the last block: rows behind the last key repeat it, every lane by an address of its own
      const uint32_t lds = uniform((int)lds_address(to));
      bool whole = true;
#pragma unroll
      for (int i = 0; i < G; ++i) {
        const int row = i * RG + lane / CH, key = min(base + row, end - 1), page = __shfl(set_ids, at + (key - base) / RG);
        const int ch = values ? v_piece<D>(row, lane % CH) : k_piece<D>(row, lane % CH);
        if (!p.none(page)) to_lds(lds + i * 1024, pool + p.at(page, place(key)) + ch * 16);
        else zero_lds(to + i * 1024);
        whole &= __ballot(p.none(page)) == 0;
      }
      return whole;
    };
    // Waits for everything but the last load(), if that was a whole one.
    auto wait_but = [](bool whole) {
      if (whole) asm volatile("s_waitcnt vmcnt(%0)" ::"i"(G) : "memory");
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    };
    load(p.k, wave, here, ids, ks, std::false_type());
    bool whole_k = false, whole_v = load(p.v, wave, here, ids, vs, std::true_type());
#pragma unroll
    for (int kk = 0; kk < D / 32; ++kk) asm volatile("" : "+v"(qf[kk]));
    for (int block = wave; block < blocks; block += kWaves) {
      const int base = first + block * 32, nth = block / kWaves, next = block + kWaves;
      const bool more = next < blocks, set_ends = (nth + 1) % SET == 0;
      if (nth % SET == 0 && block + SET * kWaves < blocks) ids_next = ids_of(nth / SET + 1);
      wait_but(whole_v);  // the values may still be on their way
      f32x4 s[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        s[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < D / 32; ++kk) {
          const int row = 16 * b + (lane & 15);
          s[b] = Kind<T>::mfma(*reinterpret_cast<const V8*>(ks + row * D * 2 + k_piece<D>(row, 4 * kk + quarter) * 16), qf[kk], s[b]);
        }
      }
      float top = -INFINITY;
      const bool partial = MASKED && (base + 32 > all_see || (base < lo_most && base + 32 > sinks));
      if (partial)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int r = 0; r < 4; ++r) s[b][r] = sees(base + 16 * b + 4 * quarter + r) ? s[b][r] : -INFINITY;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (!MASKED && base + 32 > end && 16 * b + 4 * quarter + r >= end - base) s[b][r] = -INFINITY;
          top = fmaxf(top, s[b][r]);
        }
      asm volatile("" : "+v"(top)::"memory");  // the keys have been read
      if (set_ends && more) {
        ids = ids_next;
        here = places_of(nth / SET + 1, ids);
      }
      whole_k = more && load(p.k, next, here, ids, ks, std::false_type());
      top = quarters_max(top) * c;
      if (__builtin_amdgcn_ballot_w64(outgrown<T>(top, m))) {  // as in Many
        const float mn = outgrown<T>(top, m) ? lifted<T>(top) : m, f = mn == m ? 1.f : __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        slow = __builtin_amdgcn_ballot_w64(far(m)) != 0;
        l *= f;
#pragma unroll
        for (int d = 0; d < D / 16; ++d)
#pragma unroll
          for (int r = 0; r < 4; ++r) o[d][r] *= f;
      }
      if (slow)
#pragma unroll
        for (int b = 0; b < 2; ++b) exponents(s[b], 4, c, m);
      const float cs = slow ? 1.f : c, ms = slow ? 0.f : finite_or_zero(m);
      V8 w;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float e = __builtin_amdgcn_exp2f(fmaf(s[i / 4][i % 4], cs, -ms));
        l += e;
        w[i] = (T)e;
      }
      wait_but(whole_k);
      uint32_t bad[G / 4];
      const bool spoiled = partial && clean(vs, bad);
#pragma unroll
      for (int d = 0; d < D / 16; ++d) o[d] = Kind<T>::mfma(v_operand(vs, d), w, o[d]);
      if (spoiled) {  // rows that see a value that is not finite
        asm volatile("" ::: "memory");
        store_bad(vs, bad);
        asm volatile("" ::: "memory");
        V8 seen;
#pragma unroll
        for (int i = 0; i < 8; ++i) seen[i] = sees(base + 16 * (i / 4) + 4 * quarter + i % 4) ? (T)1.f : (T)0.f;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
          const f32x4 n = Kind<T>::mfma(v_operand(vs, d), seen, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
          for (int r = 0; r < 4; ++r) o[d][r] = n[r] > 0.f ? NAN : o[d][r];
        }
      }
#pragma unroll
      for (int d = 0; d < D / 16; ++d) asm volatile("" : "+v"(o[d])::"memory");  // the values have been read
      whole_v = more && load(p.v, next, here, ids, vs, std::true_type());
    }
    l = quarters_sum(l);
  }

  // The waves' sums together: a thread's part of a row's, D / 16 elements from it % 16 of row it / 16 on, and the row's maximum and sum.
  __device__ __forceinline__ void join(float (&sum)[D / 16], float* top, float* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, quarter = lane >> 4;
    __shared__ float tops[kWaves][16], totals[kWaves][16];
    if (quarter == 0) tops[wave][lane] = m;
    __syncthreads();  // and nobody reads keys or values any more
    float mm = -INFINITY;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) mm = fmaxf(mm, tops[i][lane & 15]);
    const float f = __builtin_amdgcn_exp2f(m - finite_or_zero(mm));
    if (quarter == 0) totals[wave][lane] = l * f;
    float* sums = reinterpret_cast<float*>(sm);
#pragma unroll
    for (int d = 0; d < D / 16; ++d) *reinterpret_cast<f32x4*>(sums + (wave * 16 + (lane & 15)) * STRIDE + 16 * d + 4 * quarter) = o[d] * f;
    __syncthreads();
    const int row = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * (D / 16);
#pragma unroll
    for (int i = 0; i < D / 16; ++i) sum[i] = 0.f;
    *total = 0.f;
    mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i) sum[i] += sums[(w * 16 + row) * STRIDE + d0 + i];
      *total += totals[w][row];
      mm = fmaxf(mm, tops[w][row]);
    }
    *top = mm;
  }
};

// Sets up the poison word; a barrier of run() lies between this and its first use.
__device__ __forceinline__ void set_up(int* poison) {
  if (threadIdx.x == 0) *poison = -1;
}

// A sequence's tokens and keys.
struct Sequence {
  int q0, nq, k0, nk, tile;
};
// Tile x of a list in which sequence i has tiles(its tokens) tiles: its sequence, and which of its tiles.  A wave looks at 64 sequences at a
// time, keys' bounds along with tokens', so that one trip to memory does.  (Longest sequences first: no faster; nor is a workgroup that
// goes from tile to tile.)
template <typename A, typename F>
__device__ __forceinline__ bool find_tile(const A& a, int x, F tiles, Sequence* s) {
  const int lane = threadIdx.x & 63;
  for (int i0 = 0; i0 < a.seqs; i0 += 64) {
    const int i = min(i0 + lane, a.seqs - 1);
    const int qb = a.cu_q[i], qe = a.cu_q[i + 1], kb = a.cu_k[i], ke = a.cu_k[i + 1];
    const int b = min(max(qb, 0), a.total_q), len = i0 + lane < a.seqs ? min(max(qe, b), a.total_q) - b : 0;
    const int k = min(max(kb, 0), a.total_k), keys = min(max(ke, k), a.total_k) - k;
    const int t = tiles(len);
    int sum = t;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int u = __shfl_up(sum, d);
      if (lane >= d) sum += u;
    }
    const int before = sum - t, total = __builtin_amdgcn_readlane(sum, 63);
    const unsigned long long here = __ballot(x >= before && x < before + t);
    if (here) {
      const int at = __ffsll(here) - 1;
      *s = Sequence{__builtin_amdgcn_readlane(b, at), __builtin_amdgcn_readlane(len, at), __builtin_amdgcn_readlane(k, at),
                    __builtin_amdgcn_readlane(keys, at), x - __builtin_amdgcn_readlane(before, at)};
      return true;
    }
    x -= total;
  }
  return false;
}

// Sums of whole numbers over the wave, and over the lanes up to each.
struct AddWhole {
  __device__ __forceinline__ float operator()(float x, float y) const { return __uint_as_float(__float_as_uint(x) + __float_as_uint(y)); }
};
__device__ __forceinline__ unsigned wave_sum(unsigned v) { return __float_as_uint(hq_wave(__uint_as_float(v), AddWhole())); }
__device__ __forceinline__ unsigned running_sum(unsigned v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1, 2, 4, 8: within the rows of 16
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1 and 3, :31 into rows 2 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return v;
}

// The shares of up to 16 rows together, by one workgroup: 16 threads a row, whose loads are of two values each, side by side, and the
// shares, `step` places apart, divided among the sets of threads that there are then.  Written by others a moment ago: read past the caches
// of this XCD.  all: the rows' results; else the sums go to the place of the first of the shares, which has been read by then.
// out_row: where the result of one of the rows is.
template <typename T, int D, typename A, typename F>
__device__ __forceinline__ void join_here(const A& a, char* sm, int nrows, int64_t row0, int64_t place, int64_t step, int slots, bool all, F out_row) {
  constexpr int N = D / 16, AT_ONCE = 4;
  const int log = nrows > 8 ? 4 : nrows > 4 ? 3 : nrows > 2 ? 2 : nrows > 1, sets = 16 >> log;
  const int set = threadIdx.x >> (4 + log), row = (threadIdx.x >> 4) & ((1 << log) - 1), d0 = (threadIdx.x & 15) * 2;
  const int64_t at = row0 + min(row, nrows - 1);
  const unsigned long long* const pm = reinterpret_cast<const unsigned long long*>(a.pm) + at + place;
  const unsigned long long* const po = reinterpret_cast<const unsigned long long*>(a.po + (at + place) * D + d0);
  float m = -INFINITY, l = 0.f, o[N] = {};
  for (int s0 = set; s0 < slots; s0 += AT_ONCE * sets) {
    unsigned long long ml[AT_ONCE], v[AT_ONCE][N / 2];
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const int s = min(s0 + i * sets, slots - 1);
      ml[i] = __hip_atomic_load(pm + s * step, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
      for (int j = 0; j < N / 2; ++j) v[i][j] = __hip_atomic_load(po + s * step * (D / 2) + 16 * j, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) top = fmaxf(top, __uint_as_float((uint32_t)ml[i]));
    const float f = __builtin_amdgcn_exp2f(m - finite_or_zero(top));
    m = top;
    l *= f;
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] *= f;
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      // A share of weight 0 counts too: what is not finite in it stays so (one without keys holds zeros).
      const float w = __builtin_amdgcn_exp2f(__uint_as_float((uint32_t)ml[i]) - finite_or_zero(m));
      if (s0 + i * sets < slots) {
        l += w * __uint_as_float((uint32_t)(ml[i] >> 32));
#pragma unroll
        for (int j = 0; j < N; ++j) o[j] += w * __uint_as_float((uint32_t)(v[i][j / 2] >> 32 * (j & 1)));
      }
    }
  }
  if (sets > 1) {
    float* const sums = reinterpret_cast<float*>(sm) + threadIdx.x;  // N + 2 planes of a float a thread
    sums[0] = m;
    sums[kThreads] = l;
#pragma unroll
    for (int j = 0; j < N; ++j) sums[(2 + j) * kThreads] = o[j];
    __syncthreads();
    if (set) return;
    const int apart = 16 << log;
    float top = m;
    for (int s = 1; s < sets; ++s) top = fmaxf(top, sums[s * apart]);
    const float own = __builtin_amdgcn_exp2f(m - finite_or_zero(top));
    m = top;
    l *= own;
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] *= own;
    for (int s = 1; s < sets; ++s) {
      const float w = __builtin_amdgcn_exp2f(sums[s * apart] - finite_or_zero(top));
      l += w * sums[s * apart + kThreads];
#pragma unroll
      for (int j = 0; j < N; ++j) o[j] += w * sums[s * apart + (2 + j) * kThreads];
    }
  }
  if (row >= nrows) return;
  if (!all) {
    auto put = [](const unsigned long long* to, float x, float y) {
      __hip_atomic_store(const_cast<unsigned long long*>(to), (unsigned long long)__float_as_uint(y) << 32 | __float_as_uint(x), __ATOMIC_RELAXED,
                         __HIP_MEMORY_SCOPE_AGENT);
    };
#pragma unroll
    for (int j = 0; j < N / 2; ++j) put(po + 16 * j, o[2 * j], o[2 * j + 1]);
    if (d0 == 0) put(pm, m, l);
    return;
  }
  const bool none = m == -INFINITY;
  typedef T T2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int j = 0; j < N; j += 2)
    *reinterpret_cast<T2*>((T*)a.out + out_row(row) * D + d0 + 16 * j) = none ? T2{(T)0.f, (T)0.f} : T2{(T)result(o[j], o[j] / l), (T)result(o[j + 1], o[j + 1] / l)};
}

constexpr int kJoin = 32, kTeam = 16;  // shares that are joined at once, of that many and of more
// Shares that there is room for, two workgroups a compute unit (`side` of them for every one), and no more than two steps join: a team's counter is that
// of its first share, and a third step's first team would count on the first one's, which others may still be at.  (256 compute units: 512,
// just as many.)
constexpr int64_t share_room(int64_t cus, int64_t side) { return std::max<int64_t>(std::min<int64_t>(2 * cus / side, kJoin * kTeam), 1); }
static_assert(share_room(1024, 1) <= kJoin * kTeam, "joined in two steps on any device");
constexpr int kApart = 16;  // counters, a line of 64 bytes each: atomics on one line wait for each other (64 shares: 17.7 us, apart 14.5)

// The shares of a row together, by WAVES waves: their maxima and sums a lane each, then the sums of the values, 16 bytes a lane, several
// shares at a time; a wave takes every WAVES-th group of them.  Of the shares, those from `np` to `own` were not written.  PRE:
// the first PRE groups, if below `likely` or from `own` on, are asked for before np and the maxima are there: one trip to memory less
// where rows are few (32 rows of 64 shares 14.6 -> 12.3 us with the whole call, 1280 of 12 15.4 -> 15.0), and only more to read where
// they are many (2048 rows of 9 shares 72.8 -> 74.3).
template <typename T, int D, int WAVES, int PRE>
__device__ __forceinline__ void join_shares(const float* po, const float* pm, int64_t row, int64_t place, int step, int np, int own, int slots, int likely,
                                            T* out) {
  constexpr int LANES = D / 4, AT_ONCE = 64 / LANES, EVERY = WAVES * AT_ONCE;  // lanes of a share, shares of a load
  const int lane = threadIdx.x & 63, d = (lane % LANES) * 4, wave = WAVES == 1 ? 0 : threadIdx.x >> 6, mine0 = wave * AT_ONCE + lane / LANES;
  const float2* ml = reinterpret_cast<const float2*>(pm) + place;
  const float2 ahead = ml[(int64_t)min(lane, slots - 1) * step];
  auto sums = [&](int s) { return *reinterpret_cast<const hq_f4v*>(po + (place + (int64_t)s * step) * D + d); };
  auto early = [&](int s) { return s < slots && (s < likely || s >= own); };
  hq_f4v pre[PRE ? PRE : 1];
#pragma unroll
  for (int i = 0; i < PRE; ++i) pre[i] = sums(early(mine0 + i * EVERY) ? mine0 + i * EVERY : 0);
  auto share = [&](int s0) {
    const int s = s0 + lane;
    const float2 x = s0 ? ml[(int64_t)min(s, slots - 1) * step] : ahead;
    return s < np || (s >= own && s < slots) ? x : float2{-INFINITY, 0.f};
  };
  float m = -INFINITY;
  for (int s0 = 0; s0 < slots; s0 += 64) m = fmaxf(m, share(s0).x);
  m = hq_wave_max(m);
  const bool none = m == -INFINITY;
  const float ms = finite_or_zero(m);
  float l = 0.f;
  hq_f4v o = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < slots; s0 += 64) {
    const int here = min(slots - s0, 64);
    const float2 x = share(s0);
    // the share's weight; -1: it has no keys, and nothing was written for it (one of weight 0 counts: what is not finite in it stays so)
    const float f = x.x == -INFINITY ? -1.f : __builtin_amdgcn_exp2f(x.x - ms);
    l += x.y * f;
    int i0 = 0;
    if (PRE && s0 == 0) {
#pragma unroll
      for (int i = 0; i < PRE; ++i) {
        const int at = mine0 + i * EVERY;
        const float w = __shfl(f, at & 63);
        if (at < here && !(w < 0.f)) o += (early(at) ? pre[i] : sums(at)) * w;
      }
      i0 = PRE * EVERY;
    }
#pragma unroll 8
    for (int i = i0; i < here; i += EVERY) {
      const int at = i + mine0;
      const float w = __shfl(f, at & 63);
      if (at < here && !(w < 0.f)) o += sums(s0 + at) * w;
    }
  }
  l = hq_wave_sum(l);
#pragma unroll
  for (int x = LANES; x < 64; x <<= 1)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] += __shfl_xor(o[i], x);
  if (WAVES > 1) {
    __shared__ hq_f4v parts[WAVES][LANES];
    if (lane < LANES) parts[wave][lane] = o;
    __syncthreads();
    if (wave > 0 || lane >= LANES) return;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) o += parts[w][lane];
  }
  if (lane < LANES) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    T4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (T)(none ? 0.f : result(o[i], o[i] / l));
    *reinterpret_cast<T4*>(out + row * D + d) = v;
  }
}

// A row of few shares takes a wave, one of many a workgroup (1024 rows of 128, 33 shares: 9.3 us by waves, 7.0 by workgroups; 4096
// rows, 9 shares: 7.2 and 10.6).
constexpr int kSharesOfAWave = 16;

template <typename A>
struct Joins {  // by waves and by workgroups, and the same with loads ahead
  void (*waves)(A), (*workgroups)(A), (*waves_ahead)(A), (*workgroups_ahead)(A);
};
template <typename A>
int launch_join(const Joins<A>& by, int64_t rows, int64_t slots, hipStream_t stream, const A& a) {
  if (slots <= kSharesOfAWave)
    return hq_launch_as_is(rows < 2048 ? by.waves_ahead : by.waves, dim3((unsigned)((rows + kWaves - 1) / kWaves)), dim3(kThreads), 0, stream, a);
  return hq_launch_as_is(rows < 2048 ? by.workgroups_ahead : by.workgroups, dim3((unsigned)rows), dim3(kThreads), 0, stream, a);
}

// Scores are compared and masked by -infinity before they are scaled: a scale of zero (all keys alike) becomes one that no score notices.
float exponent_scale(float s) { return std::max(s * 1.44269504088896340736f, FLT_TRUE_MIN); }
bool bad_scale(float s) { return !(s >= 0.f) || std::isinf(s); }
// Keys of a row are numbered in 32 bits, as are the ends of loads and shares behind the last one: up to 512 shares rounded up to 128 keys, page
// numbers up to 2048 keys ahead.
constexpr int kMostKeys = INT_MAX - (1 << 17);
// One of the four kernels by type and head size: f of a Form.
template <typename T_, int D_>
struct Form {
  typedef T_ T;
  static constexpr int D = D_;
};
template <typename F>
int by_type(int dtype, int head_dim, F f) {
  if (dtype == HQ_DTYPE_F16) return head_dim == 64 ? f(Form<_Float16, 64>()) : f(Form<_Float16, 128>());
  return head_dim == 64 ? f(Form<__bf16, 64>()) : f(Form<__bf16, 128>());
}
bool misaligned(const void* p, int64_t stride) { return ((uintptr_t)p & 15) || stride % 8; }

}  // namespace
