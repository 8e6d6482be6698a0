// Attention: over whole prompts packed one behind the other, and of one query a request over a paged cache.
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

// The tiles of one sequence's keys, one head, for the four waves of Many.  Rows behind the last one repeat it.
template <typename T, int D>
struct PackedTiles {
  static constexpr int CH = D / 8, NL = 64 * CH / kThreads;  // pieces of a row; instructions of a wave for the keys of a tile
  const T *k, *v;
  int64_t ks, vs;
  int n, first;
  uint32_t koff[NL], voff[NL];
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
  __device__ __forceinline__ void load_k(int t, char* to) {
    const int base = first + t * 64;
    if (base + 64 > n) offsets(koff, (int)ks, n - base, k_piece<D>);
    load(k + base * ks, koff, to);
  }
  __device__ __forceinline__ void load_v(int t, char* to) {
    const int base = first + t * 64;
    if (base + 64 > n) offsets(voff, (int)vs, n - base, v_piece<D>);
    load(v + base * vs, voff, to);
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

// The same tiles of pages.  Rows behind the last one are whatever its page holds.
template <typename T, int D>
struct PagedTiles {
  static constexpr int CH = D / 8, NL = 64 * CH / kThreads, RG = 64 / CH;  // RG: rows of an instruction, all in one page
  Pages<T, D> p;
  int n, first;
  int ids;          // pages of the wave's instructions' rows, one a lane, of the tile to come
  Places next, now; // of the tile whose keys are loaded next, and (heads of 128, whose keys are a tile ahead) of its predecessor
  uint32_t koff, voff;
  __device__ PagedTiles(const Pages<T, D>& pages, int end) : p(pages), n(end) {}
  __device__ __forceinline__ int key(int t) const { return first + t * 64 + (int)((threadIdx.x >> 6) * NL + threadIdx.x % NL) * RG; }
  __device__ __forceinline__ void start(int f) {
    first = f;
    const int lane = threadIdx.x & 63, row = lane / CH;  // of a multiple of 16
    koff = row * D * 2 + k_piece<D>(row, lane % CH) * 16;
    voff = row * D * 2 + v_piece<D>(row, lane % CH) * 16;
    ids = p.id(min(key(0), n - 1));
  }
  // Before the first load of tile t: its pages are there, those of the tile behind it are asked for.
  __device__ __forceinline__ void advance(int t) {
    now = next;
    next.set(p, ids, key(t));
    ids = p.id(min(key(t + 1), n - 1));
  }
  __device__ __forceinline__ void load_k(int, char* to) { next.template load<D, false, NL>(p.k, 0, koff, to + (threadIdx.x >> 6) * (NL * 1024)); }
  __device__ __forceinline__ void load_v(int, char* to) {
    (D == 128 ? now : next).template load<D, true, NL>(p.v, 0, voff, to + (threadIdx.x >> 6) * (NL * 1024));
  }
};

// ---- many rows -----------------------------------------------------------------------------------------------------------
// 128 rows of a workgroup, 32 a wave.
template <typename T, int D>
struct Many {
  typedef typename Kind<T>::V8 V8;
  static constexpr int NB = 2, TILE = 64;           // blocks of 32 keys, keys of a tile
  static constexpr int CH = D / 8, NL = 64 * CH / kThreads;
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

  // In a tile that not every row sees whole, a value that is not finite would reach the rows that do not see it (0 times infinity): it
  // becomes zero, and the bits returned say which values were.
  static __device__ __forceinline__ void clean(char* values, uint32_t& bad) {
    hq_u4v* vs = reinterpret_cast<hq_u4v*>(values) + threadIdx.x;
    hq_u4v v[NL];
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < NL; ++i) v[i] = vs[i * kThreads];
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
      vs[i * kThreads] = v[i];
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
      reinterpret_cast<hq_u4v*>(values)[threadIdx.x + i * kThreads] = w;
    }
  }

  // V^T of 32 elements of the head (block d) and 16 keys (block b, half t) as the matrix core takes it: the keys in the order in which
  // the scores' registers hold them.
  static __device__ __forceinline__ V8 v_operand(const char* values, int b, int t, int d) {
    const int lane = threadIdx.x & 63;
    const int row = 32 * b + 16 * t + 4 * (lane >> 5) + ((lane >> 2) & 3);
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
        const int row = 32 * b + (lane & 31);
        const V8 a = *reinterpret_cast<const V8*>(keys + row * D * 2 + k_piece<D>(row, 2 * kk + half) * 16);
        s[b] = Kind<T>::mfma(a, qf[kk], s[b]);
      }
    }
  }
  // Which of the lane's registers are keys that the row sees: the first `left` of the wave's, less 4 in the upper lanes.
  static __device__ __forceinline__ void mask(f32x16 (&s)[NB], int left) {
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      // bit i: key i of the block is seen; a bit field of a sign and a bitwise select cost two instructions a score and no scalar register
      const int n = left - 32 * b;
      const int seen = n >= 32 ? -1 : n <= 0 ? 0 : (int)((1u << n) - 1);
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
      const int row = 32 * (j / (D / 16)) + (lane & 31);
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
  __device__ __forceinline__ void spoil(char* values, int left, uint32_t bad) {
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
          for (int i = 0; i < 8; ++i) seen[i] = 32 * b + 16 * t + 8 * (i / 4) + i % 4 < left ? (T)1.f : (T)0.f;
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

  // Keys [first, end) of src; whole: keys below it are seen by every row of the workgroup.  A tile is on its way from memory while the one
  // before it is worked on, with one barrier a tile.  Heads of 128: the scores of the next tile are in the matrix core while the vector
  // unit makes this one's weights of its own, and the next scores' maximum is taken under this tile's product with the values; the
  // keys so run a tile ahead.  Heads of 64, where the vector unit is the busier of the two and the registers saved are two waves more: one step after
  // the other (16384 tokens, heads of 128: 2186 us one after the other, 2116 so; 8192 tokens, heads of 64: 359 and 376).
  template <typename SRC>
  __device__ __forceinline__ void run(SRC& src, int first, int end, int whole, float c) {
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
    if (first >= end) return;
    const int nt = (end - first + TILE - 1) / TILE, half4 = 4 * ((threadIdx.x >> 5) & 1);
    f32x16 s0[NB], s1[NB];
    float top = 0.f;
    src.start(first);
    src.advance(0);
    src.load_k(0, sm);
    if (!K_AHEAD) src.load_v(0, sm + 2 * HALF);
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) asm volatile("" : "+v"(qf[kk]));  // here, not at every tile: the loads in flight then are the next tile's
    if (K_AHEAD) {
      src.advance(1);
      src.load_v(0, sm + 2 * HALF);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (nt > 1) src.load_k(1, sm + HALF);
      scores(s0, sm);
      if (first + TILE > all_see) mask(s0, lim - first - half4);
      top = top_of(s0);
    }
    // One tile.  K_AHEAD: its scores in s, the next one's go to n (behind the last tile they are of no tile, and not used: one way
    // through the step, as two ways that both sum into o cost the compiler a second set of its registers).
    auto step = [&](int t, auto SLOT, f32x16(&s)[NB], f32x16(&n)[NB]) __attribute__((always_inline)) {
      const int base = first + t * TILE;
      const bool partly = base + TILE > whole;
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
          if (base + 2 * TILE > all_see) mask(n, lim - base - TILE - half4);
          top = values_and_top(p, vs, n);
        } else {
          scores(s, sm + SLOT * HALF);
          if (base + TILE > all_see) mask(s, lim - base - half4);
          const bool done = raise(s, top_of(s), c);
          weights(p, s, done ? 1.f : c, done ? 0.f : finite_or_zero(m));
          values(p, vs);
        }
      }
      if (partly && spoiled(t)) spoil(vs, lim - base - half4, bad);
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
// tile half of the vector unit's work would be for rows that are not there).  Bound by memory.
template <typename T, int D>
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
    auto ids_of = [&](int set) { return p.id(min(first + (wave + kWaves * (set * SET + lane / G)) * 32 + lane % G * RG, end - 1)); };
    Places here;
    auto places_of = [&](int set, int id) {
      Places x;
      x.set(p, id, first + (wave + kWaves * (set * SET + lane / G)) * 32 + lane % G * RG);
      return x;
    };
    int ids = ids_of(0), ids_next = 0;
    here = places_of(0, ids);
    // Whether all G instructions were needed: what the waits count.
    auto load = [&](const char* pool, int block, const Places& places, int set_ids, char* to, auto values) {
      const int base = first + block * 32, at = block / kWaves % SET * G;
      if (base + 32 <= end) return places.template load<D, values, G>(pool, at, values ? voff : koff, to);
      // the last block: rows behind the last key repeat it, every lane by an address of its own
      const uint32_t lds = uniform((int)lds_address(to));
      bool whole = true;
#pragma unroll
      for (int i = 0; i < G; ++i) {
        const int row = i * RG + lane / CH, key = min(base + row, end - 1), page = __shfl(set_ids, at + (key - base) / RG);
        const int ch = values ? v_piece<D>(row, lane % CH) : k_piece<D>(row, lane % CH);
        if (!p.none(page)) to_lds(lds + i * 1024, pool + p.at(page, key) + ch * 16);
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
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (base + 32 > end && 16 * b + 4 * quarter + r >= end - base) s[b][r] = -INFINITY;
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
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        const int row = 4 * quarter + ((lane >> 2) & 3), ch = 2 * d + ((lane >> 1) & 1);
        lds_char* at = (lds_char*)vs + (lane & 1) * 8;
        typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
        union {
          s16x4 h[2];
          V8 v;
        } u;
        u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + row * D * 2 + v_piece<D>(row, ch) * 16));
        u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + (row + 16) * D * 2 + v_piece<D>(row + 16, ch) * 16));
        o[d] = Kind<T>::mfma(u.v, w, o[d]);
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

// ---- prompts -------------------------------------------------------------------------------------------------------
struct PromptArgs {
  const void *q, *k, *v;
  void* out;
  const int *cu_q, *cu_k;
  int64_t qs, ks, vs;  // elements from one token to the next
  float *po, *pm;      // shares of the sums [total_q * heads][shares][D], and {maximum, sum} [total_q * heads][shares]
  int seqs, total_q, total_k, heads, kv_heads, ratio, causal, shares;
  float c;
};

// A workgroup's rows and share of the keys.  Many rows: all keys, and the result; few: the keys are divided among `shares` workgroups.
template <typename T, int D>
__global__ __launch_bounds__(kThreads, D == 64 ? 4 : 2) void prompt_kernel(PromptArgs a) {
  typedef Many<T, D> A;
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
  w.all_see = __builtin_amdgcn_readlane(w.lim, 0);  // a later row sees as much or more
  w.any_sees = __builtin_amdgcn_readlane(w.lim, 31);
  PackedTiles<T, D> src;
  src.k = (const T*)a.k + (int64_t)k0 * a.ks + head * D;
  src.v = (const T*)a.v + (int64_t)k0 * a.vs + head * D;
  src.ks = a.ks;
  src.vs = a.vs;
  src.n = nk;
  const int each = a.shares == 1 ? nk : max(256, ((nk + a.shares - 1) / a.shares + A::TILE - 1) & -A::TILE);
  const int end = uniform(limit((uint32_t)last_row / ratio)), first = (int)min((int64_t)share * each, (int64_t)end);
  w.run(src, first, min(end, first + each), uniform(limit((uint32_t)first_row / ratio)), a.c);
  if (row > last_row) return;  // and so does the partner
  if (a.shares == 1) {
    w.put((T*)a.out + ((int64_t)(q0 + token) * a.heads + h) * D, w.lim == 0);
  } else {
    w.put_share(a.po, a.pm, ((int64_t)(q0 + token) * a.heads + h) * a.shares + share, w.lim > first);
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

// The shares of up to 16 rows together, by one workgroup: 16 threads a row, whose loads are of two values each, side by side, and the
// shares, `step` places apart, divided among the sets of threads that there are then.  Written by others a moment ago: read past the caches
// of this XCD.  all: the rows' results; else the sums go to the place of the first of the shares, which has been read by then.
template <typename T, int D>
__device__ __forceinline__ void join_here(const PagedArgs& a, char* sm, int nrows, int64_t row0, int64_t place, int64_t step, int slots, bool all) {
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
    *reinterpret_cast<T2*>((T*)a.out + at * D + d0 + 16 * j) = none ? T2{(T)0.f, (T)0.f} : T2{(T)result(o[j], o[j] / l), (T)result(o[j + 1], o[j + 1] / l)};
}

constexpr int kJoin = 32, kTeam = 16;  // shares that are joined at once, of that many and of more
constexpr int kApart = 16;  // counters, a line of 64 bytes each: atomics on one line wait for each other (64 shares: 17.7 us, apart 14.5)

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
    join_here<T, D>(a, sm, nrows, (int64_t)b0 * a.heads + head * ratio, (int64_t)(first_share - b0) * a.heads, (int64_t)unit * a.heads, members, all);
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
  PagedTiles<T, D> src(pages_of<T, D>(a, b0, head), end);
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
bool misaligned(const void* p, int64_t stride) { return ((uintptr_t)p & 15) || stride % 8; }

// Few rows leave compute units idle, and each of their workgroups with all keys: then the keys are divided, 256 a share at least, and the
// shares joined by a second launch.  Into how many parts, an estimate says, of sequences of the average length (lengths are device memory),
// in us: a tile of 64 keys takes a workgroup 1.04 alone (heads of 64: 0.88), a compute unit 0.96 (0.65) where it has more of them, and
// every share of a row is written and read.  40 tokens behind 2900 keys, 32 / 8 heads of 128: 50.9 us, in 12 shares 16.1; 512 behind
// 8000 143.8, in four 90.5; 1000 by themselves 24.0, in two 35.9; 17 sequences of up to 248, 12 / 1 heads, 11.7 and 29.1.
template <typename T, int D>
int launch_prompt(PromptArgs a, int cus, hipStream_t stream) {
  const int64_t items = ((int64_t)a.total_q * a.ratio / 128 + a.seqs) * a.kv_heads, rows = (int64_t)a.total_q * a.heads;
  const float queries = (float)a.total_q / a.seqs, keys = (float)a.total_k / a.seqs;
  const float unit = (D == 128 ? 0.96f : 0.65f) / cus * std::max(queries * a.ratio / 128, 1.f) * a.seqs * a.kv_heads;
  const float deepest = keys / 64, mean = (a.causal ? keys - std::min(queries, keys) / 2 : keys) / 64;
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
  const int rc = hq_launch_as_is(prompt_kernel<T, D>, dim3((unsigned)(items * a.shares)), dim3(kThreads), Many<T, D>::LDS, stream, a);
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
      const int64_t most = a.batch * std::max<int64_t>(1, (cap + kUnit - 1) / kUnit), room = divide ? 2 * (int64_t)cus / (a.kv_heads * tiles) : 1;
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

// One of the four kernels by type and head size.
#define HQ_BY_TYPE(fn, ...)                                                                     \
  (dtype == HQ_DTYPE_F16 ? (head_dim == 64 ? fn<_Float16, 64>(__VA_ARGS__) : fn<_Float16, 128>(__VA_ARGS__)) \
                         : (head_dim == 64 ? fn<__bf16, 64>(__VA_ARGS__) : fn<__bf16, 128>(__VA_ARGS__)))
}  // namespace

extern "C" int hq_prompt_attention(const void* q, const void* k, const void* v, void* out, int dtype, const int32_t* cu_q,
                                   const int32_t* cu_k, int seqs, int64_t total_q, int64_t total_k, int heads, int kv_heads,
                                   int head_dim, int64_t q_stride, int64_t k_stride, int64_t v_stride, float scale, int causal,
                                   void* stream) {
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
                     heads / kv_heads, causal != 0, 1, exponent_scale(scale)};
  return HQ_BY_TYPE(launch_prompt, a, dev->cus, (hipStream_t)stream);
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
  return HQ_BY_TYPE(launch_paged, a, dev->cus, (hipStream_t)stream);
}
