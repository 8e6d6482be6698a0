// Attention: over whole prompts packed one behind the other, and of one query a request over a paged cache.
//
// For a query row q: out = sum_j p_j v_j / sum_j p_j, p_j = 2^(c q.k_j - m), c = scale * log2(e), in one pass over the keys with the
// running maximum m of the row; a larger maximum scales what has been summed so far.
//
// Rows: the R = heads / kv_heads query heads of a key / value head and the tokens (or requests) are one list of rows
// (token, head of the group), so that a tile of keys in LDS serves all of them.  A wave has 32 rows.  The scores are computed
// transposed, S^T = K Q^T: the matrix core leaves a row's scores in one lane and its partner 32 lanes on, so maximum and sum are
// sums within a lane and one exchange, and the same registers are, rounded, the operand of O^T = V^T P^T without another move: the
// order of the keys in that sum is free, and the transposing LDS read fetches V's rows in the order in which S^T left them.
#include <algorithm>
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

template <typename T>
struct Kind;
template <>
struct Kind<__bf16> {
  typedef bf16x8 V8;
  static constexpr uint32_t kExp = 0x7f807f80u, kStep = 0x00800080u, kOne = 0x3f803f80u;
  static __device__ __forceinline__ f32x16 mfma(V8 a, V8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Kind<_Float16> {
  typedef f16x8 V8;
  static constexpr uint32_t kExp = 0x7c007c00u, kStep = 0x04000400u, kOne = 0x3c003c00u;
  static __device__ __forceinline__ f32x16 mfma(V8 a, V8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
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
__device__ __forceinline__ float finite_or_zero(float m) { return m == -INFINITY ? 0.f : m; }

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

// What one workgroup attends: up to 128 rows (RW = 4 waves of them, all of which see every key of a tile) or up to 32 rows (RW = 1,
// the waves share the tile's keys among them).
template <typename T, int D, int RW, bool DIRECT = false>
struct Attend {
  typedef typename Kind<T>::V8 V8;
  static constexpr int KW = kWaves / RW;            // waves that divide a tile's keys
  static constexpr int NB = RW == 4 ? 2 : 1;        // blocks of 32 keys of a wave
  static constexpr int TILE = 32 * NB * KW;         // keys of a tile
  static constexpr int CH = D / 8;                  // 16-byte pieces of a row
  static constexpr int NL = TILE * CH / kThreads;   // pieces that a thread brings
  static constexpr int STEP = kThreads / CH;        // rows between two of them
  static constexpr int BUF = 2 * TILE * D * 2;      // a tile's keys and values
  static constexpr int LDS = (DIRECT ? 2 : 1) * BUF;

  // A row's pieces are stored in an order that depends on the row, so that the lanes of a read pass meet different banks: the keys'
  // pieces by all bits of the row, which 16 lanes read piece by piece, the values' by the two bits of the four rows that a
  // transposing read takes together, 64 bytes of each.
  static __device__ __forceinline__ int k_piece(int row, int ch) { return D == 128 ? ch ^ (row & 15) : ch ^ ((row >> 1) & 7); }
  static __device__ __forceinline__ int v_piece(int row, int ch) { return D == 128 ? ch ^ ((row & 3) << 2) : ch ^ (((row >> 1) & 1) << 2); }

  char* sm;
  int* poison;  // in LDS: the tile whose values hold something that is not finite
  V8 qf[D / 16];
  f32x16 o[D / 32];
  float m = -INFINITY, l = 0.f;
  hq_u4v kr[NL], vr[NL];
  int lim;              // keys below this are seen by the lane's row
  int all_see, any_sees;  // below the first by all rows of the wave, below the second by one of them

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
  }

  template <typename SRC>
  __device__ __forceinline__ void load(const SRC& src, int base) {
    const int ch = threadIdx.x % CH, row = threadIdx.x / CH;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const T *k, *v;
      const bool there = src.at(base + row + i * STEP, &k, &v);
      kr[i] = *reinterpret_cast<const hq_u4v*>(k + ch * 8);
      vr[i] = *reinterpret_cast<const hq_u4v*>(v + ch * 8);
      if (!there) kr[i] = vr[i] = hq_u4v{0, 0, 0, 0};
    }
  }

  // DIRECT: a tile goes from memory into LDS past the registers, its second buffer is filled while the first is worked on, and one barrier
  // a tile does.  An instruction brings 1 KB, the lanes' pieces one behind the other, so it is the lane's address that follows the
  // order of the pieces.
  uint32_t koff[NL], voff[NL];
  // (Of a thread number that the compiler cannot see through where it happens inside the loop, once: nothing of it is then kept in
  // registers all along.)
  template <typename F>
  static __device__ __forceinline__ void direct_offsets(uint32_t (&off)[NL], int stride, int rows, F piece) {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int row = ((tid >> 6) * NL + i) * (64 / CH) + (tid & 63) / CH;
      off[i] = __umul24(min(row, rows - 1), 2 * stride) + piece(row, tid % CH) * 16;
    }
  }
  static __device__ __forceinline__ void direct_load(const T* from, const uint32_t (&off)[NL], char* to) {
    from = uniform(from);
    const uint32_t lds = uniform((int)((uint32_t)(uintptr_t)(lds_char*)to + (threadIdx.x >> 6) * (NL * 1024)));
#pragma unroll
    for (int i = 0; i < NL; ++i)
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds + i * 1024), "v"(off[i]), "s"(from) : "memory");
  }
  // What store() does on the way, on a tile that is in LDS.
  static __device__ __forceinline__ void clean(char* values, uint32_t (&bad)[(NL + 3) / 4]) {
    hq_u4v* vs = reinterpret_cast<hq_u4v*>(values) + threadIdx.x;
    hq_u4v v[NL];
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < NL; ++i) v[i] = vs[i * kThreads];
#pragma unroll
    for (int i = 0; i < NL; ++i)
#pragma unroll
      for (int w = 0; w < 4; ++w) any |= (v[i][w] & Kind<T>::kExp) + Kind<T>::kStep;
#pragma unroll
    for (int i = 0; i < (NL + 3) / 4; ++i) bad[i] = 0;
    if (!(any & 0x80008000u)) return;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t e = ((v[i][w] & Kind<T>::kExp) + Kind<T>::kStep) & 0x80008000u;
        bad[i / 4] |= ((e >> 15 & 1u) | (e >> 30 & 2u)) << (8 * (i % 4) + 2 * w);
        v[i][w] &= ~((e >> 15) * 0xffffu);
      }
      vs[i * kThreads] = v[i];
    }
  }

  // Into LDS.  In a tile that not every row sees whole, a value that is not finite would reach the rows that do not see it (0 times
  // infinity): it is stored as zero, and the bits returned say which values were.
  __device__ __forceinline__ void store(bool partly, uint32_t (&bad)[(NL + 3) / 4]) {
    const int ch = threadIdx.x % CH, row0 = threadIdx.x / CH;
    char* vs = sm + TILE * D * 2;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int row = row0 + i * STEP;
      *reinterpret_cast<hq_u4v*>(sm + row * D * 2 + k_piece(row, ch) * 16) = kr[i];
      if (partly) {
        if (i % 4 == 0) bad[i / 4] = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t e = ((vr[i][w] & Kind<T>::kExp) + Kind<T>::kStep) & 0x80008000u;
          if (e) {
            bad[i / 4] |= ((e >> 15 & 1u) | (e >> 30 & 2u)) << (8 * (i % 4) + 2 * w);
            vr[i][w] &= ~((e >> 15) * 0xffffu);
          }
        }
      }
      *reinterpret_cast<hq_u4v*>(vs + row * D * 2 + v_piece(row, ch) * 16) = vr[i];
    }
  }
  // The same places again, one for each value that was not finite and zero for the others.
  static __device__ __forceinline__ void store_bad(char* vs, const uint32_t (&bad)[(NL + 3) / 4]) {
    const int ch = threadIdx.x % CH, row0 = threadIdx.x / CH;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      hq_u4v w;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t b = bad[i / 4] >> (8 * (i % 4) + 2 * j);
        w[j] = (b & 1 ? Kind<T>::kOne & 0xffffu : 0u) | (b & 2 ? Kind<T>::kOne & 0xffff0000u : 0u);
      }
      if (DIRECT) {
        reinterpret_cast<hq_u4v*>(vs)[threadIdx.x + i * kThreads] = w;
      } else {
        const int row = row0 + i * STEP;
        *reinterpret_cast<hq_u4v*>(vs + row * D * 2 + v_piece(row, ch) * 16) = w;
      }
    }
  }

  // V^T of 32 elements of the head (block d) and 16 keys (block b, half t) as the matrix core takes it: see the top of the file.
  static __device__ __forceinline__ V8 v_operand(const char* values, int key0, int b, int t, int d) {
    const int lane = threadIdx.x & 63;
    const int row = key0 + 32 * b + 16 * t + 4 * (lane >> 5) + ((lane >> 2) & 3);
    const int ch = 4 * d + 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
    lds_char* vs = (lds_char*)values + (lane & 1) * 8;
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    union {
      s16x4 h[2];
      V8 v;
    } u;
    u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(vs + row * D * 2 + v_piece(row, ch) * 16));
    u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(vs + (row + 8) * D * 2 + v_piece(row + 8, ch) * 16));
    return u.v;
  }

  // The wave's part of a tile, step by step.  Scores of its rows and the keys from key0 on:
  __device__ __forceinline__ void scores(f32x16 (&s)[NB], const char* keys, int key0) const {
    const int lane = threadIdx.x & 63, half = lane >> 5;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[b][r] = 0.f;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const int row = key0 + 32 * b + (lane & 31);
        const V8 a = *reinterpret_cast<const V8*>(keys + row * D * 2 + k_piece(row, 2 * kk + half) * 16);
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
  // A maximum that has grown by less than 2^8 stays: the weights may then be up to 2^8, which neither fp32 sums nor the 16-bit
  // weights mind, and the sums need no scaling.  The scaling of 64 registers a tile was a fifth of the vector instructions.
  __device__ __forceinline__ void raise(float top) {
    if (!__builtin_amdgcn_ballot_w64(top > m + 8.f)) return;
    const float mn = top > m + 8.f ? top : m;  // each row by its own scores: its bits do not depend on its neighbours
    const float f = mn == m ? 1.f : __builtin_amdgcn_exp2f(m - mn);
    m = mn;
    l *= f;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] *= f;
  }
  __device__ __forceinline__ void weights(V8 (&p)[NB][2], const f32x16 (&s)[NB], float c) {
    const float ms = finite_or_zero(m);
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float e = __builtin_amdgcn_exp2f(fmaf(s[b][8 * t + i], c, -ms));
          sum[i & 1] += e;
          p[b][t][i] = (T)e;  // 2^-9 (bf16) or 2^-12 of a weight at most, to the nearest: as much as the result's own rounding
        }
    l += sum[0] + sum[1];
  }
  __device__ __forceinline__ void values(const V8 (&p)[NB][2], const char* values, int key0) {
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int t = 0; t < 2; ++t) o[d] = Kind<T>::mfma(v_operand(values, key0, b, t, d), p[b][t], o[d]);
  }
  // scores() of the next tile and weights() of this one, an instruction of the matrix core and its share of the others in turn: left
  // alone, the compiler moves the reads of all operands to the front and runs out of registers.
  __device__ __forceinline__ void scores_and_weights(f32x16 (&n)[NB], const char* keys, V8 (&p)[NB][2], const f32x16 (&s)[NB], float c) {
    const int lane = threadIdx.x & 63, half = lane >> 5;
    constexpr int STEPS = NB * D / 16, EACH = NB * 16 / STEPS, AHEAD = 4;
    auto operand = [&](int j) {
      const int row = 32 * (j / (D / 16)) + (lane & 31);
      return *reinterpret_cast<const V8*>(keys + row * D * 2 + k_piece(row, 2 * (j % (D / 16)) + half) * 16);
    };
    const float ms = finite_or_zero(m);
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
    auto operand = [&](int j) { return v_operand(vs, 0, j / 2 % NB, j % 2, j / (2 * NB)); };
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
  __device__ __forceinline__ void spoil(char* values, int key0, int left, const uint32_t (&bad)[(NL + 3) / 4]) {
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
          n = Kind<T>::mfma(v_operand(values, key0, b, t, d), seen, n);
        }
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] = n[r] > 0.f ? NAN : o[d][r];
    }
  }
  __device__ __forceinline__ bool spoiled(int tileno) const { return *(volatile __attribute__((address_space(3))) int*)poison == tileno; }
  __device__ __forceinline__ void note(const uint32_t (&bad)[(NL + 3) / 4], int tileno) {
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < (NL + 3) / 4; ++i) any |= bad[i];
    if (any) *poison = tileno;
  }

  // The row's sums as one of several shares; none: the row sees nothing in any of them, which share 0 says by an infinite maximum.
  __device__ __forceinline__ void put_share(float* po, float* pm, int64_t at, bool none) const {
    const int half = (threadIdx.x >> 5) & 1;
    if (m != -INFINITY)  // a share that no key went into is not read
#pragma unroll
      for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<hq_f4v*>(po + at * D + 32 * d + 8 * g + 4 * half) = hq_f4v{o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
    if (half == 0) *reinterpret_cast<float2*>(pm + 2 * at) = float2{none ? INFINITY : m, l};
  }

  // Keys [first, end) of src; whole: keys below it are seen by every row of the workgroup.
  template <typename SRC>
  __device__ __forceinline__ void run(const SRC& src, int first, int end, int whole, float c) {
    clear();
    if (first >= end) return;
    uint32_t bad[(NL + 3) / 4] = {};
    char* const vs = sm + TILE * D * 2;
    const int key0 = RW == 4 ? 0 : (threadIdx.x >> 6) * 32 * NB;
    load(src, first);
    for (int base = first, tileno = 0; base < end; base += TILE, ++tileno) {
      const bool partly = base + TILE > whole;
      __syncthreads();
      store(partly, bad);
      if (partly) note(bad, tileno);
      __syncthreads();
      if (base + TILE < end) load(src, base + TILE);
      const int left = lim - base - key0 - 4 * ((threadIdx.x >> 5) & 1);
      if (base + key0 < any_sees) {
        f32x16 s[NB];
        V8 p[NB][2];
        scores(s, sm, key0);
        if (base + key0 + 32 * NB > all_see) mask(s, left);
        raise(top_of(s) * c);
        weights(p, s, c);
        values(p, vs, key0);
      }
      if (partly && spoiled(tileno)) spoil(vs, key0, left, bad);
    }
    l = pair_sum(l);
  }

  // The same, DIRECT.  Heads of 128: the scores of the next tile are in the matrix core while the vector unit makes this one's weights
  // of its own, and the next scores' maximum is taken under this tile's product with the values; the keys so run a tile ahead.  Heads
  // of 64, where the vector unit is the busier of the two and the registers saved are two waves more: one step after the other
  // (16384 tokens, heads of 128: 2186 us one after the other, 2130 so; 8192 tokens, heads of 64: 359 and 376).
  template <typename SRC>
  __device__ __forceinline__ void run_direct(const SRC& src, int first, int end, int whole, float c) {
    clear();
    if (first >= end) return;
    constexpr int HALF = TILE * D * 2, K_AHEAD = D == 128;
    const int nt = (end - first + TILE - 1) / TILE;
    direct_offsets(koff, (int)src.ks, src.n - first, [](int row, int ch) { return k_piece(row, ch); });
    direct_offsets(voff, (int)src.vs, src.n - first, [](int row, int ch) { return v_piece(row, ch); });
    auto load_k = [&](int t, int slot) {
      const int base = first + t * TILE;
      if (base + TILE > src.n) direct_offsets(koff, (int)src.ks, src.n - base, [](int row, int ch) { return k_piece(row, ch); });
      direct_load(src.k + base * src.ks, koff, sm + slot * HALF);
    };
    auto load_v = [&](int t, int slot) {
      const int base = first + t * TILE;
      if (base + TILE > src.n) direct_offsets(voff, (int)src.vs, src.n - base, [](int row, int ch) { return v_piece(row, ch); });
      direct_load(src.v + base * src.vs, voff, sm + (2 + slot) * HALF);
    };
    const int half4 = 4 * ((threadIdx.x >> 5) & 1);
    f32x16 s0[NB], s1[NB];
    float top = 0.f;
    load_k(0, 0);
    load_v(0, 0);
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) asm volatile("" : "+v"(qf[kk]));  // here, not at every tile: the loads in flight then are the next tile's
    if (K_AHEAD) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (nt > 1) load_k(1, 1);
      scores(s0, sm, 0);
      if (first + TILE > all_see) mask(s0, lim - first - half4);
      top = top_of(s0);
    }
    // One tile.  K_AHEAD: its scores in s, the next one's go to n (behind the last tile they are of no tile, and not used: one way
    // through the step, as two ways that both sum into o cost the compiler a second set of its registers).
    auto step = [&](int t, auto SLOT, f32x16(&s)[NB], f32x16(&n)[NB]) __attribute__((always_inline)) {
      const int base = first + t * TILE;
      const bool partly = base + TILE > whole;
      char* const vs = sm + (2 + SLOT) * HALF;
      uint32_t bad[(NL + 3) / 4] = {};
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (t + 1 + K_AHEAD < nt) load_k(t + 1 + K_AHEAD, (SLOT + 1 + K_AHEAD) % 2);
      if (t + 1 < nt) load_v(t + 1, 1 - SLOT);
      if (partly) {
        clean(vs, bad);
        note(bad, t);
        __syncthreads();
      }
      if (base < any_sees) {
        V8 p[NB][2];
        if (K_AHEAD) {
          raise(top * c);
          scores_and_weights(n, sm + (1 - SLOT) * HALF, p, s, c);
          if (base + 2 * TILE > all_see) mask(n, lim - base - TILE - half4);
          top = values_and_top(p, vs, n);
        } else {
          scores(s, sm + SLOT * HALF, 0);
          if (base + TILE > all_see) mask(s, lim - base - half4);
          raise(top_of(s) * c);
          weights(p, s, c);
          values(p, vs, 0);
        }
      }
      if (partly && spoiled(t)) spoil(vs, 0, lim - base - half4, bad);
    };
    if (K_AHEAD) {
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
};

// Sets up the poison word; a barrier of run() lies between this and its first use.
__device__ __forceinline__ void set_up(int* poison) {
  if (threadIdx.x == 0) *poison = -1;
}

// Item x of a list in which entry i, bounds[i] to bounds[i + 1], cut to 0 ... most, has tiles(its length) tiles: the entry, its begin and
// length, and which of its tiles.  A wave looks at 64 entries at a time.
template <typename F>
__device__ __forceinline__ bool find_tile(const int* bounds, int n, int most, int x, F tiles, int* entry, int* begin, int* length, int* which) {
  const int lane = threadIdx.x & 63;
  for (int i0 = 0; i0 < n; i0 += 64) {
    const int i = i0 + lane;
    const int b = i < n ? min(max(bounds[i], 0), most) : 0, len = i < n ? min(max(bounds[i + 1], b), most) - b : 0;
    const int t = tiles(len);
    int sum = t;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int u = __shfl_up(sum, d);
      if (lane >= d) sum += u;
    }
    const int total = __builtin_amdgcn_readlane(sum, 63);
    if (x < total) {
      const int at = __ffsll(__ballot(sum > x)) - 1;
      *entry = i0 + at;
      *begin = __builtin_amdgcn_readlane(b, at);
      *length = __builtin_amdgcn_readlane(len, at);
      *which = x - __builtin_amdgcn_readlane(sum - t, at);
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

template <typename T>
struct PackedKeys {  // of one sequence and one head
  const T *k, *v;
  int64_t ks, vs;
  int n;
  __device__ __forceinline__ bool at(int key, const T** kp, const T** vp) const {
    key = min(key, n - 1);
    *kp = k + key * ks;
    *vp = v + key * vs;
    return true;
  }
};

// A workgroup's rows and share of the keys.  Many rows: all keys, and the result; few: the keys are divided among `shares` workgroups.
template <typename T, int D>
__global__ __launch_bounds__(kThreads, D == 64 ? 4 : 2) void prompt_kernel(PromptArgs a) {
  typedef Attend<T, D, 4, true> A;
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
  int seq, tile, q0, nq;
  if (!find_tile(a.cu_q, a.seqs, a.total_q, x, [=](int n) { return (int)((n * ratio + ROWS - 1) / ROWS); }, &seq, &q0, &nq, &tile)) return;
  const int k0 = min(max(a.cu_k[seq], 0), a.total_k), nk = min(max(a.cu_k[seq + 1], k0), a.total_k) - k0;
  const int rows = nq * ratio;
  tile = (rows + ROWS - 1) / ROWS - 1 - tile;  // the tiles with most keys come first
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
  PackedKeys<T> src{(const T*)a.k + (int64_t)k0 * a.ks + head * D, (const T*)a.v + (int64_t)k0 * a.vs + head * D, a.ks, a.vs, nk};
  const int each = a.shares == 1 ? nk : max(256, ((nk + a.shares - 1) / a.shares + A::TILE - 1) & -A::TILE);
  const int end = uniform(limit((uint32_t)last_row / ratio)), first = (int)min((int64_t)share * each, (int64_t)end);
  w.run_direct(src, first, min(end, first + each), uniform(limit((uint32_t)first_row / ratio)), a.c);
  if (row > last_row) return;
  if (a.shares == 1) {
    const float inv = 1.f / w.l;
    T* out = (T*)a.out + ((int64_t)(q0 + token) * a.heads + h) * D + 4 * (lane >> 5);
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        typedef T T4 __attribute__((ext_vector_type(4)));
        T4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (T)(w.lim == 0 ? 0.f : w.o[d][4 * g + i] * inv);  // a token that sees no key
        *reinterpret_cast<T4*>(out + 32 * d + 8 * g) = v;
      }
  } else {
    w.put_share(a.po, a.pm, ((int64_t)(q0 + token) * a.heads + h) * a.shares + share, w.lim == 0);
  }
}

// ---- one query a request, over pages -----------------------------------------------------------------------------------
struct PagedArgs {
  const void *q, *k, *v;
  void* out;
  const int *table, *lengths, *groups, *shared;
  float *po, *pm;      // partial sums [batch * heads][slots][D], and {maximum, sum} [batch * heads][slots]
  int64_t qs;
  int ngroups, batch, width, pages, page_log, heads, kv_heads, ratio;
  int np, ns;          // shares that a group's common keys, and a request's own, are divided into
  int prefix_items;    // workgroups of the common keys
  float c;
};

template <typename T, int D>
struct PagedKeys {
  const T *k, *v;
  const int* pages_of;  // the row of the table
  int head, kv_heads, page_log, pages, n;
  __device__ __forceinline__ bool at(int key, const T** kp, const T** vp) const {
    key = min(key, n - 1);
    const int page = pages_of[key >> page_log], p = (unsigned)page < (unsigned)pages ? page : 0;
    const int64_t off = ((((int64_t)p * kv_heads + head) << page_log) + (key & ((1 << page_log) - 1))) * D;
    *kp = k + off;
    *vp = v + off;
    return p == page;
  }
};

// Tokens that the requests of group g have in common: those of the first one's row that the caller says are.
__device__ __forceinline__ int shared_tokens(const PagedArgs& a, int g) {
  const int first = min(max(a.groups[g], 0), a.batch - 1);
  return min(min(max(a.shared[g], 0), max(a.lengths[first], 0)), a.width << a.page_log);
}

// Keys of share s of n, as many as make `shares` shares of whole tiles of 128, 256 at least.
__device__ __forceinline__ void share_of(int n, int shares, int s, int* first, int* end) {
  int each = (n + shares - 1) / shares;
  each = max(256, (each + 127) & ~127);
  *first = min((int64_t)s * each, (int64_t)n);
  *end = min(*first + each, n);
}

template <typename T, int D, int RW>
__device__ __forceinline__ void attend_rows(const PagedArgs& a, char* sm, int* poison, int b0, int nrows, int first_row, int head, int src_row,
                                            int first, int end, int shared_end, int slot) {
  typedef Attend<T, D, RW> A;
  typedef typename Kind<T>::V8 V8;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int slots = a.np + a.ns;
  const int last_row = min(first_row + 32 * RW, nrows) - 1;
  const int row = first_row + (RW == 4 ? wave * 32 : 0) + (lane & 31), r = min(row, last_row);
  const int b = b0 + r / a.ratio, h = head * a.ratio + r % a.ratio;
  A w;
  w.sm = sm;
  w.poison = poison;
  const T* q = (const T*)a.q + (int64_t)b * a.qs + (int64_t)h * D + 8 * (lane >> 5);
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) w.qf[kk] = *reinterpret_cast<const V8*>(q + 16 * kk);
  w.lim = min(min(max(a.lengths[b], 0), a.width << a.page_log), shared_end);
  w.all_see = uniform(wave_min(w.lim));
  w.any_sees = -uniform(wave_min(-w.lim));
  // what every row of the workgroup sees
  __shared__ int seen[kWaves];
  if (lane == 0) seen[wave] = w.all_see;
  __syncthreads();
  const int whole = min(min(seen[0], seen[1]), min(seen[2], seen[3]));
  PagedKeys<T, D> src{(const T*)a.k, (const T*)a.v, a.table + (int64_t)src_row * a.width, head, a.kv_heads, a.page_log, a.pages, end};
  w.run(src, first, end, whole, a.c);
  const int64_t at = ((int64_t)b * a.heads + h) * slots + slot;
  if (RW == 1) {  // the four waves' sums come together
    float* sum = reinterpret_cast<float*>(sm);          // [wave][D][32]
    __shared__ float top[kWaves][32], total[kWaves][32];
    __syncthreads();
    if (lane < 32) top[wave][lane] = w.m;
    __syncthreads();
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) m = fmaxf(m, top[i][lane & 31]);
    const float f = __builtin_amdgcn_exp2f(w.m - finite_or_zero(m));
    if (lane < 32) total[wave][lane] = w.l * f;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        sum[(wave * D + 32 * d + 8 * (i / 4) + 4 * (lane >> 5) + i % 4) * 32 + (lane & 31)] = w.o[d][i] * f;
    __syncthreads();
    float all = 0.f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) all += total[i][lane & 31];
    if (row > last_row) return;
    const int part = threadIdx.x >> 5;  // eight parts of the head
    if (slots == 1) {
      T* out = (T*)a.out + ((int64_t)b * a.heads + h) * D;
      const float inv = 1.f / all;
      for (int d = part * (D / 8); d < (part + 1) * (D / 8); ++d) {
        float v = 0.f;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) v += sum[(i * D + d) * 32 + (lane & 31)];
        out[d] = (T)(w.lim <= 0 ? 0.f : v * inv);
      }
    } else {
      for (int d = part * (D / 8); d < (part + 1) * (D / 8); ++d) {
        float v = 0.f;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) v += sum[(i * D + d) * 32 + (lane & 31)];
        a.po[at * D + d] = v;
      }
      if (part == 0) {
        a.pm[2 * at] = m;
        a.pm[2 * at + 1] = all;
      }
    }
  } else {
    if (row <= last_row) w.put_share(a.po, a.pm, at, false);
  }
}

template <typename T, int D>
__global__ __launch_bounds__(kThreads, 2) void paged_kernel(PagedArgs a) {
  extern __shared__ __align__(16) char sm[];
  __shared__ int poison;
  set_up(&poison);
  int x = blockIdx.x;
  if (x < a.prefix_items) {
    const int head = x % a.kv_heads;
    x /= a.kv_heads;
    const int share = x % a.np;
    int g, tile, b0, nb;
    const int ratio = a.ratio;
    if (!find_tile(a.groups, a.ngroups, a.batch, x / a.np, [=](int n) { return (int)((n * (int64_t)ratio + 127) / 128); }, &g, &b0, &nb, &tile)) return;
    const int n = shared_tokens(a, g);
    int first, end;
    share_of(n, a.np, share, &first, &end);
    if (nb * ratio <= 32)
      attend_rows<T, D, 1>(a, sm, &poison, b0, nb * ratio, 0, head, b0, first, end, n, share);
    else
      attend_rows<T, D, 4>(a, sm, &poison, b0, nb * ratio, tile * 128, head, b0, first, end, n, share);
  } else {
    x -= a.prefix_items;
    const int head = x % a.kv_heads;
    x /= a.kv_heads;
    const int share = x % a.ns, tiles = (a.ratio + 31) / 32;
    const int tile = x / a.ns % tiles, b = x / a.ns / tiles;
    int from = 0;
    for (int g = 0; g < a.ngroups; ++g)
      if (b >= a.groups[g] && b < a.groups[g + 1]) from = shared_tokens(a, g);
    const int n = min(max(a.lengths[b], 0), a.width << a.page_log);
    from = min(from, n);
    int first, end;
    share_of(n - from, a.ns, share, &first, &end);
    attend_rows<T, D, 1>(a, sm, &poison, b, a.ratio, tile * 32, head, b, from + first, from + end, INT_MAX, a.np + share);
  }
}

// The shares of a row together, one wave a row: their maxima and sums a lane each, then the sums of the values, 16 bytes a lane,
// several shares at a time.  first: shares before it were not written.
template <typename T, int D>
__device__ __forceinline__ void join_shares(const float* po, const float* pm, int64_t row, int first, int slots, bool none, T* out) {
  constexpr int LANES = D / 4, AT_ONCE = 64 / LANES;  // lanes of a share, shares of a load
  const int lane = threadIdx.x & 63, d = (lane % LANES) * 4;
  const float2* ml = reinterpret_cast<const float2*>(pm) + row * slots;
  float m = -INFINITY;
  for (int s = first + lane; s < slots; s += 64) m = fmaxf(m, ml[s].x);
  m = hq_wave_max(m);
  const float ms = finite_or_zero(m);
  float l = 0.f;
  hq_f4v o = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = first; s0 < slots; s0 += 64) {
    const int s = s0 + lane;
    const float2 mine = s < slots ? ml[s] : float2{-INFINITY, 0.f};
    const float f = __builtin_amdgcn_exp2f(mine.x - ms);
    l += mine.y * f;
    const int n = min(slots - s0, 64);
#pragma unroll 4
    for (int i = 0; i < n; i += AT_ONCE) {
      const int at = i + lane / LANES;
      const float w = __shfl(f, at & 63);
      if (at < n && w != 0.f) o += *reinterpret_cast<const hq_f4v*>(po + (row * slots + s0 + at) * D + d) * w;
    }
  }
  l = hq_wave_sum(l);
#pragma unroll
  for (int x = LANES; x < 64; x <<= 1)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] += __shfl_xor(o[i], x);
  if (lane < LANES) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    T4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (T)(none ? 0.f : o[i] / l);
    *reinterpret_cast<T4*>(out + row * D + d) = v;
  }
}

template <typename T, int D>
__global__ __launch_bounds__(kThreads) void join_paged_kernel(PagedArgs a) {
  const int64_t row = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (row >= (int64_t)a.batch * a.heads) return;
  const int b = row / a.heads;
  bool grouped = false;
  for (int g = 0; g < a.ngroups; ++g) grouped |= b >= a.groups[g] && b < a.groups[g + 1];
  // nobody wrote the common shares of a request without a group
  join_shares<T, D>(a.po, a.pm, row, grouped ? 0 : a.np, a.np + a.ns, a.lengths[b] <= 0, (T*)a.out);
}

template <typename T, int D>
__global__ __launch_bounds__(kThreads) void join_prompt_kernel(PromptArgs a) {
  const int64_t row = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (row >= (int64_t)a.total_q * a.heads) return;
  const int token = row / a.heads;
  if (token < a.cu_q[0] || token >= a.cu_q[a.seqs]) return;
  const float2 first = reinterpret_cast<const float2*>(a.pm)[row * a.shares];
  join_shares<T, D>(a.po, a.pm, row, 0, a.shares, first.x == INFINITY && first.y == 0.f, (T*)a.out);
}

// Scores are compared and masked by -infinity before they are scaled: a scale of zero (all keys alike) becomes one that no score notices.
float exponent_scale(float s) { return s * 1.44269504088896340736f > 1e-30f ? s * 1.44269504088896340736f : 1e-30f; }
bool bad_scale(float s) { return !(s >= 0.f) || std::isinf(s); }
bool misaligned(const void* p, int64_t stride) { return ((uintptr_t)p & 15) || stride % 8; }

// Few rows leave compute units idle, and each of their workgroups with all keys: then the keys are divided, so that there are up to
// two workgroups a compute unit, each with 256 keys at least.
template <typename T, int D>
int launch_prompt(PromptArgs a, int cus, hipStream_t stream) {
  const int64_t items = ((int64_t)a.total_q * a.ratio / 128 + a.seqs) * a.kv_heads;
  const int64_t want = 2 * (int64_t)cus / items, most = ((int64_t)a.total_k + 255) / 256;
  a.shares = (int)std::max<int64_t>(1, std::min(want, most));
  if (items * a.shares > INT_MAX) return HQ_ERR_TOO_LARGE;
  const int64_t rows = (int64_t)a.total_q * a.heads;
  if (a.shares > 1) {
    HqWorkspace ws;
    const int rc = hq_get_workspace(stream, (size_t)(rows * a.shares * (D + 2)), 0, &ws);
    if (rc != HQ_OK) return rc;
    a.po = ws.partial;
    a.pm = ws.partial + rows * a.shares * D;
  }
  const int rc = hq_launch_as_is(prompt_kernel<T, D>, dim3((unsigned)(items * a.shares)), dim3(kThreads), Attend<T, D, 4, true>::LDS, stream, a);
  if (rc != HQ_OK || a.shares == 1) return rc;
  return hq_launch_as_is(join_prompt_kernel<T, D>, dim3((unsigned)((rows + kWaves - 1) / kWaves)), dim3(kThreads), 0, stream, a);
}

template <typename T, int D>
int launch_paged(PagedArgs a, int cus, hipStream_t stream) {
  const int64_t cap = (int64_t)a.width << a.page_log, most = (cap + 255) / 256;
  const int tiles = (a.ratio + 31) / 32;
  const int64_t own = (int64_t)a.batch * a.kv_heads * tiles, row_tiles = (int64_t)a.batch * a.ratio / 128 + a.ngroups;
  auto shares = [&](int64_t items) {
    const int64_t want = (2 * (int64_t)cus + items - 1) / items;
    return (int)(want < most ? (want < 1 ? 1 : want) : (most < 1 ? 1 : most));
  };
  a.ns = shares(own);
  a.np = a.ngroups ? shares(row_tiles * a.kv_heads) : 0;
  const int64_t prefix = a.ngroups ? row_tiles * a.kv_heads * a.np : 0, grid = prefix + own * a.ns;
  if (grid > INT_MAX) return HQ_ERR_TOO_LARGE;
  a.prefix_items = (int)prefix;
  const int64_t slots = a.np + a.ns, rows = (int64_t)a.batch * a.heads;
  if (slots > 1) {
    HqWorkspace ws;
    const int rc = hq_get_workspace(stream, (size_t)rows * slots * (D + 2), 0, &ws);
    if (rc != HQ_OK) return rc;
    a.po = ws.partial;
    a.pm = ws.partial + rows * slots * D;
  }
  constexpr int lds = Attend<T, D, 1>::LDS > Attend<T, D, 4>::LDS ? Attend<T, D, 1>::LDS : Attend<T, D, 4>::LDS;
  constexpr int sums = kWaves * D * 32 * 4, most_lds = lds > sums ? lds : sums;
  static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(&paged_kernel<T, D>),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, most_lds);
  if (attr != hipSuccess) return (int)attr;
  int rc = hq_launch_as_is(paged_kernel<T, D>, dim3((unsigned)grid), dim3(kThreads), most_lds, stream, a);
  if (rc != HQ_OK || slots == 1) return rc;
  return hq_launch_as_is(join_paged_kernel<T, D>, dim3((unsigned)((rows + kWaves - 1) / kWaves)), dim3(kThreads), 0, stream, a);
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
  if (total_q * (heads / kv_heads) > INT_MAX - 128 || total_k > INT_MAX - 128 || k_stride > 1 << 22 || v_stride > 1 << 22)  // 32-bit offsets in a tile
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
  if (!q || !out || !lengths || (table_width && (!table || num_pages == 0 || !k_pages || !v_pages)) || (ngroups && (!groups || !shared)))
    return HQ_ERR_NULL_POINTER;
  if (q_stride < (int64_t)heads * head_dim) return HQ_ERR_BAD_SHAPE;
  if (misaligned(q, q_stride) || (((uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)out) & 15) ||
      (((uintptr_t)table | (uintptr_t)lengths | (uintptr_t)groups | (uintptr_t)shared) & 3))
    return HQ_ERR_MISALIGNED;
  if ((int64_t)table_width * page_size > INT_MAX - 256 || (int64_t)batch * heads > INT_MAX / 64) return HQ_ERR_TOO_LARGE;
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
