// Heads of queries and keys normed and rotated by their tokens' positions, to where the caller says or, the keys, into the pages of the
// cache, with the values.
//
// A head x of D elements: y = x * rsqrt(mean(x^2) + eps) * weight, and every pair (a, b) of the first `rotary` elements of y becomes
// (a c - b s, b c + a s), c and s the cosine and sine of the pair's angle at the token's position.  One pass in fp32, one rounding.
//
// A lane holds two pieces of eight elements of a head, those that are rotated against each other, so that nothing but the sum of
// the squares goes from lane to lane: D / 16 lanes a head, 64 * 16 / D heads of a token a wave, which are queries, keys or values (of several
// sets of heads one after the other, whose cosines and sines would be read once: 62.0 us with two, 64.3 with three where 60.9 here), in the
// order of memory (a token's sets in workgroups far from each other: 78 us).  Memory sees whole heads all the same, half of the wave's an instruction
// (exchange): stores of a lane's own two pieces are of half lines wherever they are not halves of a head of 128, and cost 16384 tokens of
// 32 / 8 heads of 64 34.3 us by way of the L2, which puts them together, where it is 29.7 here, and with 64 of 128 elements rotated, past the L2,
// 108 where it is 55.8.  Bound by the copy: of heads of 128 56.0 us, 6.1 TB/s of data, where a plain copy of 512 MB reaches 6.5; short calls by
// the launch and the loads that wait for another (positions, then the table's row; in the cache's form bounds and starts, then the table's
// row and the page): one token 4.4 us.
#include <algorithm>
#include <climits>
#include <cmath>

#include "hq_internal.h"

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;

struct RotateArgs {
  const hq_u4v *q, *k, *v;
  hq_u4v *qo, *ko, *vo;  // of the cache's form: ko and vo its pages
  const hq_u4v *qw, *kw; // null: no norm
  const hq_f4v* cs;      // [positions][rotary]: cosines, sines
  const int *positions;  // of the plain form
  const int *table, *starts, *cu;
  int64_t qs, ks, vs, qos, kos;  // 16-byte pieces from one token to the next
  int tokens, heads, kv_heads, rotary, known;  // known: positions of cs
  int rows, width, pages, page_log, interleaved;
  float eps;
  int q_sets, k_sets;          // sets of heads
  unsigned sets, reciprocal;   // of a token, all, two at least; 2^32 / sets, rounded up
};

template <typename T>
__device__ __forceinline__ void wide(float (&x)[8], hq_u4v v) {
  typedef T T8 __attribute__((ext_vector_type(8)));
  const T8 t = __builtin_bit_cast(T8, v);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (float)t[i];
}
template <typename T>
__device__ __forceinline__ hq_u4v narrow(const float (&x)[8]) {
  typedef T T8 __attribute__((ext_vector_type(8)));
  T8 t;
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = (T)x[i];
  return __builtin_bit_cast(hq_u4v, t);
}
// Sum over the lanes of a head.
template <int LANES>
__device__ __forceinline__ float head_sum(float v) {
  v = hq_quad(v, HqAdd());
  return LANES == 8 ? v + hq_dpp<0x141>(v) : v;  // row_half_mirror
}

// The upper lanes' first pieces against the lower lanes' second ones: what were two pieces of every lane is then the lower lanes' heads, whole, in one
// register and the upper lanes' in the other; and back.
__device__ __forceinline__ void exchange(hq_u4v& a, hq_u4v& b) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const auto s = __builtin_amdgcn_permlane32_swap(a[i], b[i], false, false);
    a[i] = s[0];
    b[i] = s[1];
  }
}

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

// A wave takes a set of a token's heads: of queries, of keys, or of values.
template <typename T, int D, bool CACHE>
__global__ __launch_bounds__(kThreads) void rotate_kernel(RotateArgs a) {
  constexpr int LANES = D / 16, HEADS = 64 / LANES, CH = D / 8;
  const unsigned wave = __builtin_amdgcn_readfirstlane(blockIdx.x * kWaves + (threadIdx.x >> 6));
  unsigned token = __umulhi(wave, a.reciprocal);  // or one more
  if (token * a.sets > wave) --token;
  const int t = token, set = wave - token * a.sets;
  if (t >= a.tokens) return;
  const int lane = threadIdx.x & 63, l = lane % LANES, np = a.rotary / 16;
  const int pa = l < np ? l : 2 * l, pb = l < np ? l + np : 2 * l + 1;
  const bool query = set < a.q_sets, key = !query && (!CACHE || set < a.q_sets + a.k_sets);
  const int heads = query ? a.heads : a.kv_heads, piece = lane < 32 ? pa : pb;
  const int h = (set - (query ? 0 : key ? a.q_sets : a.q_sets + a.k_sets)) * HEADS + (lane & 31) / LANES, h2 = h + HEADS / 2;
  const hq_u4v* const from = (query ? a.q + t * a.qs : key ? a.k + t * a.ks : a.v + t * a.vs) + piece;
  const hq_u4v* const weight = query ? a.qw : key ? a.kw : nullptr;
  hq_u4v xa = from[min(h, heads - 1) * CH], xb = from[min(h2, heads - 1) * CH], wa = {}, wb = {};
  if (weight) {
    wa = weight[pa];
    wb = weight[pb];
  }
  int row = 0;
  int64_t place;
  if (CACHE) {
    row = find_row(a.cu, a.rows, t);
    if (row >= a.rows || t < a.cu[row]) return;
    place = (int64_t)a.starts[row] + (t - a.cu[row]);
  } else {
    place = a.rotary ? a.positions[t] : 0;
  }
  const bool rotated = l < np;
  float cs[8] = {}, sn[8] = {};  // of the lane's pairs, if they are rotated
  if (rotated && (query || key)) {
    const int at = (int)min(max(place, (int64_t)0), (int64_t)a.known - 1);
    const hq_f4v* const c = a.cs + (int64_t)at * (a.rotary / 4);
    const int i0 = a.interleaved ? l : 2 * l, i1 = a.interleaved ? l + np : 2 * l + 1, sines = a.rotary / 8;
    const hq_f4v c0 = c[i0], c1 = c[i1], s0 = c[sines + i0], s1 = c[sines + i1];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      cs[i] = c0[i];
      cs[4 + i] = c1[i];
      sn[i] = s0[i];
      sn[4 + i] = s1[i];
    }
  }
  hq_u4v* to;  // of the token's head 0
  int step = CH;
  bool there = true;
  if (query) {
    to = a.qo + t * a.qos;
  } else if (CACHE) {
    const bool within = place >= 0 && place < (int64_t)a.width << a.page_log;
    const int page = within ? a.table[(int64_t)row * a.width + (place >> a.page_log)] : -1;
    there = (unsigned)page < (unsigned)a.pages;
    to = (key ? a.ko : a.vo) + (((int64_t)page * a.kv_heads << a.page_log) + (place & ((1 << a.page_log) - 1))) * CH;
    step <<= a.page_log;
  } else {
    to = a.ko + t * a.kos;
  }
  if (query || key) {
    float u[8], v[8];
    exchange(xa, xb);
    wide<T>(u, xa);
    wide<T>(v, xb);
    if (weight) {
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(u[j], u[j], fmaf(v[j], v[j], ss));
      ss = head_sum<LANES>(ss);
      float r = rsqrtf(fmaf(ss, 1.f / D, a.eps));
      if (__builtin_expect(!(ss < INFINITY), 0)) {  // bf16 holds numbers whose squares fp32 does not
        constexpr float down = 0x1p-70f;
        ss = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          u[j] *= down;
          v[j] *= down;
          ss = fmaf(u[j], u[j], fmaf(v[j], v[j], ss));
        }
        r = rsqrtf(fmaf(head_sum<LANES>(ss), 1.f / D, a.eps * down * down));
      }
      float wu[8], wv[8];
      wide<T>(wu, wa);
      wide<T>(wv, wb);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        u[j] = u[j] * r * wu[j];  // in this order: u r is sqrt(D) at most, r w has no bound
        v[j] = v[j] * r * wv[j];
      }
    }
    // The others are left out of it: turned by an angle of 0, they would take 0 times what is beside them, NaN where that is not finite, and
    // lose the sign of a zero.
    if (rotated && a.interleaved) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float u0 = u[2 * j], v0 = v[2 * j];
        u[2 * j] = u0 * cs[j] - u[2 * j + 1] * sn[j];
        u[2 * j + 1] = u[2 * j + 1] * cs[j] + u0 * sn[j];
        v[2 * j] = v0 * cs[4 + j] - v[2 * j + 1] * sn[4 + j];
        v[2 * j + 1] = v[2 * j + 1] * cs[4 + j] + v0 * sn[4 + j];
      }
    } else if (rotated) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float u0 = u[j];
        u[j] = u0 * cs[j] - v[j] * sn[j];
        v[j] = v[j] * cs[j] + u0 * sn[j];
      }
    }
    xa = narrow<T>(u);
    xb = narrow<T>(v);
    exchange(xa, xb);
  }
  if (!there) return;
  to += piece;  // whole lines, past the L2 (by way of it 32.3 us and 60.0 where these are 29.7 and 56.0)
  if (h < heads) hq_store_stream(to + (int64_t)h * step, xa);
  if (h2 < heads) hq_store_stream(to + (int64_t)h2 * step, xb);
}

template <typename T, int D, bool CACHE>
int launch_rotate(RotateArgs a, hipStream_t stream) {
  constexpr int HEADS = 64 * 16 / D;
  a.q_sets = (a.heads + HEADS - 1) / HEADS;
  a.k_sets = (a.kv_heads + HEADS - 1) / HEADS;
  a.sets = a.q_sets + (CACHE ? 2 : 1) * a.k_sets;
  a.reciprocal = (unsigned)(((1ull << 32) + a.sets - 1) / a.sets);
  const uint64_t blocks = ((uint64_t)a.tokens * a.sets + kWaves - 1) / kWaves;
  if (blocks > UINT32_MAX / kThreads) return HQ_ERR_TOO_LARGE;  // threads are numbered in 32 bits
  return hq_launch_as_is(rotate_kernel<T, D, CACHE>, dim3((unsigned)blocks), dim3(kThreads), 0, stream, a);
}
#define HQ_BY_TYPE(cache)                                                                                                        \
  (dtype == HQ_DTYPE_F16 ? (head_dim == 64 ? launch_rotate<_Float16, 64, cache>(a, s) : launch_rotate<_Float16, 128, cache>(a, s)) \
                         : (head_dim == 64 ? launch_rotate<__bf16, 64, cache>(a, s) : launch_rotate<__bf16, 128, cache>(a, s)))

// Rows of `bytes` bytes each, `stride` bytes apart.  Two of them meet nowhere, or (same) are the same rows.
struct Region {
  const void* p;
  int64_t bytes, stride;
};
bool apart(const Region& x, const Region& y, int64_t tokens, bool same) {
  const uintptr_t a = (uintptr_t)x.p, b = (uintptr_t)y.p;
  if (same && a == b && (x.stride == y.stride || tokens == 1) && x.bytes == y.bytes) return true;
  const uint64_t ax = (uint64_t)(tokens - 1) * x.stride + x.bytes, by = (uint64_t)(tokens - 1) * y.stride + y.bytes;
  if (a + ax <= b || b + by <= a) return true;
  if (x.stride != y.stride) return false;  // (one inside the other's gaps, by chance: refused)
  // columns of one wide row: where y's first begins behind one of x's
  const uint64_t d = (b >= a ? b - a : (uint64_t)x.stride - (a - b) % (uint64_t)x.stride) % (uint64_t)x.stride;
  return d >= (uint64_t)x.bytes && d + (uint64_t)y.bytes <= (uint64_t)x.stride;
}

// One stretch of memory; apart from another, or from rows, of which what lies in the gaps between them is apart too.
struct Stretch {
  const void* p;
  int64_t bytes;
};
bool apart(const Stretch& x, const Stretch& y) {
  const uintptr_t a = (uintptr_t)x.p, b = (uintptr_t)y.p;
  return !x.p || !y.p || x.bytes <= 0 || y.bytes <= 0 || a + x.bytes <= b || b + y.bytes <= a;
}
bool apart(const Region& x, int64_t tokens, const Stretch& y) {
  if (apart(Stretch{x.p, (tokens - 1) * x.stride + x.bytes}, y)) return true;
  if ((uintptr_t)y.p < (uintptr_t)x.p) return false;
  const int64_t d = (int64_t)(((uintptr_t)y.p - (uintptr_t)x.p) % (uint64_t)x.stride);
  return d >= x.bytes && y.bytes <= x.stride - d;
}
// Bytes of the pages, as far as any memory reaches.
int64_t bytes_of_pages(int pages, int heads, int page, int head_dim) {
  return (int64_t)std::min((double)(1ll << 60), 2.0 * pages * heads * page * head_dim);
}

int check(int dtype, int head_dim, int rotary, int num_positions, const float* cos_sin, int64_t tokens, int heads, int kv_heads, bool normed, float eps) {
  if (tokens < 0 || heads < 1 || kv_heads < 1 || num_positions < 0 || rotary < 0 || rotary % 16 || rotary > head_dim) return HQ_ERR_BAD_SHAPE;
  if (head_dim != 64 && head_dim != 128) return HQ_ERR_BAD_SHAPE;
  if (dtype != HQ_DTYPE_F16 && dtype != HQ_DTYPE_BF16) return HQ_ERR_BAD_ENUM;
  if (normed && (!(eps >= 0x1p-126f) || std::isinf(eps))) return HQ_ERR_BAD_SHAPE;
  if (rotary && num_positions == 0 && tokens) return HQ_ERR_BAD_SHAPE;
  if (rotary && tokens && !cos_sin) return HQ_ERR_NULL_POINTER;
  if (tokens > INT_MAX || heads > 1 << 16 || kv_heads > 1 << 16) return HQ_ERR_TOO_LARGE;
  return HQ_OK;
}
bool odd(const void* p, int64_t stride) { return ((uintptr_t)p & 15) || stride % 8; }

}  // namespace

extern "C" int hq_norm_rotate(const void* q, const void* k, void* q_out, void* k_out, int dtype, const void* q_weight, const void* k_weight,
                              const float* cos_sin, const int32_t* positions, int64_t tokens, int heads, int kv_heads, int head_dim, int rotary,
                              int num_positions, int64_t q_stride, int64_t k_stride, int64_t q_out_stride, int64_t k_out_stride, float eps,
                              int interleaved, void* stream) {
  const int rc = check(dtype, head_dim, rotary, num_positions, cos_sin, tokens, heads, kv_heads, q_weight || k_weight, eps);
  if (rc != HQ_OK) return rc;
  if (tokens == 0) return HQ_OK;
  if (!q || !k || !q_out || !k_out || (rotary && !positions)) return HQ_ERR_NULL_POINTER;
  const int64_t qn = (int64_t)heads * head_dim, kn = (int64_t)kv_heads * head_dim;
  if (q_stride < qn || q_out_stride < qn || k_stride < kn || k_out_stride < kn) return HQ_ERR_BAD_SHAPE;
  if (odd(q, q_stride) || odd(k, k_stride) || odd(q_out, q_out_stride) || odd(k_out, k_out_stride) || odd(q_weight, 0) || odd(k_weight, 0) ||
      odd(cos_sin, 0) || ((uintptr_t)positions & 3))
    return HQ_ERR_MISALIGNED;
  constexpr int64_t kMost = (int64_t)1 << 31;  // elements: bytes of all rows in 63 bits
  if (q_stride > kMost || k_stride > kMost || q_out_stride > kMost || k_out_stride > kMost) return HQ_ERR_TOO_LARGE;
  const Region qi{q, 2 * qn, 2 * q_stride}, ki{k, 2 * kn, 2 * k_stride}, qo{q_out, 2 * qn, 2 * q_out_stride}, ko{k_out, 2 * kn, 2 * k_out_stride};
  if (!apart(qo, qi, tokens, true) || !apart(ko, ki, tokens, true) || !apart(qo, ki, tokens, false) || !apart(ko, qi, tokens, false) ||
      !apart(qo, ko, tokens, false))
    return HQ_ERR_BAD_SHAPE;
  const Stretch read[] = {{q_weight, 2 * (int64_t)head_dim}, {k_weight, 2 * (int64_t)head_dim}, {rotary ? cos_sin : nullptr, 4 * (int64_t)num_positions * rotary},
                          {rotary ? positions : nullptr, 4 * tokens}};
  for (const Stretch& x : read)
    if (!apart(qo, tokens, x) || !apart(ko, tokens, x)) return HQ_ERR_BAD_SHAPE;
  const HqDevice* dev = nullptr;
  const int dc = hq_current_device(&dev);
  if (dc != HQ_OK) return dc;
  RotateArgs a{};
  a.q = (const hq_u4v*)q;
  a.k = (const hq_u4v*)k;
  a.qo = (hq_u4v*)q_out;
  a.ko = (hq_u4v*)k_out;
  a.qw = (const hq_u4v*)q_weight;
  a.kw = (const hq_u4v*)k_weight;
  a.cs = (const hq_f4v*)cos_sin;
  a.positions = positions;
  a.qs = q_stride / 8;
  a.ks = k_stride / 8;
  a.qos = q_out_stride / 8;
  a.kos = k_out_stride / 8;
  a.tokens = (int)tokens;
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.rotary = rotary;
  a.known = num_positions;
  a.interleaved = interleaved != 0;
  a.eps = eps;
  const hipStream_t s = (hipStream_t)stream;
  return HQ_BY_TYPE(false);
}

extern "C" int hq_cache_write_rotated(const void* q, const void* k, const void* v, void* q_out, void* k_pages, void* v_pages, int dtype,
                                      const void* q_weight, const void* k_weight, const float* cos_sin, const int32_t* table,
                                      const int32_t* starts, const int32_t* cu, int rows, int64_t tokens, int table_width, int num_pages,
                                      int page_size, int heads, int kv_heads, int head_dim, int rotary, int num_positions, int64_t q_stride,
                                      int64_t k_stride, int64_t v_stride, int64_t q_out_stride, float eps, int interleaved, void* stream) {
  const int rc = check(dtype, head_dim, rotary, num_positions, cos_sin, tokens, heads, kv_heads, q_weight || k_weight, eps);
  if (rc != HQ_OK) return rc;
  if (rows < 0 || table_width < 0 || num_pages < 0) return HQ_ERR_BAD_SHAPE;
  if (page_size < 1 || page_size > 1024 || (page_size & (page_size - 1))) return HQ_ERR_BAD_SHAPE;
  if (tokens == 0 || rows == 0) return HQ_OK;
  if (!q || !k || !v || !q_out || !starts || !cu || (table_width && !table) || (table_width && num_pages && (!k_pages || !v_pages)))
    return HQ_ERR_NULL_POINTER;
  const int64_t qn = (int64_t)heads * head_dim, kn = (int64_t)kv_heads * head_dim;
  if (q_stride < qn || q_out_stride < qn || k_stride < kn || v_stride < kn) return HQ_ERR_BAD_SHAPE;
  if (odd(q, q_stride) || odd(k, k_stride) || odd(v, v_stride) || odd(q_out, q_out_stride) || odd(k_pages, 0) || odd(v_pages, 0) || odd(q_weight, 0) ||
      odd(k_weight, 0) || odd(cos_sin, 0) || (((uintptr_t)table | (uintptr_t)starts | (uintptr_t)cu) & 3))
    return HQ_ERR_MISALIGNED;
  constexpr int64_t kMost = (int64_t)1 << 31;
  if (q_stride > kMost || k_stride > kMost || v_stride > kMost || q_out_stride > kMost) return HQ_ERR_TOO_LARGE;
  const Region qi{q, 2 * qn, 2 * q_stride}, ki{k, 2 * kn, 2 * k_stride}, vi{v, 2 * kn, 2 * v_stride}, qo{q_out, 2 * qn, 2 * q_out_stride};
  if (!apart(qo, qi, tokens, true) || !apart(qo, ki, tokens, false) || !apart(qo, vi, tokens, false)) return HQ_ERR_BAD_SHAPE;
  const int64_t bytes = table_width ? bytes_of_pages(num_pages, kv_heads, page_size, head_dim) : 0;
  const Stretch kp{k_pages, bytes}, vp{v_pages, bytes};
  const Stretch read[] = {{q_weight, 2 * (int64_t)head_dim}, {k_weight, 2 * (int64_t)head_dim}, {rotary ? cos_sin : nullptr, 4 * (int64_t)num_positions * rotary},
                          {table, 4 * (int64_t)rows * table_width}, {starts, 4 * (int64_t)rows}, {cu, 4 * ((int64_t)rows + 1)}};
  for (const Stretch& x : read)
    if (!apart(qo, tokens, x) || !apart(kp, x) || !apart(vp, x)) return HQ_ERR_BAD_SHAPE;
  for (const Region& x : {qi, ki, vi, qo})
    if (!apart(x, tokens, kp) || !apart(x, tokens, vp)) return HQ_ERR_BAD_SHAPE;
  if (!apart(kp, vp)) return HQ_ERR_BAD_SHAPE;
  const HqDevice* dev = nullptr;
  const int dc = hq_current_device(&dev);
  if (dc != HQ_OK) return dc;
  RotateArgs a{};
  a.q = (const hq_u4v*)q;
  a.k = (const hq_u4v*)k;
  a.v = (const hq_u4v*)v;
  a.qo = (hq_u4v*)q_out;
  a.ko = (hq_u4v*)k_pages;
  a.vo = (hq_u4v*)v_pages;
  a.qw = (const hq_u4v*)q_weight;
  a.kw = (const hq_u4v*)k_weight;
  a.cs = (const hq_f4v*)cos_sin;
  a.table = table;
  a.starts = starts;
  a.cu = cu;
  a.qs = q_stride / 8;
  a.ks = k_stride / 8;
  a.vs = v_stride / 8;
  a.qos = q_out_stride / 8;
  a.tokens = (int)tokens;
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.rotary = rotary;
  a.known = num_positions;
  a.rows = rows;
  a.width = table_width;
  a.pages = num_pages;
  a.page_log = __builtin_ctz(page_size);
  a.interleaved = interleaved != 0;
  a.eps = eps;
  const hipStream_t s = (hipStream_t)stream;
  return HQ_BY_TYPE(true);
}
