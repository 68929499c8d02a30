// vx_paged.h -- a paged key/value cache for batches: appending rotated keys
// and values, and the attention of a batch that shares a prefix.  The kernels
// work on the caller's device memory and stream; nothing is kept between
// calls.
//
// Cache: K and V pools [page][kv head][slot][head_dim] with strides for the
// first three (elements); pages of 16 to 4096 slots, a power of two, so an
// aligned run of 16 keys lies in one page.  A sequence's slot s lives in page
// table[seq][s / page_size] at s % page_size.
//
// Page ids, lengths and row starts are device data that no host check sees:
// every one is tested against its pool or bound before an address is made
// from it, and what fails the test counts as absent (a token is not written,
// a key is not seen).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "vx_kernels.h"

namespace vx {

typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

struct PagedKV {
  void *k, *v;
  int64_t page_stride, head_stride, token_stride;
  int n_pages, page_size, page_shift, n_kv_heads;
};

// the page of slot `slot` by a row of `width` page ids, -1 where there is none
__host__ __device__ inline int pg_page(const int *ids, int width, int64_t slot, int page_shift, int n_pages) {
  if (slot < 0) return -1;
  const int64_t i = slot >> page_shift;
  if (i >= width) return -1;
  const int p = ids[i];
  return p >= 0 && p < n_pages ? p : -1;
}

// one element of a row or cache type as f32, and back (one rounding, to
// nearest even)
template <typename T>
__device__ __forceinline__ float pg_f32(T x) {
  return (float)x;
}
template <typename T, int N>
struct alignas(sizeof(T) * N) PgVec {
  T x[N];
};
// N elements at p (aligned to 16 bytes, or to all of them if they are fewer)
template <typename T, int N>
__device__ __forceinline__ void pg_load(const T *p, float (&y)[N]) {
  constexpr int C = 16 / sizeof(T) < N ? 16 / sizeof(T) : N;
#pragma unroll
  for (int i = 0; i < N; i += C) {
    const PgVec<T, C> v = *(const PgVec<T, C> *)(p + i);
#pragma unroll
    for (int j = 0; j < C; j++) y[i + j] = pg_f32(v.x[j]);
  }
}
template <typename T, int N>
__device__ __forceinline__ void pg_store(T *p, const float (&y)[N]) {
  constexpr int C = 16 / sizeof(T) < N ? 16 / sizeof(T) : N;
#pragma unroll
  for (int i = 0; i < N; i += C) {
    PgVec<T, C> v;
#pragma unroll
    for (int j = 0; j < C; j++) v.x[j] = (T)y[i + j];
    *(PgVec<T, C> *)(p + i) = v;
  }
}

// ----------------------------------------------------------------- append
// Token t, position p = pos[t]: every head's pair i of the first rotary_dim
// elements turns by p theta^(-2 i / rotary_dim); K (turned) and V go to slot
// p - base of sequence seq[t], Q (turned) to q_out.
struct AppendArgs {
  PagedKV kv;
  const void *k, *v, *q;
  void *q_out;
  int64_t k_row, k_head, v_row, v_head, q_row, q_head, o_row, o_head;
  const int *pos, *seq, *table;
  int64_t table_stride;
  int table_width, base, n_tokens, n_seqs, n_heads, head_dim;
  int rotary_dim, interleaved;
  // revolutions a position for each pair: theta^(-2 i / rotary_dim) / (2 pi).
  // In 64 bits: at position 10^6 an f32 frequency is off by 0.06 radians.
  double turns[64];
};

constexpr int PA_NT = 256;

// One block a token: its 64 angles are reduced to a revolution in 64 bits and
// their sine and cosine taken once, then shared by every head through LDS.
// A thread moves two chunks of 8 elements: neighbours, or the two halves of a
// pair when pairs are (i, i + rotary_dim / 2).
template <typename RT, typename CT>
__global__ __launch_bounds__(PA_NT) void paged_append_kernel(AppendArgs a) {
  __shared__ float cs[64], sn[64];
  const int t = blockIdx.x, tid = threadIdx.x;
  const int p = a.pos[t], s = a.seq ? a.seq[t] : t;
  if (p < 0 || s < 0 || s >= a.n_seqs) return;
  const int64_t slot = (int64_t)p - a.base;
  const int page = pg_page(a.table + (int64_t)s * a.table_stride, a.table_width, slot, a.kv.page_shift, a.kv.n_pages);
  if (page < 0) return;
  const int half = a.rotary_dim >> 1;
  if (tid < half) {
    const double r = p * a.turns[tid];
    sincospif(2.0f * (float)(r - rint(r)), &sn[tid], &cs[tid]);
  }
  __syncthreads();
  const int per = a.head_dim >> 4, hkv = a.kv.n_kv_heads;
  const int heads = 2 * hkv + (a.q ? a.n_heads : 0);
  const int64_t at = page * a.kv.page_stride + (slot & (a.kv.page_size - 1)) * a.kv.token_stride;
  for (int w = tid; w < heads * per; w += PA_NT) {
    const int h = w / per, c = w - h * per;
    // elements d0.. and d1.. of the head, and the first pair they hold
    const bool turned = c < (a.rotary_dim >> 4);
    int d0 = 16 * c, d1 = d0 + 8;
    if (turned && !a.interleaved) d0 = 8 * c, d1 = d0 + half;
    float x[8], y[8];
    if (h >= hkv && h < 2 * hkv) {
      const RT *src = (const RT *)a.v + t * a.v_row + (h - hkv) * a.v_head;
      CT *dst = (CT *)a.kv.v + at + (h - hkv) * a.kv.head_stride;
      pg_load(src + d0, x);
      pg_load(src + d1, y);
      pg_store(dst + d0, x);
      pg_store(dst + d1, y);
      continue;
    }
    const RT *src = h < hkv ? (const RT *)a.k + t * a.k_row + h * a.k_head
                            : (const RT *)a.q + t * a.q_row + (h - 2 * hkv) * a.q_head;
    pg_load(src + d0, x);
    pg_load(src + d1, y);
    if (turned) {
#pragma unroll
      for (int j = 0; j < 8; j++) {
        // interleaved: x holds pairs 8 c .. 8 c + 3, y the next four
        if (a.interleaved) {
          if (j & 1) continue;
          const float c0 = cs[8 * c + j / 2], s0 = sn[8 * c + j / 2];
          const float c1 = cs[8 * c + 4 + j / 2], s1 = sn[8 * c + 4 + j / 2];
          const float u = x[j], v = x[j + 1], e = y[j], f = y[j + 1];
          x[j] = u * c0 - v * s0;
          x[j + 1] = u * s0 + v * c0;
          y[j] = e * c1 - f * s1;
          y[j + 1] = e * s1 + f * c1;
        } else {
          const float c0 = cs[8 * c + j], s0 = sn[8 * c + j];
          const float u = x[j], v = y[j];
          x[j] = u * c0 - v * s0;
          y[j] = u * s0 + v * c0;
        }
      }
    }
    if (h < hkv) {
      CT *dst = (CT *)a.kv.k + at + h * a.kv.head_stride;
      pg_store(dst + d0, x);
      pg_store(dst + d1, y);
    } else {
      RT *dst = (RT *)a.q_out + t * a.o_row + (h - 2 * hkv) * a.o_head;
      pg_store(dst + d0, x);
      pg_store(dst + d1, y);
    }
  }
}

// ----------------------------------------------------------------- attend
// Row r of sequence s, the j-th of its n_s rows: one softmax over the shared
// prefix's keys and the first clamp(lens[s] - (n_s - 1 - j), 0, max_len) keys
// of the sequence.  Columns: the n_s rows times the G query heads of a KV
// head, row-major, 16 to a wave.  Blocks of the first kind take the prefix
// with the columns of all rows, so its keys are read once for many columns
// and not once a sequence; blocks of the second kind take a sequence's own
// keys (and, where that is little, the prefix before them: `fused`).  Both
// split the key axis and leave (o, m, l) partials that a second kernel joins,
// unless there is one split in all.
struct AttendArgs {
  PagedKV kv;
  const void *q;
  void *out;
  float *lse;  // [rows][heads] or null
  int64_t q_row, q_head, o_row, o_head;
  const int *row_start, *lens, *table, *prefix_pages;
  int64_t table_stride;
  int table_width, prefix_count, prefix_len, max_len;
  int n_rows, n_seqs, n_heads, group;
  float scale;  // times log2(e)
  // the plan: column waves of a block, tiles of columns, splits and their
  // keys (multiples of 32)
  int pre_waves, pre_tiles, pre_splits, pre_chunk;
  int own_waves, own_slots, own_splits, own_chunk;
  int fused;
  float *part_o;   // [slot][row * heads + head][head_dim]
  float2 *part_ml; // [slot][row * heads + head]: maximum (log2 units), sum
};

constexpr int AT_COLS = 16;  // columns of a wave: the matrix instruction's
constexpr int AT_KEYS = 32;  // keys of a wave's step: two tiles of 16
constexpr int AT_WAVES = 4;

struct AttendPlan {
  int pre_waves, pre_tiles, pre_splits, pre_chunk, own_waves, own_slots, own_splits, own_chunk, fused;
  size_t ml_at, bytes;  // the workspace: part_o, then part_ml at ml_at
  int64_t blocks;
  int slots() const { return pre_splits + own_splits; }
  bool direct() const { return slots() == 1; }  // no partials: the blocks write the result
};

__host__ __device__ inline int64_t at_ceil(int64_t a, int64_t b) { return (a + b - 1) / b; }

inline AttendPlan attend_plan(int n_rows, int n_seqs, int n_heads, int n_kv_heads, int head_dim, int prefix_len,
                              int max_len, bool ragged, int cus) {
  AttendPlan p{};
  const int64_t g = n_heads / n_kv_heads, cols = n_rows * g;
  const int64_t want = 3 * (int64_t)cus;
  // a block's four waves go to columns as far as there are some, the rest to keys
  auto waves = [](int64_t c) { return c > 32 ? 4 : c > 16 ? 2 : 1; };
  auto split = [&](int64_t units, int64_t keys, int w, int *splits, int *chunk) {
    const int64_t step = AT_KEYS * (AT_WAVES / w);  // keys of a block's step
    int64_t n = at_ceil(want, units > 0 ? units : 1);
    const int64_t most = at_ceil(keys, 2 * step);
    n = n > most ? most : n;
    n = n < 1 ? 1 : n;
    const int64_t c = at_ceil(at_ceil(keys, n), step) * step;
    *chunk = (int)c;
    *splits = (int)at_ceil(keys, c);
  };
  p.fused = prefix_len > 0 && max_len > 0 && (int64_t)prefix_len + max_len <= 512;
  const int64_t before = p.fused ? at_ceil(prefix_len, AT_KEYS) * AT_KEYS : 0;
  p.pre_waves = waves(cols);
  if (prefix_len > 0 && !p.fused) {
    p.pre_tiles = (int)at_ceil(cols, AT_COLS * p.pre_waves);
    split((int64_t)p.pre_tiles * n_kv_heads, prefix_len, p.pre_waves, &p.pre_splits, &p.pre_chunk);
  }
  p.own_waves = waves(ragged ? cols / (n_seqs > 0 ? n_seqs : 1) : g);
  if (max_len > 0) {
    // sequence s's tiles start at slot floor(row_start[s] g / columns) + s
    const int64_t c = AT_COLS * p.own_waves;
    p.own_slots = (int)(ragged ? cols / c + n_seqs : n_seqs * at_ceil(g, c));
    if (p.fused) {
      p.own_splits = 1;
      p.own_chunk = (int)(before + at_ceil(max_len, AT_KEYS) * AT_KEYS);
    } else {
      split((int64_t)p.own_slots * n_kv_heads, max_len, p.own_waves, &p.own_splits, &p.own_chunk);
    }
  }
  const int64_t items = p.direct() ? 0 : (int64_t)p.slots() * n_rows * n_heads;
  p.ml_at = (size_t)items * head_dim * 4;
  p.bytes = p.ml_at + (size_t)items * 8;
  p.blocks = ((int64_t)p.pre_tiles * p.pre_splits + (int64_t)p.own_slots * p.own_splits) * n_kv_heads;
  return p;
}

// the largest s in [0, n) with f(s) <= x, -1 if there is none, for f that
// does not fall; every lane of the wave gets it
template <typename F>
__device__ __forceinline__ int at_search(int n, int x, F f) {
  const int lane = threadIdx.x & 63;
  int lo = 0, span = n;
  bool any = false;
  while (span > 0) {
    const int step = (span + 63) >> 6, s = lo + lane * step;
    const bool yes = lane * step < span && f(s) <= x;
    const unsigned long long m = __ballot(yes);
    if (!m) return any ? lo : -1;
    any = true;
    const int last = 63 - __clzll(m);
    const int next = lo + last * step;
    span = step == 1 ? 0 : (span - last * step < step ? span - last * step : step);
    lo = next;
    if (span <= 1) break;
  }
  return any ? lo : -1;
}

// The matrix products of one 16-key tile, by types.  An A operand's lane
// holds a key's (or a dimension's) elements, a B operand's a column's.
//   16-bit caches: v_mfma_f32_16x16x32.  f32 rows on an f16 cache are split
//     into hi and lo halves (queries after a scaling by a power of two that
//     keeps them in f16's range; weights as they are), so each product is
//     taken twice and the result is good to about 2^-21.
//   f32 caches: v_mfma_f32_16x16x4_f32, exact products.
// The score tile S^T = K Q^T leaves lane (g, c) with keys 4 g .. 4 g + 3 of
// column c.  The value product O^T = V^T P^T takes its weights from there
// without any movement, since the order of keys inside the instruction is
// free: lane group g brings the values of the same keys.  A value lane loads
// head_dim / 16 dimensions of each key, contiguous over the 16 lanes, and
// transposes key pairs in registers; instruction e then works on dimensions
// VE r + e (r the operand's row), which leaves a lane with 4 VE contiguous
// dimensions of its column.
template <typename RT, typename CT, int HD>
struct AtTypes {
  static constexpr bool F32 = sizeof(CT) == 4;
  static constexpr bool SPLIT = !F32 && sizeof(RT) == 4;
  static constexpr int VE = HD / 16;           // value instructions, dimensions a lane loads of a key
  static constexpr int KC = F32 ? HD / 16 : HD / 32;  // 16-byte chunks of a key a lane holds
};

__device__ __forceinline__ f32x4 at_mma(h8 a, h8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 at_mma(b8 a, b8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
template <typename CT>
struct At8;
template <>
struct At8<_Float16> {
  typedef h8 T;
};
template <>
struct At8<__bf16> {
  typedef b8 T;
};
template <>
struct At8<float> {
  typedef h8 T;  // unused
};

// 2^x to 1 ulp; results below the normal range are 0
__device__ __forceinline__ float at_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// the logarithm of a sum l in units of 2^m (no key: -inf; NaN stays)
__device__ __forceinline__ float at_lse(float m, float l) {
  return l == 0 ? -INFINITY : m == -INFINITY ? l : (m + log2f(l)) * 0.6931471805599453f;
}

// the first row of sequence s, inside the rows there are
__device__ __forceinline__ int at_row(const int *row_start, int s, int n_rows) {
  return min(max(row_start[s], 0), n_rows);
}

// the maximum over the four lane groups that share a column
__device__ __forceinline__ float at_max4(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float at_sum4(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

// A wave's state over its keys for one tile of columns
template <typename RT, typename CT, int HD>
struct AtWave {
  using Y = AtTypes<RT, CT, HD>;
  using E8 = typename At8<CT>::T;
  u32x4 q[Y::KC * (Y::SPLIT ? 2 : 1)];  // the column's queries: hi, then lo
  float qs;                             // the factor from products to log2 scores
  f32x4 o[Y::VE];
  float m, l;

  __device__ __forceinline__ void init(const RT *src, float scale) {
    const int g = (threadIdx.x & 63) >> 4;
    m = -INFINITY;
    l = 0;
    qs = scale;
#pragma unroll
    for (int e = 0; e < Y::VE; e++) o[e] = f32x4{0, 0, 0, 0};
    if constexpr (!Y::SPLIT) {
#pragma unroll
      for (int j = 0; j < Y::KC; j++)
        q[j] = src ? *(const u32x4 *)(src + (Y::F32 ? 16 * j + 4 * g : 32 * j + 8 * g)) : u32x4{0, 0, 0, 0};
    } else {
      float x[Y::KC][8], top = 0;
#pragma unroll
      for (int j = 0; j < Y::KC; j++) {
        if (src) {
          pg_load((const float *)src + 32 * j + 8 * g, x[j]);
        } else {
#pragma unroll
          for (int i = 0; i < 8; i++) x[j][i] = 0;
        }
#pragma unroll
        for (int i = 0; i < 8; i++) top = fmaxf(top, fabsf(x[j][i]));
      }
      top = at_max4(top);
      // |x| 2^-ex < 1, so hi and lo are normal f16 numbers down to 2^-13 of the largest
      int ex = 0;
      if (top > 0 && top < INFINITY) (void)frexpf(top, &ex);
      qs = ldexpf(scale, ex);
#pragma unroll
      for (int j = 0; j < Y::KC; j++) {
#pragma unroll
        for (int i = 0; i < 8; i++) x[j][i] = ldexpf(x[j][i], -ex);
        h8 hi, lo;
        split_n(x[j], hi, lo);
        q[j] = __builtin_bit_cast(u32x4, hi);
        q[Y::KC + j] = __builtin_bit_cast(u32x4, lo);
      }
    }
  }

  // scores of 16 keys, one row of `k` (already offset to the lane's key)
  __device__ __forceinline__ f32x4 score(const u32x4 (&k)[Y::KC]) const {
    f32x4 s{0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < Y::KC; j++) {
      if constexpr (Y::F32) {
        const f32x4 a = __builtin_bit_cast(f32x4, k[j]), b = __builtin_bit_cast(f32x4, q[j]);
#pragma unroll
        for (int i = 0; i < 4; i++) s = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], s, 0, 0, 0);
      } else {
        s = at_mma(__builtin_bit_cast(E8, k[j]), __builtin_bit_cast(E8, q[j]), s);
        if constexpr (Y::SPLIT) s = at_mma(__builtin_bit_cast(E8, k[j]), __builtin_bit_cast(E8, q[Y::KC + j]), s);
      }
    }
    return s;
  }

  // o += P V over 32 keys; v[j]: the lane's dimensions of key 4 g + (j & 3) of tile j >> 2
  __device__ __forceinline__ void values(const float (&p)[8], const uint32_t (&v)[8][Y::F32 ? Y::VE : Y::VE / 2]) {
    if constexpr (Y::F32) {
#pragma unroll
      for (int j = 0; j < 8; j++)
#pragma unroll
        for (int e = 0; e < Y::VE; e++)
          o[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, v[j][e]), p[j], o[e], 0, 0, 0);
    } else {
      E8 ph, pl;
      if constexpr (Y::SPLIT) {
        split_n(p, ph, pl);
      } else {
#pragma unroll
        for (int j = 0; j < 8; j++) ph[j] = (CT)p[j];
      }
#pragma unroll
      for (int w = 0; w < Y::VE / 2; w++) {
        u32x4 a, b;
#pragma unroll
        for (int j = 0; j < 4; j++) {  // key pairs: the low halves, the high halves
          a[j] = __builtin_amdgcn_perm(v[2 * j + 1][w], v[2 * j][w], 0x05040100u);
          b[j] = __builtin_amdgcn_perm(v[2 * j + 1][w], v[2 * j][w], 0x07060302u);
        }
        const E8 va = __builtin_bit_cast(E8, a), vb = __builtin_bit_cast(E8, b);
        o[2 * w] = at_mma(va, ph, o[2 * w]);
        o[2 * w + 1] = at_mma(vb, ph, o[2 * w + 1]);
        if constexpr (Y::SPLIT) {
          o[2 * w] = at_mma(va, pl, o[2 * w]);
          o[2 * w + 1] = at_mma(vb, pl, o[2 * w + 1]);
        }
      }
    }
  }

  // the weights of 8 scores (in log2 units; -inf: not seen), with the running
  // maximum moved where one passes it by more than 8: until then weights of up
  // to 2^8 do no harm, and the sums need not be scaled
  __device__ __forceinline__ void softmax(float (&x)[8]) {
    float top = x[0];
#pragma unroll
    for (int j = 1; j < 8; j++) top = fmaxf(top, x[j]);
    if (__any(top > m + 8.0f)) {
      const float n = fmaxf(m, at_max4(top));
      const float f = n == -INFINITY ? 1.0f : at_exp2(m - n);
      m = n;
      l *= f;
#pragma unroll
      for (int e = 0; e < Y::VE; e++) o[e] *= f;
    }
    const float z = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      x[j] = at_exp2(x[j] - z);
      l += x[j];
    }
  }
};

// whether a word of values holds one that is not finite
template <typename CT>
__device__ __forceinline__ bool at_odd(uint32_t w) {
  if constexpr (sizeof(CT) == 4) {
    return (w & 0x7f800000u) == 0x7f800000u;
  } else {
    constexpr uint32_t e = __is_same(CT, __bf16) ? 0x7f80u : 0x7c00u;
    return ((w & e) == e) | ((w >> 16 & e) == e);
  }
}

// a word of values with 0 in place of what is not finite
template <typename CT>
__device__ __forceinline__ uint32_t at_finite(uint32_t w) {
  if constexpr (sizeof(CT) == 4) return at_odd<CT>(w) ? 0 : w;
  return (at_odd<CT>(w & 0xffffu) ? 0 : w & 0xffffu) | (at_odd<CT>(w & 0xffff0000u) ? 0 : w & 0xffff0000u);
}

// 2 waves on a SIMD for f32 caches, whose tiles take twice the registers, else 3
template <typename RT, typename CT, int HD>
__global__ __launch_bounds__(64 * AT_WAVES, sizeof(CT) == 4 && HD == 128 ? 2 : 3) void paged_attend_kernel(AttendArgs a) {
  using Y = AtTypes<RT, CT, HD>;
  constexpr int VW = Y::F32 ? Y::VE : Y::VE / 2;  // 32-bit words of a value lane's key
  __shared__ f32x4 so[AT_WAVES - 1][Y::VE][64];
  __shared__ float sm[AT_WAVES - 1][64], sl[AT_WAVES - 1][64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int hkv = a.kv.n_kv_heads, kvh = blockIdx.x % hkv;
  int b = blockIdx.x / hkv, slot;

  // The block's keys are a run [k0, k1) of one or two page lists laid end to
  // end: the prefix up to `pre` (rounded up to a step), then the sequence's
  // own up to `end`.  A wave has 16 columns: row, query head, own keys seen.
  const int *ids = nullptr;
  int pre = 0, end = 0, k0, k1, row = -1, seen = 0, waves, col, last_seen = 0;
  if (b < a.pre_tiles * a.pre_splits) {
    slot = b / a.pre_tiles;
    waves = a.pre_waves;
    const int tile = b - slot * a.pre_tiles, rows = a.row_start ? at_row(a.row_start, a.n_seqs, a.n_rows) : a.n_rows;
    if (tile * waves * AT_COLS >= rows * a.group) return;
    col = (tile * waves + wave % waves) * AT_COLS + c;
    if (col < rows * a.group) row = col / a.group;
    pre = a.prefix_len;
    k0 = slot * a.pre_chunk;
    k1 = min(pre, k0 + a.pre_chunk);
  } else {
    b -= a.pre_tiles * a.pre_splits;
    slot = b / a.own_slots;
    b -= slot * a.own_slots;
    waves = a.own_waves;
    const int tc = waves * AT_COLS;
    int s, tile, r0, r1;
    if (a.row_start) {
      s = at_search(a.n_seqs, b, [&](int i) { return at_row(a.row_start, i, a.n_rows) * a.group / tc + i; });
      if (s < 0) return;
      r0 = at_row(a.row_start, s, a.n_rows);
      r1 = at_row(a.row_start, s + 1, a.n_rows);
      tile = b - (r0 * a.group / tc + s);
    } else {
      const int tiles = (a.group + tc - 1) / tc;
      s = b / tiles;
      tile = b - s * tiles;
      r0 = s;
      r1 = s + 1;
    }
    const int cols = (r1 - r0) * a.group;
    if (tile * tc >= cols) return;
    col = tile * tc + wave % waves * AT_COLS + c;
    // the j-th of n rows sees len - (n - 1 - j) keys
    const int len = min(max(a.lens[s], 0), a.max_len + (r1 - r0)) - (r1 - r0 - 1);
    auto sees = [&](int x) { return max(min(len + x / a.group, a.max_len), 0); };
    last_seen = sees(min(tile * tc + tc, cols) - 1);
    seen = sees(min(col, cols - 1));
    if (col < cols) row = r0 + col / a.group;
    pre = a.fused ? a.prefix_len : 0;
    end = last_seen;
    const int before = (pre + AT_KEYS - 1) & -AT_KEYS;
    k0 = slot * a.own_chunk;
    k1 = min(before + end, k0 + a.own_chunk);
    slot += a.pre_splits;
    const bool direct = a.pre_splits + a.own_splits == 1;
    if (k1 <= k0 && !direct) return;
    ids = a.table + (int64_t)s * a.table_stride;
  }
  const int before = (pre + AT_KEYS - 1) & -AT_KEYS;
  const int head = kvh * a.group + (row >= 0 ? col % a.group : 0);

  AtWave<RT, CT, HD> w;
  w.init(row >= 0 ? (const RT *)a.q + row * a.q_row + head * a.q_head : nullptr, a.scale);

  // what the wave's column that sees least sees: keys before it need no mask
  int least = row >= 0 ? seen : last_seen;
  least = min(least, __shfl_xor(least, 1, 64));
  least = min(least, __shfl_xor(least, 2, 64));
  least = min(least, __shfl_xor(least, 4, 64));
  least = min(least, __shfl_xor(least, 8, 64));
  least = __builtin_amdgcn_readfirstlane(least);

  // uniform base addresses, and 32-bit offsets of a lane in a tile of 16 keys
  const char *kb = (const char *)a.kv.k + kvh * a.kv.head_stride * (int64_t)sizeof(CT);
  const char *vb = (const char *)a.kv.v + kvh * a.kv.head_stride * (int64_t)sizeof(CT);
  const int ts = (int)a.kv.token_stride * (int)sizeof(CT);
  const uint32_t k_lane = c * ts + 16 * g, v_lane = 4 * g * ts + Y::VE * c * (int)sizeof(CT);
  const int key_waves = AT_WAVES / waves, key_wave = wave / waves;
  const int stride = AT_KEYS * key_waves;

  u32x4 k[2][Y::KC];
  uint32_t v[8][VW];
  for (int base = k0; base < k1; base += 1024) {
    // lane i finds the tile of keys base + 16 i .. (bytes from the pools'
    // starts); an absent tile reads the first page, and none of it is seen
    const int stop = min(k1, base + 1024);
    int page = -1, slot_in = 0;
    {
      const int x = base + 16 * lane;
      if (x < before) {
        slot_in = x;
        if (x < pre) page = pg_page(a.prefix_pages, a.prefix_count, x, a.kv.page_shift, a.kv.n_pages);
      } else if (x < stop) {
        slot_in = x - before;
        page = pg_page(ids, a.table_width, slot_in, a.kv.page_shift, a.kv.n_pages);
      }
    }
    const uint64_t have = __ballot(page >= 0);
    const int64_t my_at = page < 0 ? 0 : page * a.kv.page_stride * (int64_t)sizeof(CT) + (int64_t)(slot_in & (a.kv.page_size - 1)) * ts;
    const int at_lo = (int)my_at, at_hi = (int)(my_at >> 32);
    auto place = [&](int x, int h) -> int64_t {
      const int i = ((x - base) >> 4) + h;
      return (int64_t)__builtin_amdgcn_readlane(at_hi, i) << 32 | (uint32_t)__builtin_amdgcn_readlane(at_lo, i);
    };
    auto load_k = [&](int x) {
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const char *p = kb + place(x, h);
#pragma unroll
        for (int j = 0; j < Y::KC; j++) k[h][j] = *(const u32x4 *)(p + k_lane + 64 * j);
      }
    };
    auto load_v = [&](int x) {
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const char *p = vb + place(x, h);
#pragma unroll
        for (int i = 0; i < 4; i++, p += ts) {
          if constexpr (VW == 2) {
            const u32x2 y = *(const u32x2 *)(p + v_lane);
            v[4 * h + i][0] = y[0];
            v[4 * h + i][1] = y[1];
          } else {
#pragma unroll
            for (int z = 0; z < VW; z += 4) {
              const u32x4 y = *(const u32x4 *)(p + v_lane + 4 * z);
#pragma unroll
              for (int u = 0; u < 4; u++) v[4 * h + i][z + u] = y[u];
            }
          }
        }
      }
    };
    int x = base + AT_KEYS * key_wave;
    if (x >= stop) continue;
    load_k(x);
    load_v(x);
    // The next step's keys are asked for when this one's scores are taken, its
    // values when this one's are summed: one of the two is always on its way.
    // The last step asks for itself again, so that the number of loads in
    // flight is the same on every path and the waits can be exact.
    for (;;) {
      const int next = x + stride < stop ? x + stride : x;
      float p[8];
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const f32x4 s = w.score(k[h]);
#pragma unroll
        for (int i = 0; i < 4; i++) p[4 * h + i] = s[i] * w.qs;
      }
      load_k(next);
      const uint32_t there = (uint32_t)(have >> ((x - base) >> 4)) & 3;
      // keys of this list that are seen: by the column, by all, by any
      const bool shared = x < before;
      const int x0 = shared ? x : x - before;
      const int lim = shared ? pre : seen, all = shared ? pre : least, any = shared ? pre : end;
      uint32_t odd = 0;  // bit j: the lane's part of key j is not finite, and not seen by all
      if (all < x0 + AT_KEYS || there != 3) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const int key = x0 + 16 * (j >> 2) + 4 * g + (j & 3);
          const bool is = there >> (j >> 2) & 1;
          p[j] = is & (key < lim) ? p[j] : -INFINITY;
          // a value that no column sees may be anything, and 0 times it not 0
          const bool none = !is | (key >= any);
          bool bad = false;
#pragma unroll
          for (int y = 0; y < VW; y++) {
            v[j][y] = none ? 0 : v[j][y];
            bad |= at_odd<CT>(v[j][y]);
          }
          odd |= (uint32_t)(bad & (key >= all)) << j;
        }
      }
      w.softmax(p);
      if (__any(odd)) {
        // such elements are taken out of the common product and added to the
        // columns that see them one by one, each lane to its own dimensions
        for (int j = 0; j < 8; j++) {
          const uint64_t lanes = __ballot(odd >> j & 1);
#pragma unroll
          for (int jj = 0; jj < 8; jj++)
#pragma unroll
            for (int y = 0; y < VW; y++) v[jj][y] = jj == j && (odd >> j & 1) ? at_finite<CT>(v[jj][y]) : v[jj][y];
          float pj = p[0];
#pragma unroll
          for (int jj = 1; jj < 8; jj++) pj = jj == j ? p[jj] : pj;
          for (int gg = 0; gg < 4; gg++) {
            if (!(lanes >> (16 * gg) & 0xffff)) continue;
            const int in = 4 * gg + (j & 3);
            const float weight = __shfl(pj, 16 * gg + c, 64);
            const CT *row = (const CT *)(vb + place(x, j >> 2) + (int64_t)in * ts) + 4 * Y::VE * g;
            if (x0 + 16 * (j >> 2) + in < lim) {
#pragma unroll
              for (int i = 0; i < 4; i++) {
                float y[Y::VE];
                pg_load(row + Y::VE * i, y);
#pragma unroll
                for (int e = 0; e < Y::VE; e++)
                  if (!(fabsf(y[e]) < INFINITY)) w.o[e][i] = fmaf(weight, y[e], w.o[e][i]);
              }
            }
          }
        }
      }
      w.values(p, v);
      load_v(next);
      if (next == x) break;
      x = next;
    }
  }

  // the waves with the same columns join their states in the first one's
  w.l = at_sum4(w.l);
  if (key_waves > 1) {
    if (key_wave > 0) {
      const int at = wave - waves;
#pragma unroll
      for (int e = 0; e < Y::VE; e++) so[at][e][lane] = w.o[e];
      sm[at][lane] = w.m;
      sl[at][lane] = w.l;
    }
    __syncthreads();
    if (key_wave > 0) return;
    for (int i = 1; i < key_waves; i++) {
      const int at = wave + (i - 1) * waves;
      const float m1 = sm[at][lane], m = fmaxf(w.m, m1);
      // (a state without a maximum holds zeros, or NaN, which must not get lost)
      const float f0 = w.m == -INFINITY ? 1.0f : at_exp2(w.m - m), f1 = m1 == -INFINITY ? 1.0f : at_exp2(m1 - m);
      w.m = m;
      w.l = w.l * f0 + sl[at][lane] * f1;
#pragma unroll
      for (int e = 0; e < Y::VE; e++) w.o[e] = w.o[e] * f0 + so[at][e][lane] * f1;
    }
  }
  if (row < 0) return;
  // the lane's dimensions: 4 VE from 4 VE g on
  if (a.pre_splits + a.own_splits == 1) {
    const float r = w.l == 0 ? 0.0f : 1.0f / w.l;
    RT *out = (RT *)a.out + row * a.o_row + head * a.o_head + 4 * Y::VE * g;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      float y[Y::VE];
#pragma unroll
      for (int e = 0; e < Y::VE; e++) y[e] = w.o[e][i] * r;
      pg_store(out + Y::VE * i, y);
    }
    if (a.lse && g == 0) a.lse[(int64_t)row * a.n_heads + head] = at_lse(w.m, w.l);
    return;
  }
  const int64_t item = ((int64_t)slot * a.n_rows + row) * a.n_heads + head;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    float y[Y::VE];
#pragma unroll
    for (int e = 0; e < Y::VE; e++) y[e] = w.o[e][i];
    pg_store(a.part_o + item * HD + 4 * Y::VE * g + Y::VE * i, y);
  }
  if (g == 0) a.part_ml[item] = make_float2(w.m, w.l);
}

// Joins a row and head's partials, a wave each: lane l takes dimensions
// HD / 64 l ..
template <typename RT, int HD>
__global__ __launch_bounds__(256) void paged_attend_join_kernel(AttendArgs a) {
  constexpr int N = HD / 64;
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), items = (int64_t)a.n_rows * a.n_heads;
  if (item >= items) return;
  const int row = (int)(item / a.n_heads), head = (int)(item - (int64_t)row * a.n_heads);
  int s = row, back = 0;  // back: rows of the sequence behind this one
  if (a.row_start) {
    s = at_search(a.n_seqs, row, [&](int i) { return at_row(a.row_start, i, a.n_rows); });
    if (s < 0) return;
    const int end = at_row(a.row_start, s + 1, a.n_rows);
    if (row >= end) return;
    back = end - 1 - row;
  }
  const int seen = min(min(max(a.lens[s], 0), a.max_len + back + 1) - back, a.max_len);
  const int own = seen > 0 ? (seen + a.own_chunk - 1) / a.own_chunk : 0;
  const int parts = a.pre_splits + own;
  float m = -INFINITY;
  for (int i = lane; i < parts; i += 64) m = fmaxf(m, a.part_ml[i * items + item].x);
  m = wave_max(m);
  float l = 0, y[N];
#pragma unroll
  for (int j = 0; j < N; j++) y[j] = 0;
  for (int i = 0; i < parts; i++) {
    const float2 ml = a.part_ml[i * items + item];
    const float f = ml.x == -INFINITY ? 1.0f : at_exp2(ml.x - m);
    float x[N];
    pg_load(a.part_o + (i * items + item) * HD + N * lane, x);
    l = fmaf(ml.y, f, l);
#pragma unroll
    for (int j = 0; j < N; j++) y[j] = fmaf(x[j], f, y[j]);
  }
  const float r = l == 0 ? 0.0f : 1.0f / l;
#pragma unroll
  for (int j = 0; j < N; j++) y[j] *= r;
  pg_store((RT *)a.out + row * a.o_row + head * a.o_head + N * lane, y);
  if (a.lse && lane == 0) a.lse[item] = at_lse(m, l);
}

}  // namespace vx
