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
// head, row-major, 16 to a tile.  Blocks of the first kind take the prefix
// with the columns of all rows, so its keys are read once for 16 columns and
// not once a sequence; blocks of the second kind take a sequence's own keys.
// Both split the key axis and leave (o, m, l) partials that a second kernel
// joins.
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
  // the plan: blocks of the prefix, splits and their keys (multiples of 32)
  int pre_tiles, pre_splits, pre_chunk;
  int own_slots, own_splits, own_chunk;
  float *part_o;   // [slot][row * heads + head][head_dim]
  float2 *part_ml; // [slot][row * heads + head]: maximum (log2 units), sum
};

constexpr int AT_COLS = 16;  // columns of a tile: the matrix instruction's
constexpr int AT_KEYS = 32;  // keys of a wave's step: two tiles of 16
constexpr int AT_WAVES = 4;

struct AttendPlan {
  int pre_tiles, pre_splits, pre_chunk, own_slots, own_splits, own_chunk;
  size_t ml_at, bytes;  // the workspace: part_o, then part_ml at ml_at
  int64_t blocks;
};

__host__ __device__ inline int64_t at_ceil(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Splits: enough blocks for about four on each compute unit, at least 128
// keys a split.
inline AttendPlan attend_plan(int n_rows, int n_seqs, int n_heads, int n_kv_heads, int head_dim, int prefix_len,
                              int max_len, bool ragged, int cus) {
  AttendPlan p{};
  const int64_t g = n_heads / n_kv_heads, cols = n_rows * g;
  const int64_t want = 4 * (int64_t)cus;
  auto split = [&](int64_t units, int64_t keys, int *splits, int *chunk) {
    int64_t n = at_ceil(want, units > 0 ? units : 1);
    const int64_t most = at_ceil(keys, 128);
    n = n > most ? most : n;
    n = n < 1 ? 1 : n;
    const int64_t c = at_ceil(at_ceil(keys, n), AT_KEYS) * AT_KEYS;
    *chunk = (int)c;
    *splits = (int)at_ceil(keys, c);
  };
  if (prefix_len > 0) {
    p.pre_tiles = (int)at_ceil(cols, AT_COLS);
    split((int64_t)p.pre_tiles * n_kv_heads, prefix_len, &p.pre_splits, &p.pre_chunk);
  }
  if (max_len > 0) {
    // sequence s's tiles start at slot floor(row_start[s] g / 16) + s
    p.own_slots = (int)(ragged ? cols / AT_COLS + n_seqs : n_seqs * at_ceil(g, AT_COLS));
    split((int64_t)p.own_slots * n_kv_heads, max_len, &p.own_splits, &p.own_chunk);
  }
  const int64_t slots = p.pre_splits + p.own_splits, items = slots * n_rows * n_heads;
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

// whether an element of a value lane is not finite
template <typename CT>
__device__ __forceinline__ bool at_odd(uint32_t w) {
  if (sizeof(CT) == 4) return (w & 0x7f800000u) == 0x7f800000u;
  constexpr uint32_t e = __is_same(CT, __bf16) ? 0x7f80u : 0x7c00u;
  return (w & e) == e || ((w >> 16) & e) == e;
}

template <typename RT, typename CT, int HD>
__global__ __launch_bounds__(64 * AT_WAVES) void paged_attend_kernel(AttendArgs a) {
  using Y = AtTypes<RT, CT, HD>;
  constexpr int VW = Y::F32 ? Y::VE : Y::VE / 2;  // 32-bit words of a value lane's key
  __shared__ float so[AT_WAVES][Y::VE][64 * 4];
  __shared__ float sm[AT_WAVES][AT_COLS], sl[AT_WAVES][AT_COLS];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, g = lane >> 4, c = lane & 15;
  const int hkv = a.kv.n_kv_heads, kvh = blockIdx.x % hkv;
  int b = blockIdx.x / hkv, slot;

  // the block's keys [k0, k1) by page ids, and its column: row, head, keys seen
  const int *ids;
  int n_ids, k0, k1, row = -1, seen = 0;
  const int head = kvh * a.group;
  int col;
  if (b < a.pre_tiles * a.pre_splits) {
    slot = b / a.pre_tiles;
    col = (b - slot * a.pre_tiles) * AT_COLS + c;
    const int rows = a.row_start ? at_row(a.row_start, a.n_seqs, a.n_rows) : a.n_rows;
    if (col - c >= rows * a.group) return;
    if (col < rows * a.group) row = col / a.group;
    ids = a.prefix_pages;
    n_ids = a.prefix_count;
    k0 = slot * a.pre_chunk;
    k1 = min(a.prefix_len, k0 + a.pre_chunk);
    seen = k1;
  } else {
    b -= a.pre_tiles * a.pre_splits;
    slot = b / a.own_slots;
    b -= slot * a.own_slots;
    int s, tile, r0, r1;
    if (a.row_start) {
      s = at_search(a.n_seqs, b, [&](int i) { return at_row(a.row_start, i, a.n_rows) * a.group / AT_COLS + i; });
      if (s < 0) return;
      r0 = at_row(a.row_start, s, a.n_rows);
      r1 = at_row(a.row_start, s + 1, a.n_rows);
      tile = b - (r0 * a.group / AT_COLS + s);
    } else {
      const int tiles = (a.group + AT_COLS - 1) / AT_COLS;
      s = b / tiles;
      tile = b - s * tiles;
      r0 = s;
      r1 = s + 1;
    }
    col = tile * AT_COLS + c;
    const int cols = (r1 - r0) * a.group;
    if (col - c >= cols) return;
    const int j = min(col, cols - 1) / a.group;
    // the last column of the tile sees the most
    const int last = min(col - c + AT_COLS, cols) - 1, len = min(max(a.lens[s], 0), a.max_len + (r1 - r0));
    seen = min(len - (r1 - r0 - 1 - j), a.max_len);
    k0 = slot * a.own_chunk;
    k1 = min(min(len - (r1 - r0 - 1 - last / a.group), a.max_len), k0 + a.own_chunk);
    if (k1 <= k0) return;
    seen = min(seen, k1);
    if (col < cols) row = r0 + j;
    else seen = k1;
    ids = a.table + (int64_t)s * a.table_stride;
    n_ids = a.table_width;
    slot += a.pre_splits;
  }
  const int hq = row >= 0 ? head + (col - col / a.group * a.group) : 0;

  AtWave<RT, CT, HD> w;
  w.init(row >= 0 ? (const RT *)a.q + row * a.q_row + hq * a.q_head : nullptr, a.scale);

  // what the column that sees least sees: keys before it need no mask
  int least = seen;
  least = min(least, __shfl_xor(least, 1, 64));
  least = min(least, __shfl_xor(least, 2, 64));
  least = min(least, __shfl_xor(least, 4, 64));
  least = min(least, __shfl_xor(least, 8, 64));

  const CT *kb = (const CT *)a.kv.k + kvh * a.kv.head_stride, *vb = (const CT *)a.kv.v + kvh * a.kv.head_stride;
  const int64_t ts = a.kv.token_stride;
  const int64_t k_lane = c * ts + (Y::F32 ? 4 * g : 8 * g), v_lane = 4 * g * ts + Y::VE * c;
  for (int base = k0; base < k1; base += 1024) {
    // lane i holds the page of keys base + 16 i ..
    const int my_page = base + 16 * lane < k1 ? pg_page(ids, n_ids, base + 16 * lane, a.kv.page_shift, a.kv.n_pages) : -1;
    for (int t = wave; t < 32 && base + AT_KEYS * t < k1; t += AT_WAVES) {
      const int key0 = base + AT_KEYS * t;
      u32x4 k[2][Y::KC];
      uint32_t v[8][VW];
      bool whole = least >= key0 + AT_KEYS, there[2];
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int page = __builtin_amdgcn_readlane(my_page, 2 * t + h);
        there[h] = page >= 0;
        whole = whole && there[h];
        // an absent tile reads the pool's first page, and sees none of it
        const int64_t at = there[h] ? page * a.kv.page_stride + ((key0 + 16 * h) & (a.kv.page_size - 1)) * ts : 0;
#pragma unroll
        for (int j = 0; j < Y::KC; j++) k[h][j] = *(const u32x4 *)(kb + at + k_lane + (Y::F32 ? 16 : 32) * j);
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const CT *p = vb + at + v_lane + i * ts;
          if constexpr (VW == 2) {
            const u32x2 x = *(const u32x2 *)p;
            v[4 * h + i][0] = x[0];
            v[4 * h + i][1] = x[1];
          } else {
#pragma unroll
            for (int y = 0; y < VW; y += 4) {
              const u32x4 x = *(const u32x4 *)(p + y * 4 / sizeof(CT));
#pragma unroll
              for (int z = 0; z < 4; z++) v[4 * h + i][y + z] = x[z];
            }
          }
        }
      }
      float x[8];
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const f32x4 s = w.score(k[h]);
#pragma unroll
        for (int i = 0; i < 4; i++) x[4 * h + i] = s[i] * w.qs;
      }
      bool odd = false;
      if (!whole) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const int key = key0 + 16 * (j >> 2) + 4 * g + (j & 3);
          if (key >= seen || !there[j >> 2]) x[j] = -INFINITY;
          // a value that no column sees may be anything, and 0 times it not 0
          const bool none = key >= k1 || !there[j >> 2];
#pragma unroll
          for (int y = 0; y < VW; y++) {
            if (none) v[j][y] = 0;
            odd = odd || (key >= least && at_odd<CT>(v[j][y]));
          }
        }
      }
      w.softmax(x);
      if (!__any(odd)) {
        w.values(x, v);
      } else {
        // A value that only some columns see is not finite: one column at a
        // time, with the values it does not see put to zero.
        for (int cc = 0; cc < AT_COLS; cc++) {
          const int lim = __builtin_amdgcn_readlane(seen, cc);
          uint32_t u[8][VW];
          f32x4 keep[Y::VE];
#pragma unroll
          for (int j = 0; j < 8; j++)
#pragma unroll
            for (int y = 0; y < VW; y++)
              u[j][y] = key0 + 16 * (j >> 2) + 4 * g + (j & 3) < lim ? v[j][y] : 0;
#pragma unroll
          for (int e = 0; e < Y::VE; e++) keep[e] = w.o[e];
          w.values(x, u);
#pragma unroll
          for (int e = 0; e < Y::VE; e++)
#pragma unroll
            for (int i = 0; i < 4; i++) w.o[e][i] = c == cc ? w.o[e][i] : keep[e][i];
        }
      }
    }
  }

  // join the waves' states: each scaled to the common maximum
  w.l = at_sum4(w.l);
  if (g == 0) {
    sm[wave][c] = w.m;
    sl[wave][c] = w.l;
  }
  __syncthreads();
  float m = sm[0][c];
#pragma unroll
  for (int i = 1; i < AT_WAVES; i++) m = fmaxf(m, sm[i][c]);
  // (a state without a maximum holds zeros, or NaN, which must not get lost)
  const float f = w.m == -INFINITY ? 1.0f : at_exp2(w.m - m);
#pragma unroll
  for (int e = 0; e < Y::VE; e++) *(f32x4 *)&so[wave][e][lane * 4] = w.o[e] * f;
  __syncthreads();
  // thread (lane ln, i): dimensions VE (4 (ln >> 4) + i) .. of column ln & 15
  const int ln = tid >> 2, i = tid & 3, cc = ln & 15;
  const int row2 = __shfl(row, cc, 64), hq2 = __shfl(hq, cc, 64);
  if (row2 < 0) return;
  float y[Y::VE];
#pragma unroll
  for (int e = 0; e < Y::VE; e++) {
    y[e] = so[0][e][tid];
#pragma unroll
    for (int u = 1; u < AT_WAVES; u++) y[e] += so[u][e][tid];
  }
  const int64_t item = ((int64_t)slot * a.n_rows + row2) * a.n_heads + hq2;
  pg_store(a.part_o + item * HD + Y::VE * (4 * (ln >> 4) + i), y);
  if (ln < AT_COLS && i == 0) {
    float mm = sm[0][cc], l = 0;
#pragma unroll
    for (int u = 1; u < AT_WAVES; u++) mm = fmaxf(mm, sm[u][cc]);
#pragma unroll
    for (int u = 0; u < AT_WAVES; u++) l += sl[u][cc] * (sm[u][cc] == -INFINITY ? 1.0f : at_exp2(sm[u][cc] - mm));
    a.part_ml[item] = make_float2(mm, l);
  }
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
  if (a.lse && lane == 0) a.lse[item] = l == 0 ? -INFINITY : (m == -INFINITY ? l : (m + log2f(l)) * 0.6931471805599453f);
}

}  // namespace vx
