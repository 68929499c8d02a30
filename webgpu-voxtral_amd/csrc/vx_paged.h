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
// eight elements at p, aligned to 16 bytes, as they are, and as f32
template <typename T>
struct PgEight {
  static constexpr int W = sizeof(T) / 2, C = 16 / sizeof(T);
  u32x4 w[W];
  __device__ __forceinline__ void load(const T *p) {
#pragma unroll
    for (int i = 0; i < W; i++) w[i] = *(const u32x4 *)(p + i * C);
  }
  __device__ __forceinline__ void get(float (&y)[8]) const {
#pragma unroll
    for (int i = 0; i < W; i++) {
      const PgVec<T, C> v = __builtin_bit_cast(PgVec<T, C>, w[i]);
#pragma unroll
      for (int j = 0; j < C; j++) y[i * C + j] = (float)v.x[j];
    }
  }
};
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
struct AppendRows {
  PagedKV kv;
  const void *k, *v, *q;
  void *q_out;
  int64_t k_row, k_head, v_row, v_head, q_row, q_head, o_row, o_head;
  int rotary_dim, interleaved;
};
struct AppendArgs {
  AppendRows rows;
  const int *pos, *seq, *table;
  int64_t table_stride;
  int table_width, base, n_tokens, n_seqs, n_heads, head_dim;
  // revolutions a position for each pair: theta^(-2 i / rotary_dim) / (2 pi).
  // In 64 bits: at position 10^6 an f32 frequency is off by 0.06 radians.
  double turns[64];
};

constexpr int PA_NT = 256;

// One block a token: its 64 angles are reduced to a revolution in 64 bits and
// their sine and cosine taken once, then shared by every head through LDS.
// A thread moves chunks of 16 elements, two at a time: neighbouring eights, or
// those of the two halves of a pair when pairs are (i, i + rotary_dim / 2).
// Bound by memory where there are many tokens, by latency where there are few:
// the first two chunks are asked for before the token's page and angles are
// known (3908 f16 tokens of 32 + 8 + 8 heads, 94 MB: 30 -> 22.5 us = 4.2 TB/s;
// 8 tokens 5.1 -> 4.0 us).
template <typename RT>
struct PaChunk {
  int h, c, d0, d1;  // head (keys, values, queries), chunk, its elements' places
  bool turned;
  PgEight<RT> x, y;
  __device__ __forceinline__ void load(const AppendRows &a, int t, int w, int per) {
    const int hkv = a.kv.n_kv_heads;
    h = w / per;
    c = w - h * per;
    const RT *src = h < hkv ? (const RT *)a.k + t * a.k_row + h * a.k_head
                    : h < 2 * hkv ? (const RT *)a.v + t * a.v_row + (h - hkv) * a.v_head
                                  : (const RT *)a.q + t * a.q_row + (h - 2 * hkv) * a.q_head;
    turned = c < (a.rotary_dim >> 4) && (h < hkv || h >= 2 * hkv);
    d0 = 16 * c;
    d1 = d0 + 8;
    if (turned && !a.interleaved) d0 = 8 * c, d1 = d0 + (a.rotary_dim >> 1);
    x.load(src + d0);
    y.load(src + d1);
  }
  template <typename CT>
  __device__ __forceinline__ void store(const AppendRows &a, int t, int64_t at, const float *cs, const float *sn) const {
    const int hkv = a.kv.n_kv_heads;
    float u[8], v[8];
    x.get(u);
    y.get(v);
    if (turned) {
      if (a.interleaved) {  // u holds pairs 8 c .. 8 c + 3, v the next four
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          const float c0 = cs[8 * c + j / 2], s0 = sn[8 * c + j / 2], c1 = cs[8 * c + 4 + j / 2], s1 = sn[8 * c + 4 + j / 2];
          const float p = u[j], q = u[j + 1], e = v[j], f = v[j + 1];
          u[j] = p * c0 - q * s0;
          u[j + 1] = p * s0 + q * c0;
          v[j] = e * c1 - f * s1;
          v[j + 1] = e * s1 + f * c1;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const float c0 = cs[8 * c + j], s0 = sn[8 * c + j], p = u[j], q = v[j];
          u[j] = p * c0 - q * s0;
          v[j] = p * s0 + q * c0;
        }
      }
    }
    if (h < 2 * hkv) {
      CT *dst = h < hkv ? (CT *)a.kv.k + at + h * a.kv.head_stride : (CT *)a.kv.v + at + (h - hkv) * a.kv.head_stride;
      pg_store(dst + d0, u);
      pg_store(dst + d1, v);
    } else {
      RT *dst = (RT *)a.q_out + t * a.o_row + (h - 2 * hkv) * a.o_head;
      pg_store(dst + d0, u);
      pg_store(dst + d1, v);
    }
  }
};

template <typename RT, typename CT>
__global__ __launch_bounds__(PA_NT) void paged_append_kernel(AppendArgs args) {
  __shared__ float cs[64], sn[64];
  const AppendRows rows = args.rows;  // (the angles' table is indexed: by itself, it stays in the arguments)
  const int t = blockIdx.x, tid = threadIdx.x;
  const int per = args.head_dim >> 4, chunks = (2 * rows.kv.n_kv_heads + (rows.q ? args.n_heads : 0)) * per;
  PaChunk<RT> w0, w1;
  if (tid < chunks) w0.load(rows, t, tid, per);
  if (tid + PA_NT < chunks) w1.load(rows, t, tid + PA_NT, per);
  const int p = args.pos[t], s = args.seq ? args.seq[t] : t;
  if (p < 0 || s < 0 || s >= args.n_seqs) return;
  const int64_t slot = (int64_t)p - args.base;
  const int page = pg_page(args.table + (int64_t)s * args.table_stride, args.table_width, slot, rows.kv.page_shift, rows.kv.n_pages);
  if (page < 0) return;
  if (tid < rows.rotary_dim >> 1) {
    const double r = p * args.turns[tid];
    sincospif(2.0f * (float)(r - rint(r)), &sn[tid], &cs[tid]);
  }
  __syncthreads();
  const int64_t at = page * rows.kv.page_stride + (slot & (rows.kv.page_size - 1)) * rows.kv.token_stride;
  if (tid < chunks) w0.template store<CT>(rows, t, at, cs, sn);
  if (tid + PA_NT < chunks) w1.template store<CT>(rows, t, at, cs, sn);
  for (int i = tid + 2 * PA_NT; i < chunks; i += PA_NT) {
    w0.load(rows, t, i, per);
    w0.template store<CT>(rows, t, at, cs, sn);
  }
}

// ----------------------------------------------------------------- attend
// Row r of sequence s, the j-th of its n_s rows: one softmax over the shared
// prefix's keys and the first clamp(lens[s] - (n_s - 1 - j), 0, max_len) keys
// of the sequence.  Columns: the n_s rows times the G query heads of a KV
// head, row-major.  Blocks of the first kind take the prefix with the columns
// of all rows, so its keys are read once for many columns and not once a
// sequence; blocks of the second kind take a sequence's own keys and, where
// `fused`, the prefix before them.  Both split the key axis and leave
// (o, m, l) partials that a second kernel joins, unless there is one split in
// all.
//
// Few columns (a decode step's own keys): the block's four waves go to
// different columns, 16 each, or share columns and split the keys; a wave
// brings its keys and values from memory to registers by itself.  That is
// bound by HBM: the matrix cores are all but idle.  Many columns (wide): the
// waves bring 128 keys together through LDS, laid out as the matrix
// instruction's operands, and each takes 32 columns (16 for f32 rows) through
// all of them.  64 columns is where the two meet: a prefix of 2050 keys for 256
// columns a KV head takes 26-32 us in narrow blocks (each of four waves reads
// every key, and their partials are many) and 19 us in wide ones, and 1500 keys
// for 3520 columns 122 and 47 us.
//
// Measured: 64 sequences of 512 own keys (f16, 134 MB) 26.4 us = 5.1 TB/s, 32
// of 8192 (1.07 GB) 181 us = 5.9 TB/s; 64 of 200-900 behind 2050 shared keys
// 39.5 us and 5.3 for the join.
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
  // the plan: columns of a block (over 64: wide), tiles of columns, splits and
  // their keys (multiples of 32)
  int pre_cols, pre_wide, pre_tiles, pre_splits, pre_chunk;
  int own_cols, own_wide, own_slots, own_splits, own_chunk;
  int fused, team;
  float *part_o;   // [slot][row * heads + head][e][r]: dimension VE r + e
  float2 *part_ml; // [slot][row * heads + head]: maximum (log2 units), sum
};

constexpr int AT_COLS = 16;  // columns of a matrix instruction
constexpr int AT_KEYS = 32;  // prefixes and splits are cut in multiples of this
constexpr int AT_WAVES = 4;
constexpr int AT_STAGE = AT_KEYS * AT_WAVES;  // keys that a wide block brings at a time

struct AttendPlan {
  int pre_cols, pre_wide, pre_tiles, pre_splits, pre_chunk, own_cols, own_wide, own_slots, own_splits, own_chunk, fused, team;
  size_t ml_at, bytes;  // the workspace: part_o, then part_ml at ml_at
  int64_t blocks;
  int slots() const { return pre_splits + own_splits; }
  bool direct() const { return slots() == 1; }  // no partials: the blocks write the result
};

__host__ __device__ inline int64_t at_ceil(int64_t a, int64_t b) { return (a + b - 1) / b; }

// wide_cols: columns of a wide block (0: there is none for these types)
inline AttendPlan attend_plan(int n_rows, int n_seqs, int n_heads, int n_kv_heads, int head_dim, int prefix_len,
                              int max_len, bool ragged, int wide_cols, int cus) {
  AttendPlan p{};
  const int64_t g = n_heads / n_kv_heads, cols = n_rows * g;
  // Columns of a block that has `c` of them to choose from: a narrow block's
  // four waves go to columns as far as there are some, the rest to keys.
  auto choose = [&](int64_t c, int *block_cols, int *wide) {
    *wide = wide_cols && c >= 64;
    *block_cols = *wide ? wide_cols : AT_COLS * (c > 32 ? 4 : c > 16 ? 2 : 1);
  };
  auto step_of = [](int block_cols, int wide) { return wide ? AT_STAGE : AT_STAGE * AT_COLS / block_cols; };
  // Splits of `keys` for about `want` blocks, and of at most 2048 keys: long
  // sequences of a batch differ in length, and the longest one's last block is
  // waited for (32 x 4000-16000 keys: 285 us in 3 splits, 255 in 6, 252 in 8).
  auto split = [&](int64_t units, int64_t keys, int64_t step, int64_t want, int *splits, int *chunk) {
    int64_t n = at_ceil(want, units > 0 ? units : 1);
    const int64_t most = at_ceil(keys, step), least = at_ceil(keys, 2048);
    n = n < least ? least : n;
    n = n > most ? most : n;
    n = n < 1 ? 1 : n;
    const int64_t c = at_ceil(at_ceil(keys, n), step) * step;
    *chunk = (int)c;
    *splits = (int)at_ceil(keys, c);
  };
  choose(cols, &p.pre_cols, &p.pre_wide);
  choose(ragged ? cols / (n_seqs > 0 ? n_seqs : 1) : g, &p.own_cols, &p.own_wide);
  // Fused where the prefix costs less than a launch of the join: in wide blocks
  // (its keys serve 128 columns of the sequence as well as of others: 85 us
  // against 85 + 18 at 16 prompts behind 1500 keys), and where all keys are at
  // most 512 (4 x 1-40 behind 100: 8.4 us against 7.0 + 3.5).
  p.fused = prefix_len > 0 && max_len > 0 && (p.own_wide || (int64_t)prefix_len + max_len <= 512);
  if (prefix_len > 0 && !p.fused) {
    p.pre_tiles = (int)at_ceil(cols, p.pre_cols);
    split((int64_t)p.pre_tiles * n_kv_heads, prefix_len, step_of(p.pre_cols, p.pre_wide), cus, &p.pre_splits, &p.pre_chunk);
  }
  if (max_len > 0) {
    const int64_t before = p.fused ? at_ceil(prefix_len, AT_KEYS) * AT_KEYS : 0;
    // sequence s's tiles start at slot floor(row_start[s] g / columns) + s
    p.own_slots = (int)(ragged ? cols / p.own_cols + n_seqs : n_seqs * at_ceil(g, p.own_cols));
    split((int64_t)p.own_slots * n_kv_heads, before + max_len, step_of(p.own_cols, p.own_wide),
          p.fused && !p.own_wide ? 1 : p.own_wide ? cus : 3 * cus, &p.own_splits, &p.own_chunk);
  }
  const int64_t items = p.direct() ? 0 : (int64_t)p.slots() * n_rows * n_heads;
  // a block joins one item's partials instead of four where they are many
  p.team = p.slots() >= 24 ? AT_WAVES : 1;
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
  static constexpr int H = F32 ? 1 : 2;               // tiles of 16 keys in a wave's step
  static constexpr int STEP = 16 * H;
  static constexpr int VE = HD / 16;                  // value instructions, dimensions a lane loads of a key
  static constexpr int VW = F32 ? VE : VE / 2;        // 32-bit words of a key a value lane loads
  static constexpr int KC = F32 ? HD / 16 : HD / 32;  // 16-byte chunks of a key a lane holds
  static constexpr int WIDE = F32 ? 0 : SPLIT ? 1 : 2;  // column tiles of a wave in a wide block
};
// columns of a wide block by the sizes of row and cache elements
inline int at_wide_cols(size_t row, size_t cache) { return cache == 4 ? 0 : AT_WAVES * AT_COLS * (row == 4 ? 1 : 2); }

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

// One tile of 16 columns in a wave: queries, sums, maximum
template <typename RT, typename CT, int HD>
struct AtTile {
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

  // s += the products of chunk j of 16 keys
  __device__ __forceinline__ f32x4 score(u32x4 k, int j, f32x4 s) const {
    if constexpr (Y::F32) {
      const f32x4 a = __builtin_bit_cast(f32x4, k), b = __builtin_bit_cast(f32x4, q[j]);
#pragma unroll
      for (int i = 0; i < 4; i++) s = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], s, 0, 0, 0);
    } else {
      s = at_mma(__builtin_bit_cast(E8, k), __builtin_bit_cast(E8, q[j]), s);
      if constexpr (Y::SPLIT) s = at_mma(__builtin_bit_cast(E8, k), __builtin_bit_cast(E8, q[Y::KC + j]), s);
    }
    return s;
  }

  // the weights of a step's scores (in log2 units; -inf: not seen), with the running
  // maximum moved where one passes it by more than 8: until then weights of up
  // to 2^8 do no harm, and the sums need not be scaled
  __device__ __forceinline__ void softmax(float (&x)[4 * Y::H]) {
    float top = x[0];
#pragma unroll
    for (int j = 1; j < 4 * Y::H; j++) top = fmaxf(top, x[j]);
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
    for (int j = 0; j < 4 * Y::H; j++) {
      x[j] = at_exp2(x[j] - z);
      l += x[j];
    }
  }

  // 16-bit caches: the weights as B operands, hi and lo
  __device__ __forceinline__ void weights(const float (&p)[8], E8 (&b)[Y::SPLIT ? 2 : 1]) const {
    if constexpr (Y::SPLIT) {
      split_n(p, b[0], b[1]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) b[0][j] = (CT)p[j];
    }
  }
  __device__ __forceinline__ void value(int e, u32x4 v, const E8 (&b)[Y::SPLIT ? 2 : 1]) {
    o[e] = at_mma(__builtin_bit_cast(E8, v), b[0], o[e]);
    if constexpr (Y::SPLIT) o[e] = at_mma(__builtin_bit_cast(E8, v), b[1], o[e]);
  }

  // Adds the elements that are not finite of a step's rows (bit r of `rows`:
  // row r & 15 of the tile at `place(r >> 4)`) to the columns that see them, each lane
  // to its own dimensions.  They were taken out of the common product, where
  // 0 times them would not be 0 for the columns that do not see them.
  template <typename F>
  __device__ __forceinline__ void add_odd(uint32_t rows, const float (&p)[4 * Y::H], int limit, int ts, F place) {
    const int g = (threadIdx.x & 63) >> 4, c = threadIdx.x & 15;
    while (rows) {
      const int r = __ffs(rows) - 1, j = 4 * (r >> 4) + (r & 3);
      rows &= rows - 1;
      float pj = p[0];
#pragma unroll
      for (int i = 1; i < 4 * Y::H; i++) pj = i == j ? p[i] : pj;
      const float weight = __shfl(pj, (r & 12) * 4 + c, 64);
      const CT *row = (const CT *)(place(r >> 4) + (int64_t)(r & 15) * ts) + 4 * Y::VE * g;
      if (r < limit) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
          float y[Y::VE];
          pg_load(row + Y::VE * i, y);
#pragma unroll
          for (int e = 0; e < Y::VE; e++)
            if (!(fabsf(y[e]) < INFINITY)) o[e][i] = fmaf(weight, y[e], o[e][i]);
        }
      }
    }
  }

  // the column's result or partial; the lane's dimensions are 4 VE from 4 VE g on
  __device__ __forceinline__ void store(const AttendArgs &a, int slot, int row, int head) {
    const int g = (threadIdx.x & 63) >> 4;
    l = at_sum4(l);
    if (row < 0) return;
    if (a.pre_splits + a.own_splits == 1) {
      const float r = l == 0 ? 0.0f : 1.0f / l;
      RT *out = (RT *)a.out + row * a.o_row + head * a.o_head + 4 * Y::VE * g;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        float y[Y::VE];
#pragma unroll
        for (int e = 0; e < Y::VE; e++) y[e] = o[e][i] * r;
        pg_store(out + Y::VE * i, y);
      }
      if (a.lse && g == 0) a.lse[(int64_t)row * a.n_heads + head] = at_lse(m, l);
      return;
    }
    const int64_t item = ((int64_t)slot * a.n_rows + row) * a.n_heads + head;
#pragma unroll
    for (int e = 0; e < Y::VE; e++) *(f32x4 *)(a.part_o + item * HD + 16 * e + 4 * g) = o[e];
    if (g == 0) a.part_ml[item] = make_float2(m, l);
  }
};

// What a block works on.  Its keys are a run [k0, k1) of one or two page
// lists laid end to end: the prefix up to `pre` (then up to `before`, in whole
// steps), then a sequence's own.  Its columns are first .. first + 15 and so
// on, those below `cols` exist; column x is row r0 + x / group.
struct AtJob {
  const int *ids, *prefix_ids;
  int n_ids, n_prefix_ids;
  int pre, before, k0, k1, slot, r0, cols, first, len, group, max_len;
  // own keys that a column sees (it does not fall along the columns)
  __device__ __forceinline__ int sees(int x) const { return max(min(len + min(x, cols - 1) / group, max_len), 0); }
};

// The tiles of 16 keys of a run of up to 1024: lane i holds where keys
// base + 16 i .. lie (bytes from the pools' starts).  An absent tile points to
// the first page, and none of it is seen.
struct AtPages {
  int base, at_lo, at_hi;
  uint64_t have;
  __device__ __forceinline__ void look(const AtJob &b, const PagedKV &kv, int from, int stop, int ts, int elem) {
    base = from;
    const int x = from + 16 * (threadIdx.x & 63);
    int page = -1, slot = 0;
    if (x < b.before) {
      slot = x;
      if (x < b.pre) page = pg_page(b.prefix_ids, b.n_prefix_ids, x, kv.page_shift, kv.n_pages);
    } else if (x < stop) {
      slot = x - b.before;
      page = pg_page(b.ids, b.n_ids, slot, kv.page_shift, kv.n_pages);
    }
    have = __ballot(page >= 0);
    const int64_t at = page < 0 ? 0 : page * kv.page_stride * elem + (int64_t)(slot & (kv.page_size - 1)) * ts;
    at_lo = (int)at;
    at_hi = (int)(at >> 32);
  }
  // tile h of the step at x
  __device__ __forceinline__ int64_t place(int x, int h) const {
    const int i = ((x - base) >> 4) + h;
    return (int64_t)__builtin_amdgcn_readlane(at_hi, i) << 32 | (uint32_t)__builtin_amdgcn_readlane(at_lo, i);
  }
  // which tiles of a step of h are there, as bits
  __device__ __forceinline__ uint32_t there(int x, int h) const { return (uint32_t)(have >> ((x - base) >> 4)) & ((1u << h) - 1); }
};

// A wave's registers for the keys and values of one step
template <typename RT, typename CT, int HD>
struct AtStep {
  using Y = AtTypes<RT, CT, HD>;
  u32x4 k[Y::H][Y::KC];
  uint32_t v[4 * Y::H][Y::VW];  // the lane's dimensions of key 4 g + (j & 3) of tile j >> 2

  // Of the step at x: uniform addresses of the tiles and 32-bit offsets of the
  // lanes, so that the loads take their base from scalar registers.  The empty
  // asm keeps an offset's widening to 64 bits next to its loads: moved out of
  // the loop, it hides from the compiler that the high half is zero, and every
  // load's address becomes a pair of vector registers.
  __device__ __forceinline__ void load_k(const char *pool, const AtPages &at, int x, uint32_t lane) {
    asm volatile("" : "+v"(lane));
#pragma unroll
    for (int h = 0; h < Y::H; h++) {
      const char *p = pool + at.place(x, h);
#pragma unroll
      for (int j = 0; j < Y::KC; j++) k[h][j] = *(const u32x4 *)(p + lane + 64 * j);
    }
  }
  __device__ __forceinline__ void load_v(const char *pool, const AtPages &at, int x, uint32_t lane, int ts) {
    asm volatile("" : "+v"(lane));
#pragma unroll
    for (int h = 0; h < Y::H; h++) {
      const char *p = pool + at.place(x, h);
#pragma unroll
      for (int i = 0; i < 4; i++, p += ts) {
        if constexpr (Y::VW == 2) {
          const u32x2 y = *(const u32x2 *)(p + lane);
          v[4 * h + i][0] = y[0];
          v[4 * h + i][1] = y[1];
        } else {
#pragma unroll
          for (int z = 0; z < Y::VW; z += 4) {
            const u32x4 y = *(const u32x4 *)(p + lane + 4 * z);
#pragma unroll
            for (int u = 0; u < 4; u++) v[4 * h + i][z + u] = y[u];
          }
        }
      }
    }
  }
  // Values that no column sees (from row `any` on, or in an absent tile) may
  // be anything, and 0 times them not 0: they are put to zero.  What is not
  // finite from row `all` on, which not all columns see, is too, and its rows
  // are returned.
  __device__ __forceinline__ uint32_t clean(uint32_t there, int all, int any) {
    const int g = (threadIdx.x & 63) >> 4;
    uint32_t rows = 0;
#pragma unroll
    for (int j = 0; j < 4 * Y::H; j++) {
      const int row = 16 * (j >> 2) + 4 * g + (j & 3);
      const bool none = !(there >> (j >> 2) & 1) | (row >= any);
      bool bad = false;
#pragma unroll
      for (int y = 0; y < Y::VW; y++) {
        v[j][y] = none ? 0 : v[j][y];
        bad |= at_odd<CT>(v[j][y]);
      }
      bad &= row >= all;
      const uint64_t lanes = __ballot(bad);
      if (lanes) {
#pragma unroll
        for (int y = 0; y < Y::VW; y++) v[j][y] = bad ? at_finite<CT>(v[j][y]) : v[j][y];
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (lanes >> (16 * i) & 0xffff) rows |= 1u << (16 * (j >> 2) + 4 * i + (j & 3));
      }
    }
    return rows;
  }
  // 16-bit caches: the A operands of value instructions 2 w and 2 w + 1
  __device__ __forceinline__ void turn(int w, u32x4 &a, u32x4 &b) const {
#pragma unroll
    for (int j = 0; j < 4; j++) {  // key pairs: the low halves, the high halves
      a[j] = __builtin_amdgcn_perm(v[2 * j + 1][w], v[2 * j][w], 0x05040100u);
      b[j] = __builtin_amdgcn_perm(v[2 * j + 1][w], v[2 * j][w], 0x07060302u);
    }
  }
};

// hides what a column does not see: keys from row `limit` on, absent tiles
template <int N>
__device__ __forceinline__ void at_hide(float (&p)[N], uint32_t there, int limit) {
  const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int j = 0; j < N; j++) {
    const bool is = (there >> (j >> 2) & 1) & (16 * (j >> 2) + 4 * g + (j & 3) < limit);
    p[j] = is ? p[j] : -INFINITY;
  }
}

template <typename RT, typename CT, int HD, bool WIDE>
struct AtLds {
  using Y = AtTypes<RT, CT, HD>;
  static constexpr int JOIN = (AT_WAVES - 1) * Y::VE * 64;             // states of the waves that share columns
  static constexpr int K = WIDE ? AT_WAVES * Y::H * Y::KC * 64 : 0;    // operands of a stage's keys
  static constexpr int V = WIDE ? AT_WAVES * Y::VE * 64 : 0;           // ... and values
  u32x4 x[JOIN > K + V ? JOIN : K + V];
  float m[AT_WAVES - 1][64], l[AT_WAVES - 1][64];
  uint32_t rows[AT_WAVES];  // of each step of the stage: what clean() returned
};

// Few columns: 16 a wave; waves with the same ones split the keys.  Asking one
// step ahead took 24 sequences on an f32 cache from 35 to 25 us; steps of 16
// keys there (as many bytes in flight, half the registers) to 23.
template <typename RT, typename CT, int HD>
__device__ __forceinline__ void at_narrow(const AttendArgs &a, const AtJob &b, int cols, int kvh, u32x4 *so,
                                          float (*sm)[64], float (*sl)[64]) {
  using Y = AtTypes<RT, CT, HD>;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int col_waves = cols / AT_COLS, key_waves = AT_WAVES / col_waves, key_wave = wave / col_waves;
  const int first = b.first + wave % col_waves * AT_COLS, col = first + c;
  const int row = col < b.cols ? b.r0 + col / b.group : -1, head = kvh * b.group + col % b.group;
  const int seen = b.sees(col), least = b.sees(first), most = b.sees(first + AT_COLS - 1);
  AtTile<RT, CT, HD> w;
  w.init(row >= 0 ? (const RT *)a.q + row * a.q_row + head * a.q_head : nullptr, a.scale);

  const char *kb = (const char *)a.kv.k + kvh * a.kv.head_stride * (int64_t)sizeof(CT);
  const char *vb = (const char *)a.kv.v + kvh * a.kv.head_stride * (int64_t)sizeof(CT);
  const int ts = (int)a.kv.token_stride * (int)sizeof(CT), stride = Y::STEP * key_waves;
  const uint32_t k_lane = c * ts + 16 * g, v_lane = 4 * g * ts + Y::VE * c * (int)sizeof(CT);
  AtStep<RT, CT, HD> t;
  AtPages at;
  for (int base = b.k0; base < b.k1; base += 1024) {
    const int stop = min(b.k1, base + 1024);
    at.look(b, a.kv, base, stop, ts, sizeof(CT));
    int x = base + Y::STEP * key_wave;
    if (x >= stop) continue;
    t.load_k(kb, at, x, k_lane);
    t.load_v(vb, at, x, v_lane, ts);
    // The next step's keys are asked for when this one's scores are taken, its
    // values when this one's are summed: one of the two is always on its way.
    // The last step asks for itself again, so that the number of loads in
    // flight is the same on every path and the waits can be exact.
    for (;;) {
      const int next = x + stride < stop ? x + stride : x;
      float p[4 * Y::H];
#pragma unroll
      for (int h = 0; h < Y::H; h++) {
        f32x4 d{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < Y::KC; j++) d = w.score(t.k[h][j], j, d);
#pragma unroll
        for (int i = 0; i < 4; i++) p[4 * h + i] = d[i] * w.qs;
      }
      t.load_k(kb, at, next, k_lane);
      const uint32_t there = at.there(x, Y::H);
      const bool shared = x < b.before;
      const int x0 = shared ? x : x - b.before;  // in its list
      uint32_t rows = 0;
      if ((shared ? b.pre : least) < x0 + Y::STEP || there != (1u << Y::H) - 1) {
        at_hide(p, there, (shared ? b.pre : seen) - x0);
        rows = t.clean(there, (shared ? b.pre : least) - x0, (shared ? b.pre : most) - x0);
      }
      w.softmax(p);
      if (rows) w.add_odd(rows, p, (shared ? b.pre : seen) - x0, ts, [&](int h) { return vb + at.place(x, h); });
      if constexpr (Y::F32) {
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
          for (int e = 0; e < Y::VE; e++)
            w.o[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, t.v[j][e]), p[j], w.o[e], 0, 0, 0);
      } else {
        typename At8<CT>::T pb[Y::SPLIT ? 2 : 1];
        w.weights(p, pb);
#pragma unroll
        for (int i = 0; i < Y::VE / 2; i++) {
          u32x4 u, v;
          t.turn(i, u, v);
          w.value(2 * i, u, pb);
          w.value(2 * i + 1, v, pb);
        }
      }
      t.load_v(vb, at, next, v_lane, ts);
      if (next == x) break;
      x = next;
    }
  }

  // the waves with the same columns join their states in the first one's
  if (key_waves > 1) {
    if (key_wave > 0) {
      const int i = wave - col_waves;
#pragma unroll
      for (int e = 0; e < Y::VE; e++) so[(i * Y::VE + e) * 64 + lane] = __builtin_bit_cast(u32x4, w.o[e]);
      sm[i][lane] = w.m;
      sl[i][lane] = w.l;
    }
    __syncthreads();
    if (key_wave > 0) return;
    for (int k = 1; k < key_waves; k++) {
      const int i = wave + (k - 1) * col_waves;
      const float m1 = sm[i][lane], m = fmaxf(w.m, m1);
      // (a state without a maximum holds zeros, or NaN, which must not get lost)
      const float f0 = w.m == -INFINITY ? 1.0f : at_exp2(w.m - m), f1 = m1 == -INFINITY ? 1.0f : at_exp2(m1 - m);
      w.m = m;
      w.l = w.l * f0 + sl[i][lane] * f1;
#pragma unroll
      for (int e = 0; e < Y::VE; e++) w.o[e] = w.o[e] * f0 + __builtin_bit_cast(f32x4, so[(i * Y::VE + e) * 64 + lane]) * f1;
    }
  }
  w.store(a, b.slot, row, head);
}

// Many columns: a stage is 128 keys, 32 brought by each wave, and every wave
// takes them all through its own columns.  16 prompts of 20-90 rows behind 1500
// keys (27.5 GFLOP, bf16): 153 us in narrow blocks, 89 in wide ones with the
// prefix before each sequence's own keys and nothing to join.
template <typename RT, typename CT, int HD>
__device__ __forceinline__ void at_wide(const AttendArgs &a, const AtJob &b, int kvh, AtLds<RT, CT, HD, true> &s) {
  using Y = AtTypes<RT, CT, HD>;
  constexpr int N = Y::WIDE;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int first = b.first + wave * N * AT_COLS;
  AtTile<RT, CT, HD> w[N];
  int row[N], head[N], seen[N];
#pragma unroll
  for (int n = 0; n < N; n++) {
    const int col = first + n * AT_COLS + c;
    row[n] = col < b.cols ? b.r0 + col / b.group : -1;
    head[n] = kvh * b.group + col % b.group;
    seen[n] = b.sees(col);
    w[n].init(row[n] >= 0 ? (const RT *)a.q + row[n] * a.q_row + head[n] * a.q_head : nullptr, a.scale);
  }
  const int least = b.sees(first), most = b.sees(first + N * AT_COLS - 1);          // of the wave's columns
  const int block_least = b.sees(b.first), block_most = b.sees(b.first + AT_WAVES * N * AT_COLS - 1);
  const bool idle = first >= b.cols;

  const char *kb = (const char *)a.kv.k + kvh * a.kv.head_stride * (int64_t)sizeof(CT);
  const char *vb = (const char *)a.kv.v + kvh * a.kv.head_stride * (int64_t)sizeof(CT);
  const int ts = (int)a.kv.token_stride * (int)sizeof(CT);
  const uint32_t k_lane = c * ts + 16 * g, v_lane = 4 * g * ts + Y::VE * c * (int)sizeof(CT);
  u32x4 *const sk = s.x, *const sv = s.x + AtLds<RT, CT, HD, true>::K;
  AtStep<RT, CT, HD> t;
  AtPages at;
  for (int base = b.k0; base < b.k1; base += 1024) {
    const int stop = min(b.k1, base + 1024), end = base + ((stop - 1 - base) & -AT_KEYS);  // the last step's start
    at.look(b, a.kv, base, stop, ts, sizeof(CT));
    auto load = [&](int from) {
      const int x = min(from + AT_KEYS * wave, end);
      t.load_k(kb, at, x, k_lane);
      t.load_v(vb, at, x, v_lane, ts);
    };
    load(base);
    for (int from = base; from < stop; from += AT_STAGE) {
      {
        const int x = min(from + AT_KEYS * wave, end);
        const bool shared = x < b.before;
        const int x0 = shared ? x : x - b.before;
        const uint32_t there = at.there(x, Y::H);
        uint32_t rows = 0;
        if ((shared ? b.pre : block_least) < x0 + AT_KEYS || there != 3)
          rows = t.clean(there, (shared ? b.pre : block_least) - x0, (shared ? b.pre : block_most) - x0);
        if (lane == 0) s.rows[wave] = rows;
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
          for (int j = 0; j < Y::KC; j++) sk[((wave * 2 + h) * Y::KC + j) * 64 + lane] = t.k[h][j];
#pragma unroll
        for (int i = 0; i < Y::VE / 2; i++) {
          u32x4 u, v;
          t.turn(i, u, v);
          sv[(wave * Y::VE + 2 * i) * 64 + lane] = u;
          sv[(wave * Y::VE + 2 * i + 1) * 64 + lane] = v;
        }
      }
      __syncthreads();
      if (from + AT_STAGE < stop) load(from + AT_STAGE);
      for (int i = 0; i < AT_WAVES; i++) {
        const int x = from + AT_KEYS * i;
        const bool shared = x < b.before;
        const int x0 = shared ? x : x - b.before;
        if (x >= stop || idle || (!shared && x0 >= most)) break;
        const uint32_t there = at.there(x, Y::H);
        float p[N][8];
#pragma unroll
        for (int h = 0; h < 2; h++) {
          f32x4 d[N];
#pragma unroll
          for (int n = 0; n < N; n++) d[n] = f32x4{0, 0, 0, 0};
#pragma unroll
          for (int j = 0; j < Y::KC; j++) {
            const u32x4 k = sk[((i * 2 + h) * Y::KC + j) * 64 + lane];
#pragma unroll
            for (int n = 0; n < N; n++) d[n] = w[n].score(k, j, d[n]);
          }
#pragma unroll
          for (int n = 0; n < N; n++)
#pragma unroll
            for (int u = 0; u < 4; u++) p[n][4 * h + u] = d[n][u] * w[n].qs;
        }
        const uint32_t rows = __builtin_amdgcn_readfirstlane(s.rows[i]);
        if ((shared ? b.pre : least) < x0 + AT_KEYS || there != 3) {
#pragma unroll
          for (int n = 0; n < N; n++) at_hide(p[n], there, (shared ? b.pre : seen[n]) - x0);
        }
        typename At8<CT>::T pb[N][Y::SPLIT ? 2 : 1];
#pragma unroll
        for (int n = 0; n < N; n++) {
          w[n].softmax(p[n]);
          w[n].weights(p[n], pb[n]);
        }
        if (rows) {
#pragma unroll
          for (int n = 0; n < N; n++)
            w[n].add_odd(rows, p[n], (shared ? b.pre : seen[n]) - x0, ts, [&](int h) { return vb + at.place(x, h); });
        }
#pragma unroll
        for (int e = 0; e < Y::VE; e++) {
          const u32x4 v = sv[(i * Y::VE + e) * 64 + lane];
#pragma unroll
          for (int n = 0; n < N; n++) w[n].value(e, v, pb[n]);
        }
      }
      __syncthreads();
    }
  }
#pragma unroll
  for (int n = 0; n < N; n++) w[n].store(a, b.slot, row[n], head[n]);
}

// WIDE: some of the blocks are wide; their registers and 64 KB of LDS allow 2
// waves on a SIMD, narrow blocks alone 3 (16 KB in flight a wave).
template <typename RT, typename CT, int HD, bool WIDE>
__global__ __launch_bounds__(64 * AT_WAVES, 2) void paged_attend_kernel(AttendArgs a) {
  __shared__ AtLds<RT, CT, HD, WIDE> lds;
  const int hkv = a.kv.n_kv_heads, kvh = blockIdx.x % hkv;
  int i = blockIdx.x / hkv;
  AtJob b{};
  b.prefix_ids = a.prefix_pages;
  b.n_prefix_ids = a.prefix_count;
  b.group = a.group;
  b.max_len = a.max_len;
  bool wide;
  int cols;  // of the block
  if (i < a.pre_tiles * a.pre_splits) {
    wide = a.pre_wide;
    cols = a.pre_cols;
    b.slot = i / a.pre_tiles;
    b.first = (i - b.slot * a.pre_tiles) * cols;
    b.cols = (a.row_start ? at_row(a.row_start, a.n_seqs, a.n_rows) : a.n_rows) * a.group;
    if (b.first >= b.cols) return;
    b.pre = a.prefix_len;
    b.before = (b.pre + AT_KEYS - 1) & -AT_KEYS;
    b.k0 = b.slot * a.pre_chunk;
    b.k1 = min(b.pre, b.k0 + a.pre_chunk);
  } else {
    wide = a.own_wide;
    cols = a.own_cols;
    i -= a.pre_tiles * a.pre_splits;
    const int split = i / a.own_slots;
    i -= split * a.own_slots;
    int s, tile, rows = 1;
    if (a.row_start) {
      s = at_search(a.n_seqs, i, [&](int x) { return at_row(a.row_start, x, a.n_rows) * a.group / cols + x; });
      if (s < 0) return;
      b.r0 = at_row(a.row_start, s, a.n_rows);
      rows = at_row(a.row_start, s + 1, a.n_rows) - b.r0;
      tile = i - (b.r0 * a.group / cols + s);
    } else {
      const int tiles = (a.group + cols - 1) / cols;
      b.r0 = s = i / tiles;
      tile = i - s * tiles;
    }
    b.slot = a.pre_splits + split;
    b.first = tile * cols;
    b.cols = rows * a.group;
    if (b.first >= b.cols) return;
    // the j-th of n rows sees lens - (n - 1 - j) keys
    b.len = min(max(a.lens[s], 0), a.max_len + rows) - (rows - 1);
    b.pre = a.fused ? a.prefix_len : 0;
    b.before = (b.pre + AT_KEYS - 1) & -AT_KEYS;
    b.ids = a.table + (int64_t)s * a.table_stride;
    b.n_ids = a.table_width;
    b.k0 = split * a.own_chunk;
    const int end = b.sees(b.first + cols - 1);
    b.k1 = min(end ? b.before + end : b.pre, b.k0 + a.own_chunk);
    // an empty split is not read by the join; alone, it writes zeros
    if (b.k1 <= b.k0 && a.pre_splits + a.own_splits > 1) return;
  }
  if constexpr (WIDE) {
    if (wide) {
      at_wide<RT, CT, HD>(a, b, kvh, lds);
      return;
    }
  }
  at_narrow<RT, CT, HD>(a, b, cols, kvh, lds.x, lds.m, lds.l);
}

// Joins a row and head's partials: a wave each, or the four waves of a block
// where there are many.  Lane l takes dimensions HD / 64 l ..
template <typename RT, int HD>
__global__ __launch_bounds__(64 * AT_WAVES) void paged_attend_join_kernel(AttendArgs a) {
  constexpr int N = HD / 64, VE = HD / 16;
  __shared__ float sy[AT_WAVES][HD], sl[AT_WAVES];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t items = (int64_t)a.n_rows * a.n_heads;
  const int64_t item = a.team > 1 ? blockIdx.x : (int64_t)blockIdx.x * AT_WAVES + wave;
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
  const int pre = a.fused ? a.prefix_len : 0, before = (pre + AT_KEYS - 1) & -AT_KEYS;
  const int keys = seen > 0 ? before + seen : pre;
  const int parts = a.pre_splits + (keys > 0 ? (keys + a.own_chunk - 1) / a.own_chunk : 0);
  float m = -INFINITY;
  for (int i = lane; i < parts; i += 64) m = fmaxf(m, a.part_ml[i * items + item].x);
  m = wave_max(m);
  // the lane's dimensions N l + j lie at 16 e + r, VE r + e = N l + j
  const int at = N * lane % VE * 16 + N * lane / VE;
  float l = 0, y[N];
#pragma unroll
  for (int j = 0; j < N; j++) y[j] = 0;
  const int first = a.team > 1 ? wave : 0;
#pragma unroll 4
  for (int i = first; i < parts; i += a.team) {
    const float2 ml = a.part_ml[i * items + item];
    const float *o = a.part_o + (i * items + item) * HD + at;
    // (a part without a maximum holds zeros, or NaN, which must not get lost)
    const float f = ml.x == -INFINITY ? 1.0f : at_exp2(ml.x - m);
    l = fmaf(ml.y, f, l);
#pragma unroll
    for (int j = 0; j < N; j++) y[j] = fmaf(o[16 * j], f, y[j]);
  }
  if (a.team > 1) {
#pragma unroll
    for (int j = 0; j < N; j++) sy[wave][N * lane + j] = y[j];
    if (lane == 0) sl[wave] = l;
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int u = 1; u < AT_WAVES; u++) {
      l += sl[u];
#pragma unroll
      for (int j = 0; j < N; j++) y[j] += sy[u][N * lane + j];
    }
  }
  const float r = l == 0 ? 0.0f : 1.0f / l;
#pragma unroll
  for (int j = 0; j < N; j++) y[j] *= r;
  pg_store((RT *)a.out + row * a.o_row + head * a.o_head + N * lane, y);
  if (a.lse && lane == 0) a.lse[item] = at_lse(m, l);
}

}  // namespace vx
