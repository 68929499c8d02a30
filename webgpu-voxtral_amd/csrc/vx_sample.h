// vx_sample.h -- tokens drawn from rows of logits with temperature, top-k,
// top-p and min-p by given uniforms, on the caller's device memory.
//
// A row's order: logit descending, index ascending; NaN and -inf are not in
// it.  Weight of an entry: 2^t, t = (x - max) log2(e) / T, rounded to a
// multiple of 2^-43; sums of weights are integers, exact, and the same
// however the row is dealt to threads.  The kept entries are the shortest of
// three prefixes of the order (top_k entries; the first whose sum reaches
// top_p of the top-k sum; the entries of weight >= min_p), at least one; the
// token is the first whose running sum passes u times the kept sum.
//
// No row is sorted.  One pass over it finds the range of its values, one
// counts entries and sums weights in 2048 bins that fall with x.  Each cut
// and the draw then lie in a known bin, or in one of a few while the sums
// they go by are not known exactly; a third pass gathers the entries of those
// bins, and each gathered entry's place follows from the sums before its bin
// and from the entries of its own bin that come before it.  Where these bins
// hold more entries than the list (long runs of equal values), the
// cuts are looked for one after the other, the bin being narrowed by digits
// of (value, index) first.
//
// Bound by LDS additions and weights (two additions and some 30 instructions an
// entry) where rows are long, by the latency of about a dozen barriers where
// they are short.  A row of 8320 f32 logits takes 15.4 us in one block (load 2,
// range 2, bins 3, cuts 4, gathering and places 4), 64 of them 19; 256 of
// 131072 f32 91 us in a block each (134 MB: 1.5 TB/s); 8 of them, 16 blocks
// each, 41 us in four launches against 129 in a block each.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "vx_paged.h"

namespace vx {

struct SampleArgs {
  const void *logits;
  int64_t row_stride;
  int rows, n;
  const float *temperature, *top_p, *min_p;
  const int *top_k;
  const double *u;
  float temperature0, top_p0, min_p0;  // where the pointer is null
  int top_k0;
  int *token, *kept;
  float *prob;
  // rows dealt to several blocks: their number, the entries of one, and what
  // they hand on (SrSplit for each row)
  int chunks, chunk;
  char *split;
};

constexpr int SR_NT = 1024, SR_WAVES = SR_NT / 64;
constexpr int SR_PER = 2;  // bins and gathered entries of a thread
constexpr int SR_BINS = SR_PER * SR_NT, SR_CELLS = 2048, SR_LIST = SR_PER * SR_NT;
constexpr int SR_MAXN = 1 << 20;  // 2^43 weights: sums stay below 2^63
constexpr int SR_FIX = 43;
constexpr int SR_MAXCHUNKS = 160;

// what the blocks of a row hand on
struct SrSplit {
  uint64_t mass[SR_BINS];
  uint32_t count[SR_BINS], fill[SR_BINS];
  uint64_t list[SR_LIST];
  uint64_t first[SR_MAXCHUNKS];
  float least[SR_MAXCHUNKS];
};
static_assert(sizeof(SrSplit) % 16 == 0, "rows of it are aligned");

// the row's values as a key that rises with them; 0: not in the order
__device__ __forceinline__ uint32_t sr_key(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);  // -0 counts as 0
  return x > -INFINITY ? (b >> 31 ? ~b : b | 0x80000000u) : 0;
}
__device__ __forceinline__ float sr_value(uint32_t key) {
  return __builtin_bit_cast(float, key >> 31 ? key & 0x7fffffffu : ~key);
}
// an entry: rises along the order
__device__ __forceinline__ uint64_t sr_entry(uint32_t key, int i) { return (uint64_t)~key << 32 | (uint32_t)i; }
__device__ __forceinline__ float sr_value_of(uint64_t e) { return sr_value(~(uint32_t)(e >> 32)); }

// the bin of an entry: falls from the maximum over the range of weights, or
// that of values where it is smaller
struct SrBin {
  float max, scale;
  __device__ __forceinline__ int operator()(float x) const {
    return x == max ? 0 : (int)fminf((max - x) * scale, (float)(SR_BINS - 1));
  }
};

// What every form keeps in LDS, and behind it one of the forms' own
struct SrCommon {
  double tab[32];  // 2^(i / 32)
  uint64_t wave_m[SR_WAVES], found_m, found_e;
  uint32_t wave_c[SR_WAVES], found_c, n_list;
  int found[8];
  float wave_f[SR_WAVES];
};
// Running sums are those before a bin, with the total behind the last one.
struct SrShared : SrCommon {
  uint64_t mass[SR_BINS + 1];
  uint32_t count[SR_BINS + 1];
  uint32_t fill[SR_BINS];  // where a gathered bin's next entry goes; ~0: not gathered
  union {
    struct {
      uint64_t list[SR_LIST], sorted[SR_LIST];
    };
    struct {
      uint64_t cell_mass[SR_CELLS];
      uint32_t cell_count[SR_CELLS];
    };
  };
};
// 16-bit logits: how often each value occurs (two to a word, by bit pattern),
// and running sums over groups of 64 values, by falling value
constexpr int SR_GROUPS = 1024;
struct SrValues : SrCommon {
  uint64_t mass[SR_GROUPS + 1];
  uint32_t count[SR_GROUPS + 1];
  uint32_t often[1 << 15];
};

// The block's LDS, always by its own name: a generic pointer to it would make
// every access a flat one.
template <typename S>
__device__ __forceinline__ S &sr_lds() {
  extern __shared__ __attribute__((aligned(16))) unsigned char sr_smem[];
  return *(S *)sr_smem;
}
__device__ __forceinline__ SrShared &sr_shared() { return sr_lds<SrShared>(); }

// 2^t for t <= 0 to about 10^-11 of itself, as a multiple of 2^-43: t is
// split into k / 32 and a rest below 1/64, whose power is taken from its
// series (the quadratic and later terms, below 6e-5, in f32), times 2^(k/32)
// from a table.
struct SrWeight {
  double max, c;  // t = (x - max) c, exactly 0 at the maximum
  bool inf;       // the maximum is +inf: its entries weigh 1, all others 0
  __device__ __forceinline__ double power(float x) const {  // 2^(t + 43)
    const double t = ((double)x - max) * c;
    if (!(t > -45.0)) return 0;
    const double kd = t + 0x1.8p47;  // the sum's last bit is 1/32
    const int k = (int)(uint32_t)__builtin_bit_cast(uint64_t, kd);
    const double r = t - (kd - 0x1.8p47);
    const float f = (float)r;
    const float q = f * f * fmaf(f, fmaf(f, 0.009618129f, 0.05550411f), 0.24022651f);
    const double s = fma(r, 0.693147180559945309417, (double)q), b = sr_shared().tab[k & 31];
    return __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, fma(b, s, b)) + ((uint64_t)(int64_t)((k >> 5) + SR_FIX) << 52));
  }
  __device__ __forceinline__ uint64_t operator()(float x) const {
    if (inf) return x == INFINITY ? 1ull << SR_FIX : 0;
    return __builtin_bit_cast(uint64_t, power(x) + 0x1p52) & 0xfffffffffffffull;
  }
};

// loads that are known to be from device memory: through a generic pointer
// they would wait for LDS too
template <typename W>
__device__ __forceinline__ W sr_global(const void *p) {
  return *(const __attribute__((address_space(1))) W *)p;
}
template <typename T>
__device__ __forceinline__ T sr_element(const T *p) {
  if constexpr (sizeof(T) == 4) return __builtin_bit_cast(T, sr_global<uint32_t>(p));
  else return __builtin_bit_cast(T, sr_global<uint16_t>(p));
}
// 16 bytes of elements from i on, NaN in place of those outside from .. to - 1
template <typename T, int V = 16 / sizeof(T)>
__device__ __forceinline__ PgVec<T, V> sr_elements(const T *row, int i, int from, int to) {
  PgVec<T, V> x;
  if (i >= from && i + V <= to) {
    x = __builtin_bit_cast(PgVec<T, V>, sr_global<u32x4>(row + i));
  } else {
#pragma unroll
    for (int j = 0; j < V; j++) x.x[j] = i + j >= from && i + j < to ? sr_element(row + i + j) : (T)NAN;
  }
  return x;
}

// Entries of a row: f(index, x) for each that is in the order.
// From memory, 16 bytes a thread at a time from aligned addresses; entries
// from .. to - 1 of the row.  While four such loads are worked on, the next
// four are on their way: 64 KB a block.  (U 1: a rare path's, for its size.)
template <typename T, int U = 4>
struct SrStream {
  static constexpr int V = 16 / sizeof(T);
  const T *row;
  int from, to;
  // U times a thread's V entries, from i on (i may lie before `from`)
  __device__ __forceinline__ void load(int i, PgVec<T, V> (&x)[U]) const {
#pragma unroll
    for (int u = 0; u < U; u++, i += SR_NT * V) x[u] = sr_elements(row, i, from, to);
  }
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    vectors([&](int i, const PgVec<T, V> &x) {
#pragma unroll
      for (int j = 0; j < V; j++) {
        const float y = (float)x.x[j];
        if (y > -INFINITY) f(i + j, y);
      }
    });
  }
  // f(index, V elements), NaN where there is none; U SR_NT V elements a step
  template <typename F>
  __device__ __forceinline__ int vectors(F f) const {
    int steps = 0;
    const int off = (int)(((uintptr_t)(row + from) & 15) / sizeof(T));  // row + from - off is aligned
    int i = from - off + (int)threadIdx.x * V;
    PgVec<T, V> x[U], next[U];
    load(i, x);
#pragma unroll 1
    for (;;) {
      const int then = i + U * SR_NT * V;
      load(then, next);
#pragma unroll
      for (int u = 0; u < U; u++) f(i + u * SR_NT * V, x[u]);
      steps++;
      if (then - (int)threadIdx.x * V >= to) break;  // the same for all threads
#pragma unroll
      for (int u = 0; u < U; u++) x[u] = next[u];
      i = then;
    }
    return steps;
  }
};
// Kept in LDS from the first pass on
constexpr int SR_HOLD = 12288;
struct SrHeld {
  int n;
  static __device__ __forceinline__ float *held() {
    __shared__ float x[SR_HOLD];
    return x;
  }
  template <typename T>
  __device__ __forceinline__ void load(const SrStream<T> &from) {
    constexpr int V = 16 / sizeof(T), U = (SR_HOLD + V - 1 + SR_NT * V - 1) / (SR_NT * V);
    n = from.to;
    const int off = (int)(((uintptr_t)from.row & 15) / sizeof(T)), i0 = (int)threadIdx.x * V - off;
    PgVec<T, V> x[U];
#pragma unroll
    for (int u = 0; u < U; u++) x[u] = sr_elements(from.row, i0 + u * SR_NT * V, 0, n);
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int j = 0; j < V; j++) {
        const int i = i0 + u * SR_NT * V + j;
        if (i >= 0 && i < n) held()[i] = (float)x[u].x[j];
      }
    __syncthreads();
  }
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
#pragma unroll 4
    for (int i = threadIdx.x; i < n; i += SR_NT) {
      const float x = held()[i];
      if (x > -INFINITY) f(i, x);
    }
  }
};

// The sums of (c, m) over the lanes up to this one, by DPP: four shifts inside
// rows of 16 lanes, then the rows' totals handed on (a shift brings 0 where
// there is no lane).
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t sr_dpp(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xF, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ void sr_add_dpp(uint32_t &c, uint64_t &m) {
  const uint64_t o = (uint64_t)sr_dpp<CTRL, ROWS>((uint32_t)(m >> 32)) << 32 | sr_dpp<CTRL, ROWS>((uint32_t)m);
  c += sr_dpp<CTRL, ROWS>(c);
  m += o;
}
__device__ __forceinline__ void sr_wave_scan(uint32_t &c, uint64_t &m) {
  sr_add_dpp<0x111, 0xF>(c, m);  // row_shr 1, 2, 4, 8
  sr_add_dpp<0x112, 0xF>(c, m);
  sr_add_dpp<0x114, 0xF>(c, m);
  sr_add_dpp<0x118, 0xF>(c, m);
  sr_add_dpp<0x142, 0xA>(c, m);  // the last lane of rows 0 and 2 to rows 1 and 3
  sr_add_dpp<0x143, 0xC>(c, m);  // lane 31 to rows 2 and 3
}

// the sums of (count, mass) before each of PER items a thread, in thread
// order, in place; the totals over the block go to (tc, tm)
template <int PER>
__device__ __forceinline__ void sr_scan(uint32_t (&c)[PER], uint64_t (&m)[PER], uint32_t &tc, uint64_t &tm) {
  SrShared &s = sr_shared();
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t ac = 0, bc = 0;
  uint64_t am = 0, bm = 0;
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const uint32_t x = c[i];
    const uint64_t y = m[i];
    c[i] = ac;
    m[i] = am;
    ac += x;
    am += y;
  }
  uint32_t ic = ac;
  uint64_t im = am;
  sr_wave_scan(ic, im);
  __syncthreads();
  if (lane == 63) s.wave_c[wave] = ic, s.wave_m[wave] = im;
  __syncthreads();
  tc = 0;
  tm = 0;
#pragma unroll 4
  for (int w = 0; w < SR_WAVES; w++) {
    if (w == wave) bc = tc, bm = tm;
    tc += s.wave_c[w];
    tm += s.wave_m[w];
  }
#pragma unroll
  for (int i = 0; i < PER; i++) c[i] += bc + ic - ac, m[i] += bm + im - am;
}

// A row's settings and what follows from its range of values.  All members
// are the same in every thread.
struct SrRow {
  float temp, top_p, min_p;
  int top_k;
  double u;
  SrWeight weight;
  SrBin bin;
  uint32_t top;  // the maximum's key

  __device__ __forceinline__ void settings(const SampleArgs &a, int r) {
    temp = a.temperature ? a.temperature[r] : a.temperature0;
    top_p = a.top_p ? a.top_p[r] : a.top_p0;
    min_p = a.min_p ? a.min_p[r] : a.min_p0;
    top_k = a.top_k ? a.top_k[r] : a.top_k0;
    u = a.u[r];
  }
  // from the first entry and the least value
  __device__ __forceinline__ void range(uint64_t first, float least) {
    top = ~(uint32_t)(first >> 32);
    const float max = sr_value(top);
    weight = SrWeight{(double)max, 1.4426950408889634 / temp, max == INFINITY};
    // weights end at 2^-44, 30.5 T below the maximum
    bin = SrBin{max, fminf((float)SR_BINS / fminf(31.0f * temp, max - least), 1e30f)};
  }
  // the sum that top-p's cut reaches, and the one the draw does, by the sum they are a part of
  __device__ __forceinline__ uint64_t goal(uint64_t mass) const {
    if (!(top_p < 1.0f)) return ~0ull;
    const double t = ceil((double)fmaxf(top_p, 0.0f) * (double)mass);
    return t < 1.0 ? 1 : t < (double)mass ? (uint64_t)t : mass;
  }
  __device__ __forceinline__ uint64_t drawn(uint64_t mass) const {
    const double t = floor(u * (double)mass);
    return !(t > 0.0) ? 1 : t >= (double)mass ? mass : (uint64_t)t + 1;
  }
  // the smallest key whose weight is at least min_p (the maximum's is 1): 64
  // trials a step, each wave for itself
  __device__ __forceinline__ uint32_t min_p_key() const {
    const int lane = threadIdx.x & 63;
    uint32_t lo = 0, hi = top;  // lo: below it, hi: not below it
    while (hi - lo > 1) {
      const uint32_t by = (hi - lo + 63) / 64;
      const uint64_t at = (uint64_t)lo + (uint64_t)by * (lane + 1);
      const uint32_t k = at < hi ? (uint32_t)at : hi;
      const float x = sr_value(k);
      const bool yes = k == hi || (x > -INFINITY && !weight.inf && weight.power(x) >= (double)min_p * 0x1p43);
      const int i = __ffsll((unsigned long long)__ballot(yes)) - 1;
      const uint64_t up = (uint64_t)lo + (uint64_t)by * (i + 1);
      lo = lo + by * i;
      hi = up < hi ? (uint32_t)up : hi;
    }
    return hi;
  }
};

// whether the target-th of a running quantity lies in (before, after]
__device__ __forceinline__ bool sr_inside(uint64_t target, uint64_t before, uint64_t after) {
  return before < target && target <= after;
}

// The first entry and the least value over the block.  The entry's index is
// found where it is asked for (a greedy choice), else 0.
template <typename E>
__device__ __forceinline__ void sr_range(const E &entries, bool index, uint64_t &first, float &least) {
  SrShared &s = sr_shared();
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float max = -INFINITY, min = INFINITY;
  entries.each([&](int, float x) {
    max = fmaxf(max, x);
    min = fminf(min, x);
  });
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) {
    max = fmaxf(max, __shfl_xor(max, d, 64));
    min = fminf(min, __shfl_xor(min, d, 64));
  }
  if (lane == 0) s.wave_f[wave] = min, s.wave_m[wave] = sr_key(max);
  if (threadIdx.x == 0) s.found_c = index ? ~0u : 0;
  __syncthreads();
  uint32_t key = 0;
  least = INFINITY;
#pragma unroll
  for (int w = 0; w < SR_WAVES; w++) {
    key = s.wave_m[w] > key ? (uint32_t)s.wave_m[w] : key;
    least = fminf(least, s.wave_f[w]);
  }
  if (index && key && sr_key(max) == key) {  // a wave that has the maximum
    uint32_t at = ~0u;
    entries.each([&](int i, float x) {
      if (sr_key(x) == key) at = (uint32_t)i < at ? (uint32_t)i : at;
    });
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
      const uint32_t o = (uint32_t)__shfl_xor((int)at, d, 64);
      at = o < at ? o : at;
    }
    if (lane == 0) atomicMin(&s.found_c, at);
  }
  if (index) __syncthreads();
  first = key ? sr_entry(key, (int)s.found_c) : ~0ull;
}

// counts and sums of the entries in the bins (cleared by the caller)
template <typename E>
__device__ __forceinline__ void sr_bins(const E &entries, const SrRow &q) {
  SrShared &s = sr_shared();
  entries.each([&](int, float x) {
    const int b = q.bin(x);
    atomicAdd(&s.count[b], 1u);
    const uint64_t w = q.weight(x);
    if (w) atomicAdd((unsigned long long *)&s.mass[b], (unsigned long long)w);
  });
}

// running sums over the bins, from this thread's
__device__ __forceinline__ void sr_run(uint32_t (&c)[SR_PER], uint64_t (&m)[SR_PER]) {
  SrShared &s = sr_shared();
  uint32_t tc;
  uint64_t tm;
  sr_scan(c, m, tc, tm);
#pragma unroll
  for (int i = 0; i < SR_PER; i++) {
    s.count[threadIdx.x * SR_PER + i] = c[i];
    s.mass[threadIdx.x * SR_PER + i] = m[i];
  }
  if (threadIdx.x == 0) s.count[SR_BINS] = tc, s.mass[SR_BINS] = tm;
  __syncthreads();
}
// f(bin) for each of this thread's bins
template <typename F>
__device__ __forceinline__ void sr_own(F f) {
#pragma unroll
  for (int i = 0; i < SR_PER; i++) f((int)threadIdx.x * SR_PER + i);
}

// Where the cuts and the draw lie, as far as the bins tell: sets fill[] for
// the bins to gather.  Returns their number of entries.
struct SrCuts {
  bool k, m;         // whether top-k, min-p take anything away
  uint32_t key;      // min-p's
  int key_bin;
};
__device__ __forceinline__ uint32_t sr_choose(const SrRow &q, SrCuts &cut) {
  SrShared &s = sr_shared();
  const uint32_t total_c = s.count[SR_BINS];
  const uint64_t total = s.mass[SR_BINS];
  cut.k = q.top_k > 0 && (uint32_t)q.top_k < total_c;
  cut.m = q.min_p > 0.0f;
  cut.key = cut.m ? q.min_p_key() : 0;
  cut.key_bin = cut.m ? q.bin(sr_value(cut.key)) : SR_BINS - 1;
  if (threadIdx.x < 8) s.found[threadIdx.x] = 0;
  __syncthreads();
  // marks the bin that a sum lies in
  auto locate = [&](int i, uint64_t sum) {
    sr_own([&](int b) {
      if (sr_inside(sum, s.mass[b], s.mass[b + 1])) s.found[i] = b;
    });
  };
  int kb = 0;
  if (cut.k) {
    sr_own([&](int b) {
      if (sr_inside(q.top_k, s.count[b], s.count[b + 1])) s.found[0] = b;
    });
    __syncthreads();
    kb = s.found[0];
  }
  // bounds of the sums: of top-k's, then of what is kept
  const uint64_t klo = cut.k ? s.mass[kb] : total, khi = cut.k ? s.mass[kb + 1] : total;
  uint64_t lo = klo, hi = khi;
  const bool p = q.top_p < 1.0f;
  if (p) {
    locate(1, q.goal(klo));
    locate(2, q.goal(khi));
    __syncthreads();
    lo = s.mass[s.found[1]] < lo ? s.mass[s.found[1]] : lo;
    hi = s.mass[s.found[2] + 1] < hi ? s.mass[s.found[2] + 1] : hi;
  }
  if (cut.m) {
    lo = s.mass[cut.key_bin] < lo ? s.mass[cut.key_bin] : lo;
    hi = s.mass[cut.key_bin + 1] < hi ? s.mass[cut.key_bin + 1] : hi;
  }
  locate(3, q.drawn(lo));
  locate(4, q.drawn(hi));
  __syncthreads();
  uint32_t cs[SR_PER], n;
  uint64_t ms[SR_PER] = {}, none;
  bool take[SR_PER];
#pragma unroll
  for (int i = 0; i < SR_PER; i++) {
    const int b = threadIdx.x * SR_PER + i;
    take[i] = (cut.k && b == kb) || (p && b >= s.found[1] && b <= s.found[2]) || (cut.m && b == cut.key_bin) ||
              (b >= s.found[3] && b <= s.found[4]);
    cs[i] = take[i] ? s.count[b + 1] - s.count[b] : 0;
  }
  sr_scan(cs, ms, n, none);
#pragma unroll
  for (int i = 0; i < SR_PER; i++) s.fill[threadIdx.x * SR_PER + i] = take[i] ? cs[i] : ~0u;
  __syncthreads();
  return n;
}

// A thread's gathered entries, in order, and their places: the entries and
// weights before each
struct SrPlaces {
  uint64_t e[SR_PER], w[SR_PER], m[SR_PER];
  uint32_t c[SR_PER];
  int b[SR_PER];  // bins; -1: none
  // Of the list's n entries, those of a bin lie together, at from .. to - 1,
  // running on from the sums (c, m) before it: before(bin, from, to, c, m).
  // Each is put to its place by the number of those in its bin that come
  // before it, then their weights are summed.
  template <typename F>
  __device__ __forceinline__ void rank(const SrRow &q, uint32_t n, F before) {
    SrShared &s = sr_shared();
    uint32_t from, to;
#pragma unroll
    for (int i = 0; i < SR_PER; i++) {
      const uint32_t at = threadIdx.x + i * SR_NT;
      if (at >= n) continue;
      const uint64_t x = s.list[at];
      before(q.bin(sr_value_of(x)), from, to, c[0], m[0]);
      uint32_t place = from;
#pragma unroll 8
      for (uint32_t j = from; j < to; j++) place += s.list[j] < x;
      s.sorted[place] = x;
    }
    __syncthreads();
    uint64_t sum[SR_PER], total;
    uint32_t none[SR_PER] = {}, nothing;
#pragma unroll
    for (int i = 0; i < SR_PER; i++) {
      const uint32_t at = threadIdx.x * SR_PER + i;
      e[i] = at < n ? s.sorted[at] : ~0ull;
      b[i] = at < n ? q.bin(sr_value_of(e[i])) : -1;
      w[i] = at < n ? q.weight(sr_value_of(e[i])) : 0;
      sum[i] = w[i];
    }
    sr_scan(none, sum, nothing, total);
#pragma unroll
    for (int i = 0; i < SR_PER; i++) s.list[threadIdx.x * SR_PER + i] = sum[i];  // before each place
    __syncthreads();
#pragma unroll
    for (int i = 0; i < SR_PER; i++) {
      if (b[i] < 0) continue;
      before(b[i], from, to, c[i], m[i]);
      c[i] += threadIdx.x * SR_PER + i - from;
      m[i] += sum[i] - s.list[from];
    }
  }
  // f(i) for each entry there is
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
#pragma unroll
    for (int i = 0; i < SR_PER; i++)
      if (b[i] >= 0) f(i);
  }
  // hands on the entry whose running count or sum, it included, is the first to reach `target`
  __device__ __forceinline__ void find(bool by_count, uint64_t target) const {
    SrShared &s = sr_shared();
    each([&](int i) {
      if (by_count ? c[i] + 1 == target : sr_inside(target, m[i], m[i] + w[i]))
        s.found_c = c[i] + 1, s.found_m = m[i] + w[i], s.found_e = e[i];
    });
    __syncthreads();
  }
};

// a row's results
__device__ __forceinline__ void sr_write(const SrRow &q, uint64_t e, uint32_t count, uint64_t mass, const SampleArgs &a, int r) {
  a.token[r] = (int)(uint32_t)e;
  if (a.kept) a.kept[r] = (int)count;
  if (a.prob) a.prob[r] = (float)((q.weight.inf ? 0x1p43 : q.weight.power(sr_value_of(e))) / (double)mass);
}

// the cuts and the draw by the gathered entries' places
__device__ __forceinline__ void sr_finish(const SrRow &q, const SrCuts &cut, uint32_t n, const SampleArgs &a, int r) {
  SrShared &s = sr_shared();
  SrPlaces p;
  p.rank(q, n, [&](int b, uint32_t &from, uint32_t &to, uint32_t &c, uint64_t &m) {
    to = s.fill[b];  // behind its last entry, since all are in
    from = to - (s.count[b + 1] - s.count[b]);
    c = s.count[b];
    m = s.mass[b];
  });
  uint32_t count = s.count[SR_BINS];
  uint64_t mass = s.mass[SR_BINS];
  if (threadIdx.x == 0) s.n_list = 0, s.wave_m[0] = 0;
  if (cut.k) {
    p.find(true, q.top_k);
    count = s.found_c;
    mass = s.found_m;
  }
  __syncthreads();
  const uint64_t goal = q.goal(mass);
  if (cut.m) {
    p.each([&](int i) {
      if (p.b[i] == cut.key_bin && ~(uint32_t)(p.e[i] >> 32) >= cut.key) {
        atomicAdd(&s.n_list, 1u);
        atomicAdd((unsigned long long *)&s.wave_m[0], (unsigned long long)p.w[i]);
      }
    });
    __syncthreads();
    const uint32_t c = s.count[cut.key_bin] + s.n_list;
    if (c < count) count = c, mass = s.mass[cut.key_bin] + s.wave_m[0];
  }
  if (goal <= mass) {
    p.find(false, goal);
    if (s.found_c < count) count = s.found_c, mass = s.found_m;
  }
  const uint64_t drawn = q.drawn(mass);
  p.each([&](int i) {
    if (sr_inside(drawn, p.m[i], p.m[i] + p.w[i])) sr_write(q, p.e[i], count, mass, a, r);
  });
}

// The cuts one after the other, for bins of too many entries.
template <typename E>
struct SrSearch {
  const E &entries;
  const SrRow &q;
  // the entry that a cut falls on, the first whose running count or sum (it
  // included) is at least `target`, and its running count and sum
  __device__ __forceinline__ uint64_t find(bool by_count, uint64_t target, uint32_t &c, uint64_t &m) {
    SrShared &s = sr_shared();
    const int t = threadIdx.x;
    __syncthreads();
    sr_own([&](int b) {
      if (by_count ? sr_inside(target, s.count[b], s.count[b + 1]) : sr_inside(target, s.mass[b], s.mass[b + 1])) s.found[0] = b;
    });
    __syncthreads();
    // the entries of bin b whose leading digits, all above `bits`, are `lead`
    const int b = s.found[0];
    int bits = 64;
    uint64_t lead = 0;
    uint32_t c0 = s.count[b], left = s.count[b + 1] - c0;
    uint64_t m0 = s.mass[b];
    auto in = [&](uint64_t e, float x) { return q.bin(x) == b && (bits == 64 || e >> bits == lead); };
    // narrowed by digits of 10, 11 and 11 bits of the value, then by runs of 1024 indices
    for (int shift = 54; left > SR_LIST; shift = shift > 32 ? shift - 11 : 10) {
      for (int i = t; i < SR_CELLS; i += SR_NT) s.cell_count[i] = 0, s.cell_mass[i] = 0;
      __syncthreads();
      entries.each([&](int i, float x) {
        const uint64_t e = sr_entry(sr_key(x), i);
        if (!in(e, x)) return;
        const int cell = (int)(e >> shift) & (SR_CELLS - 1);
        atomicAdd(&s.cell_count[cell], 1u);
        atomicAdd((unsigned long long *)&s.cell_mass[cell], (unsigned long long)q.weight(x));
      });
      __syncthreads();
      constexpr int P = SR_CELLS / SR_NT;
      uint32_t cs[P], own[P], tc;
      uint64_t ms[P], own_m[P], tm;
#pragma unroll
      for (int i = 0; i < P; i++) {
        cs[i] = own[i] = s.cell_count[P * t + i];
        ms[i] = own_m[i] = s.cell_mass[P * t + i];
      }
      sr_scan(cs, ms, tc, tm);
#pragma unroll
      for (int i = 0; i < P; i++)
        if (by_count ? sr_inside(target, c0 + cs[i], c0 + cs[i] + own[i]) : sr_inside(target, m0 + ms[i], m0 + ms[i] + own_m[i])) {
          s.found[1] = P * t + i;
          s.found_c = cs[i];
          s.found_m = ms[i];
          s.n_list = own[i];
        }
      __syncthreads();
      c0 += s.found_c;
      m0 += s.found_m;
      left = s.n_list;
      lead = (bits < 64 ? lead << (bits - shift) : 0) | (uint64_t)s.found[1];
      bits = shift;
      __syncthreads();
    }
    if (t == 0) s.n_list = 0;
    __syncthreads();
    entries.each([&](int i, float x) {
      const uint64_t e = sr_entry(sr_key(x), i);
      if (!in(e, x)) return;
      const uint32_t at = atomicAdd(&s.n_list, 1u);
      if (at < SR_LIST) s.list[at] = e;
    });
    __syncthreads();
    SrPlaces p;
    p.rank(q, left, [&](int, uint32_t &from, uint32_t &to, uint32_t &pc, uint64_t &pm) { from = 0, to = left, pc = c0, pm = m0; });
    p.find(by_count, target);
    c = s.found_c;
    m = s.found_m;
    return s.found_e;
  }
  __device__ __forceinline__ void finish(const SrCuts &cut, const SampleArgs &a, int r) {
    SrShared &s = sr_shared();
    uint32_t count = s.count[SR_BINS], c;
    uint64_t mass = s.mass[SR_BINS], m, e = 0, goal = ~0ull;
    for (int step = 0; step < 3; step++) {
      uint64_t target;
      if (step == 0) {
        if (!cut.k) continue;
        target = q.top_k;
      } else if (step == 1) {
        goal = q.goal(mass);
        // where the bins before min-p's hold as much as the other cuts leave, it cuts nothing
        if (cut.m && s.count[cut.key_bin] < count && s.mass[cut.key_bin] < goal) {
          uint32_t cs[1] = {0};
          uint64_t ms[1] = {0};
          entries.each([&](int, float x) {
            if (sr_key(x) >= cut.key) cs[0]++, ms[0] += q.weight(x);
          });
          sr_scan(cs, ms, c, m);
          if (c < count) count = c, mass = m;
        }
        if (goal > mass) continue;
        target = goal;
      } else {
        target = q.drawn(mass);
      }
      e = find(step == 0, target, c, m);
      if (step < 2 && c < count) count = c, mass = m;
    }
    if (threadIdx.x == 0) sr_write(q, e, count, mass, a, r);
  }
};

// nothing to draw from, or the greedy choice: known from the first entry
__device__ __forceinline__ bool sr_simple(const SrRow &q, uint64_t first, const SampleArgs &a, int r, bool write) {
  const bool none = first == ~0ull;
  if (!none && q.temp > 0) return false;
  if (write) {
    a.token[r] = none ? -1 : (int)(uint32_t)first;
    if (a.kept) a.kept[r] = none ? 0 : 1;
    if (a.prob) a.prob[r] = none ? 0.0f : 1.0f;
  }
  return true;
}

__device__ __forceinline__ void sr_clear() {
  SrShared &s = sr_shared();
  sr_own([&](int b) { s.mass[b] = 0, s.count[b] = 0; });
  if (threadIdx.x < 32) s.tab[threadIdx.x] = exp2(threadIdx.x / 32.0);
}

template <typename E>
__device__ __forceinline__ void sr_gather(const E &entries, const SrRow &q) {
  SrShared &s = sr_shared();
  entries.each([&](int i, float x) {
    const int b = q.bin(x);
    if (s.fill[b] != ~0u) s.list[atomicAdd(&s.fill[b], 1u)] = sr_entry(sr_key(x), i);
  });
  __syncthreads();
}

// A block a row; `again`: the same entries, for the rare search
template <typename E, typename S>
__device__ __forceinline__ void sr_row(const E &entries, const S &again, const SampleArgs &a, int r) {
  SrShared &s = sr_shared();
  SrRow q;
  q.settings(a, r);
  sr_clear();
  uint64_t first;
  float least;
  sr_range(entries, !(q.temp > 0), first, least);
  if (sr_simple(q, first, a, r, threadIdx.x == 0)) return;
  q.range(first, least);
  sr_bins(entries, q);
  __syncthreads();
  uint32_t c[SR_PER];
  uint64_t m[SR_PER];
#pragma unroll
  for (int i = 0; i < SR_PER; i++) c[i] = s.count[threadIdx.x * SR_PER + i], m[i] = s.mass[threadIdx.x * SR_PER + i];
  sr_run(c, m);
  SrCuts cut;
  const uint32_t n = sr_choose(q, cut);
  if (n <= SR_LIST) {
    sr_gather(entries, q);
    sr_finish(q, cut, n, a, r);
  } else {
    SrSearch<S>{again, q}.finish(cut, a, r);
  }
}
template <typename T, bool HELD>
__global__ __launch_bounds__(SR_NT) void sample_rows_kernel(SampleArgs a) {
  const int r = blockIdx.x;
  const SrStream<T> stream{(const T *)a.logits + r * a.row_stride, 0, a.n};
  if constexpr (HELD) {
    SrHeld held;
    held.load(stream);
    sr_row(held, held, a, r);
  } else {
    sr_row(stream, SrStream<T, 1>{stream.row, 0, a.n}, a, r);
  }
}

// A block a row of 16-bit logits: a pass counts how often each of the 65536
// values occurs, which is one LDS addition an entry; everything up to the
// draw then goes by values and their numbers, with one weight a value.  A
// second pass finds the entry among those of the drawn value.  256 rows of
// 131072 bf16: 44 us (first pass 13, second 9), against 117 by bins.
// Values by falling order: the bit pattern at a place (0: the largest).
__device__ __forceinline__ uint32_t sr_place_bits(uint32_t place) { return place < 0x8000u ? 0x7fffu - place : place; }
template <typename T>
__device__ __forceinline__ float sr_place_value(uint32_t place) {
  return (float)__builtin_bit_cast(T, (uint16_t)sr_place_bits(place));
}

template <typename T>
struct SrByValue {
  // a value in its place among the others: entries and weights before it, its
  // number and weight
  struct At {
    uint32_t place, before, number;
    uint64_t before_m, w;
  };
  static __device__ __forceinline__ uint32_t often(uint32_t place) {
    const uint32_t bits = sr_place_bits(place);
    return sr_lds<SrValues>().often[bits >> 1] >> (16 * (bits & 1)) & 0xffffu;
  }
  // The value at lane l of group `group`, and the sums before it; every wave
  // does the same.
  static __device__ __forceinline__ At lane(const SrRow &q, int group) {
    const SrValues &s = sr_lds<SrValues>();
    const int l = threadIdx.x & 63;
    At v;
    v.place = 64 * group + l;
    v.number = often(v.place);
    v.w = v.number ? q.weight(sr_place_value<T>(v.place)) : 0;
    uint32_t c = v.number;
    uint64_t m = v.number * v.w;
    const uint32_t own = c;
    const uint64_t own_m = m;
    sr_wave_scan(c, m);
    v.before = s.count[group] + c - own;
    v.before_m = s.mass[group] + m - own_m;
    return v;
  }
  // lane `from`'s value in every lane
  static __device__ __forceinline__ At of(const At &v, int from) {
    At r;
    r.place = __shfl(v.place, from, 64);
    r.before = __shfl(v.before, from, 64);
    r.number = __shfl(v.number, from, 64);
    r.before_m = __shfl((unsigned long long)v.before_m, from, 64);
    r.w = __shfl((unsigned long long)v.w, from, 64);
    return r;
  }
  // the value that a running count or sum falls on
  static __device__ __forceinline__ At find(const SrRow &q, bool by_count, uint64_t target) {
    SrValues &s = sr_lds<SrValues>();
    const int t = threadIdx.x;
    __syncthreads();
    if (by_count ? sr_inside(target, s.count[t], s.count[t + 1]) : sr_inside(target, s.mass[t], s.mass[t + 1])) s.found[0] = t;
    __syncthreads();
    const At v = lane(q, s.found[0]);
    const bool is = by_count ? sr_inside(target, v.before, v.before + v.number) : sr_inside(target, v.before_m, v.before_m + v.number * v.w);
    return of(v, __ffsll((unsigned long long)__ballot(is)) - 1);
  }
  // the number of a value's entries that a sum takes
  static __device__ __forceinline__ uint32_t part(const At &v, uint64_t target) {
    return (uint32_t)((target - v.before_m + v.w - 1) / v.w);
  }
};
static_assert(SR_GROUPS == SR_NT, "a group a thread");

template <typename T>
__global__ __launch_bounds__(SR_NT) void sample_values_kernel(SampleArgs a) {
  using B = SrByValue<T>;
  SrValues &s = sr_lds<SrValues>();
  const int r = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const SrStream<T> stream{(const T *)a.logits + r * a.row_stride, 0, a.n};
  SrRow q;
  q.settings(a, r);
  for (int i = t; i < (1 << 15) / 4; i += SR_NT) ((u32x4 *)s.often)[i] = u32x4{0, 0, 0, 0};
  if (t < 32) s.tab[t] = exp2(t / 32.0);
  if (t == 0) s.found_c = 0, s.found[1] = 0x10000;
  __syncthreads();
  const uint32_t n = SrStream<T>::V * 4 * SR_NT * stream.vectors([&](int, const PgVec<T, SrStream<T>::V> &x) {
#pragma unroll
    for (int j = 0; j < SrStream<T>::V; j++) {
      const uint32_t b = __builtin_bit_cast(uint16_t, x.x[j]);
      atomicAdd(&s.often[b >> 1], b & 1 ? 0x10000u : 1u);
    }
  });
  __syncthreads();

  // Words 1024 i + t are this thread's: the positive values' for i < 16, the
  // negative ones' behind them.  What is not in the order is taken out, the
  // second zero is counted as the first, and the first value there is found.
  constexpr int WORDS = (1 << 15) / SR_NT;
  constexpr uint32_t inf = __is_same(T, __bf16) ? 0x7f80u : 0x7c00u;
  uint32_t some = 0, sum = 0, first = 0x10000;
#pragma unroll 4
  for (int i = 0; i < WORDS; i++) {
    const uint32_t at = i * SR_NT + t, all = s.often[at];
    uint32_t w = all;
    sum += (w & 0xffffu) + (w >> 16);
    if ((at > inf >> 1 && at < 0x4000u) || at >= (0x8000u | inf) >> 1) w = 0;  // NaN, -inf
    if (at == inf >> 1) w &= 0xffffu;                                          // +inf, and a NaN
    if (w != all) s.often[at] = w;
    some |= (uint32_t)(w != 0) << i;
  }
  if (t == 0) {
    const uint32_t zeros = (s.often[0] & 0xffffu) + (s.often[0x4000] & 0xffffu);
    if (zeros > 0xffffu) sum++;  // does not fit
    s.often[0] = (s.often[0] & 0xffff0000u) | (zeros & 0xffffu);
    s.often[0x4000] &= 0xffff0000u;
    some = (some & ~0x10001u) | (s.often[0] != 0) | (uint32_t)(s.often[0x4000] != 0) << 16;
  }
  if (some & 0xffffu) {
    const int i = 31 - __clz(some & 0xffffu);
    first = 0x7fffu - (2 * (i * SR_NT + t) + (s.often[i * SR_NT + t] >> 16 ? 1 : 0));
  } else if (some) {
    const int i = __ffs(some) - 1;
    first = 2 * (i * SR_NT + t) + (s.often[i * SR_NT + t] & 0xffffu ? 0 : 1);
  }
  for (int d = 32; d > 0; d >>= 1) {
    const uint32_t o = __shfl_xor(first, d, 64);
    first = o < first ? o : first;
    sum += __shfl_xor(sum, d, 64);
  }
  if (lane == 0) {
    atomicMin(&s.found[1], (int)first);
    atomicAdd(&s.found_c, sum);
  }
  __syncthreads();
  first = s.found[1];
  if (s.found_c != n) {  // a value that occurs 65536 times or more does not fit its half of a word
    __syncthreads();
    const SrStream<T, 1> again{stream.row, 0, a.n};
    sr_row(again, again, a, r);
    return;
  }
  typename B::At v{first, 0, 0, 0, 1};  // the value that is drawn, and which of its entries
  uint32_t turn = 1, count = 1;
  uint64_t mass = 1ull << SR_FIX;
  if (first > 0xffffu) {
    sr_simple(q, ~0ull, a, r, t == 0);
    return;
  }
  q.range(sr_entry(sr_key(sr_place_value<T>(first)), 0), 0);
  if (q.temp > 0) {
    // sums over groups of 64 values: 32 words, half a wave's
    const auto group = [&](int i) { return i < WORDS / 2 ? SR_GROUPS / 2 - 1 - (i * 32 + (t >> 5)) : i * 32 + (t >> 5); };
#pragma unroll 1
    for (int i = 0; i < WORDS; i++) {
      uint32_t c = 0;
      uint64_t m = 0;
      if (__any(some >> i & 1)) {
        const uint32_t w = s.often[i * SR_NT + t], b = 2 * (i * SR_NT + t);
        const uint32_t c0 = w & 0xffffu, c1 = w >> 16;
        c = c0 + c1;
        if (c0) m = c0 * q.weight((float)__builtin_bit_cast(T, (uint16_t)b));
        if (c1) m += c1 * q.weight((float)__builtin_bit_cast(T, (uint16_t)(b + 1)));
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
          c += __shfl_xor(c, d, 64);
          m += __shfl_xor((unsigned long long)m, d, 64);
        }
      }
      if ((t & 31) == 0) s.count[group(i)] = c, s.mass[group(i)] = m;
    }
    __syncthreads();
    uint32_t cs[1] = {s.count[t]};
    uint64_t ms[1] = {s.mass[t]};
    sr_scan(cs, ms, count, mass);
    s.count[t] = cs[0];
    s.mass[t] = ms[0];
    if (t == 0) s.count[SR_GROUPS] = count, s.mass[SR_GROUPS] = mass;
    __syncthreads();
    if (q.top_k > 0 && (uint32_t)q.top_k < count) {
      v = B::find(q, true, q.top_k);
      count = q.top_k;
      mass = v.before_m + (count - v.before) * v.w;
    }
    const uint64_t goal = q.goal(mass);
    if (q.min_p > 0.0f) {
      // the last place whose value's key is not below min-p's
      const uint32_t key = q.min_p_key();
      uint32_t lo = first, hi = 0x10000;  // lo: not below, hi: below
      while (hi - lo > 1) {
        const uint32_t by = (hi - lo + 63) / 64, at = lo + by * lane;
        const bool yes = at < hi && sr_key(sr_place_value<T>(at)) >= key;
        const int i = 63 - __clzll(__ballot(yes));
        hi = lo + by * (i + 1) < hi ? lo + by * (i + 1) : hi;
        lo = lo + by * i;
      }
      const typename B::At w = B::of(B::lane(q, lo >> 6), lo & 63);
      const uint32_t c = w.before + w.number;
      if (c < count) count = c, mass = w.before_m + w.number * w.w;
    }
    if (goal <= mass) {
      v = B::find(q, false, goal);
      const uint32_t some_of = B::part(v, goal), c = v.before + some_of;
      if (c < count) count = c, mass = v.before_m + some_of * v.w;
    }
    const uint64_t drawn = q.drawn(mass);
    v = B::find(q, false, drawn);
    turn = B::part(v, drawn);
  }

  // the turn-th entry of the drawn value: counted in 1024 runs of the row
  __syncthreads();
  s.often[t] = 0;
  __syncthreads();
  int shift = 0;
  while (((a.n - 1) >> shift) >= SR_NT) shift++;
  const uint32_t bits = sr_place_bits(v.place);
  const auto is_it = [&](T x) {
    const uint32_t b = __builtin_bit_cast(uint16_t, x);
    return b == bits || (bits == 0 && b == 0x8000u);
  };
  const uint32_t pair = bits * 0x10001u, sign = bits ? 0 : 0x80008000u;
  stream.vectors([&](int i, const PgVec<T, SrStream<T>::V> &x) {
    // a half word of zeros in any of the differences (or a false alarm)
    uint32_t any = 0;
#pragma unroll
    for (int j = 0; j < SrStream<T>::V; j += 2) {
      const uint32_t w = __builtin_bit_cast(uint16_t, x.x[j]) | (uint32_t)__builtin_bit_cast(uint16_t, x.x[j + 1]) << 16;
      const uint32_t d = (w ^ pair) & ~sign;
      any |= (d - 0x00010001u) & ~d;
    }
    if (!(any & 0x80008000u)) return;
#pragma unroll
    for (int j = 0; j < SrStream<T>::V; j++)
      if (is_it(x.x[j])) atomicAdd(&s.often[(i + j) >> shift], 1u);
  });
  __syncthreads();
  uint32_t cs[1] = {s.often[t]}, total;
  const uint32_t own = cs[0];
  uint64_t none[1] = {0}, nothing;
  sr_scan(cs, none, total, nothing);
  if (sr_inside(turn, cs[0], cs[0] + own)) s.found[0] = t, s.found[1] = turn - cs[0];
  __syncthreads();
  if (wave) return;
  int left = s.found[1];
  const int from = s.found[0] << shift, to = min(a.n, from + (1 << shift));
  for (int i = from; i < to; i += 64) {
    const bool is = i + lane < to && is_it(sr_element(stream.row + i + lane));
    const uint64_t m = __ballot(is);
    const int here = __popcll(m);
    if (left > here) {
      left -= here;
      continue;
    }
    if (is && __popcll(m & ((1ull << lane) - 1)) == left - 1) {
      a.token[r] = i + lane;
      if (a.kept) a.kept[r] = (int)count;
      if (a.prob)
        a.prob[r] = !(q.temp > 0) ? 1.0f : (float)((q.weight.inf ? 0x1p43 : q.weight.power(sr_place_value<T>(v.place))) / (double)mass);
    }
    break;
  }
}

// Several blocks a row, for a few long rows: the same passes as launches of
// their own, sums and gathered entries joined in memory (integers: the order
// of the blocks does not matter).
// the range of a chunk's values; clears what the next passes add to
template <typename T>
__global__ __launch_bounds__(SR_NT) void sample_range_kernel(SampleArgs a) {
  const int r = blockIdx.x / a.chunks, k = blockIdx.x - r * a.chunks;
  SrSplit &g = ((SrSplit *)a.split)[r];
  const SrStream<T> entries{(const T *)a.logits + r * a.row_stride, k * a.chunk, min(a.n, (k + 1) * a.chunk)};
  for (int i = k * SR_NT + threadIdx.x; i < SR_BINS; i += a.chunks * SR_NT) g.mass[i] = 0, g.count[i] = 0, g.fill[i] = 0;
  uint64_t first;
  float least;
  sr_range(entries, !((a.temperature ? a.temperature[r] : a.temperature0) > 0), first, least);
  if (threadIdx.x == 0) g.first[k] = first, g.least[k] = least;
}
// the row's range from its chunks'
__device__ __forceinline__ void sr_joined(const SrSplit &g, int chunks, uint64_t &first, float &least) {
  const int lane = threadIdx.x & 63;
  first = ~0ull;
  least = INFINITY;
  for (int i = lane; i < chunks; i += 64) {
    first = g.first[i] < first ? g.first[i] : first;
    least = fminf(least, g.least[i]);
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) {
    const uint64_t o = __shfl_xor((unsigned long long)first, d, 64);
    first = o < first ? o : first;
    least = fminf(least, __shfl_xor(least, d, 64));
  }
}
template <typename T>
__global__ __launch_bounds__(SR_NT) void sample_bins_kernel(SampleArgs a) {
  SrShared &s = sr_shared();
  const int r = blockIdx.x / a.chunks, k = blockIdx.x - r * a.chunks, t = threadIdx.x;
  SrSplit &g = ((SrSplit *)a.split)[r];
  const SrStream<T> entries{(const T *)a.logits + r * a.row_stride, k * a.chunk, min(a.n, (k + 1) * a.chunk)};
  SrRow q;
  q.settings(a, r);
  sr_clear();
  uint64_t first;
  float least;
  sr_joined(g, a.chunks, first, least);
  if (sr_simple(q, first, a, r, k == 0 && t == 0)) return;
  q.range(first, least);
  __syncthreads();
  sr_bins(entries, q);
  __syncthreads();
  for (int b = t; b < SR_BINS; b += SR_NT)
    if (s.count[b]) {
      atomicAdd(&g.count[b], s.count[b]);
      if (s.mass[b]) atomicAdd((unsigned long long *)&g.mass[b], (unsigned long long)s.mass[b]);
    }
}
template <typename T>
__global__ __launch_bounds__(SR_NT) void sample_gather_kernel(SampleArgs a) {
  SrShared &s = sr_shared();
  const int r = blockIdx.x / a.chunks, k = blockIdx.x - r * a.chunks, t = threadIdx.x;
  SrSplit &g = ((SrSplit *)a.split)[r];
  const SrStream<T> entries{(const T *)a.logits + r * a.row_stride, k * a.chunk, min(a.n, (k + 1) * a.chunk)};
  uint32_t c[SR_PER];
  uint64_t m[SR_PER];
#pragma unroll
  for (int i = 0; i < SR_PER; i++) c[i] = g.count[t * SR_PER + i], m[i] = g.mass[t * SR_PER + i];
  SrRow q;
  q.settings(a, r);
  sr_clear();
  uint64_t first;
  float least;
  sr_joined(g, a.chunks, first, least);
  if (sr_simple(q, first, a, r, false)) return;
  q.range(first, least);
  __syncthreads();
  sr_run(c, m);
  SrCuts cut;
  if (sr_choose(q, cut) > SR_LIST) return;
  entries.each([&](int i, float x) {
    const int b = q.bin(x);
    if (s.fill[b] != ~0u) g.list[s.fill[b] + atomicAdd(&g.fill[b], 1u)] = sr_entry(sr_key(x), i);
  });
}
template <typename T>
__global__ __launch_bounds__(SR_NT) void sample_finish_kernel(SampleArgs a) {
  SrShared &s = sr_shared();
  const int r = blockIdx.x, t = threadIdx.x;
  const SrSplit &g = ((SrSplit *)a.split)[r];
  uint32_t c[SR_PER];
  uint64_t m[SR_PER];
#pragma unroll
  for (int i = 0; i < SR_PER; i++) c[i] = g.count[t * SR_PER + i], m[i] = g.mass[t * SR_PER + i];
  SrRow q;
  q.settings(a, r);
  sr_clear();
  uint64_t first;
  float least;
  sr_joined(g, a.chunks, first, least);
  if (sr_simple(q, first, a, r, false)) return;
  q.range(first, least);
  __syncthreads();
  sr_run(c, m);
  SrCuts cut;
  const uint32_t n = sr_choose(q, cut);
  if (n <= SR_LIST) {
    for (uint32_t i = t; i < n; i += SR_NT) s.list[i] = g.list[i];
    sr_own([&](int b) {
      if (s.fill[b] != ~0u) s.fill[b] += s.count[b + 1] - s.count[b];
    });
    __syncthreads();
    sr_finish(q, cut, n, a, r);
  } else {
    const SrStream<T, 1> entries{(const T *)a.logits + r * a.row_stride, 0, a.n};
    SrSearch<SrStream<T, 1>>{entries, q}.finish(cut, a, r);
  }
}

// How rows of n are dealt out: to a block each, held in its LDS where they
// fit, or several blocks each where there are fewer rows than compute units to
// keep busy
struct SamplePlan {
  int chunks, chunk;  // 0: one block
  bool held;
  size_t bytes;  // of workspace
};
inline SamplePlan sample_plan(int rows, int n, int cus) {
  constexpr int most = 8192;
  static_assert(most * SR_MAXCHUNKS >= SR_MAXN, "chunks");
  SamplePlan p{};
  p.held = n <= SR_HOLD;
  if (!p.held && rows * 2 <= cus) {
    p.chunks = (n + most - 1) / most;
    p.chunk = ((n + p.chunks - 1) / p.chunks + 7) / 8 * 8;
    p.bytes = sizeof(SrSplit) * (size_t)rows;
  }
  return p;
}

}  // namespace vx
