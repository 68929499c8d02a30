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
constexpr int SR_BINS = SR_PER * SR_NT, SR_CELLS = 2 * SR_NT, SR_LIST = SR_PER * SR_NT;
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

// Running sums are those before a bin, with the total behind the last one.
struct SrShared {
  uint64_t mass[SR_BINS + 1];
  uint32_t count[SR_BINS + 1];
  uint32_t fill[SR_BINS];  // where a gathered bin's next entry goes; ~0: not gathered
  union {
    struct {
      uint64_t list[SR_LIST], list_w[SR_LIST];
    };
    struct {
      uint64_t cell_mass[SR_CELLS];
      uint32_t cell_count[SR_CELLS];
    };
  };
  double tab[32];  // 2^(i / 32)
  uint64_t wave_m[SR_WAVES], found_m, found_e;
  uint32_t wave_c[SR_WAVES], found_c, n_list;
  int found[8];
  float wave_f[SR_WAVES];
};

// The block's LDS, always by its own name: a generic pointer to it would make
// every access a flat one.
__device__ __forceinline__ SrShared &sr_shared() {
  __shared__ SrShared s;
  return s;
}

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

// Entries of a row: f(index, x) for each that is in the order.  Both kinds
// read 16 bytes a thread at a time from aligned addresses.
// Up to U chunks of 16 bytes a thread, kept in registers from the first pass on
template <typename T, int U>
struct SrHeld {
  static constexpr int V = 16 / sizeof(T), MOST = SR_NT * U * V - V + 1;
  float x[U * V];
  int at;  // the index of this thread's first one
  __device__ __forceinline__ void load(const T *row, int from, int to) {
    const T *p = row + from;
    const int off = (int)(((uintptr_t)p & 15) / sizeof(T));  // p - off is aligned
    at = from + (int)threadIdx.x * V - off;
    PgVec<T, V> v[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i = at + u * SR_NT * V;
      if (i >= from && i + V <= to) {
        v[u] = *(const PgVec<T, V> *)(row + i);
      } else {
#pragma unroll
        for (int j = 0; j < V; j++) v[u].x[j] = i + j >= from && i + j < to ? row[i + j] : (T)NAN;
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int j = 0; j < V; j++) x[u * V + j] = (float)v[u].x[j];
  }
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int j = 0; j < V; j++)
        if (x[u * V + j] > -INFINITY) f(at + u * SR_NT * V + j, x[u * V + j]);
  }
};
// Any number, read again in every pass
template <typename T>
struct SrStream {
  const T *row;
  int n;
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    constexpr int V = 16 / sizeof(T), U = 2;
    const int off = (int)(((uintptr_t)row & 15) / sizeof(T));
    const int chunks = (n + off + V - 1) / V;
    for (int c0 = 0; c0 < chunks; c0 += SR_NT * U) {
      PgVec<T, V> x[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int i = (c0 + u * SR_NT + (int)threadIdx.x) * V - off;
        if (i >= 0 && i + V <= n) {
          x[u] = *(const PgVec<T, V> *)(row + i);
        } else {
#pragma unroll
          for (int j = 0; j < V; j++) x[u].x[j] = i + j >= 0 && i + j < n ? row[i + j] : (T)NAN;
        }
      }
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int j = 0; j < V; j++) {
          const float y = (float)x[u].x[j];
          if (y > -INFINITY) f((c0 + u * SR_NT + (int)threadIdx.x) * V - off + j, y);
        }
    }
  }
};

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
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t oc = __shfl_up(ic, d, 64);
    const uint64_t om = __shfl_up((unsigned long long)im, d, 64);
    if (lane >= d) ic += oc, im += om;
  }
  __syncthreads();
  if (lane == 63) s.wave_c[wave] = ic, s.wave_m[wave] = im;
  __syncthreads();
  tc = 0;
  tm = 0;
#pragma unroll
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

// the first entry and the least value over the block
template <typename E>
__device__ __forceinline__ void sr_range(const E &entries, uint64_t &first, float &least) {
  SrShared &s = sr_shared();
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // the maximum alone is one instruction an entry; its first index is looked for in the wave that has it
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
  if (threadIdx.x == 0) s.found_c = ~0u;
  __syncthreads();
  uint32_t key = 0;
  least = INFINITY;
#pragma unroll
  for (int w = 0; w < SR_WAVES; w++) {
    key = s.wave_m[w] > key ? (uint32_t)s.wave_m[w] : key;
    least = fminf(least, s.wave_f[w]);
  }
  if (key && sr_key(max) == key) {
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
  __syncthreads();
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

// A thread's gathered entries and their places: the entries and weights before
// each
struct SrPlaces {
  uint64_t e[SR_PER], w[SR_PER], m[SR_PER];
  uint32_t c[SR_PER];
  int b[SR_PER];  // bins; -1: none
  // Of the list's n entries, those of a bin lie together, at from .. to - 1,
  // running on from the sums (c, m) before it: before(bin, from, to, c, m).
  template <typename F>
  __device__ __forceinline__ void rank(const SrRow &q, uint32_t n, F before) {
    SrShared &s = sr_shared();
#pragma unroll
    for (int i = 0; i < SR_PER; i++) {
      const uint32_t at = threadIdx.x + i * SR_NT;
      e[i] = at < n ? s.list[at] : ~0ull;
      b[i] = at < n ? q.bin(sr_value_of(e[i])) : -1;
      w[i] = at < n ? q.weight(sr_value_of(e[i])) : 0;
      s.list_w[at] = w[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < SR_PER; i++) {
      if (b[i] < 0) continue;
      uint32_t from, to;
      before(b[i], from, to, c[i], m[i]);
      for (uint32_t j = from; j < to; j++) {
        const uint64_t o = s.list[j], ow = s.list_w[j];
        if (o < e[i]) c[i]++, m[i] += ow;
      }
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
  sr_range(entries, first, least);
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
template <typename T, int U>
__global__ __launch_bounds__(SR_NT) void sample_held_kernel(SampleArgs a) {
  const int r = blockIdx.x;
  SrHeld<T, U> entries;
  entries.load((const T *)a.logits + r * a.row_stride, 0, a.n);
  sr_row(entries, SrStream<T>{(const T *)a.logits + r * a.row_stride, a.n}, a, r);
}
template <typename T>
__global__ __launch_bounds__(SR_NT) void sample_rows_kernel(SampleArgs a) {
  const int r = blockIdx.x;
  const SrStream<T> entries{(const T *)a.logits + r * a.row_stride, a.n};
  sr_row(entries, entries, a, r);
}

// Several blocks a row, for a few long rows: the same passes as launches of
// their own, sums and gathered entries joined in memory (integers: the order
// of the blocks does not matter).
// the range of a chunk's values; clears what the next passes add to
template <typename T, int U>
__global__ __launch_bounds__(SR_NT) void sample_range_kernel(SampleArgs a) {
  const int r = blockIdx.x / a.chunks, k = blockIdx.x - r * a.chunks;
  SrSplit &g = ((SrSplit *)a.split)[r];
  SrHeld<T, U> entries;
  entries.load((const T *)a.logits + r * a.row_stride, k * a.chunk, min(a.n, (k + 1) * a.chunk));
  for (int i = k * SR_NT + threadIdx.x; i < SR_BINS; i += a.chunks * SR_NT) g.mass[i] = 0, g.count[i] = 0, g.fill[i] = 0;
  uint64_t first;
  float least;
  sr_range(entries, first, least);
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
template <typename T, int U>
__global__ __launch_bounds__(SR_NT) void sample_bins_kernel(SampleArgs a) {
  SrShared &s = sr_shared();
  const int r = blockIdx.x / a.chunks, k = blockIdx.x - r * a.chunks, t = threadIdx.x;
  SrSplit &g = ((SrSplit *)a.split)[r];
  SrHeld<T, U> entries;
  entries.load((const T *)a.logits + r * a.row_stride, k * a.chunk, min(a.n, (k + 1) * a.chunk));
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
template <typename T, int U>
__global__ __launch_bounds__(SR_NT) void sample_gather_kernel(SampleArgs a) {
  SrShared &s = sr_shared();
  const int r = blockIdx.x / a.chunks, k = blockIdx.x - r * a.chunks, t = threadIdx.x;
  SrSplit &g = ((SrSplit *)a.split)[r];
  SrHeld<T, U> entries;
  entries.load((const T *)a.logits + r * a.row_stride, k * a.chunk, min(a.n, (k + 1) * a.chunk));
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
    const SrStream<T> entries{(const T *)a.logits + r * a.row_stride, a.n};
    SrSearch<SrStream<T>>{entries, q}.finish(cut, a, r);
  }
}

// How rows of n are dealt out: to a block each, held in its registers where
// they fit, or several blocks each where there are fewer rows than compute
// units to keep busy
struct SamplePlan {
  int chunks, chunk;  // 0: one block
  bool held;
  size_t bytes;  // of workspace
};
template <typename T>
struct SrHold {
  static constexpr int U = sizeof(T) == 4 ? 3 : 2, SPLIT_U = sizeof(T) == 4 ? 2 : 1;  // 12288 or 16384 entries; 8192
};
template <typename T>
inline SamplePlan sample_plan(int rows, int n, int cus) {
  SamplePlan p{};
  p.held = n <= SrHeld<T, SrHold<T>::U>::MOST;
  if (!p.held && rows * 2 <= cus) {
    const int most = SrHeld<T, SrHold<T>::SPLIT_U>::MOST / 8 * 8;
    p.chunks = (n + most - 1) / most;
    p.chunk = ((n + p.chunks - 1) / p.chunks + 7) / 8 * 8;
    p.bytes = sizeof(SrSplit) * (size_t)rows;
  }
  return p;
}
static_assert(SrHeld<float, 2>::MOST / 8 * 8 * SR_MAXCHUNKS >= SR_MAXN && SrHeld<_Float16, 1>::MOST / 8 * 8 * SR_MAXCHUNKS >= SR_MAXN, "chunks");

}  // namespace vx
