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
// No row is sorted.  A pass over it counts entries and sums weights in 4096
// bins that fall with x, and a cut is then looked for in the one bin where it
// lies: its entries (or all entries up to it, if they are few) are gathered
// and sorted in LDS.  A bin of too many entries (ties above all) is narrowed
// first, by digits of (value, index).
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
};

constexpr int SR_NT = 1024, SR_WAVES = SR_NT / 64;
constexpr int SR_BINS = 4096, SR_CELLS = 2048, SR_CAP = 4096;
constexpr int SR_MAXN = 1 << 20;  // 2^43 weights: sums stay below 2^63
constexpr int SR_FIX = 43;

// the row's values as a key that rises with them; 0: not in the order
__device__ __forceinline__ uint32_t sr_key(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);  // -0 counts as 0
  return x > -INFINITY ? (b >> 31 ? ~b : b | 0x80000000u) : 0;
}
__device__ __forceinline__ float sr_value(uint32_t key) {
  return __builtin_bit_cast(float, key >> 31 ? key & 0x7fffffffu : ~key);
}

// the bin of an entry: falls from the maximum over the range of weights
struct SrBin {
  float max, scale;
  __device__ __forceinline__ int operator()(float x) const {
    return x == max ? 0 : (int)fminf((max - x) * scale, (float)(SR_BINS - 1));
  }
};

// Running sums are those before an entry, with the total behind the last one.
struct SrShared {
  uint64_t mass[SR_BINS + 1];  // over the bins
  uint32_t count[SR_BINS + 1];
  uint64_t cell_mass[SR_CELLS];
  uint32_t cell_count[SR_CELLS];
  uint64_t list[SR_CAP], list_mass[SR_CAP + 1];  // gathered entries in order
  double tab[32];                                // 2^(i / 32)
  uint64_t wave_m[SR_WAVES], found_m, found_e;
  uint32_t wave_c[SR_WAVES], found_c, n_list;
  int found;
};

// The block's LDS, always by its own name: a generic pointer to it would make
// every access a flat one.
__device__ __forceinline__ SrShared &sr_shared() {
  extern __shared__ __attribute__((aligned(16))) unsigned char sr_smem[];
  return *(SrShared *)sr_smem;
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

// f(index, x) for every entry of the row, 16 bytes a thread at a time from
// aligned addresses
template <typename T, typename F>
__device__ __forceinline__ void sr_each(const T *row, int n, F f) {
  constexpr int V = 16 / sizeof(T), U = 2;
  const int off = (int)(((uintptr_t)row & 15) / sizeof(T));  // row - off is aligned
  const int chunks = (n + off + V - 1) / V;
  for (int c0 = 0; c0 < chunks; c0 += SR_NT * U) {
    PgVec<T, V> x[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int c = c0 + u * SR_NT + threadIdx.x, i = c * V - off;
      if (i >= 0 && i + V <= n) {
        x[u] = *(const PgVec<T, V> *)(row + i);
      } else {
#pragma unroll
        for (int j = 0; j < V; j++) x[u].x[j] = i + j >= 0 && i + j < n ? row[i + j] : (T)0;
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i = (c0 + u * SR_NT + threadIdx.x) * V - off;
#pragma unroll
      for (int j = 0; j < V; j++)
        if (i + j >= 0 && i + j < n) f(i + j, (float)x[u].x[j]);
    }
  }
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
  for (int w = 0; w < SR_WAVES; w++) {
    if (w == wave) bc = tc, bm = tm;
    tc += s.wave_c[w];
    tm += s.wave_m[w];
  }
#pragma unroll
  for (int i = 0; i < PER; i++) c[i] += bc + ic - ac, m[i] += bm + im - am;
}

// What a cut is looked for by: a running count or a running sum
enum SrKind { SR_COUNT, SR_MASS };

// An entry is (~key) << 32 | index, which rises along the order.  One block
// a row.
template <typename T>
struct SrRow {
  const T *row;
  int n;
  SrWeight weight;
  SrBin bin;
  // what the list holds: the entries behind running count base_c and sum base_m
  uint32_t base_c, end_c;
  uint64_t base_m, end_m;

  static __device__ __forceinline__ uint64_t entry(uint32_t key, int i) { return (uint64_t)~key << 32 | (uint32_t)i; }
  // whether the target-th of a running quantity lies in (before, after]
  static __device__ __forceinline__ bool inside(uint64_t target, uint64_t before, uint64_t after) {
    return before < target && target <= after;
  }

  // The entry that a cut falls on: the first whose running count or sum (it
  // included) is at least `target`, which the row's total is too.  Its own
  // running count and sum go to (c, m).
  __device__ __forceinline__ uint64_t find(SrKind kind, uint64_t target, uint32_t &c, uint64_t &m) {
    SrShared &s = sr_shared();
    if (!(kind == SR_COUNT ? inside(target, base_c, end_c) : inside(target, base_m, end_m))) bring(kind, target);
    __syncthreads();
    for (int i = threadIdx.x; i < (int)(end_c - base_c); i += SR_NT)
      if (kind == SR_COUNT ? base_c + i + 1 == target : inside(target, s.list_mass[i], s.list_mass[i + 1]))
        s.found_e = s.list[i], s.found_c = base_c + i + 1, s.found_m = s.list_mass[i + 1];
    __syncthreads();
    c = s.found_c;
    m = s.found_m;
    return s.found_e;
  }

  // makes the list hold the place of a cut
  __device__ __forceinline__ void bring(SrKind kind, uint64_t target) {
    SrShared &s = sr_shared();
    __syncthreads();
    for (int b = threadIdx.x; b < SR_BINS; b += SR_NT)
      if (kind == SR_COUNT ? inside(target, s.count[b], s.count[b + 1]) : inside(target, s.mass[b], s.mass[b + 1])) s.found = b;
    __syncthreads();
    // the entries of bins first .. b whose leading digits, all above `bits`, are `lead`
    const int b = s.found;
    int first = b, bits = 64;
    uint64_t lead = 0;
    uint32_t c0 = s.count[b], left = s.count[b + 1] - c0;
    uint64_t m0 = s.mass[b];
    if (s.count[b + 1] <= SR_CAP) {  // all entries up to the cut: later cuts lie among them too
      first = 0;
      left += c0;
      c0 = 0;
      m0 = 0;
    }
    auto in = [&](uint64_t e, float x) {
      const int at = bin(x);
      return at >= first && at <= b && (bits == 64 || e >> bits == lead);
    };
    // narrowed by digits of 10, 11 and 11 bits of the value, then by runs of 1024 indices
    for (int shift = 54; left > SR_CAP; shift = shift > 32 ? shift - 11 : 10) {
      for (int i = threadIdx.x; i < SR_CELLS; i += SR_NT) s.cell_count[i] = 0, s.cell_mass[i] = 0;
      __syncthreads();
      sr_each(row, n, [&](int i, float x) {
        const uint32_t k = sr_key(x);
        const uint64_t e = entry(k, i);
        if (!k || !in(e, x)) return;
        const int cell = (int)(e >> shift) & (SR_CELLS - 1);
        atomicAdd(&s.cell_count[cell], 1u);
        atomicAdd((unsigned long long *)&s.cell_mass[cell], (unsigned long long)weight(x));
      });
      __syncthreads();
      constexpr int P = SR_CELLS / SR_NT;
      uint32_t c[P], own[P], tc;
      uint64_t m[P], own_m[P], tm;
#pragma unroll
      for (int i = 0; i < P; i++) {
        c[i] = own[i] = s.cell_count[P * threadIdx.x + i];
        m[i] = own_m[i] = s.cell_mass[P * threadIdx.x + i];
      }
      sr_scan(c, m, tc, tm);
#pragma unroll
      for (int i = 0; i < P; i++)
        if (kind == SR_COUNT ? inside(target, c0 + c[i], c0 + c[i] + own[i]) : inside(target, m0 + m[i], m0 + m[i] + own_m[i])) {
          s.found = P * threadIdx.x + i;
          s.found_c = c[i];
          s.found_m = m[i];
          s.n_list = own[i];
        }
      __syncthreads();
      c0 += s.found_c;
      m0 += s.found_m;
      left = s.n_list;
      lead = (bits < 64 ? lead << (bits - shift) : 0) | (uint64_t)s.found;
      bits = shift;
      __syncthreads();
    }
    // gathered, sorted, and their sums run on
    if (threadIdx.x == 0) s.n_list = 0;
    __syncthreads();
    sr_each(row, n, [&](int i, float x) {
      const uint32_t k = sr_key(x);
      const uint64_t e = entry(k, i);
      if (!k || !in(e, x)) return;
      const uint32_t at = atomicAdd(&s.n_list, 1u);
      if (at < SR_CAP) s.list[at] = e;
    });
    int size = 2;
    while (size < (int)left) size <<= 1;
    __syncthreads();
    for (int i = left + threadIdx.x; i < size; i += SR_NT) s.list[i] = ~0ull;
    for (int k = 2; k <= size; k <<= 1)
      for (int j = k >> 1; j > 0; j >>= 1) {
        __syncthreads();
        for (int p = threadIdx.x; p < size >> 1; p += SR_NT) {
          const int x = ((p & ~(j - 1)) << 1) | (p & (j - 1)), y = x | j;
          const uint64_t u = s.list[x], v = s.list[y];
          if ((u > v) == ((x & k) == 0)) s.list[x] = v, s.list[y] = u;
        }
      }
    __syncthreads();
    constexpr int P = SR_CAP / SR_NT;
    uint32_t c[P], tc;
    uint64_t m[P], tm;
#pragma unroll
    for (int i = 0; i < P; i++) {
      const uint32_t at = threadIdx.x * P + i;
      c[i] = 1;
      m[i] = at < left ? weight(sr_value(~(uint32_t)(s.list[at] >> 32))) : 0;
    }
    sr_scan(c, m, tc, tm);
#pragma unroll
    for (int i = 0; i < P; i++) s.list_mass[threadIdx.x * P + i] = m0 + m[i];
    if (threadIdx.x == 0) s.list_mass[SR_CAP] = m0 + tm;
    base_c = c0;
    end_c = c0 + left;
    base_m = m0;
    end_m = m0 + tm;
  }

  // the count and the sum of the entries with keys of at least `key`
  __device__ __forceinline__ void from_key(uint32_t key, uint32_t &c, uint64_t &m) {
    uint32_t cs[1] = {0};
    uint64_t ms[1] = {0};
    sr_each(row, n, [&](int, float x) {
      if (sr_key(x) >= key) cs[0]++, ms[0] += weight(x);
    });
    sr_scan(cs, ms, c, m);
  }
};

template <typename T>
__global__ __launch_bounds__(SR_NT) void sample_rows_kernel(SampleArgs a) {
  SrShared &s = sr_shared();
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const T *row = (const T *)a.logits + r * a.row_stride;
  const float temp = a.temperature ? a.temperature[r] : a.temperature0;
  const float top_p = a.top_p ? a.top_p[r] : a.top_p0, min_p = a.min_p ? a.min_p[r] : a.min_p0;
  const int top_k = a.top_k ? a.top_k[r] : a.top_k0;

  // the first entry of the order
  uint64_t first = ~0ull;
  sr_each(row, a.n, [&](int i, float x) {
    const uint32_t k = sr_key(x);
    const uint64_t e = SrRow<T>::entry(k, i);
    if (k && e < first) first = e;
  });
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) {
    const uint64_t o = __shfl_xor((unsigned long long)first, d, 64);
    first = o < first ? o : first;
  }
  if (lane == 0) s.wave_m[wave] = first;
  if (tid < 32) s.tab[tid] = exp2(tid / 32.0);
  for (int i = tid; i < SR_BINS; i += SR_NT) s.mass[i] = 0, s.count[i] = 0;
  __syncthreads();
  for (int w = 0; w < SR_WAVES; w++) first = s.wave_m[w] < first ? s.wave_m[w] : first;
  if (first == ~0ull || !(temp > 0)) {  // nothing to draw from, or the greedy choice
    if (tid == 0) {
      const bool none = first == ~0ull;
      a.token[r] = none ? -1 : (int)(uint32_t)first;
      if (a.kept) a.kept[r] = none ? 0 : 1;
      if (a.prob) a.prob[r] = none ? 0.0f : 1.0f;
    }
    return;
  }
  const uint32_t top = ~(uint32_t)(first >> 32);
  const float max = sr_value(top);
  SrRow<T> q{row, a.n, {(double)max, 1.4426950408889634 / temp, max == INFINITY},
             {max, fminf((float)(SR_BINS / 31.0) / temp, 1e30f)}, 0, 0, 0, 0};

  sr_each(row, a.n, [&](int, float x) {
    if (!(x > -INFINITY)) return;
    const int b = q.bin(x);
    atomicAdd(&s.count[b], 1u);
    const uint64_t w = q.weight(x);
    if (w) atomicAdd((unsigned long long *)&s.mass[b], (unsigned long long)w);
  });
  __syncthreads();
  uint32_t count, c;
  uint64_t mass, m, e = 0;
  {
    constexpr int P = SR_BINS / SR_NT;
    uint32_t cs[P];
    uint64_t ms[P];
#pragma unroll
    for (int i = 0; i < P; i++) cs[i] = s.count[tid * P + i], ms[i] = s.mass[tid * P + i];
    sr_scan(cs, ms, count, mass);
#pragma unroll
    for (int i = 0; i < P; i++) s.count[tid * P + i] = cs[i], s.mass[tid * P + i] = ms[i];
    if (tid == 0) s.count[SR_BINS] = count, s.mass[SR_BINS] = mass;
  }
  __syncthreads();

  // the cuts, then the draw: (count, mass) of what is kept so far
  uint64_t goal = ~0ull;  // top-p: the kept sum reaches this
  for (int step = 0; step < 3; step++) {
    uint64_t target;
    if (step == 0) {
      if (!(top_k > 0 && (uint32_t)top_k < count)) continue;
      target = top_k;
    } else if (step == 1) {
      if (top_p < 1.0f) {
        const double t = ceil((double)fmaxf(top_p, 0.0f) * (double)mass);
        goal = t < 1.0 ? 1 : (uint64_t)t < mass ? (uint64_t)t : mass;
      }
      if (min_p > 0.0f) {
        // the smallest key whose weight is at least min_p (the maximum's is
        // 1): 64 trials a step, each wave for itself
        uint32_t lo = 0, hi = top;  // lo: below it, hi: not below it
        while (hi - lo > 1) {
          const uint32_t by = (hi - lo + 63) / 64;
          const uint64_t at = (uint64_t)lo + (uint64_t)by * (lane + 1);
          const uint32_t k = at < hi ? (uint32_t)at : hi;
          const float x = sr_value(k);
          const bool yes = k == hi || (x > -INFINITY && !q.weight.inf && q.weight.power(x) >= (double)min_p * 0x1p43);
          const int i = __ffsll((unsigned long long)__ballot(yes)) - 1;
          const uint64_t up = (uint64_t)lo + (uint64_t)by * (i + 1);
          lo = lo + by * i;
          hi = up < hi ? (uint32_t)up : hi;
        }
        // where the bins before it hold as much as the other cuts leave, it cuts nothing
        const int b = q.bin(sr_value(hi));
        if (s.count[b] < count && s.mass[b] < goal) {
          q.from_key(hi, c, m);
          if (c < count) count = c, mass = m;
        }
      }
      if (goal > mass) continue;
      target = goal;
    } else {
      const double t = floor(a.u[r] * (double)mass);
      target = !(t > 0.0) ? 1 : t >= (double)mass ? mass : (uint64_t)t + 1;
    }
    e = q.find(step ? SR_MASS : SR_COUNT, target, c, m);
    if (step < 2 && c < count) count = c, mass = m;
  }
  if (tid == 0) {
    a.token[r] = (int)(uint32_t)e;
    if (a.kept) a.kept[r] = (int)count;
    const double w = q.weight.inf ? 0x1p43 : q.weight.power(sr_value(~(uint32_t)(e >> 32)));
    if (a.prob) a.prob[r] = (float)(w / (double)mass);
  }
}

}  // namespace vx
