// vx_batch.h -- host side of the operators on the caller's device memory
// (vx_paged_append, vx_paged_attend, vx_sample_rows): argument checks, launch
// plans and launches.  Calls keep no state, so they may run from several
// threads at once; a failed call's message belongs to its thread.
#pragma once
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "../../include/voxtral_engine.h"
#include "vx_paged.h"
#include "vx_sample.h"

namespace vx {

inline char *batch_error() {
  static thread_local char text[512] = "";
  return text;
}

__attribute__((format(printf, 2, 3))) inline int batch_fail(int code, const char *fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(batch_error(), 512, fmt, ap);
  va_end(ap);
  return code;
}

// makes `device` current for a call
struct OnDevice {
  int before = -1;
  hipError_t status;
  explicit OnDevice(int device) {
    int now = -1;
    status = hipGetDevice(&now);
    if (status == hipSuccess && now != device) {
      status = hipSetDevice(device);
      if (status == hipSuccess) before = now;
    }
  }
  ~OnDevice() {
    if (before >= 0) (void)hipSetDevice(before);
  }
};

template <typename A>
inline int batch_launch(const char *what, void (*kernel)(A), int64_t blocks, int threads, int lds, const A &args, void *stream) {
  if (blocks > 0x7fffffff) return batch_fail(VX_E_INVALID, "%s: %lld blocks: too much for one call", what, (long long)blocks);
  void *p[] = {const_cast<A *>(&args)};
  const hipError_t s = hipLaunchKernel((const void *)kernel, dim3((unsigned)blocks), dim3(threads), p, lds, (hipStream_t)stream);
  if (s != hipSuccess) {
    (void)hipGetLastError();
    return batch_fail(VX_E_DEVICE, "%s: kernel launch failed: %s", what, hipGetErrorString(s));
  }
  return VX_OK;
}

inline size_t type_size(int type) { return type == VX_TYPE_F32 ? 4 : 2; }
inline bool type_ok(int type) { return type >= VX_TYPE_F32 && type <= VX_TYPE_BF16; }
// the pairs of row and cache types there are kernels for
inline bool types_ok(int rows, int cache) {
  return type_ok(rows) && type_ok(cache) && (rows == cache || (rows == VX_TYPE_F32 && cache == VX_TYPE_F16));
}
// a pointer and its strides (elements of `size` bytes) that 16-byte accesses can use
inline bool aligned16(const void *p, size_t size, int64_t a, int64_t b) {
  const int64_t m = 16 / (int64_t)size;
  return ((uintptr_t)p & 15) == 0 && a % m == 0 && b % m == 0;
}

inline int check_kv(const char *what, const vx_paged_kv &kv, PagedKV *out) {
  if (!kv.k || !kv.v) return batch_fail(VX_E_INVALID, "%s: NULL cache", what);
  if (kv.head_dim != 64 && kv.head_dim != 128) return batch_fail(VX_E_INVALID, "%s: head_dim %d is not 64 or 128", what, kv.head_dim);
  if (kv.page_size < 16 || kv.page_size > 4096 || (kv.page_size & (kv.page_size - 1)))
    return batch_fail(VX_E_INVALID, "%s: page_size %d is not a power of two from 16 to 4096", what, kv.page_size);
  if (kv.n_pages < 1 || kv.n_kv_heads < 1 || kv.n_kv_heads > 1024)
    return batch_fail(VX_E_INVALID, "%s: %d pages, %d KV heads", what, kv.n_pages, kv.n_kv_heads);
  const size_t es = type_size(kv.type);
  if (kv.page_stride < 0 || kv.head_stride < 0 || kv.token_stride < kv.head_dim || !aligned16(kv.k, es, kv.page_stride, kv.head_stride) ||
      !aligned16(kv.v, es, kv.token_stride, 0))
    return batch_fail(VX_E_INVALID, "%s: the cache and its strides must be multiples of 16 bytes", what);
  if (kv.token_stride > (1 << 24)) return batch_fail(VX_E_RANGE, "%s: token stride %lld", what, (long long)kv.token_stride);
  *out = PagedKV{kv.k, kv.v, kv.page_stride, kv.head_stride, kv.token_stride, kv.n_pages, kv.page_size,
                 31 - __builtin_clz((unsigned)kv.page_size), kv.n_kv_heads};
  return VX_OK;
}

// f with a value of each type in place of the row and cache types
template <typename F>
inline int with_types(int rows, int cache, F f) {
  if (rows == VX_TYPE_F32) return cache == VX_TYPE_F32 ? f(float(), float()) : f(float(), _Float16());
  return rows == VX_TYPE_F16 ? f(_Float16(), _Float16()) : f(__bf16(), __bf16());
}

inline int paged_append(const vx_append_args *p, void *stream) {
  const char *what = "vx_paged_append";
  if (!p) return batch_fail(VX_E_INVALID, "%s: NULL arguments", what);
  AppendArgs a;
  if (int rc = check_kv(what, p->kv, &a.rows.kv)) return rc;
  if (!types_ok(p->type, p->kv.type)) return batch_fail(VX_E_INVALID, "%s: rows of type %d for a cache of type %d", what, p->type, p->kv.type);
  if (p->n_tokens < 0 || p->n_seqs < 0 || p->table_width < 0 || p->n_heads < 0 || p->n_heads > 4096)
    return batch_fail(VX_E_INVALID, "%s: %d tokens, %d sequences, %d table columns, %d heads", what, p->n_tokens, p->n_seqs, p->table_width, p->n_heads);
  if (p->rotary_dim < 0 || p->rotary_dim > p->kv.head_dim || p->rotary_dim % 16)
    return batch_fail(VX_E_INVALID, "%s: rotary_dim %d is not a multiple of 16 up to head_dim %d", what, p->rotary_dim, p->kv.head_dim);
  if (p->rotary_dim && !(p->theta > 0 && std::isfinite(p->theta))) return batch_fail(VX_E_INVALID, "%s: theta %g", what, p->theta);
  if (p->n_tokens == 0) return VX_OK;
  if (!p->k || !p->v || !p->pos || (p->q && !p->q_out) || (p->table_width > 0 && p->n_seqs > 0 && !p->table))
    return batch_fail(VX_E_INVALID, "%s: NULL argument", what);
  if (!p->seq && p->n_seqs < p->n_tokens)
    return batch_fail(VX_E_INVALID, "%s: %d tokens without sequence numbers for %d sequences", what, p->n_tokens, p->n_seqs);
  const size_t es = type_size(p->type);
  if (!aligned16(p->k, es, p->k_row, p->k_head) || !aligned16(p->v, es, p->v_row, p->v_head) ||
      (p->q && (!aligned16(p->q, es, p->q_row, p->q_head) || !aligned16(p->q_out, es, p->o_row, p->o_head))))
    return batch_fail(VX_E_INVALID, "%s: rows and their strides must be multiples of 16 bytes", what);
  if (p->n_seqs == 0 || p->table_width == 0) return VX_OK;  // no place to write to
  AppendRows &r = a.rows;
  r.k = p->k, r.v = p->v, r.q = p->n_heads ? p->q : nullptr, r.q_out = p->q_out;
  r.k_row = p->k_row, r.k_head = p->k_head, r.v_row = p->v_row, r.v_head = p->v_head;
  r.q_row = p->q_row, r.q_head = p->q_head, r.o_row = p->o_row, r.o_head = p->o_head;
  r.rotary_dim = p->rotary_dim, r.interleaved = p->interleaved;
  a.pos = p->pos, a.seq = p->seq, a.table = p->table, a.table_stride = p->table_stride;
  a.table_width = p->table_width, a.base = p->base, a.n_tokens = p->n_tokens, a.n_seqs = p->n_seqs;
  a.n_heads = p->n_heads, a.head_dim = p->kv.head_dim;
  // theta^(-2 i / rotary_dim) as a product of two of 16 powers
  const double step = p->rotary_dim ? -2.0 * std::log2(p->theta) / p->rotary_dim : 0;
  double low[8];
  for (int i = 0; i < 8; i++) low[i] = std::exp2(i * step);
  for (int i = 0; i < 64; i += 8) {
    const double high = i < p->rotary_dim / 2 ? std::exp2(i * step) * 0.15915494309189533577 : 0;
    for (int j = 0; j < 8; j++) a.turns[i + j] = high * low[j];
  }
  OnDevice on(p->kv.device);
  if (on.status != hipSuccess) return batch_fail(VX_E_DEVICE, "%s: device %d: %s", what, p->kv.device, hipGetErrorString(on.status));
  return with_types(p->type, p->kv.type, [&](auto rt, auto ct) {
    return batch_launch(what, paged_append_kernel<decltype(rt), decltype(ct)>, a.n_tokens, PA_NT, 0, a, stream);
  });
}

// compute units of a device (asked for once)
inline int device_cus(int device) {
  static int known[64] = {};
  if (device < 0 || device >= 64) return 256;
  int n = __atomic_load_n(&known[device], __ATOMIC_RELAXED);
  if (n) return n;
  if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess || n < 1) {
    (void)hipGetLastError();
    return 256;
  }
  __atomic_store_n(&known[device], n, __ATOMIC_RELAXED);
  return n;
}

inline int check_attend(const char *what, const vx_attend_args *p, PagedKV *kv, AttendPlan *plan) {
  if (!p) return batch_fail(VX_E_INVALID, "%s: NULL arguments", what);
  if (int rc = check_kv(what, p->kv, kv)) return rc;
  if (!types_ok(p->type, p->kv.type)) return batch_fail(VX_E_INVALID, "%s: rows of type %d for a cache of type %d", what, p->type, p->kv.type);
  if (p->n_heads < 1 || p->n_heads > 4096 || p->n_heads % p->kv.n_kv_heads)
    return batch_fail(VX_E_INVALID, "%s: %d heads for %d KV heads", what, p->n_heads, p->kv.n_kv_heads);
  if (p->n_rows < 0 || p->n_rows > (1 << 18) || p->n_seqs < 0 || p->n_seqs > (1 << 18) || p->table_width < 0 || p->prefix_count < 0)
    return batch_fail(VX_E_INVALID, "%s: %d rows, %d sequences, %d table columns, %d prefix pages", what, p->n_rows, p->n_seqs,
                      p->table_width, p->prefix_count);
  if (p->max_len < 0 || p->max_len > (int64_t)p->table_width * p->kv.page_size || p->max_len > (1 << 28))
    return batch_fail(VX_E_RANGE, "%s: max_len %d passes the table's %d pages of %d", what, p->max_len, p->table_width, p->kv.page_size);
  if (p->prefix_len < 0 || p->prefix_len > (int64_t)p->prefix_count * p->kv.page_size || p->prefix_len > (1 << 28))
    return batch_fail(VX_E_RANGE, "%s: prefix_len %d passes %d pages of %d", what, p->prefix_len, p->prefix_count, p->kv.page_size);
  if (!std::isfinite(p->scale)) return batch_fail(VX_E_INVALID, "%s: scale %g", what, p->scale);
  if (!p->row_start && p->n_seqs != p->n_rows)
    return batch_fail(VX_E_INVALID, "%s: %d rows of %d sequences without row_start", what, p->n_rows, p->n_seqs);
  *plan = attend_plan(p->n_rows, p->n_seqs, p->n_heads, p->kv.n_kv_heads, p->kv.head_dim, p->prefix_len, p->max_len,
                      p->row_start != nullptr, at_wide_cols(type_size(p->type), type_size(p->kv.type)), device_cus(p->kv.device));
  return VX_OK;
}

inline int paged_attend(const vx_attend_args *p, void *stream) {
  const char *what = "vx_paged_attend";
  AttendArgs a;
  AttendPlan plan;
  if (int rc = check_attend(what, p, &a.kv, &plan)) return rc;
  if (p->n_rows == 0 || p->n_seqs == 0) return VX_OK;
  if (!p->q || !p->out || !p->lens || (p->max_len > 0 && !p->table) || (p->prefix_len > 0 && !p->prefix_pages))
    return batch_fail(VX_E_INVALID, "%s: NULL argument", what);
  const size_t es = type_size(p->type);
  if (!aligned16(p->q, es, p->q_row, p->q_head) || !aligned16(p->out, es, p->o_row, p->o_head))
    return batch_fail(VX_E_INVALID, "%s: rows and their strides must be multiples of 16 bytes", what);
  if (plan.bytes > p->workspace_bytes || (plan.bytes && (!p->workspace || ((uintptr_t)p->workspace & 15))))
    return batch_fail(VX_E_INVALID, "%s: workspace of %zu bytes, %zu needed (aligned to 16)", what, p->workspace_bytes, plan.bytes);
  a.q = p->q, a.out = p->out, a.lse = p->lse;
  a.q_row = p->q_row, a.q_head = p->q_head, a.o_row = p->o_row, a.o_head = p->o_head;
  a.row_start = p->row_start, a.lens = p->lens, a.table = p->table, a.prefix_pages = p->prefix_pages;
  a.table_stride = p->table_stride, a.table_width = p->table_width, a.prefix_count = p->prefix_count;
  a.prefix_len = p->prefix_len, a.max_len = p->max_len;
  a.n_rows = p->n_rows, a.n_seqs = p->n_seqs, a.n_heads = p->n_heads, a.group = p->n_heads / p->kv.n_kv_heads;
  a.scale = (p->scale == 0 ? 1.0f / sqrtf((float)p->kv.head_dim) : p->scale) * 1.4426950408889634f;
  a.pre_cols = plan.pre_cols, a.pre_wide = plan.pre_wide, a.pre_tiles = plan.pre_tiles;
  a.pre_splits = plan.pre_splits, a.pre_chunk = plan.pre_chunk;
  a.own_cols = plan.own_cols, a.own_wide = plan.own_wide, a.own_slots = plan.own_slots;
  a.own_splits = plan.own_splits, a.own_chunk = plan.own_chunk;
  a.fused = plan.fused, a.team = plan.team;
  a.part_o = (float *)p->workspace;
  a.part_ml = (float2 *)((char *)p->workspace + plan.ml_at);
  OnDevice on(p->kv.device);
  if (on.status != hipSuccess) return batch_fail(VX_E_DEVICE, "%s: device %d: %s", what, p->kv.device, hipGetErrorString(on.status));
  return with_types(p->type, p->kv.type, [&](auto r, auto c) {
    auto go = [&](auto part, auto join) {
      int rc = plan.blocks ? batch_launch(what, part, plan.blocks, 64 * AT_WAVES, 0, a, stream) : VX_OK;
      return rc || plan.direct() ? rc : batch_launch(what, join, at_ceil((int64_t)a.n_rows * a.n_heads, AT_WAVES / a.team), 64 * AT_WAVES, 0, a, stream);
    };
    using R = decltype(r);
    using C = decltype(c);
    const bool hd128 = p->kv.head_dim == 128;
    if constexpr (AtTypes<R, C, 128>::WIDE > 0) {
      if ((plan.pre_wide && plan.pre_splits) || plan.own_wide)
        return hd128 ? go(paged_attend_kernel<R, C, 128, true>, paged_attend_join_kernel<R, 128>)
                     : go(paged_attend_kernel<R, C, 64, true>, paged_attend_join_kernel<R, 64>);
    }
    return hd128 ? go(paged_attend_kernel<R, C, 128, false>, paged_attend_join_kernel<R, 128>)
                 : go(paged_attend_kernel<R, C, 64, false>, paged_attend_join_kernel<R, 64>);
  });
}

inline int check_sample(const char *what, const vx_sample_args *p, SamplePlan *plan) {
  if (!p) return batch_fail(VX_E_INVALID, "%s: NULL arguments", what);
  if (!type_ok(p->type)) return batch_fail(VX_E_INVALID, "%s: logits of type %d", what, p->type);
  if (p->rows < 0 || p->n < 1) return batch_fail(VX_E_INVALID, "%s: %d rows of %d logits", what, p->rows, p->n);
  if (p->n > SR_MAXN) return batch_fail(VX_E_RANGE, "%s: %d logits a row, more than %d", what, p->n, SR_MAXN);
  *plan = sample_plan(p->rows, p->n, device_cus(p->device));
  return VX_OK;
}

// a launch with S in dynamic LDS; what passes 64 KB is announced once for each device
template <typename S, void (*K)(SampleArgs)>
inline int sample_kernel(const char *what, int64_t blocks, const SampleArgs &a, int device, void *stream) {
  static uint64_t announced = 0;  // bits of devices
  const uint64_t bit = 1ull << (device & 63);
  if (sizeof(S) > 64 * 1024 && !(__atomic_load_n(&announced, __ATOMIC_RELAXED) & bit)) {
    const hipError_t e = hipFuncSetAttribute((const void *)K, hipFuncAttributeMaxDynamicSharedMemorySize, sizeof(S));
    if (e != hipSuccess) {
      (void)hipGetLastError();
      return batch_fail(VX_E_DEVICE, "%s: LDS size rejected: %s", what, hipGetErrorString(e));
    }
    __atomic_fetch_or(&announced, bit, __ATOMIC_RELAXED);
  }
  return batch_launch(what, K, blocks, SR_NT, sizeof(S), a, stream);
}

template <typename T>
inline int sample_launch(const char *what, const SamplePlan &plan, const SampleArgs &a, int device, void *stream) {
  if (!plan.chunks) {
    if (plan.held) return sample_kernel<SrShared, sample_rows_kernel<T, true>>(what, a.rows, a, device, stream);
    if constexpr (sizeof(T) == 2) return sample_kernel<SrValues, sample_values_kernel<T>>(what, a.rows, a, device, stream);
    else return sample_kernel<SrShared, sample_rows_kernel<T, false>>(what, a.rows, a, device, stream);
  }
  const int64_t blocks = (int64_t)a.rows * plan.chunks;
  int rc = sample_kernel<SrShared, sample_range_kernel<T>>(what, blocks, a, device, stream);
  if (!rc) rc = sample_kernel<SrShared, sample_bins_kernel<T>>(what, blocks, a, device, stream);
  if (!rc) rc = sample_kernel<SrShared, sample_gather_kernel<T>>(what, blocks, a, device, stream);
  if (!rc) rc = sample_kernel<SrShared, sample_finish_kernel<T>>(what, a.rows, a, device, stream);
  return rc;
}

inline int sample_rows(const vx_sample_args *p, void *stream) {
  const char *what = "vx_sample_rows";
  SamplePlan plan;
  if (int rc = check_sample(what, p, &plan)) return rc;
  if (!p->temperature && !(std::isfinite(p->temperature0) && p->temperature0 >= 0))
    return batch_fail(VX_E_INVALID, "%s: temperature %g", what, p->temperature0);
  if (!p->top_p && !(p->top_p0 > 0 && p->top_p0 <= 1)) return batch_fail(VX_E_INVALID, "%s: top_p %g", what, p->top_p0);
  if (!p->min_p && !(p->min_p0 >= 0 && p->min_p0 <= 1)) return batch_fail(VX_E_INVALID, "%s: min_p %g", what, p->min_p0);
  if (!p->top_k && p->top_k0 < 0) return batch_fail(VX_E_INVALID, "%s: top_k %d", what, p->top_k0);
  if (p->rows == 0) return VX_OK;
  if (!p->logits || !p->u || !p->token) return batch_fail(VX_E_INVALID, "%s: NULL argument", what);
  if ((uintptr_t)p->logits % type_size(p->type)) return batch_fail(VX_E_INVALID, "%s: logits are not aligned to their type", what);
  if (plan.bytes > p->workspace_bytes || (plan.bytes && (!p->workspace || ((uintptr_t)p->workspace & 15))))
    return batch_fail(VX_E_INVALID, "%s: workspace of %zu bytes, %zu needed (aligned to 16)", what, p->workspace_bytes, plan.bytes);
  const SampleArgs a{p->logits, p->row_stride, p->rows, p->n, p->temperature, p->top_p, p->min_p, p->top_k, p->u,
                     p->temperature0, p->top_p0, p->min_p0, p->top_k0, p->token, p->kept, p->prob,
                     plan.chunks, plan.chunk, (char *)p->workspace};
  OnDevice on(p->device);
  if (on.status != hipSuccess) return batch_fail(VX_E_DEVICE, "%s: device %d: %s", what, p->device, hipGetErrorString(on.status));
  return p->type == VX_TYPE_F32 ? sample_launch<float>(what, plan, a, p->device, stream)
         : p->type == VX_TYPE_F16 ? sample_launch<_Float16>(what, plan, a, p->device, stream)
                                  : sample_launch<__bf16>(what, plan, a, p->device, stream);
}

}  // namespace vx
