"""Host side of the batch operators, on the CPU: the argument structures'
layout, refusals that the C ABI makes before anything touches a device, the
page lookup with bad ids, and the attention's plan (every column tile and
split, each once, inside the workspace)."""
import ctypes
import os
import subprocess
import threading

import pytest

import voxtral_amd as V
from voxtral_amd import batch as B

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = "/opt/rocm/bin/hipcc"
P = 1 << 20  # an address that is never used


def kv(k=P, v=P, page_stride=32768, head_stride=2048, token_stride=128, n_pages=4, page_size=16, n_kv_heads=8, head_dim=128, type=1):
    return B._KV.pack(k, v, page_stride, head_stride, token_stride, n_pages, page_size, n_kv_heads, head_dim, type, 0)


def append(cache=None, **kw):
    a = dict(k=P, v=P, k_row=1024, k_head=128, v_row=1024, v_head=128, q=0, q_out=0, q_row=0, q_head=0, o_row=0, o_head=0, pos=P, seq=P,
             table=P, table_stride=4, table_width=4, base=0, n_tokens=3, n_seqs=2, n_heads=0, type=1, theta=1e6, rotary_dim=128,
             interleaved=1)
    assert set(kw) <= set(a)
    a.update(kw)
    return V.load_library().vx_paged_append(B._APPEND.pack(cache or kv(), *a.values()), None)


def attend(cache=None, f="vx_paged_attend", **kw):
    a = dict(q=P, out=P, lse=0, q_row=4096, q_head=128, o_row=4096, o_head=128, row_start=0, lens=P, table=P, prefix_pages=P, table_stride=4,
             table_width=4, prefix_count=2, prefix_len=20, max_len=50, n_rows=3, n_seqs=3, n_heads=32, type=1, scale=0.0, workspace=0,
             workspace_bytes=0)
    assert set(kw) <= set(a)
    a.update(kw)
    n = ctypes.c_size_t()
    rc = getattr(V.load_library(), f)(B._ATTEND.pack(cache or kv(), *a.values()), ctypes.byref(n) if "workspace" in f else None)
    return (rc, n.value) if "workspace" in f else rc


def sample(**kw):
    a = dict(logits=P, row_stride=100, temperature=0, top_p=0, min_p=0, top_k=0, u=P, token=P, kept=0, prob=0, rows=2, n=100, type=0,
             device=0, temperature0=1.0, top_p0=1.0, min_p0=0.0, top_k0=0, workspace=0, workspace_bytes=0)
    assert set(kw) <= set(a)
    a.update(kw)
    return V.load_library().vx_sample_rows(B._SAMPLE.pack(*a.values()), None)


def error():
    return V.load_library().vx_batch_error().decode()


@pytest.mark.parametrize("call,text", [
    (lambda: append(kv(k=0)), "NULL cache"),
    (lambda: append(kv(head_dim=96)), "head_dim 96"),
    (lambda: append(kv(page_size=24)), "page_size 24"),
    (lambda: append(kv(page_size=8192)), "page_size 8192"),
    (lambda: append(kv(n_pages=0)), "0 pages"),
    (lambda: append(kv(token_stride=132)), "multiples of 16"),
    (lambda: append(kv(token_stride=64)), "multiples of 16"),
    (lambda: append(kv(k=P + 8)), "multiples of 16"),
    (lambda: append(type=3), "rows of type 3"),
    (lambda: append(type=2), "rows of type 2 for a cache of type 1"),
    (lambda: append(kv(type=0), type=1), "rows of type 1 for a cache of type 0"),
    (lambda: append(n_tokens=-1), "-1 tokens"),
    (lambda: append(rotary_dim=8), "rotary_dim 8"),
    (lambda: append(rotary_dim=144), "rotary_dim 144"),
    (lambda: append(theta=0.0), "theta 0"),
    (lambda: append(theta=float("nan")), "theta"),
    (lambda: append(k=0), "NULL argument"),
    (lambda: append(q=P, n_heads=4, q_row=512, q_head=128), "NULL argument"),
    (lambda: append(seq=0), "without sequence numbers"),
    (lambda: append(k_row=1028), "multiples of 16"),
    (lambda: append(v=P + 4), "multiples of 16"),
    (lambda: attend(n_heads=12), "12 heads for 8"),
    (lambda: attend(n_heads=0), "0 heads"),
    (lambda: attend(n_rows=1 << 19, n_seqs=1 << 19), "rows"),
    (lambda: attend(max_len=65), "max_len 65"),
    (lambda: attend(prefix_len=33), "prefix_len 33"),
    (lambda: attend(scale=float("inf")), "scale"),
    (lambda: attend(n_rows=4), "without row_start"),
    (lambda: attend(lens=0), "NULL argument"),
    (lambda: attend(prefix_pages=0), "NULL argument"),
    (lambda: attend(q_head=132), "multiples of 16"),
    (lambda: attend(prefix_len=2000, prefix_count=125), "workspace of 0 bytes"),
    (lambda: attend(prefix_len=2000, prefix_count=125, workspace=P + 8, workspace_bytes=1 << 30), "aligned to 16"),
    (lambda: sample(type=7), "type 7"),
    (lambda: sample(n=0), "0 logits"),
    (lambda: sample(n=(1 << 20) + 1), "more than"),
    (lambda: sample(temperature0=float("inf")), "temperature"),
    (lambda: sample(top_p0=0.0), "top_p 0"),
    (lambda: sample(top_p0=float("nan")), "top_p"),
    (lambda: sample(min_p0=-0.1), "min_p"),
    (lambda: sample(top_k0=-1), "top_k -1"),
    (lambda: sample(u=0), "NULL argument"),
    (lambda: sample(logits=P + 2), "aligned to their type"),
    (lambda: sample(n=131072), "workspace of 0 bytes"),
    (lambda: sample(n=131072, workspace=P + 4, workspace_bytes=1 << 30), "aligned to 16"),
])
def test_refusals(call, text):
    assert call() in (V.VX_E_INVALID, V.VX_E_RANGE)
    assert text in error()


def test_null_arguments_and_empty_calls():
    L = V.load_library()
    for f in (L.vx_paged_append, L.vx_paged_attend, L.vx_sample_rows):
        assert f(None, None) == V.VX_E_INVALID and "NULL" in error()
    assert L.vx_paged_attend_workspace(None, None) == V.VX_E_INVALID
    assert append(n_tokens=0, k=0, v=0, pos=0) == V.VX_OK
    assert append(n_seqs=0) == V.VX_OK and append(table_width=0, table=0) == V.VX_OK
    assert attend(n_rows=0, n_seqs=0, q=0, out=0, lens=0, table=0) == V.VX_OK
    assert sample(rows=0, logits=0, u=0, token=0) == V.VX_OK


def test_errors_belong_to_their_thread():
    assert sample(n=0) == V.VX_E_INVALID
    seen = []

    def other():
        seen.append(error())
        sample(type=9)
        seen.append(error())

    t = threading.Thread(target=other)
    t.start()
    t.join()
    assert seen[0] == "" and "type 9" in seen[1] and "0 logits" in error()


def test_workspace_covers_every_partial():
    rc, n = attend(f="vx_paged_attend_workspace", prefix_len=2000, prefix_count=125)
    assert rc == V.VX_OK and n >= 2 * 3 * 32 * (128 + 2) * 4
    assert attend(f="vx_paged_attend_workspace") == (V.VX_OK, 0)  # one split in all: no partials
    assert attend(f="vx_paged_attend_workspace", prefix_len=0, max_len=0) == (V.VX_OK, 0)


def test_sample_workspace_by_sizes():
    L = V.load_library()
    assert L.vx_sample_rows_workspace(None, None) == V.VX_E_INVALID
    sizes = [B._sample_space(L, rows, n, kind, 0) for rows, n, kind in ((1, 8320, 0), (500, 131072, 2), (8, 131072, 0), (1, 1 << 20, 1))]
    assert sizes[:2] == [0, 0] and sizes[2] == 8 * sizes[3] > 0


PROGRAM = r"""
#include "vx_paged.h"
#include <cstdio>
#include <vector>
using namespace vx;
int main() {
  const int ids[4] = {3, -1, 7, 8};
  const int want[] = {3, 3, -1, -1, 7, -1, -1};
  const int64_t slot[] = {0, 15, 16, 31, 32, 48, 64};
  for (int i = 0; i < 7; i++)
    if (pg_page(ids, 4, slot[i], 4, 8) != want[i]) return 1;
  if (pg_page(ids, 4, -1, 4, 8) != -1 || pg_page(ids, 4, INT64_MAX, 4, 8) != -1 || pg_page(ids, 0, 0, 4, 8) != -1) return 2;
  const int heads[][2] = {{32, 8}, {16, 16}, {40, 8}, {8, 1}, {28, 4}, {1, 1}, {96, 2}, {128, 1}};
  const int rows[] = {1, 2, 5, 16, 64, 333, 4000}, lens[] = {0, 1, 31, 32, 127, 128, 1000, 16000, 200000};
  for (auto &h : heads)
    for (int r : rows)
      for (int len : lens)
        for (int pre : lens)
          for (int hd : {64, 128})
            for (bool ragged : {false, true})
            for (int wide_cols : {0, 64, 128}) {
              const int seqs = ragged ? (r + 2) / 3 : r, g = h[0] / h[1];
              const AttendPlan p = attend_plan(r, seqs, h[0], h[1], hd, pre, len, ragged, wide_cols, 256);
              if (pre && !p.fused && ((int64_t)p.pre_splits * p.pre_chunk < pre || (int64_t)(p.pre_splits - 1) * p.pre_chunk >= pre ||
                                      p.pre_chunk % 32 || (int64_t)p.pre_tiles * p.pre_cols < (int64_t)r * g))
                return 3;
              // a fused block's keys: the prefix in whole steps, then its own
              const int64_t own = len + (p.fused ? at_ceil(pre, 32) * 32 : 0);
              if (len && ((int64_t)p.own_splits * p.own_chunk < own || (int64_t)(p.own_splits - 1) * p.own_chunk >= own || p.own_chunk % 32))
                return 4;
              if (p.fused && (p.pre_splits || p.pre_tiles || !len)) return 5;
              if (p.pre_wide ? p.pre_cols != wide_cols : p.pre_cols != 16 && p.pre_cols != 32 && p.pre_cols != 64) return 9;
              if (p.own_wide ? p.own_cols != wide_cols : p.own_cols != 16 && p.own_cols != 32 && p.own_cols != 64) return 9;
              if (p.blocks > 0x7fffffff || p.ml_at % 16) return 6;
              const size_t items = (size_t)(p.pre_splits + p.own_splits) * r * h[0];
              if (!p.direct() && (p.bytes < items * (hd * 4 + 8) || p.ml_at < items * hd * 4)) return 7;
              if (!len) continue;
              // the slots of every sequence's tiles: distinct, in order, inside the grid
              std::vector<char> taken(p.own_slots, 0);
              int r0 = 0;
              for (int s = 0; s < seqs; s++) {
                const int n = !ragged ? 1 : s + 1 < seqs ? (s * 7) % 4 : r - r0;
                const int r1 = r0 + n < r ? r0 + n : r;
                const int tc = p.own_cols, tiles = (int)at_ceil((int64_t)(r1 - r0) * g, tc);
                const int64_t first = ragged ? (int64_t)r0 * g / tc + s : (int64_t)s * at_ceil(g, tc);
                for (int t = 0; t < tiles; t++)
                  if (first + t >= p.own_slots || taken[first + t]++) return 8;
                r0 = r1;
              }
            }
  puts("ok");
  return 0;
}
"""


def test_page_lookup_and_plans(tmp_path):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not installed")
    src, exe = tmp_path / "t.hip", tmp_path / "t"
    src.write_text(PROGRAM)
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O1", "-std=c++17", "-I", os.path.join(ROOT, "webgpu-voxtral_amd", "csrc"), "-o",
                    str(exe), str(src)], check=True, capture_output=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout == "ok\n", out.returncode
