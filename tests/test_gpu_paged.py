"""The paged cache's append and the shared-prefix attention on the GPU against
64-bit arithmetic."""
import math

import pytest
import torch

import voxtral_amd as V
from batch_f64 import PAIRS, TYPES, attend, half_step, turn, turn_bound

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def pools(pages, hkv, page, hd, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(pages, hkv, page, hd, generator=g).to(dtype).to(DEV) for _ in range(2)]


# ----------------------------------------------------------------- append
@pytest.mark.parametrize("rows,cache", PAIRS)
@pytest.mark.parametrize("heads,hkv,hd,page,rotary,interleaved", [(32, 8, 128, 16, 128, True), (5, 1, 64, 64, 64, False),
                                                                  (6, 3, 128, 32, 48, True), (4, 2, 64, 16, 16, False),
                                                                  (2, 2, 128, 256, 0, True)])
def test_append(rows, cache, heads, hkv, hd, page, rotary, interleaved):
    torch.manual_seed(1)
    n, seqs, width, base, theta = 37, 5, 3, 200000, 1e6
    kp, vp = pools(seqs * width, hkv, page, hd, TYPES[cache])
    k0, v0 = kp.cpu(), vp.cpu()
    qkv = torch.randn(n, heads + 2 * hkv, hd, device=DEV).to(TYPES[rows])
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + hkv], qkv[:, heads + hkv:]
    table = torch.randperm(seqs * width).to(torch.int32).view(seqs, width).to(DEV)
    slots = torch.randperm(seqs * width * page)[:n]
    seq, slot = slots // (width * page), slots % (width * page)
    pos = slot + base
    got = V.PagedKV(kp, vp).append(k, v, ints(pos.tolist()), table, seq=ints(seq.tolist()), base=base, q=q, theta=theta,
                                   rotary_dim=rotary, interleaved=interleaved)
    kw, vw, wrote = k0.double(), v0.double(), torch.zeros(k0.shape, dtype=torch.bool)
    tol = torch.zeros(k0.shape, dtype=torch.float64)
    kd = k.cpu().double()
    kt = turn(kd, pos, theta, rotary, interleaved)
    kb = turn_bound(kd, kt, TYPES[cache], rotary, interleaved)
    for t in range(n):
        p, o = int(table[seq[t], slot[t] // page]), int(slot[t] % page)
        kw[p, :, o], vw[p, :, o], tol[p, :, o], wrote[p, :, o] = kt[t], v[t].cpu().to(TYPES[cache]).double(), kb[t], True
    assert ((kp.cpu().double() - kw).abs() <= tol).all()
    assert torch.equal(kp.cpu()[~wrote], k0[~wrote])
    assert torch.equal(vp.cpu().double(), vw)
    qd = q.cpu().double()
    qt = turn(qd, pos, theta, rotary, interleaved)
    assert ((got.cpu().double() - qt).abs() <= turn_bound(qd, qt, TYPES[rows], rotary, interleaved)).all()


def test_append_skips_what_has_no_place_and_turns_in_place():
    page, width, hkv, hd = 16, 2, 2, 64
    kp, vp = pools(4, hkv, page, hd, torch.float16)
    k0, v0 = kp.clone(), vp.clone()
    table = ints([[2, 0], [1, 99], [-1, 3]])
    #       fine   seq<0 seq big  pos<0  before base  past table  page 99  page -1  fine
    seq = [0, -1, 3, 1, 0, 0, 1, 2, 2]
    pos = [10 + 5, 10, 12, -3, 9, 10 + 32, 10 + 16, 10 + 3, 10 + 31]
    n = len(seq)
    k, v, q = (torch.randn(n, h, hd, device=DEV).half() for h in (hkv, hkv, 3))
    q0 = q.clone()
    kv = V.PagedKV(kp, vp)
    out = kv.append(k, v, ints(pos), table, seq=ints(seq), base=10, q=q, q_out=q, interleaved=False)
    assert out.data_ptr() == q.data_ptr()
    full = kv.append(k, v, ints(pos), table, seq=ints(seq), base=10, q=q0)
    assert full.shape == q0.shape and not full[1:8].any()
    for t in range(1, 8):
        assert torch.equal(q[t], q0[t])
    assert not torch.equal(q[0], q0[0]) and not torch.equal(q[8], q0[8])
    vw = v0.clone()
    vw[2, :, 5], vw[3, :, 15] = v[0], v[8]
    assert torch.equal(vp, vw)
    kw = kp.clone()
    kw[2, :, 5], kw[3, :, 15] = k0[2, :, 5], k0[3, :, 15]
    assert torch.equal(kw, k0)


def test_append_far_positions_and_large_pools():
    """Positions where an f32 angle is off by whole radians, and a page whose
    offset passes 2^32 elements."""
    hkv, hd, page = 8, 128, 4096
    pages = (1 << 32) // (hkv * hd * page) + 3
    kp = torch.empty(pages, hkv, page, hd, device=DEV, dtype=torch.float16)
    vp = torch.empty_like(kp)
    kp[-1].zero_()
    vp[-1].zero_()
    pos = torch.tensor([2000000000, 2000000001])
    k, v = (torch.randn(2, hkv, hd, device=DEV).half() for _ in range(2))
    base = 2000000000 - 4094
    V.PagedKV(kp, vp).append(k, v, ints(pos.tolist()), ints([[pages - 1]]), seq=ints([0, 0]), base=base)
    at = (pos - base).tolist()
    kd = k.cpu().double()
    kt = turn(kd, pos, 1e6, hd, True)
    tol = turn_bound(kd, kt, torch.float16, hd, True)
    for t in range(2):
        assert ((kp[-1, :, at[t]].cpu().double() - kt[t]).abs() <= tol[t]).all()
        assert torch.equal(vp[-1, :, at[t]], v[t])


# ----------------------------------------------------------------- attend
def check(q, kp, vp, table, lens, row_start=None, prefix_pages=None, prefix_len=0, max_len=None, scale=None, out=None, **kw):
    kv = V.PagedKV(kp, vp)
    lse = torch.full(q.shape[:2], 7.0, device=DEV)
    got = kv.attend(q, lens, table, row_start=row_start, prefix_pages=prefix_pages, prefix_len=prefix_len, max_len=max_len,
                    scale=scale, lse=lse, out=out, **kw)
    starts = list(range(len(lens) + 1)) if row_start is None else row_start.tolist()
    want, wlse, bound = attend(q.cpu(), kp.cpu(), vp.cpu(), table.cpu(), lens.cpu(), starts,
                               [] if prefix_pages is None else prefix_pages.cpu(), prefix_len,
                               table.shape[1] * kp.shape[2] if max_len is None else max_len, scale)
    n = starts[-1]
    off = (got.cpu().double() - want).abs()[:n]
    assert torch.isfinite(got[:n]).all()
    assert (off <= bound[:n]).all(), f"off by {float((off / bound[:n].clamp(min=1e-300)).max()):.2f} of the bound"
    empty = wlse[:n] == -math.inf
    assert torch.equal(lse.cpu()[:n] == -math.inf, empty)
    d = (lse.cpu().double()[:n] - wlse[:n]).abs()[~empty]
    # the score's own bound, as a part of out's: max|v| of a normal sample is over 1/2
    assert not len(d) or (d <= 4 * bound[:n].amax(2)[~empty] + 1e-5).all()
    assert (lse.cpu()[n:] == 7.0).all()
    return got


SHAPES = [
    # heads, kv heads, hd, page, prefix, own lengths, rows of each sequence (None: one)
    (32, 8, 128, 16, 100, [1, 17, 40, 33], None),
    (32, 8, 128, 64, 0, [1, 2, 300], None),
    (8, 8, 64, 32, 31, [0, 64, 5], None),
    (5, 1, 128, 16, 1, [16, 0], None),
    (40, 2, 64, 128, 700, [129, 1000], None),
    (4, 4, 128, 16, 33, [0, 0], None),
    (1, 1, 64, 16, 0, [1], None),
    (32, 8, 128, 16, 70, [5, 40, 3, 90], [5, 7, 1, 30]),
    (7, 1, 64, 32, 0, [33, 4, 9], [33, 6, 0]),
    (16, 16, 128, 64, 129, [200, 8, 1], [19, 2, 1]),
]


@pytest.mark.parametrize("rows,cache", PAIRS)
@pytest.mark.parametrize("heads,hkv,hd,page,prefix,lens,counts", SHAPES)
def test_attend(rows, cache, heads, hkv, hd, page, prefix, lens, counts):
    torch.manual_seed(3)
    width = max(1, -(-max(lens) // page))
    pre = -(-prefix // page)
    total = len(lens) * width + pre
    kp, vp = pools(total, hkv, page, hd, TYPES[cache], 4)
    order = torch.randperm(total).to(torch.int32).to(DEV)
    counts_ = counts or [1] * len(lens)
    start = [sum(counts_[:i]) for i in range(len(lens) + 1)]
    q = torch.randn(start[-1], heads, hd, device=DEV).to(TYPES[rows]) * 2
    check(q, kp, vp, order[:len(lens) * width].view(len(lens), width), ints(lens), ints(start) if counts else None,
          order[len(lens) * width:], prefix)


@pytest.mark.parametrize("rows,cache", PAIRS)
def test_attend_many_sequences_and_long_contexts(rows, cache):
    """More sequences than a wave searches at once, uneven rows, and contexts
    of several splits with a bound on lengths that the longest passes."""
    torch.manual_seed(5)
    n, hkv, hd, page = 150, 2, 64, 16
    counts = [int(x) for x in torch.randint(0, 4, (n,))]
    start = [sum(counts[:i]) for i in range(n + 1)]
    lens = [int(x) for x in torch.randint(0, 60, (n,))]
    width = 4
    kp, vp = pools(n * width + 2, hkv, page, hd, TYPES[cache], 6)
    table = torch.arange(n * width, dtype=torch.int32, device=DEV).view(n, width)
    q = torch.randn(start[-1], 6, hd, device=DEV).to(TYPES[rows])
    check(q, kp, vp, table, ints(lens), ints(start), ints([n * width + 1, n * width]), 21)
    lens, width = [3000, 1, 2047, 700], 188
    kp, vp = pools(4 * width, 1, page, hd, TYPES[cache], 7)
    table = torch.randperm(4 * width).to(torch.int32).view(4, width).to(DEV)
    q = torch.randn(4, 4, hd, device=DEV).to(TYPES[rows])
    check(q, kp, vp, table, ints(lens), max_len=2900, scale=0.3)
    check(q, kp, vp, table, ints(lens), prefix_pages=table[0], prefix_len=3000, max_len=17)


@pytest.mark.parametrize("rows,cache", PAIRS)
def test_attend_shared_prefix_in_wide_blocks(rows, cache):
    """More columns than a narrow block takes, over a prefix of several splits
    that ends inside a page and a step, next to own keys of several splits."""
    torch.manual_seed(18)
    n, hkv, hd, page, prefix = 37, 2, 128, 16, 777
    lens = [int(x) for x in torch.randint(0, 500, (n,))]
    lens[3], lens[9] = 0, 512
    width, pre = 32, -(-prefix // page)
    kp, vp = pools(n * width + pre, hkv, page, hd, TYPES[cache], 19)
    order = torch.randperm(n * width + pre).to(torch.int32).to(DEV)
    q = torch.randn(n, 8, hd, device=DEV).to(TYPES[rows]) * 1.5
    kp[order[n * width + pre - 1].item(), :, prefix % page:] = math.nan
    vp[order[n * width + pre - 1].item(), :, prefix % page:] = math.nan
    table = order[:n * width].view(n, width)
    bad = order[n * width:].clone()
    check(q, kp, vp, table, ints(lens), prefix_pages=bad, prefix_len=prefix)
    bad[7] = -1  # a hole of 16 keys
    bad[8] = 1 << 20
    check(q, kp, vp, table, ints(lens), prefix_pages=bad, prefix_len=prefix)


@pytest.mark.parametrize("rows,cache", PAIRS)
def test_attend_leaves_what_is_not_its_own(rows, cache):
    """Rows behind the last sequence stay as they were; NaN and infinities in
    slots that no row sees, in pages of nobody and in padding rows change
    nothing; a value that only later rows see reaches only them."""
    torch.manual_seed(8)
    hkv, hd, page, heads = 2, 128, 16, 8
    lens, counts = [21, 0, 18], [3, 2, 4]
    start = [0, 3, 5, 9]
    kp, vp = pools(9, hkv, page, hd, TYPES[cache], 9)
    table = ints([[0, 1, 8], [2, 3, 8], [4, 5, 8]])
    for pool in (kp, vp):
        pool[8] = math.nan
        pool[7] = math.inf
        pool[1, :, 5:] = math.nan
        pool[2:4] = -math.inf
        pool[5, :, 2:] = math.nan
        pool[6, :, 13:] = math.nan
    q = torch.randn(12, heads, hd, device=DEV).to(TYPES[rows])
    q[9:] = math.nan
    out = torch.full_like(q, 3.0)
    clean = check(q, kp, vp, table, ints(lens), ints(start), ints([6]), 13, out=out)
    assert (out[9:] == 3.0).all()
    # a NaN in the newest value of sequence 2: its last row alone sees it
    vp[5, 1, 1, 3] = math.nan
    vp[4, 0, 15, 7] = math.inf  # slot 15: rows 6.. see it
    again = V.PagedKV(kp, vp).attend(q, ints(lens), table, row_start=ints(start), prefix_pages=ints([6]), prefix_len=13)
    bad = ~torch.isfinite(again[:9])
    want = torch.zeros_like(bad)
    want[8, 4:, 3] = True
    want[6:9, :4, 7] = True  # row 5 sees slots 0 .. 14
    assert torch.equal(bad, want)
    assert torch.equal(again[:9][~want], clean[:9][~want])
    # a query that is not finite spoils its own head alone
    vp[5, 1, 1, 3] = vp[4, 0, 15, 7] = 0.5
    clean = V.PagedKV(kp, vp).attend(q, ints(lens), table, row_start=ints(start), prefix_pages=ints([6]), prefix_len=13)
    q[4, 2, 9] = math.nan
    again = V.PagedKV(kp, vp).attend(q, ints(lens), table, row_start=ints(start), prefix_pages=ints([6]), prefix_len=13)
    want = torch.zeros_like(bad)
    want[4, 2] = True
    assert torch.equal(torch.isnan(again[:9]), want) and torch.equal(again[:9][~want], clean[:9][~want])


@pytest.mark.parametrize("rows,cache", PAIRS)
def test_attend_with_bad_ids_and_bounds(rows, cache):
    """Page ids outside the pool hide their keys; lengths are cut to the
    bound, negative ones are none; row starts are cut to the rows there are."""
    torch.manual_seed(10)
    hkv, hd, page = 2, 64, 16
    kp, vp = pools(6, hkv, page, hd, TYPES[cache], 11)
    q = torch.randn(4, 4, hd, device=DEV).to(TYPES[rows])
    table = ints([[0, -1, 2], [6, 1 << 30, -(1 << 31)], [3, 4, 5], [1, 1, 1]])
    check(q, kp, vp, table, ints([48, 48, 1 << 30, -5]), prefix_pages=ints([77, 2]), prefix_len=20)
    check(q, kp, vp, table, ints([40, 17, -(1 << 31), (1 << 31) - 1]), max_len=33)
    kv = V.PagedKV(kp, vp)
    out = torch.full_like(q, 3.0)
    kv.attend(q, ints([5, 5, 5, 5]), table, row_start=ints([0, 1, 2, 3, 4000]), out=out)
    kv.attend(q, ints([5, 5, 5, 5]), table, row_start=ints([-9, -2, 7, 2, 1]), out=out)
    torch.cuda.synchronize()


def test_attend_strides_and_offsets_past_32_bits():
    """Token-major pools with gaps, queries inside a wider row, and pages whose
    offsets pass 2^32 elements."""
    torch.manual_seed(12)
    hkv, hd, page, heads = 8, 128, 256, 32
    wide = torch.randn(5, page, 2 * hkv + 1, hd, device=DEV).half()
    kp, vp = wide[:, :, :hkv].transpose(1, 2), wide[:, :, hkv:2 * hkv].transpose(1, 2)
    rows = torch.randn(3, heads + 4, hd + 8, device=DEV).half()
    q, out = rows[:, 2:heads + 2, :hd], torch.zeros(3, heads, 2 * hd, device=DEV, dtype=torch.float16)[:, :, hd:]
    check(q, kp, vp, ints([[4, 0], [1, 1], [2, 3]]), ints([300, 9, 256]), prefix_pages=ints([3]), prefix_len=77, out=out)
    pages = (1 << 32) // (hkv * hd * 4096) + 2
    big = torch.empty(2, pages, hkv, 4096, hd, device=DEV, dtype=torch.float16)
    big[:, -1].normal_()
    small = big[:, -1:].cpu()
    table = ints([[pages - 1]])
    lens = ints([4096])
    got = V.PagedKV(big[0], big[1]).attend(q[:1], lens, table)
    want, _, bound = attend(q[:1].cpu(), small[0], small[1], torch.tensor([[0]]), [4096], [0, 1], [], 0, 4096)
    assert ((got.cpu().double() - want).abs() <= bound).all()


def test_large_values_keep_f32_range():
    """f32 rows far outside f16's range on an f16 cache, f32 caches too."""
    torch.manual_seed(13)
    kp, vp = pools(2, 1, 16, 64, torch.float16)
    q = torch.randn(2, 4, 64, device=DEV)
    q[0] *= 3e7
    q[1] *= 1e-12
    check(q, kp, vp, ints([[0], [1]]), ints([16, 11]), scale=1e-6)
    check(q, kp.float() * 1e5, vp.float() * 1e8, ints([[0], [1]]), ints([16, 11]), scale=1e-11)


def test_a_run_of_steps_streams_and_graphs():
    """Append and attend as a batch uses them, eagerly, on another stream and
    replayed from a graph: the cache and outputs agree bit for bit."""
    torch.manual_seed(14)
    seqs, heads, hkv, hd, page, prefix, width, steps = 5, 8, 2, 128, 16, 50, 4, 24
    pre = ints([0, 1, 2, 3])
    table = (torch.arange(seqs * width, dtype=torch.int32) + 4).view(seqs, width).to(DEV)

    def fresh():
        kv = V.PagedKV(*pools(4 + seqs * width, hkv, page, hd, torch.float16, 15))
        lens = ints([3, 0, 9, 17, 1])
        pos = lens + prefix
        data = [torch.randn(seqs, heads + 2 * hkv, hd, generator=torch.Generator().manual_seed(i)).half().to(DEV) for i in range(steps)]
        return kv, lens, pos, data

    def step(kv, x, lens, pos, **kw):
        q = kv.append(x[:, heads:heads + hkv], x[:, heads + hkv:], pos, table, base=prefix, q=x[:, :heads], **kw)
        lens += 1
        pos += 1
        return kv.attend(q, lens, table, prefix_pages=pre, prefix_len=prefix, **kw)

    kv, lens, pos, data = fresh()
    want = [step(kv, x, lens, pos).clone() for x in data]
    check(data[0][:, :heads].contiguous(), kv.k_pages, kv.v_pages, table, lens, prefix_pages=pre, prefix_len=prefix)

    side = torch.cuda.Stream()
    kv2, lens, pos, data = fresh()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [step(kv2, x, lens, pos) for x in data]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(kv2.k_pages, kv.k_pages)

    kv3, lens, pos, data = fresh()
    x = torch.empty_like(data[0])
    with torch.cuda.stream(side):
        for i in range(2):  # warm the allocator, on values that are put back
            x.copy_(data[i])
            step(kv3, x, lens, pos)
        lens -= 2
        pos -= 2
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y = step(kv3, x, lens, pos)
    torch.cuda.synchronize()
    for i in range(steps):
        x.copy_(data[i])
        graph.replay()
        assert torch.equal(y, want[i]), i
        (torch.randn(100, 100, device=DEV) @ torch.randn(100, 100, device=DEV)).sum()
        torch.cuda.synchronize()
    assert torch.equal(kv3.k_pages, kv.k_pages) and torch.equal(kv3.v_pages, kv.v_pages)


def test_a_given_workspace_and_stream():
    torch.manual_seed(16)
    kp, vp = pools(240, 2, 16, 64, torch.bfloat16)
    kv = V.PagedKV(kp, vp)
    table = torch.arange(240, dtype=torch.int32, device=DEV).view(4, 60)
    q, lens = torch.randn(4, 4, 64, device=DEV).bfloat16(), ints([960, 3, 50, 400])
    want = kv.attend(q, lens, table)
    need = kv.attend_workspace(4, 4, 4, 60)
    assert need > 0
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    assert torch.equal(kv.attend(q, lens, table, workspace=ws), want)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = kv.attend(q, lens, table, stream=side)
    side.synchronize()
    assert torch.equal(got, want)
    with pytest.raises(V.VoxtralError, match="workspace of"):
        kv.attend(q, lens, table, workspace=ws[:need - 16])


def test_refusals_of_tensors():
    kp, vp = pools(4, 2, 16, 64, torch.float16)
    kv = V.PagedKV(kp, vp)
    table, lens, q = ints([[0, 1], [2, 3]]), ints([3, 4]), torch.zeros(2, 4, 64, device=DEV).half()
    k = torch.zeros(2, 2, 64, device=DEV).half()
    for err, match, call in (
            (ValueError, "differ", lambda: V.PagedKV(kp, vp[:2])),
            (ValueError, "on cpu", lambda: V.PagedKV(kp, vp.cpu())),
            (TypeError, "torch tensor", lambda: V.PagedKV(kp, [1])),
            (TypeError, "float32, float16 or bfloat16", lambda: V.PagedKV(kp.double(), vp.double())),
            (ValueError, "not contiguous", lambda: V.PagedKV(kp.transpose(2, 3), vp.transpose(2, 3))),
            (V.VoxtralError, "power of two", lambda: V.PagedKV(kp[:, :, :12], vp[:, :, :12]).attend(q, lens, table)),
            (V.VoxtralError, "head_dim 32", lambda: V.PagedKV(kp[..., :32], vp[..., :32]).attend(q[..., :32], lens, table)),
            (TypeError, "int32", lambda: kv.attend(q, lens.long(), table)),
            (TypeError, "int32", lambda: kv.attend(q, lens, table.long())),
            (ValueError, "2 elements, not 3", lambda: kv.attend(q, lens, table, row_start=lens)),
            (ValueError, "shape", lambda: kv.attend(q[..., :32], lens, table)),
            (V.VoxtralError, "3 heads for 2", lambda: kv.attend(q[:, :3], lens, table)),
            (V.VoxtralError, "rows of type 2", lambda: kv.attend(q.bfloat16(), lens, table)),
            (V.VoxtralError, "without row_start", lambda: kv.attend(q[:1], lens, table)),
            (V.VoxtralError, "max_len 33", lambda: kv.attend(q, lens, table, max_len=33)),
            (V.VoxtralError, "prefix_len 17", lambda: kv.attend(q, lens, table, prefix_pages=ints([1]), prefix_len=17)),
            (ValueError, "scale", lambda: kv.attend(q, lens, table, scale=0)),
            (V.VoxtralError, "scale", lambda: kv.attend(q, lens, table, scale=math.nan)),
            (ValueError, "gradient", lambda: kv.attend(q.clone().requires_grad_(), lens, table)),
            (V.VoxtralError, "multiples of 16", lambda: kv.attend(torch.zeros(2, 4, 65, device=DEV).half()[..., :64], lens, table)),
            (ValueError, "lse", lambda: kv.attend(q, lens, table, lse=torch.zeros(2, 4, device=DEV).half())),
            (ValueError, "out of range", lambda: kv.attend(q, lens, table, max_len=1 << 40)),
            (ValueError, "out of range", lambda: kv.append(k, k, lens, table, base=1 << 31)),
            (TypeError, "v is", lambda: kv.append(k, k.float(), lens, table)),
            (V.VoxtralError, "rotary_dim 24", lambda: kv.append(k, k, lens, table, rotary_dim=24)),
            (V.VoxtralError, "theta", lambda: kv.append(k, k, lens, table, theta=-1.0)),
            (V.VoxtralError, "without sequence numbers", lambda: kv.append(k, k, lens, table[:1])),
            (TypeError, "q is", lambda: kv.append(k, k, lens, table, q=q.float()))):
        with pytest.raises(err, match=match):
            call()


def test_nothing_to_do():
    kp, vp = pools(2, 2, 16, 64, torch.float16)
    k0 = kp.clone()
    kv = V.PagedKV(kp, vp)
    none = torch.zeros(0, 2, 64, device=DEV).half()
    kv.append(none, none, ints([]), ints([[0], [1]]), seq=ints([]))
    assert kv.attend(none, ints([]), torch.zeros(0, 3, dtype=torch.int32, device=DEV)).shape == none.shape
    k = torch.randn(2, 2, 64, device=DEV).half()
    kv.append(k, k, ints([0, 1]), torch.zeros(2, 0, dtype=torch.int32, device=DEV))
    assert torch.equal(kp, k0)
    q = torch.randn(2, 4, 64, device=DEV).half()
    lse = torch.zeros(2, 4, device=DEV)
    out = kv.attend(q, ints([4, 4]), torch.zeros(2, 0, dtype=torch.int32, device=DEV), lse=lse)
    assert not out.any() and (lse == -math.inf).all()


def test_results_do_not_change_from_call_to_call():
    torch.manual_seed(17)
    kp, vp = pools(200, 2, 16, 128, torch.float16)
    table = torch.randperm(200).to(torch.int32).view(4, 50).to(DEV)
    q, lens = torch.randn(4, 8, 128, device=DEV), ints([800, 13, 555, 320])
    outs = [V.PagedKV(kp, vp).attend(q, lens, table, prefix_pages=table[1], prefix_len=799) for _ in range(5)]
    assert all(torch.equal(o, outs[0]) for o in outs)
    assert half_step(torch.float16) == 2.0 ** -11
