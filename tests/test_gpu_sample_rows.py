"""sample_rows on the GPU against 64-bit arithmetic: the same tokens and
numbers of kept entries wherever no cut or draw lies within 1e-9 of another
choice (weights are good to about 1e-11, sums exact)."""
import math

import pytest
import torch

import voxtral_amd as V
from batch_f64 import TYPES, sample

pytestmark = pytest.mark.gpu
DEV = "cuda"
EDGE = 1e-9


def check(logits, u, temperature, top_k, top_p, min_p, most_edges=0.02):
    """Settings are numbers or lists of one for each row."""
    rows = logits.shape[0]

    def full(v):
        return list(v) if isinstance(v, (list, tuple)) else [v] * rows

    def given(v, dtype):
        return torch.tensor(v, dtype=dtype, device=DEV) if isinstance(v, (list, tuple)) else v

    token, kept, prob = V.sample_rows(logits, torch.tensor(u, dtype=torch.float64, device=DEV), given(temperature, torch.float32),
                                      given(top_k, torch.int32), given(top_p, torch.float32), given(min_p, torch.float32))
    x, edges = logits.cpu(), 0
    t, k, p, m = (torch.tensor(full(v), dtype=torch.float32).tolist() for v in (temperature, top_k, top_p, min_p))
    for r in range(rows):
        want = sample(x[r], u[r], t[r], int(k[r]), p[r], m[r])
        if want[3] < EDGE:
            edges += 1
            continue
        assert (int(token[r]), int(kept[r])) == want[:2], (r, t[r], k[r], p[r], m[r])
        # weights to 1e-11, one rounding to f32
        assert abs(float(prob[r]) - want[2]) <= want[2] * (2.0 ** -24 + 1e-9) + 1e-30
    assert edges <= max(1, most_edges * rows)
    return token, kept, prob


def uniforms(n, seed):
    return torch.rand(n, generator=torch.Generator().manual_seed(seed), dtype=torch.float64).tolist()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n", [1, 2, 7, 64, 1000, 4097, 8320, 50001, 131072])
def test_settings(dtype, n):
    rows = 12
    g = torch.Generator().manual_seed(n)
    x = (torch.randn(rows, n, generator=g) * 3).to(TYPES[dtype]).to(DEV)
    u = uniforms(rows, n + 1)
    check(x, u, 1.0, 0, 1.0, 0.0)
    check(x, u, 0.7, 50, 0.9, 0.05)
    check(x, u, [0.0, 0.3, 1.0, 1.7] * 3, [0, 1, 40, n, 5000, 0] * 2, [1.0, 0.9, 0.5, 0.999] * 3, [0.0, 0.0, 0.2, 1e-4] * 3)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_flat_rows_and_ties(dtype):
    """Rows whose cuts lie among tens of thousands of entries, all equal ones,
    few distinct values, and one value far above."""
    n, g = 131072, torch.Generator().manual_seed(2)
    x = torch.zeros(6, n)
    x[0] = torch.randn(n, generator=g) * 0.01
    x[2] = torch.randint(0, 3, (n,), generator=g).float()
    x[3] = torch.randint(0, 40, (n,), generator=g).float() * 0.25
    x[4, 77] = 5.0
    x[5] = torch.randn(n, generator=g).abs()
    x = x.to(TYPES[dtype]).to(DEV)
    for seed, (k, p, m) in enumerate([(0, 1.0, 0.0), (0, 0.9, 0.0), (60000, 0.5, 0.0), (0, 1.0, 0.3), (70001, 0.97, 0.1), (6000, 1.0, 0.0)]):
        check(x, uniforms(6, seed), 1.0, k, p, m, most_edges=0.5)
    check(x, [0.0] * 6, 1e-6, 0, 0.5, 0.0, most_edges=0.5)
    check(x, [1 - 2.0 ** -53] * 6, 30.0, 0, 1.0, 0.0, most_edges=0.5)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_many_long_rows(dtype):
    """Rows enough to keep the GPU busy with a block each: ordinary, flat, few
    distinct values, and one value more than 65536 times."""
    n, rows, g = 70001, 130, torch.Generator().manual_seed(7)
    x = torch.randn(rows, n, generator=g) * 2.5
    x[1::5] *= 0.004
    x[2::5] = torch.randint(0, 5, (26, n), generator=g).float() * 0.5
    x[3::5, 1000:] = -1.25
    x[4::5, 7] = 14.0
    x[0, 50000:], x[5] = -math.inf, math.nan
    x[10, ::2] = 0.0
    x[10, 1::2] = -0.0
    x = x.to(TYPES[dtype]).to(DEV)
    r = torch.rand(4, rows, generator=g)
    t = torch.where(r[0] < 0.15, 0.0, 0.3 + r[0]).tolist()
    k = torch.where(r[1] < 0.4, 0.0, r[1] * torch.tensor([60.0, 70000.0]).repeat(65)).int().tolist()
    p = torch.where(r[2] < 0.3, 1.0, 0.3 + 0.699 * r[2]).tolist()
    m = torch.where(r[3] < 0.5, 0.0, 0.3 * r[3]).tolist()
    check(x, uniforms(rows, 8), t, k, p, m, most_edges=0.1)
    check(x[:, 1:], uniforms(rows, 9), 0.9, 0, 0.95, 0.0, most_edges=0.1)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_entries_that_are_not_finite(dtype):
    x = torch.randn(9, 300, generator=torch.Generator().manual_seed(3)) * 2
    x[0] = -math.inf
    x[1] = math.nan
    x[2, ::2], x[2, 1::4] = math.nan, -math.inf
    x[3, 17] = math.inf
    x[4, 100:200:10] = math.inf
    x[5] = math.inf
    x[6, 1:] = -math.inf
    x[7, :299] = math.nan
    x[8, 5], x[8, 6] = math.nan, -math.nan
    x = x.to(TYPES[dtype]).to(DEV)
    for k, p, m in ((0, 1.0, 0.0), (3, 0.9, 0.0), (0, 0.5, 0.4)):
        for u in (0.0, 0.31, 0.999):
            check(x, [u] * 9, 1.0, k, p, m, most_edges=1.0)
    token, kept, prob = check(x, [0.5] * 9, 0.0, 0, 1.0, 0.0)
    assert token.tolist()[:2] == [-1, -1] and kept.tolist()[:2] == [0, 0] and prob.tolist()[:2] == [0.0, 0.0]
    assert token.tolist()[3:8] == [17, 100, 0, 0, 299]


def test_zeros_of_both_signs_are_equal_and_extremes():
    x = torch.zeros(4, 50)
    x[0, ::2] = -0.0
    x[1] = -3.4e38
    x[1, 9] = 3.4e38
    x[2] = torch.arange(50) * 1e-44
    x[3] = 3.4e38
    x = x.to(DEV)
    token, _, _ = check(x, [0.0, 0.7, 0.3, 0.99], 1.0, 0, 1.0, 0.0, most_edges=1.0)
    assert token.tolist()[:2] == [0, 9]
    check(x, [0.5] * 4, [1e-40, 1e30, 1.0, 1e38], [7, 0, 3, 5], 1.0, 0.0, most_edges=1.0)
    token, _, _ = V.sample_rows(x, torch.tensor([math.nan, 2.0, -1.0, 0.5], dtype=torch.float64, device=DEV),
                                top_p=torch.tensor([-1.0, 2.0, 0.0, math.nan], device=DEV),
                                top_k=torch.tensor([-4, 1 << 30, 0, 0], dtype=torch.int32, device=DEV))
    assert all(0 <= t < 50 for t in token.tolist())


def test_alignment_strides_and_outputs():
    """Rows that start at any element, rows inside wider ones, given outputs."""
    g = torch.Generator().manual_seed(4)
    for dtype in TYPES.values():
        wide = (torch.randn(5, 1013, generator=g) * 3).to(dtype).to(DEV)
        for off in (0, 1, 3, 7):
            check(wide[:, off:off + 1001], uniforms(5, off), 0.9, 0, 0.95, 0.0)
    x, u = wide.float(), torch.tensor(uniforms(5, 9), dtype=torch.float64, device=DEV)
    out = tuple(torch.zeros(8, dtype=t, device=DEV)[3:] for t in (torch.int32, torch.int32, torch.float32))
    got = V.sample_rows(x, u, out=out)
    assert all(a is b for a, b in zip(got, out))
    assert all(torch.equal(a, b) for a, b in zip(V.sample_rows(x, u), out))


def test_frequencies():
    """20000 draws of one row follow the kept weights: each token's count is
    within 5 standard deviations."""
    x = torch.randn(1, 40, generator=torch.Generator().manual_seed(5)).to(DEV).expand(20000, 40)
    u = torch.rand(20000, generator=torch.Generator().manual_seed(6), dtype=torch.float64).to(DEV)
    token, kept, _ = V.sample_rows(x, u, temperature=0.8, top_p=0.9)
    n = int(kept[0])
    p = torch.softmax(x[0].double() / 0.8, 0).cpu()
    top = p.argsort(descending=True)[:n]
    p = p[top] / p[top].sum()
    count = torch.bincount(token.cpu().long(), minlength=40)
    assert int(count.sum()) == 20000 == int(count[top].sum())
    assert ((count[top].double() - 20000 * p).abs() <= 5 * (20000 * p * (1 - p)).sqrt() + 1).all()


def test_graph_and_streams():
    x, u = torch.randn(3, 9001, device=DEV), torch.rand(3, device=DEV, dtype=torch.float64)
    side = torch.cuda.Stream()
    out = V.sample_rows(x, u, top_p=0.9)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        V.sample_rows(x, u, top_p=0.9, out=out)
    for i in range(4):
        x.normal_()
        u.uniform_()
        graph.replay()
        torch.cuda.synchronize()
        want = V.sample_rows(x, u, top_p=0.9)
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i


def test_refusals():
    x, u = torch.randn(3, 50, device=DEV), torch.rand(3, device=DEV, dtype=torch.float64)
    for err, match, call in (
            (TypeError, "torch tensor", lambda: V.sample_rows([1.0], u)),
            (ValueError, "on cpu", lambda: V.sample_rows(x.cpu(), u)),
            (ValueError, "2 dimensions|dimensions, not 2", lambda: V.sample_rows(x[0], u)),
            (TypeError, "float64", lambda: V.sample_rows(x, u.float())),
            (TypeError, "float32, float16", lambda: V.sample_rows(x.double(), u)),
            (ValueError, "elements, not 3", lambda: V.sample_rows(x, u[:2])),
            (ValueError, "not contiguous", lambda: V.sample_rows(x.t()[:3], u)),
            (TypeError, "int32", lambda: V.sample_rows(x, u, top_k=u)),
            (V.VoxtralError, "temperature -1", lambda: V.sample_rows(x, u, temperature=-1.0)),
            (V.VoxtralError, "top_p 0", lambda: V.sample_rows(x, u, top_p=0.0)),
            (V.VoxtralError, "min_p 1.5", lambda: V.sample_rows(x, u, min_p=1.5)),
            (V.VoxtralError, "top_k -1", lambda: V.sample_rows(x, u, top_k=-1)),
            (V.VoxtralError, "0 logits", lambda: V.sample_rows(x[:, :0], u)),
            (V.VoxtralError, "more than 1048576", lambda: V.sample_rows(torch.zeros(1, 1 << 20, device=DEV).expand(3, -1).repeat(1, 2), u))):
        with pytest.raises(err, match=match):
            call()
    assert V.sample_rows(x[:0], u[:0])[0].shape == (0,)
