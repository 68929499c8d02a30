"""The batch operators (paged append, shared-prefix attention, row sampling)
in 64 bits on the CPU, written out sequence by sequence, and the bounds that
the GPU tests hold results to."""
import math

import torch

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
PAIRS = [("f32", "f32"), ("f32", "f16"), ("f16", "f16"), ("bf16", "bf16")]
U32 = 2.0 ** -24  # half a step of f32


def half_step(t):
    return torch.finfo(t).eps / 2


def turn(x, pos, theta, rotary_dim, interleaved):
    """x [t][heads][hd] (float64) turned by pos [t]."""
    y = x.clone()
    half = rotary_dim // 2
    for i in range(half):
        a = pos.double() * theta ** (-2.0 * i / rotary_dim)
        c, s = a.cos()[:, None], a.sin()[:, None]
        u, w = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        y[:, :, u] = x[:, :, u] * c - x[:, :, w] * s
        y[:, :, w] = x[:, :, u] * s + x[:, :, w] * c
    return y


def turn_bound(x, y, dtype, rotary_dim, interleaved):
    """How far a turned element may be from y: the angle's revolution is
    rounded to f32 (2^-26 of one, 9.4e-8 radians), sine and cosine are good to
    2 ulp (1.2e-7), two products and a sum round (1.8e-7 of |u| + |w|): 4e-7
    of |u| + |w| in all, and the result is rounded to its type."""
    a, b = x.abs(), x.abs()
    half = rotary_dim // 2
    for i in range(half):
        u, w = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        b[:, :, u] = a[:, :, u] + a[:, :, w]
        b[:, :, w] = b[:, :, u]
    return 4e-7 * b + (y.abs() + 4e-7 * b) * half_step(dtype) + torch.finfo(dtype).tiny * half_step(dtype)


def line(pool, pages, n):
    """The first n slots of a page list: [n][kv heads][hd] in float64, and
    which of them have a page."""
    n_pages, hkv, size, hd = pool.shape
    out = torch.zeros(n, hkv, hd, dtype=torch.float64)
    there = torch.zeros(n, dtype=torch.bool)
    for i in range(n):
        p = int(pages[i // size]) if i // size < len(pages) else -1
        if 0 <= p < n_pages:
            out[i] = pool[p, :, i % size].double()
            there[i] = True
    return out, there


def attend(q, kp, vp, table, lens, row_start, prefix_pages, prefix_len, max_len, scale=None):
    """(out, lse, bound) of every row up to row_start[-1], in float64.  All
    arguments on the CPU.  bound: how far `out` may be off.

    With S the largest sum |q_i k_i| scale of a row and s its largest |score|,
    an f32 score is off by at most d = U32 (2 hd S + 4 s + 16) (its products
    and sums, the factor, the exponent's argument and exp2); a split f16
    product adds 2^-21 S.  Weights off by a factor 1 + d move out by 2 d
    max|v|; the sums over keys add U32 keys max|v| at most; weights rounded to
    16 bits u max|v|; the result's own rounding u |out|."""
    t, heads, hd = q.shape
    hkv = kp.shape[1]
    g = heads // hkv
    scale = hd ** -0.5 if scale is None else scale
    u_out, split = half_step(q.dtype), q.dtype == torch.float32 and kp.dtype != torch.float32
    u_w = 2.0 ** -21 if split else (half_step(kp.dtype) if kp.dtype != torch.float32 else 0.0)
    out, lse, bound = torch.zeros(t, heads, hd, dtype=torch.float64), torch.full((t, heads), -math.inf, dtype=torch.float64), torch.zeros(t, heads, hd, dtype=torch.float64)
    pre = [line(x, prefix_pages, prefix_len) for x in (kp, vp)] if prefix_len else None
    for b in range(len(lens)):
        r0, r1 = int(row_start[b]), int(row_start[b + 1])
        for r in range(r0, r1):
            n = max(0, min(int(lens[b]) - (r1 - 1 - r), max_len))
            k, there = line(kp, table[b], n)
            v, _ = line(vp, table[b], n)
            if pre:
                k, v, there = torch.cat([pre[0][0], k]), torch.cat([pre[1][0], v]), torch.cat([pre[0][1], there])
            k, v = k[there], v[there]
            if not len(k):
                continue
            for h in range(heads):
                qh = q[r, h].double()
                s = k[:, h // g] @ qh * scale
                lse[r, h] = torch.logsumexp(s, 0)
                p = torch.softmax(s, 0)
                vh = v[:, h // g]
                out[r, h] = p @ vh
                big = float((k[:, h // g].abs() @ qh.abs()).max()) * abs(scale)
                d = U32 * (2 * hd * big + 4 * float(s.abs().max()) + 16) + (2.0 ** -21 * big if split else 0)
                vmax = float(vh.abs().max())
                bound[r, h] = vmax * (2 * d + U32 * len(k) + u_w) + u_out * out[r, h].abs() + torch.finfo(q.dtype).tiny
    return out, lse, bound


def sample(x, u, temperature, top_k, top_p, min_p):
    """(token, kept, prob, edge) of one row x (1-D); edge: how near, relative
    to the kept sum, a cut or the draw comes to another choice."""
    x = x.double()
    ok = torch.isfinite(x) | (x == math.inf)
    ids = torch.nonzero(ok)[:, 0]
    if not len(ids):
        return -1, 0, 0.0, 1.0
    y, order = torch.sort(x[ids], descending=True, stable=True)
    order = ids[order]
    if not temperature > 0:
        return int(order[0]), 1, 1.0, 1.0
    if y[0] == math.inf:
        w = (y == math.inf).double()
    else:
        w = torch.exp((y - y[0]) / temperature)
    edge = 1.0
    if top_k > 0:
        w, order = w[:top_k], order[:top_k]
    n = len(w)
    if top_p < 1:
        c = torch.cumsum(w, 0)
        goal = max(top_p, 0.0) * c[-1]
        n = max(1, int(((c - w) < goal).sum()))
        edge = min(edge, float((c - goal).abs().min() / c[-1]))
    if min_p > 0:
        n = min(n, max(1, int((w >= min(min_p, 1.0)).sum())))
        d = (w - min_p).abs()
        if min_p < 1 and w[0] != w[-1]:
            edge = min(edge, float(d[w != 1].min()) if bool((w != 1).any()) else 1.0)
    w = w[:n]
    c = torch.cumsum(w, 0)
    j = min(int((c <= u * c[-1]).sum()), n - 1)
    if n > 1:  # behind the last entry there is no other choice
        edge = min(edge, float((c[:-1] - u * c[-1]).abs().min() / c[-1]))
    return int(order[j]), n, float(w[j] / c[-1]), edge
