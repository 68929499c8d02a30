"""The operators of a batched decode, as timed cases: appending rotated keys
and values to a paged cache, the attention of a batch that shares a long
prefix, and sampling rows of logits with temperature, top-k, top-p and min-p
from given uniforms.  Inputs are torch tensors on the GPU.  `run` computes a
case in its plain form (32-bit torch, 64 bits for angles and running masses)
or, where `own` is true, through voxtral_amd.  `exact` restates each operator
in 64 bits, sequence by sequence."""
import math
import os
import random
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
own = False  # set by the caller: True runs the framework's operators

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEV = "cuda"
THETA = 1e6


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one new token for each of a few utterances, the engine's own types (f32 rows, f16 cache): the smallest append
        _append("append_decode_8", 8, 1, 1, 4096, "f32", "f16", 64),
        # a decode step of a wide batch, sequences at far positions
        _append("append_decode_200", 200, 1, 1, 130000, "bf16", "bf16", 16, halves=True),
        # the prompts of a batch: ragged runs of tokens, queries, keys and values of every one rotated
        _append("append_prompts", 24, 40, 300, 2048, "f16", "f16", 64),
        # the first steps of a few short utterances: the smallest attention
        _attend("attend_small", 4, 100, 1, 40, "f16", "f16", 16),
        # an ordinary batch: one voice prompt, suffixes of text and frames
        _attend("attend_64", 64, 2050, 200, 900, "f16", "f16", 64),
        # the engine's default precision
        _attend("attend_f32", 24, 300, 1, 700, "f32", "f32", 32),
        # long own contexts next to a long prefix, f32 rows on an f16 cache: the largest call
        _attend("attend_long", 32, 8000, 4000, 16000, "f32", "f16", 128),
        # many texts after one prompt, each in one go: several query rows a sequence
        _attend("attend_prompts", 16, 1500, 0, 200, "bf16", "bf16", 16, rows_lo=20, rows_hi=90),
        # one semantic code: the smallest sampling call
        _sample("sample_1", 1, 8320, "f32"),
        # the semantic codes of a batch
        _sample("sample_64", 64, 8320, "f32"),
        # text logits of a few sequences
        _sample("sample_vocab_8", 8, 131072, "f32"),
        # text logits of a wide batch; 16 bits make long runs of equal values
        _sample("sample_vocab_256", 256, 131072, "bf16"),
    ]


def _append(name, seqs, lo, hi, far, rows, cache, page, heads=32, kv_heads=8, hd=128, halves=False):
    return {"name": name, "kind": "append", "seqs": seqs, "lo": lo, "hi": hi, "far": far, "rows": rows, "cache": cache,
            "page": page, "heads": heads, "kv_heads": kv_heads, "hd": hd, "halves": halves}


def _attend(name, seqs, prefix, lo, hi, rows, cache, page, heads=32, kv_heads=8, hd=128, rows_lo=1, rows_hi=1):
    # lo..hi: keys of its own that a sequence has before its query rows' own
    return {"name": name, "kind": "attend", "seqs": seqs, "prefix": prefix, "lo": lo, "hi": hi, "rows": rows, "cache": cache,
            "page": page, "heads": heads, "kv_heads": kv_heads, "hd": hd, "rows_lo": rows_lo, "rows_hi": rows_hi}


def _sample(name, rows, n, dtype):
    return {"name": name, "kind": "sample", "rows": rows, "n": n, "dtype": dtype}


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.499)))))))


def draw(rng):
    kind = rng.choice(("append", "attend", "attend", "sample"))
    pair = rng.choice((("f32", "f32"), ("f32", "f16"), ("f16", "f16"), ("bf16", "bf16")))
    heads, kv_heads = rng.choice(((32, 8), (32, 8), (16, 16), (40, 8), (8, 1), (28, 4)))
    page, hd = rng.choice((16, 32, 64, 128)), rng.choice((128, 128, 64))
    if kind == "append":
        seqs = _log(rng, 1, 256)
        hi = rng.choice((1, _log(rng, 1, max(1, 4000 // seqs))))
        c = _append("", seqs, min(hi, 1 + hi // 4), hi, _log(rng, 600, 200000), *pair, page, heads, kv_heads, hd, rng.random() < 0.5)
    elif kind == "attend":
        seqs = _log(rng, 1, 256)
        rows_hi = rng.choice((1, 1, 1, _log(rng, 2, 4 + 700 // seqs)))
        hi = _log(rng, 1, max(8, min(16000, 100000 // (seqs + rows_hi))))
        prefix = rng.choice((0, _log(rng, 1, 400), _log(rng, 100, 8000)))
        c = _attend("", seqs, prefix, hi // rng.choice((1, 2, 8)), hi, *pair, page, heads, kv_heads, hd, 1 + rows_hi // 4, rows_hi)
    else:
        n = _log(rng, 100, 131072)
        c = _sample("", _log(rng, 1, max(1, min(512, (256 << 17) // n // 2))), n, rng.choice(tuple(TYPES)))
    del c["name"]
    return c


# ----------------------------------------------------------------- inputs
def _spans(case, seed):
    """Of each sequence of an append or attend case: its first own position, by the seed, and its number of rows, by the case alone."""
    r, shape = random.Random(seed), random.Random(str(sorted((k, v) for k, v in case.items() if k != "name")))
    if case["kind"] == "append":
        n = [shape.randint(case["lo"], case["hi"]) for _ in range(case["seqs"])]
        return [r.randint(0, max(512, case["hi"]) - k) for k in n], n
    n = [shape.randint(case["rows_lo"], case["rows_hi"]) for _ in range(case["seqs"])]
    return [r.randint(case["lo"], case["hi"]) for _ in range(case["seqs"])], n


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case)
    if case["kind"] == "sample":
        return _prepare_sample(s, g)
    rows, cache = TYPES[case["rows"]], TYPES[case["cache"]]
    first, n = _spans(case, seed)
    hd, hkv, page = case["hd"], case["kv_heads"], case["page"]
    t = sum(n)
    s["seq"] = _ints([i for i, k in enumerate(n) for _ in range(k)])
    s["at"] = _ints([j for k in n for j in range(k)])
    s["row_start"] = _ints([sum(n[:i]) for i in range(len(n) + 1)])
    if case["kind"] == "append":
        # own positions start behind a prefix of `far` positions, less what the table holds
        longest = max(512, case["hi"])
        s["base"] = max(0, case["far"] - longest)
        s["pos"] = _ints([s["base"] + f + j for f, k in zip(first, n) for j in range(k)])
        # one product's output, as a program has it: queries, keys and values of a token side by side
        h = case["heads"] + 2 * hkv
        qkv = torch.randn(t, h, hd, device=DEV, generator=g).to(rows)
        s["q"], s["k"], s["v"] = qkv[:, :case["heads"]], qkv[:, case["heads"]:case["heads"] + hkv], qkv[:, case["heads"] + hkv:]
        s["q_out"] = torch.empty(t, case["heads"], hd, device=DEV, dtype=rows)
        extra = 0
    else:
        longest = case["hi"] + case["rows_hi"]
        s["lens"] = _ints([f + k for f, k in zip(first, n)])
        s["max_len"], s["max_rows"] = longest, case["rows_hi"]
        s["q"] = torch.randn(t, case["heads"], hd, device=DEV, generator=g).to(rows)
        s["out"] = torch.empty_like(s["q"])
        extra = -(-case["prefix"] // page)
    width = -(-longest // page)
    pages = len(n) * width + extra
    order = torch.randperm(pages, device=DEV, generator=g).to(torch.int32)
    s["table"] = order[:len(n) * width].view(len(n), width).contiguous()
    s["prefix_pages"] = order[len(n) * width:].contiguous()
    s["kp"] = torch.empty(pages, hkv, page, hd, device=DEV, dtype=cache)
    s["vp"] = torch.empty_like(s["kp"])
    if case["kind"] == "append":
        s["kp"].zero_()
        s["vp"].zero_()
    else:
        for x in (s["kp"], s["vp"]):  # some keys stand out, as they do in a trained model
            x.copy_(torch.randn(x.shape, device=DEV, generator=g, dtype=torch.float32 if cache == torch.float32 else torch.float16))
        s["kp"].mul_((0.7 + torch.rand(pages, 1, page, 1, device=DEV, generator=g)).to(cache))
    return s


def _prepare_sample(s, g):
    rows, n = s["rows"], s["n"]
    x = torch.randn(rows, n, device=DEV, generator=g) * 2.5
    top = torch.randint(0, n, (rows, 12), device=DEV, generator=g)
    s["logits"] = x.scatter_add_(1, top, 6 * torch.rand(rows, 12, device=DEV, generator=g)).to(TYPES[s["dtype"]])
    s["u"] = torch.rand(rows, device=DEV, generator=g, dtype=torch.float64)
    # settings differ from request to request: greedy ones and ones without a truncation among them
    r = torch.rand(4, rows, device=DEV, generator=g)
    s["temperature"] = torch.where(r[0] < 0.1, 0.0, 0.6 + 0.7 * r[0])
    s["top_k"] = torch.where(r[1] < 0.5, 0, 1 + (r[1] * 100).to(torch.int32)).to(torch.int32)
    s["top_p"] = torch.where(r[2] < 0.25, 1.0, 0.75 + 0.24 * r[2])
    s["min_p"] = torch.where(r[3] < 0.5, 0.0, 0.1 * r[3])
    return s


# -------------------------------------------------------------------- run
def run(s):
    if own:
        return _run_own(s)
    return {"append": _plain_append, "attend": _plain_attend, "sample": _plain_sample}[s["kind"]](s)


def _run_own(s):
    V = s.get("V")
    if V is None:  # a program imports the package and wraps its cache once
        path = os.path.join(ROOT, "webgpu-voxtral_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        import voxtral_amd as V
        s["V"] = V
        if s["kind"] != "sample":
            s["kv"] = V.PagedKV(s["kp"], s["vp"])
    if s["kind"] == "append":
        q = s["kv"].append(s["k"], s["v"], s["pos"], s["table"], seq=s["seq"], base=s["base"], q=s["q"], q_out=s["q_out"],
                           theta=THETA, interleaved=not s["halves"])
        return q, s["kp"], s["vp"]
    if s["kind"] == "attend":
        return s["kv"].attend(s["q"], s["lens"], s["table"], row_start=None if s["rows_hi"] == 1 else s["row_start"],
                              prefix_pages=s["prefix_pages"], prefix_len=s["prefix"], max_len=s["max_len"], out=s["out"])
    return V.sample_rows(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])


def _turn(x, pos, halves):
    """x [t][heads][hd] rotated, in 32 bits; the angles in 64."""
    hd = x.shape[2]
    f = THETA ** (-torch.arange(0, hd, 2, device=DEV, dtype=torch.float64) / hd)
    a = pos.double()[:, None] * f
    c, d = a.cos().float()[:, None], a.sin().float()[:, None]
    x = x.float()
    u, w = (x[..., :hd // 2], x[..., hd // 2:]) if halves else (x[..., 0::2], x[..., 1::2])
    y = (u * c - w * d, u * d + w * c)
    return torch.cat(y, 2) if halves else torch.stack(y, 3).reshape(x.shape)


def _plain_append(s):
    seq, slot = s["seq"].long(), s["pos"].long() - s["base"]
    page, off = s["table"][seq, slot // s["page"]].long(), slot % s["page"]
    s["kp"][page, :, off] = _turn(s["k"], s["pos"], s["halves"]).to(s["kp"].dtype)
    s["vp"][page, :, off] = s["v"].to(s["vp"].dtype)
    s["q_out"].copy_(_turn(s["q"], s["pos"], s["halves"]))
    return s["q_out"], s["kp"], s["vp"]


def _plain_attend(s):
    n, hkv, hd, page, m = s["seqs"], s["kv_heads"], s["hd"], s["page"], s["max_rows"]
    g, length, prefix = s["heads"] // hkv, s["max_len"], s["prefix"]
    at = torch.arange(length, device=DEV)
    pages = s["table"][:, at // page].long()

    def keys(pool):  # [n][hkv][length][hd]
        return pool[pages, :, (at % page).expand(n, length)].float().transpose(1, 2)

    def shared(pool):  # [hkv][prefix][hd]
        p = torch.arange(prefix, device=DEV)
        return pool[s["prefix_pages"][p // page].long(), :, p % page].float().transpose(0, 1)

    start = s["row_start"].long()
    count = (start[1:] - start[:-1])[:, None]
    j = torch.arange(m, device=DEV)
    rows = (start[:-1, None] + j).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][rows].float().view(n, m, hkv, g, hd).permute(0, 2, 3, 1, 4).reshape(n, hkv, g * m, hd) / math.sqrt(hd)
    seen = (s["lens"].long()[:, None] - (count - 1 - j)).clamp(min=0)  # [n][m]
    own_s = (q @ keys(s["kp"]).transpose(2, 3)).view(n, hkv, g, m, length)
    own_s = own_s.masked_fill(at >= seen[:, None, None, :, None], -math.inf).view(n, hkv, g * m, length)
    q = q.transpose(0, 1).reshape(hkv, n * g * m, hd)
    pre_s = (q @ shared(s["kp"]).transpose(1, 2)).view(hkv, n, g * m, prefix).transpose(0, 1)
    top = own_s.amax(3, keepdim=True)
    if prefix:
        top = torch.maximum(top, pre_s.amax(3, keepdim=True))
    top = top.masked_fill(top == -math.inf, 0.0)  # the padded rows of short sequences may see no key
    own_s, pre_s = (own_s - top).exp(), (pre_s - top).exp()
    total = own_s.sum(3, keepdim=True) + pre_s.sum(3, keepdim=True)
    o = own_s @ keys(s["vp"])
    o = o + (pre_s.transpose(0, 1).reshape(hkv, n * g * m, prefix) @ shared(s["vp"])).view(hkv, n, g * m, hd).transpose(0, 1)
    o = (o / total).view(n, hkv, g, m, hd).permute(0, 3, 1, 2, 4).reshape(n, m, s["heads"], hd)
    s["out"].copy_(o[s["seq"].long(), s["at"].long()])
    return s["out"]


def _plain_sample(s):
    x, order = s["logits"].float().sort(dim=1, descending=True, stable=True)
    t = s["temperature"].double()[:, None]
    rank = torch.arange(s["n"], device=DEV)
    w = ((x.double() - x[:, :1].double()) / t.clamp(min=1e-300)).exp()
    k = s["top_k"][:, None]
    kept = (k <= 0) | (rank < k)
    w = w * kept
    c = w.cumsum(1)
    p = s["top_p"].double()[:, None]
    kept &= (p >= 1) | (c - w < p * c[:, -1:])
    kept &= w >= s["min_p"].double()[:, None]
    kept &= t > 0
    kept[:, 0] = True
    mass = (w * kept).sum(1, keepdim=True)
    number = kept.sum(1)
    j = (kept & (c <= s["u"][:, None] * mass)).sum(1).minimum(number - 1)[:, None]
    return order.gather(1, j)[:, 0].to(torch.int32), number.to(torch.int32), (w.gather(1, j) / mass)[:, 0].float()


# ------------------------------------------------------------------- work
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def work(case):
    if case["kind"] == "sample":
        # a difference, a scaling, an exponential, a comparison and a sum for each logit
        return {"bytes": case["rows"] * (case["n"] * _SIZE[case["dtype"]] + 36), "flops": 5 * case["rows"] * case["n"]}
    first, n = _spans(case, 1)
    es, ec, hd = _SIZE[case["rows"]], _SIZE[case["cache"]], case["hd"]
    if case["kind"] == "append":
        t = sum(n)
        return {"bytes": t * hd * (2 * case["heads"] * es + 2 * case["kv_heads"] * (es + ec)) + 12 * t,
                "flops": 3 * t * hd * (case["heads"] + case["kv_heads"])}
    keys = case["prefix"] + sum(f + k for f, k in zip(first, n))
    pairs = sum(k * (case["prefix"] + f) + k * (k + 1) // 2 for f, k in zip(first, n))
    return {"bytes": 2 * keys * case["kv_heads"] * hd * ec + 2 * sum(n) * case["heads"] * hd * es,
            "flops": 4 * hd * case["heads"] * pairs}


# ------------------------------------------------------------------ exact
def exact(case, seed):
    return {"append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}[case["kind"]](prepare(case, seed))


def _exact_append(s):
    hd, half = s["hd"], s["hd"] // 2
    i = torch.arange(half, device=DEV, dtype=torch.float64)
    a = s["pos"].double()[:, None, None] * torch.exp(i * (-2 * math.log(THETA) / hd))
    u, w = (torch.arange(half), torch.arange(half) + half) if s["halves"] else (2 * torch.arange(half), 2 * torch.arange(half) + 1)

    def turn(x):
        x, y = x.double(), torch.empty(x.shape, dtype=torch.float64, device=DEV)
        y[..., u] = x[..., u] * a.cos() - x[..., w] * a.sin()
        y[..., w] = x[..., w] * a.cos() + x[..., u] * a.sin()
        return y

    kp, vp = s["kp"].double(), s["vp"].double()
    k, v = turn(s["k"]), s["v"].double()
    seq, slot = s["seq"].tolist(), (s["pos"] - s["base"]).tolist()
    table = s["table"].cpu()
    pages = torch.stack([table[b, x // s["page"]] for b, x in zip(seq, slot)]).long().to(DEV)
    offs = torch.tensor([x % s["page"] for x in slot], device=DEV)
    for h in range(s["kv_heads"]):
        kp[pages, h, offs] = k[:, h]
        vp[pages, h, offs] = v[:, h]
    return turn(s["q"]), kp, vp


def _exact_attend(s):
    hkv, hd, page = s["kv_heads"], s["hd"], s["page"]
    g = s["heads"] // hkv
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
    start, lens = s["row_start"].tolist(), s["lens"].tolist()

    def line(pool, ids, length):  # [length][hkv][hd] of the pages in order
        return pool[ids.long()].double().transpose(1, 2).reshape(-1, hkv, hd)[:length]

    for b in range(s["seqs"]):
        ids = s["table"][b, :-(-lens[b] // page)]
        k, v = (torch.cat([line(x, s["prefix_pages"], s["prefix"]), line(x, ids, lens[b])]) for x in (s["kp"], s["vp"]))
        n = start[b + 1] - start[b]
        q = s["q"][start[b]:start[b + 1]].double()
        last = s["prefix"] + lens[b] - (n - 1) + torch.arange(n, device=DEV)
        hidden = torch.arange(k.shape[0], device=DEV)[None, :] >= last[:, None]
        for h in range(hkv):
            x = torch.matmul(q[:, h * g:(h + 1) * g].reshape(n * g, hd), k[:, h].t().contiguous()) * hd ** -0.5
            x = x.view(n, g, -1).masked_fill(hidden[:, None], -math.inf)
            out[start[b]:start[b + 1], h * g:(h + 1) * g] = torch.matmul(torch.softmax(x, 2).view(n * g, -1), v[:, h].contiguous()).view(n, g, hd)
    return out


def _exact_sample(s):
    token, number, prob = [], [], []
    for b in range(s["rows"]):
        x, t, k = s["logits"][b].double(), float(s["temperature"][b]), int(s["top_k"][b])
        p, lo, u = float(s["top_p"][b]), float(s["min_p"][b]), float(s["u"][b])
        x, order = torch.sort(x, descending=True, stable=True)
        if t <= 0:
            x, order, t = x[:1], order[:1], 1.0
        x, order = (x[:k], order[:k]) if k > 0 else (x, order)
        w = torch.exp((x - x[0]) / t)
        if p < 1:
            before = torch.cumsum(w, 0) - w
            w = w[:max(1, int((before < p * w.sum()).sum()))]
        w = w[:max(1, int((w >= lo).sum()))]
        c = torch.cumsum(w, 0)
        j = min(int((c <= u * c[-1]).sum()), w.numel() - 1)
        token.append(int(order[j]))
        number.append(w.numel())
        prob.append(float(w[j] / c[-1]))
    return (torch.tensor(token, dtype=torch.int32), torch.tensor(number, dtype=torch.int32),
            torch.tensor(prob, dtype=torch.float64))
