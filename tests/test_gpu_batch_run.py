"""The batch operators together, as a decode loop uses them: append, attend, a
projection, sample, the drawn token's row appended next."""
import threading

import pytest
import torch

import voxtral_amd as V
from batch_f64 import attend, sample, turn

pytestmark = pytest.mark.gpu
DEV = "cuda"
SEQS, HEADS, HKV, HD, PAGE, PREFIX, WIDTH, VOCAB, STEPS = 6, 8, 2, 64, 16, 70, 3, 700, 30


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


class Loop:
    def __init__(self, seed):
        g = torch.Generator().manual_seed(seed)
        pre = -(-PREFIX // PAGE)
        self.kv = V.PagedKV(*(torch.zeros(pre + SEQS * WIDTH, HKV, PAGE, HD, device=DEV, dtype=torch.float16) for _ in range(2)))
        order = torch.randperm(pre + SEQS * WIDTH, generator=g).to(torch.int32).to(DEV)
        self.pre, self.table = order[:pre], order[pre:].view(SEQS, WIDTH)
        self.rows = torch.randn(VOCAB, HEADS + 2 * HKV, HD, generator=g).to(DEV)  # a token's queries, keys and values
        self.head = (torch.randn(HEADS * HD, VOCAB, generator=g) * 0.1).to(DEV)
        # the shared prefix, by the same operator: one sequence of its own
        x = self.rows[torch.randint(0, VOCAB, (PREFIX,), generator=g).to(DEV)]
        self.kv.append(x[:, HEADS:HEADS + HKV], x[:, HEADS + HKV:], torch.arange(PREFIX, dtype=torch.int32, device=DEV),
                       self.pre.view(1, -1), seq=ints([0] * PREFIX))
        self.lens, self.token = ints([0] * SEQS), torch.arange(SEQS, device=DEV)
        self.u = torch.rand(STEPS, SEQS, generator=g, dtype=torch.float64).to(DEV)

    def step(self, u):
        x = self.rows[self.token]
        q = self.kv.append(x[:, HEADS:HEADS + HKV], x[:, HEADS + HKV:], self.lens + PREFIX, self.table, base=PREFIX, q=x[:, :HEADS])
        self.lens += 1
        y = self.kv.attend(q, self.lens, self.table, prefix_pages=self.pre, prefix_len=PREFIX)
        logits = y.reshape(SEQS, -1) @ self.head
        token, kept, prob = V.sample_rows(logits, u, temperature=0.9, top_k=50, top_p=0.95, min_p=0.02)
        self.token.copy_(token)
        return q, y, logits, token, kept


def test_a_decode_loop_step_by_step():
    loop = Loop(1)
    for i in range(STEPS):
        pos = (loop.lens + PREFIX).cpu()
        x = loop.rows[loop.token].cpu().double()
        q, y, logits, token, kept = loop.step(loop.u[i])
        want_q = turn(x[:, :HEADS], pos, 1e6, HD, True)
        assert (q.cpu().double() - want_q).abs().max() <= 1e-5
        if i % 6 == 5:
            want, _, bound = attend(q.cpu(), loop.kv.k_pages.cpu(), loop.kv.v_pages.cpu(), loop.table.cpu(), loop.lens.cpu(),
                                    list(range(SEQS + 1)), loop.pre.cpu(), PREFIX, WIDTH * PAGE)
            assert ((y.cpu().double() - want).abs() <= bound).all()
        for s in range(SEQS):
            t, n, _, edge = sample(logits[s].cpu(), float(loop.u[i, s]), 0.9, 50, float(torch.tensor(0.95)), float(torch.tensor(0.02)))
            assert edge < 1e-9 or (int(token[s]), int(kept[s])) == (t, n)


def test_loops_replayed_from_graphs_and_side_by_side():
    """A graph of the whole step replayed, with eager work in between, and two
    loops run by two threads on streams of their own: every token as eagerly."""
    want = []
    for seed in (1, 2):
        loop = Loop(seed)
        want.append(torch.stack([loop.step(loop.u[i])[3].clone() for i in range(STEPS)]))
    loop = Loop(1)
    u = loop.u[0].clone()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):  # (the projection's library makes its workspace)
        loop.step(u)
    torch.cuda.synchronize()
    loop = Loop(1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        token = loop.step(u)[3]
    for i in range(STEPS):
        u.copy_(loop.u[i])
        graph.replay()
        assert torch.equal(token, want[0][i]), i
        (torch.ones(64, device=DEV) * i).sum()
        torch.cuda.synchronize()
    got = [None, None]

    def run(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            loop = Loop(k + 1)
            got[k] = torch.stack([loop.step(loop.u[i])[3].clone() for i in range(STEPS)]).cpu()

    threads = [threading.Thread(target=run, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for k in range(2):
        assert got[k] is not None and torch.equal(got[k], want[k].cpu())
