"""A serving loop of all its operators together: plan, append, attention over shared prefixes, sampling, first call by
call, then as a captured graph that is replayed while conversations end and begin.  Each operator's result is held
against its definition on the inputs that it had, with the tolerances of its own tests."""
import math

import numpy as np
import pytest

from test_paged_gpu import TINY, U
from test_sample_rows_gpu import _one
from yalm_b200 import PagedBatch, sample_rows

pytestmark = pytest.mark.gpu

H, K, D, P = 8, 2, 64, 16
S, ROWS, VOCAB, WIDTH = 24, 320, 503, 400  # a table so wide that prefixes are computed apart
PREFIX, STARTS = [256, 160], [0, 11, 24]


class Server:
    def __init__(self, dtype):
        import torch
        g = torch.Generator(device="cuda").manual_seed(3)
        i32 = dict(dtype=torch.int32, device="cuda")
        rnd = lambda *shape, sd=1.0: torch.randn(*shape, generator=g, device="cuda") * sd
        self.dtype, n_pages = dtype, 300
        self.k = torch.full((n_pages, K, P, D), math.nan, dtype=dtype, device="cuda")
        self.v = self.k.clone()
        self.table = torch.full((S, WIDTH), -1, **i32)
        self.q_start, self.kv_len = torch.zeros(S + 1, **i32), torch.zeros(S, **i32)
        self.free, self.n_free = torch.randperm(n_pages, generator=g, device="cuda").int(), torch.tensor([n_pages], **i32)
        self.status, self.new_len, self.kept = torch.zeros(4, **i32), torch.zeros(S, **i32), torch.zeros(S, **i32)
        self.pos, self.slots = torch.zeros(ROWS, **i32), torch.zeros(ROWS, dtype=torch.int64, device="cuda")
        self.b = PagedBatch(self.k, self.v, self.table, self.q_start, self.kv_len, H, ROWS)
        self.work = torch.zeros(self.b.shared_scratch_bytes(2), dtype=torch.uint8, device="cuda")
        self.group_start, self.prefix_len = torch.tensor(STARTS, **i32), torch.tensor(PREFIX, **i32)
        self.emb, self.w_qkv = rnd(VOCAB, 96), rnd(96, (H + 2 * K) * D, sd=0.15)
        self.w_out = rnd(H * D, VOCAB, sd=0.2)
        self.inv_freq = 1e4 ** (-torch.arange(D // 2, device="cuda") / (D / 2))
        self.prompt = torch.randint(0, VOCAB, (ROWS,), generator=g, device="cuda")
        self.tokens, self.prob = torch.zeros(S, **i32), torch.zeros(S, device="cuda")
        self.coin = torch.zeros(S, device="cuda")
        self.temperature = torch.tensor([0.0, 0.7, 1.0, 1.3], device="cuda").repeat(S // 4)
        self.top_k = torch.tensor([0, 40, 5], **i32).repeat(S // 3)
        self.top_p = torch.tensor([1.0, 0.9], device="cuda").repeat(S // 2)
        self.q, self.out = torch.zeros(ROWS, H * D, dtype=dtype, device="cuda"), torch.zeros(ROWS, H * D, dtype=dtype, device="cuda")

    def step(self, shared=True):
        import torch
        self.b.plan(self.new_len, self.free, self.n_free, self.status, kept=self.kept, pos=self.pos, slots=self.slots)
        row = torch.arange(ROWS, device="cuda")
        seq = torch.searchsorted(self.q_start[1:].contiguous(), row, right=True).clamp(max=S - 1)
        # single tokens go on with what was drawn last, prompts with the prompt's tokens
        token = torch.where(self.new_len[seq] == 1, self.tokens[seq].long(), self.prompt[row])
        self.b.append(self.emb[token] @ self.w_qkv, self.q, self.inv_freq, D, pos=self.pos)
        if shared:
            self.b.attend_shared(self.q, self.out, self.work, self.group_start, self.prefix_len)
        else:
            self.b.attend(self.q, self.out, self.work)
        last = (self.q_start[1:].long() - 1).clamp(min=0)
        self.logits = self.out[last].float() @ self.w_out
        sample_rows(self.logits, self.coin, self.tokens, prob=self.prob, temperature=self.temperature, top_k=self.top_k,
                    top_p=self.top_p)

    def check(self, kv, new):
        """kv: cached slots before the step."""
        import torch
        torch.cuda.synchronize()
        assert self.status.tolist() == [0, 0, 0, -1] and self.b.status(self.work) == 0
        n = [max(x, 0) for x in new]
        start = np.concatenate(([0], np.cumsum(n))).tolist()
        after = [0 if x < 0 else c + x for c, x in zip(kv, new)]
        assert self.q_start.tolist() == start and self.kv_len.tolist() == after
        table, u = self.table.long(), U["f16" if self.dtype is torch.float16 else "bf16"]
        for s in range(S):
            if not n[s]:
                continue
            rows = torch.arange(start[s], start[s + 1], device="cuda")
            at = torch.arange(after[s] - n[s], after[s], device="cuda")
            assert torch.equal(self.pos[rows].long(), at)
            assert torch.equal(self.slots[rows], table[s, at // P] * P + at % P)
            t = torch.arange(after[s], device="cuda")
            seen = t[None] <= at[:, None]
            q = self.q[rows].double().view(-1, H, D)
            for h in range(H):
                k, v = (x[table[s, t // P], h // (H // K), t % P].double() for x in (self.k, self.v))
                sc = (q[:, h] @ k.T / 8.0)
                mag = (q[:, h].abs() @ k.abs().T / 8.0 * seen).amax(-1, keepdim=True)
                w = torch.softmax(sc.masked_fill(~seen, -math.inf), -1)
                tol = u * (w @ v).abs() + (u + 2.0 ** -16 + 2 * 2.0 ** -20 * mag) * (w @ v.abs()) + TINY
                got = self.out[rows].double().view(-1, H, D)[:, h]
                assert ((got - w @ v).abs() <= tol).all()
        x = self.logits.double().cpu().numpy()
        f = lambda t: t.double().tolist()
        for s, (c, T, k, p) in enumerate(zip(f(self.coin), f(self.temperature), self.top_k.tolist(), f(self.top_p))):
            token, prob = _one(x[s], c, T, k, p, 0.0)
            assert int(self.tokens[s]) == token and abs(float(self.prob[s]) - prob) <= 2.0 ** -24 * prob + 2.0 ** -42
        return after


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_conversations_behind_shared_prefixes(gpu, dtype):
    import torch
    srv, rng = Server(getattr(torch, dtype)), np.random.default_rng(5)

    def go(new, kv, run):
        srv.new_len.copy_(torch.tensor(new))
        srv.coin.copy_(torch.from_numpy(rng.random(S).astype(np.float32)))
        run()
        return srv.check(kv, new)

    # the prefixes, each by the first of its group; then the others begin with their pages
    for g, first in enumerate(STARTS[:-1]):
        go([PREFIX[g] if s == first else 0 for s in range(S)], srv.kv_len.tolist(), lambda: srv.step(shared=False))
    for g in range(2):
        for s in range(STARTS[g], STARTS[g + 1]):
            srv.table[s, : PREFIX[g] // P] = srv.table[STARTS[g], : PREFIX[g] // P]
            srv.kv_len[s] = PREFIX[g]
            srv.kept[s] = PREFIX[g] // P
    kv = go([1 + int(x) for x in rng.integers(0, 9, S)], srv.kv_len.tolist(), srv.step)
    kv = go([1] * S, kv, srv.step)
    torch.cuda.synchronize()
    before = {k: getattr(srv, k).clone() for k in ("table", "kv_len", "free", "n_free", "k", "v", "tokens")}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        srv.step()
    for k, v in before.items():
        getattr(srv, k).copy_(v)
    for i in range(12):
        new = [1] * S
        for s in range(S):
            group = 0 if s < STARTS[1] else 1
            if s not in STARTS and i in (3, 7) and s % 5 == i % 5:
                new[s] = -1
            elif kv[s] == 0:  # a new conversation in the place of one that ended
                new[s] = 0
                srv.kv_len[s] = kv[s] = PREFIX[group]
            elif kv[s] == PREFIX[group]:
                new[s] = 7
        kv = go(new, kv, graph.replay)
