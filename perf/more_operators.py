"""The operators at the two ends and in the middle of a serving step over a paged KV cache, as a serving
program calls them:

 - kind "plan": from the number of tokens that every sequence brings, the batch's row starts, the caches' new
   lengths, the pages that the new tokens need (taken from a list of free ones, to which the pages of ended
   sequences go back), and every token's position and slot;
 - kind "shared": attention of the new tokens of sequences whose caches begin with the same pages, a long
   prefix, computed once for all of them;
 - kind "sample": a token for every row of logits, with temperature, top-k, top-p and min-p from a given random number.

A "plan" case: `seqs` sequences, of which the first `singles` bring one token, every eighth of the others none and the
rest up to `new`; `ended` of them end; up to `ctx` slots are cached before; `pad` rows lie behind the last token.
A "shared" case: `groups` groups of together `seqs` sequences, each group with a prefix of up to `prefix` slots, each
sequence with up to `own` cached slots of its own behind it and up to `new` new tokens; `loose` more sequences share
nothing.  `mix` (0: every sequence has just these lengths; else the seed of ragged ones).
A "sample" case: `rows` of `vocab` logits, `gap` elements more from row to row, `how` the rows are drawn from.
"""
import math
import random

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
# the largest listed cases: (token, slot, head) triples, cached elements of K; logits; sequences, tokens, pages
CELLS = 256 * 17600 * 64
CACHE = (16384 + 256 * 1088) * 8 * 128
LOGITS = 256 * 131072
PLAN = 16384 * 64


def _plan(name, seqs, new, ctx, page, singles=0, ended=0, mix=0, pad=0):
    return dict(name=name, kind="plan", seqs=seqs, new=new, ctx=ctx, page=page, singles=singles, ended=ended, mix=mix,
                pad=pad)


def _shared(name, heads, kv_heads, head_dim, page, dtype, groups, seqs, prefix, own_ctx, new=1, loose=0, mix=0, pad=0):
    return dict(name=name, kind="shared", heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page, dtype=dtype,
                groups=groups, seqs=seqs, prefix=prefix, own=own_ctx, new=new, loose=loose, mix=mix, pad=pad)


def _sample(name, rows, vocab, dtype, how, gap=0):
    return dict(name=name, kind="sample", rows=rows, vocab=vocab, dtype=dtype, how=how, gap=gap)


def listed():
    return [
        # the next token of one conversation: the call's own latency
        _plan("plan 1 sequence", 1, 1, 36, 16, singles=1),
        # a step of a busy server: 200 conversations, chunks of new prompts beside them, some that ended, a padded batch
        _plan("plan 256 sequences", 256, 300, 2000, 16, singles=200, ended=9, mix=5, pad=11),
        # a very large batch of short prompts, as offline scoring brings them
        _plan("plan 16384 sequences", 16384, 64, 500, 32, singles=3000, ended=500, mix=3),
        # three short answers to one short prompt on the smallest model: the call's own latency
        _shared("shared 3 singles", 8, 2, 64, 16, "f16", 1, 3, 256, 20),
        # 64 conversations behind one system prompt, one token each
        _shared("shared 64 singles prefix 8192", 32, 8, 128, 16, "f16", 1, 64, 8192, 700, mix=4),
        # four system prompts of different lengths, some conversations without one, on a wide model, padded
        _shared("shared 4 groups bf16", 64, 8, 128, 32, "bf16", 4, 57, 5000, 400, loose=4, mix=8, pad=3),
        # guesses of five tokens for each conversation, checked at once, narrow heads
        _shared("shared 24 drafts of 5 hd 64", 16, 2, 64, 64, "f16", 1, 24, 4096, 300, new=5, mix=6),
        # many samples of one long document
        _shared("shared 256 singles prefix 16384", 64, 8, 128, 64, "bf16", 1, 256, 16384, 1024, mix=2),
        # one row of a vocabulary of this repository's models
        _sample("sample 1 row", 1, 32000, "f32", "nucleus"),
        # a serving step of 61 conversations with settings of their own, rows of a padded vocabulary
        _sample("sample 61 rows mixed", 61, 49999, "f32", "mixed", gap=17),
        # a large vocabulary, 16-bit logits, ties among them
        _sample("sample 64 rows bf16", 64, 131072, "bf16", "mixed"),
        # many samples at a high temperature without limits but min-p
        _sample("sample 256 rows", 256, 131072, "f32", "hot"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "shared", "shared", "sample"])
    if kind == "plan":
        c = dict(kind=kind, seqs=_log(rng, 1, 16384), new=_log(rng, 1, 4096), ctx=_log(rng, 1, 8192) - 1,
                 page=rng.choice([16, 32, 64, 128, 256]), singles=0, ended=0, mix=rng.randrange(1, 1 << 20),
                 pad=rng.choice([0, rng.randrange(1, 9)]))
        while c["seqs"] * (c["new"] + c["ctx"] // 8) > PLAN:
            c["new"], c["ctx"] = max(1, c["new"] // 2), c["ctx"] // 2
        c["singles"] = rng.randrange(0, c["seqs"] + 1)
        c["ended"] = rng.randrange(0, c["seqs"] // 4 + 1)
        return c
    if kind == "sample":
        c = dict(kind=kind, rows=_log(rng, 1, 256), vocab=_log(rng, 1000, 262144), dtype=rng.choice(sorted(TYPES)),
                 how=rng.choice(["nucleus", "mixed", "mixed", "hot"]), gap=rng.choice([0, rng.randrange(1, 40)]))
        while c["rows"] * c["vocab"] > LOGITS:
            c["rows"] = c["rows"] * 3 // 4
        return c
    heads, kv_heads, head_dim = rng.choice([(8, 2, 64), (8, 8, 64), (32, 8, 128), (8, 2, 128), (4, 1, 128),
                                            (64, 8, 128), (16, 16, 128), (12, 2, 128), (16, 2, 64)])
    c = dict(kind=kind, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=rng.choice([16, 32, 64, 128, 256]),
             dtype=rng.choice(["f16", "bf16"]), groups=rng.choice([1, 1, 2, rng.randrange(1, 9)]), seqs=0,
             prefix=_log(rng, 64, 32768), own=_log(rng, 1, 2048) - 1, new=rng.choice([1, 1, 1, rng.randrange(2, 17)]),
             loose=rng.choice([0, 0, rng.randrange(1, 6)]), mix=rng.choice([0, rng.randrange(1, 1 << 20)]),
             pad=rng.choice([0, 0, rng.randrange(1, 9)]))
    c["seqs"] = c["groups"] * _log(rng, 1, 256 // c["groups"])
    while ((c["seqs"] + c["loose"]) * c["new"] * (c["prefix"] + c["own"] + c["new"]) * heads > CELLS
           or (c["groups"] * c["prefix"] + (c["seqs"] + c["loose"]) * (c["own"] + c["new"] + 256)) * kv_heads * head_dim
           > CACHE):
        if c["seqs"] > 2 * c["groups"] and rng.random() < 0.5:
            c["seqs"] = c["seqs"] * 3 // 4
        else:
            c["prefix"], c["own"] = max(64, c["prefix"] * 3 // 4), c["own"] * 3 // 4
    return c


def _ints(v, dtype=torch.int32):
    return torch.tensor(np.asarray(v), dtype=dtype, device="cuda")


def prepare(case, seed):
    return {"plan": _prepare_plan, "shared": _prepare_shared, "sample": _prepare_sample}[case["kind"]](case, seed)


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"plan": _own_plan, "shared": _own_shared, "sample": _own_sample}[kind](state)
    return {"plan": _run_plan, "shared": _run_shared, "sample": _run_sample}[kind](state)


def exact(case, seed):
    return {"plan": _exact_plan, "shared": _exact_shared, "sample": _exact_sample}[case["kind"]](case, seed)


def work(case):
    return {"plan": _work_plan, "shared": _work_shared, "sample": _work_sample}[case["kind"]](case)


# ---------------------------------------------------------------------------------------------- plan
def _plan_lengths(case):
    """What every sequence brings (-1: it ends) and has cached, as arrays."""
    r = np.random.default_rng(case["mix"])
    S = case["seqs"]
    new = np.where(np.arange(S) < case["singles"], 1, r.integers(1, case["new"] + 1, S) if case["mix"] else case["new"])
    new[case["singles"]:][::8] = 0
    kv = r.integers(0, case["ctx"] + 1, S) if case["mix"] else np.full(S, case["ctx"])
    new[r.permutation(S)[: case["ended"]]] = -1
    kept = np.where(np.arange(S) % 3 == 0, kv // case["page"] // 2, 0)  # pages of a prefix that others share
    return new, kv, kept


def _prepare_plan(case, seed):
    new, kv, kept = _plan_lengths(case)
    P, S = case["page"], case["seqs"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    held, then = -(-kv // P), -(-(kv + np.maximum(new, 0)) // P)
    total = int(held.sum())
    pages = int(total + (then - held).sum()) + 40
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    width = int(then.max()) + 1
    table = torch.full((S, width), -1, dtype=torch.int32, device="cuda")
    row, at = np.repeat(np.arange(S), held), np.arange(total) - np.repeat(np.cumsum(held) - held, held)
    table[torch.from_numpy(row).cuda(), torch.from_numpy(at).cuda()] = order[:total]
    free = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
    free[: pages - total] = order[total:]
    T = int(np.maximum(new, 0).sum()) + case["pad"]
    i32 = dict(dtype=torch.int32, device="cuda")
    return dict(case=case, new_len=_ints(new), kv_before=_ints(kv), kept=_ints(kept), page_table=table, free=free,
                n_free_before=_ints([pages - total]), n_free=torch.zeros(1, **i32), q_start=torch.zeros(S + 1, **i32),
                kv_len=torch.zeros(S, **i32), pos=torch.zeros(T, **i32), status=torch.zeros(4, **i32),
                slots=torch.zeros(T, dtype=torch.int64, device="cuda"),
                k_pages=torch.empty((pages, 1, P, 64), dtype=torch.float16, device="cuda"),
                v_pages=torch.empty((pages, 1, P, 64), dtype=torch.float16, device="cuda"))


PLANNED = ("q_start", "kv_len", "page_table", "free", "n_free", "pos", "slots", "status")


def _own_plan(st):
    b = st.get("batch")
    if b is None:
        from yalm_b200 import PagedBatch
        b = st["batch"] = PagedBatch(st["k_pages"], st["v_pages"], st["page_table"], st["q_start"], st["kv_len"], 1,
                                     st["pos"].shape[0])
    b.plan(st["new_len"], st["free"], st["n_free"], st["status"], kv_before=st["kv_before"],
           n_free_before=st["n_free_before"], kept=st["kept"], pos=st["pos"], slots=st["slots"])
    return {k: st[k] for k in PLANNED}


def _run_plan(st):
    P, table, free = st["case"]["page"], st["page_table"], st["free"]
    new, kv = st["new_len"].long(), st["kv_before"].long()
    ended, n = new < 0, new.clamp(min=0)
    held = (kv + P - 1) // P
    # the pages of ended sequences, behind the free ones
    col = torch.arange(table.shape[1], device="cuda")
    back = table[ended[:, None] & (col >= st["kept"].long()[:, None]) & (col < held[:, None])]
    free0 = st["n_free_before"].long()
    free[free0 + torch.arange(back.shape[0], device="cuda")] = back
    free0 = free0 + back.shape[0]
    # the new pages, from the end of the list
    after = torch.where(ended, 0, kv + n)
    more = torch.where(ended, 0, (after + P - 1) // P - held)
    first = more.cumsum(0) - more
    want = ~ended[:, None] & (col >= held[:, None]) & (col < (held + more)[:, None])
    at = free0 - 1 - (first[:, None] + col - held[:, None])
    table[want] = free[at[want]]
    st["n_free"].copy_(free0 - more.sum())
    st["kv_len"].copy_(after)
    st["q_start"][0] = 0
    st["q_start"][1:] = n.cumsum(0)
    # the tokens
    T = st["pos"].shape[0] - st["case"]["pad"]
    seq = torch.repeat_interleave(torch.arange(n.shape[0], device="cuda"), n, output_size=T)
    pos = kv[seq] + torch.arange(T, device="cuda") - st["q_start"].long()[seq]
    st["pos"][:T] = pos.int()
    st["slots"][:T] = table[seq, pos // P].long() * P + pos % P
    st["status"].zero_()
    st["status"][3] = -1
    return {k: st[k] for k in PLANNED}


def _exact_plan(case, seed):
    st = _prepare_plan(case, seed)
    P = case["page"]
    new, kv, kept, free = (st[k].tolist() for k in ("new_len", "kv_before", "kept", "free"))
    table = st["page_table"].cpu().numpy()
    n_free, pos, slots, q_start, after = st["n_free_before"].item(), [], [], [0], []
    for s, n in enumerate(new):
        if n < 0:
            for j in range(kept[s], -(-kv[s] // P)):
                free[n_free] = int(table[s, j])
                n_free += 1
    for s, n in enumerate(new):
        have = kv[s] if n >= 0 else 0
        for t in range(have, have + max(n, 0)):
            if t % P == 0:
                n_free -= 1
                table[s, t // P] = free[n_free]
            pos.append(t)
            slots.append(int(table[s, t // P]) * P + t % P)
        after.append(have + max(n, 0))
        q_start.append(q_start[-1] + max(n, 0))
    out = dict(q_start=q_start, kv_len=after, free=free, n_free=[n_free], pos=pos + [0] * case["pad"],
               slots=slots + [0] * case["pad"], status=[0, 0, 0, -1])
    out = {k: _ints(v, torch.int64 if k == "slots" else torch.int32) for k, v in out.items()}
    out["page_table"] = torch.from_numpy(table).cuda()
    return {k: out[k] for k in PLANNED}


def _work_plan(case):
    new, kv, kept = _plan_lengths(case)
    P = case["page"]
    held = -(-kv // P)
    n = np.maximum(new, 0)
    back = int(np.maximum(held - kept, 0)[new < 0].sum())
    more = int((-(-(kv + n) // P) - held)[new >= 0].sum())
    T = int(n.sum())
    return {"bytes": 8 * len(kv) + 8 * len(kv) + 8 * (back + more) + 12 * T + 4 * case["ended"] + 32, "flops": 2 * T}


# -------------------------------------------------------------------------------------------- shared
def _shared_lengths(case):
    """The groups' first sequences and prefixes; each sequence's new tokens and cache length with them."""
    r = random.Random(case["mix"])
    G, P = case["groups"], case["page"]
    some = lambda n, low: r.randint(low, n) if case["mix"] and n > low else n
    cuts = sorted(r.sample(range(1, case["seqs"]), G - 1)) if case["mix"] else [case["seqs"] * g // G for g in range(1, G)]
    start = [0] + cuts + [case["seqs"]]
    prefix = [max(1, some(case["prefix"], case["prefix"] // 4) // P) * P for _ in range(G)]
    new, kv = [], []
    for g in range(G):
        for _ in range(start[g], start[g + 1]):
            new.append(some(case["new"], 1))
            kv.append(prefix[g] + some(case["own"], 0) + new[-1])
    for _ in range(case["loose"]):
        new.append(some(case["new"], 1))
        kv.append(some(case["prefix"], 0) // 2 + some(case["own"], 0) + new[-1])
    return start, prefix, new, kv


def _prepare_shared(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    start, prefix, new, kv = _shared_lengths(case)
    H, K, D, P, dt = case["heads"], case["kv_heads"], case["head_dim"], case["page"], TYPES[case["dtype"]]
    width = max(-(-n // P) for n in kv)
    table = np.full((len(kv), width), -1, dtype=np.int32)
    # the pool, a few more pages than are in use, handed out in no order
    total = sum(-(-n // P) for n in kv) - sum((start[i + 1] - start[i] - 1) * (p // P) for i, p in enumerate(prefix))
    order = torch.randperm(total + 3, generator=g, device="cuda").to(torch.int32).cpu().numpy()
    used = 0
    for s, n in enumerate(kv):
        group = next((i for i in range(len(prefix)) if start[i] <= s < start[i + 1]), None)
        have = 0
        if group is not None and s > start[group]:
            have = prefix[group] // P
            table[s, :have] = table[start[group], :have]
        more = -(-n // P) - have
        table[s, have: have + more] = order[used: used + more]
        used += more
    T = sum(new) + case["pad"]

    def cache(gain):
        x = torch.empty((total + 3, K, P, D), dtype=dt, device="cuda")
        return x.normal_(0.0, gain, generator=g)

    return dict(case=case, start=start, prefix=prefix, new=new, kv=kv, page_table=torch.from_numpy(table).cuda(),
                q_start=_ints([0] + list(np.cumsum(new))), kv_len=_ints(kv), group_start=_ints(start),
                prefix_len=_ints(prefix), k_pages=cache(1.4), v_pages=cache(1.0),
                q=torch.empty((T, H * D), device="cuda").normal_(0.0, 1.4, generator=g).to(dt),
                out=torch.zeros((T, H * D), dtype=dt, device="cuda"))


def _own_shared(st):
    b = st.get("batch")
    if b is None:
        from yalm_b200 import PagedBatch
        b = st["batch"] = PagedBatch(st["k_pages"], st["v_pages"], st["page_table"], st["q_start"], st["kv_len"],
                                     st["case"]["heads"], st["q"].shape[0])
        st["scratch"] = torch.zeros(b.shared_scratch_bytes(st["case"]["groups"]), dtype=torch.uint8, device="cuda")
    b.attend_shared(st["q"], st["out"], st["scratch"], st["group_start"], st["prefix_len"])
    return st["out"]


def _run_shared(st):
    c = st["case"]
    H, K, D, P = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    first = 0
    for s, (n, m) in enumerate(zip(st["new"], st["kv"])):
        pages = st["page_table"][s, : -(-m // P)].long()
        k = st["k_pages"][pages].float().permute(1, 0, 2, 3).reshape(K, -1, D)[:, :m]
        v = st["v_pages"][pages].float().permute(1, 0, 2, 3).reshape(K, -1, D)[:, :m]
        q = st["q"][first: first + n].float().view(n, K, H // K, D).permute(1, 2, 0, 3).reshape(K, -1, D)
        x = torch.matmul(q, k.transpose(1, 2)).view(K, H // K, n, m) * (1.0 / math.sqrt(D))
        if n > 1:
            hidden = torch.arange(m, device="cuda") > torch.arange(m - n, m, device="cuda")[:, None]
            x.masked_fill_(hidden, -math.inf)
        p = (x - x.amax(-1, keepdim=True)).exp()
        o = torch.matmul(p.view(K, -1, m), v).view(K, H // K, n, D) / p.sum(-1, keepdim=True)
        st["out"][first: first + n] = o.permute(2, 0, 1, 3).reshape(n, H * D).to(st["out"].dtype)
        first += n
    return st["out"]


def _exact_shared(case, seed):
    st = _prepare_shared(case, seed)
    H, K, D, P = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    G = H // K
    out = st["out"].double()
    q = st["q"].double().view(-1, H, D)
    first = 0
    for s, (n, m) in enumerate(zip(st["new"], st["kv"])):
        slot = torch.arange(m, device="cuda")
        page = st["page_table"][s].long()[slot // P]
        for h in range(K):
            k, v = st["k_pages"][page, h, slot % P].double(), st["v_pages"][page, h, slot % P].double()
            for i in range(n):
                seen = m - n + i + 1
                w = torch.softmax(q[first + i, h * G: (h + 1) * G] @ k[:seen].T / math.sqrt(D), -1)
                out[first + i].view(H, D)[h * G: (h + 1) * G] = w @ v[:seen]
        first += n
    return out


def _work_shared(case):
    start, prefix, new, kv = _shared_lengths(case)
    H, K, D, e = case["heads"], case["kv_heads"], case["head_dim"], SIZE[case["dtype"]]
    slots = sum(kv) - sum((start[g + 1] - start[g] - 1) * p for g, p in enumerate(prefix))
    pairs = sum(m - n + i + 1 for n, m in zip(new, kv) for i in range(n))
    return {"bytes": 2 * sum(new) * H * D * e + 2 * slots * K * D * e, "flops": 4 * pairs * H * D}


# -------------------------------------------------------------------------------------------- sample
LEAST = 2.0 ** -47  # of the largest weight: what is less is never drawn


def _prepare_sample(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    R, V = case["rows"], case["vocab"]
    x = torch.empty((R, V + case["gap"]), device="cuda").normal_(0.0, 2.0, generator=g)
    # a few dozen tokens stand out, as they do behind a context
    likely = (torch.randint(0, V, (R, 1), generator=g, device="cuda") + torch.arange(40, device="cuda") * (V // 41)) % V
    x.scatter_add_(1, likely, torch.rand((R, 40), generator=g, device="cuda") * 9.0)
    pick = lambda *v: torch.tensor(v, device="cuda")[torch.randint(0, len(v), (R,), generator=g, device="cuda")]
    how = case["how"]
    if how == "nucleus":
        par = dict(temperature=pick(0.8), top_k=pick(50), top_p=pick(0.95), min_p=None)
    elif how == "hot":
        par = dict(temperature=pick(1.3, 1.7), top_k=None, top_p=None, min_p=pick(0.0, 0.02))
    else:
        par = dict(temperature=pick(0.0, 0.6, 0.8, 1.0, 1.2), top_k=pick(0, 0, 20, 64, 1000), top_p=pick(1.0, 0.9, 0.97),
                   min_p=pick(0.0, 0.0, 0.05))
    return dict(case=case, logits=x.to(TYPES[case["dtype"]])[:, :V], coin=torch.rand(R, generator=g, device="cuda"),
                tokens=torch.zeros(R, dtype=torch.int32, device="cuda"), prob=torch.zeros(R, device="cuda"),
                **{k: v if v is None else v.int() if k == "top_k" else v.float() for k, v in par.items()})


def _own_sample(st):
    from yalm_b200 import sample_rows
    sample_rows(st["logits"], st["coin"], st["tokens"], prob=st["prob"], temperature=st["temperature"],
                top_k=st["top_k"], top_p=st["top_p"], min_p=st["min_p"])
    return {"tokens": st["tokens"], "prob": st["prob"]}


def _run_sample(st):
    x = st["logits"].double()  # 64 bits: running sums next to a border decide the token
    R, V = x.shape
    full = lambda v, other: (torch.full((R,), other, device="cuda") if v is None else v).double()[:, None]
    T, k, p, least = full(st["temperature"], 1.0), full(st["top_k"], 0.0), full(st["top_p"], 1.0), full(st["min_p"], 0.0)
    x, order = x.sort(dim=-1, descending=True, stable=True)
    rank = torch.arange(V, device="cuda")
    w = torch.where(T > 0, ((x - x[:, :1]) / T.clamp(min=1e-30)).exp(), (rank == 0).double())
    w = torch.where((w >= LEAST) & ((rank < k) | (k < 1)), w, 0.0)
    total = w.cumsum(-1)
    before = torch.cat((torch.zeros_like(total[:, :1]), total[:, :-1]), -1)
    w = torch.where(((before < p * total[:, -1:]) | (p >= 1) | (rank == 0)) & (w >= least), w, 0.0)
    w = torch.zeros_like(w).scatter_(1, order, w)  # in the order of the tokens again
    total = w.cumsum(-1)
    hit = (total >= st["coin"].double()[:, None] * total[:, -1:]) & (w > 0)
    token = torch.where(hit, rank, V).amin(-1)
    st["tokens"].copy_(token)
    st["prob"].copy_(w.gather(1, token[:, None])[:, 0] / total[:, -1])
    return {"tokens": st["tokens"], "prob": st["prob"]}


def _exact_sample(case, seed):
    st = _prepare_sample(case, seed)
    logits, coin = st["logits"].float().cpu().numpy().astype(np.float64), st["coin"].tolist()
    R = case["rows"]
    col = lambda k, other: [other] * R if st[k] is None else st[k].tolist()
    tokens, prob = [], []
    for x, c, T, k, p, least in zip(logits, coin, col("temperature", 1.0), col("top_k", 0), col("top_p", 1.0),
                                    col("min_p", 0.0)):
        if T <= 0:
            tokens.append(int(np.argmax(x)))
            prob.append(1.0)
            continue
        w = np.exp((x - x.max()) / T)
        w[w < LEAST] = 0.0
        if 0 < k < len(w) or p < 1:
            best = np.lexsort((np.arange(len(x)), -x))
            if 0 < k < len(w):
                best = best[:k]
            if p < 1:
                run_sum = np.cumsum(w[best])
                best = best[: int(np.searchsorted(run_sum, p * run_sum[-1])) + 1]
            only = np.zeros_like(w)
            only[best] = w[best]
            w = only
        w[w < least] = 0.0
        alive = np.flatnonzero(w)
        run_sum = np.cumsum(w[alive])
        at = alive[int(np.searchsorted(run_sum, c * run_sum[-1]))]
        tokens.append(int(at))
        prob.append(w[at] / run_sum[-1])
    return {"tokens": _ints(tokens), "prob": _ints(prob, torch.float64)}


def _work_sample(case):
    n = case["rows"] * case["vocab"]
    return {"bytes": n * SIZE[case["dtype"]] + 28 * case["rows"], "flops": 4 * n}
