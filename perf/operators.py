"""The paged-cache operators as a serving program calls them: the per-head norm, rotation and append
of new tokens into a paged KV cache (kind "append"), and the attention of those tokens over the
cache (kind "attend"), for batches of sequences that bring a whole prompt, a chunk of one, or a
single token each.

A case names the heads, the page size, the element type, how many sequences there are (`seqs`), how
many new tokens a sequence brings at most (`new`; the first `singles` sequences bring one), how many
tokens are cached before them at most (`ctx`), `mix` (0: every sequence has just these lengths;
else the seed of ragged ones) and `pad`, the rows of the token-major buffers behind the last sequence.
`window`: how many slots back a token sees, itself counted (0: all of them).
"""
import math
import random

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
CELLS = 2048 * 16384 * 32  # scores of the largest listed case, over all query heads
CACHE = 64 * 8 * 4096 * 128 + (1 << 22)  # cached elements of K of the largest listed case, with its padding


def _case(name, kind, heads, kv_heads, head_dim, page, dtype, seqs, new, ctx, singles=0, mix=0, pad=0, src="f32",
          norm=True, half=False, rotary=None, window=0):
    c = dict(name=name, kind=kind, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page, dtype=dtype,
             seqs=seqs, new=new, ctx=ctx, singles=singles, mix=mix, pad=pad)
    if kind == "append":
        c.update(src=src, norm=norm, half=half, rotary=head_dim if rotary is None else rotary)
    else:
        c.update(window=window)
    return c


def listed():
    return [
        # one token of one short conversation on the smallest model: the call's own latency
        _case("append 1 token", "append", 8, 2, 64, 16, "f16", 1, 1, 36),
        # a serving step of 64 conversations, one token each, fp32 projections, a batch padded to a captured size
        _case("append 61 singles", "append", 32, 8, 128, 16, "f16", 61, 1, 400, singles=61, mix=11, pad=3),
        # chunks of three prompts on a wide model, part of the head rotated, pairs half a rotation apart
        _case("append 3 chunks bf16", "append", 64, 8, 128, 32, "bf16", 3, 700, 900, mix=5, src="bf16", half=True,
              rotary=96),
        # a whole long prompt
        _case("append 8192 tokens", "append", 32, 8, 128, 64, "f16", 1, 8192, 0, src="f16"),
        # one token after a short prompt: the call's own latency
        _case("attend 1 token ctx 36", "attend", 8, 2, 64, 16, "f16", 1, 1, 36),
        # one token of one long conversation: the cache is split over the whole GPU
        _case("attend 1 token ctx 32767", "attend", 32, 8, 128, 64, "f16", 1, 1, 32767),
        # a serving step of 64 conversations of very different lengths
        _case("attend 64 singles", "attend", 32, 8, 128, 16, "bf16", 64, 1, 4095, singles=64, mix=3),
        # the same on one of four tensor-parallel ranks, and a batch padded to a captured size
        _case("attend 29 singles rank", "attend", 8, 2, 128, 32, "f16", 29, 1, 8000, singles=29, mix=9, pad=3),
        # a prompt's chunk over the part that is cached
        _case("attend chunk 512", "attend", 32, 8, 128, 16, "f16", 1, 512, 2690),
        # a mixed step: chunks of three prompts beside single tokens of thirteen conversations
        _case("attend mixed bf16", "attend", 64, 8, 128, 32, "bf16", 16, 300, 2000, singles=13, mix=7),
        # ragged prompts of a small model with narrow heads and a sliding window
        _case("attend 5 prompts hd 64", "attend", 8, 2, 64, 64, "f16", 5, 1500, 0, mix=2, window=512),
        # the last chunk of a very long prompt
        _case("attend chunk 2048 ctx 14336", "attend", 32, 8, 128, 64, "f16", 1, 2048, 14336),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    heads, kv_heads, head_dim = rng.choice([(8, 2, 64), (8, 8, 64), (32, 8, 128), (8, 2, 128), (4, 1, 128),
                                            (64, 8, 128), (16, 16, 128), (12, 2, 128), (16, 2, 64)])
    c = dict(kind=rng.choice(["append", "attend", "attend"]), heads=heads, kv_heads=kv_heads, head_dim=head_dim,
             page=rng.choice([16, 32, 64, 128, 256]), dtype=rng.choice(["f16", "bf16"]), seqs=_log(rng, 1, 64),
             new=1 if rng.random() < 0.4 else _log(rng, 2, 4096), ctx=_log(rng, 1, 32768) - 1, singles=0,
             mix=rng.choice([0, rng.randrange(1, 1 << 20)]), pad=rng.choice([0, 0, rng.randrange(1, 9)]))
    if c["new"] == 1:
        c["singles"] = c["seqs"]
    elif c["seqs"] > 1 and rng.random() < 0.3:
        c["singles"] = rng.randrange(1, c["seqs"])
    if c["kind"] == "append":
        c["ctx"] //= c["seqs"]  # a pool that the new tokens are a fair part of
        c.update(src=rng.choice(["f32", "f16", "bf16"]), norm=rng.random() < 0.8, half=rng.random() < 0.5,
                 rotary=rng.choice([0, head_dim // 2, head_dim, head_dim]))
    else:
        c["window"] = rng.choice([0, 0, 0, _log(rng, 1, 4096)])
    # no more work or memory than the largest listed case
    while (c["seqs"] * c["new"] * (c["ctx"] + c["new"]) * heads > CELLS
           or c["seqs"] * (c["ctx"] + c["new"] + 256) * kv_heads * head_dim > CACHE
           or c["seqs"] * c["new"] * (heads + 2 * kv_heads) * head_dim > 8192 * 48 * 128):
        if c["seqs"] > 1 and rng.random() < 0.6:
            c["seqs"] = max(1, c["seqs"] * 3 // 4)
            c["singles"] = c["seqs"] if c["new"] == 1 else min(c["singles"], c["seqs"] - 1)
        elif c["new"] > 1 and rng.random() < 0.5:
            c["new"] = max(2, c["new"] * 3 // 4)
        else:
            c["ctx"] = c["ctx"] * 3 // 4
    return c


def _lengths(case):
    """Each sequence's new tokens and its cache length with them."""
    r = random.Random(case["mix"])
    new, kv = [], []
    for s in range(case["seqs"]):
        n = 1 if s < case["singles"] else r.randint(max(1, case["new"] // 3), case["new"]) if case["mix"] else case["new"]
        c = r.randint(case["ctx"] // 16, case["ctx"]) if case["mix"] else case["ctx"]
        new.append(n)
        kv.append(c + n)
    return new, kv


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    new, kv = _lengths(case)
    H, K, D, P = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    dt = TYPES[case["dtype"]]
    need = [-(-n // P) for n in kv]
    total, width = sum(need), max(need)
    # the pool: a few more pages than are in use, handed out in no order
    pages = total + 3
    order = torch.randperm(pages, generator=g, device="cuda")[:total].to(torch.int32)
    row = np.repeat(np.arange(len(kv)), need)
    col = np.concatenate([np.arange(n) for n in need])
    table = torch.full((len(kv), width), -1, dtype=torch.int32, device="cuda")
    table[torch.from_numpy(row).cuda(), torch.from_numpy(col).cuda()] = order

    def cache(gain):
        x = torch.empty((pages, K, P, D), dtype=dt, device="cuda")
        return x.normal_(0.0, gain, generator=g)

    T = sum(new) + case["pad"]
    st = dict(case=case, page_table=table, q_start=_ints([0] + list(np.cumsum(new))), kv_len=_ints(kv),
              most_new=max(new), k_pages=cache(1.4), v_pages=cache(1.0),
              q_out=torch.zeros((T, H * D), dtype=dt, device="cuda"))
    if case["kind"] == "append":
        x = torch.empty((T, (H + 2 * K) * D), device="cuda").normal_(0.0, 1.5, generator=g)
        st["qkv"] = x.to(TYPES[case["src"]])
        w = torch.empty((2, D), device="cuda").normal_(1.2, 0.2, generator=g)
        st["q_norm"], st["k_norm"] = (w[0].clone(), w[1].clone()) if case["norm"] else (None, None)
        R = case["rotary"]
        st["inv_freq"] = torch.tensor([1e6 ** (-2.0 * j / R) for j in range(R // 2)] or [0.0], dtype=torch.float32,
                                      device="cuda")
    else:
        st["q"] = torch.empty((T, H * D), device="cuda").normal_(0.0, 1.4, generator=g).to(dt)
    return st


def run(state):
    if own:
        return _own(state)
    return _append(state) if state["case"]["kind"] == "append" else _attend(state)


EPS = 1e-6


def _own(state):
    """The calls that a serving program makes, with the batch descriptor and the workspace that it keeps."""
    from yalm_b200 import PagedBatch

    c = state["case"]
    b = state.get("batch")
    if b is None:
        b = state["batch"] = PagedBatch(state["k_pages"], state["v_pages"], state["page_table"], state["q_start"],
                                        state["kv_len"], c["heads"], state["q_out"].shape[0])
        if c["kind"] == "attend":
            state["scratch"] = torch.zeros(b.scratch_bytes(), dtype=torch.uint8, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    if c["kind"] == "append":
        b.append(state["qkv"], state["q_out"], state["inv_freq"], c["rotary"], q_norm=state["q_norm"],
                 k_norm=state["k_norm"], eps=EPS, half=c["half"], stream=stream)
        return {"q": state["q_out"], "k": state["k_pages"], "v": state["v_pages"]}
    b.attend(state["q"], state["q_out"], state["scratch"], window=c["window"], stream=stream)
    return state["q_out"]


# ------------------------------------------------------------------------------------ plain forms
def _norm(x, w):
    if w is None:
        return x
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w


def _turn(x, cos, sin, half):
    """x [T, heads, dim]: the first 2 * cos.shape[1] elements of each head rotated by pairs."""
    r = 2 * cos.shape[1]
    y, rest = x[..., :r], x[..., r:]
    a, b = (y[..., : r // 2], y[..., r // 2:]) if half else (y[..., 0::2], y[..., 1::2])
    c, s = cos[:, None], sin[:, None]
    u, v = a * c - b * s, a * s + b * c
    y = torch.cat((u, v), -1) if half else torch.stack((u, v), -1).flatten(-2)
    return torch.cat((y, rest), -1)


def _append(st):
    c = st["case"]
    H, K, D, P, R = c["heads"], c["kv_heads"], c["head_dim"], c["page"], c["rotary"]
    start = st["q_start"].long()
    n = st["qkv"].shape[0] - c["pad"]
    tok = torch.arange(n, device="cuda")
    seq = (tok[:, None] >= start[None, 1:]).sum(1)
    at = st["kv_len"].long()[seq] - start[seq + 1] + tok  # the token's slot in its sequence, and its position
    x = st["qkv"][:n].float()
    q, k, v = x[:, : H * D].view(n, H, D), x[:, H * D: (H + K) * D].view(n, K, D), x[:, (H + K) * D:].view(n, K, D)
    q, k = _norm(q, st["q_norm"]), _norm(k, st["k_norm"])
    angle = at.double()[:, None] * st["inv_freq"].double()[: R // 2]
    cos, sin = angle.cos().float(), angle.sin().float()
    dt = st["k_pages"].dtype
    page = st["page_table"].long()[seq, at // P]
    st["q_out"][:n] = _turn(q, cos, sin, c["half"]).to(dt).flatten(1)
    st["k_pages"][page, :, at % P] = _turn(k, cos, sin, c["half"]).to(dt)
    st["v_pages"][page, :, at % P] = v.to(dt)
    return {"q": st["q_out"], "k": st["k_pages"], "v": st["v_pages"]}


def _attend(st):
    c = st["case"]
    H, K, D, P, N = c["heads"], c["kv_heads"], c["head_dim"], c["page"], st["most_new"]
    start, kv, table = st["q_start"].long(), st["kv_len"].long(), st["page_table"].long()
    S, G = kv.shape[0], H // K
    i = torch.arange(N, device="cuda")
    tok = start[:-1, None] + i  # [S, N]
    real = tok < start[1:, None]
    pos = kv[:, None] - (start[1:] - start[:-1])[:, None] + i
    q = st["q"][tok.clamp(max=st["q"].shape[0] - 1)].float().view(S, N, K, G, D).permute(0, 2, 3, 1, 4)
    L = table.shape[1] * P
    k = st["k_pages"][table.clamp(min=0)].float().permute(0, 2, 1, 3, 4).reshape(S, K, L, D)
    s = torch.matmul(q.reshape(S, K, G * N, D), k.transpose(2, 3)).view(S, K, G, N, L) * (1.0 / math.sqrt(D))
    del k
    slot = torch.arange(L, device="cuda")
    seen = (slot <= pos[..., None]) & (table >= 0).repeat_interleave(P, 1)[:, None]  # [S, N, L]
    if c["window"]:
        seen &= slot > pos[..., None] - c["window"]
    s.masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True).clamp(min=-3e38)
    p = s.sub_(top).exp_()
    v = st["v_pages"][table.clamp(min=0)].float().permute(0, 2, 1, 3, 4).reshape(S, K, L, D)
    o = torch.matmul(p.view(S, K, G * N, L), v).view(S, K, G, N, D)
    total = p.sum(-1, keepdim=True)
    o = torch.where(total > 0, o / total, 0.0)
    o = o.permute(0, 3, 1, 2, 4).reshape(S, N, H * D)
    st["q_out"][tok[real]] = o[real].to(st["q_out"].dtype)
    return st["q_out"]


# ----------------------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    return _exact_append(st) if case["kind"] == "append" else _exact_attend(st)


def _exact_append(st):
    c = st["case"]
    new, kv = _lengths(c)
    H, K, D, P, R = c["heads"], c["kv_heads"], c["head_dim"], c["page"], c["rotary"]
    q_out, k_pages, v_pages = st["q_out"].double(), st["k_pages"].double(), st["v_pages"].double()
    first = 0
    for s, (n, m) in enumerate(zip(new, kv)):
        x = st["qkv"][first: first + n].double().view(n, H + 2 * K, D)
        out = x.clone()
        if c["norm"]:
            rms = ((x ** 2).sum(-1, keepdim=True) / D + EPS) ** 0.5
            out[:, :H] = x[:, :H] / rms[:, :H] * st["q_norm"].double()
            out[:, H: H + K] = x[:, H: H + K] / rms[:, H: H + K] * st["k_norm"].double()
        at = torch.arange(m - n, m, device="cuda")
        for j in range(R // 2):
            e, f = (j, j + R // 2) if c["half"] else (2 * j, 2 * j + 1)
            z = torch.polar(torch.ones(n, 1, dtype=torch.float64, device="cuda"),
                            at.double()[:, None] * st["inv_freq"][j].double())
            w = torch.complex(out[:, : H + K, e], out[:, : H + K, f]) * z
            out[:, : H + K, e], out[:, : H + K, f] = w.real, w.imag
        q_out[first: first + n] = out[:, :H].flatten(1)
        page = st["page_table"][s].long()[at // P]
        k_pages[page, :, at % P] = out[:, H: H + K]
        v_pages[page, :, at % P] = out[:, H + K:]
        first += n
    return {"q": q_out, "k": k_pages, "v": v_pages}


def _exact_attend(st):
    c = st["case"]
    new, kv = _lengths(c)
    H, K, D, P = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    G = H // K
    out = st["q_out"].double()
    first = 0
    for s, (n, m) in enumerate(zip(new, kv)):
        ids = st["page_table"][s, : -(-m // P)].long()
        t, p = torch.arange(m, device="cuda")[None], torch.arange(m - n, m, device="cuda")[:, None]
        hidden = (t > p) | (t <= p - (c["window"] or m + 1))
        for h in range(K):
            k = st["k_pages"][ids, h].double().reshape(-1, D)[:m]
            v = st["v_pages"][ids, h].double().reshape(-1, D)[:m]
            for a in range(h * G, (h + 1) * G):
                q = st["q"][first: first + n, a * D: (a + 1) * D].double()
                w = (q @ k.T / math.sqrt(D)).masked_fill_(hidden, -math.inf)
                w = torch.softmax(w, -1)
                out[first: first + n, a * D: (a + 1) * D] = w @ v
        first += n
    return out


def work(case):
    new, kv = _lengths(case)
    H, K, D, e = case["heads"], case["kv_heads"], case["head_dim"], SIZE[case["dtype"]]
    T = sum(new)
    if case["kind"] == "append":
        return {"bytes": T * (H + 2 * K) * D * (SIZE[case["src"]] + e) + (8 * D if case["norm"] else 0),
                "flops": T * (6 * (H + K) * D)}
    W = case["window"] or 1 << 30
    # (token, slot) pairs that the mask leaves, and the slots that any token sees
    pairs = sum(min(p + 1, W) for n, m in zip(new, kv) for p in range(m - n, m))
    slots = sum(min(m, n - 1 + W) for n, m in zip(new, kv))
    return {"bytes": 2 * T * H * D * e + 2 * slots * K * D * e, "flops": 4 * pairs * H * D}
