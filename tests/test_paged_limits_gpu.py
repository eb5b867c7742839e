"""The paged-cache operators where they end: waits that run out, streams, sequences far longer than a block's share,
values that are not finite.  Plain implementations and tolerances are those of test_paged_gpu.py where nothing else is
said."""
import math

import pytest

from test_paged_gpu import Step
from yalm_b200 import _lib

pytestmark = pytest.mark.gpu


@pytest.fixture
def wait_budget():
    """Sets the clocks that a wait may take; the default comes back at the end."""
    def use(clocks):
        _lib.check(_lib.lib().yb_paged_attention_wait_budget(clocks))
    yield use
    use(0)


@pytest.mark.parametrize("clocks", [1, 500, 2000, 6000, 20000])
@pytest.mark.parametrize("new,kv,nh,nkv,hd,ps,dtype", [
    ([1, 1, 260, 300], [4000, 900, 1500, 700], 32, 8, 128, 16, "f16"),
    ([1] * 30, [700] * 30, 8, 2, 64, 64, "bf16"),
])
def test_a_wait_that_runs_out_ends_the_call(gpu, wait_budget, new, kv, nh, nkv, hd, ps, dtype, clocks):
    """The kernel gives up, says so in the workspace's first word and returns, with nothing in flight: the next call in
    the same workspace is right.  A budget of one clock always runs out: the first queries are a trip to memory away."""
    import torch
    s = Step(new, kv, nh, nkv, hd, ps, dtype, seed=91)
    b = s.batch()
    scratch = torch.zeros(b.scratch_bytes(), dtype=torch.uint8, device="cuda")
    word = scratch[:4].view(torch.int32)
    want = s.check(scratch=scratch, batch=b)
    assert int(word) == 0
    for _ in range(5):
        wait_budget(clocks)
        got = s.attend(scratch=scratch, batch=b).double()
        bits = int(word)
        assert bits in ((1,) if clocks == 1 else (0, 1))
        if not bits:
            assert torch.equal(got, want)
        wait_budget(0)
        word.zero_()
        assert torch.equal(s.attend(scratch=scratch, batch=b).double(), want)
        assert int(word) == 0


def test_status_tells_of_a_wait_that_ran_out(gpu, wait_budget):
    """Of any of the calls since the last look, on any stream, captured ones too."""
    import torch
    s = Step([40, 1], [300, 200], 8, 2, 64, 32, "f16", seed=92)
    b = s.batch()
    scratch = torch.zeros(b.scratch_bytes(), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(s.q)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    wait_budget(1)
    b.attend(s.q, out, scratch, stream=side.cuda_stream)
    wait_budget(0)
    b.attend(s.q, out, scratch, stream=side.cuda_stream)
    assert b.status(scratch) == 1
    assert b.status(scratch) == 0
    wait_budget(1)
    with torch.cuda.graph(graph):
        b.attend(s.q, out, scratch, stream=torch.cuda.current_stream().cuda_stream)
    wait_budget(0)
    assert b.status(scratch) == 0
    graph.replay()
    assert b.status(scratch) == 1
    s.check(scratch=scratch, batch=b)
    assert b.status(scratch) == 0


def test_calls_without_a_stream_run_on_torchs_current_one(gpu):
    """Inside torch.cuda.stream() and inside a capture; a long kernel before them holds their inputs back."""
    import torch
    s = Step([40, 1], [300, 200], 8, 2, 64, 32, "f16", seed=93)
    b, want = s.batch(), s.check()
    scratch = torch.zeros(b.scratch_bytes(), dtype=torch.uint8, device="cuda")
    q, out = torch.zeros_like(s.q), torch.empty_like(s.q)
    qkv, rows = torch.zeros(s.n, 768, device="cuda"), torch.randn(s.n, 768, device="cuda")
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(50_000_000)
        q.copy_(s.q)
        b.attend(q, out, scratch)
        side.synchronize()
        assert torch.equal(out.double(), want)
        torch.cuda._sleep(50_000_000)
        qkv.copy_(rows)
        b.append(qkv, out, None, 0)
        side.synchronize()
        assert torch.equal(out, rows[:, :512].half())
    out.zero_()
    with torch.cuda.graph(graph):
        b.append(qkv, q, None, 0)
        b.attend(q, out, scratch)
    torch.cuda.synchronize()
    assert not out.any()
    graph.replay()
    torch.cuda.synchronize()
    s.q = q
    ref, tol = s.attend64()
    assert ((out.double() - ref).abs() <= tol).all()


def test_steps_whose_lengths_are_advanced_on_the_device(gpu):
    """A captured step that begins by writing its own lengths and pages, replayed through page borders."""
    import torch
    nh, nkv, hd, ps, steps = 8, 2, 64, 16, 40
    s = Step([0, 0, 0], [5, 47, 130], nh, nkv, hd, ps, "f16", seed=94, spare=12)
    width = s.page_table.shape[1] + 4
    used = {p for t in s.table for p in t}
    free = [p for p in range(s.n_pages) if p not in used]
    full = [[p for p in t if p >= 0] for t in s.table]
    for t, m in zip(full, s.kv):
        while len(t) < -(-(m + steps) // ps):
            t.append(free.pop())
    table = torch.tensor([t + [-1] * (width - len(t)) for t in full], dtype=torch.int32, device="cuda")
    s.page_table = torch.full_like(table, -1)
    s.n, s.new, s.starts = 3, [1, 1, 1], [0, 1, 2, 3]
    s.q_start = torch.zeros(4, dtype=torch.int32, device="cuda")
    b = s.batch()
    qkv = torch.zeros(3, (nh + 2 * nkv) * hd, device="cuda")
    s.q = torch.zeros(3, nh * hd, device="cuda").half()
    out, scratch = torch.zeros_like(s.q), torch.zeros(b.scratch_bytes(), dtype=torch.uint8, device="cuda")
    rows = torch.randn(steps, *qkv.shape, generator=s.g, device="cuda")
    one, starts = torch.ones_like(s.kv_len), torch.arange(4, dtype=torch.int32, device="cuda")
    at = torch.arange(width, device="cuda")[None] * ps
    graph = torch.cuda.CUDAGraph()
    kv = s.kv_len.clone()
    with torch.cuda.graph(graph):
        s.q_start.copy_(starts)
        s.page_table.copy_(torch.where(at <= s.kv_len[:, None], table, -1))
        s.kv_len.add_(one)
        b.append(qkv, s.q, None, 0)
        b.attend(s.q, out, scratch)
    assert torch.equal(s.kv_len, kv)
    for i in range(steps):
        qkv.copy_(rows[i])
        graph.replay()
        torch.cuda.synchronize()
        s.kv = [m + 1 for m in s.kv]
        ref, tol = s.attend64()
        assert ((out.double() - ref).abs() <= tol).all(), i
    assert b.status(scratch) == 0


# ------------------------------------------------------------------------------------- very long caches
def _row64(q, k, v, scale, u):
    """(output, tolerance) of one query head over k, v [slots][head_dim], in 64 bits.  Beside the terms of
    test_paged_gpu.py: the tensor cores' additions need not round to nearest, so a sum is off by up to 2^-23 of it in each
    of the 1024 additions (of 16 slots) after which it is joined to the rest, and by 2^-22 in each such join (a product
    and a sum rounded to nearest); however long the cache."""
    q, k, v = q.double(), k.double(), v.double()
    sc = (k @ q) * scale
    mag = float(((k.abs() @ q.abs()) * scale).max())
    w = (sc - sc.max()).exp()
    w /= w.sum()
    o, size = w @ v, w @ v.abs()
    joins = min(k.shape[0] // 16, 1024) + 2 * (k.shape[0] // 16384)
    return o, u * o.abs() + (u + 2.0 ** -16 + 2 * 2.0 ** -20 * mag + joins * 2.0 ** -23) * size + 2.0 ** -25


def _long(slots, nkv, hd, ps, dtype, seed):
    """A cache of one sequence with values of one sign, so that a biased sum shows, in pages in random order; and its
    keys and values in the order of the slots."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = -(-slots // ps)
    k = (torch.randn(n, nkv, ps, hd, generator=g, device="cuda") * 1.4).to(dtype)
    v = (torch.rand(n, nkv, ps, hd, generator=g, device="cuda") + 0.5).to(dtype)
    order = torch.randperm(n, generator=g, device="cuda")
    table = order.to(torch.int32)[None].contiguous()

    def slots_of(x, head, lo, hi):
        a, b = lo // ps, -(-hi // ps)
        return x[order[a:b], head].reshape(-1, hd)[lo - a * ps: hi - a * ps]
    return g, k, v, table, slots_of


@pytest.mark.parametrize("slots,new,window,nh,nkv,hd,ps,dtype", [
    (200_003, 1, 0, 4, 1, 128, 16, "f16"),
    (200_003, 1, 0, 8, 2, 64, 16, "bf16"),
    (1 << 21, 1, 0, 4, 1, 128, 256, "f16"),  # the longest cache there is
    (1 << 21, 1, 0, 1, 1, 64, 16, "f16"),
    ((1 << 21) - 77, 2, 0, 16, 1, 64, 64, "bf16"),
    (1_000_003, 3, 1000, 4, 1, 128, 16, "f16"),
    (1_000_003, 3, 100_003, 4, 1, 128, 64, "f16"),
    (1 << 21, 3, 1 << 20, 8, 1, 128, 32, "bf16"),
    (1 << 21, 300, (1 << 21) - 100, 2, 2, 64, 256, "f16"),
])
def test_caches_up_to_the_longest(gpu, slots, new, window, nh, nkv, hd, ps, dtype):
    import torch
    from test_paged_gpu import U, _types
    dt = _types()[dtype]
    g, k, v, table, slots_of = _long(slots, nkv, hd, ps, dt, seed=slots % 1000 + new)
    from yalm_b200 import PagedBatch
    i32 = dict(dtype=torch.int32, device="cuda")
    b = PagedBatch(k, v, table, torch.tensor([0, new], **i32), torch.tensor([slots], **i32), nh, new)
    q = (torch.randn(new, nh * hd, generator=g, device="cuda") * 1.4).to(dt)
    out, scratch = torch.full_like(q, 7.0), torch.zeros(b.scratch_bytes(), dtype=torch.uint8, device="cuda")
    b.attend(q, out, scratch, window=window)
    assert b.status(scratch) == 0
    for i in sorted({0, new // 2, new - 1}):
        for h in sorted({0, nh // 2, nh - 1}):
            p = slots - new + i
            lo = max(0, p - window + 1) if window else 0
            o, tol = _row64(q[i, h * hd: (h + 1) * hd], slots_of(k, h * nkv // nh, lo, p + 1),
                            slots_of(v, h * nkv // nh, lo, p + 1), 1 / math.sqrt(hd), U[dtype])
            err = (out[i, h * hd: (h + 1) * hd].double() - o).abs()
            assert (err <= tol).all(), (i, h, float((err / tol).max()))


@pytest.mark.parametrize("slots,hd,dtype", [(120_000, 128, "f16"), (120_000, 64, "bf16"), (1 << 20, 128, "bf16"),
                                            (1 << 21, 64, "f16")])
def test_long_units_that_no_cut_shortens(gpu, slots, hd, dtype):
    """As many sequences as blocks over the same pages: each block carries one row's sums over the whole cache."""
    import torch
    from test_paged_gpu import U, _types
    from yalm_b200 import PagedBatch
    dt, n = _types()[dtype], _lib.lib().yb_num_sms()
    g, k, v, table, slots_of = _long(slots, 1, hd, 64, dt, seed=hd)
    i32 = dict(dtype=torch.int32, device="cuda")
    b = PagedBatch(k, v, table.expand(n, -1).contiguous(), torch.arange(n + 1, **i32),
                   torch.full((n,), slots, **i32), 2, n)
    q = (torch.randn(n, 2 * hd, generator=g, device="cuda") * 1.4).to(dt)
    out, scratch = torch.full_like(q, 7.0), torch.zeros(b.scratch_bytes(), dtype=torch.uint8, device="cuda")
    b.attend(q, out, scratch)
    assert b.status(scratch) == 0
    keys, values = slots_of(k, 0, 0, slots), slots_of(v, 0, 0, slots)
    for i in (0, 1, n // 2, n - 1):
        for h in range(2):
            o, tol = _row64(q[i, h * hd: (h + 1) * hd], keys, values, 1 / math.sqrt(hd), U[dtype])
            err = out[i, h * hd: (h + 1) * hd].double() - o
            assert (err.abs() <= tol).all(), (i, h, float((err.abs() / tol).max()))


@pytest.mark.parametrize("nh,window", [(1, 0), (16, 300)])
def test_as_many_tokens_as_there_may_be(gpu, nh, window):
    """A prompt of 2^20 tokens, appended and attended to: sampled rows."""
    import torch
    from test_paged_gpu import U
    from yalm_b200 import PagedBatch
    n, hd, ps = 1 << 20, 64, 256
    i32 = dict(dtype=torch.int32, device="cuda")
    g, k, v, table, slots_of = _long(n, 1, hd, ps, torch.float16, seed=nh)
    k.zero_()
    v.zero_()
    b = PagedBatch(k, v, table, torch.tensor([0, n], **i32), torch.tensor([n], **i32), nh, n)
    qkv = torch.randn(n, (nh + 2) * hd, generator=g, device="cuda", dtype=torch.float16)
    qkv[:, (nh + 1) * hd:] = qkv[:, (nh + 1) * hd:].abs()
    q = torch.empty(n, nh * hd, device="cuda", dtype=torch.float16)
    inv = torch.tensor([1e6 ** (-2.0 * j / hd) for j in range(hd // 2)], device="cuda")
    b.append(qkv, q, inv, hd, clip=3.0)
    rows = sorted({0, 1, 255, 256, 65535, 65536, n // 2, n - 257, n - 1} |
                  set(torch.randint(0, n, (12,), generator=g, device="cuda").tolist()))
    at = torch.tensor(rows, device="cuda")
    x = qkv[at].double().clamp(-3, 3).view(-1, nh + 2, hd)
    a, c = x[:, : nh + 1, 0::2], x[:, : nh + 1, 1::2]
    ang = at.double()[:, None, None] * inv.double()
    want = torch.stack((a * ang.cos() - c * ang.sin(), a * ang.sin() + c * ang.cos()), -1).flatten(-2)
    size = torch.stack((a.abs() + c.abs(),) * 2, -1).flatten(-2)
    tol = U["f16"] * want.abs() + 2.0 ** -18 * size + 2.0 ** -25
    assert ((q[at].double().view(-1, nh, hd) - want[:, :nh]).abs() <= tol[:, :nh]).all()
    key, value = slots_of(k, 0, 0, n)[at].double(), slots_of(v, 0, 0, n)[at]
    assert ((key - want[:, nh]).abs() <= tol[:, nh]).all()
    assert torch.equal(value, qkv[at, (nh + 1) * hd:].clamp(-3, 3))
    out, scratch = torch.full_like(q, 7.0), torch.zeros(b.scratch_bytes(), dtype=torch.uint8, device="cuda")
    b.attend(q, out, scratch, window=window)
    assert b.status(scratch) == 0
    keys, values = slots_of(k, 0, 0, n), slots_of(v, 0, 0, n)
    for p in rows:
        lo = max(0, p - window + 1) if window else 0
        for h in sorted({0, nh - 1}):
            o, tol = _row64(q[p, h * hd: (h + 1) * hd], keys[lo: p + 1], values[lo: p + 1], 1 / math.sqrt(hd), U["f16"])
            err = out[p, h * hd: (h + 1) * hd].double() - o
            assert (err.abs() <= tol).all(), (p, h, float((err.abs() / tol).max()))


@pytest.mark.parametrize("dtype,hd", [("f16", 64), ("f16", 128), ("bf16", 128)])
@pytest.mark.parametrize("slots,top_at,second", [(1 << 20, 5, 0), (1 << 20, (1 << 20) - 3, 0), (300_000, 299_000, 7.9),
                                                 (700, 3, 0)])
def test_many_small_weights_beside_a_large_one(gpu, dtype, hd, slots, top_at, second):
    """Weights of 2^-20 to 2^-33 of the largest, which together are up to a fifth of it; the largest comes first, last, or
    after one (2^-7.9 of it) whose maximum then serves for the rest.  Tolerance: in fp16 a weight below 2^-21 of that maximum
    is rounded by up to 2^-32 of it, which the other terms, relative to each weight, do not hold."""
    import torch
    from test_paged_gpu import U, _types
    from yalm_b200 import PagedBatch
    dt = _types()[dtype]
    g, k, v, table, slots_of = _long(slots, 1, hd, 64, dt, seed=slots % 97 + hd)
    score = torch.rand(slots, generator=g, device="cuda") * 13 + 20
    if second:
        score[: slots // 100] = 40.0
        score[slots // 100] = second
    score[top_at] = 0.0
    k.zero_()
    at = torch.arange(slots, device="cuda")
    k[table[0].long()[at // 64], 0, at % 64, 0] = (score * -math.log(2)).to(dt)
    i32 = dict(dtype=torch.int32, device="cuda")
    b = PagedBatch(k, v, table, torch.tensor([0, 1], **i32), torch.tensor([slots], **i32), 2, 1)
    q = torch.zeros(1, 2 * hd, device="cuda", dtype=dt)
    q[0, 0], q[0, hd] = 8.0, 16.0  # the second head: all weights squared
    out, scratch = torch.full_like(q, 7.0), torch.zeros(b.scratch_bytes(), dtype=torch.uint8, device="cuda")
    b.attend(q, out, scratch, scale=0.125)
    assert b.status(scratch) == 0
    keys, values = slots_of(k, 0, 0, slots), slots_of(v, 0, 0, slots)
    for h in range(2):
        qh = q[0, h * hd: (h + 1) * hd]
        o, tol = _row64(qh, keys, values, 0.125, U[dtype])
        if dtype == "f16":
            s = (keys.double() @ qh.double()) * 0.125
            tol = tol + slots * 2.0 ** -32 * float(values.max()) / float((s - s.max()).exp().sum())
        err = (out[0, h * hd: (h + 1) * hd].double() - o).abs()
        assert (err <= tol).all(), (h, float((err / tol).max()))


@pytest.mark.parametrize("busy", [[0, 1, 40_000, 65_535], [65_535], None])
def test_as_many_sequences_as_there_may_be(gpu, busy):
    """2^16 sequences of up to 40 slots: a few with one new token (none in the rest), or all of them."""
    import torch
    from test_paged_gpu import U
    from yalm_b200 import PagedBatch
    n, nh, nkv, hd, ps = 1 << 16, 4, 2, 64, 16
    g = torch.Generator(device="cuda").manual_seed(95)
    i32 = dict(dtype=torch.int32, device="cuda")
    new = torch.ones(n, **i32) if busy is None else torch.zeros(n, **i32).index_fill_(0, torch.tensor(busy, device="cuda"), 1)
    kv = torch.randint(1, 41, (n,), generator=g, **i32)
    start = torch.cat((torch.zeros(1, **i32), new.cumsum(0, dtype=torch.int32)))
    T = int(start[-1])
    pages = 3 * n
    table = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).view(n, 3)
    k, v = (torch.randn(pages, nkv, ps, hd, generator=g, device="cuda", dtype=torch.float16) for _ in range(2))
    b = PagedBatch(k, v, table, start, kv, nh, T + 1)
    qkv = torch.randn(T + 1, (nh + 2 * nkv) * hd, generator=g, device="cuda", dtype=torch.float16)
    q = torch.full((T + 1, nh * hd), 7.0, device="cuda", dtype=torch.float16)
    out, scratch = q.clone(), torch.zeros(b.scratch_bytes(), dtype=torch.uint8, device="cuda")
    b.append(qkv, q, None, 0)
    b.attend(q, out, scratch)
    assert b.status(scratch) == 0
    assert (out[T] == 7).all() and torch.equal(q[:T], qkv[:T, : nh * hd]) and (q[T] == 7).all()
    seqs = new.nonzero().flatten()
    seqs = seqs[torch.linspace(0, T - 1, min(T, 500), device="cuda").long()]
    for s in seqs.tolist():
        m, row = int(kv[s]), int(start[s])
        own_k, own_v = (x[table[s].long()].transpose(1, 2).reshape(-1, nkv, hd)[:m] for x in (k, v))
        assert torch.equal(own_k[m - 1].flatten(), qkv[row, nh * hd: (nh + nkv) * hd])
        assert torch.equal(own_v[m - 1].flatten(), qkv[row, (nh + nkv) * hd:])
        for h in range(nh):
            o, tol = _row64(q[row, h * hd: (h + 1) * hd], own_k[:, h // 2], own_v[:, h // 2], 1 / math.sqrt(hd), U["f16"])
            err = (out[row, h * hd: (h + 1) * hd].double() - o).abs()
            assert (err <= tol).all(), (s, h, float((err / tol).max()))


# ---------------------------------------------------------------------------------------------- append
@pytest.mark.parametrize("hd,R,half", [(128, 128, False), (128, 128, True), (128, 96, False), (128, 96, True), (64, 8, False),
                                       (64, 8, True), (64, 62, False), (64, 0, False), (64, 0, True), (128, 0, True)])
@pytest.mark.parametrize("src,dtype", [("f32", "f16"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("norms", ["", "q", "k", "qk"])
def test_append_with_either_norm_and_values_that_are_not_finite(gpu, hd, R, half, src, dtype, norms):
    """One norm without the other, half-split pairs over nothing; infinities and NaN spoil what the definition says
    they do: without a norm their pair, or themselves alone where nothing is rotated, with one their head (an infinity
    makes the finite ones 0)."""
    import torch
    from test_paged_gpu import _append64, _types
    nh, nkv, ps, n = 6, 3, 16, 40
    s = Step([n], [n + 70], nh, nkv, hd, ps, dtype, seed=hd + R)
    g = s.g
    qkv = (torch.randn(n, (nh + 2 * nkv) * hd, generator=g, device="cuda") * 2).to(_types()[src])
    for bad in (math.inf, -math.inf, math.nan):
        where = torch.randint(0, qkv.numel(), (24,), generator=g, device="cuda")
        qkv.view(-1)[where] = bad
    w = 1 + 0.3 * torch.randn(2, hd, generator=g, device="cuda")
    qn, kn = (w[0].clone() if "q" in norms else None), (w[1].clone() if "k" in norms else None)
    inv = torch.tensor([1e4 ** (-2.0 * j / max(R, 1)) for j in range(R // 2)] or [0.0], device="cuda")
    pos = torch.randint(1, 5000, (n,), dtype=torch.int32, generator=g, device="cuda")
    q = torch.empty_like(s.q)
    s.batch().append(qkv, q, inv if R else None, R, q_norm=qn, k_norm=kn, eps=1e-6, half=half, pos=pos)
    torch.cuda.synchronize()
    ref, tol = _append64(s, qkv, qn, kn, 1e-6, inv, R, half, pos, math.inf)
    slot = torch.arange(70, 70 + n, device="cuda")
    page = s.page_table[0].long()[slot // ps]
    got = torch.cat((q.view(n, nh, hd), s.k[page, :, slot % ps], s.v[page, :, slot % ps]), 1).double()
    assert torch.equal(got.isnan(), ref.isnan())
    assert torch.equal(got.isinf(), ref.isinf()) and torch.equal(got[got.isinf()], ref[ref.isinf()])
    fine = ref.isfinite()
    assert fine.float().mean() > 0.3 and not fine.all()
    assert ((got - ref).abs()[fine] <= tol[fine]).all()
