"""Attention over shared prefixes (yb_paged_attention_shared_dev) against the definition in 64 bits that the
tests of yb_paged_attention_dev use, with their tolerances: a prefix that is computed apart splits a row's sums
in one more place, whose join is two more products and a sum in fp32, far below the 2^-16 that is allowed for those."""
import math
import random

import pytest

from test_paged_gpu import Step, _types
from yalm_b200 import PagedBatch, YalmB200Error

pytestmark = pytest.mark.gpu


class Shared(Step):
    """A Step whose sequences from starts[g] to starts[g + 1] have the first one's pages for prefix[g] slots.  wide: its
    table is so long that sharing could save the 64 MB from which on prefixes are computed apart."""

    def __init__(self, starts, prefix, own, new, nh, nkv, hd, ps, dtype, seed, wide=True, **kw):
        import torch
        S = len(own)
        group = [next((g for g in range(len(prefix)) if starts[g] <= s < starts[g + 1]), None) for s in range(S)]
        kv = [(0 if group[s] is None else prefix[group[s]]) + own[s] + new[s] for s in range(S)]
        super().__init__(new, kv, nh, nkv, hd, ps, dtype, seed, **kw)
        for s in range(S):
            if group[s] is not None and s > starts[group[s]]:
                full = prefix[group[s]] // ps  # whole pages; the rest are each one's own, with the same contents
                first = starts[group[s]]
                own_pages = self.table[s][:full]
                self.table[s][:full] = self.table[first][:full]
                rest = prefix[group[s]] % ps
                if rest:
                    for x in (self.k, self.v):
                        x[self.table[s][full], :, :rest] = x[self.table[first][full], :, :rest]
                for page in own_pages:  # nothing may look there
                    self.k[page], self.v[page] = math.nan, math.nan
        i32 = dict(dtype=torch.int32, device="cuda")
        self.page_table = torch.tensor(self.table, **i32)
        if wide and S > 1:
            width = min(int(64e6 / ((S - 1) * nkv * hd * 4) / ps) + 1, (1 << 21) // ps)
            if width > self.page_table.shape[1]:
                more = torch.full((S, width - self.page_table.shape[1]), -1, **i32)
                self.page_table = torch.cat((self.page_table, more), 1).contiguous()
        self.group_start, self.prefix_len = torch.tensor(starts, **i32), torch.tensor(prefix, **i32)

    def attend(self, window=0, scale=None, out=None, q=None, scratch=None, batch=None):
        import torch
        assert not window
        b = batch or self.batch()
        if out is None:
            out = torch.full((self.n, self.nh * self.hd), 7.0, device="cuda").to(_types()[self.dtype])
        if scratch is None:
            scratch = torch.full((b.shared_scratch_bytes(len(self.prefix_len)),), 0xff, dtype=torch.uint8, device="cuda")
            scratch[:4] = 0
        b.attend_shared(self.q if q is None else q, out, scratch, self.group_start, self.prefix_len, scale=scale)
        torch.cuda.synchronize()
        assert int(scratch[:4].view(torch.int32)) == 0
        return out


def _ragged(n, most, seed, low=0):
    r = random.Random(seed)
    return [r.randint(low, most) for _ in range(n)]


# (groups' first sequences, prefixes, own cached slots, new tokens, heads, kv heads, head_dim, page size, type)
CASES = [
    ([0, 3], [256], [20, 0, 7], [1, 1, 1], 8, 2, 64, 16, "f16"),
    ([0, 2], [128], [0, 0], [1, 1], 8, 2, 128, 16, "f16"),
    ([0, 2], [127], [4, 0], [1, 1], 8, 2, 128, 16, "bf16"),  # less than a tile
    ([0, 2], [0], [200, 300], [1, 1], 8, 2, 128, 16, "f16"),
    ([0, 1], [1000], [20], [1], 8, 2, 128, 16, "f16"),  # a group of one
    ([0, 64], [1024], _ragged(64, 300, 1), [1] * 64, 32, 8, 128, 16, "f16"),
    ([0, 65], [1000], _ragged(65, 300, 2), [1] * 65, 32, 8, 128, 64, "bf16"),  # two units, 1000: no whole tiles
    ([0, 200], [3000], _ragged(200, 40, 3), [1] * 200, 16, 16, 128, 32, "f16"),  # no sharing of heads
    ([0, 33], [2048], _ragged(33, 100, 4), [1] * 33, 16, 1, 128, 128, "bf16"),  # 16 query heads a kv head
    ([0, 30], [1500], _ragged(30, 100, 5), [1] * 30, 12, 2, 128, 16, "f16"),  # 6: rows that fill no tile
    ([0, 24], [777], _ragged(24, 300, 6), [5] * 24, 16, 2, 64, 256, "f16"),
    ([0, 20], [900], _ragged(20, 300, 7), _ragged(20, 16, 8, 1), 8, 2, 64, 16, "bf16"),
    ([0, 20], [900], _ragged(20, 300, 9), _ragged(20, 2, 10), 8, 2, 64, 32, "f16"),  # some bring no token
    ([2, 9, 9, 30], [640, 500, 1300], _ragged(37, 200, 11), [1] * 37, 8, 2, 128, 16, "f16"),  # loose ones, a group of none
    ([0, 5, 11, 40, 41, 60], [4096, 128, 333, 2000, 700], _ragged(60, 500, 12), _ragged(60, 3, 13, 1), 64, 8, 128, 32,
     "bf16"),
    ([0, 6], [5000], [0, 0, 0, 0, 0, 0], [1] * 6, 4, 1, 128, 64, "f16"),  # few rows over many blocks
    ([0, 20], [900], _ragged(20, 300, 14), _ragged(20, 8, 15, 1), 16, 16, 128, 16, "f16"),  # up to 8 tokens of one head
    ([0, 20], [900], _ragged(20, 300, 16), _ragged(20, 8, 17, 1), 4, 4, 64, 64, "bf16"),
    ([0, 12], [700], [0] * 12, [1] * 12, 16, 2, 128, 256, "f16"),
    ([0, 3], [512], [100, 200, 0], [300, 257, 900], 8, 2, 128, 16, "f16"),  # chunks, which do not share
    ([0, 10], [2000], [100] * 10, [400] + [1] * 9, 32, 8, 128, 16, "bf16"),  # one long chunk among single tokens
    ([0, 40], [2000], [100] * 40, [200] + [1] * 39, 32, 8, 128, 16, "f16"),
]


@pytest.mark.parametrize("starts,prefix,own,new,nh,nkv,hd,ps,dtype", CASES)
def test_outputs_match_the_definition(gpu, starts, prefix, own, new, nh, nkv, hd, ps, dtype):
    Shared(starts, prefix, own, new, nh, nkv, hd, ps, dtype, seed=sum(prefix) + nh).check()


def test_many_groups_and_sequences(gpu):
    G = 2048
    starts = [2 * g for g in range(G)] + [2 * G]
    Shared(starts, [128 + 16 * (g % 9) for g in range(G)], _ragged(2 * G, 9, 1), [1] * (2 * G), 2, 1, 64, 16, "f16",
           seed=5).check()


def test_padded_rows_are_left_alone(gpu):
    st = Shared([0, 30], [600], _ragged(30, 50, 2), [1] * 30, 8, 2, 128, 16, "f16", seed=6, pad=5)
    assert (st.check()[-5:] == 7).all()


def test_row_strides(gpu):
    import torch
    st = Shared([0, 30], [600], _ragged(30, 50, 2), [2] * 30, 8, 2, 64, 16, "bf16", seed=7)
    wide = torch.full((st.n, 2 * 512), 7.0, device="cuda").to(torch.bfloat16)
    q = torch.cat((st.q, st.q), 1)[:, :512]
    got = st.attend(out=wide[:, 512:], q=q)
    assert torch.equal(got, st.attend()) and (wide[:, :512] == 7).all()


def test_pages_that_are_not_there(gpu):
    """A missing page of the prefix is missing for all, one of a sequence's own for it alone."""
    st = Shared([0, 20], [1000], _ragged(20, 300, 3, 1), [1] * 20, 8, 2, 128, 16, "f16", seed=8)
    for j in (0, 7, 8, 9, 10, 11, 12, 13, 14, 15, 33):
        for s in range(20):
            st.page_table[s, j] = -1
    st.page_table[4, 63] = st.n_pages
    st.page_table[5, :] = -1  # the table of one that is not the first: its prefix is the group's all the same
    st.page_table[5, :56] = st.page_table[0, :56]
    st.check()


def test_whole_prefix_missing(gpu):
    st = Shared([0, 20], [512], [0] * 20, [1] * 20, 8, 2, 128, 16, "f16", seed=9)
    st.page_table[:, :32] = -1
    st.page_table[3, 32] = -1  # and its one slot beside: no slot at all, zeros
    assert (st.check()[3] == 0).all()


def test_a_prefix_longer_than_what_is_cached(gpu):
    """It is cut to what all the group's sequences have before their new tokens."""
    import torch
    st = Shared([0, 20], [1024], _ragged(20, 300, 4), [1] * 20, 8, 2, 128, 16, "f16", seed=10)
    want = st.check()
    for p in (1 << 30, 5000):
        st.prefix_len.fill_(p)
        st.kv_len[7] = 700  # shorter than the prefix: its token is at slot 699
        st.kv[7] = 700
        st.check()
    st.prefix_len.fill_(-4)
    st.check()
    st.kv_len.zero_()
    st.kv = [0] * 20
    assert (st.check() == 0).all()
    assert want.shape == (20, 8 * 128)


def test_sequences_that_bring_nothing_may_come_first(gpu):
    """A group's pages are read through a row that means something: that of an ended sequence may hold anything."""
    new = [0, 0] + [1] * 18 + [0, 0, 0] + [2] * 17
    st = Shared([0, 20, 40], [1000, 700], [0, 0] + [40] * 18 + [0] * 3 + [9] * 17, new, 8, 2, 128, 16, "f16", seed=11)
    for s in range(40):
        if not new[s]:
            st.page_table[s, :] = st.n_pages + s if s % 2 else -1
            st.kv_len[s] = st.kv[s] = 0
    st.check()


def test_group_starts_out_of_range(gpu):
    import torch
    st = Shared([0, 20], [1024], _ragged(20, 300, 4), [1] * 20, 8, 2, 128, 16, "f16", seed=11)
    for starts in ([-5, 100], [0, 1 << 30], [20, 20], [25, 30]):
        st.group_start.copy_(torch.tensor(starts))
        st.check()
    # values that decrease: whatever comes out, no index leaves a buffer (by the planning kernel's own checks)
    st.group_start = torch.tensor([0, 15, 5, 20, 3], dtype=torch.int32, device="cuda")
    st.prefix_len = torch.full((4,), 1024, dtype=torch.int32, device="cuda")
    st.attend()


def test_results_repeat_and_take_a_dirty_workspace(gpu):
    import torch
    st = Shared([0, 64], [4096], _ragged(64, 600, 5), [1] * 64, 32, 8, 128, 16, "f16", seed=12)
    a = st.attend()
    b = st.batch()
    scratch = torch.randint(0, 255, (b.shared_scratch_bytes(1),), dtype=torch.uint8, device="cuda")
    scratch[:4] = 0
    for _ in range(3):
        assert torch.equal(a, st.attend(scratch=scratch))
    # the same workspace serves the form without prefixes
    out = torch.empty_like(a)
    b.attend(st.q, out, scratch)
    ref, tol = st.attend64()
    assert ((out.double() - ref).abs() <= tol).all()
    assert b.status(scratch) == 0


def test_small_batches_take_the_other_call(gpu):
    import torch
    st = Shared([0, 9], [1000], _ragged(9, 300, 6), [1] * 9, 8, 2, 128, 16, "f16", seed=16, wide=False)
    assert torch.equal(st.check().half(), Step.attend(st))
    wide = Shared([0, 9], [1000], _ragged(9, 300, 6), [1] * 9, 8, 2, 128, 16, "f16", seed=16)
    assert not torch.equal(wide.check().half(), Step.attend(st))  # (sums are split elsewhere)


def test_without_groups_it_is_the_other_call(gpu):
    import torch
    st = Shared([0], [], _ragged(9, 600, 6), [1] * 9, 8, 2, 128, 16, "f16", seed=13)
    assert torch.equal(st.attend(), Step.attend(st))


def test_replayed_graph_follows_new_lengths_and_groups(gpu):
    import torch
    S = 40
    st = Shared([0, S], [1024], _ragged(S, 600, 7), [1] * S, 16, 4, 128, 16, "bf16", seed=14)
    st.group_start = torch.tensor([0, 10, S], dtype=torch.int32, device="cuda")
    st.prefix_len = torch.tensor([1024, 1024], dtype=torch.int32, device="cuda")
    b, out = st.batch(), torch.full((S, 16 * 128), 7.0, device="cuda").to(torch.bfloat16)
    scratch = torch.zeros(b.shared_scratch_bytes(2), dtype=torch.uint8, device="cuda")
    b.attend_shared(st.q, out, scratch, st.group_start, st.prefix_len)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        b.attend_shared(st.q, out, scratch, st.group_start, st.prefix_len)
    for i, (starts, prefix) in enumerate((([0, 10, S], [1024, 512]), ([3, 30, 30], [640, 9]), ([0, 1, S], [1024, 300]))):
        st.kv = [1025 + (i * 37 + 11 * s) % (st.kv[s] - 1024) for s in range(S)]
        st.kv_len.copy_(torch.tensor(st.kv))
        st.group_start.copy_(torch.tensor(starts))
        st.prefix_len.copy_(torch.tensor(prefix))
        st.q.copy_(torch.randn(st.q.shape, generator=st.g, device="cuda"))
        g.replay()
        torch.cuda.synchronize()
        ref, tol = st.attend64()
        assert ((out.double() - ref).abs() <= tol).all()


def test_two_streams_with_a_workspace_each(gpu):
    import torch
    sts = [Shared([0, 40], [2048], _ragged(40, 400, i), [1] * 40, 16, 4, 128, 16, "f16", seed=20 + i) for i in range(2)]
    want = [st.attend() for st in sts]
    streams = [torch.cuda.Stream() for _ in sts]
    outs = [torch.zeros_like(w) for w in want]
    bs = [st.batch() for st in sts]
    work = [torch.zeros(b.shared_scratch_bytes(1), dtype=torch.uint8, device="cuda") for b in bs]
    torch.cuda.synchronize()
    for _ in range(5):
        for st, b, w, o, s in zip(sts, bs, work, outs, streams):
            with torch.cuda.stream(s):
                b.attend_shared(st.q, o, w, st.group_start, st.prefix_len)
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)


def test_refusals(gpu):
    import torch
    st = Shared([0, 4], [256], [1] * 4, [1] * 4, 8, 2, 64, 16, "f16", seed=15)
    b = st.batch()
    w = torch.zeros(b.shared_scratch_bytes(1), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(st.q)
    i32 = dict(dtype=torch.int32, device="cuda")
    for bad in (lambda: b.attend_shared(st.q, out, w[:-1], st.group_start, st.prefix_len),
                lambda: b.attend_shared(st.q, out, w, st.group_start[:1], st.prefix_len),
                lambda: b.attend_shared(st.q, out, w, st.group_start.long(), st.prefix_len),
                lambda: b.attend_shared(st.q, out, w, st.group_start, st.prefix_len.float()),
                lambda: b.attend_shared(st.q, out, w, st.group_start.cpu(), st.prefix_len),
                lambda: b.attend_shared(st.q.float(), out, w, st.group_start, st.prefix_len),
                lambda: b.attend_shared(st.q[:, :8], out, w, st.group_start, st.prefix_len)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(YalmB200Error):
        b.shared_scratch_bytes(2049)
    with pytest.raises(YalmB200Error):
        b.attend_shared(st.q, out, w, st.group_start, st.prefix_len, scale=0.0)
    many = torch.zeros(2050, **i32)
    with pytest.raises(YalmB200Error):
        b.attend_shared(st.q, out, w, many, many[:2049])


@pytest.fixture
def wait_budget():
    """Sets the clocks that a wait may take; the default comes back at the end."""
    from yalm_b200 import _lib

    def use(clocks):
        _lib.check(_lib.lib().yb_paged_attention_wait_budget(clocks))
    yield use
    use(0)


@pytest.mark.parametrize("clocks", [1, 500, 2000, 6000])
@pytest.mark.parametrize("new", [[1] * 30, [1] * 20 + [40, 300] + [1] * 8])
def test_a_wait_that_runs_out_ends_the_call(gpu, wait_budget, new, clocks):
    """In either kernel: told in the workspace's first word, with nothing in flight, and the next call is right."""
    import torch
    st = Shared([0, 30], [1500], _ragged(30, 400, 21), new, 16, 4, 128, 16, "f16", seed=22)
    b = st.batch()
    scratch = torch.zeros(b.shared_scratch_bytes(1), dtype=torch.uint8, device="cuda")
    want, out = st.check(scratch=scratch, batch=b), torch.empty_like(st.q)
    for _ in range(3):
        wait_budget(clocks)
        b.attend_shared(st.q, out, scratch, st.group_start, st.prefix_len)
        bits = b.status(scratch)
        assert bits in ((1,) if clocks == 1 else (0, 1))
        if not bits:
            assert torch.equal(out.double(), want)
        wait_budget(0)
        assert torch.equal(st.attend(scratch=scratch, batch=b).double(), want)


def test_pools_past_32_bit_offsets(gpu):
    """Pages whose elements lie past 2^31 and whose bytes lie past 2^32, of the prefix and of the sequences' own."""
    import torch
    st = Shared([0, 12], [512], _ragged(12, 300, 23, 1), [1] * 12, 16, 8, 128, 256, "f16", seed=24)
    n_pages = 11000
    k = torch.empty(n_pages, 8, 256, 128, dtype=torch.float16, device="cuda")
    v = torch.empty_like(k)
    assert k.numel() > 2 ** 31
    old = st.page_table.clone()
    for i, page in enumerate(sorted(set(old.flatten().tolist()) - {-1})):
        to = 10999 - 7 * i
        k[to], v[to] = st.k[page], st.v[page]
        st.page_table[old == page] = to
    st.k, st.v, st.n_pages = k, v, n_pages
    st.check()


@pytest.mark.parametrize("slots,hd,dtype", [(1 << 20, 64, "f16"), (300_000, 128, "bf16")])
def test_long_sums_of_few_rows(gpu, slots, hd, dtype):
    """As many loose sequences as warps have room for, over the same pages, values of one sign: a warp carries one
    row's sums over thousands of steps, which must not lose what an addition of the tensor cores cuts off."""
    import torch
    from test_paged_gpu import U
    n, ps, dt = 1300, 256, _types()[dtype]
    g = torch.Generator(device="cuda").manual_seed(25)
    pages = -(-slots // ps)
    k = (torch.randn(pages, 1, ps, hd, generator=g, device="cuda") * 0.3).to(dt)
    v = (torch.rand(pages, 1, ps, hd, generator=g, device="cuda") + 0.5).to(dt)
    i32 = dict(dtype=torch.int32, device="cuda")
    table = torch.randperm(pages, generator=g, device="cuda").int().expand(n, -1).contiguous()
    b = PagedBatch(k, v, table, torch.arange(n + 1, **i32), torch.full((n,), slots, **i32), 2, n)
    q = torch.randn(n, 2 * hd, generator=g, device="cuda").to(dt)
    out, scratch = torch.empty_like(q), torch.zeros(b.shared_scratch_bytes(1), dtype=torch.uint8, device="cuda")
    b.attend_shared(q, out, scratch, torch.tensor([0, 0], **i32), torch.zeros(1, **i32))
    assert b.status(scratch) == 0
    keys, values = (x[table[0].long(), 0].reshape(-1, hd)[:slots].double() for x in (k, v))
    for i in (0, 1, n // 2, n - 1):
        for h in range(2):
            sc = keys @ q[i, h * hd: (h + 1) * hd].double() / math.sqrt(hd)
            w = torch.softmax(sc, 0)
            mag = float((keys.abs() @ q[i, h * hd: (h + 1) * hd].double().abs()).max()) / math.sqrt(hd)
            o = w @ values
            # the weights' roundings average over the slots: the output's own, and those of the sums
            tol = U[dtype] * o.abs() + (2.0 ** -15 + 2 * 2.0 ** -20 * mag) * (w @ values.abs())
            assert ((out[i, h * hd: (h + 1) * hd].double() - o).abs() <= tol).all()
