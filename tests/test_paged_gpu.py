"""The paged-cache append and attention kernels (yb_paged_append_dev, yb_paged_attention_dev) against their
definitions computed in 64 bits, sequence by sequence and head by head.

Tolerances, with u = half a step of the output type (2^-11 fp16, 2^-8 bf16, relative) and 2^-25 for the
fp16 outputs below the normal range:
 - append: one rounding u to the type; before it norm, angle and rotation in fp32: the square sum of up
   to 128 terms (pairwise over a warp: under 2^-20 relative with the root and the division), sine and cosine
   of an angle reduced in 64 bits (2^-22), two products and a sum: 2^-18 of the pair's magnitude covers it.
   Values are neither normed nor rotated: their one rounding alone.
 - attention: the output's rounding u; each probability's rounding to the type, u of sum w|v|; scores
   summed in fp32 over head_dim products, 2^-20 of scale * sum |q k| absolute, which is that much relative in
   a weight; exponentials and the sums over the slots in fp32, 2^-16 of sum w|v| together."""
import math

import pytest

from yalm_b200 import PagedBatch, YalmB200Error

pytestmark = pytest.mark.gpu

U = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = 2.0 ** -25


def _types():
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


class Step:
    """A batch of sequences with `new` new tokens and kv cached slots each, in pages handed out in random
    order from a pool that holds NaN wherever nothing was stored."""

    def __init__(self, new, kv, nh, nkv, hd, ps, dtype, seed, pad=0, spare=3, gain=1.4):
        import torch
        self.new, self.kv, self.nh, self.nkv, self.hd, self.ps, self.dtype = new, kv, nh, nkv, hd, ps, dtype
        g = self.g = torch.Generator(device="cuda").manual_seed(seed)
        dt = _types()[dtype]
        need = [-(-n // ps) for n in kv]
        self.n_pages = sum(need) + spare
        order = torch.randperm(self.n_pages, generator=g, device="cuda").tolist()
        width = max(need + [1]) + 1
        self.table = [[order.pop() for _ in range(n)] + [-1] * (width - n) for n in need]
        self.n = sum(new) + pad
        self.k = torch.full((self.n_pages, nkv, ps, hd), math.nan, device="cuda").to(dt)
        self.v = self.k.clone()
        for s, m in enumerate(kv):
            for t0 in range(0, m, ps):
                c = min(ps, m - t0)
                for x, sd in ((self.k, gain), (self.v, 1.0)):
                    x[self.table[s][t0 // ps], :, :c] = (torch.randn(nkv, c, hd, generator=g, device="cuda") * sd).to(dt)
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        self.starts = starts
        i32 = dict(dtype=torch.int32, device="cuda")
        self.q_start, self.kv_len = torch.tensor(starts, **i32), torch.tensor(kv, **i32)
        self.page_table = torch.tensor(self.table, **i32)
        self.q = (torch.randn(self.n, nh * hd, generator=g, device="cuda") * gain).to(dt)

    def batch(self, **kw):
        a = dict(k_pages=self.k, v_pages=self.v, page_table=self.page_table, q_start=self.q_start, kv_len=self.kv_len,
                 n_heads=self.nh, n_tokens=self.n)
        a.update(kw)
        return PagedBatch(**a)

    def attend(self, window=0, scale=None, out=None, q=None, scratch=None, batch=None):
        import torch
        b = batch or self.batch()
        if out is None:
            out = torch.full((self.n, self.nh * self.hd), 7.0, device="cuda").to(_types()[self.dtype])
        if scratch is None:
            scratch = torch.zeros(b.scratch_bytes(), dtype=torch.uint8, device="cuda")
        b.attend(self.q if q is None else q, out, scratch, window=window, scale=scale,
                 stream=torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        return out

    def attend64(self, window=0, scale=None):
        """(outputs, tolerance) in 64 bits; rows of no sequence are left at 7."""
        import torch
        scale = 1 / math.sqrt(self.hd) if scale is None else scale
        G, u = self.nh // self.nkv, U[self.dtype]
        out = torch.full((self.n, self.nh, self.hd), 7.0, dtype=torch.float64, device="cuda")
        tol = torch.zeros_like(out)
        qd = self.q.double().view(self.n, self.nh, self.hd)
        for s, (n, m) in enumerate(zip(self.new, self.kv)):
            if n == 0:
                continue
            r = slice(self.starts[s], self.starts[s] + n)
            ids = self.page_table[s].long()
            here = ((ids >= 0) & (ids < self.n_pages)).repeat_interleave(self.ps)[:m]
            ids = torch.where((ids >= 0) & (ids < self.n_pages), ids, 0)
            p = torch.arange(m - n, m, device="cuda")[:, None]
            t = torch.arange(m, device="cuda")[None]
            seen = (t <= p) & here[None]
            if window:
                seen &= t > p - window
            for h in range(self.nh):
                k = self.k[ids, h // G].double().reshape(-1, self.hd)[:m]
                v = self.v[ids, h // G].double().reshape(-1, self.hd)[:m]
                k, v = torch.where(here[:, None], k, 0.0), torch.where(here[:, None], v, 0.0)
                sc = (qd[r, h] @ k.T) * scale
                mag = ((qd[r, h].abs() @ k.abs().T) * scale * seen).amax(-1, keepdim=True) if m else sc.new_zeros(n, 1)
                sc = sc.masked_fill(~seen, -math.inf)
                top = sc.amax(-1, keepdim=True).clamp(min=-1e300) if m else sc.new_zeros(n, 1)
                w = (sc - top).exp()
                tot = w.sum(-1, keepdim=True)
                w = torch.where(tot > 0, w / tot, 0.0)
                o = w @ v
                out[r, h] = o
                tol[r, h] = u * o.abs() + (u + 2.0 ** -16 + 2 * 2.0 ** -20 * mag) * (w @ v.abs()) + TINY
        return out.flatten(1), tol.flatten(1)

    def check(self, window=0, scale=None, **kw):
        got = self.attend(window, scale, **kw).double()
        ref, tol = self.attend64(window, scale)
        err = (got - ref).abs()
        assert not err.isnan().any()
        assert (err <= tol).all(), (float((err / tol.clamp(min=TINY)).max()), float(err.max()))
        return got


# (new tokens, cached slots with them, heads, kv heads, head_dim, page size, type, window)
ATTEND = [
    ([1], [1], 8, 2, 64, 16, "f16", 0),  # the first token of all
    ([1], [37], 8, 2, 64, 16, "bf16", 0),
    ([1], [128], 32, 8, 128, 128, "f16", 0),  # exactly a tile
    ([1], [129], 32, 8, 128, 256, "f16", 0),
    ([1], [5000], 32, 8, 128, 64, "f16", 0),  # one row split over many blocks
    ([1], [5000], 4, 1, 128, 16, "bf16", 0),
    ([1, 1, 1], [300, 17, 1025], 16, 16, 128, 32, "f16", 0),  # no sharing of heads
    ([1] * 40, [3 + 97 * i for i in range(40)], 8, 2, 128, 16, "bf16", 0),
    ([1] * 300, [1 + (i * 7) % 50 for i in range(300)], 8, 2, 64, 16, "f16", 0),  # more sequences than threads of a warp
    ([5], [5], 8, 2, 64, 16, "f16", 0),
    ([77], [77], 32, 8, 128, 16, "f16", 0),
    ([256], [256], 8, 8, 128, 64, "bf16", 0),
    ([257], [1000], 8, 2, 128, 32, "f16", 0),
    ([1000], [1000], 8, 2, 64, 64, "f16", 0),
    ([513], [3202], 32, 8, 128, 16, "f16", 0),
    ([130, 1, 0, 64, 1], [130, 900, 40, 700, 1], 64, 8, 128, 32, "bf16", 0),  # mixed, one sequence without new tokens
    ([0, 0, 3, 0], [0, 10, 3, 5], 8, 2, 64, 16, "f16", 0),
    ([60, 33], [61, 200], 12, 2, 128, 32, "f16", 0),  # six heads share one
    ([50], [90], 5, 1, 64, 16, "bf16", 0),
    ([50], [90], 16, 1, 64, 16, "f16", 0),
    ([40, 1], [700, 700], 9, 3, 128, 16, "f16", 0),
    ([1, 1], [700, 5], 32, 8, 128, 16, "f16", 100),  # windows
    ([300], [300], 8, 2, 64, 64, "f16", 1),
    ([300], [900], 8, 2, 128, 16, "bf16", 130),
    ([700, 1, 20], [700, 2000, 600], 32, 8, 128, 32, "f16", 333),
    ([4, 9], [2, 5], 8, 2, 64, 16, "f16", 0),  # fewer slots than tokens: the first tokens see none
    ([300], [7], 8, 2, 128, 16, "f16", 0),
    ([2], [0], 8, 2, 128, 16, "f16", 0),  # an empty cache
]


@pytest.mark.parametrize("new,kv,nh,nkv,hd,ps,dtype,window", ATTEND)
def test_attention_matches_64_bits(gpu, new, kv, nh, nkv, hd, ps, dtype, window):
    Step(new, kv, nh, nkv, hd, ps, dtype, seed=len(new) + kv[0], pad=2).check(window)


@pytest.mark.parametrize("hd,ps,dtype", [(128, 16, "f16"), (64, 256, "bf16")])
def test_pages_that_are_not_there_are_masked(gpu, hd, ps, dtype):
    """Entries outside [0, n_pages) in the middle of a sequence, over its first slots and over all of them."""
    import torch
    s = Step([1, 70, 33, 1], [800, 1100, 33, 600], 8, 2, hd, ps, dtype, seed=5)
    t = s.page_table
    for row, lo, hi in ((0, 1, 3), (1, 0, 2), (1, 3, 4), (2, 0, 3)):
        t[row, lo:hi] = -1
    t[1, 2] = s.n_pages
    t[3, :] = 2 ** 31 - 1
    s.check()
    got = s.check(window=150)
    assert (got[104] == 0).all()  # the last sequence has no page: zeros
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("new,kv,window,hd,ps", [([1], [1000], 100, 128, 16), ([90, 1], [700, 333], 130, 64, 64),
                                                 ([200], [2000], 7, 128, 256)])
def test_slots_before_the_first_window_may_hold_anything(gpu, new, kv, window, hd, ps):
    import torch
    s = Step(new, kv, 8, 2, hd, ps, "f16", seed=63)
    ref, tol = s.attend64(window)
    for row, (n, m) in enumerate(zip(new, kv)):
        for t in range(m - n - window + 1):
            s.k[s.table[row][t // ps], :, t % ps] = math.nan
            s.v[s.table[row][t // ps], :, t % ps] = math.inf if t % 2 else math.nan
    got = s.attend(window).double()
    assert ((got - ref).abs() <= tol).all()


def test_large_scores_and_other_scales(gpu):
    """Scores of several hundred, where only the differences to the row's maximum matter; rising along the
    cache, so that the running maximum keeps growing; another scale."""
    import torch
    s = Step([1, 200], [3000, 700], 8, 2, 128, 32, "bf16", seed=9, gain=8.0)
    s.check()
    s.check(scale=0.01)
    s = Step([64], [2048], 8, 2, 128, 32, "f16", seed=10)
    ramp = torch.linspace(0.0, 8.0, 2048, device="cuda")
    for t0 in range(0, 2048, 32):
        s.k[s.table[0][t0 // 32]] = ramp[t0:t0 + 32, None].expand(2, 32, 128).half()
    s.q.fill_(1.0)
    s.check()


def test_strided_rows_and_untouched_rows(gpu):
    """q and out as column ranges of wider tensors; rows behind the last sequence and the columns beside stay."""
    import torch
    s = Step([3, 100], [50, 333], 8, 2, 64, 16, "f16", seed=21, pad=5)
    wide_q = torch.randn(s.n, 512 + 256, device="cuda").half()
    wide_q[:, 128:640] = s.q
    wide_o = torch.full((s.n, 1024), 7.0, device="cuda").half()
    s.q = wide_q[:, 128:640]
    s.check(q=s.q, out=wide_o[:, 256:768])
    assert (wide_o[:, :256] == 7).all() and (wide_o[:, 768:] == 7).all()
    assert (wide_o[s.starts[-1]:] == 7).all()


def test_rows_before_the_first_sequence_stay(gpu):
    import torch
    s = Step([3, 9], [50, 33], 8, 2, 64, 16, "f16", seed=22, pad=4)
    s.starts = [4, 7, 16]
    s.q_start.copy_(torch.tensor(s.starts))
    got = s.check()
    assert (got[:4] == 7).all()


def test_attention_is_deterministic_and_leaves_its_workspace_ready(gpu):
    import torch
    s = Step([1, 1, 260], [4000, 900, 1500], 32, 8, 128, 16, "bf16", seed=31)
    b = s.batch()
    scratch = torch.zeros(b.scratch_bytes(), dtype=torch.uint8, device="cuda")
    first = s.attend(scratch=scratch, batch=b)
    other = Step([1] * 7, [2000] * 7, 8, 2, 128, 32, "f16", seed=32)
    assert b.scratch_bytes() == other.batch().scratch_bytes()
    for _ in range(20):
        other.check(scratch=scratch)
        assert torch.equal(s.attend(scratch=scratch, batch=b), first)


def test_attention_in_a_graph_follows_new_lengths(gpu):
    """A captured launch replayed after the lengths, the table and the rows changed: the kernel reads them
    when it runs.  On a stream that is not the default one."""
    import torch
    s = Step([1, 40, 1], [900, 500, 2000], 8, 2, 128, 16, "f16", seed=41, pad=30)
    b = s.batch()
    scratch = torch.zeros(b.scratch_bytes(), dtype=torch.uint8, device="cuda")
    out = torch.full((s.n, 1024), 7.0, device="cuda").half()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        b.attend(s.q, out, scratch, stream=torch.cuda.current_stream().cuda_stream)
    for new, kv in (([1, 40, 1], [900, 500, 2000]), ([30, 1, 30], [777, 500, 130]), ([0, 0, 70], [3, 5, 1999]),
                    ([1, 1, 1], [1, 1, 1])):
        s.new, s.kv = new, kv
        s.starts = [0, new[0], new[0] + new[1], sum(new)]
        s.q_start.copy_(torch.tensor(s.starts))
        s.kv_len.copy_(torch.tensor(kv))
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        ref, tol = s.attend64()
        assert ((out.double() - ref).abs() <= tol).all(), (new, kv)


def test_lengths_out_of_range_stay_inside_the_buffers(gpu):
    """q_start and kv_len outside what the header allows are clamped: nothing outside is touched, the other
    sequences are right."""
    import torch
    s = Step([4, 3, 5], [40, 30, 48], 8, 2, 64, 16, "f16", seed=51)
    guard = torch.full((3 * s.n, 512), 7.0, device="cuda").half()
    out = guard[s.n: 2 * s.n]
    s.kv_len[1] = -5
    s.q_start[3] = 10 ** 6  # clamped to the 12 rows there are
    s.new, s.kv = [4, 3, 5], [40, 0, 48]
    s.check(out=out)
    assert (guard[: s.n] == 7).all() and (guard[2 * s.n:] == 7).all()
    s.q_start.copy_(torch.tensor([7, 3, -4, 12]))  # not increasing: any rows, but inside
    s.kv_len.copy_(torch.tensor([40, 10 ** 9, 48]))
    s.attend(out=out)
    assert (guard[: s.n] == 7).all() and (guard[2 * s.n:] == 7).all()


def test_rows_do_not_touch_each_other(gpu):
    """A query that is not finite spoils its own head's row alone."""
    import torch
    s = Step([70, 1], [300, 200], 8, 2, 128, 16, "f16", seed=55)
    clean = s.attend()
    s.q[5, 3 * 128] = math.nan
    s.q[69, 0] = math.inf
    s.q[70, 7 * 128 + 5] = -math.inf
    got = s.attend().view(s.n, 8, 128)
    bad = torch.zeros(s.n, 8, dtype=torch.bool, device="cuda")
    bad[5, 3] = bad[69, 0] = bad[70, 7] = True
    assert got[5, 3].isnan().all()
    assert torch.equal(got[~bad], clean.view(s.n, 8, 128)[~bad])


def test_sequences_share_a_prefix(gpu):
    """Two sequences whose first pages are the same ones."""
    s = Step([40, 3], [500, 300], 8, 2, 64, 32, "bf16", seed=56)
    for i in range(8):
        s.table[1][i] = s.table[0][i]
    s.page_table[1, :8] = s.page_table[0, :8]
    s.check()
    s.check(window=77)


def test_many_sequences(gpu):
    """More sequences than a block has threads, most of them without new tokens."""
    n = 3000
    new = [1 if i % 7 == 0 else 0 for i in range(n)]
    new[1234] = 150
    kv = [1 + (i * 13) % 40 for i in range(n)]
    kv[1234] = 400
    Step(new, kv, 4, 2, 64, 16, "f16", seed=57).check()


def test_pools_past_32_bit_offsets(gpu):
    """Pages whose elements lie past 2^31 and whose bytes lie past 2^32, for the reads and the stores."""
    import torch
    nh, nkv, hd, ps, n_pages = 16, 8, 128, 256, 11000  # 2.9e9 elements in either cache
    k = torch.empty(n_pages, nkv, ps, hd, dtype=torch.float16, device="cuda")
    v = torch.empty_like(k)
    assert k.numel() > 2 ** 31
    s = Step([3, 80], [600, 300], nh, nkv, hd, ps, "f16", seed=58)
    old, far = [list(t) for t in s.table], [10999, 8192, 8193, 10500, 2]
    for row in range(2):
        for i, page in enumerate(old[row]):
            if page >= 0:
                to = far.pop()
                k[to], v[to] = s.k[page], s.v[page]
                s.table[row][i] = to
    s.k, s.v, s.n_pages = k, v, n_pages
    s.page_table.copy_(torch.tensor(s.table))
    s.check()
    qkv = torch.randn(s.n, (nh + 2 * nkv) * hd, device="cuda")
    out = torch.empty_like(s.q)
    s.batch().append(qkv, out, None, 0, stream=torch.cuda.current_stream().cuda_stream)
    for at, (row, slot) in enumerate([(0, t) for t in (597, 598, 599)] + [(1, t) for t in range(220, 300)]):
        page, r = s.table[row][slot // ps], slot % ps
        want = qkv[at].half().view(nh + 2 * nkv, hd)
        assert torch.equal(k[page, :, r], want[nh: nh + nkv]) and torch.equal(v[page, :, r], want[nh + nkv:])
    assert torch.equal(out, qkv[:, : nh * hd].half())


def test_two_streams_at_once(gpu):
    """Calls on two streams, each with its own workspace."""
    import torch
    a = Step([1] * 5, [3000] * 5, 32, 8, 128, 16, "f16", seed=59)
    b = Step([300], [1200], 8, 2, 64, 64, "bf16", seed=60)
    want = [x.attend() for x in (a, b)]
    runs = []
    for x in (a, b):
        batch = x.batch()
        runs.append((x, batch, torch.zeros(batch.scratch_bytes(), dtype=torch.uint8, device="cuda"),
                     [torch.full_like(want[len(runs)], 7.0) for _ in range(20)], torch.cuda.Stream()))
    torch.cuda.synchronize()
    for i in range(20):
        for x, batch, scratch, outs, stream in runs:
            batch.attend(x.q, outs[i], scratch, stream=stream.cuda_stream)
    torch.cuda.synchronize()
    for w, run in zip(want, runs):
        assert all(torch.equal(w, o) for o in run[3])


def test_workspace_needs_no_initial_value(gpu):
    import torch
    s = Step([1, 130], [4000, 900], 32, 8, 128, 32, "f16", seed=62)
    b = s.batch()
    s.check(scratch=torch.full((b.scratch_bytes(),), 0xFF, dtype=torch.uint8, device="cuda"), batch=b)


def test_host_memory_is_refused(gpu):
    import torch
    s = Step([2], [20], 8, 2, 64, 16, "f16", seed=61)
    b = s.batch()
    scratch = torch.zeros(b.scratch_bytes(), dtype=torch.uint8, device="cuda")
    b.c.kv_len_dev = torch.tensor([20], dtype=torch.int32).data_ptr()
    with pytest.raises(YalmB200Error):
        b.attend(s.q, torch.empty_like(s.q), scratch)
    with pytest.raises(YalmB200Error):
        b.append(torch.zeros(2, 768, device="cuda"), s.q, torch.zeros(32, device="cuda"), 64)


# ---------------------------------------------------------------------------------------------- append
def _append64(s, qkv, qn, kn, eps, inv, R, half, pos, clip):
    """(q, {(page, head, row): (k, v)}, ...) in 64 bits: q rows, k and v rows, and each one's tolerance."""
    import torch
    H, K, D, u = s.nh, s.nkv, s.hd, U[s.dtype]
    x = qkv.double().clamp(-clip, clip).view(s.n, H + 2 * K, D)
    y = x.clone()
    for lo, hi, w in ((0, H, qn), (H, H + K, kn)):
        if w is not None:
            y[:, lo:hi] = x[:, lo:hi] / (x[:, lo:hi].square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    mag = y.abs().clone()
    j = torch.arange(R // 2, device="cuda")
    e, f = (j, j + R // 2) if half else (2 * j, 2 * j + 1)
    ang = pos.double()[:, None] * inv.double()[: R // 2]
    c, sn = ang.cos()[:, None], ang.sin()[:, None]
    a, b = y[:, : H + K, e].clone(), y[:, : H + K, f].clone()
    y[:, : H + K, e], y[:, : H + K, f] = a * c - b * sn, a * sn + b * c
    mag[:, : H + K, e] = a.abs() + b.abs()
    mag[:, : H + K, f] = a.abs() + b.abs()
    tol = u * y.abs() + 2.0 ** -18 * mag + TINY
    tol[:, H + K:] = u * y[:, H + K:].abs() + TINY
    return y, tol


APPEND = [
    ([1], [37], 8, 2, 64, 16, "f16", "f32", 64, False, True),
    ([1], [1], 32, 8, 128, 16, "bf16", "f32", 128, True, True),
    ([1] * 61, [1 + 13 * i for i in range(61)], 32, 8, 128, 16, "f16", "f32", 128, False, True),
    ([1] * 300, [1 + (i * 7) % 50 for i in range(300)], 8, 2, 64, 16, "f16", "f16", 64, True, False),
    ([100, 0, 333], [300, 5, 333], 64, 8, 128, 32, "bf16", "bf16", 96, True, True),
    ([100, 0, 333], [300, 5, 333], 64, 8, 128, 32, "f16", "bf16", 96, False, True),
    ([250], [250], 12, 2, 128, 256, "f16", "f16", 0, False, True),
    ([250], [7000], 5, 1, 64, 64, "bf16", "f32", 8, True, False),
    ([17, 18], [100017, 40], 16, 16, 128, 128, "f16", "f32", 128, True, True),  # far positions
    ([9], [4], 8, 2, 64, 16, "f16", "f32", 62, False, True),  # fewer slots than tokens
]


@pytest.mark.parametrize("new,kv,nh,nkv,hd,ps,dtype,src,R,half,norm", APPEND)
def test_append_matches_64_bits(gpu, new, kv, nh, nkv, hd, ps, dtype, src, R, half, norm):
    import torch
    s = Step([0] * len(new), kv, nh, nkv, hd, ps, dtype, seed=kv[0] + R)
    s.new, s.n = new, sum(new) + 3
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s.q_start.copy_(torch.tensor(starts))
    width = (nh + 2 * nkv) * hd
    g = s.g
    wide = (torch.randn(s.n, width + 64, generator=g, device="cuda") * 2).to(_types()[src])
    qkv = wide[:, 32: 32 + width]
    wide_q = torch.full((s.n, nh * hd + 64), 7.0, device="cuda").to(_types()[dtype])
    q_out = wide_q[:, 16: 16 + nh * hd]
    qn, kn = ((1 + 0.3 * torch.randn(2, hd, generator=g, device="cuda")) if norm else (None, None))
    inv = torch.tensor([1e4 ** (-2.0 * j / max(R, 1)) for j in range(R // 2)] or [0.0], device="cuda")
    k0, v0 = s.k.clone(), s.v.clone()
    s.batch().append(qkv, q_out, inv, R, q_norm=qn, k_norm=kn, eps=1e-6, half=half, clip=5.0,
                     stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    pos = torch.cat([torch.arange(m - n, m) for n, m in zip(new, kv)] + [torch.zeros(3)]).long().cuda()
    ref, tol = _append64(s, qkv, qn, kn, 1e-6, inv, R, half, pos, 5.0)
    T, H, K = sum(new), nh, nkv
    err = (q_out[:T].double().view(T, H, hd) - ref[:T, :H]).abs()
    assert (err <= tol[:T, :H]).all(), float((err / tol[:T, :H]).max())
    assert (wide_q[T:] == 7).all() and (wide_q[:, :16] == 7).all() and (wide_q[:, 16 + nh * hd:] == 7).all()
    touched = torch.zeros(s.n_pages, ps, dtype=torch.bool, device="cuda")
    for i, (n, m) in enumerate(zip(new, kv)):
        for r in range(n):
            t = m - n + r
            if t < 0:
                continue
            page, row, at = s.table[i][t // ps], t % ps, starts[i] + r
            touched[page, row] = True
            for x, lo in ((s.k, H), (s.v, H + K)):
                e = (x[page, :, row].double() - ref[at, lo: lo + K]).abs()
                assert (e <= tol[at, lo: lo + K]).all(), (i, r)
    keep = ~touched[:, None, :, None].expand_as(s.k)
    for x, x0 in ((s.k, k0), (s.v, v0)):  # nothing else in the pool changed (bits, NaN among them)
        assert torch.equal(x.view(torch.int16)[keep], x0.view(torch.int16)[keep])


def test_append_drops_tokens_without_a_page_and_takes_positions(gpu):
    import torch
    s = Step([6, 5], [20, 40], 8, 2, 64, 16, "f16", seed=71)
    s.page_table[0, 1] = -1  # slots 16..19 of the first sequence: the last four tokens
    s.page_table[1, 2] = s.n_pages  # slots 32..39 of the second
    qkv = torch.randn(s.n, 768, device="cuda")
    pos = torch.randint(0, 5000, (s.n,), dtype=torch.int32, device="cuda")
    inv = torch.tensor([1e4 ** (-2.0 * j / 64) for j in range(32)], device="cuda")
    k0, v0 = s.k.clone(), s.v.clone()
    out = torch.empty_like(s.q)
    s.batch().append(qkv, out, inv, 64, pos=pos, stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    ref, tol = _append64(s, qkv, None, None, 0.0, inv, 64, False, pos, 1e30)
    assert ((out.double().view(s.n, 8, 64) - ref[:, :8]).abs() <= tol[:, :8]).all()
    e = (s.k[s.table[0][0], :, 14].double() - ref[0, 8:10]).abs()
    assert (e <= tol[0, 8:10]).all()  # token 0 of the first sequence: slot 14
    changed = (s.k.view(torch.int16) != k0.view(torch.int16)).flatten(1).any(1)
    assert changed.nonzero().flatten().tolist() == [s.table[0][0]]
    changed = (s.v.view(torch.int16) != v0.view(torch.int16)).flatten(1).any(1)
    assert changed.nonzero().flatten().tolist() == [s.table[0][0]]


def test_append_then_attend_in_a_graph(gpu):
    """A serving run: prompts in chunks, then single tokens, append and attend captured together and
    replayed with new lengths, against the attention over keys and values kept aside in 64 bits."""
    import torch
    nh, nkv, hd, ps, T = 8, 2, 128, 16, 48
    lens = [150, 33, 1]
    g = torch.Generator(device="cuda").manual_seed(81)
    total = [n + 6 for n in lens]  # prompt and six generated tokens
    i32 = dict(dtype=torch.int32, device="cuda")
    n_pages = sum(-(-n // ps) for n in total)
    free = torch.randperm(n_pages, generator=g, device="cuda").tolist()
    width = max(-(-n // ps) for n in total)
    k = torch.full((n_pages, nkv, ps, hd), math.nan, device="cuda").half()
    v = k.clone()
    table, q_start, kv_len = torch.full((3, width), -1, **i32), torch.zeros(4, **i32), torch.zeros(3, **i32)
    b = PagedBatch(k, v, table, q_start, kv_len, nh, T)
    qkv = torch.zeros(T, (nh + 2 * nkv) * hd, device="cuda")
    q, out = torch.zeros(T, nh * hd, device="cuda").half(), torch.zeros(T, nh * hd, device="cuda").half()
    qn, kn = 1 + 0.2 * torch.randn(2, hd, generator=g, device="cuda")
    inv = torch.tensor([1e4 ** (-2.0 * j / hd) for j in range(hd // 2)], device="cuda")
    scratch = torch.zeros(b.scratch_bytes(), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        st = torch.cuda.current_stream().cuda_stream
        b.append(qkv, q, inv, hd, q_norm=qn, k_norm=kn, stream=st)
        b.attend(q, out, scratch, stream=st)
    rows = [torch.randn(n, (nh + 2 * nkv) * hd, generator=g, device="cuda") for n in total]
    done = [0, 0, 0]
    while any(d < n for d, n in zip(done, total)):
        take, room = [], T
        for d, n, p in zip(done, total, lens):
            c = min(p - d if d < p else 1, room - 2) if d < n else 0
            take.append(max(c, 0))
            room -= take[-1]
        at, starts = 0, [0]
        for s in range(3):
            qkv[at: at + take[s]] = rows[s][done[s]: done[s] + take[s]]
            for t in range(done[s], done[s] + take[s]):
                if t % ps == 0:
                    table[s, t // ps] = free.pop()
            done[s] += take[s]
            at += take[s]
            starts.append(at)
        q_start.copy_(torch.tensor(starts))
        kv_len.copy_(torch.tensor(done))
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        for s in range(3):
            m, n = done[s], take[s]
            if not n:
                continue
            x = rows[s][:m].double().view(m, nh + 2 * nkv, hd)
            y = x.clone()
            for lo, hi, w in ((0, nh, qn), (nh, nh + nkv, kn)):
                y[:, lo:hi] = x[:, lo:hi] / (x[:, lo:hi].square().mean(-1, keepdim=True) + 1e-5).sqrt() * w.double()
            ang = torch.arange(m, device="cuda").double()[:, None] * inv.double()
            z = torch.polar(torch.ones_like(ang), ang)[:, None] * torch.view_as_complex(
                y[:, : nh + nkv].reshape(m, nh + nkv, hd // 2, 2).contiguous())
            y[:, : nh + nkv] = torch.view_as_real(z).flatten(-2)
            keys, vals = y[:, nh: nh + nkv].half().double(), y[:, nh + nkv:].half().double()
            hidden = torch.arange(m, device="cuda")[None] > torch.arange(m - n, m, device="cuda")[:, None]
            for h in range(nh):
                sc = y[m - n:, h].half().double() @ keys[:, h // 4].T / math.sqrt(hd)
                w = torch.softmax(sc.masked_fill(hidden, -math.inf), -1)
                ref = w @ vals[:, h // 4]
                got = out[starts[s]: starts[s] + n, h * hd: (h + 1) * hd].double()
                # a stored key may differ from its 64-bit value's rounding by one step (2^-10 of |k|), which moves
                # a score by at most 2^-10 * scale * sum |q k|, under 2^-10 * 12 here, and so does a query
                tol = U["f16"] * ref.abs() + (2.0 ** -11 + 2.0 ** -16 + 2 * 12 * 2.0 ** -10) * (w @ vals[:, h // 4].abs())
                assert ((got - ref).abs() <= tol).all()
        assert (out[starts[-1]:] == 7).all()
