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
