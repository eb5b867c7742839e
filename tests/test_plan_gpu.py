"""The plan of a serving step (yb_paged_plan_dev) against its definition, sequence by sequence and page by page:
whole numbers, which have to be equal."""
import random

import pytest

from yalm_b200 import PagedBatch, YalmB200Error

pytestmark = pytest.mark.gpu


class State:
    """Caches of kv slots each in pages handed out in random order, and a list of the free ones."""

    def __init__(self, kv, P, spare, width, n_tokens, seed=0, kept=None, holes=0):
        import torch
        r = random.Random(seed)
        held = [-(-n // P) for n in kv]
        self.P, self.width, self.n_tokens, self.kv, self.kept = P, width, n_tokens, list(kv), kept
        self.n_pages = max(1, sum(held) + spare)
        ids = list(range(self.n_pages))
        r.shuffle(ids)
        self.table = [[ids.pop() if j < h else -1 for j in range(width)] for h in held]
        for _ in range(holes):
            s = r.randrange(len(kv))
            if held[s]:
                self.table[s][r.randrange(held[s])] = r.choice([-1, self.n_pages, 1 << 30])
        self.free = ids + [-7] * (self.n_pages - len(ids))
        self.n_free = len(ids)
        i32 = dict(dtype=torch.int32, device="cuda")
        S = len(kv)
        self.t = dict(table=torch.tensor(self.table, **i32).view(S, width), free=torch.tensor(self.free, **i32),
                      n_free=torch.tensor([self.n_free], **i32), kv_len=torch.tensor(self.kv, **i32).view(S),
                      q_start=torch.full((S + 1,), 55, **i32), status=torch.full((4,), 9, **i32),
                      pos=torch.full((n_tokens,), -3, **i32),
                      slots=torch.full((n_tokens,), -3, dtype=torch.int64, device="cuda"))
        k = torch.empty((self.n_pages, 1, P, 64), dtype=torch.float16, device="cuda")
        self.batch = PagedBatch(k, k.clone(), self.t["table"], self.t["q_start"], self.t["kv_len"], 1, n_tokens)
        self.kept_t = None if kept is None else torch.tensor(kept, **i32)

    def plan(self, new, **kw):
        import torch
        t = self.t
        self.new_t = torch.tensor(new, dtype=torch.int32, device="cuda")
        a = dict(kept=self.kept_t, pos=t["pos"], slots=t["slots"])
        a.update(kw)
        self.batch.plan(self.new_t, t["free"], t["n_free"], t["status"], **a)

    def expect(self, new):
        """Advances the host's copy by the definition; returns what the device is to hold."""
        P, S, cap = self.P, len(self.kv), self.width * self.P
        kv = [min(max(v, 0), cap) for v in self.kv]
        for s, n in enumerate(new):
            if n < 0:
                kept = max(0, self.kept[s]) if self.kept else 0
                for j in range(kept, -(-kv[s] // P)):
                    page = self.table[s][j]
                    if 0 <= page < self.n_pages:
                        self.free[self.n_free] = page
                        self.n_free += 1
        rows = sum(max(n, 0) for n in new)
        long = [s for s, n in enumerate(new) if n >= 0 and kv[s] + n > cap]
        need = sum(-(-(kv[s] + n) // P) - -(-kv[s] // P) for s, n in enumerate(new) if n >= 0 and s not in set(long))
        status = [(1 if need > self.n_free else 0) | (2 if rows > self.n_tokens else 0) | (4 if long else 0),
                  max(0, need - self.n_free), min(max(0, rows - self.n_tokens), 2 ** 31 - 1), long[0] if long else -1]
        q_start, pos, slots = [0], [], []
        for s, n in enumerate(new):
            n = 0 if status[0] else max(n, 0)
            base = 0 if new[s] < 0 else kv[s]
            for t in range(base, base + n):
                if t % P == 0:
                    self.n_free -= 1
                    self.table[s][t // P] = self.free[self.n_free]
                page = self.table[s][t // P]
                pos.append(t)
                slots.append(page * P + t % P if 0 <= page < self.n_pages else -1)
            q_start.append(q_start[-1] + n)
            kv[s] = base + n
        self.kv = kv
        return dict(q_start=q_start, kv_len=kv, status=status, n_free=[self.n_free], free=self.free[: self.n_free],
                    table=self.table, pos=pos + [-3] * (self.n_tokens - len(pos)),
                    slots=slots + [-3] * (self.n_tokens - len(slots)))

    def compare(self, want):
        import torch
        torch.cuda.synchronize()
        for k, v in want.items():
            got = self.t[k].tolist()
            assert (got[: len(v)] if k == "free" else got) == v, k


def _step(st, new, **kw):
    want_pos, want_slots = (st.t[k].clone() for k in ("pos", "slots"))
    st.plan(new, **kw)
    want = st.expect(new)
    n = want["q_start"][-1]
    want["pos"][n:], want["slots"][n:] = want_pos[n:].tolist(), want_slots[n:].tolist()
    st.compare(want)
    return want


CASES = [  # (cached, new, page size, spare pages, table width, rows)
    ([0], [1], 16, 3, 4, 1),
    ([0], [0], 16, 0, 1, 1),
    ([15, 16, 17], [1, 1, 1], 16, 3, 3, 4),
    ([16], [-1], 16, 0, 2, 1),
    ([100, 3, 64, 0], [-1, 200, -5, 0], 32, 2, 20, 210),
    ([0, 0, 0], [256, 257, 255], 256, 4, 3, 800),
    ([5000], [3000], 16, 190, 600, 3000),
    ([1] * 1024, [1] * 1024, 16, 0, 2, 1024),
    ([16 * (i % 3) for i in range(1024)], [1 if i % 5 else -1 for i in range(1024)], 16, 900, 4, 1030),
    ([16 * (i % 3) for i in range(1025)], [(i % 4) - 1 for i in range(1025)], 16, 900, 4, 2000),  # two kernels
    ([7], [8193], 64, 200, 200, 8193),  # two kernels for the rows' sake
    ([5] * 9000, [(700 if i == 3 else 0) if i < 8000 else i % 3 for i in range(9000)], 16, 2000, 60, 3000),  # far apart
    ([5] * 60000, [1 if i % 20000 == 7 else 0 for i in range(60000)], 16, 9, 2, 9000),
    ([i % 90 for i in range(20000)], [(i * 7) % 12 - 1 for i in range(20000)], 32, 30000, 4, 100000),
]


@pytest.mark.parametrize("kv,new,P,spare,width,rows", CASES)
@pytest.mark.parametrize("kept", [False, True])
def test_plans_match_the_definition(gpu, kv, new, P, spare, width, rows, kept):
    st = State(kv, P, spare, width, rows, seed=len(kv), kept=[(s * 3) % 4 for s in range(len(kv))] if kept else None)
    assert not _step(st, new)["status"][0] or kept  # pages that are kept may be missed


def test_most_sequences_that_a_batch_has(gpu):
    S = 65536
    st = State([i % 17 for i in range(S)], 16, 20000, 2, 70000, seed=3)
    assert _step(st, [1 if i % 11 else -1 for i in range(S)])["status"] == [0, 0, 0, -1]


def test_steps_in_place_one_after_another(gpu):
    r = random.Random(5)
    st = State([0] * 40, 16, 700, 16, 600, seed=1)
    for _ in range(60):
        new = [r.choice([0, 1, 1, 1, 1, 30, -1]) if kv < 200 else -1 for kv in st.kv]
        assert _step(st, new)["status"][0] == 0
    assert sorted(st.free[: st.n_free] + [p for row, kv in zip(st.table, st.kv) for p in row[: -(-kv // 16)]]) == \
        list(range(st.n_pages))  # no page is lost or given twice


@pytest.mark.parametrize("big", [False, True])
@pytest.mark.parametrize("kv,new,spare,width,rows,bits", [
    ([3, 40, 9], [20, -1, 60], 1, 8, 100, 1),  # the page that an ended sequence gives back is not enough
    ([3, 40, 9], [20, 30, 60], 9, 8, 50, 2),
    ([3, 40, 9], [20, 100, 190], 90, 8, 500, 4),
    ([3, 40, 9], [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1], 4, 8, 500, 6),
    ([3, 40, 9], [20, 30, 100], 3, 8, 50, 3)])
def test_a_step_that_does_not_fit_takes_nothing(gpu, big, kv, new, spare, width, rows, bits):
    more = 1100 if big else 0  # a batch that takes the cluster of blocks
    st = State(kv + [0] * more, 16, spare, width, rows, seed=2)
    assert _step(st, new + [0] * more)["status"][0] == bits


def test_state_of_its_own_can_be_planned_again(gpu):
    import torch
    for S in (30, 1500):
        kv, new = [(i * 13) % 70 for i in range(S)], [(i * 7) % 20 - 1 for i in range(S)]
        st = State(kv, 16, 3 * S, 8, 20 * S, seed=4)
        before = {k: st.t[k].clone() for k in ("kv_len", "n_free")}
        want = None
        for _ in range(3):
            st.plan(new, kv_before=before["kv_len"], n_free_before=before["n_free"])
            want = want or st.expect(new)
            st.compare(want)
        assert torch.equal(before["kv_len"], torch.tensor(kv, dtype=torch.int32, device="cuda"))


def test_pages_that_are_not_there(gpu):
    st = State([100] * 30, 16, 50, 10, 400, seed=6, holes=60)
    _step(st, [10] * 30)
    st = State([100] * 30, 16, 50, 10, 400, seed=7, holes=60)
    _step(st, [-1 if i % 2 else 5 for i in range(30)])


def test_lengths_and_counts_out_of_range(gpu):
    import torch
    st = State([0, 20, 5], 16, 9, 3, 40, seed=8)
    st.t["kv_len"].copy_(torch.tensor([-4, 1 << 30, 5]))
    st.kv = [-4, 1 << 30, 5]
    _step(st, [3, 0, 8])
    st.t["n_free"].fill_(-5)
    st.n_free = 0
    assert _step(st, [1, 0, 40])["status"][0] == 6  # 41 tokens for 40 rows, and 13 + 40 slots in a row of 48
    assert _step(st, [20, 0, 20])["status"] == [1, 3, 0, -1]
    st.t["n_free"].fill_(1 << 30)
    st.n_free = st.n_pages
    st.free = [p if 0 <= p < st.n_pages else 0 for p in st.free]
    st.t["free"].copy_(torch.tensor(st.free))
    assert _step(st, [1, 0, 20])["status"][0] == 0


def test_without_positions_or_slots(gpu):
    for S in (9, 1200):
        for drop in ("pos", "slots"):
            st = State([5] * S, 16, 2 * S, 4, 20 * S, seed=9)
            old = st.t[drop].clone()
            st.plan([12] * S, **{drop: None})
            want = st.expect([12] * S)
            want[drop] = old.tolist()
            st.compare(want)


def test_no_sequences_and_no_rows(gpu):
    import torch
    st = State([], 16, 5, 1, 4)
    st.plan([])
    torch.cuda.synchronize()
    assert st.t["q_start"].tolist() == [0] and st.t["status"].tolist() == [0, 0, 0, -1] and st.t["n_free"].tolist() == [5]
    st = State([40, 3], 16, 5, 4, 0)
    _step(st, [-1, 0])
    assert _step(st, [0, 1])["status"][0] == 2


def test_replayed_graph_follows_new_requests(gpu):
    import torch
    for S in (50, 1100):
        st = State([0] * S, 16, 8 * S, 16, 12 * S, seed=10)
        st.plan([0] * S)
        st.expect([0] * S)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        keep = st.new_t
        with torch.cuda.graph(g):
            st.batch.plan(keep, st.t["free"], st.t["n_free"], st.t["status"], pos=st.t["pos"], slots=st.t["slots"])
        r = random.Random(S)
        for _ in range(6):
            new = [r.choice([0, 1, 11, -1]) for _ in range(S)]
            keep.copy_(torch.tensor(new))
            old = {k: st.t[k].tolist() for k in ("pos", "slots")}
            g.replay()
            want = st.expect(new)
            n = want["q_start"][-1]
            for k in old:
                want[k][n:] = old[k][n:]
            st.compare(want)


def test_refusals(gpu):
    import torch
    st = State([5, 9], 16, 4, 4, 8)
    i32 = dict(dtype=torch.int32, device="cuda")
    t, new = st.t, torch.zeros(2, **i32)
    with pytest.raises(ValueError):
        st.batch.plan(new[:1], t["free"], t["n_free"], t["status"])
    with pytest.raises(ValueError):
        st.batch.plan(new, t["free"][1:], t["n_free"], t["status"])
    with pytest.raises(ValueError):
        st.batch.plan(new.long(), t["free"], t["n_free"], t["status"])
    with pytest.raises(ValueError):
        st.batch.plan(new, t["free"], t["n_free"], t["status"][:3])
    with pytest.raises(ValueError):
        st.batch.plan(new, t["free"], t["n_free"], t["status"], slots=t["pos"])
    with pytest.raises(ValueError):
        st.batch.plan(new.cpu(), t["free"], t["n_free"], t["status"])
    with pytest.raises(YalmB200Error):
        from yalm_b200 import _lib
        host = torch.zeros(4, dtype=torch.int32)
        _lib.call("yb_paged_plan_dev", st.batch._ref, new.data_ptr(), t["kv_len"].data_ptr(), None, t["free"].data_ptr(),
                  t["n_free"].data_ptr(), t["n_free"].data_ptr(), None, None, host.data_ptr(), None)
