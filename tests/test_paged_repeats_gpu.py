"""Batches whose blocks go from units of one row tile to units of two, again and again: outputs within the tolerances of
test_paged_gpu, and the same bits in thousands of calls."""
import random

import pytest

from test_paged_gpu import Step
from test_paged_shared_gpu import Shared

pytestmark = pytest.mark.gpu


def _repeats(st, call, runs=4000, at_once=50):
    import torch
    want = st.check()
    want = want.to(st.q.dtype)
    outs = [torch.full_like(want, 7.0) for _ in range(at_once)]
    for _ in range(runs // at_once):
        for o in outs:
            call(o)
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)
        for o in outs:
            o.fill_(7.0)


def _prompts(n, gq, seed):
    """Single tokens and short prompts of one or two row tiles, in every order."""
    r, qb = random.Random(seed), 128 // gq
    new = [r.choice([1, 1, qb, qb + 1, 2 * qb, 2 * qb + 3, 3 * qb + 1]) for _ in range(n)]
    return new, [n + r.randint(0, 300) for n in new]


@pytest.mark.parametrize("nh,nkv,hd,n,dtype", [(64, 8, 128, 300, "f16"), (16, 1, 128, 900, "bf16"), (32, 8, 64, 200, "f16"),
                                               (8, 8, 128, 120, "f16")])
def test_short_prompts_repeat(gpu, nh, nkv, hd, n, dtype):
    import torch
    new, kv = _prompts(n, nh // nkv, n)
    st = Step(new, kv, nh, nkv, hd, 16, dtype, seed=n)
    b = st.batch()
    scratch = torch.zeros(b.scratch_bytes(), dtype=torch.uint8, device="cuda")
    _repeats(st, lambda o: b.attend(st.q, o, scratch))
    assert b.status(scratch) == 0


@pytest.mark.parametrize("nh,nkv,hd,S,prefix,own,dtype", [(64, 8, 128, 69, 128, 2000, "f16"), (64, 8, 128, 106, 128, 1900, "bf16"),
                                                          (16, 2, 64, 150, 256, 900, "f16"), (16, 1, 128, 40, 384, 300, "f16")])
def test_prefixes_of_groups_that_end_in_one_tile_repeat(gpu, nh, nkv, hd, S, prefix, own, dtype):
    import torch
    r = random.Random(S)
    st = Shared([0, S], [prefix], [r.randint(0, own) for _ in range(S)], [1] * S, nh, nkv, hd, 32, dtype, seed=S)
    b = st.batch()
    scratch = torch.zeros(b.shared_scratch_bytes(1), dtype=torch.uint8, device="cuda")
    _repeats(st, lambda o: b.attend_shared(st.q, o, scratch, st.group_start, st.prefix_len), runs=10000)
    assert b.status(scratch) == 0
