"""Refusals of the paged-cache entry points beyond those of test_paged_cpu.py, and what the class hands to them; no GPU."""
from yalm_b200 import _lib


def test_wait_budgets_out_of_range_are_refused():
    L = _lib.lib()
    for bad in (-1, 4 * 10 ** 9 + 1):
        assert L.yb_paged_attention_wait_budget(bad) == _lib.YB_E_INVALID
        assert _lib.last_error()
    for good in (1, 4 * 10 ** 9, 0):
        assert L.yb_paged_attention_wait_budget(good) == 0


def _batch():
    import torch

    from yalm_b200 import PagedBatch
    k, i32 = torch.zeros(3, 2, 16, 64, dtype=torch.float16), dict(dtype=torch.int32)
    return PagedBatch(k, k.clone(), torch.zeros(2, 1, **i32), torch.zeros(3, **i32), torch.zeros(2, **i32), 8, 4)


def test_status_reads_and_clears_the_workspaces_first_word():
    import pytest
    import torch
    b = _batch()
    for scratch in (torch.zeros(b.scratch_bytes(), dtype=torch.uint8), torch.zeros(2, b.scratch_bytes(), dtype=torch.int32)):
        assert b.status(scratch) == 0
        scratch.view(-1).view(torch.uint8)[:8] = 255
        assert b.status(scratch) == 0xFFFFFFFF
        assert b.status(scratch) == 0
        assert (scratch.view(-1).view(torch.uint8)[4:8] == 255).all()  # the word alone
    with pytest.raises(ValueError):
        b.status(torch.zeros(b.scratch_bytes() - 1, dtype=torch.uint8))
