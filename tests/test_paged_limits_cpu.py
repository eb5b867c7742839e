"""Refusals of the paged-cache entry points beyond those of test_paged_cpu.py, and what the class hands to them; no GPU."""
from yalm_b200 import _lib


def test_wait_budgets_out_of_range_are_refused():
    L = _lib.lib()
    for bad in (-1, 4 * 10 ** 9 + 1):
        assert L.yb_paged_attention_wait_budget(bad) == _lib.YB_E_INVALID
        assert _lib.last_error()
    for good in (1, 4 * 10 ** 9, 0):
        assert L.yb_paged_attention_wait_budget(good) == 0
