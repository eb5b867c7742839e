"""Refusals of the plan and the sampler (yb_paged_plan_dev, yb_sample_rows_dev): every bad size, NULL or alignment
returns an error code with a message before any CUDA call, so without a GPU too; a dummy non-NULL address is never
dereferenced on these paths."""
import ctypes

import pytest

from yalm_b200 import _lib

P = 4096  # an aligned address that nothing reads


def _batch(**kw):
    c = dict(n_seqs=2, n_tokens=5, n_heads=8, n_kv_heads=2, head_dim=64, dtype=1, page_size=16, n_pages=9, max_pages=4,
             q_start_dev=P, kv_len_dev=P, page_table_dev=P, k_pages=P, v_pages=P)
    c.update(kw)
    return _lib.yb_paged_batch(**c)


def _plan(b, **kw):
    c = dict(new_len=P, kv_before=P, kept=None, free_pages=P, n_free_before=P, n_free=P, pos=P, slots=P, status=P)
    c.update(kw)
    return _lib.lib().yb_paged_plan_dev(ctypes.byref(b) if b else None, *c.values(), None)


def _sample(**kw):
    c = dict(tokens=P, prob=P, logits=P, stride=100, dtype=0, rows=2, vocab=100, coin=P, temperature=P, top_k=P, top_p=P,
             min_p=P)
    c.update(kw)
    return _lib.lib().yb_sample_rows_dev(*c.values(), None)


@pytest.mark.parametrize("kw", [{"new_len": None}, {"kv_before": None}, {"free_pages": None}, {"n_free_before": None},
                                {"n_free": None}, {"status": None}, {"new_len": P + 1}, {"kept": P + 2}, {"pos": P + 3},
                                {"slots": P + 4}, {"status": P + 2}, {"free_pages": P + 1}])
def test_bad_plan_arguments_are_refused(kw):
    assert _plan(_batch(), **kw) == _lib.YB_E_INVALID
    assert _lib.last_error()


@pytest.mark.parametrize("kw,code", [({"page_size": 24}, _lib.YB_E_UNSUPPORTED), ({"n_seqs": -1}, _lib.YB_E_INVALID),
                                     ({"n_seqs": 65537}, _lib.YB_E_UNSUPPORTED), ({"q_start_dev": None}, _lib.YB_E_INVALID),
                                     ({"n_tokens": (1 << 20) + 1}, _lib.YB_E_UNSUPPORTED),
                                     ({"n_tokens": 0, "page_table_dev": None}, _lib.YB_E_INVALID),
                                     ({"n_seqs": 0, "q_start_dev": None}, _lib.YB_E_INVALID)])
def test_bad_batches_are_refused_by_the_plan(kw, code):
    assert _plan(_batch(**kw)) == code
    assert _lib.last_error()


def test_null_batch_is_refused():
    assert _plan(None) == _lib.YB_E_INVALID


@pytest.mark.parametrize("kw,code", [
    ({"tokens": None}, _lib.YB_E_INVALID), ({"logits": None}, _lib.YB_E_INVALID), ({"coin": None}, _lib.YB_E_INVALID),
    ({"dtype": 3}, _lib.YB_E_UNSUPPORTED), ({"dtype": -1}, _lib.YB_E_UNSUPPORTED), ({"rows": -1}, _lib.YB_E_INVALID),
    ({"vocab": 0}, _lib.YB_E_INVALID), ({"rows": 65537}, _lib.YB_E_UNSUPPORTED),
    ({"vocab": (1 << 20) + 1, "stride": 1 << 21}, _lib.YB_E_UNSUPPORTED), ({"stride": 99}, _lib.YB_E_INVALID),
    ({"stride": (1 << 31) + 1}, _lib.YB_E_INVALID), ({"logits": P + 2}, _lib.YB_E_INVALID),
    ({"logits": P + 1, "dtype": 1}, _lib.YB_E_INVALID), ({"tokens": P + 2}, _lib.YB_E_INVALID),
    ({"prob": P + 1}, _lib.YB_E_INVALID), ({"min_p": P + 2}, _lib.YB_E_INVALID), ({"top_k": P + 1}, _lib.YB_E_INVALID)])
def test_bad_sampler_arguments_are_refused(kw, code):
    assert _sample(**kw) == code
    assert _lib.last_error()


def test_no_rows_need_no_gpu():
    assert _sample(rows=0) == 0
