"""Refusals of the plan, the attention over shared prefixes and the sampler (yb_paged_plan_dev,
yb_paged_attention_shared_dev, yb_sample_rows_dev): every bad size, NULL or alignment returns an error code with a
message before any CUDA call, so without a GPU too; a dummy non-NULL address is never dereferenced on these paths.  And
the arithmetic by which the attention shares out its work, against counting."""
import ctypes
import os
import subprocess

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


def _shared(b, **kw):
    c = dict(n_groups=1, group_start=P, prefix_len=P, out=P, out_stride=512, q=P, q_stride=512, scale=0.125, scratch=P)
    c.update(kw)
    return _lib.lib().yb_paged_attention_shared_dev(ctypes.byref(b) if b else None, *c.values(), None)


WIDE = dict(n_seqs=40, max_pages=4000)  # a table so long that prefixes are computed apart


@pytest.mark.parametrize("kw,code", [
    ({"n_groups": -1}, _lib.YB_E_INVALID), ({"n_groups": 2049}, _lib.YB_E_UNSUPPORTED), ({"group_start": None}, _lib.YB_E_INVALID),
    ({"prefix_len": None}, _lib.YB_E_INVALID), ({"group_start": P + 1}, _lib.YB_E_INVALID),
    ({"prefix_len": P + 2}, _lib.YB_E_INVALID), ({"out": None}, _lib.YB_E_INVALID), ({"q": P + 8}, _lib.YB_E_INVALID),
    ({"out_stride": 500}, _lib.YB_E_INVALID), ({"scale": 0.0}, _lib.YB_E_INVALID), ({"scratch": None}, _lib.YB_E_INVALID),
    ({"scratch": P + 8}, _lib.YB_E_INVALID)])
def test_bad_shared_attention_arguments_are_refused(kw, code):
    assert _shared(_batch(**WIDE), **kw) == code
    assert _lib.last_error()


def test_bad_batches_are_refused_by_the_shared_attention():
    for kw, code in (({"head_dim": 80}, _lib.YB_E_UNSUPPORTED), ({"n_heads": 7}, _lib.YB_E_INVALID),
                     ({"page_table_dev": None}, _lib.YB_E_INVALID), ({"page_size": 8}, _lib.YB_E_UNSUPPORTED)):
        assert _shared(_batch(**{**WIDE, **kw})) == code
        assert _lib.lib().yb_paged_attention_shared_scratch_bytes(ctypes.byref(_batch(**{**WIDE, **kw})), 1) == 0
    big = dict(n_seqs=65536, n_tokens=65536, n_heads=512, n_kv_heads=512, max_pages=(1 << 21) // 16)
    assert _shared(_batch(**big), out_stride=512 * 64, q_stride=512 * 64) == _lib.YB_E_UNSUPPORTED
    assert _shared(None) == _lib.YB_E_INVALID


def test_the_shared_workspace_serves_the_other_call_too():
    for kw in (WIDE, {}, dict(n_seqs=3, n_tokens=900, head_dim=128)):
        b = _batch(**kw)
        plain = _lib.lib().yb_paged_attention_scratch_bytes(ctypes.byref(b))
        assert 0 < plain < _lib.lib().yb_paged_attention_shared_scratch_bytes(ctypes.byref(b), 1)


def test_empty_shared_batches_need_no_gpu():
    for kw in ({"n_seqs": 0}, {"n_tokens": 0}):
        assert _shared(_batch(**{**WIDE, **kw})) == 0


def test_shared_work_axis_against_counting(tmp_path):
    here, csrc = os.path.dirname(os.path.abspath(__file__)), os.path.join(os.path.dirname(_lib.__file__), "csrc")
    exe = str(tmp_path / "axis")
    subprocess.run(["g++", "-O2", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", "-I" + csrc, "-o", exe,
                    os.path.join(here, "paged_shared_axis_check.cpp")], check=True, timeout=300)
    r = subprocess.run([exe, "20000"], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout + r.stderr


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
