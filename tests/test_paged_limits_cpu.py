"""Refusals of the paged-cache entry points beyond those of test_paged_cpu.py, and what the class hands to them; no GPU."""
import ctypes

import pytest

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


P = 4096  # an aligned address that nothing reads


def _descriptor(**kw):
    c = dict(n_seqs=2, n_tokens=5, n_heads=8, n_kv_heads=2, head_dim=64, dtype=1, page_size=16, n_pages=9, max_pages=4,
             q_start_dev=P, kv_len_dev=P, page_table_dev=P, k_pages=P, v_pages=P)
    c.update(kw)
    return _lib.yb_paged_batch(**c)


def _append(b, width, **kw):
    c = dict(q_out=P, q_out_stride=width, qkv=P, qkv_stride=3 * width, qkv_dtype=0, q_norm=None, k_norm=None, eps=1e-5,
             inv_freq=P, rotary_dim=64, half=0, pos=None, clip=3e38)
    c.update(kw)
    return _lib.lib().yb_paged_append_dev(ctypes.byref(b), *c.values(), None)


def _attend(b, width, **kw):
    c = dict(out=P, out_stride=width, q=P, q_stride=width, scale=0.125, window=0, scratch=P)
    c.update(kw)
    return _lib.lib().yb_paged_attention_dev(ctypes.byref(b), *c.values(), None)


def test_the_attentions_limit_of_work_is_the_documented_one_and_its_own():
    """At the limit the call passes on to the buffers' check (these are no device memory), one unit more is refused.
    The append has no such limit."""
    L = _lib.lib()
    sms = L.yb_num_sms() or 148
    H = 512  # a kv head a query head: units of 256 queries
    tiles = (1 << 21) // 128 + 3
    last = (sms * (2 ** 31 - 1) - 1) // (H * tiles)  # units
    for units, refused in ((last, False), (last + 1, True), (60000, True)):
        n = next(n for n in range(units, 0, -1) if n // 256 + n <= units)  # as many sequences as tokens
        rest = units - n // 256 - n
        b = _descriptor(n_seqs=n + rest, n_tokens=n + rest, n_heads=H, n_kv_heads=H, max_pages=(1 << 21) // 16)
        assert (n + rest) // 256 + n + rest == units
        rc = _attend(b, H * 64)
        assert (rc == _lib.YB_E_UNSUPPORTED) == refused and rc != 0
        assert ("too many slots" in _lib.last_error()) == refused
        assert (L.yb_paged_attention_scratch_bytes(ctypes.byref(b)) == 0) == refused
        assert _append(b, H * 64) not in (0, _lib.YB_E_UNSUPPORTED)


@pytest.mark.parametrize("name", ["q_start_dev", "kv_len_dev", "page_table_dev"])
@pytest.mark.parametrize("off", [1, 2, 3])
def test_misaligned_lengths_and_tables_are_refused(name, off):
    """A word read at such an address would end the context."""
    b = _descriptor(**{name: P + off})
    for call in (_append, _attend):
        assert call(b, 512) == _lib.YB_E_INVALID
        assert "4-byte aligned" in _lib.last_error()
    assert _lib.lib().yb_paged_attention_scratch_bytes(ctypes.byref(b)) == 0


@pytest.mark.parametrize("name", ["q_norm", "k_norm", "inv_freq", "pos"])
@pytest.mark.parametrize("off", [1, 2, 3])
def test_misaligned_vectors_are_refused(name, off):
    assert _append(_descriptor(), 512, **{name: P + off}) == _lib.YB_E_INVALID
    assert "4-byte aligned" in _lib.last_error()


def test_scales_that_overflow_are_refused():
    """The kernel's factor is scale * log2(e)."""
    for scale in (3e38, 2.4e38):
        assert _attend(_descriptor(), 512, scale=scale) == _lib.YB_E_INVALID
        assert "scale" in _lib.last_error()
    assert _attend(_descriptor(n_tokens=0), 512, scale=2.3e38) == 0


@pytest.mark.parametrize("window,handed", [(0, 0), (5, 5), (2 ** 31 - 1, 2 ** 31 - 1), (2 ** 31, 2 ** 31 - 1),
                                           (2 ** 32, 2 ** 31 - 1), (2 ** 32 + 5, 2 ** 31 - 1), (10 ** 30, 2 ** 31 - 1)])
def test_windows_wider_than_an_int_see_everything(window, handed):
    """A C int would take their low bits: 2^32 + 5 as a window of 5."""
    import torch
    b = _batch()
    seen = []
    b._attend = lambda *a: seen.append(ctypes.c_int(a[6]).value) or 0
    q = torch.zeros(4, 512, dtype=torch.float16)
    b.attend(q, q.clone(), torch.zeros(b.scratch_bytes(), dtype=torch.uint8), window=window)
    assert seen == [handed]


@pytest.mark.parametrize("window", [-1, -2 ** 31, -2 ** 32 + 5, -2 ** 32])
def test_negative_windows_are_refused(window):
    import torch
    b = _batch()
    q = torch.zeros(4, 512, dtype=torch.float16)
    with pytest.raises(_lib.YalmB200Error):
        b.attend(q, q.clone(), torch.zeros(b.scratch_bytes(), dtype=torch.uint8), window=window)


def test_inputs_are_read_by_coherent_loads():
    """The kernels start while the one before them may still be writing lengths, tables and rows (programmatic launch);
    non-coherent loads need memory that nothing writes while the kernel lives, wherever in the kernel they stand."""
    import os
    import re
    csrc = os.path.join(os.path.dirname(_lib.__file__), "csrc")
    for name in ("paged.cuh", "paged_append.cu", "paged_attn.cu"):
        code = re.sub(r"//.*", "", open(os.path.join(csrc, name)).read())
        assert not re.search(r"__ldg\b|ld\.global\.nc|__restrict__", code), name


def test_work_axis_against_counting(tmp_path):
    """The closed forms by which the attention's blocks share out the work (csrc/paged_axis.cuh), compiled for the
    host: lengths up to the limits, every key tile walked once, every cut unit's parts where the merge looks."""
    import os
    import subprocess
    here = os.path.dirname(os.path.abspath(__file__))
    csrc = os.path.join(os.path.dirname(_lib.__file__), "csrc")
    exe = str(tmp_path / "axis")
    subprocess.run(["g++", "-O2", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", "-I" + csrc, "-o", exe,
                    os.path.join(here, "paged_axis_check.cpp")], check=True, timeout=300)
    r = subprocess.run([exe, "1500"], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout + r.stderr
