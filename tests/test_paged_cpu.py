"""Refusals of the paged-cache entry points (include/yalm_b200.h, yb_paged_*): every bad shape, NULL,
stride or alignment returns an error code with a message before any CUDA call, so without a GPU
too; a dummy non-NULL address is never dereferenced on these paths.  And the descriptor's layout."""
import ctypes

import pytest

from yalm_b200 import _lib

P = 4096  # a 16-byte aligned address that nothing reads


def _batch(**kw):
    c = dict(n_seqs=2, n_tokens=5, n_heads=8, n_kv_heads=2, head_dim=64, dtype=1, page_size=16, n_pages=9, max_pages=4,
             q_start_dev=P, kv_len_dev=P, page_table_dev=P, k_pages=P, v_pages=P)
    c.update(kw)
    return _lib.yb_paged_batch(**c)


def _append(b, **kw):
    c = dict(q_out=P, q_out_stride=512, qkv=P, qkv_stride=768, qkv_dtype=0, q_norm=None, k_norm=None, eps=1e-5,
             inv_freq=P, rotary_dim=64, half=0, pos=None, clip=3e38)
    c.update(kw)
    return _lib.lib().yb_paged_append_dev(ctypes.byref(b) if b else None, *c.values(), None)


def _attend(b, **kw):
    c = dict(out=P, out_stride=512, q=P, q_stride=512, scale=0.125, window=0, scratch=P)
    c.update(kw)
    return _lib.lib().yb_paged_attention_dev(ctypes.byref(b) if b else None, *c.values(), None)


BAD_BATCHES = [
    ({"dtype": 0}, _lib.YB_E_UNSUPPORTED), ({"dtype": 3}, _lib.YB_E_UNSUPPORTED),
    ({"head_dim": 80}, _lib.YB_E_UNSUPPORTED), ({"head_dim": 0}, _lib.YB_E_UNSUPPORTED),
    ({"n_heads": 7}, _lib.YB_E_INVALID), ({"n_kv_heads": 0}, _lib.YB_E_INVALID), ({"n_heads": 0}, _lib.YB_E_INVALID),
    ({"n_heads": 64, "n_kv_heads": 2}, _lib.YB_E_UNSUPPORTED),
    ({"page_size": 24}, _lib.YB_E_UNSUPPORTED), ({"page_size": 8}, _lib.YB_E_UNSUPPORTED),
    ({"page_size": 512}, _lib.YB_E_UNSUPPORTED), ({"page_size": 0}, _lib.YB_E_UNSUPPORTED),
    ({"n_seqs": -1}, _lib.YB_E_INVALID), ({"n_tokens": -1}, _lib.YB_E_INVALID), ({"n_pages": 0}, _lib.YB_E_INVALID),
    ({"max_pages": 0}, _lib.YB_E_INVALID), ({"max_pages": (1 << 21) // 16 + 1}, _lib.YB_E_UNSUPPORTED),
    ({"n_tokens": (1 << 20) + 1}, _lib.YB_E_UNSUPPORTED), ({"n_seqs": 65537}, _lib.YB_E_UNSUPPORTED),
    ({"n_pages": 1 << 27}, _lib.YB_E_UNSUPPORTED),
    ({"q_start_dev": None}, _lib.YB_E_INVALID), ({"kv_len_dev": None}, _lib.YB_E_INVALID),
    ({"page_table_dev": None}, _lib.YB_E_INVALID), ({"k_pages": None}, _lib.YB_E_INVALID),
    ({"v_pages": None}, _lib.YB_E_INVALID), ({"k_pages": P + 8}, _lib.YB_E_INVALID),
    ({"v_pages": P + 2}, _lib.YB_E_INVALID),
]


@pytest.mark.parametrize("kw,code", BAD_BATCHES)
def test_bad_batches_are_refused(kw, code):
    for call in (_append, _attend):
        assert call(_batch(**kw)) == code
        assert _lib.last_error()
    assert _lib.lib().yb_paged_attention_scratch_bytes(ctypes.byref(_batch(**kw))) == 0


@pytest.mark.parametrize("kw,code", [
    ({"q_out": None}, _lib.YB_E_INVALID), ({"qkv": None}, _lib.YB_E_INVALID), ({"q_out": P + 8}, _lib.YB_E_INVALID),
    ({"qkv": P + 4}, _lib.YB_E_INVALID), ({"q_out_stride": 511}, _lib.YB_E_INVALID),
    ({"q_out_stride": 516}, _lib.YB_E_INVALID), ({"qkv_stride": 767}, _lib.YB_E_INVALID),
    ({"qkv_stride": 770}, _lib.YB_E_INVALID), ({"qkv_stride": 772, "qkv_dtype": 1}, _lib.YB_E_INVALID),
    ({"qkv_dtype": 3}, _lib.YB_E_UNSUPPORTED), ({"qkv_dtype": -1}, _lib.YB_E_UNSUPPORTED),
    ({"rotary_dim": 66}, _lib.YB_E_INVALID), ({"rotary_dim": 3}, _lib.YB_E_INVALID),
    ({"rotary_dim": -2}, _lib.YB_E_INVALID), ({"rotary_dim": 36, "half": 1}, _lib.YB_E_INVALID),
    ({"inv_freq": None}, _lib.YB_E_INVALID), ({"eps": -1.0}, _lib.YB_E_INVALID),
    ({"eps": float("nan")}, _lib.YB_E_INVALID), ({"clip": 0.0}, _lib.YB_E_INVALID),
    ({"clip": float("nan")}, _lib.YB_E_INVALID)])
def test_bad_append_arguments_are_refused(kw, code):
    assert _append(_batch(), **kw) == code
    assert _lib.last_error()


@pytest.mark.parametrize("kw", [
    {"out": None}, {"q": None}, {"out": P + 4}, {"q": P + 8}, {"out_stride": 504}, {"q_stride": 500},
    {"q_stride": 516}, {"scale": 0.0}, {"scale": -1.0}, {"scale": float("nan")}, {"scale": float("inf")},
    {"window": -1}, {"scratch": None}, {"scratch": P + 8}])
def test_bad_attention_arguments_are_refused(kw):
    assert _attend(_batch(), **kw) == _lib.YB_E_INVALID
    assert _lib.last_error()


def test_null_batch_is_refused():
    assert _append(None) == _lib.YB_E_INVALID
    assert _attend(None) == _lib.YB_E_INVALID
    assert _lib.lib().yb_paged_attention_scratch_bytes(None) == 0


def test_empty_batches_need_no_gpu():
    """No sequence or no row: nothing to launch."""
    for kw in ({"n_seqs": 0}, {"n_tokens": 0}):
        assert _append(_batch(**kw)) == 0
        assert _attend(_batch(**kw)) == 0


def test_empty_tensors_need_no_gpu():
    """Tensors without elements have no address; their batch is empty, not refused."""
    import torch

    from yalm_b200 import PagedBatch
    k, i32 = torch.zeros(3, 2, 16, 64, dtype=torch.float16), dict(dtype=torch.int32)
    for n_seqs, n_tokens in ((0, 0), (2, 0), (0, 4)):
        b = PagedBatch(k, k.clone(), torch.zeros(n_seqs, 4, **i32), torch.zeros(n_seqs + 1, **i32),
                       torch.zeros(n_seqs, **i32), 8, n_tokens)
        q = torch.zeros(n_tokens, 512, dtype=torch.float16)
        b.append(torch.zeros(n_tokens, 768), q, torch.zeros(32), 64)
        b.attend(q, q.clone(), torch.zeros(b.scratch_bytes(), dtype=torch.uint8))


def test_more_key_tiles_than_a_block_can_count_are_refused():
    big = dict(n_seqs=65536, n_tokens=65536, n_heads=512, n_kv_heads=512, max_pages=(1 << 21) // 16)
    assert _attend(_batch(**big), out_stride=512 * 64, q_stride=512 * 64) == _lib.YB_E_UNSUPPORTED
    assert "too many slots" in _lib.last_error()
    big["n_seqs"], big["n_tokens"] = 4096, 0  # the same table for fewer sequences
    assert _attend(_batch(**big), out_stride=512 * 64, q_stride=512 * 64) == 0


def test_descriptor_matches_the_header():
    """The ctypes structure has the header's fields in the header's order."""
    import re
    src = open(_lib.HEADER).read()
    body = re.search(r"typedef struct yb_paged_batch \{(.*?)\} yb_paged_batch;", src, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    names = re.findall(r"(\w+);", body)
    assert names == [n for n, _ in _lib.yb_paged_batch._fields_]
    assert ctypes.sizeof(_lib.yb_paged_batch) == 9 * 4 + 4 + 5 * 8


def test_batch_class_refuses_wrong_tensors():
    import torch

    from yalm_b200 import PagedBatch
    k = torch.zeros(3, 2, 16, 64, dtype=torch.float16)
    i32 = dict(dtype=torch.int32)
    ok = (k, k.clone(), torch.zeros(2, 1, **i32), torch.zeros(3, **i32), torch.zeros(2, **i32))
    b = PagedBatch(*ok, 8, 4)
    assert b.c.n_seqs == 2 and b.c.page_size == 16 and b.c.max_pages == 1 and b.c.n_pages == 3

    def swapped(i, t):
        return tuple(t if j == i else x for j, x in enumerate(ok))

    for bad in (swapped(1, k.float()), swapped(1, k[:2]), swapped(2, torch.zeros(2, 1)), swapped(3, torch.zeros(2, **i32)),
                swapped(4, torch.zeros(2)), swapped(0, k.transpose(1, 2)), swapped(2, torch.zeros(2, **i32)),
                swapped(0, k.double())):
        with pytest.raises(ValueError):
            PagedBatch(*bad, 8, 4)
    with pytest.raises(ValueError):
        b.attend(torch.zeros(4, 512), torch.zeros(4, 512), torch.zeros(1))
    with pytest.raises(ValueError):
        b.append(torch.zeros(4, 768), torch.zeros(4, 500, dtype=torch.float16), torch.zeros(32), 64)
    with pytest.raises(ValueError):
        b.append(torch.zeros(4, 768), torch.zeros(4, 512, dtype=torch.float16), torch.zeros(31), 64)
