"""Which batches the attention over shared prefixes refuses for their size (yb_paged_attention_shared_dev), without a GPU; and
that what it takes can be counted in 31 bits, by the shares that its planning kernel makes."""
import ctypes
import random

import pytest

from yalm_b200 import _lib

P = 4096  # an aligned address that nothing reads


def _batch(**kw):
    c = dict(n_seqs=65536, n_tokens=65536, n_heads=128, n_kv_heads=128, head_dim=64, dtype=1, page_size=16, n_pages=9,
             max_pages=(1 << 21) // 16, q_start_dev=P, kv_len_dev=P, page_table_dev=P, k_pages=P, v_pages=P)
    c.update(kw)
    return _lib.yb_paged_batch(**c)


def _shared(b, n_groups):
    w = b.n_heads * b.head_dim
    return _lib.lib().yb_paged_attention_shared_dev(ctypes.byref(b), n_groups, P, P, P, w, P, w, 0.125, P, None)


def test_batches_whose_warps_could_have_too_many_steps():
    """A fifth of what one SM may have without prefixes: the planning kernel may leave few SMs for single tokens."""
    size = _lib.lib().yb_paged_attention_shared_scratch_bytes
    for b, ok in ((_batch(), False), (_batch(n_seqs=2048, n_tokens=2048), True), (_batch(max_pages=1 << 14), True)):
        assert _lib.lib().yb_paged_attention_scratch_bytes(ctypes.byref(b)) > 0
        assert (size(ctypes.byref(b), 1) > 0) == ok
        if not ok:
            assert _shared(b, 1) == _lib.YB_E_UNSUPPORTED and "on this device" in _lib.last_error()


@pytest.mark.parametrize("head_dim", [64, 128])
def test_shares_of_what_is_taken_fit(head_dim):
    """The planning kernel's choice of SMs (paged_shared.cu) for work at the limit, split in every way between key tiles and
    steps of few rows, of which a unit of one tile has 8."""
    grid, most = 148, (2 ** 31 - 1) // 5 * 148
    step = 1.0 if head_dim == 128 else 0.6
    r = random.Random(head_dim)
    worst = 0
    for i in range(400):
        tiles = int(most * (1 - 10 ** r.uniform(-5, 0))) if i else 0
        few = 8 * (most - tiles)
        best, blocks = float("inf"), 0
        for n in range(grid + 1):
            a = 6 + 2.2 * tiles / n if n else (float("inf") if tiles else 0)
            b = 3 + few * step * 0.136 / (grid - n) if n < grid else (float("inf") if few else 0)
            t = max(a, b, few * step * 0.0013)
            if t < best:
                best, blocks = t, n
        worst = max(worst, tiles / max(blocks, 1), few / (12 * max(grid - blocks, 1)))
    assert worst < 2 ** 31 - 1
