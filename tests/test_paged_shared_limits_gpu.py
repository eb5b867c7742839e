"""Attention over shared prefixes (yb_paged_attention_shared_dev) at its largest sizes and at the edges of its rules,
against the definition in 64 bits with the tolerances of test_paged_gpu."""
import math

import pytest

from test_paged_gpu import TINY, U
from yalm_b200 import PagedBatch

pytestmark = pytest.mark.gpu


def test_room_for_the_most_tokens_and_heads(gpu):
    """65536 sequences, 2^20 rows and 16 query heads of a kv head of 128: records of 2^24 rows, whose maxima lie 2^31
    floats behind their sums.  A few sequences have a token each, the first of all among them."""
    import torch
    S, rows, hd, ps, prefix, live = 65536, 1 << 20, 128, 256, 1024, 40
    g = torch.Generator(device="cuda").manual_seed(31)
    i32 = dict(dtype=torch.int32, device="cuda")
    n_pages = prefix // ps + live
    k, v = (torch.randn(n_pages, 1, ps, hd, generator=g, device="cuda").half() for _ in range(2))
    table = torch.full((S, prefix // ps + 1), -1, **i32)
    table[:live, : prefix // ps] = torch.arange(prefix // ps, **i32)
    table[:live, prefix // ps] = torch.arange(prefix // ps, n_pages, **i32)
    kv_len = torch.zeros(S, **i32)
    kv_len[:live] = prefix + 1 + torch.arange(live, **i32) * 5
    q_start = torch.arange(S + 1, **i32).clamp(max=live)
    b = PagedBatch(k, v, table, q_start, kv_len, 16, rows)
    q = torch.zeros(rows, 16 * hd, dtype=torch.float16, device="cuda")
    q[:live] = torch.randn(live, 16 * hd, generator=g, device="cuda").half()
    out = torch.full((rows, 16 * hd), 7.0, dtype=torch.float16, device="cuda")
    scratch = torch.empty(b.shared_scratch_bytes(1), dtype=torch.uint8, device="cuda")
    scratch[:4] = 0
    b.attend_shared(q, out, scratch, torch.tensor([0, live], **i32), torch.tensor([prefix], **i32))
    assert b.status(scratch) == 0
    for s in range(live):
        n = int(kv_len[s])
        keys, values = (x[table[s].long(), 0].reshape(-1, hd)[:n].double() for x in (k, v))
        qs = q[s].double().view(16, hd)
        w = torch.softmax(qs @ keys.T / math.sqrt(hd), -1)
        mag = (qs.abs() @ keys.abs().T).amax(-1, keepdim=True) / math.sqrt(hd)
        o, u = w @ values, U["f16"]
        tol = u * o.abs() + (u + 2.0 ** -16 + 2 * 2.0 ** -20 * mag) * (w @ values.abs()) + TINY
        assert ((out[s].double().view(16, hd) - o).abs() <= tol).all(), s
    assert (out[live:] == 7).all()


@pytest.mark.parametrize("width", [8, 60000])  # of the table: prefixes are computed apart with the second
@pytest.mark.parametrize("host", ["group_start", "prefix_len"])
def test_groups_are_the_devices_memory_whatever_the_batch(gpu, width, host):
    import torch
    from yalm_b200 import _lib
    i32 = dict(dtype=torch.int32, device="cuda")
    k = torch.zeros(8, 2, 16, 64, dtype=torch.float16, device="cuda")
    b = PagedBatch(k, k.clone(), torch.zeros(3, width, **i32), torch.arange(4, **i32), torch.full((3,), 20, **i32), 4, 3)
    q = torch.zeros(3, 256, dtype=torch.float16, device="cuda")
    out, scratch = torch.empty_like(q), torch.zeros(b.shared_scratch_bytes(1), dtype=torch.uint8, device="cuda")
    t = dict(group_start=torch.tensor([0, 3], **i32), prefix_len=torch.tensor([16], **i32))

    def call():
        return _lib.lib().yb_paged_attention_shared_dev(b._ref, 1, t["group_start"].data_ptr(), t["prefix_len"].data_ptr(),
                                                        out.data_ptr(), 256, q.data_ptr(), 256, 0.125, scratch.data_ptr(), None)
    torch.cuda.synchronize()
    assert call() == 0 and b.status(scratch) == 0
    t[host] = t[host].cpu()
    assert call() == _lib.YB_E_INVALID and host in _lib.last_error()
