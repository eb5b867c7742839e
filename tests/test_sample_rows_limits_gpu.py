"""The sampler for rows of logits (yb_sample_rows_dev) where the blocks of a row and the borders of its sums meet, against
the definition of test_sample_rows_gpu."""
import numpy as np
import pytest

from test_sample_rows_gpu import _check, _logits
from yalm_b200 import sample_rows

pytestmark = pytest.mark.gpu


def _likely(R, V, dtype, seed, n):
    """Rows of which n tokens hold nearly all of the weight."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = _logits(R, V, "f32", seed, 1.0, peaks=False)
    at = torch.rand(R, V, generator=g, device="cuda").argsort(1)[:, :n]
    return x.scatter(1, at, 14 + torch.randn(R, n, generator=g, device="cuda")).to(getattr(torch, dtype))


@pytest.mark.parametrize("R,V,dtype", [(1, 32000, "float32"), (7, 60001, "bfloat16"), (61, 49999, "float32"), (120, 60000, "float16"),
                                       (300, 20000, "float32")])
def test_top_p_among_hundreds_repeats(gpu, R, V, dtype):
    """Rows that the first block finishes by itself, with more tokens than are compared each with each, while the others of
    its cluster leave: in 1 to 8 blocks a row, often."""
    import torch
    x = _likely(R, V, dtype, R, 900)
    rng = np.random.default_rng(R)
    p = [(0.9, 0.5, 0.99, 0.7)[r % 4] for r in range(R)]
    coin = rng.random(R).astype(np.float32)
    _check(x, coin.tolist(), top_p=p)
    coins, ps = torch.from_numpy(coin).cuda(), torch.tensor(p, device="cuda")
    runs = torch.full((200, R), -1, dtype=torch.int32, device="cuda")
    for out in runs:
        sample_rows(x, coins, out, top_p=ps)
    torch.cuda.synchronize()
    assert (runs == runs[0]).all() and (runs[0] >= 0).all()
