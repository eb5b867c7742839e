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


@pytest.mark.parametrize("V", [4096, 40000])
def test_a_sum_that_is_just_the_coins_share(gpu, V):
    """A row whose second half repeats its first: with coin 1/2 the sum up to the middle is the share, to the last unit.
    Half of such sums have more than the 53 bits of a 64-bit number and would be rounded up past the middle."""
    import torch
    R = 64
    tokens = torch.full((R,), -1, dtype=torch.int32, device="cuda")
    for seed in range(4):
        x = torch.cat([_logits(R, V // 2, "f32", 77 + seed, 0.05, peaks=False)] * 2, 1)
        sample_rows(x, torch.full((R,), 0.5, device="cuda"), tokens)
        assert tokens.tolist() == [V // 2 - 1] * R, seed


@pytest.mark.parametrize("coin", [2.0 ** -149, 2.0 ** -126, 1e-40, 2.0 ** -64, 2.0 ** -41, 1e-12, 1.0 - 2.0 ** -24, 0.5 + 2.0 ** -24])
def test_coins_of_every_exponent(gpu, coin):
    """The smallest numbers, numbers that have no bit above the sum's last one, and the largest below 1."""
    x = _logits(6, 30001, "f32", 91, 0.3)
    _check(x, [coin] * 6)
    _check(x, [coin] * 6, top_p=[coin] * 3 + [0.9] * 3)
