"""The sampler for rows of logits (yb_sample_rows_dev) against its definition: weights in 64 bits, rounded to
multiples of 2^-43 of the largest, then whole numbers, whose sums are exact.  Tokens have to be equal.

A weight of 64 bits may be off by a few units of its last place on either side, which moves the rounded one by a
unit where it lies within 2^-50 of a half: nothing that a token here hangs on.  Probabilities: two exact sums, one
division in 64 bits and the rounding to fp32, 2^-24 relative; 2^-42 absolute covers a unit in the smallest weights."""
import math

import numpy as np
import pytest

from yalm_b200 import YalmB200Error, sample_rows

pytestmark = pytest.mark.gpu

ONE = 2.0 ** 43


def _dt(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def _share(x, total):
    """The least whole number that is at least x * total, 1 .. total."""
    if not x > 0:
        return 1
    if x >= 1:
        return total
    n, d = float(x).as_integer_ratio()
    return min(max(-(-n * total // d), 1), total)


def _one(x, coin, T, k, p, least):
    """(token, probability) of one row."""
    x = np.where(np.isnan(x), -np.inf, x)
    m = x.max()
    if m == -np.inf:
        return 0, 0.0
    if not T > 0:
        return int(np.argmax(x)), 1.0
    T = min(max(T, 2.0 ** -60), 2.0 ** 90)
    with np.errstate(all="ignore"):
        w = (x == m).astype(np.float64) if m == np.inf else np.exp((x - m) / T)
    n = np.rint(w * ONE).astype(np.uint64)
    if 0 < k < len(x) or p < 1:
        order = np.lexsort((np.arange(len(x)), -x))
        order = order[n[order] > 0]
        if 0 < k < len(x):
            order = order[:k]
        run = np.cumsum(n[order])
        if p < 1:
            order = order[: int(np.searchsorted(run, np.uint64(_share(p, int(run[-1]))))) + 1]
        only = np.zeros_like(n)
        only[order] = n[order]
        n = only
    if least > 0:
        n[w < min(least, 1.0)] = 0
    run = np.cumsum(n)
    total = int(run[-1])
    t = int(np.searchsorted(run, np.uint64(_share(coin, total))))
    return t, int(n[t]) / total


def _run(x, coin, **par):
    import torch
    R = x.shape[0]
    ten = {k: None if v is None else torch.tensor(v, dtype=torch.int32 if k == "top_k" else torch.float32, device="cuda")
           for k, v in par.items()}
    tokens, prob = torch.full((R,), -9, dtype=torch.int32, device="cuda"), torch.full((R,), -9.0, device="cuda")
    sample_rows(x, torch.tensor(coin, dtype=torch.float32, device="cuda"), tokens, prob=prob, **ten)
    torch.cuda.synchronize()
    return tokens.tolist(), prob.tolist()


def _check(x, coin, **par):
    R = x.shape[0]
    tokens, prob = _run(x, coin, **par)
    x64 = x.float().cpu().numpy().astype(np.float64)
    f32 = lambda v: [float(np.float32(c)) for c in v]
    col = lambda name, other: f32(par[name]) if par.get(name) is not None else [other] * R
    k = par.get("top_k") or [0] * R
    for r, (c, T, p, least) in enumerate(zip(f32(coin), col("temperature", 1.0), col("top_p", 1.0), col("min_p", 0.0))):
        t, q = _one(x64[r].copy(), c, T, k[r], p, least)
        assert tokens[r] == t, (r, tokens[r], t, dict(c=c, T=T, k=k[r], p=p, least=least))
        assert abs(prob[r] - q) <= 2.0 ** -24 * q + 2.0 ** -42, (r, prob[r], q)


def _logits(R, V, dtype, seed, spread=2.0, peaks=True):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(R, V, generator=g, device="cuda") * spread
    if peaks:
        at = torch.randint(0, V, (R, min(V, 30)), generator=g, device="cuda")
        x = x.scatter(1, at, torch.rand(at.shape, generator=g, device="cuda") * 9 + 2)
    return x.to(_dt(dtype))


KINDS = {  # each row takes the next of every list
    "plain": {},
    "temperature": dict(temperature=[0.3, 0.0, 1.0, 1.7, 5.0]),
    "top_k": dict(top_k=[1, 2, 50, 0, 1000, 7]),
    "top_p": dict(top_p=[0.9, 0.1, 0.99, 1.0, 0.5]),
    "min_p": dict(min_p=[0.05, 0.5, 0.0, 1.0, 0.001]),
    "all": dict(temperature=[0.7, 1.0, 1.4, 0.0], top_k=[40, 0, 300, 5, 100000], top_p=[0.95, 0.8, 1.0], min_p=[0.0, 0.1]),
}


@pytest.mark.parametrize("kind", sorted(KINDS))
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("R,V", [(3, 1), (5, 2), (4, 31), (6, 33), (17, 1000), (5, 4096), (5, 4097), (9, 32000), (7, 50001),
                                 (12, 131072), (160, 8193)])
def test_rows_match_the_definition(gpu, kind, dtype, R, V):
    rng = np.random.default_rng(R * V)
    par = {k: [v[r % len(v)] for r in range(R)] for k, v in KINDS[kind].items()}
    _check(_logits(R, V, dtype, R + V), rng.random(R).tolist(), **par)


@pytest.mark.parametrize("kind", ["all", "top_p", "plain"])
@pytest.mark.parametrize("R,V,dtype", [(260, 20000, "f32"), (256, 32000, "bf16"), (300, 60000, "f32"), (300, 131072, "f16")])
def test_batches_of_many_rows(gpu, kind, R, V, dtype):
    """As many rows as take one or two blocks each, staged in shared memory or not."""
    rng = np.random.default_rng(R + V)
    par = {k: [v[r % len(v)] for r in range(R)] for k, v in KINDS[kind].items()}
    _check(_logits(R, V, dtype, 9), rng.random(R).tolist(), **par)


@pytest.mark.parametrize("V", [300000, 1 << 20])  # longer than shared memory takes
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_long_rows(gpu, dtype, V):
    rng = np.random.default_rng(V)
    par = {k: [v[r % len(v)] for r in range(8)] for k, v in KINDS["all"].items()}
    _check(_logits(8, V, dtype, 7), rng.random(8).tolist(), **par)


def test_batches_of_long_rows(gpu):
    """As many rows as there are places for blocks, each longer than the 2^17 logits whose weights a block's sums hold."""
    import torch
    R, V = 290, 1 << 20
    x = torch.zeros(R, V, dtype=torch.bfloat16, device="cuda")
    x[1::2] = _logits(1, V, "bf16", 8, 1e-2, peaks=False)
    rng = np.random.default_rng(8)
    coin, p = rng.random(R).tolist(), [(0.5, 0.9, 1.0, 0.3)[r // 2 % 4] for r in range(R)]
    tokens, prob = _run(x, coin, top_p=p)
    for r in (0, 1, 2, 3, 4, 5, 6, 7, 144, 145, 288, 289):
        t, q = _one(x[r].float().cpu().numpy().astype(np.float64), float(np.float32(coin[r])), 1.0, 0, float(np.float32(p[r])), 0.0)
        assert tokens[r] == t and abs(prob[r] - q) <= 2.0 ** -24 * q + 2.0 ** -42, (r, tokens[r], t, prob[r], q)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("spread", [0.0, 1e-3, 0.02, 0.5])
def test_limits_among_many_tokens_alike(gpu, dtype, spread):
    """Tens of thousands of tokens in one bin: the place is narrowed down by value, then by index."""
    R, V = 8, 100003
    x = _logits(R, V, dtype, 11, spread, peaks=False)
    rng = np.random.default_rng(3)
    _check(x, rng.random(R).tolist(), top_p=[0.5, 0.01, 0.999, 0.3, 0.9, 0.7, 0.2, 0.6])
    _check(x, rng.random(R).tolist(), top_k=[5000, 2048, 2049, 99999, 100002, 1, 60000, 30000])
    _check(x, rng.random(R).tolist(), top_k=[5000, 2048, 2049, 99999, 100002, 1, 60000, 30000],
           top_p=[0.5, 0.01, 0.999, 0.3, 0.9, 0.7, 0.2, 0.6], min_p=[0.0, 0.99] * 4)


def test_equal_weights_share_evenly(gpu):
    import torch
    x = torch.full((9, 4), -3.25, device="cuda")
    coin = [0.0, 0.1, 0.25, 0.2500001, 0.5, 0.75, 0.76, 0.9999999, 1.0]
    assert _run(x, coin)[0] == [0, 0, 0, 1, 1, 2, 3, 3, 3]
    assert _run(x, coin, top_p=[0.5] * 9)[0] == [0, 0, 0, 0, 0, 1, 1, 1, 1]  # ties go to the lowest index
    assert _run(x, coin, top_k=[3] * 9)[0] == [0, 0, 0, 0, 1, 2, 2, 2, 2]
    assert _run(x, coin, min_p=[1.0] * 9)[0] == [0, 0, 0, 1, 1, 2, 3, 3, 3]
    assert _run(x, coin, temperature=[0.0] * 9) == ([0] * 9, [1.0] * 9)


INF, NAN = math.inf, math.nan


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [64, 9000])
def test_masked_and_infinite_logits(gpu, dtype, V):
    import torch
    lowest = torch.finfo(_dt(dtype)).min
    rows = []
    for fill, some in ((-INF, [(3, 1.0)]), (-INF, [(5, 0.5), (V - 1, 0.25), (9, NAN)]), (NAN, [(V - 2, -7.0)]),
                       (lowest, [(7, 1.0), (11, 0.0)]), (lowest, []), (-INF, []), (NAN, []), (1.0, [(4, INF), (40, INF)]),
                       (-INF, [(6, INF)]), (NAN, [(2, INF), (3, -INF)]), (0.0, [(1, -0.0)]), (-INF, [(8, lowest)]),
                       (-INF, [(V - 1, torch.finfo(_dt(dtype)).max), (0, lowest)])):
        x = torch.full((V,), fill)
        for i, v in some:
            x[i] = v
        rows.append(x)
    x = torch.stack(rows).to(_dt(dtype)).cuda()
    R = x.shape[0]
    rng = np.random.default_rng(V)
    for par in ({}, dict(temperature=[0.0] * R), dict(top_k=[2] * R), dict(top_p=[0.6] * R, top_k=[1] * R),
                dict(min_p=[0.4] * R), dict(temperature=[INF] * R), dict(temperature=[1e-38] * R, top_p=[0.5] * R)):
        for coin in (rng.random(R).tolist(), [1.0] * R):
            _check(x, coin, **par)
    empty = [5, 6]
    tokens, prob = _run(x, [0.5] * R)
    assert [tokens[r] for r in empty] == [0, 0] and [prob[r] for r in empty] == [0.0, 0.0]


def test_settings_out_of_range(gpu):
    x = _logits(7, 5000, "f32", 21)
    odd = [NAN, -1.0, 0.0, 2.0, INF, -INF, 0.3]
    k = [-3, 0, 5000, 6000, 2 ** 31 - 1, -2 ** 31, 4999]
    _check(x, odd)
    _check(x, [0.7] * 7, temperature=odd)
    _check(x, [0.7] * 7, top_k=k)
    # (a NaN is no limit)
    for name in ("top_p", "min_p"):
        tokens, prob = _run(x, [0.7] * 7, **{name: odd})
        clean, clean_prob = _run(x, [0.7] * 7, **{name: [1.0 if name == "top_p" else 0.0] + odd[1:]})
        assert tokens == clean and prob == clean_prob
        _check(x[1:], [0.7] * 6, **{name: odd[1:]})


def test_strides_and_alignments(gpu):
    import torch
    rng = np.random.default_rng(5)
    for dtype in ("f32", "f16", "bf16"):
        big = _logits(6, 20011, dtype, 31)
        for x in (big[:, 1:], big[:, 3:20000], big[::2, 5:-2], big[1:2, 7:], big[:, 4:5]):
            par = {k: [v[r % len(v)] for r in range(x.shape[0])] for k, v in KINDS["all"].items()}
            _check(x, rng.random(x.shape[0]).tolist(), **par)
    x = _logits(1, 1000, "f32", 32)
    _check(x.expand(4, 1000)[:1], [0.3])


def test_rows_past_32_bit_offsets(gpu):
    import torch
    x = torch.empty((3, (1 << 30) + 40), dtype=torch.float16, device="cuda")[:, :33000]
    x.copy_(_logits(3, 33000, "f16", 41))
    _check(x, [0.2, 0.5, 0.9], top_p=[0.9] * 3)


def test_many_rows(gpu):
    rng = np.random.default_rng(6)
    R = 3000
    par = {k: [v[r % len(v)] for r in range(R)] for k, v in KINDS["all"].items()}
    _check(_logits(R, 257, "f16", 51), rng.random(R).tolist(), **par)


def test_replayed_graphs_and_two_streams(gpu):
    import torch
    R, V = 20, 32000
    x = _logits(R, V, "f32", 61)
    rng = np.random.default_rng(7)
    coin = torch.zeros(R, device="cuda")
    p, k = torch.full((R,), 0.9, device="cuda"), torch.full((R,), 64, dtype=torch.int32, device="cuda")
    outs = [torch.zeros(R, dtype=torch.int32, device="cuda") for _ in range(2)]
    for o in outs:
        sample_rows(x, coin, o, top_p=p, top_k=k)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        sample_rows(x, coin, outs[0], top_p=p, top_k=k)
    side = torch.cuda.Stream()
    for i in range(4):
        c = rng.random(R).astype(np.float32)
        coin.copy_(torch.from_numpy(c))
        x.copy_(_logits(R, V, "f32", 70 + i))
        torch.cuda.synchronize()
        g.replay()
        with torch.cuda.stream(side):
            sample_rows(x, coin, outs[1], top_p=p, top_k=k)
        torch.cuda.synchronize()
        want = [_one(v.astype(np.float64), float(cc), 1.0, 64, float(np.float32(0.9)), 0.0)[0]
                for v, cc in zip(x.cpu().numpy(), c)]
        assert outs[0].tolist() == want and outs[1].tolist() == want


def test_draws_follow_the_weights(gpu):
    """Evenly spread coins draw every token as often as its probability says, to one in the number of coins."""
    import torch
    R, V = 4096, 40
    row = torch.randn(V, device="cuda", generator=torch.Generator(device="cuda").manual_seed(8)) * 2
    tokens, _ = _run(row.expand(R, V).contiguous(), [(r + 0.5) / R for r in range(R)], top_k=[10] * R)
    n = np.bincount(tokens, minlength=V)
    w = np.exp(row.double().cpu().numpy())
    w[np.argsort(-w)[10:]] = 0
    assert np.abs(n - R * w / w.sum()).max() <= 1.0


def test_refusals(gpu):
    import torch
    x = torch.zeros(2, 8, device="cuda")
    coin, tok = torch.zeros(2, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    for bad in (lambda: sample_rows(x.t(), coin, tok), lambda: sample_rows(x, coin[:1], tok),
                lambda: sample_rows(x, coin, tok.long()), lambda: sample_rows(x, coin.cpu(), tok),
                lambda: sample_rows(x.double(), coin, tok), lambda: sample_rows(x, coin, tok, top_k=coin),
                lambda: sample_rows(x, coin, tok, temperature=coin.double()), lambda: sample_rows(x[0], coin, tok)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(YalmB200Error):
        sample_rows(x.cpu(), coin.cpu(), tok.cpu())  # not memory of the GPU
    with pytest.raises(YalmB200Error):
        sample_rows(x[:1].expand(2, 8), coin, tok)  # rows on top of one another
    sample_rows(x[:0], coin[:0], tok[:0])
