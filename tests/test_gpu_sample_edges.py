"""``sample_tokens`` at the ends of the temperatures' range and among thousands of ties.

The comparison and its tolerances are ``test_gpu_sample.check``'s. A row's noise is small at
one token alone, so the row answers whether that token is kept.
"""

from __future__ import annotations

import math

import pytest
import torch

import fpv2
from tests.test_gpu_sample import check, inputs

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
INF = math.inf
MOST = torch.finfo(torch.float32).max


def probed(values, ranks, seed):
    """Rows of the same shuffled logits; row r's noise singles out the token of rank ranks[r]."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.cat([torch.full((n,), v) for v, n in values])
    x = x[torch.randperm(len(x), generator=gen)]
    order = torch.sort(x.double(), descending=True, stable=True).indices
    noise = torch.empty(len(ranks), len(x)).exponential_(generator=gen).clamp_min_(0.5)
    noise[torch.arange(len(ranks)), order[torch.tensor(ranks)]] = 1e-20
    return x.expand(len(ranks), -1).contiguous(), noise.to(DEV)


def kept(values, p, heat, k):
    """How many tokens the nucleus of the first k holds, float64."""
    x = torch.cat([torch.full((n,), v) for v, n in values]).double()
    x = x.sort(descending=True).values[:k or None]
    w = ((x - x[0]) / heat).exp()
    return int((torch.cumsum(w, 0) - w < p * w.sum()).sum())


@pytest.mark.parametrize("rows,vocab", [(6, 9001), (6, 151937)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heat", [7e37, 1e38, MOST])
def test_unfiltered_rows_at_the_largest_temperatures(rows, vocab, dtype, heat):
    logits, noise = inputs(rows, vocab, dtype, seed=vocab)
    logits[1, ::3] = -INF
    logits[2, ::3] = torch.finfo(dtype).min
    logits[3, ::5] = math.nan
    logits[4] = -INF
    logits[5, 3::1000] = INF
    check(logits, noise, temperature=heat)
    tokens, logprobs = fpv2.sample_tokens(logits, noise, temperature=MOST, return_logprobs=True)
    for endless in (INF, torch.full((rows,), INF, device=DEV)):   # as the largest number
        got, lp = fpv2.sample_tokens(logits, noise, temperature=endless, return_logprobs=True)
        assert torch.equal(got, tokens) and torch.equal(lp, logprobs)


@pytest.mark.parametrize("settings", [
    dict(top_p=0.7), dict(top_p=0.5, min_p=0.4), dict(min_p=0.5), dict(top_k=7), dict(top_k=4999, top_p=0.4),
    dict(top_k=300, top_p=0.9),
])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heat", [1e38, MOST])
def test_filters_at_the_largest_temperatures(dtype, settings, heat):
    logits, noise = inputs(5, 9001, dtype, seed=3)
    logits[1, ::3] = -INF
    logits[2, ::3] = torch.finfo(dtype).min
    logits[4] = -INF
    check(logits, noise, temperature=heat, **settings)
    tokens = fpv2.sample_tokens(logits, noise, temperature=MOST, **settings)
    assert torch.equal(fpv2.sample_tokens(logits, noise, temperature=INF, **settings), tokens)


@pytest.mark.parametrize("values,heat,p,k", [
    ([(0.05, 1), (0.035, 4000), (-0.004, 4000)], 1.0, 0.52, 0),     # both sides of zero
    ([(0.04, 3000), (0.03125, 3000), (0.015625, 3000)], 1.0, 0.5, 0),
    ([(0.04, 3000), (0.0, 3000), (-0.03, 3000)], 1.0, 0.9, 0),
    ([(3.0, 2), (0.003, 5000), (-0.002, 5000), (-1e-5, 3000)], 0.9, 0.8, 0),
    ([(0.05, 1), (0.035, 4000), (-0.004, 4000)], 1.0, 0.55, 7500),  # of the first k
    ([(0.05, 1), (0.035, 4000), (-0.004, 4000)], 1.0, 0.9999, 7500),
    ([(1e-3 * (50 - i), 211) for i in range(100)], 1.0, 0.63, 0),
    ([(1e-3 * (50 - i), 211) for i in range(100)], 1.0, 0.63, 20001),
    ([(0.25 * (4 - i), 4500) for i in range(9)], 0.7, 0.6, 0),
    ([(0.0, 9000)], 1.0, 0.37, 0),
])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("more_rows", [False, True])   # few CTAs a row
def test_the_nucleus_of_thousands_of_ties(values, heat, p, k, dtype, more_rows):
    if dtype == torch.float16:
        values = [(float(torch.tensor(v).half()), n) for v, n in values]
    count = kept(values, p, heat, k)
    total = sum(n for _, n in values)
    ranks = [min(max(count + d, 0), total - 1) for d in (-300, -40, -9, -3, -2, -1, 0, 1, 2, 8, 39, 299)]
    logits, noise = probed(values, ranks * (12 if more_rows else 1), seed=count)
    check(logits.to(dtype).to(DEV), noise, temperature=heat, top_p=p, top_k=k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_nucleus_that_ends_past_32_nats(dtype):
    """2^26 tokens of e^-32.25 each weigh 6.6e-7 of the first one, more than 1 - top_p."""
    vocab, p = 2**26, 1 - 2.0**-24
    x = torch.full((3, vocab), -32.25, dtype=dtype, device=DEV)
    x[:, 12345] = 0
    noise = torch.ones(3, vocab, device=DEV)
    w = math.exp(-32.25)
    count = math.ceil((p * (1 + (vocab - 1) * w) - 1) / w)   # of the equal ones that are kept, lowest first
    for r, rank in enumerate((1_000_000, count - vocab // 100, count + vocab // 100)):
        noise[r, rank if rank < 12345 else rank + 1] = 1e-30
    got = fpv2.sample_tokens(x, noise, top_p=p).tolist()
    assert got == [1_000_001, count - vocab // 100 + 1, 12345]
