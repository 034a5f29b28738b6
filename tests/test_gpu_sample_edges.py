"""``sample_tokens`` at the largest temperatures: the comparison and its tolerances are
``test_gpu_sample.check``'s.
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
