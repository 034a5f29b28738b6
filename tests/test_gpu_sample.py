"""``sample_tokens`` against the definition in float64.

Tokens have to be equal. Where the definition itself hangs on less than float32 can
tell -- the best two scores within 1e-5 of each other, or another token when top_p
moves by 4e-6 of itself or min_p by 1e-5 -- either answer is taken. Log-probabilities:
z within (|z| + 1) 2^-22 and the sum of weights within 2^-18 (150 float32 additions a
thread, exponents to 2^-21).
"""

from __future__ import annotations

import math

import pytest
import torch

import fpv2

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
INF = math.inf


def pick(x, e, heat, k, p, least):
    """(token, runner-up score gap) of one row, float64."""
    x = torch.where(torch.isnan(x), -INF, x)
    if bool((x == -INF).all()):
        return -1, INF
    if not heat > 0:
        return int((x == x.max()).nonzero()[0]), INF
    top = x.max()
    z = torch.where(x == top, 0.0, (x - top) / heat)
    by = torch.sort(x, descending=True, stable=True).indices
    if k > 0:
        by = by[:k]
    w = torch.exp(z[by])
    keep = torch.ones_like(w, dtype=torch.bool)
    if not p >= 1:
        keep &= torch.cumsum(w, 0) - w < p * w.sum()
    if not least <= 0:
        keep &= w >= least
    keep[0] = True
    by = by[keep]
    by = by[z[by] > -INF].sort().values
    noise = e[by]
    score = torch.where(noise > 0, z[by] - torch.log(noise), -3.4e38)
    best = torch.sort(score, descending=True, stable=True)
    gap = float(best.values[0] - best.values[1]) if by.numel() > 1 else INF
    return int(by[best.indices[0]]), gap


def check(logits, noise, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    rows, vocab = logits.shape

    def per_row(value, dtype):
        return value if isinstance(value, torch.Tensor) else torch.full((rows,), value, dtype=dtype, device=DEV)

    heat, k = per_row(temperature, torch.float32), per_row(top_k, torch.int32)
    p, least = per_row(top_p, torch.float32), per_row(min_p, torch.float32)
    got, lp = fpv2.sample_tokens(logits, noise, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p,
                                 return_logprobs=True)
    alone = fpv2.sample_tokens(logits, noise, temperature=heat, top_k=k, top_p=p, min_p=least)
    assert got.dtype == torch.int64 and torch.equal(got, alone)
    x, e = logits.double().cpu(), noise.double().cpu()
    for r in range(rows):
        h, kr, pr, mr = float(heat[r]), int(k[r]), float(p[r]), float(least[r])
        token, gap = pick(x[r], e[r], h, kr, pr, mr)
        mine = int(got[r])
        if mine != token:
            near = {pick(x[r], e[r], h, kr, pr * (1 + a), mr * (1 + b))[0]
                    for a in (-4e-6, 0, 4e-6) for b in (-1e-5, 0, 1e-5)}
            assert gap < 1e-5 or mine in near, (r, mine, token, gap)
        if token < 0:
            assert float(lp[r]) == -INF
            continue
        row = torch.where(torch.isnan(x[r]), -INF, x[r])
        h = h if h > 0 else 1.0
        if float(row.max()) == INF:
            want = -math.log(float((row == INF).sum()))
        else:
            z = (row - row.max()) / h
            want = float(z[mine] - torch.logsumexp(z, 0))
        assert abs(float(lp[r]) - want) <= (abs(want) + 1) * 2.0**-22 + 2.0**-18, (r, float(lp[r]), want)
    return got


def inputs(rows, vocab, dtype, seed, spread=2.5):
    gen = torch.Generator().manual_seed(seed)
    logits = (spread * torch.randn(rows, vocab, generator=gen)).to(dtype).to(DEV)
    noise = torch.empty(rows, vocab).exponential_(generator=gen).clamp_min_(1e-30).to(DEV)
    return logits, noise


@pytest.mark.parametrize("rows,vocab,dtype", [
    (3, 1, torch.float32),
    (2, 5, torch.bfloat16),
    (9, 1000, torch.float16),
    (5, 32001, torch.bfloat16),
    (2, 151936, torch.bfloat16),
    (2, 151937, torch.float32),
    (160, 4099, torch.float16),     # one CTA a row
    (1, 700001, torch.float32),     # more than the clusters hold: read again each time
])
@pytest.mark.parametrize("settings", [
    dict(),
    dict(temperature=0.0),
    dict(temperature=0.7, top_k=50, top_p=0.9),
    dict(top_p=0.9),
    dict(temperature=1.4, top_p=0.5, min_p=0.01),
    dict(min_p=0.1),
    dict(top_k=1500, top_p=0.97),
    dict(top_k=1, top_p=0.2),
    dict(top_k=9000),
])
def test_matches_the_definition(rows, vocab, dtype, settings):
    logits, noise = inputs(rows, vocab, dtype, seed=vocab + rows)
    check(logits, noise, **settings)


def test_settings_for_each_row():
    logits, noise = inputs(24, 20011, torch.bfloat16, seed=1)
    gen = torch.Generator().manual_seed(2)
    check(logits, noise,
          temperature=(torch.rand(24, generator=gen) * 2 - 0.2).clamp_min(0).to(DEV),
          top_k=torch.randint(-1, 3000, (24,), generator=gen, dtype=torch.int32).to(DEV),
          top_p=(torch.rand(24, generator=gen) * 1.2).to(DEV),
          min_p=(torch.rand(24, generator=gen) * 0.2 - 0.1).to(DEV))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("settings", [
    dict(), dict(top_k=7), dict(top_k=4999, top_p=0.4), dict(top_p=0.31), dict(top_k=3, min_p=0.9),
    dict(temperature=0.0), dict(top_p=0.9999999), dict(top_p=1e-9), dict(min_p=1.5),
    dict(top_p=0.0), dict(temperature=1e-3, top_p=0.7), dict(temperature=1e30, top_p=0.7),
])
def test_equal_masked_and_extreme_logits(dtype, settings):
    vocab = 9001
    _, noise = inputs(8, vocab, dtype, seed=4)
    x = torch.zeros(8, vocab)                         # row 0: every logit equal
    x[1] = torch.arange(vocab) % 5                    # five values, 1800 times each
    x[2] = -INF
    x[2, 5000:5010] = 1.0                             # all but ten masked
    x[3] = torch.finfo(dtype).min                     # masked with the lowest value
    x[3, 17::1000] = torch.linspace(-3, 3, 9)
    x[4] = torch.linspace(-8, 8, vocab)
    x[4, ::7] = math.nan
    x[5] = -INF                                       # nothing left
    x[6, 1::4000] = INF                               # three infinite ones
    x[7, ::2] = -0.0                                  # zeros of both signs
    check(x.to(dtype).to(DEV), noise, **settings)


def test_noise_out_of_contract_never_wins_against_good_noise():
    logits, noise = inputs(3, 400, torch.float32, seed=6)
    noise[:, ::2] = 0.0
    noise[:, 1::4] = math.nan
    got = fpv2.sample_tokens(logits, noise)
    assert bool((got % 4 == 3).all())


def test_strides_streams_and_repeats():
    logits, noise = inputs(6, 5003, torch.bfloat16, seed=7)
    wide = torch.zeros(6, 5010, dtype=torch.bfloat16, device=DEV)
    wide[:, 3:5006] = logits
    wide_noise = torch.zeros(6, 5009, device=DEV)
    wide_noise[:, 1:5004] = noise
    want = check(logits, noise, top_p=0.8)
    assert torch.equal(fpv2.sample_tokens(wide[:, 3:5006], wide_noise[:, 1:5004], top_p=0.8), want)
    turned = logits.t().contiguous().t()
    assert torch.equal(fpv2.sample_tokens(turned, noise, top_p=0.8), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fpv2.sample_tokens(logits, noise, top_p=0.8)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    assert fpv2.sample_tokens(logits[:0], noise[:0]).shape == (0,)


def test_draws_follow_the_probabilities():
    # 20000 rows of the same five logits: each share within 5 standard deviations
    rows = 20000
    x = torch.tensor([1.0, 0.0, -1.0, 0.5, -30.0])
    gen = torch.Generator().manual_seed(11)
    noise = torch.empty(rows, 5).exponential_(generator=gen).clamp_min_(1e-30)
    got = fpv2.sample_tokens(x.expand(rows, 5).contiguous().to(DEV), noise.to(DEV), temperature=0.8, top_k=3)
    p = torch.softmax(torch.tensor([1.0, 0.0, 0.5]) / 0.8, 0)
    share = torch.bincount(got.cpu(), minlength=5).double() / rows
    assert float(share[2]) == 0 and float(share[4]) == 0
    for i, at in enumerate((0, 1, 3)):
        assert abs(float(share[at]) - float(p[i])) <= 5 * math.sqrt(float(p[i]) / rows)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 7), (2, 4099), (1, 151937), (40, 30011), (700, 513)])
@pytest.mark.parametrize("temperature", [0.0, 0.6, 1.7])
def test_unfiltered_rows(rows, vocab, dtype, temperature):
    """Whole rows: rising and falling ones (whose running maximum keeps moving), far offsets,
    masked stretches, odd starts in memory."""
    logits, noise = inputs(rows, vocab + 3, dtype, seed=rows + vocab)
    at = torch.arange(vocab + 3, device=DEV) / vocab
    logits[0::4] += (at * 60).to(dtype)
    logits[1::4] -= (at * 60).to(dtype)
    logits[2::4] += 300
    logits[:, : vocab // 3: 2] = -INF
    logits[:, vocab // 2] = math.nan
    check(logits[:, 3:], noise[:, 3:], temperature=temperature)
    check(logits[:, 1:-2], noise[:, 2:-1], temperature=temperature)
