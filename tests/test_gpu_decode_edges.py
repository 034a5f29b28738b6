"""``decode_attention`` where infinities are seen and where weights are small, against float64.

Tolerance: as in ``test_gpu_decode`` but for the weights' 16-bit form, which is two parts
in both types: 2^-16 of a weight in bfloat16, 2^-21 in float16 and there no finer than
2^-32 of a part's largest weight, so n 2^-32 of the largest weight and value in all. A
weight is an exponential of 2^-22 of itself.
"""

from __future__ import annotations

import math

import pytest
import torch

import fpv2
from tests.test_gpu_decode import U, problem

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
DP = {torch.bfloat16: 2.0**-16, torch.float16: 2.0**-21}


def formula(q, k, v, tables, lengths, scale, window=0, sinks=0):
    """(i, t, keys' values, weights, score error, wanted output) of every row, float64."""
    b, new, hq, dim = q.shape
    page, hkv = k.shape[1:3]
    for i, n in enumerate(lengths.tolist()):
        pages = tables[i, :-(-n // page)].long()
        ki = k[pages].flatten(0, 1)[:n].double().repeat_interleave(hq // hkv, 1)
        vi = v[pages].flatten(0, 1)[:n].double().repeat_interleave(hq // hkv, 1)
        at = torch.arange(n, device=DEV)
        for t in range(new):
            p = n - new + t
            sees = at <= p
            if window:
                sees &= (at < sinks) | (at > p - window)
            qt, kt, vt = q[i, t].double(), ki[sees], vi[sees]
            pr = torch.softmax(torch.einsum("hd,lhd->hl", qt, kt) * scale, -1)
            e = dim * 2.0**-23 * abs(scale) * torch.einsum("hd,lhd->hl", qt.abs(), kt.abs()).amax(-1)
            yield i, t, vt, pr, e, torch.einsum("hl,lhd->hd", pr, vt)


def check_weights(q, k, v, tables, lengths, scale, out):
    n_max = int(lengths.max())
    for i, t, vt, pr, e, want in formula(q, k, v, tables, lengths, scale):
        size = torch.einsum("hl,lhd->hd", pr, vt.abs())
        rel = 2 * e + DP[q.dtype] + 2.0**-22 + (n_max / 16 + 160) * 2.0**-23
        tol = U[q.dtype] * want.abs() + rel[:, None] * size
        if q.dtype == torch.float16:
            tol = tol + n_max * 2.0**-32 * pr.amax(-1)[:, None] * vt.abs().amax(0)
        err = (out[i, t].double() - want).abs()
        assert bool((err <= tol).all()), (i, t, float((err / tol).max()))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths,new,hq,hkv,dim,window,sinks", [
    ([40, 3], 1, 8, 2, 128, 0, 0),        # finished by one warp
    ([6000], 1, 8, 2, 128, 0, 0),         # cut into parts and joined
    ([300, 77], 1, 4, 4, 96, 50, 3),
    ([300, 77], 3, 16, 2, 256, 0, 0),     # two row blocks
    ([2000, 60], 4, 64, 8, 64, 100, 4),   # four row blocks, several new tokens
])
def test_infinities_that_a_query_sees(lengths, new, hq, hkv, dim, window, sinks, dtype):
    q, k, v, tables, n = problem(lengths, new, hq, hkv, dim, 16, dtype, seed=dim + new)
    key = [x - new - 5 if x - new > 5 else 0 for x in lengths]   # seen by every row
    for i, j in enumerate(key):
        page, row = int(tables[i, j // 16]), j % 16
        v[page, row, :, 0] = math.inf
        v[page, row, :, 7] = -math.inf
        v[page, row, :, dim - 1] = math.nan
        v[page, row, :, 12] = math.inf
        page, row = int(tables[i, (j + 1) // 16]), (j + 1) % 16
        v[page, row, :, 12] = -math.inf   # both: no value
    scale = dim ** -0.5
    out = fpv2.decode_attention(q, k, v, tables, n, scale=scale, window=window, sinks=sinks)
    for i, t, vt, pr, e, want in formula(q, k, v, tables, n, scale, window, sinks):
        got = out[i, t].double()
        assert torch.equal(got.isnan(), want.isnan()), (i, t)
        assert torch.equal(got == math.inf, want == math.inf) and torch.equal(got == -math.inf, want == -math.inf)
        assert bool(want[:, 0].eq(math.inf).all()) and bool(want[:, 12].isnan().all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths,new,hq,hkv,dim", [
    ([2, 5, 16, 3], 1, 8, 2, 128),
    ([9, 40], 3, 16, 2, 256),
    ([21, 33], 4, 64, 8, 64),
    ([4000, 7], 1, 8, 2, 96),
])
def test_weights_keep_their_bits_where_values_cancel(lengths, new, hq, hkv, dim, dtype):
    q, k, v, tables, n = problem([max(x, new) for x in lengths], new, hq, hkv, dim, 16, dtype, seed=dim)
    scale = dim ** -0.5
    out = fpv2.decode_attention(q, k, v, tables, n, scale=scale)
    check_weights(q, k, v, tables, n, scale, out)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("nats", [12.0, 17.5, 20.0])
def test_one_heavy_key_and_a_long_even_tail(nats, dtype):
    """150 sequences over the same pages, so that a part holds tens of thousands of keys."""
    length, dim, page = 32768, 64, 64
    gen = torch.Generator().manual_seed(7)
    k = 0.05 * torch.randn(length // page, page, 8, dim, generator=gen)
    k[0, 0] = 0
    k[0, 0, :, 0] = nats / 4
    v = 1 + 0.5 * torch.randn(length // page, page, 8, dim, generator=gen)
    v[0, 0] = 0   # what is left is the tail's
    k, v = k.to(dtype).to(DEV), v.to(dtype).to(DEV)
    q = torch.zeros(150, 1, 8, dim, dtype=dtype, device=DEV)
    q[..., 0] = 4
    tables = torch.arange(length // page, dtype=torch.int32, device=DEV).expand(150, -1).contiguous()
    n = torch.full((150,), length, dtype=torch.int32, device=DEV)
    out = fpv2.decode_attention(q, k, v, tables, n, scale=1.0)
    check_weights(q[:1], k, v, tables[:1], n[:1], 1.0, out[:1])
    check_weights(q[-1:], k, v, tables[-1:], n[-1:], 1.0, out[-1:])
