"""``decode_attention`` where infinities are seen, against float64."""

from __future__ import annotations

import math

import pytest
import torch

import fpv2
from tests.test_gpu_decode import problem

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


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
