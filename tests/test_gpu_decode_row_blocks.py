"""``decode_attention`` with every number of row blocks and row groups a head dimension has,
against the formula in float64 (``test_gpu_decode.check``)."""

from __future__ import annotations

import pytest
import torch

import fpv2
from tests.test_gpu_decode import check, problem

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths,new,hq,hkv,dim,page,window,sinks", [
    ([900, 31], 3, 16, 4, 64, 16, 0, 0),       # 12 rows a KV head: two blocks
    ([900, 31, 2], 3, 20, 2, 64, 32, 70, 3),   # 30: four blocks
    ([900, 31], 7, 40, 4, 64, 16, 0, 0),       # 70: three groups of four blocks
    ([900, 31], 3, 16, 4, 96, 16, 0, 0),
    ([3000, 31, 4], 5, 24, 4, 96, 24, 64, 2),  # 30: two groups of two blocks
    ([900, 31], 3, 16, 4, 256, 16, 0, 0),
    ([3000, 31, 4], 5, 24, 4, 256, 20, 64, 2),
    ([900, 31], 12, 32, 4, 128, 16, 0, 0),     # 96: six groups
])
def test_row_blocks(lengths, new, hq, hkv, dim, page, window, sinks, dtype):
    q, k, v, tables, n = problem(lengths, new, hq, hkv, dim, page, dtype, seed=new + dim)
    out, lse = fpv2.decode_attention(q, k, v, tables, n, scale=dim ** -0.5, window=window, sinks=sinks,
                                     return_lse=True)
    check(q, k, v, tables, n, dim ** -0.5, window, sinks, out, lse)
