"""``qk_norm_rope`` writing long chunks into a cache, and inside a captured graph.

The chunks are long enough for a lane group to go through several heads of its token (query,
key and value heads in turn, their weights, and tokens whose slot is out of range in
between). Compared with the formula in float64 within ``test_gpu_qk_rope``'s tolerance, and
half a step of float16's smallest numbers: among this many outputs some are that small.
"""

from __future__ import annotations

import pytest
import torch

import fpv2
from tests.test_gpu_qk_rope import U, formula, inputs

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def close(got, want, size):
    tol = U[got.dtype] * want.abs() + 24 * 2.0**-24 * size + (2.0**-25 if got.dtype == torch.float16 else 0)
    return bool(((got.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("tokens,hq,hkv,dim,rot,page,dtype", [
    (4001, 8, 2, 128, 128, 16, torch.bfloat16),    # 16-byte packs
    (4001, 12, 4, 80, 40, 24, torch.float16),      # 8-byte packs, lanes past the head's end
    (3500, 10, 2, 64, 64, 5, torch.float16),
    (3000, 6, 1, 256, 128, 64, torch.bfloat16),
    (3000, 5, 3, 96, 64, 16, torch.float32),
])
@pytest.mark.parametrize("heads_first,interleaved", [(False, False), (True, True), (True, False)])
def test_long_chunks_into_the_cache(tokens, hq, hkv, dim, rot, page, dtype, heads_first, interleaved):
    q, k, v, pos, qw, kw = inputs(tokens, hq, hkv, dim, dtype, seed=dim + page)
    table = fpv2.rope_table(500, rot, theta=1e6, device=DEV)
    pages = tokens // page + 3
    gen = torch.Generator().manual_seed(page)
    slots = torch.randperm(pages * page, generator=gen)[:tokens]
    slots[5::97] = -1
    slots[6::501] = pages * page
    slots = slots.to(DEV)
    kc = torch.full((pages, page, hkv, dim), 7.0, dtype=dtype, device=DEV)
    vc = torch.full((pages, 2, page, hkv, dim), 7.0, dtype=dtype, device=DEV)   # pages apart
    gq, none = fpv2.qk_norm_rope(q, k, pos, table, q_weight=qw, k_weight=kw, eps=1e-5, interleaved=interleaved,
                                 heads_first=heads_first, v=v, k_cache=kc, v_cache=vc[:, 1], slots=slots)
    assert none is None
    assert close(gq.transpose(0, 1) if heads_first else gq, *formula(q, qw, table, pos, 1e-5, interleaved))
    ok = (slots >= 0) & (slots < pages * page)
    want, size = formula(k, kw, table, pos, 1e-5, interleaved)
    flat_k, flat_v = kc.view(-1, hkv, dim), vc[:, 1].reshape(-1, hkv, dim)
    assert close(flat_k[slots[ok]], want[ok], size[ok])
    assert torch.equal(flat_v[slots[ok]], v[ok])
    free = torch.ones(pages * page, dtype=torch.bool, device=DEV)
    free[slots[ok]] = False
    assert bool((flat_k[free] == 7).all()) and bool((flat_v[free] == 7).all()) and bool((vc[:, 0] == 7).all())


@pytest.mark.parametrize("tokens", [3, 4001])
def test_in_a_graph(tokens):
    q, k, v, pos, qw, kw = inputs(tokens, 8, 2, 128, torch.bfloat16, seed=1)
    table = fpv2.rope_table(500, 128, device=DEV)
    caches = torch.zeros(2, tokens // 16 + 1, 16, 2, 128, dtype=torch.bfloat16, device=DEV)
    slots = torch.arange(tokens, device=DEV)

    def call():
        return fpv2.qk_norm_rope(q, k, pos, table, q_weight=qw, v=v, k_cache=caches[0], v_cache=caches[1], slots=slots)[0]

    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    pos.copy_(pos.flip(0))   # the graph follows its inputs
    slots.copy_(slots.flip(0))
    caches.zero_()
    graph.replay()
    mine, kept = got.clone(), caches.clone()
    caches.zero_()
    want = call()
    assert torch.equal(mine, want) and torch.equal(kept, caches) and bool(kept.any())
