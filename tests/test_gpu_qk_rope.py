"""``qk_norm_rope`` against the formula in float64.

Tolerance: the output's rounding, u |y| with u = 2^-8 (bfloat16), 2^-11 (float16) or
2^-24, plus the float32 arithmetic. The sum of squares takes at most 13 roundings,
halved by the root, the reciprocal root 4, the rest of the norm 3 and the rotation 2,
in units of 2^-24 of the pair's magnitude |a| + |b|: under 24 in all.
"""

from __future__ import annotations

import pytest
import torch

import fpv2
from fpv2 import _lib

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


def formula(x, weight, table, positions, eps, interleaved):
    """(y, |a| + |b|) in float64, dimension by dimension."""
    x = x.double()
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.double()
    rot = table.shape[1]
    pos = positions.long().clamp(0, table.shape[0] - 1)
    out, size = y.clone(), y.abs()
    for i in range(rot // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
        c, s = table[pos, i].double()[:, None], table[pos, rot // 2 + i].double()[:, None]
        out[..., a] = y[..., a] * c - y[..., b] * s
        out[..., b] = y[..., b] * c + y[..., a] * s
        size[..., a] = size[..., b] = y[..., a].abs() + y[..., b].abs()
    return out, size


def close(got, want, size):
    err = (got.double() - want).abs()
    return bool((err <= U[got.dtype] * want.abs() + 24 * 2.0**-24 * size).all())


def inputs(tokens, hq, hkv, dim, dtype, seed, span=500):
    gen = torch.Generator().manual_seed(seed)
    qkv = (torch.randn(tokens, hq + 2 * hkv, dim, generator=gen) * 3).to(dtype).to(DEV)
    pos = torch.randint(0, span, (tokens,), generator=gen, dtype=torch.int32).to(DEV)
    qw = torch.randn(dim, generator=gen).to(dtype).to(DEV)
    kw = torch.randn(dim, generator=gen).to(dtype).to(DEV)
    return qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:], pos, qw, kw


@pytest.mark.parametrize("tokens,hq,hkv,dim,rot,dtype", [
    (1, 32, 8, 128, 128, torch.bfloat16),
    (7, 6, 2, 64, 64, torch.float16),
    (33, 5, 1, 96, 48, torch.float32),
    (3, 8, 8, 256, 128, torch.bfloat16),
    (5, 3, 3, 80, 80, torch.float16),      # 10 chunks of 8, the rotation in halves of 5
    (9, 4, 2, 80, 40, torch.bfloat16),     # a half that is no multiple of 8
    (4, 2, 1, 37, 6, torch.float32),       # nothing divides
    (2, 1, 1, 2, 2, torch.float16),
    (1500, 4, 2, 128, 128, torch.float32),
])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("weights", [False, True])
def test_matches_the_formula(tokens, hq, hkv, dim, rot, dtype, interleaved, weights):
    q, k, _, pos, qw, kw = inputs(tokens, hq, hkv, dim, dtype, seed=tokens + dim)
    table = fpv2.rope_table(500, rot, theta=1e6, device=DEV)
    kwargs = dict(q_weight=qw, k_weight=kw) if weights else {}
    gq, gk = fpv2.qk_norm_rope(q, k, pos, table, eps=1e-5, interleaved=interleaved, **kwargs)
    assert gq.shape == q.shape and gk.shape == k.shape and gq.dtype == dtype
    assert close(gq, *formula(q, qw if weights else None, table, pos, 1e-5, interleaved))
    assert close(gk, *formula(k, kw if weights else None, table, pos, 1e-5, interleaved))
    hq_first, hk_first = fpv2.qk_norm_rope(q, k, pos.long(), table, eps=1e-5, interleaved=interleaved,
                                           heads_first=True, **kwargs)
    assert torch.equal(hq_first, gq.transpose(0, 1)) and torch.equal(hk_first, gk.transpose(0, 1))
    assert hq_first.is_contiguous()


@pytest.mark.parametrize("dim,page,dtype,packed", [
    (128, 16, torch.bfloat16, False),
    (64, 5, torch.float16, True),
    (80, 8, torch.bfloat16, False),
    (30, 4, torch.float32, True),
])
def test_writes_the_cache_and_nothing_else(dim, page, dtype, packed):
    tokens, hq, hkv, pages = 23, 4, 2, 9
    q, k, v, pos, qw, kw = inputs(tokens, hq, hkv, dim, dtype, seed=dim)
    table = fpv2.rope_table(500, dim if dim % 4 == 0 else 6, device=DEV)
    if packed:   # k and v pages interleaved in one pool
        pool = torch.full((pages, 2, page, hkv, dim), 7.0, dtype=dtype, device=DEV)
        kc, vc = pool[:, 0], pool[:, 1]
    else:
        kc = torch.full((pages, page, hkv, dim), 7.0, dtype=dtype, device=DEV)
        vc = kc.clone()
    gen = torch.Generator().manual_seed(3)
    slots = torch.randperm(pages * page, generator=gen)[:tokens]
    slots[4], slots[11], slots[12] = -1, pages * page, -(2**40)   # not written
    slots = slots.to(DEV)
    ref_q, ref_k = fpv2.qk_norm_rope(q, k, pos, table, q_weight=qw, k_weight=kw)
    got_q, none = fpv2.qk_norm_rope(q, k, pos, table, q_weight=qw, k_weight=kw, v=v, k_cache=kc, v_cache=vc,
                                    slots=slots)
    assert none is None and torch.equal(got_q, ref_q)
    want_k = torch.full((pages * page, hkv, dim), 7.0, dtype=dtype, device=DEV)
    want_v = want_k.clone()
    ok = (slots >= 0) & (slots < pages * page)
    want_k[slots[ok]] = ref_k[ok]
    want_v[slots[ok]] = v[ok]
    assert torch.equal(kc.reshape(-1, hkv, dim), want_k) and torch.equal(vc.reshape(-1, hkv, dim), want_v)


def test_odd_alignment_and_strides_give_the_same_bits_as_the_formula():
    tokens, hq, hkv, dim = 6, 3, 2, 64
    gen = torch.Generator().manual_seed(8)
    flat = torch.randn(tokens * 600 + 1, generator=gen).to(torch.bfloat16).to(DEV)
    q = flat[1:].as_strided((tokens, hq, dim), (599, 71, 1))      # odd strides, odd base
    k = flat.as_strided((tokens, hkv, dim), (600, 64, 1), 300)
    pos = torch.arange(tokens, device=DEV, dtype=torch.int32)
    table = fpv2.rope_table(50, dim, device=DEV)
    gq, gk = fpv2.qk_norm_rope(q, k, pos, table)
    assert close(gq, *formula(q, None, table, pos, 1e-6, False))
    assert close(gk, *formula(k, None, table, pos, 1e-6, False))
    last = k.transpose(1, 2).contiguous().transpose(1, 2)        # head dimension not contiguous
    assert torch.equal(fpv2.qk_norm_rope(q, last, pos, table)[1], gk)


def test_positions_are_clamped_zero_rows_stay_finite_and_no_tokens_are_fine():
    q = torch.zeros(2, 2, 64, dtype=torch.float16, device=DEV)
    table = fpv2.rope_table(10, 64, device=DEV)
    pos = torch.tensor([-5, 10**6], device=DEV, dtype=torch.int64)
    gq, gk = fpv2.qk_norm_rope(q, q, pos, table)
    assert torch.equal(gq, q) and torch.equal(gk, q)
    x = torch.randn(2, 2, 64, generator=torch.Generator().manual_seed(1)).half().to(DEV)
    inside = torch.tensor([0, 9], device=DEV)
    assert torch.equal(fpv2.qk_norm_rope(x, x, pos, table)[0], fpv2.qk_norm_rope(x, x, inside, table)[0])
    before = _lib.launch_count()
    gq, gk = fpv2.qk_norm_rope(q[:0], q[:0], pos[:0], table)
    assert gq.shape == (0, 2, 64) and _lib.launch_count() == before


def test_side_stream_and_mixed_weight_type():
    q, k, _, pos, qw, kw = inputs(300, 8, 2, 128, torch.bfloat16, seed=2)
    table = fpv2.rope_table(500, 128, device=DEV)
    want, _ = formula(q, qw.float(), table, pos, 1e-6, False)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        gq, _ = fpv2.qk_norm_rope(q, k, pos, table, q_weight=qw.float())
    torch.cuda.current_stream().wait_stream(side)
    assert close(gq, want, formula(q, qw.float(), table, pos, 1e-6, False)[1])


@pytest.mark.parametrize("dim,rot", [(96, 64), (80, 40), (80, 80), (56, 16), (160, 32)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_heads_narrower_than_their_lanes_after_infinite_ones(dim, rot, dtype):
    """Nothing of an earlier call's infinities, left in on-chip memory, gets into the norm."""
    full = torch.full((3000, 24, 256), float("inf"), dtype=dtype, device=DEV)
    table = fpv2.rope_table(500, 64, device=DEV)
    pos = torch.zeros(3000, dtype=torch.int32, device=DEV)
    fpv2.qk_norm_rope(full[:, :20], full[:, 20:], pos, table)
    q, k, _, pos, qw, kw = inputs(3000, 20, 4, dim, dtype, seed=dim)
    table = fpv2.rope_table(500, rot, device=DEV)
    for interleaved in (False, True):
        fpv2.qk_norm_rope(full[:, :20], full[:, 20:], torch.zeros_like(pos), table)
        gq, gk = fpv2.qk_norm_rope(q, k, pos, table, q_weight=qw, k_weight=kw, eps=1e-5, interleaved=interleaved)
        assert close(gq, *formula(q, qw, table, pos, 1e-5, interleaved))
        assert close(gk, *formula(k, kw, table, pos, 1e-5, interleaved))
