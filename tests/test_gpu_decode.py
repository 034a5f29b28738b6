"""``decode_attention`` against the formula in float64.

Tolerance, from the arithmetic: scores are exact products summed in float32 over D
terms, so each is off by at most e = D 2^-23 scale sum|q k|; that moves the weights by
2 e, their 16-bit form by dP (2^-11 in float16, 2^-16 in bfloat16's two parts) and the
sums over n keys by (n / 16 + 160) 2^-23 (tiles of a part, then the joined parts); all
relative to A = sum p |v|. The output's own rounding adds u |o| (2^-8, 2^-11). The
log-sum-exp is off by e plus 2^-20 of its size.
"""

from __future__ import annotations

import math

import pytest
import torch

import fpv2
from fpv2 import _lib

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
DP = {torch.bfloat16: 2.0**-16, torch.float16: 2.0**-11}


def problem(lengths, new, hq, hkv, dim, page, dtype, seed, spare=3):
    gen = torch.Generator().manual_seed(seed)
    b = len(lengths)
    width = max(1, max(-(-n // page) for n in lengths))
    total = sum(-(-n // page) for n in lengths) + spare
    order = torch.randperm(total, generator=gen).int()
    tables = torch.full((b, width), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(lengths):
        need = -(-n // page)
        tables[i, :need] = order[at:at + need]
        at += need
    k = torch.randn(total, page, hkv, dim, generator=gen).to(dtype)
    v = torch.randn(total, page, hkv, dim, generator=gen).to(dtype)
    q = torch.randn(b, new, hq, dim, generator=gen).to(dtype)
    return q.to(DEV), k.to(DEV), v.to(DEV), tables.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV)


def check(q, k, v, tables, lengths, scale, window, sinks, out, lse):
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
            if not bool(sees.any()):
                assert bool((out[i, t] == 0).all())
                assert bool((lse[i, t] == -math.inf).all())
                continue
            qt, kt, vt = q[i, t].double(), ki[sees], vi[sees]
            s = torch.einsum("hd,lhd->hl", qt, kt) * scale
            pr = torch.softmax(s, -1)
            want = torch.einsum("hl,lhd->hd", pr, vt)
            size = torch.einsum("hl,lhd->hd", pr, vt.abs())
            e = dim * 2.0**-23 * abs(scale) * torch.einsum("hd,lhd->hl", qt.abs(), kt.abs()).amax(-1)
            rel = 2 * e + DP[q.dtype] + (n / 16 + 160) * 2.0**-23
            err = (out[i, t].double() - want).abs()
            tol = U[q.dtype] * want.abs() + rel[:, None] * size
            assert bool((err <= tol).all()), (i, t, float((err / tol).max()))
            wl = torch.logsumexp(s, -1)
            assert bool(((lse[i, t].double() - wl).abs() <= e + 2.0**-20 * wl.abs().clamp_min(1)).all())


@pytest.mark.parametrize("lengths,new,hq,hkv,dim,page,dtype,window,sinks", [
    ([1], 1, 32, 8, 128, 16, torch.bfloat16, 0, 0),
    ([517], 1, 32, 8, 128, 16, torch.bfloat16, 0, 0),
    ([9001], 1, 8, 2, 128, 64, torch.float16, 0, 0),            # cut into many parts
    ([3000], 1, 4, 1, 64, 16, torch.bfloat16, 0, 0),            # one KV head: many parts a CTA
    ([0, 1, 15, 16, 17, 0, 300, 4097], 1, 12, 4, 96, 16, torch.float16, 0, 0),
    ([2500, 33, 0, 700], 1, 16, 16, 64, 7, torch.float16, 0, 0),   # pages that end inside a tile, G = 1
    ([129, 1000, 4], 1, 64, 8, 256, 20, torch.bfloat16, 0, 0),
    ([640] * 40, 1, 8, 2, 256, 128, torch.float16, 0, 0),
    ([100, 3, 1, 0, 2000], 4, 64, 8, 64, 32, torch.float16, 64, 4),   # rows that see nothing, sinks, several tokens
    ([777, 5000], 5, 24, 8, 128, 16, torch.bfloat16, 0, 0),     # G T = 15
    ([777, 50], 9, 24, 8, 128, 1, torch.bfloat16, 0, 0),        # G T = 27: two row blocks; pages of one key
    ([4000, 90, 17], 1, 8, 2, 128, 16, torch.bfloat16, 33, 0),
    ([4000, 90, 17], 2, 8, 2, 96, 16, torch.bfloat16, 100, 130),
    ([5000, 10], 1, 8, 2, 64, 24, torch.bfloat16, 1, 1),
    ([300] * 70, 1, 4, 2, 128, 16, torch.bfloat16, 0, 0),       # more sequences than a warp scans at once
    ([40, 2000], 1, 40, 40, 128, 16, torch.float16, 0, 0),
])
def test_matches_the_formula(lengths, new, hq, hkv, dim, page, dtype, window, sinks):
    q, k, v, tables, n = problem(lengths, new, hq, hkv, dim, page, dtype, seed=sum(lengths) + dim)
    scale = dim ** -0.5
    out, lse = fpv2.decode_attention(q, k, v, tables, n, scale=scale, window=window, sinks=sinks, return_lse=True)
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    check(q, k, v, tables, n, scale, window, sinks, out, lse)
    again = fpv2.decode_attention(q, k, v, tables, n, scale=scale, window=window, sinks=sinks)
    assert torch.equal(again, out)   # bit for bit
    if new == 1:
        flat, flat_lse = fpv2.decode_attention(q[:, 0], k, v, tables, n, scale=scale, window=window, sinks=sinks,
                                               return_lse=True)
        assert flat.shape == q[:, 0].shape and torch.equal(flat, out[:, 0]) and torch.equal(flat_lse, lse[:, 0])


@pytest.mark.parametrize("scale", [0.0, -0.09, 0.4])
@pytest.mark.parametrize("new,hq,dim,window", [(1, 8, 128, 0), (3, 8, 128, 50), (4, 16, 64, 200)])
def test_scales_of_any_sign(scale, new, hq, dim, window):
    q, k, v, tables, n = problem([700, 2, 0, 1900], new, hq, 2, dim, 16, torch.float16, seed=hq + new)
    out, lse = fpv2.decode_attention(q, k, v, tables, n, scale=scale, window=window, return_lse=True)
    check(q, k, v, tables, n, scale, window, 0, out, lse)


def test_strided_caches_queries_and_tables():
    q, k, v, tables, n = problem([300, 41], 1, 8, 2, 128, 16, torch.bfloat16, seed=3)
    want = fpv2.decode_attention(q, k, v, tables, n, scale=0.1)
    both = torch.stack([k, v], 1)                                  # [pages, 2, page, heads, dim]
    heads = torch.stack([k, v]).transpose(2, 3).contiguous().transpose(2, 3)   # heads outside the rows
    wide = torch.cat([tables, tables], 1)[:, :tables.shape[1]]
    assert torch.equal(fpv2.decode_attention(q, both[:, 0], both[:, 1], wide, n, scale=0.1), want)
    assert torch.equal(fpv2.decode_attention(q, heads[0], heads[1], tables.t().contiguous().t(), n, scale=0.1), want)
    fused = torch.zeros(2, 1, 12, 129, dtype=q.dtype, device=DEV)   # odd strides: copied
    fused[:, :, 2:10, 1:] = q
    assert torch.equal(fpv2.decode_attention(fused[:, :, 2:10, 1:], k, v, tables, n, scale=0.1), want)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_what_a_query_does_not_see_does_not_touch_it(bad, dtype):
    window, sinks, new = 50, 3, 3
    q, k, v, tables, n = problem([400, 60, 2], new, 8, 2, 128, 16, dtype, seed=5)
    want, wl = fpv2.decode_attention(q, k, v, tables, n, scale=0.09, window=window, sinks=sinks, return_lse=True)
    # rows past the end, keys between the sinks and the window, and every unused page
    k2, v2 = k.clone(), v.clone()
    used = set()
    for i, length in enumerate(n.tolist()):
        low = max(0, length - new - window + 1)
        for j in range(-(-length // 16) * 16):
            page, row = int(tables[i, j // 16]), j % 16
            used.add(page)
            if j >= length or sinks <= j < low:
                k2[page, row] = bad
                v2[page, row] = bad
    for page in set(range(k.shape[0])) - used:
        k2[page] = bad
        v2[page] = bad
    got, gl = fpv2.decode_attention(q, k2, v2, tables, n, scale=0.09, window=window, sinks=sinks, return_lse=True)
    assert torch.equal(got, want) and torch.equal(gl, wl)
    # the newest token's own key and value: the drafts before it must not notice
    page, row = int(tables[0, 399 // 16]), 399 % 16
    k2[page, row] = bad
    v2[page, row] = bad
    got, gl = fpv2.decode_attention(q, k2, v2, tables, n, scale=0.09, window=window, sinks=sinks, return_lse=True)
    assert not bool(torch.isfinite(got[0, 2].float()).all())
    check(q[:, :2], k, v, tables, torch.tensor([399, 59, 1], device=DEV), 0.09, window, sinks, got[:, :2], gl[:, :2])


def test_lengths_and_pages_out_of_range_are_clamped():
    q, k, v, tables, n = problem([64, 64], 1, 4, 2, 64, 16, torch.float16, seed=6)
    full = fpv2.decode_attention(q, k, v, tables, n, scale=0.1)
    over = torch.tensor([10**6, -7], dtype=torch.int32, device=DEV)
    got = fpv2.decode_attention(q, k, v, tables, over, scale=0.1)
    assert torch.equal(got[0], full[0]) and bool((got[1] == 0).all())
    wild = tables.clone()
    wild[0, 1], wild[0, 2] = 2**31 - 1, -(2**31)
    kept = tables.clone()
    kept[0, 1], kept[0, 2] = k.shape[0] - 1, 0
    assert torch.equal(fpv2.decode_attention(q, k, v, wild, n, scale=0.1),
                       fpv2.decode_attention(q, k, v, kept, n, scale=0.1))
    _lib.device_status()   # a build that reports clamped entries has noted these
    none = fpv2.decode_attention(q[:0], k, v, tables[:0], n[:0], scale=0.1)
    assert none.shape == (0, 1, 4, 64)


def test_large_scores_negative_scale_and_equal_keys():
    q, k, v, tables, n = problem([900], 1, 8, 2, 128, 16, torch.bfloat16, seed=9)
    for scale in (4.0, -0.3):
        out, lse = fpv2.decode_attention(q, k, v, tables, n, scale=scale, return_lse=True)
        check(q, k, v, tables, n, scale, 0, 0, out, lse)
    k.fill_(0.5)   # every key the same: the plain mean
    out, lse = fpv2.decode_attention(q, k, v, tables, n, scale=0.2, return_lse=True)
    check(q, k, v, tables, n, 0.2, 0, 0, out, lse)


def test_offsets_past_32_bits():
    # 2^31 + elements between the first and the last page
    page, hkv, dim = 16, 2, 64
    pages = 2**31 // (page * hkv * dim) + 40
    k = torch.empty(pages, page, hkv, dim, dtype=torch.float16, device=DEV)
    v = torch.empty(pages, page, hkv, dim, dtype=torch.float16, device=DEV)
    gen = torch.Generator().manual_seed(4)
    tables = torch.tensor([[pages - 1, 0, pages - 20]], dtype=torch.int32, device=DEV)
    for p in tables[0].tolist():
        k[p] = torch.randn(page, hkv, dim, generator=gen).half().to(DEV)
        v[p] = torch.randn(page, hkv, dim, generator=gen).half().to(DEV)
    q = torch.randn(1, 1, 8, dim, generator=gen).half().to(DEV)
    n = torch.tensor([45], dtype=torch.int32, device=DEV)
    out, lse = fpv2.decode_attention(q, k, v, tables, n, scale=0.125, return_lse=True)
    check(q, k, v, tables, n, 0.125, 0, 0, out, lse)


def test_side_stream_and_graph():
    q, k, v, tables, n = problem([3000, 100], 1, 8, 2, 128, 16, torch.bfloat16, seed=12)
    want = fpv2.decode_attention(q, k, v, tables, n, scale=0.1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fpv2.decode_attention(q, k, v, tables, n, scale=0.1)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = fpv2.decode_attention(q, k, v, tables, n, scale=0.1)
    n.copy_(torch.tensor([500, 100], dtype=torch.int32))   # the graph follows the lengths
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(kept, fpv2.decode_attention(q, k, v, tables, n, scale=0.1))
