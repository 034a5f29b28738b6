"""Argument checks of the decode step's operators, without a GPU.

Wrong shapes, types and missing tensors are refused before any launch, CPU tensors
and inputs that need gradients are refused too, and the C entry points return a
status for scalars out of contract.
"""

from __future__ import annotations

import ctypes

import pytest
import torch

import fpv2
from fpv2 import _lib

BF = torch.bfloat16


def _rope_args(**change):
    a = dict(q=torch.zeros(3, 4, 64, dtype=BF), k=torch.zeros(3, 2, 64, dtype=BF),
             positions=torch.zeros(3, dtype=torch.int32), table=torch.zeros(8, 64))
    kw = {}
    for name, value in change.items():
        (a if name in a else kw)[name] = value
    return list(a.values()), kw


@pytest.mark.parametrize("change,match", [
    (dict(q=torch.zeros(3, 64, dtype=BF)), "shape"),
    (dict(k=torch.zeros(2, 2, 64, dtype=BF)), "same tokens"),
    (dict(k=torch.zeros(3, 2, 32, dtype=BF)), "same tokens"),
    (dict(k=torch.zeros(3, 0, 64, dtype=BF)), "heads"),
    (dict(k=torch.zeros(3, 2, 64)), "share"),
    (dict(q=torch.zeros(3, 4, 320, dtype=BF), k=torch.zeros(3, 2, 320, dtype=BF)), "head dimension"),
    (dict(q=torch.zeros(3, 4, 64, dtype=torch.int32), k=torch.zeros(3, 2, 64, dtype=torch.int32)), "dtype"),
    (dict(positions=torch.zeros(2, dtype=torch.int32)), "positions"),
    (dict(positions=torch.zeros(3)), "positions"),
    (dict(table=torch.zeros(8, 64, dtype=BF)), "table"),
    (dict(table=torch.zeros(0, 64)), "table"),
    (dict(table=torch.zeros(8, 63)), "rotary"),
    (dict(table=torch.zeros(8, 66)), "rotary"),
    (dict(q_weight=torch.ones(32, dtype=BF)), "weights"),
    (dict(q_weight=torch.ones(64, dtype=BF), k_weight=torch.ones(64)), "weights"),
    (dict(v=torch.zeros(3, 2, 64, dtype=BF)), "go together"),
    (dict(v=torch.zeros(3, 2, 64, dtype=BF), k_cache=torch.zeros(2, 8, 2, 64, dtype=BF),
          v_cache=torch.zeros(2, 8, 2, 64, dtype=BF)), "go together"),
    (dict(v=torch.zeros(3, 2, 64, dtype=BF), k_cache=torch.zeros(2, 8, 3, 64, dtype=BF),
          v_cache=torch.zeros(2, 8, 3, 64, dtype=BF), slots=torch.zeros(3, dtype=torch.int64)), "caches"),
    (dict(v=torch.zeros(3, 2, 64, dtype=BF), k_cache=torch.zeros(2, 8, 2, 64, dtype=BF),
          v_cache=torch.zeros(3, 8, 2, 64, dtype=BF), slots=torch.zeros(3, dtype=torch.int64)), "identical"),
    (dict(v=torch.zeros(3, 2, 64, dtype=BF), k_cache=torch.zeros(2, 8, 2, 64, dtype=BF),
          v_cache=torch.zeros(2, 8, 2, 64, dtype=BF), slots=torch.zeros(3, dtype=torch.int32)), "slots"),
    (dict(q=torch.zeros(3, 4, 64, dtype=BF, requires_grad=True)), "no backward"),
    (dict(), "CUDA"),
])
def test_qk_norm_rope_refuses(change, match):
    args, kw = _rope_args(**change)
    with pytest.raises(ValueError, match=match):
        fpv2.qk_norm_rope(*args, **kw)


def _decode_args(**change):
    a = dict(q=torch.zeros(2, 4, 64, dtype=BF), k_cache=torch.zeros(5, 8, 2, 64, dtype=BF),
             v_cache=torch.zeros(5, 8, 2, 64, dtype=BF), block_tables=torch.zeros(2, 3, dtype=torch.int32),
             lengths=torch.zeros(2, dtype=torch.int32))
    kw = {"scale": 1.0}
    for name, value in change.items():
        (a if name in a else kw)[name] = value
    return list(a.values()), kw


@pytest.mark.parametrize("change,match", [
    (dict(q=torch.zeros(4, 64, dtype=BF)), "shape"),
    (dict(q=torch.zeros(2, 4, 64)), "dtype"),
    (dict(k_cache=torch.zeros(5, 8, 2, 64, dtype=torch.float16)), "dtype"),
    (dict(v_cache=torch.zeros(5, 8, 2, 32, dtype=BF)), "identical"),
    (dict(q=torch.zeros(2, 4, 128, dtype=BF)), "head dimension"),
    (dict(q=torch.zeros(2, 3, 64, dtype=BF)), "divisible"),
    (dict(q=torch.zeros(2, 0, 4, 64, dtype=BF)), "at least one"),
    (dict(k_cache=torch.zeros(0, 8, 2, 64, dtype=BF), v_cache=torch.zeros(0, 8, 2, 64, dtype=BF)), "empty"),
    (dict(block_tables=torch.zeros(2, 3, dtype=torch.int64)), "block_tables"),
    (dict(block_tables=torch.zeros(1, 3, dtype=torch.int32)), "block_tables"),
    (dict(block_tables=torch.zeros(2, 0, dtype=torch.int32)), "no pages"),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), "lengths"),
    (dict(lengths=torch.zeros(2)), "lengths"),
    (dict(window=-1), "window"),
    (dict(sinks=-1), "window"),
    (dict(q=torch.zeros(2, 4, 64, dtype=BF, requires_grad=True)), "no backward"),
    (dict(), "CUDA"),
])
def test_decode_attention_refuses(change, match):
    args, kw = _decode_args(**change)
    with pytest.raises(ValueError, match=match):
        fpv2.decode_attention(*args, **kw)


@pytest.mark.parametrize("change,match", [
    (dict(logits=torch.zeros(5)), "shape"),
    (dict(noise=torch.ones(2, 6)), "shape"),
    (dict(logits=torch.zeros(2, 0), noise=torch.ones(2, 0)), "vocabulary"),
    (dict(logits=torch.zeros(2, 5, dtype=torch.float64)), "dtype"),
    (dict(noise=torch.ones(2, 5, dtype=BF)), "noise"),
    (dict(temperature=torch.ones(3)), "temperature"),
    (dict(top_k=torch.ones(2)), "top_k"),
    (dict(top_k=2**40), "top_k"),
    (dict(top_p=torch.ones(2, dtype=BF)), "top_p"),
    (dict(min_p=torch.ones(2, 1)), "min_p"),
    (dict(logits=torch.zeros(2, 5, requires_grad=True)), "no backward"),
    (dict(), "CUDA"),
])
def test_sample_tokens_refuses(change, match):
    a = dict(logits=torch.zeros(2, 5), noise=torch.ones(2, 5))
    a.update(change)
    with pytest.raises(ValueError, match=match):
        fpv2.sample_tokens(a.pop("logits"), a.pop("noise"), **a)


def test_rope_table_rows_and_refusals():
    t = fpv2.rope_table(5, 4, theta=100.0)
    assert t.shape == (5, 4) and t.dtype == torch.float32
    angle = torch.tensor([3.0, 3.0 / 10.0], dtype=torch.float64)
    assert torch.equal(t[3], torch.cat([angle.cos(), angle.sin()]).float())
    for bad in ((0, 4), (5, 3), (5, 0)):
        with pytest.raises(ValueError, match="rotary_dim"):
            fpv2.rope_table(*bad)


def test_entry_points_return_status_without_gpu():
    lib = _lib.lib()
    before = _lib.launch_count()
    nine = (ctypes.c_int64 * 9)(*[64] * 9)
    six = (ctypes.c_int64 * 6)(*[64] * 6)

    def decode(batch=1, new=1, hq=4, hkv=2, dim=64, strides=nine, pages=2, page=16, width=2, scale=1.0,
               window=0, dtype=1, ptr=1 << 20, nbytes=1 << 40):
        return lib.fpv2_decode_attention(ptr, ptr, ptr, dtype, batch, new, hq, hkv, dim, strides, ptr, 2, width,
                                         ptr, pages, page, scale, window, 0, ptr, None, ptr, nbytes, None)

    bad = [decode(dtype=2), decode(batch=-1), decode(new=0), decode(hq=3), decode(dim=80), decode(pages=0),
           decode(width=1 << 30), decode(scale=float("nan")), decode(window=-1), decode(strides=None),
           decode(ptr=None), decode(nbytes=8), decode(strides=(ctypes.c_int64 * 9)(*[4] * 9))]
    assert bad == [_lib.ERR_INVALID_ARGUMENT] * len(bad)
    assert decode(batch=0) == _lib.OK

    def rope(dtype=1, tokens=1, hq=1, dim=64, rot=64, table=8, eps=1e-6, ptr=1 << 20, k_cache=None, strides=six):
        return lib.fpv2_qk_norm_rope(ptr, ptr, ptr, dtype, tokens, hq, 1, dim, strides, ptr, 0, ptr, table, rot, 0,
                                     None, None, dtype, eps, ptr, ptr, strides, k_cache, None, None, None, 0, 0,
                                     None)

    bad = [rope(dtype=7), rope(tokens=-1), rope(hq=0), rope(dim=257), rope(rot=63), rope(rot=66), rope(table=0),
           rope(eps=-1.0), rope(ptr=None), rope(k_cache=1 << 20), rope(strides=None)]
    assert bad == [_lib.ERR_INVALID_ARGUMENT] * len(bad)
    assert rope(tokens=0) == _lib.OK

    def sample(dtype=1, rows=1, vocab=8, ptr=1 << 20):
        return lib.fpv2_sample_tokens(ptr, dtype, rows, vocab, vocab, ptr, vocab, None, 1.0, None, 0, None, 1.0,
                                      None, 0.0, ptr, None, None)

    bad = [sample(dtype=3), sample(rows=-1), sample(vocab=0), sample(ptr=None), sample(ptr=(1 << 20) + 1)]
    assert bad == [_lib.ERR_INVALID_ARGUMENT] * len(bad)
    assert sample(rows=0) == _lib.OK
    assert lib.fpv2_decode_workspace_bytes(1, 3, 2, 64) == 0
    assert lib.fpv2_decode_workspace_bytes(1, 32, 8, 128) > 0
    assert _lib.launch_count() == before
