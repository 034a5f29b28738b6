"""Argument checks of the decode step's operators, without a GPU.

Wrong shapes, types and missing tensors are refused before any launch, CPU tensors
and inputs that need gradients are refused too, and the C entry points return a
status for scalars out of contract.
"""

from __future__ import annotations

import ctypes
import re
from pathlib import Path

import pytest
import torch

import fpv2
from fpv2 import _lib, decode

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


def _structure(name: str) -> type[ctypes.Structure]:
    """A parameter structure as include/fpv2_b200.h declares it."""
    text = (Path(__file__).resolve().parents[1] / "include" / "fpv2_b200.h").read_text()
    body = re.search(r"typedef struct \{([^}]*)\} " + name + ";", text).group(1)
    fields = []
    for line in re.sub(r"/\*.*?\*/", "", body, flags=re.S).split(";"):
        line = line.strip()
        if not line:
            continue
        kind = ctypes.c_double if line.startswith("double") else ctypes.c_int64
        names = re.sub(r"^(const\s+)?\w+", "", line).replace("*", " ")
        fields += [(f.strip(), kind) for f in names.split(",")]
    return type(name, (ctypes.Structure,), {"_fields_": fields})


@pytest.mark.parametrize("name,pack", [
    ("fpv2_qk_norm_rope_params", decode._pack_rope),
    ("fpv2_decode_attention_params", decode._pack_decode),
    ("fpv2_sample_tokens_params", decode._pack_sample),
])
def test_packed_parameters_have_the_declared_layout(name, pack):
    kind = _structure(name)
    values = [float(i) if t is ctypes.c_double else i for i, (_, t) in enumerate(kind._fields_)]
    assert pack(*values) == bytes(kind(*values))


def test_entry_points_return_status_without_gpu():
    lib = _lib.lib()
    before = _lib.launch_count()
    some = 1 << 20   # a pointer that is never followed

    def call(entry, good, **change):
        kind = _structure(entry + "_params")
        fields = {n: some if n not in good else good[n] for n, _ in kind._fields_}
        fields.update(change)
        return getattr(lib, entry)(bytes(kind(**{n: v or 0 for n, v in fields.items()})), None)

    def decode_call(**change):
        good = dict(dtype=1, batch=1, new_tokens=1, q_heads=4, kv_heads=2, head_dim=64, table_width=2,
                    num_pages=2, page_size=16, window=0, sinks=0, scale=1.0, workspace_bytes=1 << 40)
        return call("fpv2_decode_attention", good, **change)

    bad = [decode_call(**c) for c in (
        dict(dtype=2), dict(batch=-1), dict(new_tokens=0), dict(q_heads=3), dict(q_heads=1 << 30),
        dict(head_dim=80), dict(num_pages=0), dict(table_width=1 << 30), dict(scale=float("nan")),
        dict(window=-1), dict(sinks=1 << 40), dict(q=None), dict(lengths=None), dict(workspace_bytes=8),
        dict(k_row_stride=4), dict(q_head_stride=3), dict(k_pages=some + 2), dict(workspace=some + 8))]
    assert bad == [_lib.ERR_INVALID_ARGUMENT] * len(bad)
    assert decode_call(batch=0) == _lib.OK

    def rope_call(**change):
        good = dict(dtype=1, tokens=1, q_heads=1, kv_heads=1, head_dim=64, table_positions=8, rotary_dim=64,
                    interleaved=0, positions_int64=0, weight_dtype=1, eps=1e-6, k_cache=0, v_cache=0)
        return call("fpv2_qk_norm_rope", good, **change)

    bad = [rope_call(**c) for c in (
        dict(dtype=7), dict(tokens=-1), dict(q_heads=0), dict(head_dim=257), dict(rotary_dim=63),
        dict(rotary_dim=66), dict(table_positions=0), dict(eps=-1.0), dict(q=None), dict(weight_dtype=5),
        dict(k_cache=some), dict(k_cache=some, v_cache=some, slots=None),
        dict(k_cache=some, v_cache=some, page_size=0))]
    assert bad == [_lib.ERR_INVALID_ARGUMENT] * len(bad)
    assert rope_call(tokens=0) == _lib.OK

    def sample_call(**change):
        good = dict(dtype=1, rows=1, vocab=8, temperature_all=1.0, top_k_all=0, top_p_all=1.0, min_p_all=0.0)
        return call("fpv2_sample_tokens", good, **change)

    bad = [sample_call(**c) for c in (
        dict(dtype=3), dict(rows=-1), dict(vocab=0), dict(logits=None), dict(noise=None),
        dict(logits=some + 1))]
    assert bad == [_lib.ERR_INVALID_ARGUMENT] * len(bad)
    assert sample_call(rows=0) == _lib.OK
    for entry in ("fpv2_qk_norm_rope", "fpv2_decode_attention", "fpv2_sample_tokens"):
        assert getattr(lib, entry)(None, None) == _lib.ERR_INVALID_ARGUMENT
    assert lib.fpv2_decode_workspace_bytes(1, 3, 2, 64) == 0
    assert lib.fpv2_decode_workspace_bytes(1, 32, 8, 128) > 0
    assert _lib.launch_count() == before
