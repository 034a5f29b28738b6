"""``eps`` and ``scale`` come as float64 and are used in float32: what that type has no finite
number for is refused, and an ``eps`` below its smallest number still keeps zeros finite."""

from __future__ import annotations

import pytest
import torch

import fpv2
from fpv2 import _lib
from tests.test_decode_step_cpu import _structure

SOME = 1 << 20   # a pointer that is never followed


def _call(entry, good, **change):
    kind = _structure(entry + "_params")
    fields = {n: good.get(n, SOME) for n, _ in kind._fields_}
    fields.update(change)
    return getattr(_lib.lib(), entry)(bytes(kind(**fields)), None)


@pytest.mark.parametrize("eps", [3.5e38, 1e300, float("inf"), float("nan"), -1e-300])
def test_eps_out_of_range(eps):
    good = dict(dtype=1, tokens=0, q_heads=1, kv_heads=1, head_dim=64, table_positions=8, rotary_dim=64,
                interleaved=0, positions_int64=0, weight_dtype=1, eps=1e-6, k_cache=0, v_cache=0)
    assert _call("fpv2_qk_norm_rope", good) == _lib.OK
    assert _call("fpv2_qk_norm_rope", good, eps=eps) == _lib.ERR_INVALID_ARGUMENT
    assert _call("fpv2_qk_norm_rope", good, eps=3.4e38) == _lib.OK


@pytest.mark.parametrize("scale", [3e38, -3e38, 1e39, 1e300, float("inf"), float("nan")])
def test_scale_out_of_range(scale):
    good = dict(dtype=1, batch=0, new_tokens=1, q_heads=4, kv_heads=2, head_dim=64, table_width=2, num_pages=2,
                page_size=16, window=0, sinks=0, scale=1.0, workspace_bytes=1 << 40)
    assert _call("fpv2_decode_attention", good) == _lib.OK
    assert _call("fpv2_decode_attention", good, scale=scale) == _lib.ERR_INVALID_ARGUMENT
    assert _call("fpv2_decode_attention", good, scale=-2e38) == _lib.OK


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 37])
@pytest.mark.parametrize("eps", [1e-60, 1e-44])
def test_zeros_stay_zeros_with_the_least_eps(dim, eps):
    q = torch.zeros(3, 2, dim, device="cuda")
    q[1, 0, 5] = 2.0
    table = fpv2.rope_table(4, 2, device="cuda")
    pos = torch.zeros(3, dtype=torch.int32, device="cuda")
    got, _ = fpv2.qk_norm_rope(q, q, pos, table, eps=eps)
    want = torch.zeros_like(q)
    want[1, 0, 5] = dim ** 0.5
    assert torch.equal(got == 0, want == 0) and bool(((got - want).abs() <= 8 * 2.0**-24 * want).all())
