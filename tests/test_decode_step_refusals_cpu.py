"""Derivatives that the decode step's operators do not have are refused, not dropped; without a GPU."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import fpv2

BF = torch.bfloat16


def _rope(**change):
    a = dict(q=torch.zeros(3, 4, 64), k=torch.zeros(3, 2, 64), positions=torch.zeros(3, dtype=torch.int32),
             table=torch.zeros(8, 64), q_weight=torch.ones(64), k_weight=torch.ones(64), v=torch.zeros(3, 2, 64),
             k_cache=torch.zeros(2, 8, 2, 64), v_cache=torch.zeros(2, 8, 2, 64),
             slots=torch.zeros(3, dtype=torch.int64))
    a.update({n: f(a[n]) for n, f in change.items()})
    return fpv2.qk_norm_rope(a.pop("q"), a.pop("k"), a.pop("positions"), a.pop("table"), **a)


def _decode(**change):
    a = dict(q=torch.zeros(2, 4, 64, dtype=BF), k_cache=torch.zeros(5, 8, 2, 64, dtype=BF),
             v_cache=torch.zeros(5, 8, 2, 64, dtype=BF))
    a.update({n: f(a[n]) for n, f in change.items()})
    return fpv2.decode_attention(*a.values(), torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32),
                                 scale=1.0)


def _sample(**change):
    a = dict(logits=torch.zeros(2, 5), temperature=torch.ones(2))
    a.update({n: f(a[n]) for n, f in change.items()})
    return fpv2.sample_tokens(a["logits"], torch.ones(2, 5), temperature=a["temperature"])


CALLS = [(_rope, n) for n in ("q", "k", "table", "q_weight", "k_weight", "v", "k_cache", "v_cache")]
CALLS += [(_decode, n) for n in ("q", "k_cache", "v_cache")] + [(_sample, n) for n in ("logits", "temperature")]


@pytest.mark.parametrize("call,name", CALLS)
def test_a_forward_mode_tangent_is_refused(call, name):
    with forward_ad.dual_level(), torch.no_grad():
        with pytest.raises(ValueError, match="forward-mode"):
            call(**{name: lambda t: forward_ad.make_dual(t, torch.ones_like(t))})
        with pytest.raises(ValueError, match="CUDA"):   # none of them has one: on to the next check
            call()


@pytest.mark.parametrize("call,name", CALLS)
def test_an_input_that_requires_grad_is_refused(call, name):
    with pytest.raises(ValueError, match="no backward"):
        call(**{name: lambda t: t.clone().requires_grad_()})
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
        call(**{name: lambda t: t.clone().requires_grad_()})
