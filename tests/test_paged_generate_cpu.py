"""The generation example refuses on the host what would index past its page tables on the GPU."""

from __future__ import annotations

import sys
from pathlib import Path

import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))

import paged_generate as G  # noqa: E402

SHAPE = G.Shape(layers=1, hidden=64, q_heads=2, kv_heads=1, head_dim=64, inner=64, vocab=50, max_tokens=200)


def _model(requests=2):
    return G.PagedModel(SHAPE, G.random_weights(SHAPE, device="cpu"), requests)


def _ids(n):
    return torch.zeros(n, dtype=torch.int64)


@pytest.mark.parametrize("request_, tokens, match", [
    (2, 5, "request"), (-1, 5, "request"), (0, 201, "max_tokens"), (0, 0, "max_tokens"),
])
def test_prefill_refuses(request_, tokens, match):
    with pytest.raises(ValueError, match=match):
        _model().prefill(request_, _ids(tokens))


def test_decode_refuses():
    model = _model()
    with pytest.raises(ValueError, match="token"):
        model.decode(_ids(1))
    model.held = [200, 3]
    with pytest.raises(ValueError, match="max_tokens"):
        model.decode(_ids(2))


@pytest.mark.parametrize("prompts, new, match", [
    ((150, 3), 52, "max_tokens"), ((5,), 2, "requests"), ((5, 5, 5), 2, "requests"),
])
def test_generate_refuses(prompts, new, match):
    with pytest.raises(ValueError, match=match):
        G.generate(_model(), [_ids(n) for n in prompts], new)


def test_what_fits_goes_on_to_the_operators():
    with pytest.raises(ValueError, match="CUDA"):
        G.generate(_model(), [_ids(150), _ids(3)], 51)
