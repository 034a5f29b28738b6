"""``sample_tokens`` inside a captured graph."""

from __future__ import annotations

import pytest
import torch

import fpv2
from tests.test_gpu_sample import inputs

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("settings", [dict(), dict(temperature=0.0), dict(top_k=50, top_p=0.9), dict(top_p=0.9)])
@pytest.mark.parametrize("each", [False, True])
def test_in_a_graph(settings, each):
    logits, noise = inputs(6, 50003, torch.bfloat16, seed=8)
    if each:
        settings = {name: torch.full((6,), value, dtype=torch.int32 if name == "top_k" else torch.float32, device=DEV)
                    for name, value in settings.items()}
    fpv2.sample_tokens(logits, noise, **settings)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens, logprobs = fpv2.sample_tokens(logits, noise, return_logprobs=True, **settings)
    logits.copy_(logits.flip(0) + 1)   # the graph follows its inputs
    noise.copy_(noise.flip(1))
    graph.replay()
    want, lp = fpv2.sample_tokens(logits, noise, return_logprobs=True, **settings)
    assert torch.equal(tokens, want) and torch.equal(logprobs, lp)
