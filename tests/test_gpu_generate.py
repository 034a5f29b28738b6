"""The example's prefill and decode against the same decoder in float32 with dense attention.

With alpha 0 every block is selected, so the sparse prefill is exact attention. The
model runs in bfloat16: each of a layer's dozen roundings is off by up to 2^-8 of its
value, independently, and two layers and the head have about 30, so the logits'
relative error (2-norm) stays within 2^-8 sqrt(30) = 0.021; twice that is allowed.
"""

from __future__ import annotations

import sys
from pathlib import Path

import pytest
import torch
import torch.nn.functional as F

import fpv2
from fpv2 import _lib

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))

import paged_generate as G  # noqa: E402

pytestmark = pytest.mark.gpu


def dense_logits(shape, weights, ids):
    """Logits [tokens, vocab] of the whole sequence, float32, without fpv2."""
    s, n = shape, ids.numel()
    wf = lambda t: t.float()  # noqa: E731
    pos = torch.arange(n, device=ids.device, dtype=torch.float64)[:, None]
    freq = s.theta ** (-torch.arange(s.head_dim // 2, device=ids.device, dtype=torch.float64) / (s.head_dim // 2))
    cos, sin = (pos * freq).cos().float()[:, None], (pos * freq).sin().float()[:, None]

    def rope(x):
        a, b = x.chunk(2, -1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    x = wf(weights["embed"][ids])
    mask = torch.ones(n, n, dtype=torch.bool, device=ids.device).tril()
    for b in weights["blocks"]:
        h = F.rms_norm(x, (s.hidden,), wf(b["ln1"]), eps=1e-6)
        qkv = (h @ wf(b["qkv"]).T).view(n, -1, s.head_dim)
        q, k, v = qkv.split([s.q_heads, s.kv_heads, s.kv_heads], 1)
        q = rope(F.rms_norm(q, (s.head_dim,), wf(b["qn"]), eps=1e-6))
        k = rope(F.rms_norm(k, (s.head_dim,), wf(b["kn"]), eps=1e-6))
        k, v = (t.repeat_interleave(s.q_heads // s.kv_heads, 1) for t in (k, v))
        score = torch.einsum("qhd,khd->hqk", q, k) * s.head_dim**-0.5
        o = torch.einsum("hqk,khd->qhd", score.masked_fill(~mask, -torch.inf).softmax(-1), v)
        x = x + o.reshape(n, -1) @ wf(b["o"]).T
        h = F.rms_norm(x, (s.hidden,), wf(b["ln2"]), eps=1e-6)
        x = x + (F.silu(h @ wf(b["gate"]).T) * (h @ wf(b["up"]).T)) @ wf(b["down"]).T
    return F.rms_norm(x, (s.hidden,), wf(weights["norm"]), eps=1e-6) @ wf(weights["head"]).T


def test_prefill_and_decode_match_the_dense_decoder():
    shape = G.Shape(layers=2, hidden=256, q_heads=8, kv_heads=2, head_dim=64, inner=512, vocab=997, page_size=16,
                    max_tokens=700)
    weights = G.random_weights(shape, seed=3)
    cfg = fpv2.FPV2Config(alpha=0.0, tile_q=32, last_n_blocks=0, score_chunk_tiles=8)
    gen = torch.Generator(device="cuda").manual_seed(4)
    ids = [torch.randint(0, shape.vocab, (n,), generator=gen, device="cuda") for n in (600, 211, 1)]
    new = [torch.randint(0, shape.vocab, (3,), generator=gen, device="cuda") for _ in range(3)]   # a step's tokens
    model = G.PagedModel(shape, weights, 3, cfg)
    got = [torch.stack([model.prefill(r, x, chunk=256) for r, x in enumerate(ids)])]
    got += [model.decode(step) for step in new]
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    for r in range(3):
        whole = torch.cat([ids[r], torch.stack(new)[:, r]])
        want = dense_logits(shape, weights, whole)[len(ids[r]) - 1:]
        mine = torch.stack([g[r] for g in got]).float()
        assert mine.shape == want.shape
        assert float((mine - want).norm() / want.norm()) <= 2 * 0.021


def test_generate_repeats_and_follows_the_filters():
    shape = G.Shape(layers=1, hidden=128, q_heads=4, kv_heads=1, head_dim=64, inner=256, vocab=500, max_tokens=300)
    weights = G.random_weights(shape, seed=5)
    prompts = [torch.arange(5, 260, device="cuda") % shape.vocab, torch.arange(40, device="cuda")]
    runs = []
    for _ in range(2):
        torch.manual_seed(0)   # page order
        runs.append(G.generate(G.PagedModel(shape, weights, 2), prompts, 8, seed=9))
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])
    assert runs[0][0].shape == (2, 8) and bool((runs[0][1] <= 0).all())
    greedy, _ = G.generate(G.PagedModel(shape, weights, 2), prompts, 4, temperature=0.0)
    top1, _ = G.generate(G.PagedModel(shape, weights, 2), prompts, 4, top_k=1, seed=3)
    assert torch.equal(greedy, top1)
