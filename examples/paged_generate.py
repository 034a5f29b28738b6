"""Sparse prefill and token-by-token generation over one paged KV cache.

A small decoder (random weights; RMS norms, per-head q/k norms, rotary embedding,
grouped-query attention, SwiGLU) serves a batch of requests. Each prompt is prefilled
in chunks with block-sparse attention, then all requests generate together:

    prefill chunk   qk_norm_rope -> pool_pages -> block_scores_and_select
                    -> compact_block_indices -> sparse_attention_paged
    decode step     qk_norm_rope -> decode_attention -> sample_tokens

Both write and read the same page pools. Run on a B200:

    python examples/paged_generate.py --prompts 3 --prompt-tokens 4000 --new-tokens 32
"""

from __future__ import annotations

import argparse
import sys
from dataclasses import dataclass
from pathlib import Path

import torch
import torch.nn.functional as F

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "flashprefillv2-mlx_b200"))

import fpv2  # noqa: E402


@dataclass(frozen=True)
class Shape:
    layers: int = 4
    hidden: int = 1024
    q_heads: int = 32
    kv_heads: int = 8
    head_dim: int = 128
    inner: int = 2816
    vocab: int = 32000
    page_size: int = 16
    max_tokens: int = 8192
    theta: float = 1e6


def random_weights(shape: Shape, seed: int = 0, device: str = "cuda") -> dict:
    gen = torch.Generator(device=device).manual_seed(seed)

    def w(rows: int, cols: int) -> torch.Tensor:
        return (torch.randn(rows, cols, generator=gen, device=device) * cols**-0.5).to(torch.bfloat16)

    s, one = shape, lambda n: torch.ones(n, dtype=torch.bfloat16, device=device)
    heads = s.q_heads + 2 * s.kv_heads
    blocks = [dict(ln1=one(s.hidden), qkv=w(heads * s.head_dim, s.hidden), qn=one(s.head_dim), kn=one(s.head_dim),
                   o=w(s.hidden, s.q_heads * s.head_dim), ln2=one(s.hidden), gate=w(s.inner, s.hidden),
                   up=w(s.inner, s.hidden), down=w(s.hidden, s.inner)) for _ in range(s.layers)]
    return dict(embed=w(s.vocab, s.hidden) * 30, blocks=blocks, norm=one(s.hidden), head=w(s.vocab, s.hidden))


class PagedModel:
    """The decoder and its page pools; request ``r`` owns the pages of ``tables[r]``."""

    def __init__(self, shape: Shape, weights: dict, requests: int, config: fpv2.FPV2Config | None = None):
        s = self.shape = shape
        self.weights = weights
        device = weights["embed"].device
        group = s.q_heads // s.kv_heads
        # 128 packed query rows a selection tile; no raw scores
        self.config = config or fpv2.FPV2Config(alpha=0.1, tile_q=128 // group, last_n_blocks=0, score_chunk_tiles=8)
        block = self.config.block_k
        pages = (s.max_tokens + block - 1) // block * block // s.page_size
        self.table = fpv2.rope_table(s.max_tokens, s.head_dim, theta=s.theta, device=device)
        pool = (s.layers, 2, requests * pages, s.page_size, s.kv_heads, s.head_dim)
        self.cache = torch.zeros(pool, dtype=torch.bfloat16, device=device)
        order = torch.randperm(requests * pages, device=device, dtype=torch.int32)
        self.tables = order.view(requests, pages)
        self.lengths = torch.zeros(requests, dtype=torch.int32, device=device)
        self.held = [0] * requests   # the same on the host: a position past the pools is refused there

    def _slots(self, requests: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
        page = self.shape.page_size
        return self.tables[requests, positions // page].long() * page + positions % page

    def _block(self, x: torch.Tensor, layer: int, positions: torch.Tensor, slots: torch.Tensor, attend,
               heads_first: bool) -> torch.Tensor:
        s, b = self.shape, self.weights["blocks"][layer]
        h = F.rms_norm(x, (s.hidden,), b["ln1"], eps=1e-6)
        qkv = (h @ b["qkv"].T).view(-1, s.q_heads + 2 * s.kv_heads, s.head_dim)
        q, k, v = qkv.split([s.q_heads, s.kv_heads, s.kv_heads], 1)
        kc, vc = self.cache[layer]
        q, _ = fpv2.qk_norm_rope(q, k, positions, self.table, q_weight=b["qn"], k_weight=b["kn"], eps=1e-6,
                                 heads_first=heads_first, v=v, k_cache=kc, v_cache=vc, slots=slots)
        x = x + attend(q, kc, vc).reshape(-1, s.q_heads * s.head_dim) @ b["o"].T
        h = F.rms_norm(x, (s.hidden,), b["ln2"], eps=1e-6)
        return x + (F.silu(h @ b["gate"].T) * (h @ b["up"].T)) @ b["down"].T

    def _logits(self, x: torch.Tensor) -> torch.Tensor:
        return F.rms_norm(x, (self.shape.hidden,), self.weights["norm"], eps=1e-6) @ self.weights["head"].T

    @torch.no_grad()
    def prefill(self, request: int, ids: torch.Tensor, chunk: int = 2048) -> torch.Tensor:
        """Logits ``[vocab]`` after the prompt ``ids``, prefilled in chunks."""
        s, cfg = self.shape, self.config
        if not 0 <= request < len(self.held):
            raise ValueError(f"request must be in [0, {len(self.held)})")
        if not 0 < ids.numel() <= s.max_tokens:
            raise ValueError(f"a prompt must have 1 to max_tokens = {s.max_tokens} tokens")
        for offset in range(0, ids.numel(), chunk):
            n = min(chunk, ids.numel() - offset)
            length = offset + n
            rows = (n + cfg.tile_q - 1) // cfg.tile_q * cfg.tile_q
            keys = (max(length, offset + rows) + cfg.block_k - 1) // cfg.block_k * cfg.block_k
            positions = torch.arange(offset, length, device=ids.device)
            slots = self._slots(torch.full_like(positions, request), positions)
            pages = self.tables[request, :keys // s.page_size].contiguous()

            def attend(q, kc, vc):
                q = F.pad(q, (0, 0, 0, rows - n))
                pooled_k = fpv2.pool_pages(kc, pages, cfg.block_k, keys)
                pooled_v = fpv2.pool_pages(vc, pages, cfg.block_k, keys)
                selected, _ = fpv2.block_scores_and_select(q, pooled_k, scale=s.head_dim**-0.5, config=cfg,
                                                           offset=offset, query_length=n)
                lists = fpv2.compact_block_indices(selected, config=cfg, offset=offset, query_length=n,
                                                   key_length=length)
                out = fpv2.sparse_attention_paged(q, kc, vc, pages, pooled_k, pooled_v, *lists,
                                                  scale=s.head_dim**-0.5, config=cfg, offset=offset,
                                                  query_length=n, key_length=length)
                return out[:, :n].transpose(0, 1)

            x = self.weights["embed"][ids[offset:length]]
            for layer in range(s.layers):
                x = self._block(x, layer, positions, slots, attend, heads_first=True)
        self.lengths[request] = self.held[request] = ids.numel()
        return self._logits(x[-1])

    @torch.no_grad()
    def decode(self, ids: torch.Tensor) -> torch.Tensor:
        """Logits ``[requests, vocab]`` after one more token of every request."""
        s = self.shape
        if len(ids) != len(self.held):
            raise ValueError("every request needs its token")
        if max(self.held) >= s.max_tokens:
            raise ValueError(f"a request would pass max_tokens = {s.max_tokens}")
        self.held = [n + 1 for n in self.held]
        positions = self.lengths.long()
        slots = self._slots(torch.arange(len(ids), device=ids.device), positions)
        lengths = self.lengths + 1

        def attend(q, kc, vc):
            return fpv2.decode_attention(q, kc, vc, self.tables, lengths, scale=s.head_dim**-0.5)

        x = self.weights["embed"][ids]
        for layer in range(s.layers):
            x = self._block(x, layer, positions, slots, attend, heads_first=False)
        self.lengths.copy_(lengths)
        return self._logits(x)


def generate(model: PagedModel, prompts: list[torch.Tensor], new_tokens: int, *, temperature: float = 0.8,
             top_k: int = 50, top_p: float = 0.95, seed: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    """``new_tokens`` tokens for each prompt and their log-probabilities."""
    if len(prompts) != len(model.held):
        raise ValueError(f"the model holds {len(model.held)} requests")
    if max(ids.numel() for ids in prompts) + new_tokens - 1 > model.shape.max_tokens:
        raise ValueError(f"prompt and new tokens would pass max_tokens = {model.shape.max_tokens}")
    logits = torch.stack([model.prefill(r, ids) for r, ids in enumerate(prompts)])
    gen = torch.Generator(device=logits.device).manual_seed(seed)
    noise = torch.empty(logits.shape, device=logits.device)
    tokens, logprobs = [], []
    for step in range(new_tokens):
        noise.exponential_(generator=gen)
        ids, lp = fpv2.sample_tokens(logits, noise, temperature=temperature, top_k=top_k, top_p=top_p,
                                     return_logprobs=True)
        tokens.append(ids)
        logprobs.append(lp)
        if step + 1 < new_tokens:
            logits = model.decode(ids)
    return torch.stack(tokens, 1), torch.stack(logprobs, 1)


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--prompts", type=int, default=3)
    ap.add_argument("--prompt-tokens", type=int, default=4000)
    ap.add_argument("--new-tokens", type=int, default=32)
    args = ap.parse_args()
    shape = Shape(max_tokens=args.prompt_tokens + args.new_tokens)
    model = PagedModel(shape, random_weights(shape), args.prompts)
    gen = torch.Generator(device="cuda").manual_seed(1)
    prompts = [torch.randint(0, shape.vocab, (max(1, args.prompt_tokens - 37 * r),), generator=gen, device="cuda")
               for r in range(args.prompts)]
    generate(model, prompts, 2)   # warm-up
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    tokens, logprobs = generate(model, prompts, args.new_tokens)
    end.record()
    torch.cuda.synchronize()
    print(f"{args.prompts} prompts, {args.new_tokens} new tokens each: {start.elapsed_time(end):.1f} ms")
    for r, row in enumerate(tokens.tolist()):
        print(f"request {r}: mean log-probability {float(logprobs[r].mean()):.3f}, tokens {row[:12]} ...")


if __name__ == "__main__":
    main()
