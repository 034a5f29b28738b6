"""The operators of the decode step that are measured, their cases and their plain forms.

``qk_norm_rope``: RMS norm of every query and key head, rotary embedding and the
write of K and V into their cache pages. ``decode_attention``: attention of the
newest token (or the newest few) of each sequence over its paged K/V.
``sample_tokens``: the next token of each row of logits from given random
numbers. With ``own`` false ``run`` computes them with elementary torch
operations in float32, else through the package's public calls.
"""

import math
import os
import sys

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_package = None


def _fpv2():
    global _package
    if _package is None:
        sys.path.insert(0, os.path.abspath("flashprefillv2-mlx_b200"))
        import fpv2

        _package = fpv2
    return _package


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------


def _rope(name, tokens, q_heads, kv_heads, dim, rotary, dtype, *, norm=True, interleaved=False, cache=0,
          heads_first=False):
    return {"op": "rope", "name": name, "tokens": tokens, "q_heads": q_heads, "kv_heads": kv_heads,
            "dim": dim, "rotary": rotary, "dtype": dtype, "norm": norm, "interleaved": interleaved,
            "cache": cache, "heads_first": heads_first}


def _decode(name, batch, longest, shortest, new, q_heads, kv_heads, dim, page, dtype, *, window=0, sinks=0,
            lse=False):
    return {"op": "decode", "name": name, "batch": batch, "longest": longest, "shortest": shortest,
            "new": new, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "dtype": dtype, "window": window, "sinks": sinks, "lse": lse}


def _sample(name, rows, vocab, dtype, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, logprobs=False):
    return {"op": "sample", "name": name, "rows": rows, "vocab": vocab, "dtype": dtype,
            "temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p,
            "logprobs": logprobs}


def listed():
    return [
        # one request, one new token of a 32/8-head layer written to its page: pure latency
        _rope("rope_1_token", 1, 32, 8, 128, 128, "bf16", cache=16),
        # a decode step of many requests, pages of 64
        _rope("rope_batch_192", 192, 64, 8, 128, 128, "f16", cache=64),
        # a 2048-token prefill chunk, queries laid out for the prefill attention, K and V paged
        _rope("rope_chunk_2048", 2048, 32, 8, 128, 128, "bf16", cache=16, heads_first=True),
        # a long odd prompt without a cache: no norm weights, part of each head rotated, adjacent pairs
        _rope("rope_prompt_31007_f32", 31007, 16, 4, 96, 64, "f32", norm=False, interleaved=True),
        # a short chat of one request: latency
        _decode("decode_1x517", 1, 517, 517, 1, 32, 8, 128, 16, "bf16"),
        # one request behind a 64k prefill: the length is split over the GPU and joined
        _decode("decode_1x65536", 1, 65536, 65536, 1, 32, 8, 128, 16, "bf16"),
        # a full serving batch of ragged lengths
        _decode("decode_64_ragged", 64, 16384, 129, 1, 32, 8, 128, 64, "bf16", lse=True),
        # four drafted tokens a request checked at once in a layer with a sliding window and sinks
        _decode("decode_24_window_draft", 24, 20011, 3, 4, 64, 8, 64, 32, "f16", window=4096, sinks=4),
        # one request with the usual filters over a 151936-token vocabulary: latency
        _sample("sample_1_topk_topp", 1, 151936, "bf16", temperature=0.7, top_k=50, top_p=0.9),
        # a batch drawn from the nucleus of float32 logits, with log-probabilities
        _sample("sample_64_nucleus", 64, 151936, "f32", temperature=0.8, top_p=0.9, logprobs=True),
        # rollouts: the whole distribution, nothing filtered, with log-probabilities
        _sample("sample_200_all", 200, 151936, "bf16", logprobs=True),
        # a smaller odd vocabulary under every filter
        _sample("sample_33_minp_odd", 33, 50003, "f16", temperature=1.3, top_k=1000, top_p=0.97, min_p=0.02),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rope", "decode", "decode", "sample"])
    if op == "rope":
        tokens = _spread(rng, 1, 16000)
        dim = rng.choice([64, 80, 96, 128, 128, 256])
        q_heads, kv_heads = rng.choice([(32, 8), (64, 8), (16, 16), (12, 4), (8, 1)])
        cache = rng.choice([0, 16, 24, 64])
        dtype = rng.choice(["bf16", "bf16", "f16"] if cache else ["bf16", "f16", "f32"])
        value = (q_heads + 2 * kv_heads) * dim * (4 if dtype == "f32" else 2)
        tokens = min(tokens, 31007 * 20 * 96 * 4 // value)
        case = _rope(None, tokens, q_heads, kv_heads, dim, rng.choice([dim, dim, dim // 2]), dtype,
                     norm=rng.random() < 0.8, interleaved=rng.random() < 0.3, cache=cache,
                     heads_first=rng.random() < 0.4)
    elif op == "decode":
        batch = _spread(rng, 1, 64)
        dim = rng.choice([64, 96, 128, 128, 256])
        q_heads, kv_heads = rng.choice([(32, 8), (64, 8), (8, 8), (12, 4), (8, 2), (6, 1)])
        longest = _spread(rng, 1, min(65536, 220_000_000 // (batch * kv_heads * dim)))
        windowed = rng.random() < 0.35
        case = _decode(None, batch, longest, max(1, longest // rng.choice([1, 4, 100])),
                       rng.choice([1, 1, 1, 2, 5]), q_heads, kv_heads, dim,
                       rng.choice([8, 16, 20, 64, 128]), rng.choice(["bf16", "f16"]),
                       window=_spread(rng, 16, 8192) if windowed else 0,
                       sinks=rng.choice([0, 4, 130]) if windowed else 0, lse=rng.random() < 0.5)
    else:
        rows = _spread(rng, 1, 200)
        case = _sample(None, rows, min(_spread(rng, 1000, 262144), 22_000_000 // rows),
                       rng.choice(["bf16", "f16", "f32"]), temperature=rng.choice([0.0, 0.6, 1.0, 1.7]),
                       top_k=rng.choice([0, 0, 20, 300]), top_p=rng.choice([1.0, 0.95, 0.8, 0.3]),
                       min_p=rng.choice([0.0, 0.0, 0.05]), logprobs=rng.random() < 0.5)
    del case["name"]
    return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    {"rope": _prepare_rope, "decode": _prepare_decode, "sample": _prepare_sample}[case["op"]](case, gen, state)
    return state


def _prepare_rope(c, gen, s):
    dtype = _TYPES[c["dtype"]]
    n, hq, hkv, d = c["tokens"], c["q_heads"], c["kv_heads"], c["dim"]
    # q, k and v are views of one fused projection's output
    qkv = torch.randn(n, hq + 2 * hkv, d, generator=gen, device="cuda") * 1.7
    qkv = qkv.to(dtype)
    s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    s["q_weight"] = s["k_weight"] = None
    if c["norm"]:
        s["q_weight"] = (1 + 0.2 * torch.randn(d, generator=gen, device="cuda")).to(dtype)
        s["k_weight"] = (1 + 0.2 * torch.randn(d, generator=gen, device="cuda")).to(dtype)
    # the rotation table of the model, [positions, rotary]: cosines, then sines
    span = 65536
    half = c["rotary"] // 2
    freq = 1e6 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
    angle = torch.arange(span, dtype=torch.float64, device="cuda")[:, None] * freq
    s["table"] = torch.cat([angle.cos(), angle.sin()], -1).float()
    if n > 1024:   # a prompt's consecutive positions
        s["positions"] = torch.arange(n, device="cuda", dtype=torch.int32) + 4096
    else:          # one position for each of a batch's requests
        s["positions"] = torch.randint(0, span, (n,), generator=gen, device="cuda", dtype=torch.int32)
    if c["cache"]:
        page = c["cache"]
        pages = -(-n // page) + 2
        s["k_cache"] = torch.zeros(pages, page, hkv, d, dtype=dtype, device="cuda")
        s["v_cache"] = torch.zeros(pages, page, hkv, d, dtype=dtype, device="cuda")
        order = torch.randperm(pages, generator=gen, device="cuda")
        at = torch.arange(n, device="cuda")
        s["slots"] = order[at // page] * page + at % page


def _prepare_decode(c, gen, s):
    dtype = _TYPES[c["dtype"]]
    b, d, page, hkv = c["batch"], c["dim"], c["page"], c["kv_heads"]
    fill = torch.rand(b, generator=gen, device="cuda", dtype=torch.float64)
    low, high = math.log(c["shortest"]), math.log(c["longest"])
    lengths = torch.exp(low + fill * (high - low)).round().int()
    lengths[0] = c["longest"]
    s["lengths"] = lengths
    width = -(-c["longest"] // page)
    # pages of all requests in one pool, handed out in random order; the tables' unused ends hold -1
    need = (lengths + page - 1) // page
    used = torch.arange(width, device="cuda")[None, :] < need[:, None]
    total = int(need.sum())
    tables = torch.full((b, width), -1, dtype=torch.int32, device="cuda")
    tables[used] = torch.randperm(total, generator=gen, device="cuda").int()
    s["tables"] = tables
    s["k_cache"] = torch.randn(total, page, hkv, d, generator=gen, device="cuda", dtype=dtype)
    s["v_cache"] = torch.randn(total, page, hkv, d, generator=gen, device="cuda", dtype=dtype)
    first = tables[:, 0].long()
    s["k_cache"][first, 0] *= 2   # the first token draws weight, as sinks do
    s["q"] = torch.randn(b, c["new"], c["q_heads"], d, generator=gen, device="cuda").to(dtype)


def _prepare_sample(c, gen, s):
    rows, vocab = c["rows"], c["vocab"]
    # a bulk of unlikely tokens and some that stand out by a few nats
    logits = 2.2 * torch.randn(rows, vocab, generator=gen, device="cuda")
    at = torch.randint(0, vocab, (rows, 1), generator=gen, device="cuda")
    at = (at + torch.arange(40, device="cuda") * (vocab // 40)) % vocab
    logits.scatter_(1, at, 11 - 6 * torch.rand(rows, 40, generator=gen, device="cuda"))
    s["logits"] = logits.to(_TYPES[c["dtype"]])
    s["noise"] = torch.empty(rows, vocab, device="cuda").exponential_(generator=gen).clamp_min_(1e-30)
    # every request has its own settings, spread around the case's
    wide = torch.rand(rows, generator=gen, device="cuda")
    s["temperature"] = c["temperature"] * (0.9 + 0.2 * wide)
    s["top_k"] = (c["top_k"] * (0.8 + 0.2 * wide)).int()
    s["top_p"] = c["top_p"] - (0.05 * wide if c["top_p"] < 1 else 0 * wide)
    s["min_p"] = c["min_p"] * wide


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def run(state):
    op = state["case"]["op"]
    if op == "rope":
        return _own_rope(state) if own else _plain_rope(state)
    if op == "decode":
        return _own_decode(state) if own else _plain_decode(state)
    return _own_sample(state) if own else _plain_sample(state)


def _own_rope(s):
    c = s["case"]
    paged = {"v": s["v"], "k_cache": s["k_cache"], "v_cache": s["v_cache"], "slots": s["slots"]} if c["cache"] else {}
    q, k = _fpv2().qk_norm_rope(s["q"], s["k"], s["positions"], s["table"], q_weight=s["q_weight"],
                                k_weight=s["k_weight"], eps=1e-6, interleaved=c["interleaved"],
                                heads_first=c["heads_first"], **paged)
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]} if c["cache"] else {"q": q, "k": k}


def _own_decode(s):
    c = s["case"]
    got = _fpv2().decode_attention(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["lengths"],
                                   scale=c["dim"] ** -0.5, window=c["window"], sinks=c["sinks"],
                                   return_lse=c["lse"])
    return {"out": got[0], "lse": got[1]} if c["lse"] else {"out": got}


def _own_sample(s):
    c = s["case"]
    got = _fpv2().sample_tokens(s["logits"], s["noise"], temperature=s["temperature"], top_k=s["top_k"],
                                top_p=s["top_p"], min_p=s["min_p"], return_logprobs=c["logprobs"])
    return {"tokens": got[0], "logprobs": got[1]} if c["logprobs"] else {"tokens": got}


def _plain_norm_rope(x, weight, cos, sin, interleaved):
    x = x.float()
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
    if weight is not None:
        x = x * weight.float()
    rot = 2 * cos.shape[-1]
    part, rest = x[..., :rot], x[..., rot:]
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = part[..., :rot // 2], part[..., rot // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, rest], -1)


def _plain_rope(s):
    c = s["case"]
    row = s["table"][s["positions"].long()]
    cos, sin = row[:, None, :c["rotary"] // 2], row[:, None, c["rotary"] // 2:]
    q = _plain_norm_rope(s["q"], s["q_weight"], cos, sin, c["interleaved"]).to(s["q"].dtype)
    k = _plain_norm_rope(s["k"], s["k_weight"], cos, sin, c["interleaved"]).to(s["k"].dtype)
    if c["heads_first"]:
        q = q.transpose(0, 1).contiguous()
    if not c["cache"]:
        return {"q": q, "k": k.transpose(0, 1).contiguous() if c["heads_first"] else k}
    shape = (-1,) + tuple(s["k_cache"].shape[2:])
    s["k_cache"].view(shape)[s["slots"]] = k
    s["v_cache"].view(shape)[s["slots"]] = s["v"]
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_decode(s):
    c = s["case"]
    b, new, hq, d = s["q"].shape
    hkv = c["kv_heads"]
    group = hq // hkv
    tables = s["tables"].long().clamp_min(0)
    longest = tables.shape[1] * c["page"]
    k = s["k_cache"][tables].view(b, longest, hkv, d).permute(0, 2, 3, 1).float()
    q = s["q"].view(b, new, hkv, group, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, new * group, d).float()
    scores = (torch.matmul(q, k) * d ** -0.5).view(b, hkv, new, group, longest)
    del k
    at = torch.arange(longest, device="cuda")
    pos = s["lengths"][:, None] - new + torch.arange(new, device="cuda")[None, :]
    seen = at <= pos[..., None]
    if c["window"]:
        seen &= (at < c["sinks"]) | (at > pos[..., None] - c["window"])
    scores = scores.masked_fill(~seen[:, None, :, None, :], -math.inf)
    top = scores.amax(-1, keepdim=True)
    weight = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = weight.sum(-1, keepdim=True)
    v = s["v_cache"][tables].view(b, longest, hkv, d).permute(0, 2, 1, 3).float()
    out = torch.matmul(weight.view(b, hkv, new * group, longest), v).view(b, hkv, new, group, d)
    out = torch.where(total > 0, out / total.clamp_min(1e-30), 0.0)
    out = out.permute(0, 2, 1, 3, 4).reshape(b, new, hq, d).to(s["q"].dtype)
    if not c["lse"]:
        return {"out": out}
    lse = (top + torch.log(total))[..., 0]
    return {"out": out, "lse": lse.permute(0, 2, 1, 3).reshape(b, new, hq)}


def _plain_sample(s):
    c = s["case"]
    x = s["logits"].float()
    rows, vocab = x.shape
    x = torch.where(torch.isnan(x), -math.inf, x)
    top = x.amax(-1, keepdim=True)
    greedy = (s["temperature"] == 0)[:, None]
    z = (x - top) / torch.where(greedy, 1.0, s["temperature"][:, None])
    z_sorted, order = torch.sort(z, dim=-1, descending=True, stable=True)
    w = torch.exp(z_sorted)
    rank = torch.arange(vocab, device="cuda")
    k = s["top_k"][:, None]
    keep = (rank < k) | (k <= 0)
    run_up = torch.cumsum(w * keep, -1)
    before = torch.cat([torch.zeros_like(run_up[:, :1]), run_up[:, :-1]], -1)
    p = s["top_p"][:, None]
    keep &= (before < p * run_up[:, -1:]) | (p >= 1)
    keep &= w >= s["min_p"][:, None]
    keep |= rank == 0
    kept = torch.zeros_like(keep).scatter_(1, order, keep)
    score = torch.where(kept, z - torch.log(s["noise"]), -math.inf)
    score = torch.where(greedy, x, score)
    best = score == score.amax(-1, keepdim=True)
    tokens = torch.where(best, rank, vocab).amin(-1)
    if not c["logprobs"]:
        return {"tokens": tokens}
    logprobs = z.gather(1, tokens[:, None])[:, 0] - torch.log(w.sum(-1))
    return {"tokens": tokens, "logprobs": logprobs}


# ---------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# ---------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "decode": _exact_decode, "sample": _exact_sample}[case["op"]](case, s)


def _exact_rope(c, s):
    n, half = c["tokens"], c["rotary"] // 2
    turn = torch.complex(*s["table"].double()[s["positions"].long()].split(half, -1))[:, None, :]

    def one(x, weight):
        x = x.double()
        y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / c["dim"] + 1e-6)
        if weight is not None:
            y = y * weight.double()
        first = range(0, 2 * half, 2) if c["interleaved"] else range(half)
        a = torch.tensor(list(first), device="cuda")
        b = a + (1 if c["interleaved"] else half)
        pair = torch.complex(y[..., a], y[..., b]) * turn
        y[..., a], y[..., b] = pair.real, pair.imag
        return y

    q, k = one(s["q"], s["q_weight"]), one(s["k"], s["k_weight"])
    if c["heads_first"]:
        q = q.permute(1, 0, 2).contiguous()
    if not c["cache"]:
        return {"q": q, "k": k.permute(1, 0, 2).contiguous() if c["heads_first"] else k}
    caches = []
    for new in (k, s["v"].double()):
        cache = torch.zeros(s["k_cache"].shape, dtype=torch.float64, device="cuda")
        for page in range(-(-n // c["cache"])):
            at = int(s["slots"][page * c["cache"]])
            rows = new[page * c["cache"]:(page + 1) * c["cache"]]
            cache[at // c["cache"], :rows.shape[0]] = rows
        caches.append(cache)
    return {"q": q, "k_cache": caches[0], "v_cache": caches[1]}


def _exact_decode(c, s):
    group = c["q_heads"] // c["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:3], -math.inf, dtype=torch.float64, device="cuda")
    for b, length in enumerate(s["lengths"].tolist()):
        pages = s["tables"][b, :-(-length // c["page"])].long()
        k = s["k_cache"][pages].flatten(0, 1)[:length].double().repeat_interleave(group, 1)
        v = s["v_cache"][pages].flatten(0, 1)[:length].double().repeat_interleave(group, 1)
        for t in range(c["new"]):
            pos = length - c["new"] + t
            keys = set(range(pos + 1)) if not c["window"] else (
                set(range(min(c["sinks"], pos + 1))) | set(range(max(0, pos - c["window"] + 1), pos + 1)))
            if not keys:
                continue
            at = torch.tensor(sorted(keys), device="cuda")
            score = torch.einsum("hd,lhd->hl", s["q"][b, t].double(), k[at]) / math.sqrt(c["dim"])
            lse[b, t] = torch.logsumexp(score, -1)
            out[b, t] = torch.einsum("hl,lhd->hd", torch.softmax(score, -1), v[at])
    return {"out": out, "lse": lse} if c["lse"] else {"out": out}


def _exact_sample(c, s):
    tokens, logprobs = [], []
    for r in range(c["rows"]):
        x = s["logits"][r].double()
        heat = float(s["temperature"][r])
        z = x / (heat if heat > 0 else 1.0)
        whole = torch.logsumexp(z, 0)
        if heat == 0:
            token = int((x == x.max()).nonzero()[0])
        else:
            by = torch.argsort(-x, stable=True)
            k = int(s["top_k"][r])
            by = by[:k] if k > 0 else by
            share = torch.softmax(z[by], 0)
            ahead = torch.cumsum(share, 0) - share
            p = float(s["top_p"][r])
            count = int((ahead < p).sum()) if p < 1 else by.numel()
            least = float(s["min_p"][r]) * float(share[0])
            by = by[:max(1, count)]
            by = by[share[:by.numel()] >= least]
            token = int(by[torch.argmax(z[by] - torch.log(s["noise"][r].double()[by]))])
        tokens.append(token)
        logprobs.append(z[token] - whole)
    got = {"tokens": torch.tensor(tokens, device="cuda")}
    if c["logprobs"]:
        got["logprobs"] = torch.stack(logprobs)
    return got


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------


def work(case):
    c = case
    size = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "rope":
        heads = c["q_heads"] + c["kv_heads"] * (2 if c["cache"] else 1)
        values = c["tokens"] * heads * c["dim"]
        return {"bytes": 2 * values * size + c["tokens"] * (4 * c["rotary"] + 4 + (8 if c["cache"] else 0)),
                "flops": 7 * values}
    if c["op"] == "decode":
        # the expected length of the log-uniform spread; the first request has the longest
        low, high, b = c["shortest"], c["longest"], c["batch"]
        mean = (high - low) / math.log(high / low) if high > low else high
        seen = [min(x, c["window"] + c["new"] + c["sinks"]) if c["window"] else x for x in (high, mean)]
        keys = seen[0] + (b - 1) * seen[1]
        rows = c["new"] * c["q_heads"]
        return {"bytes": 2 * keys * c["kv_heads"] * c["dim"] * size + 2 * b * rows * c["dim"] * size
                + 4 * keys / c["page"] + 4 * b + (4 * b * rows if c["lse"] else 0),
                "flops": 4 * keys * rows * c["dim"]}
    # every logit, and the noise of what is kept: k tokens, all of them, or (a nucleus) at least one
    kept = c["top_k"] or (c["vocab"] if c["top_p"] >= 1 and c["temperature"] > 0 else 1)
    return {"bytes": c["rows"] * (c["vocab"] * size + 4 * kept + 24 + (4 if c["logprobs"] else 0)),
            "flops": 4 * c["rows"] * c["vocab"]}
