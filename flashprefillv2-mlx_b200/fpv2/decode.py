"""The decode step next to the sparse prefill (no reference counterpart: the
reference leaves it to its model library).

``qk_norm_rope`` norms and rotates the query and key heads and writes K and V into
the page pools that ``pool_pages`` / ``sparse_attention_paged`` prefill from and
``decode_attention`` reads; ``decode_attention`` attends the newest tokens of every
sequence over them; ``sample_tokens`` picks the next tokens. The kernels have no
derivatives: inputs that require grad are refused while grad mode is on, and those with
a forward-mode tangent always.
"""

from __future__ import annotations

import functools
import struct

import torch
from torch.autograd import forward_ad

from fpv2 import _lib

DECODE_HEAD_DIMS = (64, 96, 128, 256)
_HALF = (torch.float16, torch.bfloat16)
_INT32_MAX = 2**31 - 1

# The parameter structures of include/fpv2_b200.h, field by field (null pointers are 0).
# These calls are short on the GPU, so their host side avoids what costs microseconds:
# many ctypes arguments, views, Stream objects.
_pack_rope = struct.Struct("@3q 5q 6q 2q 3q 1q 2q 1q 1d 2q 4q 2q 6q 3q").pack
_pack_decode = struct.Struct("@3q 1q 5q 3q 6q 3q 1q 4q 1d 3q 1q").pack
_pack_sample = struct.Struct("@5q 2q 1q1d 2q 1q1d 1q1d 2q").pack


def _refuse_grad(what: str) -> None:
    raise ValueError(f"{what} has no backward; call it under torch.no_grad()")


def _refuse_tangents(what: str, *tensors: object) -> None:
    """Outside a forward-mode level (-1) no tensor has a tangent, and nothing is looked at."""
    if getattr(forward_ad, "_current_level", 0) < 0:
        return
    for t in tensors:
        if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError(f"{what} has no forward-mode derivative; pass tensors without tangents")


def _call(fn, device: int, params: bytes) -> None:
    """One library call on ``device`` and its current stream."""
    if device == torch.cuda.current_device():
        rc = fn(params, _lib.stream_of_device(device))
    else:
        with torch.cuda.device(device):
            rc = fn(params, _lib.stream_of_device(device))
    if rc:
        _lib.check(rc)


@functools.lru_cache(maxsize=None)
def _workspace_bytes(new: int, q_heads: int, kv_heads: int, dim: int) -> int:
    return int(_lib.lib().fpv2_decode_workspace_bytes(new, q_heads, kv_heads, dim))


def rope_table(positions: int, rotary_dim: int, *, theta: float = 10000.0,
               device: torch.device | str | None = None) -> torch.Tensor:
    """Rotation table ``[positions, rotary_dim]`` for ``qk_norm_rope``: the cosines of
    ``p * theta ** (-2 i / rotary_dim)``, then their sines, computed in float64 and
    rounded to float32."""
    if positions <= 0 or rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError("positions must be positive and rotary_dim even and positive")
    half = rotary_dim // 2
    freq = theta ** (-torch.arange(half, dtype=torch.float64, device=device) / half)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], -1).float()


def qk_norm_rope(
    q: torch.Tensor,
    k: torch.Tensor,
    positions: torch.Tensor,
    table: torch.Tensor,
    *,
    q_weight: torch.Tensor | None = None,
    k_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    interleaved: bool = False,
    heads_first: bool = False,
    v: torch.Tensor | None = None,
    k_cache: torch.Tensor | None = None,
    v_cache: torch.Tensor | None = None,
    slots: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """RMS norm of every query and key head, then rotary embedding, in one pass.

    ``q`` is ``[tokens, q_heads, dim]`` and ``k`` ``[tokens, kv_heads, dim]`` (any token
    and head strides, so views of one fused projection do). Each head is divided by
    ``sqrt(mean(x^2) + eps)``, multiplied by ``q_weight`` / ``k_weight`` ``[dim]`` where
    given, and its first ``table.shape[1]`` dimensions are rotated by the row of
    ``table`` (see ``rope_table``) of the token's position (int32 or int64, clamped
    into the table): pairs ``(i, i + rotary / 2)``, or ``(2i, 2i + 1)`` with
    ``interleaved``. Float32 arithmetic, rounded once.

    Returns ``(q, k)`` as ``[tokens, heads, dim]``, or ``[heads, tokens, dim]`` (the
    prefill operators' layout) with ``heads_first``. With ``v``, ``k_cache``, ``v_cache``
    (page pools ``[pages, page_size, kv_heads, dim]``, any strides) and ``slots`` (int64
    ``[tokens]``, ``page * page_size + row``; negative or past the pool: the token is
    not written) k and v go into the cache and the returned k is None. Slots must
    not repeat.
    """
    qshape, kshape = q.shape, k.shape
    if len(qshape) != 3 or len(kshape) != 3:
        raise ValueError("q and k must have shape [tokens, heads, dim]")
    tokens, q_heads, dim = qshape
    kv_heads = kshape[1]
    if kshape[0] != tokens or kshape[2] != dim:
        raise ValueError("q and k must have the same tokens and head dimension")
    if not q_heads or not kv_heads:
        raise ValueError("q and k must have heads")
    if not 0 < dim <= 256:
        raise ValueError("head dimension must be in [1, 256]")
    dtype = q.dtype
    code = _lib.dtype_code(dtype)
    if k.dtype != dtype:
        raise ValueError("q and k must share their dtype")
    wide = positions.dtype == torch.int64
    if positions.shape != (tokens,) or not (wide or positions.dtype == torch.int32):
        raise ValueError("positions must be an int32 or int64 tensor [tokens]")
    if table.ndim != 2 or table.dtype != torch.float32 or not table.shape[0]:
        raise ValueError("table must be a float32 tensor [positions, rotary_dim]")
    span, rotary = table.shape
    if not rotary or rotary % 2 or rotary > dim:
        raise ValueError("rotary_dim must be even and in [2, head_dim]")
    weight_code = code
    if q_weight is not None:
        if q_weight.shape != (dim,) or k_weight is not None and q_weight.dtype != k_weight.dtype:
            raise ValueError("norm weights must share one dtype and have shape [head_dim]")
        weight_code = _lib.dtype_code(q_weight.dtype)
    if k_weight is not None:
        if k_weight.shape != (dim,):
            raise ValueError("norm weights must share one dtype and have shape [head_dim]")
        weight_code = _lib.dtype_code(k_weight.dtype)
    paged = k_cache is not None
    if (v is not None) != paged or (v_cache is not None) != paged or (slots is not None) != paged:
        raise ValueError("v, k_cache, v_cache and slots go together")
    kc = vc = (0, 0, 0)
    if paged:
        if v.shape != kshape or v.dtype != dtype:
            raise ValueError("v must have the shape and dtype of k")
        cshape = k_cache.shape
        if len(cshape) != 4 or cshape[2] != kv_heads or cshape[3] != dim or k_cache.dtype != dtype \
                or v_cache.dtype != dtype:
            raise ValueError("caches must have shape [pages, page_size, kv_heads, dim] and k's dtype")
        if v_cache.shape != cshape or not cshape[0] or not cshape[1]:
            raise ValueError("k_cache and v_cache must have identical non-empty shapes")
        kc, vc = k_cache.stride(), v_cache.stride()
        if kc[3] != 1 or vc[3] != 1:
            raise ValueError("a cache's head dimension must be contiguous")
        if slots.shape != (tokens,) or slots.dtype != torch.int64:
            raise ValueError("slots must be an int64 tensor [tokens]")
    if torch.is_grad_enabled() and (
            q.requires_grad or k.requires_grad or table.requires_grad
            or q_weight is not None and q_weight.requires_grad
            or k_weight is not None and k_weight.requires_grad
            or paged and (v.requires_grad or k_cache.requires_grad or v_cache.requires_grad)):
        _refuse_grad("qk_norm_rope")
    _refuse_tangents("qk_norm_rope", q, k, table, q_weight, k_weight, v, k_cache, v_cache)
    device = q.get_device()
    if device < 0 or k.get_device() != device or positions.get_device() != device or table.get_device() != device \
            or q_weight is not None and q_weight.get_device() != device \
            or k_weight is not None and k_weight.get_device() != device \
            or paged and (v.get_device() != device or k_cache.get_device() != device
                          or v_cache.get_device() != device or slots.get_device() != device):
        _lib.require_cuda(q, k, positions, table, q_weight, k_weight, v, k_cache, v_cache, slots)
    # the head dimension contiguous (a copy only where it is not), the small ones as a whole
    qs, ks = q.stride(), k.stride()
    if qs[2] != 1:
        q = q.contiguous()
        qs = q.stride()
    if ks[2] != 1:
        k = k.contiguous()
        ks = k.stride()
    positions, table = positions.contiguous(), table.contiguous()
    if q_weight is not None:
        q_weight = q_weight.contiguous()
    if k_weight is not None:
        k_weight = k_weight.contiguous()
    if heads_first:
        q_out = q.new_empty((q_heads, tokens, dim))
        qo_t, qo_h, ko_t, ko_h = dim, tokens * dim, dim, tokens * dim
    else:
        q_out = q.new_empty(qshape)
        qo_t, qo_h, ko_t, ko_h = q_heads * dim, dim, kv_heads * dim, dim
    if paged:
        k_out, k_out_ptr = None, 0
        vs = v.stride()
        if vs[2] != 1:
            v = v.contiguous()
            vs = v.stride()
        slots = slots.contiguous()
        v_ptr, kc_ptr, vc_ptr, slots_ptr = v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), slots.data_ptr()
        pages, page_size = cshape[0], cshape[1]
    else:
        k_out = q.new_empty((kv_heads, tokens, dim) if heads_first else kshape)
        k_out_ptr = k_out.data_ptr()
        vs = (0, 0)
        v_ptr = kc_ptr = vc_ptr = slots_ptr = pages = page_size = 0
    _call(_lib.lib().fpv2_qk_norm_rope, device, _pack_rope(
        q.data_ptr(), k.data_ptr(), v_ptr, code, tokens, q_heads, kv_heads, dim, qs[0], qs[1], ks[0], ks[1],
        vs[0], vs[1], positions.data_ptr(), wide, table.data_ptr(), span, rotary, bool(interleaved),
        0 if q_weight is None else q_weight.data_ptr(), 0 if k_weight is None else k_weight.data_ptr(),
        weight_code, eps, q_out.data_ptr(), k_out_ptr, qo_t, qo_h, ko_t, ko_h, kc_ptr, vc_ptr,
        kc[0], kc[1], kc[2], vc[0], vc[1], vc[2], slots_ptr, pages, page_size))
    return q_out, k_out


def _address(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


def _rows(x: torch.Tensor) -> torch.Tensor:
    """``x`` with a contiguous last dimension (a copy only where it is not)."""
    return x if x.stride(-1) == 1 else x.contiguous()


def decode_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_tables: torch.Tensor,
    lengths: torch.Tensor,
    *,
    scale: float,
    window: int = 0,
    sinks: int = 0,
    return_lse: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Attention of the newest token (or the newest few) of each sequence over its paged K/V.

    ``q`` is ``[batch, heads, dim]``, or ``[batch, new, heads, dim]`` for several new
    tokens (drafts to verify); ``k_cache`` and ``v_cache`` are page pools ``[pages,
    page_size, kv_heads, dim]`` with any page, row and head strides (multiples of 8
    elements); ``block_tables`` int32 ``[batch, max_pages]`` holds each sequence's
    pages and ``lengths`` int32 ``[batch]`` its keys, the new tokens' included.
    Query ``t`` sits at position ``p = length - new + t`` and sees the keys ``j <= p``
    with ``j < sinks`` or ``j > p - window``; ``window=0`` sees all of them. A query
    without a visible key gets zeros. float16 / bfloat16, head_dim 64, 96, 128 or
    256, any page size. Returns the output in ``q``'s shape, and with ``return_lse``
    the float32 log-sum-exp of the scaled scores (without the last dimension).
    """
    shape, kshape = q.shape, k_cache.shape
    if len(shape) == 3:
        (batch, q_heads, dim), new = shape, 1
    elif len(shape) == 4:
        batch, new, q_heads, dim = shape
    else:
        raise ValueError("q must have shape [batch, heads, dim] or [batch, new, heads, dim]")
    if len(kshape) != 4:
        raise ValueError("k_cache must have shape [pages, page_size, kv_heads, dim]")
    dtype = q.dtype
    if dtype not in _HALF or k_cache.dtype != dtype or v_cache.dtype != dtype:
        raise ValueError("q and the caches must share float16 or bfloat16 dtype")
    if v_cache.shape != kshape:
        raise ValueError("k_cache and v_cache must have identical shapes")
    pages, page_size, kv_heads, kdim = kshape
    if dim != kdim or dim not in DECODE_HEAD_DIMS:
        raise ValueError(f"head dimension must be one of {DECODE_HEAD_DIMS}")
    if not kv_heads or not q_heads or q_heads % kv_heads:
        raise ValueError("query heads must be divisible by KV heads")
    if not new:
        raise ValueError("q must hold at least one new token a sequence")
    if not pages or not page_size:
        raise ValueError("the caches are empty")
    tshape = block_tables.shape
    if len(tshape) != 2 or block_tables.dtype != torch.int32 or tshape[0] != batch:
        raise ValueError("block_tables must be an int32 tensor [batch, max_pages]")
    if lengths.shape != (batch,) or lengths.dtype != torch.int32:
        raise ValueError("lengths must be an int32 tensor [batch]")
    width = tshape[1]
    if not width:
        raise ValueError("block_tables holds no pages")
    if not (0 <= window <= _INT32_MAX and 0 <= sinks <= _INT32_MAX):
        raise ValueError("window and sinks must be non-negative 32-bit integers")
    if torch.is_grad_enabled() and (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad):
        _refuse_grad("decode_attention")
    _refuse_tangents("decode_attention", q, k_cache, v_cache)
    device = q.get_device()
    if device < 0 or k_cache.get_device() != device or v_cache.get_device() != device \
            or block_tables.get_device() != device or lengths.get_device() != device:
        _lib.require_cuda(q, k_cache, v_cache, block_tables, lengths)
    out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(shape)
    lse = q.new_empty(shape[:-1], dtype=torch.float32) if return_lse else None
    if batch:
        qs, ks, vs = q.stride(), k_cache.stride(), v_cache.stride()
        token_stride = qs[1] if len(shape) == 4 else 0
        if qs[-1] != 1 or (qs[0] | token_stride | qs[-2]) & 1 or q.data_ptr() & 3:
            q = q.clone(memory_format=torch.contiguous_format)
            qs = q.stride()
            token_stride = qs[1] if len(shape) == 4 else 0
        if ks[3] != 1 or vs[3] != 1:
            raise ValueError("a cache's head dimension must be contiguous")
        if block_tables.stride(1) != 1:
            block_tables = block_tables.contiguous()
        lengths = lengths.contiguous()
        nbytes = _workspace_bytes(new, q_heads, kv_heads, dim)
        workspace = q.new_empty(nbytes, dtype=torch.uint8)
        _call(_lib.lib().fpv2_decode_attention, device, _pack_decode(
            q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), _lib.dtype_code(dtype), batch, new, q_heads,
            kv_heads, dim, qs[0], token_stride, qs[-2], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
            block_tables.data_ptr(), block_tables.stride(0), width, lengths.data_ptr(), pages, page_size,
            window, sinks, scale, out.data_ptr(), _address(lse), workspace.data_ptr(), nbytes))
    return (out, lse) if return_lse else out


def _setting(value, name: str, dtype: torch.dtype, rows: int, plain: float):
    """(tensor, scalar) of a per-row or common setting."""
    if isinstance(value, torch.Tensor):
        if value.shape != (rows,) or value.dtype != dtype:
            raise ValueError(f"{name} must be a number or a {dtype} tensor [rows]")
        return value.contiguous(), plain
    return None, value


def sample_tokens(
    logits: torch.Tensor,
    noise: torch.Tensor,
    *,
    temperature: float | torch.Tensor = 1.0,
    top_k: int | torch.Tensor = 0,
    top_p: float | torch.Tensor = 1.0,
    min_p: float | torch.Tensor = 0.0,
    return_logprobs: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """The next token of each row of ``logits`` ``[rows, vocab]`` from given random numbers.

    ``noise`` is float32 ``[rows, vocab]`` of positive, exponentially distributed
    numbers (``torch.empty(...).exponential_()``). Each setting is one number or a
    tensor ``[rows]`` (float32; int32 for ``top_k``). With ``z = (x - max) / T`` and
    ``w = exp(z)``, tokens in the order of (x descending, index ascending) pass
    ``top_k`` (the first k; 0 or less: all), then ``top_p`` (the shortest prefix of
    those whose weight reaches ``top_p`` of theirs; 1 or more: all), then ``min_p``
    (``w >= min_p``); the first token always stays. The result, int64 ``[rows]``, is the
    argmax of ``z - log(noise)`` over what is left: a draw with probabilities
    proportional to ``w``. ``T <= 0`` takes the lowest index of the maximum; an infinite
    ``T`` counts as float32's largest number. NaN logits count as -inf; a row without a
    logit above -inf gives -1. With ``return_logprobs`` also float32 ``[rows]``: the
    token's log-probability under ``softmax(x / T)`` over the whole row (``T = 1`` where
    ``T <= 0``).
    """
    if logits.ndim != 2 or logits.shape != noise.shape:
        raise ValueError("logits and noise must have the same shape [rows, vocab]")
    rows, vocab = logits.shape
    if not vocab:
        raise ValueError("logits must have a vocabulary")
    code = _lib.dtype_code(logits.dtype)
    if noise.dtype != torch.float32:
        raise ValueError("noise must have float32 dtype")
    heat, heat_all = _setting(temperature, "temperature", torch.float32, rows, 1.0)
    k, k_all = _setting(top_k, "top_k", torch.int32, rows, 0)
    p, p_all = _setting(top_p, "top_p", torch.float32, rows, 1.0)
    least, least_all = _setting(min_p, "min_p", torch.float32, rows, 0.0)
    if not -_INT32_MAX <= k_all <= _INT32_MAX:
        raise ValueError("top_k must be a 32-bit integer")
    if torch.is_grad_enabled() and (logits.requires_grad or heat is not None and heat.requires_grad):
        _refuse_grad("sample_tokens")
    _refuse_tangents("sample_tokens", logits, heat)
    device = logits.get_device()
    if device < 0 or noise.get_device() != device or heat is not None and heat.get_device() != device \
            or k is not None and k.get_device() != device or p is not None and p.get_device() != device \
            or least is not None and least.get_device() != device:
        _lib.require_cuda(logits, noise, heat, k, p, least)
    logits, noise = _rows(logits), _rows(noise)
    tokens = logits.new_empty(rows, dtype=torch.int64)
    logprobs = logits.new_empty(rows, dtype=torch.float32) if return_logprobs else None
    _call(_lib.lib().fpv2_sample_tokens, device, _pack_sample(
        logits.data_ptr(), code, rows, vocab, logits.stride(0), noise.data_ptr(), noise.stride(0),
        _address(heat), heat_all, _address(k), int(k_all), _address(p), p_all, _address(least), least_all,
        tokens.data_ptr(), _address(logprobs)))
    return (tokens, logprobs) if return_logprobs else tokens
