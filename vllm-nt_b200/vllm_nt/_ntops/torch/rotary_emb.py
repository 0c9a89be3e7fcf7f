"""In-place rotary embedding on the sm_100a kernels (replaces
vllm_nt/_ntops/torch/rotary_emb.py and the cos/sin gather of
vllm_nt/_ntops/oot_support.py:164-204): NeoX heads with a table of their own dtype as vLLM
rounds them, the interleaved layout and fp32 tables with one rounding, and the table itself."""

from __future__ import annotations

import math

import torch

from vllm_nt._ntops import capi
from vllm_nt._ntops.torch._ext import ops, overload

_SCALINGS = {None: capi.ROPE_NONE, "none": capi.ROPE_NONE, "linear": capi.ROPE_LINEAR, "ntk": capi.ROPE_NTK,
             "yarn": capi.ROPE_YARN}


def _heads(t: torch.Tensor, num_tokens: int, head_size: int) -> torch.Tensor:
    v = t.view(num_tokens, -1, head_size)
    if v.stride(-1) != 1:
        raise ValueError("rotary_embedding needs unit stride in the head dimension")
    return v


def rotary_embedding(
    positions: torch.Tensor,
    query: torch.Tensor,
    key: torch.Tensor | None,
    head_size: int,
    cos_sin_cache: torch.Tensor,
    rotary_dim: int | None = None,
    interleaved: bool = False,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Rotates the first ``rotary_dim`` dims of every head of query (and key) in place, with
    cos/sin = cos_sin_cache[positions] split in halves.  Pairs are (i, i + rotary_dim / 2)
    (NeoX), or (2i, 2i + 1) with ``interleaved``.  NeoX pairs and a cache of query's dtype
    (vLLM's _match_cos_sin_cache_dtype) are rounded as vLLM's torch path rounds them; an fp32
    cache of 16-bit heads, and interleaved pairs, are rotated in fp32 and rounded once.  Heads
    that are a column slice (the rotary part at a head's end) are passed as the 3-D slice."""
    rot = cos_sin_cache.shape[-1] if rotary_dim is None else rotary_dim
    if interleaved or cos_sin_cache.dtype != query.dtype:
        _rotary_either_layout(positions, query, key, head_size, cos_sin_cache, rot, interleaved)
        return query, key
    if (positions.is_contiguous() and cos_sin_cache.is_contiguous() and query.dim() == 2
            and query.stride(-1) == 1 and (key is None or (key.dim() == 2 and key.stride(-1) == 1))):
        # vLLM's [tokens, heads * head_size] slices of the qkv projection go straight in
        ops().rotary_embedding_neox(positions, query, key, cos_sin_cache, head_size, rot)
        return query, key
    positions = positions.reshape(-1)
    if not positions.is_contiguous():
        positions = positions.contiguous()
    n = positions.shape[0]
    cache = cos_sin_cache if cos_sin_cache.stride(-1) == 1 else cos_sin_cache.contiguous()
    q = _heads(query, n, head_size)
    k = _heads(key, n, head_size) if key is not None else None
    ops().rotary_embedding_neox(positions, q, k, cache, int(head_size), int(rot))
    return query, key


def _token_rows(shape, n, head_size):
    """[tokens, heads * head_size] or [tokens, heads, head_size]: rows that go to the kernel as they are."""
    return (len(shape) == 2 or (len(shape) == 3 and shape[2] == head_size)) and shape[0] == n


def _rotary_either_layout(positions, query, key, head_size, cos_sin_cache, rot, interleaved):
    if not positions.is_contiguous():
        positions = positions.contiguous()
    if not cos_sin_cache.is_contiguous() and cos_sin_cache.stride(-1) != 1:
        cos_sin_cache = cos_sin_cache.contiguous()
    n = positions.numel()
    if not _token_rows(query.shape, n, head_size):
        query = _heads(query, n, head_size)
    if key is not None and not _token_rows(key.shape, n, head_size):
        key = _heads(key, n, head_size)
    overload("rotary_embedding")(positions, query, key, cos_sin_cache, head_size, rot, interleaved)


def rope_cos_sin_cache(
    num_positions: int,
    rotary_dim: int,
    base: float = 10000.0,
    *,
    scaling: str | None = None,
    factor: float = 1.0,
    original_max_position: int | None = None,
    beta_fast: float = 32.0,
    beta_slow: float = 1.0,
    magnitude: float | None = None,
    freq_divisors: torch.Tensor | None = None,
    first_position: int = 0,
    dtype: torch.dtype = torch.float32,
    device: torch.device | str | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """The [num_positions, rotary_dim] table cat(cos, sin) of position * frequency that the
    rotary kernels read, angles formed in 64 bits.  ``scaling`` stretches the frequencies
    base^(-2i/d) to contexts ``factor`` times as long: ``"linear"`` divides them by factor,
    ``"ntk"`` raises base to base * factor^(d/(d-2)), ``"yarn"`` divides those that turn less
    than ``beta_slow`` times over ``original_max_position`` positions, keeps those that turn more
    than ``beta_fast`` times and blends between.  ``freq_divisors`` (float32 [d/2]) divide the
    frequencies one by one (a divisor of 0 or NaN leaves NaN in its columns).  cos and sin are
    multiplied by ``magnitude`` (None: 0.1 ln(factor) + 1 for yarn with factor > 1, else 1).  ``out`` may be given instead of dtype and device."""
    if scaling not in _SCALINGS:
        raise ValueError(f"rope_cos_sin_cache: unknown scaling {scaling!r}")
    if scaling == "yarn" and original_max_position is None:
        raise ValueError("rope_cos_sin_cache: yarn needs original_max_position")
    if magnitude is None:
        magnitude = 0.1 * math.log(factor) + 1.0 if scaling == "yarn" and factor > 1.0 else 1.0
    if out is None:
        out = torch.empty(num_positions, rotary_dim, dtype=dtype, device="cuda" if device is None else device)
    elif out.dim() != 2 or out.shape[0] != num_positions:
        raise ValueError("rope_cos_sin_cache: out must be [num_positions, >= rotary_dim]")
    overload("rope_cos_sin_cache")(out, first_position, rotary_dim, base, _SCALINGS[scaling], factor,
                                   original_max_position or 0, beta_fast, beta_slow, magnitude, freq_divisors)
    return out


def rotary_embedding_and_cache(
    positions: torch.Tensor,
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    head_size: int,
    cos_sin_cache: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    slot_mapping: torch.Tensor,
    rotary_dim: int | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """rotary_embedding(positions, query, key, ...) followed by
    store_kvcache(key, value, key_cache, value_cache, slot_mapping) in one kernel: q/k are
    rotated in place and the rotated key rows and the value rows land in the paged caches
    [blocks, block_size, kv_heads, head_size].  Bit-identical to the two calls in sequence.
    Tokens past ``slot_mapping.numel()`` (vLLM's padded rows) are rotated only."""
    rot = cos_sin_cache.shape[-1] if rotary_dim is None else rotary_dim
    positions = positions.reshape(-1)
    if not positions.is_contiguous():
        positions = positions.contiguous()
    slots = slot_mapping.reshape(-1)
    if not slots.is_contiguous():
        slots = slots.contiguous()
    cache = cos_sin_cache if cos_sin_cache.stride(-1) == 1 else cos_sin_cache.contiguous()
    n = positions.shape[0]
    q = query if query.dim() == 2 and query.stride(-1) == 1 else _heads(query, n, head_size)
    k = key if key.dim() == 2 and key.stride(-1) == 1 else _heads(key, n, head_size)
    v = value if value.dim() == 2 and value.stride(-1) == 1 else _heads(value, n, head_size)
    ops().rope_and_cache(positions, q, k, v, cache, key_cache, value_cache, slots, int(head_size), int(rot))
    return query, key


def apply_rotary_emb(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """Reference signature (vllm_nt/_ntops/torch/rotary_emb.py:7-9): x [T, H, R] rotated in
    place with per-token cos/sin [T, 1, R/2] (or [T, R/2]).  Implemented by handing the
    kernel a per-token cos|sin table and positions 0..T-1."""
    t, _, r = x.shape
    table = torch.cat((cos.reshape(t, r // 2), sin.reshape(t, r // 2)), dim=-1).to(x.dtype)
    pos = torch.arange(t, device=x.device, dtype=torch.int64)
    if x.stride(-1) != 1:
        raise ValueError("apply_rotary_emb needs unit stride in the last dimension")
    ops().rotary_embedding_neox(pos, x, None, table.contiguous(), r, r)
    return x
