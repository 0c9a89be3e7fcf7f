"""Latent attention on sm_100a: every head's keys and values come from one latent vector a token
(plus one shared rotary key), which is all that is cached.  The paged cache is
[blocks, block_size, 576]: the normalised latent (512), then the rotated key (64)."""

from __future__ import annotations

import torch

from vllm_nt._ntops.torch._ext import ops, overload


def _flat(t: torch.Tensor) -> torch.Tensor:
    if t.dim() != 1:
        t = t.reshape(-1)
    return t if t.is_contiguous() else t.contiguous()


def _int32(t: torch.Tensor) -> torch.Tensor:
    if t.dtype != torch.int32:
        t = t.to(torch.int32)
    return t if t.is_contiguous() else t.contiguous()


def latent_rope_and_cache(
    positions: torch.Tensor,
    query: torch.Tensor | None,
    latent: torch.Tensor,
    key: torch.Tensor,
    cos_sin_cache: torch.Tensor,
    kv_cache: torch.Tensor,
    slot_mapping: torch.Tensor,
    *,
    norm_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    latent_out: torch.Tensor | None = None,
    interleaved: bool = True,
) -> None:
    """One layer's rows into the latent cache in one kernel: ``latent`` [T, 512] is RMS-normalised
    with ``norm_weight`` (unchanged if None), ``key`` [T, 64] and ``query`` [T, heads, 64] (the
    rotary columns of the query heads, or None) are rotated in place, and
    kv_cache[slot_mapping[t]] = [latent | key].  ``latent_out`` [T, 512] (it may be ``latent``)
    receives the normalised rows.  Tokens past ``slot_mapping.numel()`` and those with a negative
    slot (vLLM's padded rows) are not stored."""
    overload("latent_rope_and_cache")(_flat(positions), query, latent, key, norm_weight, eps, cos_sin_cache, interleaved,
                                      kv_cache, latent_out, _flat(slot_mapping))


def latent_workspace_bytes() -> int:
    """Bytes of latent_attention's workspace on the current device (one size for every call)."""
    return int(ops().latent_attention_workspace_size())


def latent_attention(
    out: torch.Tensor,
    q_latent: torch.Tensor,
    q_rope: torch.Tensor,
    kv_cache: torch.Tensor,
    seq_lens: torch.Tensor,
    block_table: torch.Tensor,
    scale: float,
    *,
    query_start_loc: torch.Tensor | None = None,
    max_query_len: int | None = None,
    max_seq_len: int | None = None,
    lse: torch.Tensor | None = None,
    workspace: torch.Tensor | None = None,
) -> torch.Tensor:
    """out[t, h] = softmax(scale * (q_latent[t, h] . latent_j + q_rope[t, h] . key_j)) latent_j
    over the cached rows j of t's sequence up to t's own position (absorbed form: q_latent is
    the head's query taken through the key up-projection, and out goes through the value one).

    q_latent/out [T, heads, 512], q_rope [T, heads, 64]; sequence b's queries are rows
    query_start_loc[b] .. [b + 1], the last of its seq_lens[b] cached tokens; without
    ``query_start_loc`` every sequence has T / len(seq_lens) of them (1: a decode batch).
    ``max_query_len`` bounds the query counts (None: T) and is worth giving: query rows are grouped
    for it, and 96 decodes of 16 heads take a tenth longer without it; sequences with more queries are
    skipped and reported.  ``max_seq_len`` bounds the lengths (None: the block table's capacity) and
    only sizes the launch.  ``lse`` float32 [T, heads] receives the natural log of the
    softmax sums.  ``workspace`` may be passed to avoid an allocation per call."""
    if query_start_loc is not None:
        query_start_loc = _int32(query_start_loc)
    if block_table.dtype != torch.int32:
        block_table = block_table.to(torch.int32)
    overload("latent_attention")(out, lse, q_latent, q_rope, kv_cache, query_start_loc, _int32(seq_lens), block_table,
                                 q_latent.shape[0] if max_query_len is None else max_query_len, max_seq_len or 0, scale,
                                 workspace)
    return out


def latent_attention_prefill(
    out: torch.Tensor,
    query: torch.Tensor,
    k_nope: torch.Tensor,
    k_rope: torch.Tensor,
    value: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    cu_seqlens_k: torch.Tensor,
    max_query_len: int,
    scale: float,
    causal: bool = True,
    lse: torch.Tensor | None = None,
) -> torch.Tensor:
    """Varlen attention over keys and values expanded from the latent: query [Tq, heads, 192],
    k_nope and value [Tk, heads, 128] (slices of the up-projection's rows go in as they are),
    k_rope [Tk, 64] shared by the heads, out [Tq, heads, 128]; sequence b's queries and keys at
    rows cu_seqlens_q[b] .. [b + 1] and cu_seqlens_k[b] .. [b + 1], causal masking aligned to the
    end of its keys.  ``lse`` float32 [Tq, heads] receives the natural log of the softmax sums,
    with which two parts of a context can be merged."""
    overload("latent_attention_prefill")(out, lse, query, k_nope, k_rope, value, _int32(cu_seqlens_q),
                                         _int32(cu_seqlens_k), max_query_len, scale, causal)
    return out
