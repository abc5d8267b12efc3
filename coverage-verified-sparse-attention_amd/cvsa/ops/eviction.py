"""Eviction from the paged cache by accumulated attention weight.

:func:`add_key_weights` keeps account of how much attention each cached key
has received; :func:`evict_tokens` cuts every sequence to the tokens with the
most of it, in place, each KV head by itself.  Both take caches of bf16 and of
8 bits (:func:`cvsa.ops.append_chunk_kv`).  After a cut a key's place in the
cache is no longer its position: new keys and queries are rotated by
:func:`cvsa.ops.qk_norm_rope` with positions that the caller counts, and
appended without a rotation.

Neither has a counterpart in the reference, whose cache keeps every token.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _i32, _block_tables, _check_seqs, _lib, _ptr
from .chunk import (_BF16, ChunkLayout, _call, _check_caches, _rows, _same_device,
                    _tables)


def _check_weights(who: str, weights: torch.Tensor, B: int, H_kv: int, keys: int) -> int:
    """Their capacity of keys."""
    if weights.dim() != 3 or weights.shape[0] != B or weights.shape[1] != H_kv \
            or weights.shape[2] < keys or weights.dtype is not torch.float32 \
            or not weights.is_contiguous():
        raise ValueError(f"{who}: weights must be contiguous float32 [{B}, {H_kv}, >= {keys}] (all "
                         f"keys of the block tables), got {tuple(weights.shape)} {weights.dtype}")
    return weights.shape[2]


def add_key_weights(weights: torch.Tensor, q: torch.Tensor, lse: torch.Tensor,
                    k_cache: torch.Tensor, block_tables: torch.Tensor,
                    context_lens: torch.Tensor, layout: ChunkLayout, num_kv_heads: int,
                    num_q_per_kv: int, block_size: int, causal: bool = True,
                    scale: Optional[float] = None, window: int = 0,
                    k_scales: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Add the attention weight that a chunk's queries give to each key.

    ``weights`` [B, H_kv, S] fp32, S at least the keys of a block table's row,
    is updated in place and returned: of the key in slot j of sequence b and
    KV head h it becomes (0 where the chunk itself brought the key, else what
    it was) + the sum of exp(scale q . k - lse) over the chunk's tokens of b
    and the query heads of h that see the key.  q, block tables, context
    lengths, layout, causal and scale as :func:`cvsa.ops.chunk_attention` has
    them, and ``lse`` ([T, H_q] fp32) what it returned; rows with -inf give
    nothing.  ``window``: only the last tokens of each sequence's chunk count
    (0: all).  Entries past a context, and of sequences without tokens in the
    chunk, are left as they are; keys of blocks outside the pool get nothing.
    So a chunk for which this is not called leaves its keys what their slots
    held, and the caller sets those to 0.
    Sums are of 32 bits, in an order that does not vary.
    """
    who = "add_key_weights"
    dev = _same_device(q, lse, k_cache, block_tables, context_lens, weights, k_scales)
    num_blocks, H_kv, D = _check_caches(who, k_cache, k_cache, block_size, k_scales, k_scales)
    if H_kv != num_kv_heads:
        raise ValueError(f"{who}: head counts do not match the cache")
    bt, bt_stride, ctx = _tables(who, layout, dev, block_tables, context_lens)
    B, W = bt.shape
    if bt_stride < W:  # a row that sequences share
        bt, bt_stride = bt.contiguous(), W
    S = _check_weights(who, weights, B, H_kv, W * block_size)
    T, H_q, G = layout.total, num_kv_heads * num_q_per_kv, num_q_per_kv
    q, *q_at = _rows(who, "q", q, T, H_q, D, _BF16)
    # The kernel counts in 32 bits from the first of up to 128 rows to the others.
    if (126 + G) // G * q_at[1] + (G - 1) * q_at[2] >= 1 << 31:
        q = q[:T].contiguous()
        q_at = [q.data_ptr(), H_q * D, D]
    if lse.dim() != 2 or lse.shape[0] < T or lse.shape[1] != H_q or lse.dtype is not torch.float32:
        raise ValueError(f"{who}: lse must be [{T}, {H_q}] float32, got {tuple(lse.shape)} "
                         f"{lse.dtype}")
    lse = lse.contiguous()
    window = int(window)
    if window < 0:
        raise ValueError(f"{who}: window must not be negative")
    scale = D ** -0.5 if scale is None else float(scale)
    if T:
        L = _lib.load()
        # Allocated for the call, so no two calls, streams or captured graphs
        # share it.
        key = ("add_key_weights", H_q, H_kv, D, S, window)
        need = layout._workspace_bytes.get(key)
        if need is None:
            need = L.cvsa_add_key_weights_workspace_bytes(layout.cu_host, B, *key[1:])
            layout._workspace_bytes[key] = need
        ws = torch.empty(need, device=dev, dtype=torch.uint8) if need else None
        _call(dev, who, L.cvsa_add_key_weights, weights.data_ptr(), S, *q_at, lse.data_ptr(),
              k_cache.data_ptr(), _ptr(k_scales), num_blocks, bt.data_ptr(), bt_stride,
              ctx.data_ptr(), layout.cu_seqlens.data_ptr(), layout.cu_host, B, H_q, H_kv, D,
              block_size, W, scale, int(bool(causal)), window, _ptr(ws), need)
    return weights


def evict_tokens(weights: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 block_tables: torch.Tensor, context_lens: torch.Tensor, keep: int,
                 block_size: int, sinks: int = 0, recent: int = 0,
                 k_scales: Optional[torch.Tensor] = None,
                 v_scales: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Cut every sequence of more than ``keep`` tokens to ``keep``.

    For each KV head by itself the first ``sinks`` tokens stay, the last
    ``recent`` and, of those between, the ones of the largest ``weights``
    ([B, H_kv, S] fp32, see :func:`add_key_weights`); ties go to the lowest
    slot, NaN counts as the largest.  The fewest rows move: a slot below keep
    - recent whose token stays is not touched, the others of them get the kept
    tokens from slot keep - recent on, in order, and the last ``recent`` tokens
    go to the end, in order.  Keys, values and weights move together; what is
    behind slot ``keep`` is left as it is.

    The caches are changed in place, the tables are not: the caller takes
    context_lens.clamp(max=keep) as the new lengths, once for all layers.
    What was learned of pages before no longer holds: ``reset()`` a CVSABackend
    (its selections, Quest's extremes), ``invalidate()`` a QuestPageMeta.
    Pages must belong to one sequence alone, and keys and values have caches
    (and scales) of their own.  In caches of 8 bits a page that tokens come to
    gets the largest scale of its tokens' pages, to which they are brought
    (exact but for values that become subnormal).

    Returns [B, H_kv, keep] int32, the old slot of each new one (-1 past a
    shorter context).
    """
    who = "evict_tokens"
    dev = _same_device(weights, k_cache, v_cache, block_tables, context_lens, k_scales, v_scales)
    num_blocks, H_kv, D = _check_caches(who, k_cache, v_cache, block_size, k_scales, v_scales)
    _check_seqs(who, weights.shape[0], block_tables, context_lens)
    bt, ctx = _block_tables(block_tables), _i32(context_lens)
    B, W = bt.shape
    S = _check_weights(who, weights, B, H_kv, W * block_size)
    keep, sinks, recent = int(keep), int(sinks), int(recent)
    if sinks < 0 or recent < 0 or keep < 1 or sinks + recent > keep:
        raise ValueError(f"{who}: {sinks} first and {recent} last tokens of {keep} kept")
    kept = torch.empty(B, H_kv, keep, device=dev, dtype=torch.int32)
    L = _lib.load()
    need = L.cvsa_evict_tokens_workspace_bytes(B, H_kv, D, block_size, W,
                                               16 if k_scales is None else 8, keep, sinks, recent)
    ws = torch.empty(need, device=dev, dtype=torch.uint8) if need else None
    _call(dev, who, L.cvsa_evict_tokens, weights.data_ptr(), S, k_cache.data_ptr(),
          v_cache.data_ptr(), _ptr(k_scales), _ptr(v_scales), num_blocks, bt.data_ptr(),
          bt.stride(0) if B > 1 else W, W, ctx.data_ptr(), B, H_kv, D, block_size, keep, sinks,
          recent, kept.data_ptr(), _ptr(ws), need)
    return kept
