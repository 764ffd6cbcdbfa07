"""KV-cache in-place update: the reference's planned ``stackkernels.torch.cache``
API (``docs/user_guide/dropout_cache_sampling.md:66-72``; the reference module
``src/stackkernels/torch/cache.py`` is still a stub).

ROCm device tensors run the HIP kernel; CPU tensors and ``backend='reference'``
run the same update with torch indexing.
"""

from __future__ import annotations

import torch

from stackkernels_amd._core.cache.kv_update import kv_cache_update as _core_kv_cache_update
from stackkernels_amd._core.cache.kv_update import validate_cache_update
from stackkernels_amd._core.cache.quantized import (
    _integer,
    layout_of,
    table_operand,
    validate_page_plan,
    validate_q8_update,
)
from stackkernels_amd._core.cache.quantized import kv_cache_update_q8 as _core_kv_cache_update_q8
from stackkernels_amd._core.cache.quantized import kv_page_plan as _core_kv_page_plan
from stackkernels_amd._reference.torch import quantized
from stackkernels_amd.torch._dispatch import should_use_hip


def kv_cache_update(
    k: torch.Tensor,
    v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    slot_indices: torch.Tensor,
    paged: bool = False,
    *,
    rope_cos: torch.Tensor | None = None,
    rope_sin: torch.Tensor | None = None,
    start_pos: int | torch.Tensor = 0,
) -> None:
    """Insert new key/value rows into the caches in place.

    ``k_cache[b, h, slot_indices[b, t], :] = k[b, h, t, :]`` (and for v) for every
    batch row b, KV head h and new token t.

    Args:
        k, v: (B, H_kv, T, D) new keys and values.
        k_cache, v_cache: (B, H_kv, S_cache, D) caches (any b/h/s strides, contiguous D),
            updated in place.
        slot_indices: integer (B, T) cache positions.  A position outside
            ``[0, S_cache)`` skips its token (pad ragged batches with -1).  Positions
            must be distinct within a batch row (within the pool when paged).
        paged: the caches are page pools (num_pages, H_kv, page_size, D) shared by
            all rows, and a position s is row ``s % page_size`` of page
            ``s // page_size`` (S_cache = num_pages * page_size).
        rope_cos, rope_sin: optional (max_seq_len, D) RoPE tables: the new keys are
            rotated (the reference's ``apply_rope`` on k) as they are written, new
            token t of row b at position ``start_pos + t``; values are copied as
            they are.
        start_pos: int, or integer (B,) tensor of per-row positions of token 0.
    """
    rope = rope_cos is not None or rope_sin is not None
    if should_use_hip(k_cache):
        extra = dict(rope_cos=rope_cos, rope_sin=rope_sin, start_pos=start_pos) if rope else {}
        _core_kv_cache_update(k, v, k_cache, v_cache, slot_indices, paged, **extra)
        return
    b, _, t, s, _ = validate_cache_update(k, v, k_cache, v_cache, slot_indices, paged)
    if rope:
        from stackkernels_amd.torch.attention import _rope_reference

        k = _rope_reference(k, rope_cos, rope_sin, start_pos)
    slots = slot_indices.to("cpu", torch.int64)
    if paged:
        ps = k_cache.shape[2]
        for i in range(b):
            for j in range(t):
                pos = int(slots[i, j])
                if 0 <= pos < s:
                    k_cache[pos // ps, :, pos % ps] = k[i, :, j].to(k_cache.dtype)
                    v_cache[pos // ps, :, pos % ps] = v[i, :, j].to(v_cache.dtype)
        return
    for i in range(b):
        pos = slots[i]
        keep = (pos >= 0) & (pos < s)
        if bool(keep.any()):
            idx = pos[keep].to(k_cache.device)
            sel = keep.nonzero().flatten().to(k.device)
            k_cache[i][:, idx] = k[i][:, sel].to(k_cache.dtype)
            v_cache[i][:, idx] = v[i][:, sel].to(v_cache.dtype)


def kv_cache_update_q8(
    k: torch.Tensor,
    v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    cache_seqlens: torch.Tensor,
    new_lens: torch.Tensor | None = None,
    block_table: torch.Tensor | None = None,
    *,
    block_size: int = 32,
    rope_cos: torch.Tensor | None = None,
    rope_sin: torch.Tensor | None = None,
    start_pos: int | torch.Tensor = 0,
) -> None:
    """Append new keys and values to a cache held in 8 bits, in place.

    The cache holds codes, ``int8`` or ``float8_e4m3fn``, and one float32 scale for
    each block of ``block_size`` tokens and KV head; an element's value is its code
    times its block's scale.  New token t of row b becomes token
    ``cache_seqlens[b] + t``.  A block takes the scale its new values need (int8:
    largest magnitude / 127; e4m3: the smallest power of two that brings it to 448
    or less), or keeps its own where it already holds tokens of the row and its own
    is larger; where the scale grows, the older codes of the block are rounded to
    it.  In e4m3 that keeps older values exactly, down to the subnormal range; in
    int8 it costs at most half a step of the new scale each time.  Rounding is to
    nearest, ties to even.  Infinities and NaN do not count for the scale; they
    saturate, and NaN becomes 0 in int8.

    Args:
        k, v: (B, H_kv, T, D) new keys and values; D a multiple of 16 up to 256.
        k_cache, v_cache: codes, (B, H_kv, S_cache, D) or page pools (num_pages,
            H_kv, page_size, D); 16-byte-aligned rows, contiguous D.
        k_scale, v_scale: float32 (B, H_kv, ceil(S_cache / block_size)) or
            (num_pages, H_kv, page_size / block_size).
        cache_seqlens: integer (B,) tokens each row holds before the call.
        new_lens: optional integer (B,): row b has ``new_lens[b]`` of the T tokens
            (the first ones); the others are not written.
        block_table: integer (B, max_pages) for a paged cache: token n of row b lies
            in page ``block_table[b, n // page_size]``.  Tokens past the row's
            capacity or in a page outside the pool are skipped.  Two rows must not
            write the same block.
        block_size: tokens per scale, a multiple of 32 that divides page_size.
        rope_cos, rope_sin, start_pos: rotate the new keys, token t of row b at
            position ``start_pos + t`` (typically ``start_pos=cache_seqlens``), in
            float32 before they are rounded to codes.
    """
    rope = rope_cos is not None or rope_sin is not None
    if should_use_hip(k_cache):
        _core_kv_cache_update_q8(k, v, k_cache, v_cache, k_scale, v_scale, cache_seqlens, new_lens,
                                 block_table, block_size, rope_cos, rope_sin, start_pos)
        return
    b, _, t, _, _, _ = validate_q8_update(
        *(layout_of(x) for x in (k, v, k_cache, v_cache, k_scale, v_scale)),
        block_table is not None, block_size)
    lens = _integer(cache_seqlens, "cache_seqlens", (b,)).tolist()
    news = [t] * b if new_lens is None else _integer(new_lens, "new_lens", (b,)).tolist()
    table = None if block_table is None else table_operand(block_table, b).tolist()
    with torch.no_grad():
        if rope:
            from stackkernels_amd.torch.attention import _rope_reference

            k = _rope_reference(k.float(), rope_cos, rope_sin, start_pos)
        quantized.append(k, v, k_cache, v_cache, k_scale, v_scale, lens, news, table, block_size)


def kv_page_plan(
    block_table: torch.Tensor,
    cache_seqlens: torch.Tensor,
    new_lens: torch.Tensor,
    free_pages: torch.Tensor,
    free_state: torch.Tensor,
    page_size: int,
    *,
    max_new: int = 1,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Block tables and slot maps of a serving step, built on the device.

    Row b holds ``cache_seqlens[b]`` tokens in the pages ``block_table[b, 0 ..
    ceil(cache_seqlens[b] / page_size))``.  A positive ``new_lens[b]`` is the number
    of tokens it gains in this step (at most ``max_new``), a negative one the number
    of its last tokens that it gives up (rejected drafts; all of them when the
    request is done).  Nothing is copied to the host, so the plan, the append and
    the attention of a step can be captured into one graph.

    Rows that grow take pages from the front of the ring ``free_pages`` in row order.
    A row that does not fit its table, or whose pages, summed over it and the rows
    before it, are more than the ring holds, does not grow at all: its length stays
    and its slots are -1.  Rows that shrink put the pages they no longer need behind
    the ring's end, for the next call.

    Args:
        block_table: int32 (B, max_pages), changed in place: pages are stored behind
            those a row holds, entries past a row's pages are not cleared.
        cache_seqlens, new_lens: integer (B,).
        free_pages: int32 (N,) ring of free page ids, changed in place; N at least
            the number of pages there are.
        free_state: integer (2,): place of the ring's first id, how many there are.
        page_size: tokens per page.
        max_new: width of the slot map.

    Returns:
        ``slot_indices`` int64 (B, max_new), for ``kv_cache_update(..., paged=True)``:
        the slot of each new token, -1 past a row's own; the new ``cache_seqlens``
        int32 (B,) and ``free_state`` int32 (2,).  The inputs of these names are left
        as they are: a call with the same inputs gives the same results again.
    """
    if should_use_hip(block_table):
        return _core_kv_page_plan(block_table, cache_seqlens, new_lens, free_pages, free_state,
                                  page_size, max_new)
    b, _ = validate_page_plan(block_table, cache_seqlens, new_lens, free_pages, free_state,
                              page_size, max_new)
    table, ring = block_table.tolist(), free_pages.tolist()
    slots, lens, state = quantized.page_plan(
        table, _integer(cache_seqlens, "cache_seqlens", (b,)).tolist(),
        _integer(new_lens, "new_lens", (b,)).tolist(), ring,
        _integer(free_state, "free_state", (2,)).tolist(), page_size, max_new)
    dev = block_table.device
    if b:
        block_table.copy_(torch.tensor(table, dtype=torch.int32).view_as(block_table))
    free_pages.copy_(torch.tensor(ring, dtype=torch.int32))
    return (torch.tensor(slots, dtype=torch.int64, device=dev).view(b, max_new),
            torch.tensor(lens, dtype=torch.int32, device=dev),
            torch.tensor(state, dtype=torch.int32, device=dev))


__all__ = ["kv_cache_update", "kv_cache_update_q8", "kv_page_plan"]
