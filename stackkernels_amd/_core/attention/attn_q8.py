"""Launcher of attention over a cache held in 8-bit codes (``sk_attn_q8``): one or
more query tokens per row, contiguous or paged, per-row key and query counts."""

from __future__ import annotations

import ctypes
import functools
import math

import torch

from stackkernels_amd._core.attention import _lib
from stackkernels_amd._core.attention._common import _SUPPORTED, kernel_operand
from stackkernels_amd._core.cache.quantized import (
    check_cache_strides,
    check_q8_devices,
    int32_operand,
    layout_of,
    rope_tail,
    table_operand,
    validate_q8_cache,
)


@functools.lru_cache(maxsize=512)
def plan_q8(code: int, b: int, hq: int, hkv: int, sq: int, sk: int, d: int,
            is_causal: bool) -> tuple[int, int]:
    """(split count, workspace bytes) the library takes for a shape."""
    ns, nb = ctypes.c_int(0), ctypes.c_size_t(0)
    _lib.check(_lib.load().sk_attn_q8_plan(code, b, hq, hkv, sq, sk, d, int(is_causal),
                                           ctypes.byref(ns), ctypes.byref(nb)),
               "flash_attention_q8 plan")
    return ns.value, nb.value


def validate_q8_attention(q, k, v, ks, vs, width: int | None, block_size: int) -> tuple:
    """(units, KV heads, tokens per unit, keys a row can have), each tensor given as
    ``layout_of``; ``width``: the block table's, None for a contiguous cache."""
    if len(q[0]) != 4:
        raise ValueError(f"Expected 4D q (B, H, S, D), got {len(q[0])}D")
    b, hq, _, d = q[0]
    units, hkv, rows = validate_q8_cache(k, v, ks, vs, b, d, width is not None, block_size)
    if hkv == 0 or hq % hkv != 0:
        raise ValueError(f"Query heads ({hq}) must be divisible by KV heads ({hkv}) for GQA/MQA")
    return units, hkv, rows, rows if width is None else width * rows


def table_width(q, cache_seqlens, block_table) -> int | None:
    if block_table is None:
        return None
    if cache_seqlens is None:
        raise ValueError("a paged cache (block_table) needs cache_seqlens")
    return table_operand(block_table, q.shape[0]).shape[1]


@functools.lru_cache(maxsize=512)
def _attention_shape(q, k, v, ks, vs, width, block_size: int, is_causal: bool):
    units, hkv, rows, sk = validate_q8_attention(q, k, v, ks, vs, width, block_size)
    if q[2] not in _SUPPORTED:
        raise NotImplementedError(f"dtype {q[2]} has no HIP kernel (supported: {_SUPPORTED})")
    check_cache_strides(k, v)
    b, hq, sq, d = q[0]
    st, unit = q[1], 3 if q[2] == torch.float32 else 7
    as_is = st[3] == 1 and not (st[0] | st[1] | st[2]) & unit
    code = _lib.dtype_code(q[2])
    out = (hq * sq * d, sq * d, d)
    shape = _lib.q8_shape(
        (code, _lib.code_type(k[2]), b, hq, hkv, sq, units, rows, width or 0, block_size, d,
         int(is_causal)),
        (st[:3], out, k[1][:3], v[1][:3], ks[1], vs[1]))
    return shape, as_is, (code, b, hq, hkv, sq, sk, d, is_causal)


def attention_q8(q, k, v, k_scale, v_scale, is_causal: bool = False, sm_scale: float | None = None,
                 cache_seqlens=None, block_table=None, query_lens=None, block_size: int = 32,
                 rope_cos=None, rope_sin=None, start_pos=0,
                 num_splits: int | None = None) -> torch.Tensor:
    """See ``stackkernels_amd.torch.flash_attention_q8``."""
    dev = q.device
    width = table_width(q, cache_seqlens, block_table)
    cache = (k, v, k_scale, v_scale)
    rest = tuple(layout_of(t) for t in cache)
    shape, as_is, dims = _attention_shape(layout_of(q), *rest, width, block_size, bool(is_causal))
    check_q8_devices(dev, q, cache)
    if not as_is or q.data_ptr() & 15:
        q = kernel_operand(q)
        shape = _attention_shape(layout_of(q), *rest, width, block_size, bool(is_causal))[0]
    _, b, hq, _, sq, _, d, _ = dims
    lens = None if cache_seqlens is None else int32_operand(cache_seqlens, "cache_seqlens", (b,), dev)
    q_lens = None if query_lens is None else int32_operand(query_lens, "query_lens", (b,), dev)
    table = None if width is None else int32_operand(block_table, "block_table", (b, width), dev)
    rope, _keep = rope_tail(rope_cos, rope_sin, start_pos, b, d, dev)
    out = torch.empty((b, hq, sq, d), dtype=q.dtype, device=dev)
    if width == 0:
        return out.zero_()
    ns, nb = plan_q8(*dims)
    if num_splits is not None:
        ns, nb = int(num_splits), int(num_splits) * b * hq * sq * 257 * 4
    ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None
    with _lib.device_guard(dev):
        rc = _lib.load().sk_attn_q8(
            shape, q.data_ptr(), k.data_ptr(), v.data_ptr(), k_scale.data_ptr(),
            v_scale.data_ptr(), out.data_ptr(), None if ws is None else ws.data_ptr(), nb, ns,
            None if table is None else table.data_ptr(), None if lens is None else lens.data_ptr(),
            None if q_lens is None else q_lens.data_ptr(), *rope,
            1.0 / math.sqrt(d) if sm_scale is None else float(sm_scale), _lib.stream_ptr(dev))
    if rc:
        _lib.check(rc, "flash_attention_q8")
    return out


__all__ = ["attention_q8", "plan_q8", "table_width", "validate_q8_attention"]
