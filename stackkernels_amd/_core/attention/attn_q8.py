"""Launcher of attention over a cache held in 8-bit codes (``sk_attn_q8``): one or
more query tokens per row, contiguous or paged, per-row key and query counts."""

from __future__ import annotations

import ctypes
import functools

import torch

from stackkernels_amd._core.attention import _lib
from stackkernels_amd._core.attention._common import check_device, default_scale, kernel_operand
from stackkernels_amd._core.attention._rope import rope_args
from stackkernels_amd._core.cache.quantized import (
    check_codes,
    int32_operand,
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


def validate_q8_attention(q, k, v, k_scale, v_scale, cache_seqlens, block_table, query_lens,
                          block_size) -> tuple[int, int, int, int, int]:
    """(units, KV heads, tokens per unit, keys a row can have, table width)."""
    if q.dim() != 4:
        raise ValueError(f"Expected 4D q (B, H, S, D), got {q.dim()}D")
    b, hq, sq, d = q.shape
    units, hkv, rows = validate_q8_cache(k, v, k_scale, v_scale, b, d, block_table is not None,
                                         block_size)
    if hkv == 0 or hq % hkv != 0:
        raise ValueError(f"Query heads ({hq}) must be divisible by KV heads ({hkv}) for GQA/MQA")
    width = 0
    if block_table is not None:
        if cache_seqlens is None:
            raise ValueError("a paged cache (block_table) needs cache_seqlens")
        width = table_operand(block_table, b).shape[1]
    return units, hkv, rows, width * rows if block_table is not None else rows, width


def attention_q8(q, k, v, k_scale, v_scale, is_causal: bool = False, sm_scale: float | None = None,
                 cache_seqlens=None, block_table=None, query_lens=None, block_size: int = 32,
                 rope_cos=None, rope_sin=None, start_pos=0,
                 num_splits: int | None = None) -> torch.Tensor:
    """See ``stackkernels_amd.torch.flash_attention_q8``."""
    units, hkv, rows, sk, width = validate_q8_attention(q, k, v, k_scale, v_scale, cache_seqlens,
                                                        block_table, query_lens, block_size)
    b, hq, sq, d = q.shape
    dev = check_device(q)
    check_codes(dev, k, v, k_scale, v_scale)
    lens = None if cache_seqlens is None else int32_operand(cache_seqlens, "cache_seqlens", b, dev)
    q_lens = None if query_lens is None else int32_operand(query_lens, "query_lens", b, dev)
    table = None
    if block_table is not None:
        table = table_operand(block_table, b).to(device=dev, dtype=torch.int32).contiguous()
    rope = rope_args(rope_cos, rope_sin, start_pos, b, d, dev)
    q = kernel_operand(q)
    code = _lib.dtype_code(q.dtype)
    ns, nb = plan_q8(code, b, hq, hkv, sq, sk, d, bool(is_causal))
    if num_splits is not None:
        nb = nb // max(ns, 1) * num_splits if ns > 1 else num_splits * b * hq * sq * 257 * 4
        ns = int(num_splits)
    ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None
    out = torch.empty((b, hq, sq, d), dtype=q.dtype, device=dev)
    lib = _lib.load()
    with _lib.device_guard(dev):
        rc = lib.sk_attn_q8(
            code, _lib.code_type(k.dtype), q.data_ptr(), k.data_ptr(), v.data_ptr(),
            k_scale.data_ptr(), v_scale.data_ptr(), out.data_ptr(),
            None if ws is None else ws.data_ptr(), nb, ns, b, hq, hkv, sq, units, rows, width,
            block_size, d, _lib.strides3(q), _lib.strides3(k), _lib.strides3(v),
            _lib.strides3(k_scale), _lib.strides3(v_scale), _lib.strides3(out),
            None if table is None else table.data_ptr(), None if lens is None else lens.data_ptr(),
            None if q_lens is None else q_lens.data_ptr(), int(bool(is_causal)),
            *(rope.args if rope is not None else _lib.NO_ROPE), default_scale(d, sm_scale),
            _lib.stream_ptr(dev))
    _lib.check(rc, "flash_attention_q8")
    return out


__all__ = ["attention_q8", "plan_q8", "validate_q8_attention"]
