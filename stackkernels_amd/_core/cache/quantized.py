"""Launchers of the 8-bit cache's writer (``sk_kv_cache_update_q8``) and of the
page plan (``sk_kv_page_plan``), and the shape rules of the cache format."""

from __future__ import annotations

import torch

from stackkernels_amd._core.attention import _lib
from stackkernels_amd._core.attention._common import check_device, kernel_operand
from stackkernels_amd._core.attention._rope import rope_args
from stackkernels_amd._reference.torch.quantized import CODE_DTYPES


def _integer(x, name: str, shape: tuple) -> torch.Tensor:
    if not isinstance(x, torch.Tensor):
        x = torch.as_tensor(x)
    if tuple(x.shape) != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(x.shape)}")
    if x.dtype.is_floating_point or x.dtype == torch.bool:
        raise ValueError(f"{name} must be an integer tensor, got {x.dtype}")
    return x


def int32_operand(x, name: str, b: int, dev) -> torch.Tensor:
    """``x`` (B,) as the kernels read it: int32 on ``dev``."""
    return _integer(x, name, (b,)).to(device=dev, dtype=torch.int32).contiguous()


def table_operand(table, b: int) -> torch.Tensor:
    """A block table as an integer (B, max_pages) tensor."""
    if not isinstance(table, torch.Tensor):
        table = torch.as_tensor(table)
    if table.dim() != 2 or table.shape[0] != b:
        raise ValueError(f"block_table must have shape ({b}, max_pages), got {tuple(table.shape)}")
    return _integer(table, "block_table", tuple(table.shape))


def validate_q8_cache(k_cache, v_cache, k_scale, v_scale, b: int, d: int, paged: bool,
                      block_size: int) -> tuple[int, int, int]:
    """(units, KV heads, tokens per unit) of a cache of 8-bit codes; raises ValueError
    (NotImplementedError for a type or head dim without a kernel)."""
    for name, t in (("k", k_cache), ("v", v_cache)):
        if t.dim() != 4:
            raise ValueError(f"Expected 4D codes for {name} (units, H, S, D), got {t.dim()}D")
    if k_cache.shape != v_cache.shape:
        raise ValueError(f"k and v cache shapes differ: {tuple(k_cache.shape)} vs "
                         f"{tuple(v_cache.shape)}")
    if k_cache.dtype != v_cache.dtype:
        raise ValueError(f"k and v cache types differ: {k_cache.dtype} vs {v_cache.dtype}")
    if k_cache.dtype not in CODE_DTYPES:
        raise NotImplementedError(f"cache dtype {k_cache.dtype} unsupported (int8, float8_e4m3fn)")
    units, h, rows, dc = k_cache.shape
    if dc != d:
        raise ValueError(f"Head dimension mismatch: the cache has {dc}, expected {d}")
    if d % 16 != 0 or d > 256:
        raise NotImplementedError(f"an 8-bit cache needs a head dim that is a multiple of 16 up to "
                                  f"256, got {d}")
    if block_size <= 0 or block_size % 32 != 0:
        raise ValueError(f"block_size must be a positive multiple of 32, got {block_size}")
    if paged and (rows <= 0 or rows % block_size != 0):
        raise ValueError(f"page_size ({rows}) must be a positive multiple of block_size "
                         f"({block_size})")
    if not paged and units != b:
        raise ValueError(f"Batch mismatch: the cache has {units} rows, expected {b}")
    want = (units, h, -(-rows // block_size))
    for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
        if tuple(t.shape) != want:
            raise ValueError(f"{name} must have shape {want}, got {tuple(t.shape)}")
        if t.dtype != torch.float32:
            raise ValueError(f"{name} must be float32, got {t.dtype}")
    return units, h, rows


def check_codes(dev, k_cache, v_cache, k_scale, v_scale) -> None:
    """Devices and layouts of a cache the kernels address in place (never copied)."""
    for name, t in (("k cache", k_cache), ("v cache", v_cache), ("k_scale", k_scale),
                    ("v_scale", v_scale)):
        if t.device != dev:
            raise ValueError(f"tensors on different devices: {dev} and {t.device} ({name})")
    for name, t in (("k", k_cache), ("v", v_cache)):
        st = t.stride()
        if st[3] != 1 or (st[0] | st[1] | st[2]) & 15 or t.data_ptr() & 15:
            raise ValueError(f"the {name} cache needs a contiguous head dim and 16-byte-aligned rows, "
                             f"got strides {tuple(st)}")


def validate_q8_update(k, v, k_cache, v_cache, k_scale, v_scale, block_table, block_size):
    """(B, KV heads, T, D, units, tokens per unit) of an append."""
    for name, t in (("k", k), ("v", v)):
        if t.dim() != 4:
            raise ValueError(f"Expected 4D tensor for {name} (B, H, T, D), got {t.dim()}D")
    if k.shape != v.shape:
        raise ValueError(f"k and v shapes differ: {tuple(k.shape)} vs {tuple(v.shape)}")
    b, h, t, d = k.shape
    units, hc, rows = validate_q8_cache(k_cache, v_cache, k_scale, v_scale, b, d,
                                        block_table is not None, block_size)
    if hc != h:
        raise ValueError(f"the cache has {hc} KV heads, the new keys {h}")
    return b, h, t, d, units, rows


def kv_cache_update_q8(k, v, k_cache, v_cache, k_scale, v_scale, cache_seqlens, new_lens=None,
                       block_table=None, block_size: int = 32, rope_cos=None, rope_sin=None,
                       start_pos=0) -> None:
    """Append k, v (B, Hkv, T, D) to a cache of 8-bit codes, in place; see
    ``stackkernels_amd.torch.kv_cache_update_q8``."""
    b, h, t, d, units, rows = validate_q8_update(k, v, k_cache, v_cache, k_scale, v_scale,
                                                 block_table, block_size)
    dev = check_device(k, v)
    check_codes(dev, k_cache, v_cache, k_scale, v_scale)
    lens = int32_operand(cache_seqlens, "cache_seqlens", b, dev)
    news = None if new_lens is None else int32_operand(new_lens, "new_lens", b, dev)
    table = None
    if block_table is not None:
        table = table_operand(block_table, b).to(device=dev, dtype=torch.int32).contiguous()
    rope = rope_args(rope_cos, rope_sin, start_pos, b, d, dev)
    k, v = kernel_operand(k), kernel_operand(v)
    lib = _lib.load()
    with _lib.device_guard(dev):
        rc = lib.sk_kv_cache_update_q8(
            _lib.dtype_code(k.dtype), _lib.code_type(k_cache.dtype), k.data_ptr(), v.data_ptr(),
            k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
            lens.data_ptr(), None if news is None else news.data_ptr(),
            None if table is None else table.data_ptr(), b, h, t, units, rows,
            0 if table is None else table.shape[1], block_size, d, _lib.strides3(k),
            _lib.strides3(v), _lib.strides3(k_cache), _lib.strides3(v_cache),
            _lib.strides3(k_scale), _lib.strides3(v_scale),
            *(rope.args if rope is not None else _lib.NO_ROPE), _lib.stream_ptr(dev))
    _lib.check(rc, "kv_cache_update_q8")


def validate_page_plan(block_table, cache_seqlens, new_lens, free_pages, free_state, page_size,
                       max_new) -> tuple[int, int]:
    """(B, max_pages); the tensors that a plan changes must be int32 as they are."""
    if not isinstance(block_table, torch.Tensor) or block_table.dim() != 2:
        raise ValueError("block_table must be a (B, max_pages) tensor")
    b, width = block_table.shape
    if not isinstance(free_pages, torch.Tensor) or free_pages.dim() != 1 or free_pages.numel() == 0:
        raise ValueError("free_pages must be a 1-D tensor of at least one id")
    for name, t in (("block_table", block_table), ("free_pages", free_pages)):
        if t.dtype != torch.int32:
            raise ValueError(f"{name} is changed in place and must be int32, got {t.dtype}")
        if t.numel() and t.stride(-1) != 1:
            raise ValueError(f"{name} is changed in place and needs a contiguous last dim")
    if b > 1 and block_table.stride(0) < width:
        raise ValueError("block_table rows overlap")
    _integer(cache_seqlens, "cache_seqlens", (b,))
    _integer(new_lens, "new_lens", (b,))
    _integer(free_state, "free_state", (2,))
    if page_size <= 0:
        raise ValueError(f"page_size must be positive, got {page_size}")
    if max_new < 0:
        raise ValueError(f"max_new must not be negative, got {max_new}")
    return b, width


def kv_page_plan(block_table, cache_seqlens, new_lens, free_pages, free_state, page_size: int,
                 max_new: int = 1) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(slot_indices, cache_seqlens, free_state) after a step; see
    ``stackkernels_amd.torch.kv_page_plan``."""
    b, width = validate_page_plan(block_table, cache_seqlens, new_lens, free_pages, free_state,
                                  page_size, max_new)
    dev = block_table.device
    if not block_table.is_cuda or free_pages.device != dev:
        raise RuntimeError("the HIP page plan needs block_table and free_pages on one ROCm device; got "
                           f"{dev} and {free_pages.device}")
    lens = int32_operand(cache_seqlens, "cache_seqlens", b, dev)
    news = int32_operand(new_lens, "new_lens", b, dev)
    state = _integer(free_state, "free_state", (2,)).to(device=dev, dtype=torch.int32).contiguous()
    slots = torch.empty((b, max_new), dtype=torch.int64, device=dev)
    out = torch.empty((b,), dtype=torch.int32, device=dev)
    now = torch.empty((2,), dtype=torch.int32, device=dev)
    if b == 0:
        now.copy_(state)
    lib = _lib.load()
    with _lib.device_guard(dev):
        rc = lib.sk_kv_page_plan(block_table.data_ptr(), lens.data_ptr(), news.data_ptr(),
                                 free_pages.data_ptr(), state.data_ptr(), slots.data_ptr(),
                                 out.data_ptr(), now.data_ptr(), b, width,
                                 max(block_table.stride(0), width), page_size, max_new,
                                 free_pages.numel(), _lib.stream_ptr(dev))
    _lib.check(rc, "kv_page_plan")
    return slots, out, now


__all__ = ["check_codes", "int32_operand", "kv_cache_update_q8", "kv_page_plan", "table_operand",
           "validate_page_plan", "validate_q8_cache", "validate_q8_update"]
