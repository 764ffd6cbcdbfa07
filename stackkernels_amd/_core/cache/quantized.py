"""Launchers of the 8-bit cache's writer (``sk_kv_cache_update_q8``) and of the
page plan (``sk_kv_page_plan``), and the shape rules of the cache format.

A serving loop makes these calls once per layer and step, so what depends on
shapes, strides and types alone is checked once per combination (``lru_cache``)."""

from __future__ import annotations

import functools

import torch

from stackkernels_amd._core.attention import _lib
from stackkernels_amd._core.attention._common import _SUPPORTED, kernel_operand
from stackkernels_amd._core.attention._rope import RopeArgs
from stackkernels_amd._reference.torch.quantized import CODE_DTYPES


def _integer(x, name: str, shape: tuple) -> torch.Tensor:
    if not isinstance(x, torch.Tensor):
        x = torch.as_tensor(x)
    if tuple(x.shape) != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(x.shape)}")
    if x.dtype.is_floating_point or x.dtype == torch.bool:
        raise ValueError(f"{name} must be an integer tensor, got {x.dtype}")
    return x


def int32_operand(x, name: str, shape: tuple, dev) -> torch.Tensor:
    """``x`` as the kernels read it: contiguous int32 on ``dev``."""
    if (type(x) is torch.Tensor and x.dtype is torch.int32 and x.shape == shape
            and x.get_device() == dev.index and x.is_contiguous()):
        return x
    return _integer(x, name, shape).to(device=dev, dtype=torch.int32).contiguous()


def table_operand(table, b: int) -> torch.Tensor:
    """A block table as an integer (B, max_pages) tensor."""
    if not isinstance(table, torch.Tensor):
        table = torch.as_tensor(table)
    if table.dim() != 2 or table.shape[0] != b:
        raise ValueError(f"block_table must have shape ({b}, max_pages), got {tuple(table.shape)}")
    return _integer(table, "block_table", tuple(table.shape))


def rope_tail(cos, sin, start_pos, b: int, d: int, dev) -> tuple[tuple, RopeArgs | None]:
    """(the rotation's arguments of a call, what must live until it returns)."""
    if cos is None and sin is None:
        return _lib.NO_ROPE, None
    if (type(cos) is torch.Tensor and type(sin) is torch.Tensor and cos.dtype is torch.float32
            and sin.dtype is torch.float32 and cos.is_contiguous() and sin.is_contiguous()
            and cos.shape == sin.shape and cos.dim() == 2 and cos.shape[1] == d and d % 16 == 0
            and cos.get_device() == dev.index == sin.get_device()
            and not (cos.data_ptr() | sin.data_ptr()) & 15):
        # Tables as a program keeps them: what RopeArgs would find, without its copies.
        rows = cos.shape[0]
        if type(start_pos) is int:
            return (cos.data_ptr(), sin.data_ptr(), _lib.SK_F32, rows, d, None, start_pos), None
        if (type(start_pos) is torch.Tensor and start_pos.dtype is torch.int32
                and start_pos.shape == (b,) and start_pos.get_device() == dev.index
                and start_pos.is_contiguous()):
            return (cos.data_ptr(), sin.data_ptr(), _lib.SK_F32, rows, d, start_pos.data_ptr(),
                    0), None
    rope = RopeArgs(cos, sin, start_pos, b, d, dev)
    return rope.args, rope


def layout_of(t: torch.Tensor) -> tuple:
    return t.shape, t.stride(), t.dtype


def validate_q8_cache(k, v, ks, vs, b: int, d: int, paged: bool, block_size: int) -> tuple:
    """(units, KV heads, tokens per unit) of a cache of 8-bit codes, each tensor given
    as ``layout_of``; raises ValueError (NotImplementedError for a type or head dim
    without a kernel)."""
    for name, t in (("k", k), ("v", v)):
        if len(t[0]) != 4:
            raise ValueError(f"Expected 4D codes for {name} (units, H, S, D), got {len(t[0])}D")
    if k[0] != v[0]:
        raise ValueError(f"k and v cache shapes differ: {tuple(k[0])} vs {tuple(v[0])}")
    if k[2] != v[2]:
        raise ValueError(f"k and v cache types differ: {k[2]} vs {v[2]}")
    if k[2] not in CODE_DTYPES:
        raise NotImplementedError(f"cache dtype {k[2]} unsupported (int8, float8_e4m3fn)")
    units, h, rows, dc = k[0]
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
    for name, t in (("k_scale", ks), ("v_scale", vs)):
        if tuple(t[0]) != want:
            raise ValueError(f"{name} must have shape {want}, got {tuple(t[0])}")
        if t[2] != torch.float32:
            raise ValueError(f"{name} must be float32, got {t[2]}")
    return units, h, rows


def check_cache_strides(k, v) -> None:
    """The kernels address codes in place (they are never copied)."""
    for name, t in (("k", k), ("v", v)):
        st = t[1]
        if st[3] != 1 or (st[0] | st[1] | st[2]) & 15:
            raise ValueError(f"the {name} cache needs a contiguous head dim and strides that are "
                             f"multiples of 16, got {tuple(st)}")


def check_q8_devices(dev, x: torch.Tensor, cache: tuple) -> None:
    """Kernel calls: every tensor on x's ROCm device, codes 16-byte aligned."""
    if not x.is_cuda:
        raise RuntimeError("the HIP kernels of the 8-bit cache need ROCm device tensors; got a tensor "
                           f"on {x.device} (use backend 'auto' or 'reference' for CPU tensors)")
    for t in cache:
        if t.get_device() != dev.index:
            raise ValueError(f"tensors on different devices: {dev} and {t.device}")
    if (cache[0].data_ptr() | cache[1].data_ptr()) & 15:
        raise ValueError("the k and v caches must be 16-byte aligned")


def validate_q8_update(k, v, kc, vc, ks, vs, paged: bool, block_size: int) -> tuple:
    """(B, KV heads, T, D, units, tokens per unit) of an append (``layout_of`` each)."""
    for name, t in (("k", k), ("v", v)):
        if len(t[0]) != 4:
            raise ValueError(f"Expected 4D tensor for {name} (B, H, T, D), got {len(t[0])}D")
    if k[0] != v[0]:
        raise ValueError(f"k and v shapes differ: {tuple(k[0])} vs {tuple(v[0])}")
    b, h, t, d = k[0]
    units, hc, rows = validate_q8_cache(kc, vc, ks, vs, b, d, paged, block_size)
    if hc != h:
        raise ValueError(f"the cache has {hc} KV heads, the new keys {h}")
    return b, h, t, d, units, rows


@functools.lru_cache(maxsize=512)
def _update_shape(k, v, kc, vc, ks, vs, width: int | None, block_size: int):
    b, h, t, d, units, rows = validate_q8_update(k, v, kc, vc, ks, vs, width is not None,
                                                 block_size)
    if k[2] != v[2]:
        raise ValueError(f"dtype mismatch: {k[2]} and {v[2]}")
    if k[2] not in _SUPPORTED:
        raise NotImplementedError(f"dtype {k[2]} has no HIP kernel (supported: {_SUPPORTED})")
    check_cache_strides(kc, vc)
    unit = 3 if k[2] == torch.float32 else 7
    as_is = all((x[1][3] == 1 or d == 1) and not (x[1][0] | x[1][1] | x[1][2]) & unit
                for x in (k, v))
    shape = _lib.q8_shape(
        (_lib.dtype_code(k[2]), _lib.code_type(kc[2]), b, h, h, t, units, rows, width or 0,
         block_size, d, 0),
        (k[1][:3], v[1][:3], kc[1][:3], vc[1][:3], ks[1], vs[1]))
    return shape, b, d, as_is


def kv_cache_update_q8(k, v, k_cache, v_cache, k_scale, v_scale, cache_seqlens, new_lens=None,
                       block_table=None, block_size: int = 32, rope_cos=None, rope_sin=None,
                       start_pos=0) -> None:
    """Append k, v (B, Hkv, T, D) to a cache of 8-bit codes, in place; see
    ``stackkernels_amd.torch.kv_cache_update_q8``."""
    dev = k.device
    width = None if block_table is None else table_operand(block_table, k.shape[0]).shape[1]
    cache = (k_cache, v_cache, k_scale, v_scale)
    rest = tuple(layout_of(t) for t in cache)
    shape, b, d, as_is = _update_shape(layout_of(k), layout_of(v), *rest, width, block_size)
    check_q8_devices(dev, k, (*cache, v))
    if not as_is or (k.data_ptr() | v.data_ptr()) & 15:
        k, v = kernel_operand(k), kernel_operand(v)
        shape = _update_shape(layout_of(k), layout_of(v), *rest, width, block_size)[0]
    lens = int32_operand(cache_seqlens, "cache_seqlens", (b,), dev)
    news = None if new_lens is None else int32_operand(new_lens, "new_lens", (b,), dev)
    table = None if width is None else int32_operand(block_table, "block_table", (b, width), dev)
    rope, _keep = rope_tail(rope_cos, rope_sin, start_pos, b, d, dev)
    if width == 0:
        return
    with _lib.device_guard(dev):
        rc = _lib.load().sk_kv_cache_update_q8(
            shape, k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
            k_scale.data_ptr(), v_scale.data_ptr(), lens.data_ptr(),
            None if news is None else news.data_ptr(), None if table is None else table.data_ptr(),
            *rope, _lib.stream_ptr(dev))
    if rc:
        _lib.check(rc, "kv_cache_update_q8")


@functools.lru_cache(maxsize=512)
def _plan_layout(table, ring, page_size: int, max_new: int) -> tuple[int, int]:
    if len(table[0]) != 2:
        raise ValueError("block_table must be a (B, max_pages) tensor")
    if len(ring[0]) != 1 or ring[0][0] == 0:
        raise ValueError("free_pages must be a 1-D tensor of at least one id")
    for name, t in (("block_table", table), ("free_pages", ring)):
        if t[2] != torch.int32:
            raise ValueError(f"{name} is changed in place and must be int32, got {t[2]}")
        if t[1][-1] != 1 and t[0][-1] > 1:
            raise ValueError(f"{name} is changed in place and needs a contiguous last dim")
    b, width = table[0]
    if b > 1 and table[1][0] < width:
        raise ValueError("block_table rows overlap")
    if page_size <= 0:
        raise ValueError(f"page_size must be positive, got {page_size}")
    if max_new < 0:
        raise ValueError(f"max_new must not be negative, got {max_new}")
    return b, width


def validate_page_plan(block_table, cache_seqlens, new_lens, free_pages, free_state, page_size,
                       max_new) -> tuple[int, int]:
    """(B, max_pages); the tensors that a plan changes must be int32 as they are."""
    if not isinstance(block_table, torch.Tensor):
        raise ValueError("block_table must be a (B, max_pages) tensor")
    if not isinstance(free_pages, torch.Tensor):
        raise ValueError("free_pages must be a 1-D tensor of at least one id")
    b, width = _plan_layout(layout_of(block_table), layout_of(free_pages), page_size, max_new)
    _integer(cache_seqlens, "cache_seqlens", (b,))
    _integer(new_lens, "new_lens", (b,))
    _integer(free_state, "free_state", (2,))
    return b, width


def kv_page_plan(block_table, cache_seqlens, new_lens, free_pages, free_state, page_size: int,
                 max_new: int = 1) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(slot_indices, cache_seqlens, free_state) after a step; see
    ``stackkernels_amd.torch.kv_page_plan``."""
    if not isinstance(block_table, torch.Tensor) or not isinstance(free_pages, torch.Tensor):
        raise ValueError("block_table and free_pages must be tensors")
    table = layout_of(block_table)
    b, width = _plan_layout(table, layout_of(free_pages), page_size, max_new)
    dev = block_table.device
    if not block_table.is_cuda or free_pages.get_device() != dev.index:
        raise RuntimeError("the HIP page plan needs block_table and free_pages on one ROCm device; got "
                           f"{dev} and {free_pages.device}")
    lens = int32_operand(cache_seqlens, "cache_seqlens", (b,), dev)
    news = int32_operand(new_lens, "new_lens", (b,), dev)
    state = int32_operand(free_state, "free_state", (2,), dev)
    if b == 0:
        return (torch.empty((0, max_new), dtype=torch.int64, device=dev), torch.empty_like(lens),
                state.clone())
    slots = torch.empty((b, max_new), dtype=torch.int64, device=dev)
    out, now = torch.empty_like(lens), torch.empty_like(state)
    with _lib.device_guard(dev):
        rc = _lib.load().sk_kv_page_plan(
            block_table.data_ptr(), lens.data_ptr(), news.data_ptr(), free_pages.data_ptr(),
            state.data_ptr(), slots.data_ptr(), out.data_ptr(), now.data_ptr(), b, width,
            max(table[1][0], width), page_size, max_new, free_pages.shape[0], _lib.stream_ptr(dev))
    if rc:
        _lib.check(rc, "kv_page_plan")
    return slots, out, now


__all__ = ["check_cache_strides", "check_q8_devices", "int32_operand", "kv_cache_update_q8",
           "kv_page_plan", "layout_of", "rope_tail", "table_operand", "validate_page_plan",
           "validate_q8_cache", "validate_q8_update"]
