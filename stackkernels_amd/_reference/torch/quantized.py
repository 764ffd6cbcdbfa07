"""The 8-bit key/value cache in plain torch: the path of CPU tensors and of
``backend='reference'``, and the statement of what the kernels compute.

A cache holds 8-bit codes (``int8`` or ``float8_e4m3fn``) and one float32 scale
per block of ``block_size`` tokens and KV head; an element's value is
``scale * code``.
"""

from __future__ import annotations

import math

import torch

TINY_SCALE = 2.0 ** -126
CODE_DTYPES = (torch.int8, torch.float8_e4m3fn)


def needed_scale(amax: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """float32 scale that a block with largest magnitude ``amax`` (float32) asks for:
    ``amax / 127`` in int8; in e4m3 the smallest power of two that brings it to
    448 or less; at least 2^-126."""
    if dtype == torch.int8:
        return (amax * (1.0 / 127.0)).clamp(min=TINY_SCALE)
    m, e = torch.frexp(amax)
    e = torch.where(m > 0.875, e - 8, e - 9).clamp(min=-126)
    return torch.where(amax > 0, ((e + 127) << 23).view(torch.float32), TINY_SCALE)


def encode(x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """Nearest codes (ties to even, saturated) of values divided by their scale."""
    if dtype == torch.int8:
        return torch.round(x.nan_to_num(nan=0.0).clamp(-127, 127)).to(torch.int8)
    return x.clamp(-448, 448).to(torch.float8_e4m3fn)


def append(k, v, k_cache, v_cache, k_scale, v_scale, starts, news, table, block_size) -> None:
    """Write the first ``news[b]`` tokens of row b (keys rotated already) as tokens
    ``starts[b]``, ... of its cache; ``table`` (lists of pages) for a paged pool."""
    rows = k_cache.shape[2]
    for b, (start, n) in enumerate(zip(starts, news)):
        start = max(start, 0)
        cap = rows if table is None else len(table[b]) * rows
        stop = min(start + min(max(n, 0), k.shape[2]), cap)
        if stop <= start:
            continue
        for lo in range(start // block_size * block_size, stop, block_size):
            unit, row = b, lo
            if table is not None:
                unit, row = table[b][lo // rows], lo % rows
                if not 0 <= unit < k_cache.shape[0]:
                    continue
            a, z = max(lo, start), min(lo + block_size, stop)
            for x, cache, scale in ((k, k_cache, k_scale), (v, v_cache, v_scale)):
                x = x[b, :, a - start:z - start].to(cache.device, torch.float32)  # (H, n, D)
                mag = x.abs()
                amax = torch.where(mag < math.inf, mag, 0).flatten(1).amax(1)
                now = needed_scale(amax, cache.dtype)
                codes = cache[unit, :, row:row + block_size].view(torch.uint8)
                if a > lo:
                    had = scale[unit, :, row // block_size]
                    now = torch.where(had > now, had, now)
                    old = codes[:, :a - lo]
                    moved = encode(old.contiguous().view(cache.dtype).float()
                                   * (had / now)[:, None, None], cache.dtype).view(torch.uint8)
                    old.copy_(torch.where((had < now)[:, None, None], moved, old))
                inv = (torch.ones_like(now) / now)[:, None, None]
                codes[:, a - lo:z - lo] = encode(x * inv, cache.dtype).view(torch.uint8)
                scale[unit, :, row // block_size] = now


def values(codes: torch.Tensor, scale: torch.Tensor, block_size: int, dtype=torch.float32):
    """What (..., S, D) codes with scales (..., ceil(S / block_size)) stand for."""
    s = scale.to(dtype).repeat_interleave(block_size, dim=-1)[..., :codes.shape[-2]]
    return codes.to(dtype) * s.unsqueeze(-1)


def row_values(cache, scale, b: int, n: int, pages, block_size: int, dtype=torch.float32):
    """(values (H, m, D) of the first n tokens of row b, their token numbers): tokens
    in a page outside the pool are left out."""
    if pages is None:
        return (values(cache[b, :, :n], scale[b, :, :-(-n // block_size)], block_size, dtype),
                torch.arange(n))
    rows = cache.shape[2]
    parts, at = [cache.new_empty((cache.shape[1], 0, cache.shape[3]), dtype=dtype)], []
    for i in range(-(-n // rows)):
        m = min(rows, n - i * rows)
        if 0 <= pages[i] < cache.shape[0]:
            parts.append(values(cache[pages[i], :, :m], scale[pages[i], :, :-(-m // block_size)],
                                block_size, dtype))
            at += range(i * rows, i * rows + m)
    return torch.cat(parts, dim=1), torch.tensor(at, dtype=torch.int64)


def attention(q, k_cache, v_cache, k_scale, v_scale, lens, q_lens, table, block_size, is_causal,
              sm_scale):
    """softmax(sm_scale q k^T) v over each row's own keys; zeros for a query past the
    row's own or with no key."""
    hq, hkv = q.shape[1], k_cache.shape[1]
    out = torch.zeros_like(q, memory_format=torch.contiguous_format)
    for b, (n, m) in enumerate(zip(lens, q_lens)):
        pages = None if table is None else table[b]
        k, at = row_values(k_cache, k_scale, b, n, pages, block_size)
        v, _ = row_values(v_cache, v_scale, b, n, pages, block_size)
        if m == 0 or at.numel() == 0:
            continue
        x = q[b, :, :m].float().reshape(hkv, hq // hkv * m, -1)
        s = torch.matmul(x, k.transpose(-1, -2)) * sm_scale
        s = s.view(hkv, hq // hkv, m, -1)
        if is_causal:
            hidden = at.to(q.device)[None] > torch.arange(n - m, n, device=q.device)[:, None]
            s = s.masked_fill(hidden, -math.inf)
        dead = (s == -math.inf).all(-1, keepdim=True)
        w = torch.softmax(s.masked_fill(dead, 0.0), dim=-1).masked_fill(dead, 0.0)
        o = torch.matmul(w.view(hkv, -1, w.shape[-1]), v)
        out[b, :, :m] = o.view(hq, m, -1).to(q.dtype)
    return out


def page_plan(table, lens, news, ring, state, page_size: int, max_new: int):
    """``sk_kv_page_plan`` on Python numbers: ``table`` and ``ring`` are changed in
    place; returns (slots, new lengths, state) as lists."""
    size, width = len(ring), len(table[0]) if table else 0
    cap = width * page_size
    head, count = state[0] % size, min(max(state[1], 0), size)
    taken, asked, back = 0, 0, 0
    slots, out, puts = [], [], []
    for b, (n, d) in enumerate(zip(lens, news)):
        n = min(max(n, 0), cap)
        want = max(n + min(d, max_new), 0)
        po = -(-n // page_size)
        if want > cap:
            want = n
        pn = -(-want // page_size)
        if pn > po:
            first = asked
            asked += pn - po
            if asked > count:
                want = n
            else:
                taken += pn - po
                for j in range(po, pn):
                    table[b][j] = ring[(head + first + j - po) % size]
        for j in range(pn, po):
            if count + back < size:
                puts.append(((head + count + back) % size, table[b][j]))
            back += 1
        out.append(want)
        row = [-1] * max_new
        for t in range(max(want - n, 0)):
            page = table[b][(n + t) // page_size]
            if page >= 0:
                row[t] = page * page_size + (n + t) % page_size
        slots.append(row)
    for i, page in puts:
        ring[i] = page
    return slots, out, [(head + taken) % size, min(size, count - taken + back)]


__all__ = ["CODE_DTYPES", "TINY_SCALE", "append", "attention", "encode", "needed_scale",
           "page_plan", "row_values", "values"]
