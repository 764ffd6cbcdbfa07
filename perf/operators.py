"""Serving from a key/value cache held in 8 bits: what is timed, and the same
in elementary torch operations.

A server's step has three calls, and each is an operator here:

``plan``    block tables and slot maps from request lengths: rows that grow take
            pages from a ring of free ones, rows that shrink (rejected drafts,
            finished requests) give theirs back.
``append``  new keys (rotated) and values into a cache of 8-bit codes, float8
            e4m3 or int8, with one scale for each block of tokens and head.
``decode``  one query token per row over such a cache.
``attend``  several query tokens per row over it: drafted tokens, a chunk of a
            prompt behind what the cache holds, a long prompt.

A case is a dict of plain values.  Lengths (``Sk``, ``T``, ``Sq``) are the
longest of the batch; with ``ragged`` the rows' own lengths are drawn below.
``page`` 0 means a contiguous cache.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TINY = 2.0 ** -126


def listed():
    return [
        # A decode step's plan: every request one token further, some done or rolled back.
        dict(name="plan_step", kind="plan", B=256, T=1, page=64, Sk=4096),
        # The plan of a prefill batch: thousands of new tokens a request.
        dict(name="plan_prompts", kind="plan", B=48, T=8192, page=32, Sk=2048),
        # A decode step's append: one token per request into half-filled blocks.
        dict(name="append_step", kind="append", dtype="bf16", code="int8", B=64, Hkv=8, D=128, T=1,
             Sk=512, page=64, block=32, rope=True, ragged=False),
        # A chunk of prompts of different lengths behind what the rows hold.
        dict(name="append_chunk", kind="append", dtype="fp16", code="e4m3", B=8, Hkv=8, D=128,
             T=2048, Sk=1500, page=0, block=64, rope=True, ragged=True),
        # One user's decode with a short cache: latency and launches.
        dict(name="decode_one", kind="decode", dtype="bf16", code="int8", B=1, Hq=32, Hkv=8,
             Sk=1000, D=128, page=0, block=32, rope=False, ragged=False),
        # A server's decode step: ragged lengths in a paged pool, RoPE fused.
        dict(name="decode_paged", kind="decode", dtype="bf16", code="e4m3", B=32, Hq=32, Hkv=8,
             Sk=4096, D=128, page=64, block=64, rope=True, ragged=True),
        # A full batch over long caches, 4.3 GB of codes.
        dict(name="decode_batch", kind="decode", dtype="bf16", code="int8", B=64, Hq=32, Hkv=8,
             Sk=32768, D=128, page=0, block=128, rope=False, ragged=False),
        # Few KV heads and very long contexts (MQA).
        dict(name="decode_mqa", kind="decode", dtype="fp16", code="e4m3", B=8, Hq=64, Hkv=1,
             Sk=131072, D=128, page=0, block=32, rope=False, ragged=False),
        # A 32-bit model with wide heads.
        dict(name="decode_f32", kind="decode", dtype="fp32", code="e4m3", B=4, Hq=16, Hkv=4,
             Sk=8001, D=256, page=0, block=32, rope=False, ragged=True),
        # Drafted tokens checked in one pass.
        dict(name="attend_draft", kind="attend", dtype="bf16", code="int8", B=16, Hq=64, Hkv=8,
             Sq=5, Sk=6000, D=64, page=32, block=32, rope=True, ragged=True),
        # One chunk of a long prompt against what the cache already holds.
        dict(name="attend_chunk", kind="attend", dtype="bf16", code="e4m3", B=1, Hq=32, Hkv=8,
             Sq=512, Sk=16000, D=128, page=0, block=64, rope=True, ragged=False),
        # Long prompts behind a shared prefix: bound by the matrix products.
        dict(name="attend_long", kind="attend", dtype="bf16", code="int8", B=2, Hq=32, Hkv=8,
             Sq=4096, Sk=16384, D=128, page=128, block=128, rope=False, ragged=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_once(rng):
    kind = rng.choice(["plan", "append", "append", "decode", "decode", "attend", "attend"])
    c = dict(kind=kind)
    if kind == "plan":
        t = rng.choice([1, 1, _log_int(rng, 2, 8192)])
        c.update(B=_log_int(rng, 1, 2000 if t < 64 else 64), T=t, page=rng.choice([16, 32, 64, 128, 256]),
                 Sk=_log_int(rng, 16, 16384))
        return c
    page = rng.choice([0, 0, 32, 64, 128, 256])
    block = rng.choice([n for n in (32, 64, 128) if page % n == 0])
    c.update(dtype=rng.choice(["bf16", "bf16", "bf16", "fp16", "fp16", "fp32"]),
             code=rng.choice(["int8", "e4m3"]), D=rng.choice([64, 64, 80, 96, 128, 128, 128, 256]),
             page=page, block=block, rope=rng.random() < 0.5, ragged=rng.random() < 0.6)
    heads = rng.choice([(8, 8), (12, 12), (32, 32), (16, 4), (32, 8), (32, 4), (64, 8), (24, 2),
                        (32, 1), (64, 1)])
    if kind == "append":
        c.update(Hkv=heads[1], B=_log_int(rng, 1, 64), T=rng.choice([1, _log_int(rng, 2, 4096)]),
                 Sk=_log_int(rng, 1, 4096))
    elif kind == "decode":
        c.update(Hq=heads[0], Hkv=heads[1], B=_log_int(rng, 1, 64), Sk=_log_int(rng, 1, 131072))
    else:
        sq = rng.choice([_log_int(rng, 2, 16), _log_int(rng, 17, 4096)])
        c.update(Hq=heads[0], Hkv=heads[1], B=_log_int(rng, 1, 16), Sq=sq,
                 Sk=sq + _log_int(rng, 1, 30000))
    return c


def _cost(case):
    """Rough seconds of a pass, only to keep drawn cases below the largest listed one."""
    w = work(case)
    return max(w["flops"] / (1e14 if case.get("dtype") == "fp32" else 5e14), w["bytes"] / 5e12)


def draw(rng):
    most = max(_cost(c) for c in listed()) / 2
    while True:
        c = _draw_once(rng)
        if _cost(c) <= most:
            return c


def work(case):
    """Bytes and operations a pass cannot do without (means over the drawn lengths)."""
    kind, B = case["kind"], case["B"]
    if kind == "plan":
        T, page = case["T"], case["page"]
        pages = B * ((T + 1) / 2 if T > 1 else 1) / page
        # lengths read and written, ids read and stored, one slot a token
        return {"bytes": 12 * B + 4 * B + 8 * pages + 8 * B * T, "flops": 0}
    e = 4 if case["dtype"] == "fp32" else 2
    Hkv, D, block = case["Hkv"], case["D"], case["block"]
    share = 0.5 if case["ragged"] else 1.0
    if kind == "append":
        new = B * max(1, case["T"] * share)
        data = 2 * new * Hkv * D * (e + 1)
        # scales of the blocks, rotation table rows
        data += 2 * 4 * Hkv * max(B, new / block) + (2 * 4 * D * new if case["rope"] else 0)
        return {"bytes": data, "flops": 4 * new * Hkv * D}
    Hq, Sk = case["Hq"], case["Sk"]
    if kind == "decode":
        keys = max(1.0, Sk * share)
        data = 2 * B * Hkv * keys * (D + 4 / block) + 2 * B * Hq * D * e
        return {"bytes": data, "flops": 4 * B * Hq * keys * D}
    Sq = case["Sq"]
    keys = Sq + (Sk - Sq) * share
    rows = max(1.0, Sq * (0.75 if case["ragged"] else 1.0))
    data = 2 * B * Hkv * keys * (D + 4 / block) + 2 * B * Hq * Sq * D * e
    return {"bytes": data, "flops": 4 * D * B * Hq * rows * (keys - rows / 2)}


# ---------------------------------------------------------------- the format

def _needed_scale(amax, code):
    """Scale a block's largest magnitude asks for (32 bits): amax / 127 in int8; in
    e4m3 the smallest power of two that brings it to 448 or less, so that a later,
    larger scale of the block moves older codes by an exact factor."""
    if code == "int8":
        return (amax * (1.0 / 127.0)).clamp(min=TINY)
    m, e = torch.frexp(amax)
    e = torch.where(m > 0.875, e - 8, e - 9).clamp(min=-126)
    return torch.where(amax > 0, ((e + 127) << 23).view(torch.float32), TINY)


def _to_code(x, code):
    """Nearest code (ties to even) of values already divided by their scale."""
    if code == "int8":
        return torch.round(x.clamp(-127, 127)).to(torch.int8)
    return x.clamp(-448, 448).to(torch.float8_e4m3fn)


def _made_cache(g, dev, shape, block, code, spread):
    """Codes and scales of normal keys or values whose size differs by head and block."""
    units, h, rows, d = shape
    nb = -(-rows // block)
    codes = torch.empty(shape, device=dev, dtype=CODES[code])
    scales = torch.empty(units, h, nb, device=dev)
    step = max(1, (1 << 26) // max(1, h * nb * block * d))
    for u in range(0, units, step):
        n = min(step, units - u)
        x = torch.randn(n, h, nb, block, d, generator=g, device=dev)
        x *= torch.exp(spread * torch.randn(n, h, nb, 1, 1, generator=g, device=dev))
        s = _needed_scale(x.abs().amax(dim=(-1, -2)), code)
        scales[u:u + n] = s
        c = _to_code(x * (torch.ones_like(s) / s)[..., None, None], code)
        codes[u:u + n] = c.view(n, h, nb * block, d)[:, :, :rows]
    return codes, scales


def _tables(rows, d, dev):
    """Rotation tables (rows, D), angles in 64 bits."""
    f = 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device=dev) / d)
    a = torch.arange(rows, dtype=torch.float64, device=dev)[:, None] * f[None]
    a = torch.cat([a, a], dim=1)
    return a.cos().float(), a.sin().float()


# ------------------------------------------------------------------- inputs

def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    kind, B, page = case["kind"], case["B"], case["page"]

    def ints(lo, hi, n=B):
        return torch.randint(lo, hi + 1, (n,), generator=g, device=dev, dtype=torch.int32)

    def perm(n):
        return torch.randperm(n, generator=g, device=dev).to(torch.int32)

    if kind == "plan":
        T, Sk = case["T"], case["Sk"]
        lens = ints(0, Sk)
        new = torch.ones_like(lens) if T == 1 else ints(0, T)
        # one row in eight is done or gives back some of its last tokens
        back = torch.rand(B, generator=g, device=dev) < 0.125
        new = torch.where(back, -torch.minimum(lens, ints(1, Sk)), new)
        per_row = -(-(Sk + T) // page)
        held = -(-Sk // page)
        ids = perm(B * per_row)
        table = torch.full((B, per_row), -1, device=dev, dtype=torch.int32)
        table[:, :held] = ids[:B * held].view(B, held)
        ring = torch.full((B * per_row,), -1, device=dev, dtype=torch.int32)
        free = ids[B * held:]
        head = B * per_row // 3
        at = (head + torch.arange(free.numel(), device=dev)) % ring.numel()
        ring[at] = free
        state = torch.tensor([head, free.numel()], device=dev, dtype=torch.int32)
        return dict(case=case, table=table, lens=lens, new=new, ring=ring, state=state)

    dt, code = DTYPES[case["dtype"]], case["code"]
    Hkv, Sk, D, block = case["Hkv"], case["Sk"], case["D"], case["block"]
    T = case["T"] if kind == "append" else case.get("Sq", 1)
    s = dict(case=case)
    unit = max(page, block)
    if kind == "append":
        s["lens"] = ints(0, Sk) if case["ragged"] else ints(max(0, Sk - unit), Sk)
        s["new"] = ints(1, T) if case["ragged"] else torch.full_like(s["lens"], T)
        room = (Sk + T + 3 * unit) // unit * unit
    elif kind == "decode":
        s["lens"] = ints(1, Sk) if case["ragged"] else torch.full((B,), Sk, device=dev, dtype=torch.int32)
        room = Sk
    else:
        # each row's own queries are the last of its keys
        s["new"] = ints((T + 1) // 2, T) if case["ragged"] else torch.full((B,), T, device=dev, dtype=torch.int32)
        s["lens"] = s["new"] + (ints(0, Sk - T) if case["ragged"] else Sk - T)
        room = Sk
    if page:
        per_row = -(-room // page)
        s["table"] = perm(B * per_row).view(B, per_row)
        shape = (B * per_row, Hkv, page, D)
    else:
        s["table"] = None
        shape = (B, Hkv, room, D)
    s["kc"], s["ks"] = _made_cache(g, dev, shape, block, code, 0.5)
    s["vc"], s["vs"] = _made_cache(g, dev, shape, block, code, 0.5)
    if case["rope"]:
        s["cos"], s["sin"] = _tables(Sk + T, D, dev)

    def projected(heads, n):
        # a projection's (B, n, heads, D) output, seen head by head
        x = torch.randn(B, n, heads, D, generator=g, device=dev)
        return x.to(dt).transpose(1, 2)

    # position of each row's first new token
    if kind == "append":
        s["pos"] = s["lens"]
        s["k"], s["v"] = projected(Hkv, T), projected(Hkv, T)
    else:
        s["pos"] = s["lens"] - s["new"] if "new" in s else s["lens"] - 1
        s["q"] = projected(case["Hq"], T)
    return s


# -------------------------------------------------------------- plain forms

def _plan(s):
    page, T = s["case"]["page"], s["case"]["T"]
    table, ring = s["table"], s["ring"]
    B, width = table.shape
    N = ring.numel()
    head, count = s["state"][0].long(), s["state"][1].long()
    old = s["lens"].long()
    new = s["new"].long()
    want = (old + new).clamp(min=0)
    fits = want <= width * page
    po, pn = (old + page - 1) // page, (want + page - 1) // page
    need = torch.where((new > 0) & fits, pn - po, 0)
    cum = need.cumsum(0)
    granted = (new <= 0) | (fits & ((need == 0) | (cum <= count)))
    used = torch.where(granted, need, 0)
    lens = torch.where(granted, want, old)
    back = torch.where(new < 0, po - pn, 0)
    behind = back.cumsum(0) - back
    # pages given back join the ring's end
    j = torch.arange(width, device=table.device)[None]
    gives = (j >= pn[:, None]) & (j < po[:, None]) & (new < 0)[:, None]
    slot = (head + count + behind[:, None] + j - pn[:, None]) % N
    out = torch.cat([ring, ring.new_zeros(1)])
    out.scatter_(0, torch.where(gives, slot, N).flatten(), table.flatten())
    # pages taken come from its front
    takes = (j >= po[:, None]) & (j < pn[:, None]) & (used > 0)[:, None]
    got = ring[(head + (cum - need)[:, None] + j - po[:, None]) % N]
    table = torch.where(takes, got, table)
    t = torch.arange(T, device=table.device)[None]
    pos = old[:, None] + t
    at = table.gather(1, (pos // page).clamp(max=width - 1)).long()
    slots = torch.where((t < (lens - old)[:, None]) & (at >= 0), at * page + pos % page, -1)
    n = used.sum()
    state = torch.stack([(head + n) % N, count - n + back.sum()]).to(torch.int32)
    return table, slots, lens.to(torch.int32), out[:N], state


def _rotated(x, cos, sin, start):
    """x (B, H, T, D) in 32 bits, token t of row b rotated to position start[b] + t."""
    t = torch.arange(x.shape[2], device=x.device)
    pos = start.long()[:, None] + t[None]
    c, n = cos[pos][:, None], sin[pos][:, None]
    a, b = x.chunk(2, dim=-1)
    return x * c + torch.cat([-b, a], dim=-1) * n


def _append(s):
    case = s["case"]
    code, block, page, T, B = (case[n] for n in ("code", "block", "page", "T", "B"))
    start, new = s["lens"].long(), s["new"].long()
    dev = start.device
    n_blocks = (T + block - 2) // block + 1
    first = start // block
    blk = first[:, None] + torch.arange(n_blocks, device=dev)[None]  # (B, n)
    pos = blk[..., None] * block + torch.arange(block, device=dev)  # (B, n, block)
    t = pos - start[:, None, None]
    fresh = (t >= 0) & (t < new[:, None, None])
    older = (t < 0)[:, :, None, :, None]
    written = fresh.any(-1)[:, :, None]
    if page:
        unit = s["table"].long().gather(1, (pos // page).view(B, -1)).view_as(pos)
        row = pos % page
    else:
        unit = torch.arange(B, device=dev)[:, None, None].expand_as(pos)
        row = pos
    cell = unit[..., 0], slice(None), row[..., 0] // block
    src = t.clamp(0, T - 1)
    for name in ("k", "v"):
        x = s[name].float()
        if name == "k" and case["rope"]:
            x = _rotated(x, s["cos"], s["sin"], s["pos"])
        x = x.transpose(1, 2)[torch.arange(B, device=dev)[:, None, None], src]  # (B, n, block, H, D)
        x = x.permute(0, 1, 3, 2, 4)
        f = fresh[:, :, None, :, None]
        amax = torch.where(f, x.abs(), 0).amax(dim=(-1, -2))  # (B, n, H)
        need = _needed_scale(amax, code)
        cache, scale = s[name + "c"], s[name + "s"]
        had = scale[cell]
        now = torch.where(older.any(-2).squeeze(-1), torch.maximum(had, need), need)
        now = torch.where(written, now, had)
        fresh_codes = _to_code(x * (torch.ones_like(now) / now)[..., None, None], code)
        bits = cache.view(torch.uint8)
        held = bits[unit, :, row].permute(0, 1, 3, 2, 4)  # (B, n, H, block, D)
        moved = _to_code(held.contiguous().view(CODES[code]).float() * (had / now)[..., None, None], code)
        kept = torch.where(older & written[..., None, None] & (now > had)[..., None, None],
                           moved.view(torch.uint8), held)
        put = torch.where(f, fresh_codes.view(torch.uint8), kept)
        bits[unit, :, row] = put.permute(0, 1, 3, 2, 4)
        scale[cell] = now
    return s["kc"], s["vc"], s["ks"], s["vs"]


def _values(s, name, dtype, rows=slice(None)):
    """The cache's values (B, H, room, D): codes times their block's scale."""
    c, sc, block = s[name + "c"], s[name + "s"], s["case"]["block"]
    if s["table"] is not None:
        at = s["table"][rows].long()
        b, n = at.shape
        c = c.view(torch.uint8)[at].transpose(1, 2).contiguous().view(c.dtype)  # (B, H, n, page, D)
        sc = sc[at].transpose(1, 2).reshape(b, c.shape[1], -1)
        c = c.view(b, c.shape[1], -1, c.shape[-1])
    else:
        c, sc = c[rows], sc[rows]
    return c.to(dtype) * sc.to(dtype).repeat_interleave(block, dim=-1)[:, :, :c.shape[2], None]


def _attend(s):
    case = s["case"]
    q = s["q"].float()
    B, Hq, Sq, D = q.shape
    Hkv = case["Hkv"]
    lens = s["lens"].long()
    own_q = s["new"].long() if "new" in s else torch.ones_like(lens)
    if case["rope"]:
        q = _rotated(q, s["cos"], s["sin"], s["pos"])
    k = _values(s, "k", torch.float32)
    q = q.reshape(B, Hkv, Hq // Hkv * Sq, D) * (1.0 / math.sqrt(D))
    scores = torch.matmul(q, k.transpose(-1, -2)).view(B, Hkv, Hq // Hkv, Sq, -1)
    del k
    i = torch.arange(Sq, device=q.device)
    last = (lens - own_q)[:, None] + i[None]  # last key that query i sees
    j = torch.arange(scores.shape[-1], device=q.device)
    seen = (j[None, None] <= last[..., None]) & (i[None] < own_q[:, None])[..., None]
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    scores.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = scores.sum(dim=-1, keepdim=True)
    v = _values(s, "v", torch.float32)
    out = torch.matmul(scores.view(B, Hkv, -1, scores.shape[-1]), v).view(B, Hkv, Hq // Hkv, Sq, D)
    out = out / torch.where(total > 0, total, 1.0)
    return out.view(B, Hq, Sq, D).to(s["q"].dtype)


# ---------------------------------------------------------------- one pass

def run(state):
    case = state["case"]
    kind = case["kind"]
    if not own:
        if kind == "plan":
            return _plan(state)
        if kind == "append":
            return _append(state)
        return _attend(state)
    from stackkernels_amd.torch import (flash_attention_q8, flash_decode_q8, kv_cache_update_q8,
                                        kv_page_plan)

    if kind == "plan":
        slots, lens, now = kv_page_plan(state["table"], state["lens"], state["new"], state["ring"],
                                        state["state"], case["page"], max_new=case["T"])
        return state["table"], slots, lens, state["ring"], now
    rope = {}
    if case["rope"]:
        rope = dict(rope_cos=state["cos"], rope_sin=state["sin"], start_pos=state["pos"])
    if kind == "append":
        kv_cache_update_q8(state["k"], state["v"], state["kc"], state["vc"], state["ks"],
                           state["vs"], state["lens"], state["new"], state["table"],
                           block_size=case["block"], **rope)
        return state["kc"], state["vc"], state["ks"], state["vs"]
    cache = (state["kc"], state["vc"], state["ks"], state["vs"])
    if kind == "decode":
        lens = state["lens"] if case["ragged"] or case["page"] else None
        return flash_decode_q8(state["q"], *cache, cache_seqlens=lens, block_table=state["table"],
                               block_size=case["block"], **rope)
    return flash_attention_q8(state["q"], *cache, is_causal=True, cache_seqlens=state["lens"],
                              block_table=state["table"], query_lens=state["new"],
                              block_size=case["block"], **rope)


# ------------------------------------------------------- 64-bit definitions

def exact(case, seed):
    """The definitions row by row in 64 bits (whole numbers for a plan)."""
    s = prepare(case, seed)
    if case["kind"] == "plan":
        return _exact_plan(s)
    if case["kind"] == "append":
        return _exact_append(s)
    return _exact_attend(s)


def _exact_plan(s):
    page, T = s["case"]["page"], s["case"]["T"]
    table, ring = s["table"].cpu().tolist(), s["ring"].cpu().tolist()
    old, new = s["lens"].cpu().tolist(), s["new"].cpu().tolist()
    head, count = s["state"].cpu().tolist()
    n, width = len(ring), len(table[0])
    front, end, short = head, head + count, False
    lens, slots = [], torch.full((len(old), T), -1, dtype=torch.int64)
    for b, (o, d) in enumerate(zip(old, new)):
        want = max(o + d, 0)
        po, pn = -(-o // page), -(-want // page)
        if d < 0:
            for p in table[b][pn:po]:
                ring[end % n] = p
                end += 1
        elif want > width * page or (pn > po and (short or front + pn - po > head + count)):
            short = short or want <= width * page
            want = o
        else:
            for j in range(po, pn):
                table[b][j] = ring[front % n]
                front += 1
        lens.append(want)
        if want > o:
            pos = torch.arange(o, want)
            at = torch.tensor(table[b])[pos // page]
            slots[b, :want - o] = torch.where(at >= 0, at * page + pos % page, -1)
    return (torch.tensor(table, dtype=torch.int32), slots, torch.tensor(lens, dtype=torch.int32),
            torch.tensor(ring, dtype=torch.int32),
            torch.tensor([front % n, end - front], dtype=torch.int32))


def _exact_append(s):
    case = s["case"]
    block, page, int8 = case["block"], case["page"], case["code"] == "int8"
    most = 127.0 if int8 else 448.0

    def rounded(x):
        x = x.clamp(-most, most)
        if int8:
            return torch.round(x)
        e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
        step = torch.exp2(e - 3)
        return torch.round(x / step) * step

    out = []
    lens, new = s["lens"].tolist(), s["new"].tolist()
    for name in ("k", "v"):
        codes, scales = s[name + "c"].double(), s[name + "s"].double()
        for b, (o, m) in enumerate(zip(lens, new)):
            x = s[name][b, :, :m].double()  # (H, m, D)
            if name == "k" and case["rope"]:
                c, n = s["cos"][o:o + m].double(), s["sin"][o:o + m].double()
                half = x.shape[-1] // 2
                x = torch.cat([x[..., :half] * c[:, :half] - x[..., half:] * n[:, :half],
                               x[..., half:] * c[:, half:] + x[..., :half] * n[:, half:]], dim=-1)
            for lo in range(o // block * block, o + m, block):
                u, r0 = (int(s["table"][b, lo // page]), lo % page) if page else (b, lo)
                a, z = max(lo, o), min(lo + block, o + m)
                y = x[:, a - o:z - o]
                amax = y.abs().amax(dim=(1, 2)).clamp(min=1e-300)
                need = amax / 127.0 if int8 else torch.exp2(torch.ceil(torch.log2(amax / 448.0)))
                need = need.clamp(min=TINY)
                had = scales[u, :, r0 // block].clone()
                now = torch.maximum(had, need) if a > lo else need
                rows = codes[u, :, r0:r0 + block]
                if a > lo:
                    moved = rounded(rows[:, :a - lo] * (had / now)[:, None, None])
                    rows[:, :a - lo] = torch.where((now > had)[:, None, None], moved, rows[:, :a - lo])
                rows[:, a - lo:z - lo] = rounded(y / now[:, None, None])
                scales[u, :, r0 // block] = now
        out.append((codes, scales))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def _exact_attend(s):
    case = s["case"]
    q = s["q"]
    B, Hq, Sq, D = q.shape
    group = Hq // case["Hkv"]
    out = torch.zeros(B, Hq, Sq, D, dtype=torch.float64, device=q.device)
    lens = s["lens"].tolist()
    rows = s["new"].tolist() if "new" in s else [1] * B
    for b in range(B):
        n, m = lens[b], rows[b]
        k = _values(s, "k", torch.float64, slice(b, b + 1))[0, :, :n]
        v = _values(s, "v", torch.float64, slice(b, b + 1))[0, :, :n]
        x = q[b, :, :m].double()
        if case["rope"]:
            c, t = s["cos"][n - m:n].double(), s["sin"][n - m:n].double()
            half = D // 2
            x = torch.cat([x[..., :half] * c[:, :half] - x[..., half:] * t[:, :half],
                           x[..., half:] * c[:, half:] + x[..., :half] * t[:, half:]], dim=-1)
        hidden = torch.arange(n, device=q.device)[None] > torch.arange(n - m, n, device=q.device)[:, None]
        for h in range(Hq):
            p = (x[h] @ k[h // group].t()) / math.sqrt(D)
            p = torch.softmax(p.masked_fill(hidden, -math.inf), dim=-1)
            out[b, h, :m] = p @ v[h // group]
    return out
