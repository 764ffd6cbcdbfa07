"""GPU tests of the 8-bit cache: page plans, the append and attention over codes.

The append and the plan are compared with the CPU path bit for bit; attention with
a 64-bit oracle, within the bound that ``_q8.attention64`` counts."""

import math

import pytest
import torch

from stackkernels_amd._core.attention.attn_q8 import attention_q8
from stackkernels_amd._reference.torch.rope import precompute_freqs
from stackkernels_amd.torch import (
    flash_attention_q8,
    flash_decode_q8,
    kv_cache_update_q8,
    kv_page_plan,
)

import _q8

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ----------------------------------------------------------------- page plan

@pytest.mark.parametrize("b,width,page,max_new,spare", [
    (1, 1, 16, 1, 0), (7, 5, 16, 1, 3), (7, 5, 16, 40, 8), (255, 4, 64, 1, 60), (256, 4, 64, 1, 300),
    (257, 4, 64, 1, 5), (1000, 3, 32, 2, 200), (40, 9, 32, 17, 4), (33, 90, 32, 2500, 900),
    (300, 40, 16, 300, 900), (5, 3, 1, 2, 2), (3, 200, 32, 5000, 300), (4, 4, 16, 0, 3)])
def test_page_plan(device, b, width, page, max_new, spare):
    model = _q8.PlanModel(page, width, max_new)
    for seed in range(3):
        pages, lens, news, free, head, size = _q8.random_plan(b, width, page, max_new, spare, seed)
        table, ring, state = _q8.plan_tensors(pages, free, head, size, width, "cuda")
        args = (i32(lens), i32(news))
        want_slots, want_lens = model.step(pages, lens, news, free)
        got = kv_page_plan(table, *args, ring, state, page, max_new=max_new)
        _q8.check_plan(table, ring, got[2], got[0], got[1], pages, want_slots, want_lens, free)
        again = kv_page_plan(table, *args, ring, state, page, max_new=max_new)
        assert all(torch.equal(x, y) for x, y in zip(got, again))


def test_page_plan_strided_table_and_steps(device):
    """Many steps on a table that is a slice of a wider one; nothing outside it changes."""
    b, width, page = 19, 6, 16
    wide = torch.full((b, width + 5), -3, dtype=torch.int32, device="cuda")
    model = _q8.PlanModel(page, width, 3)
    pages, lens, news, free, head, size = _q8.random_plan(b, width, page, 3, 40, 11)
    table, ring, state = _q8.plan_tensors(pages, free, head, size, width, "cuda")
    wide[:, 2:2 + width] = table
    table = wide[:, 2:2 + width]
    now = i32(lens)
    g = torch.Generator().manual_seed(5)
    for _ in range(40):
        slots, now, state = kv_page_plan(table, now, i32(news), ring, state, page, max_new=3)
        want_slots, lens = model.step(pages, lens, news, free)
        _q8.check_plan(table, ring, state, slots, now, pages, want_slots, lens, free)
        news = torch.randint(-4, 4, (b,), generator=g).tolist()
        news[int(torch.randint(0, b, (1,), generator=g))] = -1000
    assert bool((wide[:, :2] == -3).all()) and bool((wide[:, 2 + width:] == -3).all())


# -------------------------------------------------------------------- append

def _append_both(dtype, code, d, block, paged, t, starts, news, rope=False, values=None, hkv=2,
                 page=64, cap=200):
    b = len(starts)
    k, v = _q8.randn(b, t, hkv, d, seed=1), _q8.randn(b, hkv, t, d, seed=2) * 3
    if values is not None:
        values(k, v)
    k, v = k.to(dtype).transpose(1, 2), v.to(dtype)
    table = None
    if paged:
        width = -(-cap // page)
        table = torch.randperm(b * width, generator=torch.Generator().manual_seed(3)).view(b, width)
        table[-1, -1] = b * width + 7
        shape = (b * width, hkv, page)
    else:
        shape = (b, hkv, cap)
    kc, ks = _q8.make_cache(*shape, d, block, code, seed=4)
    vc, vs = _q8.make_cache(*shape, d, block, code, seed=5)
    kw = dict(block_size=block)
    if rope:
        cos, sin = precompute_freqs(d, cap + t)
        kw.update(rope_cos=cos, rope_sin=sin, start_pos=torch.tensor(starts))
    # the device's cache: a slice of a larger one, heads and rows apart
    big = torch.zeros(shape[0], hkv + 1, shape[2] + 2, d + 16, dtype=torch.uint8, device="cuda")
    views = []
    for c in (kc, vc):
        w = big.clone().view(c.dtype)[:, 1:, 1:-1, :d]
        w.view(torch.uint8).copy_(c.view(torch.uint8).cuda())
        views.append(w)
    scales = []
    for s in (ks, vs):
        w = torch.zeros(s.shape[0], s.shape[2], s.shape[1], device="cuda").transpose(1, 2)
        w.copy_(s)
        scales.append(w)
    n = None if news is None else torch.tensor(news)
    kv_cache_update_q8(k, v, kc, vc, ks, vs, torch.tensor(starts), n, table, **kw)
    if rope:
        kw.update(rope_cos=kw["rope_cos"].cuda(), rope_sin=kw["rope_sin"].cuda(),
                  start_pos=kw["start_pos"].cuda())
    kv_cache_update_q8(k.cuda(), v.cuda(), *views, *scales, i32(starts),
                       None if news is None else i32(news), None if table is None else table.cuda(), **kw)
    for got, want in zip(views, (kc, vc)):
        got = got.cpu()
        diff = got.view(torch.uint8) != want.view(torch.uint8)
        if code == "e4m3":  # two encodings are NaN (0x7f and 0xff): which one is not promised
            diff &= ~(got.float().isnan() & want.float().isnan())
        assert not bool(diff.any()), int(diff.sum())
    for got, want in zip(scales, (ks, vs)):
        assert torch.equal(got.cpu().view(torch.int32), want.view(torch.int32))


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("d,block,paged", [(64, 32, True), (128, 64, False), (80, 32, False),
                                           (256, 64, True), (16, 32, False), (96, 32, True)])
def test_append_matches_reference(device, code, dtype, d, block, paged):
    _append_both(DTYPES[dtype], code, d, block, paged, 1, [0, 31, 32, 63, 64, 199, 200, -5], None)
    _append_both(DTYPES[dtype], code, d, block, paged, 75, [0, 1, 31, 32, 100, 150, 190, 5],
                 [75, 74, 1, 0, 60, 75, 33, -2])


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("fp16", 64), ("fp32", 96), ("bf16", 256)])
def test_append_rotates(device, code, dtype, d):
    _append_both(DTYPES[dtype], code, d, 64, True, 70, [0, 3, 64, 100], [70, 69, 33, 1], rope=True)
    _append_both(DTYPES[dtype], code, d, 32, False, 1, [0, 3, 64, 199], None, rope=True)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_append_long_blocks(device, code):
    """A block with more new elements than a workgroup keeps in registers."""
    _append_both(torch.bfloat16, code, 256, 512, True, 700, [0, 100, 511], [700, 650, 513], page=512,
                 cap=1536)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_append_extreme_values(device, code):
    def values(k, v):
        k[0] = 0
        k[1] *= 1e-38
        k[2] *= 1e37
        k[3, 5], k[3, 6, 0, 3], k[3, 7, 0, 3] = math.inf, -math.inf, math.nan
        v[0] *= 1e-44
        v[1, :, 1:] = math.nan
        v[2] = math.inf

    _append_both(torch.float32, code, 64, 32, False, 40, [0, 7, 30, 32], [40, 40, 39, 11], values=values)


# ----------------------------------------------------------------- attention

def _attend(dtype, code, hq, hkv, sq, d, block, page, lens, q_lens=None, causal=True, rope=False,
            splits=None, scale=None, poison=True, table_change=None, seed=0):
    b = len(lens)
    cap = max(max(lens), 1)
    q = _q8.randn(b, sq, hq, d, seed=seed).to(dtype).transpose(1, 2)
    table = None
    if page:
        width = -(-cap // page)
        table = torch.randperm(b * width + 2, generator=torch.Generator().manual_seed(3))[:b * width]
        table = table.view(b, width)
        if table_change is not None:
            table_change(table)
        shape = (b * width + 2, hkv, page)
    else:
        shape = (b, hkv, cap)
    kc, ks = _q8.make_cache(*shape, d, block, code, seed=seed + 1)
    vc, vs = _q8.make_cache(*shape, d, block, code, seed=seed + 2)
    ql = [sq] * b if q_lens is None else q_lens
    sc = d ** -0.5 if scale is None else scale
    qr, kw = q, {}
    if rope:
        cos, sin = precompute_freqs(d, cap + sq + 1)
        starts = [max(n - m, 0) for n, m in zip(lens, ql)]
        qr = torch.stack([_q8.rotate64(q[i].double(), cos, sin, starts[i]) for i in range(b)])
        kw = dict(rope_cos=cos.cuda(), rope_sin=sin.cuda(), start_pos=i32(starts))
    want, tol = _q8.attention64(qr, kc, vc, ks, vs, block, lens, ql,
                                None if table is None else table.tolist(), causal, sc,
                                splits or 1, dtype, rope)
    # Every code and scale behind the rows' lengths is NaN on the device.
    dk, dv, dks, dvs = (x.clone().cuda() for x in (kc, vc, ks, vs))
    if poison:
        bad = 0x7F
        for i in range(b):
            if page:
                for j in range(table.shape[1]):
                    p, n = int(table[i, j]), max(min(lens[i] - j * page, page), 0)
                    if 0 <= p < shape[0]:
                        dk.view(torch.uint8)[p, :, n:] = bad
                        dv.view(torch.uint8)[p, :, n:] = bad
                        dks[p, :, -(-n // block):] = math.nan
                        dvs[p, :, -(-n // block):] = math.nan
            else:
                n = lens[i]
                dk.view(torch.uint8)[i, :, n:] = bad
                dv.view(torch.uint8)[i, :, n:] = bad
                dks[i, :, -(-n // block):] = math.nan
                dvs[i, :, -(-n // block):] = math.nan
    got = attention_q8(q.cuda(), dk, dv, dks, dvs, causal, scale, i32(lens),
                       None if table is None else table.cuda(),
                       None if q_lens is None else i32(q_lens), block, num_splits=splits, **kw)
    assert got.dtype == dtype and got.is_contiguous()
    _q8.check_within(got, want, tol)
    for i in range(b):
        assert bool((got[i, :, ql[i]:] == 0).all())
    return got


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("d", [16, 64, 80, 96, 128, 256])
def test_decode_head_dims(device, code, dtype, d):
    _attend(DTYPES[dtype], code, 4, 2, 1, d, 32, 0, [1, 31, 32, 33, 0, 127, 128, 129, 300], causal=False)
    _attend(DTYPES[dtype], code, 4, 1, 1, d, 64, 64, [1, 63, 64, 65, 0, 255, 256, 300])


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("hq,hkv", [(2, 2), (6, 2), (16, 1), (17, 1), (40, 1), (64, 1), (70, 1), (96, 2)])
def test_decode_groups(device, code, dtype, hq, hkv):
    _attend(DTYPES[dtype], code, hq, hkv, 1, 64, 32, 32, [200, 77, 1], splits=3)
    _attend(DTYPES[dtype], code, hq, hkv, 1, 128, 128, 0, [200, 77, 1])


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("sq", [2, 3, 5, 16, 33, 130])
def test_queries(device, code, dtype, sq):
    for causal in (True, False):
        _attend(DTYPES[dtype], code, 6, 2, sq, 64, 32, 32, [sq, 200, 150, 2, 0, 300],
                [sq, sq, sq - 1, sq, 1, 0], causal=causal)
    _attend(DTYPES[dtype], code, 4, 4, sq, 128, 64, 0, [sq + 1, 260, 131])


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [16, 64, 80, 96, 128, 256])
def test_many_rows(device, code, dtype, d):
    """Chunks of more rows than a decode's: ragged, paged with the smallest pages and
    contiguous, split and whole, rotated, and pages outside the pool."""
    def change(table):
        table[0, 1], table[0, 3] = -1, 10 ** 6

    _attend(DTYPES[dtype], code, 4, 2, 40, d, 32, 32, [40, 200, 39, 1, 0, 260], [40, 37, 39, 5, 1, 40],
            table_change=change)
    _attend(DTYPES[dtype], code, 4, 2, 70, d, 64, 0, [300, 70, 7], [70, 69, 7], splits=3)
    _attend(DTYPES[dtype], code, 2, 2, 129, d, 128, 128, [140, 257], causal=False)
    _attend(DTYPES[dtype], code, 8, 1, 20, d, 32, 64, [150, 77], rope=True)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("sq", [1, 5, 40])
def test_uneven_scales(device, code, sq):
    """V scales that differ by far more than fp16 holds, zeros among them: what is small
    next to the rest may vanish, the sum of the weights may not."""
    b, hq, hkv, n, d = 2, 4, 2, 320, 64
    kc, ks = _q8.make_cache(b, hkv, n, d, 32, code, seed=1)
    vc, vs = _q8.make_cache(b, hkv, n, d, 32, code, seed=2)
    size = torch.tensor([1.0, 1e-12, 0.0, 1e6, 1e-30, 1.0, 1e-38, 3.0, 0.0, 1e-4])
    for order in (torch.arange(10), torch.arange(9, -1, -1)):
        v2, k2 = vs * size[order], ks.clone()
        k2[:, :, 4] = 0
        q = _q8.randn(b, hq, sq, d, seed=3).bfloat16()
        for splits in (1, 3):
            got = attention_q8(q.cuda(), kc.cuda(), vc.cuda(), k2.cuda(), v2.cuda(), True,
                               num_splits=splits)
            want, tol = _q8.attention64(q, kc, vc, k2, v2, 32, [n] * b, [sq] * b, None, True, d ** -0.5,
                                        splits)
            _q8.check_within(got, want, tol)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("fp16", 256), ("fp32", 64), ("bf16", 96)])
def test_splits(device, code, dtype, d):
    """Explicit split counts: pieces without a key, single keys, more pieces than tiles."""
    for splits in (1, 2, 5, 16, 40):
        _attend(DTYPES[dtype], code, 4, 2, 1, d, 32, 64, [513, 100, 1, 0], splits=splits)
        _attend(DTYPES[dtype], code, 4, 2, 7, d, 32, 0, [300, 7, 3], splits=splits)


@pytest.mark.parametrize("dtype,d,sq", [("bf16", 128, 1), ("fp16", 64, 4), ("fp32", 96, 3), ("bf16", 80, 40)])
def test_rotated_queries(device, dtype, d, sq):
    _attend(DTYPES[dtype], "int8", 4, 2, sq, d, 32, 64, [200, 64, 41], rope=True)


@pytest.mark.parametrize("scale", [0.5, -0.2, 0.0])
def test_scales_of_scores(device, scale):
    _attend(torch.bfloat16, "e4m3", 4, 2, 3, 64, 32, 32, [100, 33], scale=scale)


def test_pages_outside_the_pool(device):
    def change(table):
        table[0, 0], table[0, 2], table[1, 1] = -1, 10 ** 6, 2 ** 31 - 1
        table[2] = -5

    for sq in (1, 4):
        got = _attend(torch.bfloat16, "e4m3", 4, 2, sq, 64, 32, 32, [128, 70, 60], table_change=change)
        assert bool((got[2] == 0).all())


def test_strided_cache_in_place(device):
    """Codes and scales that are slices of a (tokens, heads) layout are read in place."""
    b, hq, hkv, n, d = 3, 8, 2, 150, 64
    kc, ks = _q8.make_cache(b, hkv, n, d, 32, "int8", seed=1)
    vc, vs = _q8.make_cache(b, hkv, n, d, 32, "int8", seed=2)
    both = torch.zeros(b, n + 3, 2, hkv, d + 32, dtype=torch.int8, device="cuda")
    both[:, 1:n + 1, 0, :, 16:16 + d] = kc.transpose(1, 2).cuda()
    both[:, 1:n + 1, 1, :, 16:16 + d] = vc.transpose(1, 2).cuda()
    k, v = (both[:, 1:n + 1, i, :, 16:16 + d].transpose(1, 2) for i in (0, 1))
    sc = torch.zeros(b, ks.shape[2], hkv, 2, device="cuda")
    sc[..., 0], sc[..., 1] = ks.transpose(1, 2).cuda(), vs.transpose(1, 2).cuda()
    q = _q8.randn(b, hq, 4, d).bfloat16()
    got = flash_attention_q8(q.cuda(), k, v, sc[..., 0].transpose(1, 2), sc[..., 1].transpose(1, 2), True)
    want, tol = _q8.attention64(q, kc, vc, ks, vs, 32, [n] * b, [4] * b, None, True, d ** -0.5)
    _q8.check_within(got, want, tol)
    # one cache for all rows of the batch, and one row of keys for all tokens
    got = flash_decode_q8(q[:, :, :1].cuda(), kc[:1].cuda().expand(b, -1, -1, -1),
                          vc[:1].cuda().expand(b, -1, -1, -1), ks[:1].cuda().expand(b, -1, -1),
                          vs[:1].cuda().expand(b, -1, -1))
    ex = [x[:1].expand(b, *x.shape[1:]) for x in (kc, vc, ks, vs)]
    want, tol = _q8.attention64(q[:, :, :1], *ex, 32, [n] * b, [1] * b, None, False, d ** -0.5)
    _q8.check_within(got, want, tol)


def test_nan_key_reaches_only_its_row(device):
    kc, ks = _q8.make_cache(2, 1, 300, 64, 32, "e4m3", seed=1)
    vc, vs = _q8.make_cache(2, 1, 300, 64, 32, "e4m3", seed=2)
    kc.view(torch.uint8)[0, 0, 250, 3] = 0x7F
    q = _q8.randn(2, 4, 1, 64).bfloat16().cuda()
    for splits in (1, 4):
        out = attention_q8(q, kc.cuda(), vc.cuda(), ks.cuda(), vs.cuda(), num_splits=splits)
        assert bool(out[0].isnan().all()) and bool(out[1].isfinite().all())
        seen = attention_q8(q, kc.cuda(), vc.cuda(), ks.cuda(), vs.cuda(), cache_seqlens=i32([250, 300]),
                            num_splits=splits)
        assert bool(seen.isfinite().all())


def test_empty_calls(device):
    kc = torch.zeros(2, 2, 0, 64, dtype=torch.int8, device="cuda")
    s = torch.zeros(2, 2, 0, device="cuda")
    q = torch.ones(2, 4, 3, 64, device="cuda").half()
    assert bool((flash_attention_q8(q, kc, kc, s, s, True) == 0).all())
    kv_cache_update_q8(q[:, :2], q[:, :2], kc, kc.clone(), s, s.clone(), i32([0, 0]))
    assert flash_attention_q8(q[:, :, :0], kc, kc, s, s).shape == (2, 4, 0, 64)
    assert flash_attention_q8(q[:0], kc[:0], kc[:0], s[:0], s[:0]).shape == (0, 4, 3, 64)
    slots, lens, state = kv_page_plan(i32([]).view(0, 3), i32([]), i32([]), i32([1]), i32([0, 1]), 16)
    assert slots.shape == (0, 1) and lens.shape == (0,) and state.tolist() == [0, 1]


# ------------------------------------------------------------------- serving

@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_serving_steps_captured(device, code):
    """Plan, append and decode as a server runs them, captured once and replayed:
    every replay equals the eager step on a second copy of the state."""
    b, hq, hkv, d, page, block, width = 5, 8, 2, 64, 64, 32, 4
    pool = b * width + 1
    cos, sin = (x.cuda() for x in precompute_freqs(d, width * page + 8))

    def state():
        return dict(kc=torch.zeros(pool, hkv, page, d, dtype=_q8.CODES[code], device="cuda"),
                    vc=torch.zeros(pool, hkv, page, d, dtype=_q8.CODES[code], device="cuda"),
                    ks=torch.zeros(pool, hkv, page // block, device="cuda"),
                    vs=torch.zeros(pool, hkv, page // block, device="cuda"),
                    table=torch.full((b, width), -1, dtype=torch.int32, device="cuda"),
                    ring=torch.arange(pool, dtype=torch.int32, device="cuda"),
                    free=i32([0, pool]), lens=i32([0] * b), news=i32([1] * b),
                    q=torch.zeros(b, hq, 1, d, dtype=torch.bfloat16, device="cuda"),
                    kv=torch.zeros(2, b, hkv, 1, d, dtype=torch.bfloat16, device="cuda"))

    def step(s):
        _, lens, free = kv_page_plan(s["table"], s["lens"], s["news"], s["ring"], s["free"], page)
        kv_cache_update_q8(s["kv"][0], s["kv"][1], s["kc"], s["vc"], s["ks"], s["vs"], s["lens"],
                           lens - s["lens"], s["table"], block_size=block, rope_cos=cos, rope_sin=sin,
                           start_pos=s["lens"])
        out = flash_decode_q8(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], cache_seqlens=lens,
                              block_table=s["table"], block_size=block, rope_cos=cos, rope_sin=sin,
                              start_pos=lens - 1)
        s["lens"].copy_(lens)
        s["free"].copy_(free)
        return out

    eager, graph = state(), state()
    warm = state()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(warm)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step(graph)
    for i in range(70):
        torch.manual_seed(i)
        q = torch.randn(b, hq, 1, d, device="cuda").bfloat16()
        kv = torch.randn(2, b, hkv, 1, d, device="cuda").bfloat16() * (1 + i % 7)
        news = [1] * b
        news[i % b] = -40 if i % 23 == 22 else 0 if i % 9 == 8 else 1
        for s in (eager, graph):
            s["q"].copy_(q)
            s["kv"].copy_(kv)
            s["news"].copy_(i32(news))
        want = step(eager)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want), i
        for name in ("lens", "free", "table", "ring", "ks", "vs"):
            assert torch.equal(eager[name], graph[name]), (i, name)
    held = eager["lens"].tolist()
    assert max(held) > 60 and eager["free"][1].item() == pool - sum(-(-n // page) for n in held)


def test_side_stream(device):
    """Work queued on a stream of its own is ordered on that stream."""
    kc, ks = (x.cuda() for x in _q8.make_cache(4, 2, 500, 128, 32, "int8", seed=1))
    vc, vs = (x.cuda() for x in _q8.make_cache(4, 2, 500, 128, 32, "int8", seed=2))
    q = _q8.randn(4, 8, 1, 128).bfloat16().cuda()
    want = flash_decode_q8(q, kc, vc, ks, vs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late = torch.zeros_like(q)
        torch.cuda._sleep(10_000_000)
        late.copy_(q)
        got = flash_decode_q8(late, kc, vc, ks, vs)
    side.synchronize()
    assert torch.equal(got, want)


def test_long_cache_offsets(device):
    """Codes more than 2^31 bytes into a pool, and tokens far into one long row."""
    page, d, hkv = 64, 128, 8
    per = hkv * page * d
    pages = (1 << 31) // per + 40
    pool = torch.zeros(pages, hkv, page, d, dtype=torch.int8, device="cuda")
    ks, vs = torch.ones(pages, hkv, 2, device="cuda"), torch.ones(pages, hkv, 2, device="cuda")
    last = pages - 1
    k, v = _q8.randn(1, hkv, 70, d, seed=1).bfloat16(), _q8.randn(1, hkv, 70, d, seed=2).bfloat16()
    table = torch.tensor([[last, last - 1]])
    vpool = torch.zeros_like(pool)
    kv_cache_update_q8(k.cuda(), v.cuda(), pool, vpool, ks, vs, i32([0]), None, table.cuda())
    q = _q8.randn(1, 16, 1, d, seed=3).bfloat16()
    got = flash_decode_q8(q.cuda(), pool, vpool, ks, vs, cache_seqlens=i32([70]), block_table=table.cuda())
    tail = [x[last - 1:].cpu() for x in (pool, vpool, ks, vs)]
    want, tol = _q8.attention64(q, *tail, 32, [70], [1], [[1, 0]], False, d ** -0.5)
    _q8.check_within(got, want, tol)
    assert not bool(pool[:last - 1].any())
