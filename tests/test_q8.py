"""The 8-bit cache on the CPU: the reference path of the append, the page plan and
the attention against 64-bit oracles, and what the public calls refuse."""

import math

import pytest
import torch

from stackkernels_amd._reference.torch.quantized import encode, needed_scale
from stackkernels_amd.torch import (
    flash_attention_q8,
    flash_decode_q8,
    kv_cache_update_q8,
    kv_page_plan,
)

import _q8


def test_needed_scale():
    a = torch.tensor([0.0, 1.0, 448.0, 449.0, 3.5, 3.51, 1e-40, 3e38])
    s = needed_scale(a, torch.float8_e4m3fn).double()
    assert s[0] == 2.0 ** -126 and s[6] == 2.0 ** -126
    for x, y in zip(a.double().tolist(), s.tolist()):
        assert math.frexp(y)[0] == 0.5 and x / y <= 448
        assert y == 2.0 ** -126 or x / (y / 2) > 448
    s = needed_scale(a, torch.int8).double()
    assert s[0] == 2.0 ** -126
    assert torch.allclose(s[1:6], a.double()[1:6] / 127, rtol=2.0 ** -22, atol=0)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_encode_rounds_to_nearest(code):
    dt = _q8.CODES[code]
    if code == "int8":
        x = torch.tensor([0.5, 1.5, -0.5, 126.6, 300.0, -300.0, math.inf, -math.inf, math.nan])
        assert encode(x, dt).tolist() == [0, 2, 0, 127, 127, -127, 127, -127, 0]
        return
    x = torch.cat([_q8.randn(2000) * 30, torch.tensor([1000.0, -1000.0, math.inf])])
    y = encode(x, dt).float()
    assert y[-3:].tolist() == [448.0, -448.0, 448.0]
    err = (y - x)[:-3].abs()
    assert bool((err <= torch.maximum(x[:-3].abs() * 2.0 ** -4, torch.tensor(2.0 ** -10))).all())
    assert encode(torch.tensor([math.nan]), dt).float().isnan().all()


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("block", [32, 64])
def test_append_values(code, paged, block):
    """Appends of different lengths, one behind the other: every value the cache
    stands for is within its rounding bound of what was appended.  int8: half a
    step of the block's scale, and half a step of each scale that a later append
    moved it to; e4m3: one rounding to the code (2^-4 relative, 2^-10 of the
    scale among subnormals) and one among the subnormals of a larger scale."""
    b, h, d, page, width = 3, 2, 32, 64, 4
    cap = page * width
    dt = _q8.CODES[code]
    table = torch.randperm(b * width, generator=torch.Generator().manual_seed(3)).view(b, width)
    shape = (b * width + 1, h, page, d) if paged else (b, h, cap, d)
    kc, vc = torch.zeros(shape, dtype=dt), torch.zeros(shape, dtype=dt)
    # what an earlier user of the cache left behind does not count
    ks = torch.full((shape[0], h, shape[2] // block), 1e30)
    vs = ks.clone()
    want = {"k": torch.zeros(b, h, cap, d), "v": torch.zeros(b, h, cap, d)}
    bound = {"k": torch.zeros(b, h, cap, d, dtype=torch.float64),
             "v": torch.zeros(b, h, cap, d, dtype=torch.float64)}
    lens = torch.zeros(b, dtype=torch.int64)

    def row(cache, scale, i):
        if paged:
            cache = torch.cat([cache[p] for p in table[i]], dim=1)
            scale = torch.cat([scale[p] for p in table[i]], dim=1)
        else:
            cache, scale = cache[i], scale[i]
        s = scale.double().repeat_interleave(block, dim=-1)[:, :cap]
        return cache.float().double() * s[..., None], s

    for step in range(12):
        t = [1, 1, 5, 40, 1, 33, 2, 1, 64, 1, 3, 1][step]
        news = torch.tensor([t, max(t - 2, 0), t // 2])
        size = math.exp(_q8.randn(1, seed=step).item())
        k, v = size * _q8.randn(b, h, t, d, seed=step + 1), _q8.randn(b, h, t, d, seed=step + 50)
        before = {n: [row(c, s, i)[1] for i in range(b)]
                  for n, c, s in (("k", kc, ks), ("v", vc, vs))}
        kv_cache_update_q8(k, v, kc, vc, ks, vs, lens, news, table if paged else None,
                           block_size=block)
        for name, x, c, s in (("k", k, kc, ks), ("v", v, vc, vs)):
            for i in range(b):
                n, m = int(lens[i]), min(int(news[i]), cap - int(lens[i]))
                want[name][i, :, n:n + m] = x[i, :, :m]
                got, sc = row(c, s, i)
                moved = (sc > before[name][i])[:, :n, None]
                if code == "int8":
                    bound[name][i, :, :n] += 0.5001 * moved * sc[:, :n, None]
                    bound[name][i, :, n:n + m] = 0.5001 * sc[:, n:n + m, None]
                else:
                    bound[name][i, :, :n] += moved * sc[:, :n, None] * 2.0 ** -10
                    bound[name][i, :, n:n + m] = torch.maximum(
                        x[i, :, :m].double().abs() * 2.0 ** -4, sc[:, n:n + m, None] * 2.0 ** -10)
                e = (got[:, :n + m] - want[name][i, :, :n + m].double()).abs()
                assert bool((e <= bound[name][i, :, :n + m]).all()), (step, name, i)
        lens = torch.minimum(lens + news, torch.tensor(cap))


def test_append_leaves_other_rows():
    """Rows behind the last token, other blocks' scales, skipped pages and tokens past
    the capacity."""
    kc = torch.randint(-100, 100, (3, 2, 64, 16), dtype=torch.int8)
    vc, ks, vs = kc.clone(), torch.rand(3, 2, 2), torch.rand(3, 2, 2)
    old = [x.clone() for x in (kc, vc, ks, vs)]
    k = _q8.randn(2, 2, 40, 16)
    table = torch.tensor([[1, 5], [-1, 2]])
    kv_cache_update_q8(k, k, kc, vc, ks, vs, torch.tensor([60, 60]), torch.tensor([40, 10]), table)
    # row 0: tokens 60..63 in page 1, the rest in a page outside the pool; row 1: 60..63
    # in page -1, 64..69 in page 2
    assert torch.equal(kc[0], old[0][0]) and torch.equal(ks[0], old[2][0])
    assert torch.equal(kc[1, :, :32], old[0][1, :, :32]) and torch.equal(ks[1, :, 0], old[2][1, :, 0])
    assert torch.equal(kc[2, :, 6:], old[0][2, :, 6:]) and torch.equal(vs[2, :, 1], old[3][2, :, 1])
    assert not torch.equal(kc[2, :, :6], old[0][2, :, :6])
    kc, ks = old[0].clone(), old[2].clone()
    kv_cache_update_q8(k, k, kc[:2], vc[:2], ks[:2], vs[:2], torch.tensor([64, 70]))
    assert torch.equal(kc, old[0]) and torch.equal(ks, old[2])


def test_append_non_finite():
    k = torch.ones(1, 1, 4, 16)
    k[0, 0, 1, 0], k[0, 0, 2, 0], k[0, 0, 3, 0] = math.inf, -math.inf, math.nan
    for code, top in (("int8", 127.0), ("e4m3", 448.0)):
        c = torch.zeros(1, 1, 32, 16, dtype=_q8.CODES[code])
        s = torch.zeros(1, 1, 1)
        kv_cache_update_q8(k, k, c, c.clone(), s, s.clone(), torch.tensor([0]))
        assert s.item() == needed_scale(torch.ones(1), c.dtype).item()
        got = c.float()[0, 0, :4, 0].tolist()
        assert got[1:3] == [top, -top] and (got[3] == 0 if code == "int8" else math.isnan(got[3]))


@pytest.mark.parametrize("b,width,page,max_new,spare", [
    (1, 1, 16, 1, 0), (7, 5, 16, 1, 3), (7, 5, 16, 40, 8), (40, 9, 32, 17, 4), (40, 9, 32, 100, 500),
    (5, 3, 1, 2, 2)])
def test_page_plan(b, width, page, max_new, spare):
    model = _q8.PlanModel(page, width, max_new)
    for seed in range(5):
        pages, lens, news, free, head, size = _q8.random_plan(b, width, page, max_new, spare, seed)
        table, ring, state = _q8.plan_tensors(pages, free, head, size, width, "cpu")
        args = (torch.tensor(lens), torch.tensor(news))
        want_slots, want_lens = model.step(pages, lens, news, free)
        got = kv_page_plan(table, *args, ring, state, page, max_new=max_new)
        _q8.check_plan(table, ring, got[2], got[0], got[1], pages, want_slots, want_lens, free)
        again = kv_page_plan(table, *args, ring, state, page, max_new=max_new)
        assert all(torch.equal(x, y) for x, y in zip(got, again))


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_reference(code, paged, causal):
    b, hq, hkv, sq, d, page = 4, 4, 2, 5, 32, 64
    shape = (9, hkv, page) if paged else (b, hkv, 150)
    kc, ks = _q8.make_cache(*shape, d, 32, code, seed=1)
    vc, vs = _q8.make_cache(*shape, d, 32, code, seed=2)
    table = [[3, 1, 8], [0, -1, 2], [99, 5, 6], [4, 7, 4]] if paged else None
    lens, q_lens = [150, 149, 3, 0], [5, 4, 5, 2]
    q = _q8.randn(b, hq, sq, d)
    want, tol = _q8.attention64(q, kc, vc, ks, vs, 32, lens, q_lens, table, causal, d ** -0.5)
    got = flash_attention_q8(q, kc, vc, ks, vs, causal, cache_seqlens=torch.tensor(lens),
                             block_table=None if table is None else torch.tensor(table),
                             query_lens=torch.tensor(q_lens))
    _q8.check_within(got, want, tol)


def _case(**kw):
    a = dict(q=torch.zeros(2, 4, 1, 32), k=torch.zeros(2, 2, 64, 32, dtype=torch.int8),
             v=torch.zeros(2, 2, 64, 32, dtype=torch.int8), k_scale=torch.ones(2, 2, 2),
             v_scale=torch.ones(2, 2, 2))
    a.update(kw)
    return a


@pytest.mark.parametrize("change,error,text", [
    (dict(k=torch.zeros(2, 2, 64, 32)), ValueError, "types differ"),
    (dict(k=torch.zeros(2, 2, 64, 32), v=torch.zeros(2, 2, 64, 32)), NotImplementedError, "cache dtype"),
    (dict(k_scale=torch.ones(2, 2, 3)), ValueError, "k_scale must have shape"),
    (dict(v_scale=torch.ones(2, 2, 2).half()), ValueError, "v_scale must be float32"),
    (dict(block_size=48), ValueError, "multiple of 32"),
    (dict(block_size=0), ValueError, "multiple of 32"),
    (dict(q=torch.zeros(2, 4, 1, 16)), ValueError, "Head dimension"),
    (dict(q=torch.zeros(2, 3, 1, 32)), ValueError, "divisible"),
    (dict(q=torch.zeros(3, 4, 1, 32)), ValueError, "Batch mismatch"),
    (dict(q=torch.zeros(2, 4, 32)), ValueError, "4D"),
    (dict(cache_seqlens=torch.ones(3, dtype=torch.int32)), ValueError, "cache_seqlens"),
    (dict(cache_seqlens=torch.ones(2)), ValueError, "integer"),
    (dict(block_table=torch.zeros(2, 1, dtype=torch.int32)), ValueError, "needs cache_seqlens"),
    (dict(block_table=torch.zeros(2, dtype=torch.int32), cache_seqlens=torch.ones(2, dtype=torch.int32)),
     ValueError, "max_pages"),
    (dict(q=torch.zeros(2, 4, 1, 32, requires_grad=True)), RuntimeError, "backward"),
    (dict(rope_cos=torch.zeros(4, 32)), ValueError, "both cos and sin"),
])
def test_attention_refusals(change, error, text):
    for fn in (flash_decode_q8, flash_attention_q8):
        with pytest.raises(error, match=text):
            fn(**_case(**change))


def test_more_refusals():
    with pytest.raises(AssertionError, match="q_len == 1"):
        flash_decode_q8(**_case(q=torch.zeros(2, 4, 2, 32)))
    with pytest.raises(ValueError, match="query_lens"):
        flash_attention_q8(**_case(), query_lens=torch.ones(1, dtype=torch.int32))
    wide = dict(q=torch.zeros(2, 4, 1, 24), k=torch.zeros(2, 2, 64, 24, dtype=torch.int8),
                v=torch.zeros(2, 2, 64, 24, dtype=torch.int8))
    with pytest.raises(NotImplementedError, match="multiple of 16"):
        flash_decode_q8(**_case(**wide))
    pool = dict(block_table=torch.zeros(2, 1, dtype=torch.int32),
                cache_seqlens=torch.ones(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="multiple of block_size"):
        flash_decode_q8(**_case(**pool), block_size=128)

    x = torch.zeros(2, 2, 3, 32)
    c, s = torch.zeros(2, 2, 64, 32, dtype=torch.int8), torch.ones(2, 2, 2)
    lens = torch.zeros(2, dtype=torch.int32)
    for bad, text in ((dict(k=x[0]), "4D"), (dict(v=x[:, :, :2]), "shapes differ"),
                      (dict(k=x[:, :1], v=x[:, :1]), "KV heads"),
                      (dict(new_lens=lens[:1]), "new_lens"), (dict(cache_seqlens=lens.float()), "integer")):
        a = dict(k=x, v=x, k_cache=c, v_cache=c, k_scale=s, v_scale=s, cache_seqlens=lens)
        a.update(bad)
        with pytest.raises(ValueError, match=text):
            kv_cache_update_q8(**a)

    table, ring = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(5, dtype=torch.int32)
    state = torch.tensor([0, 5], dtype=torch.int32)
    for bad, text in ((dict(block_table=table.long()), "int32"), (dict(free_pages=ring.long()), "int32"),
                      (dict(block_table=table.t()), "must have shape|contiguous"),
                      (dict(free_pages=ring[:0]), "at least one"), (dict(free_state=state[:1]), "free_state"),
                      (dict(block_table=table[:1].expand(2, 4)), "overlap"),
                      (dict(page_size=0), "positive"), (dict(max_new=-1), "negative")):
        a = dict(block_table=table, cache_seqlens=lens, new_lens=lens, free_pages=ring,
                 free_state=state, page_size=16)
        a.update(bad)
        with pytest.raises(ValueError, match=text):
            kv_page_plan(**a)
