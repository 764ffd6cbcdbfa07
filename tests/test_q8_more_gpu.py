"""GPU tests of the 8-bit cache under less usual calls: every number of column blocks,
blocks with infinities past what a workgroup keeps, host threads and graphs at once,
a row longer than 2^31 bytes, and refusals of the launchers."""

import math
import threading

import pytest
import torch

from stackkernels_amd.torch import (
    flash_attention_q8,
    flash_decode_q8,
    kv_cache_update_q8,
    kv_page_plan,
)

import _q8
from test_q8_gpu import _append_both, _attend, i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("rows", [16, 17, 32, 33, 47, 48, 49, 64])
def test_column_blocks(device, code, d, rows):
    """One to four blocks of 16 rows, whole and split, ragged and paged."""
    _attend(torch.bfloat16, code, rows, 1, 1, d, 32, 32, [500, 260, 255, 1, 0], causal=False, splits=3)
    _attend(torch.float16, code, rows, 1, 1, d, 32, 0, [700, 300])


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("d,rows,sq", [(64, 1, 1), (64, 40, 1), (64, 64, 1), (128, 8, 3), (128, 33, 1),
                                       (128, 60, 1), (128, 4, 40), (64, 2, 70), (256, 8, 5)])
def test_rotated_fp16_queries_keep_their_precision(device, monkeypatch, code, d, rows, sq):
    """Rotated fp16 queries enter the scores with 22 bits: the bound counts no rounding
    of theirs (a rotation's own roundings, three of 2^-24, are among the D + 16 of
    2^-23 that it counts for a score)."""
    bound = _q8.attention64
    monkeypatch.setattr(_q8, "attention64", lambda *a: bound(*a[:-1], False))
    _attend(torch.float16, code, rows, 1, sq, d, 32, 64, [300, 140, 77], rope=True)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("rope", [False, True])
@pytest.mark.parametrize("token", [0, 300, 505])
def test_append_not_finite_anywhere(device, code, rope, token):
    """One infinity or NaN among values that a workgroup keeps, and among those that
    it reads again."""
    def values(k, v):
        k[0, token % 40, 1, 3], v[0, 1, token % 40, 200] = math.inf, math.nan
        k[1, token, 0, 130], v[1, 0, token, 0] = -math.inf, -math.inf
        k[2, token, 1, 255], v[2, 1, token, 255] = math.nan, math.inf

    for dtype in (torch.bfloat16, torch.float32):
        _append_both(dtype, code, 256, 512, False, 510, [0, 1, 300], None, rope=rope, values=values,
                     cap=1024)
        _append_both(dtype, code, 256, 32, True, 510, [0, 1, 300], [40, 510, 509], rope=rope,
                     values=values, cap=1024)


@pytest.mark.parametrize("b,hkv", [(1, 1), (3, 1), (5, 3), (9, 2)])
def test_append_few_blocks(device, b, hkv):
    """Numbers of blocks that are no multiple of the XCDs."""
    for t in (1, 33, 70):
        _append_both(torch.bfloat16, "int8", 64, 32, False, t, [7 * i for i in range(b)], None, hkv=hkv)


def _job(seed, hq, hkv, sq, d, code, page, dtype):
    """A server's step on a cache of its own: the cache's bytes and the output."""
    b, block, cap = 6, 32, 1024
    lens = torch.randint(0, cap - 64, (b,), generator=torch.Generator().manual_seed(seed)).tolist()
    table = None
    shape = (b, hkv, cap)
    if page:
        width = cap // page
        table = torch.randperm(b * width, generator=torch.Generator().manual_seed(seed)).view(b, width)
        table = table.int().cuda()
        shape = (b * width, hkv, page)
    kc, ks = (x.cuda() for x in _q8.make_cache(*shape, d, block, code, seed=seed))
    vc, vs = (x.cuda() for x in _q8.make_cache(*shape, d, block, code, seed=seed + 1))
    q = _q8.randn(b, hq, sq, d, seed=seed).to(dtype).cuda()
    k, v = (_q8.randn(b, hkv, sq, d, seed=seed + i).to(dtype).cuda() for i in (2, 3))
    held = i32(lens)

    def run():
        mine = [x.clone() for x in (kc, vc, ks, vs)]
        kv_cache_update_q8(k, v, *mine, held, None, table)
        out = flash_attention_q8(q, *mine, True, None, held + sq, table)
        return (out, *(x.view(torch.uint8) for x in mine))

    return run


JOBS = [
    (10, 8, 2, 1, 128, "int8", 64, torch.bfloat16),
    (20, 32, 1, 2, 64, "e4m3", 0, torch.float16),
    (30, 8, 8, 40, 128, "e4m3", 32, torch.bfloat16),
    (40, 4, 4, 3, 256, "int8", 0, torch.float32),
    (50, 16, 2, 33, 64, "int8", 128, torch.float16),
]


def test_concurrent_threads_and_streams(device):
    """Calls from several host threads, each on its own stream, share nothing."""
    jobs = [_job(*j) for j in JOBS]
    expect = [job() for job in jobs]
    torch.cuda.synchronize()
    got, errors = [[] for _ in jobs], []
    start = threading.Barrier(len(jobs))

    def worker(i):
        try:
            stream = torch.cuda.Stream()
            start.wait()
            with torch.cuda.stream(stream):
                for _ in range(4):
                    got[i].append(jobs[i]())
            stream.synchronize()
        except Exception as e:  # noqa: BLE001 -- reported by the main thread
            errors.append(f"{i}: {e!r}")

    threads = [threading.Thread(target=worker, args=(i,)) for i in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=100)
    assert not errors and not any(t.is_alive() for t in threads)
    for want, runs in zip(expect, got):
        assert len(runs) == 4
        for run in runs:
            assert all(torch.equal(x, y) for x, y in zip(want, run))


def test_two_graphs_at_once(device):
    """Two captured steps replayed side by side, several times, with eager work and
    synchronizations between: each has its workspace to itself."""
    jobs = [_job(*j) for j in JOBS[:2]]
    expect = [job() for job in jobs]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for job in jobs:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            job()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(job())
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for i in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        if i % 2:
            jobs[i % len(jobs)]()
        torch.cuda.synchronize()
        for want, out in zip(expect, outs):
            assert all(torch.equal(x, y) for x, y in zip(want, out)), i
            for x in out:
                x.zero_()
        torch.cuda.synchronize()


def test_row_past_two_gibibytes(device):
    """The last keys of a contiguous row of more than 2^31 bytes of codes.  All keys
    before them have a score of 0 and values of 0: with scores of 50 and more behind
    them they weigh less than 1.7e7 e^-50 < 4e-15 of the sum."""
    d, tail = 128, 100
    s = (1 << 31) // d + 4096 + 13
    k = torch.zeros(1, 1, s, d, dtype=torch.int8, device="cuda")
    v = torch.zeros_like(k)
    g = torch.Generator().manual_seed(1)
    kt = torch.randint(60, 90, (tail, d), generator=g).to(torch.int8)
    vt = torch.randint(-127, 128, (tail, d), generator=g).to(torch.int8)
    k[0, 0, -tail:], v[0, 0, -tail:] = kt.cuda(), vt.cuda()
    scale = torch.full((1, 1, -(-s // 32)), 1 / 128, device="cuda")
    q = torch.ones(1, 2, 1, d, dtype=torch.bfloat16)
    got = flash_decode_q8(q.cuda(), k, v, scale, scale, 1.0)
    small = torch.full((1, 1, 4), 1 / 128)
    want, tol = _q8.attention64(q, kt[None, None], vt[None, None], small, small, 32, [tail], [1], None,
                                False, 1.0, splits=256, dtype=torch.bfloat16)
    _q8.check_within(got, want, tol + 4e-15)
    new = _q8.randn(1, 1, 3, d).bfloat16().cuda()
    kv_cache_update_q8(new, new, k, v, scale, scale, i32([s - 3]))
    assert bool((k[0, 0, -3:] != 0).any(-1).all()) and not bool(k[0, 0, :4096].any())
    assert torch.equal(k[0, 0, -3:], v[0, 0, -3:])


def test_launcher_refusals(device):
    kc, ks = (x.cuda() for x in _q8.make_cache(2, 2, 64, 64, 32, "int8"))
    q = torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16, device="cuda")
    new = q[:, :2]
    with pytest.raises(ValueError, match="different devices"):
        flash_decode_q8(q, kc, kc.cpu(), ks, ks)
    with pytest.raises(ValueError, match="different devices"):
        kv_cache_update_q8(new, new, kc, kc.clone(), ks, ks.cpu(), i32([0, 0]))
    with pytest.raises(NotImplementedError, match="dtype"):
        flash_decode_q8(q.double(), kc, kc, ks, ks)
    shared = kc[:1].expand(2, 2, 64, 64)
    with pytest.raises(ValueError, match="overlap"):
        kv_cache_update_q8(new, new, shared, shared, ks, ks.clone(), i32([0, 0]))
    flash_decode_q8(q, shared, shared, ks, ks)  # (reading is fine)
    with pytest.raises(ValueError, match="16"):
        flash_decode_q8(q, kc.transpose(2, 3), kc.transpose(2, 3), ks, ks)
    with pytest.raises(RuntimeError, match="one ROCm device"):
        kv_page_plan(i32([[0, 1]]), i32([0]), i32([1]), torch.zeros(4, dtype=torch.int32), i32([0, 4]), 32)
    q.requires_grad_(True)
    with pytest.raises(RuntimeError, match="no backward"):
        flash_decode_q8(q, kc, kc, ks, ks)
