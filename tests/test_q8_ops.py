"""The 8-bit cache's C entry points refuse bad arguments before a launch (their
pointers here are no device memory), and its torch.library ops trace."""

import ctypes
import os

import pytest
import torch

import stackkernels_amd.torch  # noqa: F401  (registers the ops)
from stackkernels_amd.torch import flash_attention_q8, kv_cache_update_q8

import _q8


@pytest.fixture(scope="module")
def lib():
    from stackkernels_amd._core.attention import _lib
    from stackkernels_amd.csrc import build

    if not os.path.exists(_lib.LIB_PATH):
        build.build()
    return _lib.load()


SIZES = dict(dtype=2, code=3, b=2, hq=4, hkv=2, s=3, units=2, rows=128, pages=0, block=32, d=64,
             causal=0)
NO_ROPE = (None, None, 0, 0, 0, None, 0)


def _shape(strides, **kw):
    from stackkernels_amd._core.attention import _lib

    x = dict(SIZES, **kw)
    st = dict(x0=(2048, 512, 64), x1=(2048, 512, 64), k=(16384, 8192, 64), v=(16384, 8192, 64),
              ks=(8, 4, 1), vs=(8, 4, 1))
    st.update(strides or {})
    return _lib.q8_shape(tuple(x[n] for n in SIZES),
                         (st["x0"], st["x1"], st["k"], st["v"], st["ks"], st["vs"]))


SHAPE_REFUSALS = [
    (dict(dtype=7), "dtype"),
    (dict(code=0), "code type"),
    (dict(b=-1), "invalid sizes"),
    (dict(hkv=0), "invalid sizes"),
    (dict(d=72), "multiple of 16"),
    (dict(d=272), "multiple of 16"),
    (dict(block=16), "block_size"),
    (dict(block=0), "block_size"),
    (dict(block=(1 << 24) + 32), "block_size"),
    (dict(units=3), "contiguous cache"),
    (dict(pages=4, units=9, rows=80), "page_size"),
    (dict(pages=4, units=0, rows=64), "pool"),
    (dict(pages=1 << 26, units=9, rows=64), "overflows"),
    (dict(rows=0x7fffffff), "too long"),
    (dict(strides=dict(k=(16384, 8192, 72))), "multiple of 16"),
    (dict(strides=dict(v=(-16384, 8192, 64))), "non-negative"),
    (dict(strides=dict(k=(16384, 8192, 48))), "less than the head dim"),
    (dict(strides=dict(k=(16384, 8192, 1 << 24))), "too large"),
    (dict(strides=dict(ks=(-8, 4, 1))), "non-negative"),
    (dict(strides=dict(vs=(1 << 32, 4, 1))), "too large"),
    (dict(strides=dict(x0=(2048, 512, 63))), "stride"),
]


@pytest.mark.parametrize("kw,text", SHAPE_REFUSALS)
def test_shapes_refused(lib, kw, text):
    from stackkernels_amd._core.attention import _lib

    kw = dict(kw)
    shape = _shape(kw.pop("strides", None), **kw)
    table = 16 if kw.get("pages") else None
    rc = lib.sk_attn_q8(shape, 16, 16, 16, 16, 16, 16, None, 0, 1, table, 16, None, *NO_ROPE, 0.125,
                        None)
    assert rc in (_lib.SK_EINVAL, _lib.SK_EUNSUPPORTED) and text in _lib.last_error()
    rc = lib.sk_kv_cache_update_q8(shape, 16, 16, 16, 16, 16, 16, 16, None, table, *NO_ROPE, None)
    assert rc in (_lib.SK_EINVAL, _lib.SK_EUNSUPPORTED) and text in _lib.last_error()


@pytest.mark.parametrize("strides", [
    dict(k=(16384, 8192, 0)), dict(v=(16384, 0, 64)), dict(k=(0, 8192, 64)),
    dict(ks=(8, 4, 0)), dict(vs=(8, 0, 1)), dict(vs=(0, 4, 1))])
def test_append_refuses_shared_rows(lib, strides):
    """A cache whose rows or scales are one and the same can be read, not written."""
    from stackkernels_amd._core.attention import _lib

    rc = lib.sk_kv_cache_update_q8(_shape(strides), 16, 16, 16, 16, 16, 16, 16, None, None, *NO_ROPE,
                                   None)
    assert rc == _lib.SK_EINVAL and "overlap" in _lib.last_error()


def test_append_argument_errors(lib):
    from stackkernels_amd._core.attention import _lib

    def upd(k=16, kc=16, ks=16, lens=16, table=None, rope=NO_ROPE, **kw):
        return lib.sk_kv_cache_update_q8(_shape(None, **kw), k, 16, kc, 16, ks, 16, lens, None, table,
                                         *rope, None)

    assert upd(k=None) == _lib.SK_EINVAL and "k" in _lib.last_error()
    assert upd(k=24) == _lib.SK_EINVAL
    assert upd(kc=None) == _lib.SK_EINVAL and "k_cache" in _lib.last_error()
    assert upd(ks=None) == _lib.SK_EINVAL and "k_scale" in _lib.last_error()
    assert upd(lens=None) == _lib.SK_EINVAL and "cache_seqlens" in _lib.last_error()
    assert upd(pages=4, rows=64, units=9) == _lib.SK_EINVAL and "block_table" in _lib.last_error()
    assert upd(rope=(16, None, 0, 128, 64, None, 0)) == _lib.SK_EINVAL
    assert upd(rope=(16, 16, 0, 128, 64, None, 126)) == _lib.SK_EINVAL  # token 2 past the table
    assert lib.sk_kv_cache_update_q8(None, 16, 16, 16, 16, 16, 16, 16, None, None, *NO_ROPE,
                                     None) == _lib.SK_EINVAL
    assert upd(s=0) == _lib.SK_OK  # nothing to write: no launch
    assert upd(b=0, units=0) == _lib.SK_OK


def test_attention_argument_errors(lib):
    from stackkernels_amd._core.attention import _lib

    def att(q=16, kc=16, vs=16, ws=None, nb=0, ns=1, table=None, lens=16, **kw):
        return lib.sk_attn_q8(_shape(None, **kw), q, kc, 16, 16, vs, 16, ws, nb, ns, table, lens, None,
                              *NO_ROPE, 0.125, None)

    assert att(q=None) == _lib.SK_EINVAL and "q" in _lib.last_error()
    assert att(kc=None) == _lib.SK_EINVAL and "k_cache" in _lib.last_error()
    assert att(vs=None) == _lib.SK_EINVAL and "v_scale" in _lib.last_error()
    assert att(hq=3) != _lib.SK_OK
    assert att(ns=257) == _lib.SK_EINVAL and "num_splits" in _lib.last_error()
    assert att(ns=-1) == _lib.SK_EINVAL
    need = 2 * 4 * 3 * 4 * (64 + 1) * 4  # rows x splits x (columns + 1) floats
    assert att(ns=4) == _lib.SK_EWORKSPACE
    assert att(ns=4, ws=16, nb=need - 1) == _lib.SK_EWORKSPACE and "needed" in _lib.last_error()
    assert att(ns=4, ws=24, nb=need) == _lib.SK_EWORKSPACE
    paged = dict(pages=4, rows=64, units=9)
    assert att(**paged) == _lib.SK_EINVAL and "block_table" in _lib.last_error()
    assert att(table=16, lens=None, **paged) == _lib.SK_EINVAL
    assert att(s=0) == _lib.SK_OK
    assert att(b=0, units=0) == _lib.SK_OK


def test_plan_of_empty_shapes(lib):
    """No division by a size of zero, one split, no workspace."""
    for dims in ((2, 2, 4, 2, 0, 100, 64), (0, 0, 4, 2, 0, 0, 64), (1, 2, 4, 2, 1, 0, 128),
                 (2, 0, 4, 2, 5, 100, 256)):
        ns, nb = ctypes.c_int(-1), ctypes.c_size_t(1)
        assert lib.sk_attn_q8_plan(*dims, 0, ctypes.byref(ns), ctypes.byref(nb)) == 0
        assert ns.value == 1 and nb.value == 0


def test_plan_of_the_longest_caches(lib):
    """A hundred million keys and 2^31 - 2^16 of them: no count overflows, and one row's
    many keys are shared out."""
    for dtype, sq in ((2, 1), (2, 100), (0, 1), (1, 40)):
        for sk in (100_000_000, 0x7fff0000):
            ns, nb = ctypes.c_int(-1), ctypes.c_size_t(0)
            assert lib.sk_attn_q8_plan(dtype, 1, 8, 1, sq, sk, 128, 1, ctypes.byref(ns),
                                       ctypes.byref(nb)) == 0
            assert 16 <= ns.value <= 256


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("d", [16, 64, 128, 256])
def test_plan_splits_fit(lib, dtype, d):
    """Every shape's plan is one that the call accepts, with keys for each split."""
    for b in (1, 7, 64):
        for hq, hkv in ((8, 8), (32, 8), (64, 1)):
            for sq in (1, 5, 300):
                for sk in (1, 31, 1000, 131072):
                    ns, nb = ctypes.c_int(-1), ctypes.c_size_t(1)
                    assert lib.sk_attn_q8_plan(dtype, b, hq, hkv, sq, sk, d, 1, ctypes.byref(ns),
                                               ctypes.byref(nb)) == 0
                    assert 1 <= ns.value <= max(1, (sk + 31) // 32)
                    columns = 64 if d <= 64 else 128 if d <= 128 else 256
                    want = b * hq * sq * ns.value * (columns + 1) * 4 if ns.value > 1 else 0
                    assert nb.value == want


def test_page_plan_argument_errors(lib):
    from stackkernels_amd._core.attention import _lib

    def plan(B=2, pages=4, stride=4, size=32, T=1, n=9, ptrs=(16, 32, 48, 64, 80, 96, 1024, 2048)):
        return lib.sk_kv_page_plan(*ptrs, B, pages, stride, size, T, n, None)

    assert plan(B=-1) == _lib.SK_EINVAL
    assert plan(size=0) == _lib.SK_EINVAL and "page_size" in _lib.last_error()
    assert plan(n=0) == _lib.SK_EINVAL and "free_pages" in _lib.last_error()
    assert plan(stride=3) == _lib.SK_EINVAL and "stride" in _lib.last_error()
    assert plan(pages=1 << 20, stride=1 << 20, size=4096) == _lib.SK_EINVAL
    for i in range(8):
        ptrs = [16, 32, 48, 64, 80, 96, 1024, 2048]
        ptrs[i] = None
        assert plan(ptrs=ptrs) == _lib.SK_EINVAL and "NULL" in _lib.last_error()
    assert plan(ptrs=(16, 32, 48, 64, 80, 96, 32, 2048)) == _lib.SK_EINVAL  # lengths in place
    assert plan(ptrs=(16, 32, 48, 64, 80, 96, 1024, 80)) == _lib.SK_EINVAL  # state in place
    assert plan(B=0) == _lib.SK_OK


def test_build_refuses_spills():
    """The kernel of few rows counts its loads: a build that spills is refused."""
    from stackkernels_amd.csrc import build

    text = "Function Name: _ZN2sk14q8_attn_kernelI\n ScratchSize [bytes/lane]: %d"
    build._check_no_scratch("sk_attn_q8.hip", text % 0)
    with pytest.raises(RuntimeError, match="spills 8 bytes"):
        build._check_no_scratch("sk_attn_q8.hip", text % 8)


def _inputs(code, seed=0):
    kc, ks = _q8.make_cache(2, 2, 96, 32, 32, code, seed)
    vc, vs = _q8.make_cache(2, 2, 96, 32, 32, code, seed + 1)
    return kc, vc, ks, vs


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_ops_match_calls(code):
    kc, vc, ks, vs = _inputs(code)
    lens, new = torch.tensor([40, 7]), torch.tensor([5, 3])
    k, v = _q8.randn(2, 2, 5, 32), _q8.randn(2, 2, 5, 32, seed=1)
    cos, sin = _q8.randn(100, 32, seed=3), _q8.randn(100, 32, seed=4)
    mine = [t.clone() for t in (kc, vc, ks, vs)]
    kv_cache_update_q8(k, v, *mine, lens, new, rope_cos=cos, rope_sin=sin, start_pos=lens)
    theirs = [t.clone() for t in (kc, vc, ks, vs)]
    torch.ops.stackkernels_amd.kv_cache_update_q8(k, v, *theirs, lens, new, None, 32, cos, sin, lens, 0)
    for x, y in zip(mine, theirs):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    q = _q8.randn(2, 4, 5, 32, seed=2)
    want = flash_attention_q8(q, *mine, True, 0.2, lens + new, None, new, rope_cos=cos, rope_sin=sin,
                              start_pos=3)
    got = torch.ops.stackkernels_amd.attention_q8(q, *mine, True, 0.2, lens + new, None, new, 32, cos,
                                                  sin, None, 3)
    assert torch.equal(want, got)


def test_ops_compile():
    """A step of append and attention in one graph, and opcheck on both ops."""
    lens = torch.tensor([40, 7])
    ops = torch.ops.stackkernels_amd

    def step(k, v, q, kc, vc, ks, vs):
        ops.kv_cache_update_q8(k, v, kc, vc, ks, vs, lens, None, None, 32, None, None, None, 0)
        return ops.attention_q8(q, kc, vc, ks, vs, True, 0.2, lens + 1, None, None, 32, None, None,
                                None, 0)

    k, v, q = _q8.randn(2, 2, 1, 32), _q8.randn(2, 2, 1, 32, seed=1), _q8.randn(2, 4, 1, 32, seed=2)
    mine, theirs = _inputs("int8"), _inputs("int8")
    want = step(k, v, q, *mine)
    got = torch.compile(step, backend="aot_eager", fullgraph=True)(k, v, q, *theirs)
    assert torch.equal(want, got)
    for x, y in zip(mine, theirs):
        assert torch.equal(x, y)
    cache = _inputs("int8")
    torch.library.opcheck(ops.attention_q8, (q, *cache, True, 0.2, lens, None, None, 32, None, None,
                                             None, 0))
    torch.library.opcheck(ops.kv_cache_update_q8, (k, v, *cache, lens, None, None, 32, None, None, None,
                                                   0))
