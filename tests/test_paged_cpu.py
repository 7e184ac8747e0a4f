"""Argument checks of the batch operators (paged plan and append, paged and
packed attention): every refusal happens on the host, before a context is
needed, so they are tested without a GPU."""

import ctypes

import pytest

from rustllm_amd import abi

lib = abi.load()
NULL = ctypes.c_void_p()
ARGUMENT, SHAPE, MISMATCH, DTYPE, CONTIGUOUS, FORMAT, DEVICE = 1, 2, 3, 5, 6, 8, 9


def buf(n, es, addr=0x10000):
    return abi.RlBuffer(addr, n, n * es)


def call(name, *args):
    conv = [ctypes.byref(a) if isinstance(a, abi.RlBuffer) else a for a in args]
    return getattr(lib, name)(NULL, *conv), abi.last_error()


def u64s(*v):
    return (ctypes.c_uint64 * len(v))(*v)


def test_plan_validation():
    def go(s=3, blocks=4, pages=10, page=16, tokens=7, free=5, cached=None, fresh=None,
           table=None, offsets=None, context=None, slots=None, positions=None, taken=None):
        return call("rl_paged_plan", cached or buf(s, 4), fresh or buf(s, 4), s,
                    buf(free, 4) if isinstance(free, int) else free, table or buf(s * blocks, 4),
                    blocks, pages, page, offsets or buf(s + 1, 4), context or buf(s, 4), tokens,
                    slots or buf(tokens, 4), positions or buf(tokens, 4), taken or buf(1, 4))

    assert go()[0] == DEVICE
    assert go(free=0)[0] == DEVICE  # no free page is a state, not a mistake
    assert go(page=1)[0] == DEVICE and go(page=1 << 20)[0] == DEVICE
    for bad in (dict(s=0), dict(blocks=0), dict(tokens=0)):
        st, msg = go(**bad)
        assert st == SHAPE and "greater than zero" in msg
    st, msg = go(page=24)
    assert st == SHAPE and "power of two, got 24" in msg
    assert go(page=0)[0] == SHAPE and go(pages=0)[0] == SHAPE
    st, msg = go(pages=1 << 28)  # 2^28 pages of 16: slots would reach 2^32
    assert st == SHAPE and "u32 slots" in msg
    for name in ("cached", "fresh", "table", "offsets", "context", "slots", "positions", "taken"):
        st, msg = go(**{name: buf(2, 4)})
        assert st == SHAPE and "expected" in msg, name
        st, msg = go(**{name: buf(8, 2)})
        assert st == DTYPE and "U32" in msg, name
    assert go(free=buf(5, 2))[0] == DTYPE
    assert go(free=abi.RlBuffer(None, 5, 20))[0] == ARGUMENT
    st, msg = call("rl_paged_plan", *[None] * 2, 3, None, None, 4, 10, 16, None, None, 7, None,
                   None, None)
    assert st == ARGUMENT and "null" in msg


@pytest.mark.parametrize("dt,es", [("f32", 4), ("f16", 2)])
def test_append_validation(dt, es):
    t, qh, kvh = 5, 4, 2

    def go(d=8, q=None, k=None, v=None, rows=32, cos=None, sin=None, positions=None, slots=None,
           q_out=None, kp=None, vp=None, pages=3, page=4, lens=(None, None, None)):
        views = []
        for view, heads, n in zip((q, k, v), (qh, kvh, kvh), lens):
            dims, strides = view or ((t, heads, d), (heads * d, d, 1))
            views += [buf(t * heads * d if n is None else n, es), u64s(*dims), u64s(*strides)]
        return call(f"rl_qkv_rope_paged_append_{dt}", *views, cos or buf(rows * d // 2, 4),
                    sin or buf(rows * d // 2, 4), rows, positions or buf(t, 4),
                    slots or buf(t, 4), q_out or buf(t * qh * d, es),
                    kp or buf(pages * kvh * page * d, es), vp or buf(pages * kvh * page * d, es),
                    pages, page)

    assert go()[0] == DEVICE
    assert go(q=((t, qh, 8), (8, t * 8, 1)))[0] == DEVICE  # head-major rows
    st, msg = go(d=7)
    assert st == SHAPE and "even" in msg
    assert go(k=((t, 0, 8), (16, 8, 1)))[0] == SHAPE
    assert go(k=((t - 1, kvh, 8), (16, 8, 1)))[0] == MISMATCH
    assert go(k=((t, kvh, 4), (16, 8, 1)))[0] == MISMATCH
    assert go(v=((t, 1, 8), (16, 8, 1)))[0] == MISMATCH
    st, msg = go(q=((t, qh, 8), (64, 16, 2)), lens=(1 << 12, None, None))
    assert st == CONTIGUOUS and "unit innermost stride" in msg
    st, msg = go(lens=(None, t * kvh * 8 - 1, None))
    assert st == SHAPE and "reaches past the end" in msg
    assert go(cos=buf(32 * 4 - 1, 4))[0] == SHAPE
    assert go(sin=buf(32 * 4, 2))[0] == DTYPE
    assert go(rows=0)[0] == SHAPE
    assert go(positions=buf(t - 1, 4))[0] == SHAPE and go(slots=buf(t + 1, 4))[0] == SHAPE
    st, msg = go(page=12)
    assert st == SHAPE and "power of two" in msg
    st, msg = go(q_out=buf(3, es))
    assert st == SHAPE and "paged append output" in msg
    st, msg = go(kp=buf(3 * 2 * 4 * 8 - 8, es))
    assert st == SHAPE and "key pages buffer has 184 elements, expected [3, 2, 4, 8]" in msg
    assert go(vp=buf(8, es))[0] == SHAPE
    assert go(vp=abi.RlBuffer(0x1000, 192, 192 * 3))[0] == DTYPE


@pytest.mark.parametrize("dt,es", [("f32", 4), ("f16", 2)])
def test_paged_attention_validation(dt, es):
    def go(s=2, t=5, qh=6, kvh=2, d=64, pages=9, page=16, blocks=4, mq=3, mc=64, scale=0.125,
           q=None, kp=None, vp=None, table=None, offsets=None, context=None, ws=None, out=None):
        pool = pages * kvh * page * d
        return call(f"rl_paged_attention_{dt}", q or buf(t * qh * d, es), kp or buf(pool, es),
                    vp or buf(pool, es), table or buf(s * blocks, 4), offsets or buf(s + 1, 4),
                    context or buf(s, 4), s, t, qh, kvh, d, pages, page, blocks, mq, mc,
                    ctypes.c_float(scale), ws or buf(1 << 20, 1), out or buf(t * qh * d, es))

    assert go()[0] == DEVICE
    assert go(d=48)[0] == DEVICE and go(d=512)[0] == DEVICE and go(page=1, mc=4)[0] == DEVICE
    for bad in (dict(s=0), dict(t=0), dict(qh=0), dict(d=0), dict(mq=0), dict(mc=0),
                dict(blocks=0)):
        st, msg = go(**bad)
        assert st == SHAPE and "greater than zero" in msg, bad
    st, msg = go(kvh=4)
    assert st == FORMAT and "Q heads 6 must be divisible by non-zero KV heads 4" in msg
    assert go(kvh=0)[0] == FORMAT
    st, msg = go(d=520)
    assert st == SHAPE and "head size 520 exceeds 512" in msg
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        st, msg = go(scale=scale)
        assert st == SHAPE and "positive and finite" in msg
    st, msg = go(mc=65)
    assert st == SHAPE and "exceeds a table row" in msg
    st, msg = go(t=1 << 31, qh=2, kvh=2)
    assert st == SHAPE and "exceed one launch" in msg
    st, msg = go(pages=1 << 29, page=16)
    assert st == SHAPE and "u32 slots" in msg
    st, msg = go(s=1 << 22, kvh=2)
    assert st == SHAPE and "exceed one launch" in msg
    st, msg = go(s=1, t=127, qh=1 << 22, kvh=1 << 22, d=1)  # rows alone and heads alone would fit
    assert st == SHAPE and "exceed one launch" in msg
    st, msg = go(s=1 << 31, qh=1 << 29, kvh=1 << 29, t=1, d=1)
    assert st == SHAPE and "exceed one launch" in msg
    st, msg = go(mc=1 << 31, blocks=1 << 28)
    assert st == SHAPE and "key range exceeds" in msg
    assert go(page=20)[0] == SHAPE
    for name in ("q", "kp", "vp", "out"):
        assert go(**{name: buf(7, es)})[0] == SHAPE, name
    for name in ("q", "kp", "vp"):
        assert go(**{name: abi.RlBuffer(0x1000, 8, 24)})[0] == DTYPE, name
    for name in ("table", "offsets", "context"):
        assert go(**{name: buf(1, 4)})[0] == SHAPE, name
        assert go(**{name: buf(8, 2)})[0] == DTYPE, name
    st, msg = go(ws=abi.RlBuffer(None, 8, 8))
    assert st == ARGUMENT and "workspace" in msg


@pytest.mark.parametrize("dt,es", [("f32", 4), ("f16", 2)])
def test_packed_attention_validation(dt, es):
    t, qh, kvh = 9, 6, 2

    def go(d=64, s=3, mq=5, scale=0.125, q=None, k=None, v=None, lens=(None, None, None),
           offsets=None, out=None):
        views = []
        for view, heads, n in zip((q, k, v), (qh, kvh, kvh), lens):
            dims, strides = view or ((t, heads, d), (heads * d, d, 1))
            views += [buf(t * heads * d if n is None else n, es), u64s(*dims), u64s(*strides)]
        return call(f"rl_packed_attention_{dt}", *views, offsets or buf(s + 1, 4), s, mq,
                    ctypes.c_float(scale), out or buf(t * qh * d, es))

    assert go()[0] == DEVICE
    assert go(s=0)[0] == SHAPE and go(mq=0)[0] == SHAPE
    assert go(k=((t, 4, 64), (128, 64, 1)), v=((t, 4, 64), (128, 64, 1)),
              lens=(None, 4096, 4096))[0] == FORMAT
    assert go(k=((t, kvh, 32), (128, 64, 1)))[0] == MISMATCH
    assert go(v=((t - 1, kvh, 64), (128, 64, 1)))[0] == MISMATCH
    assert go(q=((t, qh, 64), (qh * 64, 64, 0)))[0] == CONTIGUOUS
    st, msg = go(lens=(None, None, t * kvh * 64 - 1))
    assert st == SHAPE and "reaches past the end" in msg
    assert go(scale=0.0)[0] == SHAPE
    assert go(offsets=buf(3, 4))[0] == SHAPE and go(offsets=buf(4, 2))[0] == DTYPE
    assert go(out=buf(3, es))[0] == SHAPE
    most = (1 << 64) - 1  # extents whose sum passes 2^128 by six
    st, msg = go(q=((most, 4, 8), (most, most, 1)), lens=(4096, None, None))
    assert st == SHAPE and "reaches past the end" in msg
    st, msg = call(f"rl_packed_attention_{dt}", buf(8, es), None, None, buf(8, es), None, None,
                   buf(8, es), None, None, buf(4, 4), 3, 5, ctypes.c_float(1.0), buf(8, es))
    assert st == ARGUMENT and "null" in msg


def test_workspace_validation():
    out = abi.RlBuffer()
    st, _ = call("rl_paged_attention_workspace", 4, 2, out)
    assert st == DEVICE and not out.data
    assert call("rl_paged_attention_workspace", 0, 2, out)[0] == SHAPE
    assert call("rl_paged_attention_workspace", 4, 0, out)[0] != DEVICE
    assert call("rl_paged_attention_workspace", 1 << 22, 2, out)[0] == SHAPE
    assert lib.rl_paged_attention_workspace(NULL, 4, 2, None) == ARGUMENT
