"""Rotary, cache and one-token attention entry points without a GPU: refusals before any HIP call, and the frequencies."""
import math

import numpy as np
import pytest

P16, P8, P2 = 0x1000, 0x1008, 0x1002
OK, NULL, SHAPE, ALIGN, WORKSPACE = 0, 1, 2, 3, 9


@pytest.fixture(scope="module")
def lib():
    from machx_inference_engine_amd import _lib
    return _lib.load(), _lib.parse_header()


class Call:
    """A valid call's arguments by name; `with_(...)` replaces some and gives the status.  Nothing here reaches the GPU: every one of them is refused."""

    def __init__(self, lib, name, **values):
        self.fn, self.names, self.values = getattr(lib[0], name), [n for n, _ in lib[1][name][1]], values

    def with_(self, **other):
        v = {**self.values, **other}
        assert set(other) <= set(self.names), other
        return self.fn(*[v[n] if n in v else (None if n == "s" else P16) for n in self.names])


HEADS = dict(T=4, Hq=32, Hkv=8, D=128, q_stride=4096, k_stride=1024, v_stride=1024, q_out_stride=4096, n_rot=128, interleaved=0, mscale=1.0, n_pages=10, page_size=16)


def test_rope_refusals(lib):
    c = Call(lib, "mx_rope", T=4, n_heads=8, D=128, x_stride=1024, y_stride=1024, n_rot=128, interleaved=0, mscale=1.0)
    for p in ("x", "y", "positions", "freqs"):
        assert c.with_(**{p: None}) == NULL, p
    for bad in (dict(T=0), dict(n_heads=0), dict(D=0), dict(D=120), dict(D=272), dict(n_rot=0), dict(n_rot=144), dict(n_rot=24), dict(x_stride=1020), dict(x_stride=1016),
                dict(y_stride=1016), dict(T=1 << 31, n_heads=65535)):
        assert c.with_(**bad) == SHAPE, bad
    for bad in (dict(x=P8), dict(y=P8), dict(positions=P2), dict(freqs=0x1004)):
        assert c.with_(**bad) == ALIGN, bad


@pytest.mark.parametrize("fmt", ["f16", "q8_0"])
def test_write_refusals(lib, fmt):
    planes = ("k_cache", "v_cache") if fmt == "f16" else ("k_qs", "k_d", "v_qs", "v_d")
    c = Call(lib, "mx_rope_kv_write_" + fmt, **HEADS)
    for p in ("q", "k", "v", "q_out", "positions", "slots", "freqs") + planes:
        assert c.with_(**{p: None}) == NULL, p
    for bad in (dict(T=0), dict(Hq=0), dict(Hkv=0), dict(D=0), dict(D=264, n_rot=16), dict(D=120), dict(n_rot=8), dict(n_rot=130), dict(q_stride=4088), dict(k_stride=1016),
                dict(v_stride=1025), dict(q_out_stride=8), dict(n_pages=0), dict(page_size=0), dict(page_size=24), dict(page_size=8), dict(n_pages=1 << 27, page_size=16)):
        assert c.with_(**bad) == SHAPE, bad
    for bad in (dict(q=P8), dict(k=P8), dict(v=P2), dict(q_out=P8), dict(slots=P2), dict(positions=0x1001), dict(freqs=0x1004)) + tuple({p: 0x1001} for p in planes):
        assert c.with_(**bad) == ALIGN, bad
    w = Call(lib, "mx_kv_write_" + fmt, **HEADS)
    for p in ("k", "v", "slots") + planes:
        assert w.with_(**{p: None}) == NULL, p
    assert w.with_(T=0) == SHAPE and w.with_(k_stride=1000) == SHAPE and w.with_(page_size=17) == SHAPE
    if fmt == "q8_0":
        assert c.with_(D=112, n_rot=16) == SHAPE and w.with_(D=80) == SHAPE


@pytest.mark.parametrize("fmt", ["f16", "q8_0"])
def test_launches_of_too_many_threads(lib, fmt):
    r = Call(lib, "mx_rope", T=1 << 26, n_heads=8, D=128, x_stride=1024, y_stride=1024, n_rot=128, interleaved=0, mscale=1.0)
    assert r.with_() == r.with_(T=0xFFFFFFFF) == r.with_(n_heads=1, D=16, n_rot=16, T=1 << 31) == SHAPE
    c, w = Call(lib, "mx_rope_kv_write_" + fmt, **HEADS), Call(lib, "mx_kv_write_" + fmt, **HEADS)
    for bad in (dict(T=1 << 26), dict(T=0xFFFFFFFF), dict(T=1 << 26, D=96)):
        assert c.with_(n_rot=96, **bad) == w.with_(**bad) == SHAPE, bad
    if fmt == "q8_0":                                          # three workgroups a token
        assert c.with_(T=1 << 23, D=96, n_rot=96) == SHAPE
    k = Call(lib, "mx_kv_read_" + fmt, max_pages=4, total_rows=1 << 28, B=1, Hkv=8, D=128, n_pages=10, page_size=16)
    assert k.with_() == k.with_(total_rows=1 << 27, B=1 << 23) == SHAPE
    a = Call(lib, "mx_attn_decode_" + fmt, q_stride=1 << 20, max_pages=4, B=65535, Hq=8192, Hkv=1, D=128, n_pages=10, page_size=16, max_len=2048, window=0, scale=0.1, out_q8=None,
             ws_bytes=1 << 60)
    assert a.with_() == a.with_(Hq=2048, Hkv=2048) == SHAPE


@pytest.mark.parametrize("fmt", ["f16", "q8_0"])
def test_read_refusals(lib, fmt):
    planes = ("k_cache", "v_cache") if fmt == "f16" else ("k_qs", "k_d", "v_qs", "v_d")
    c = Call(lib, "mx_kv_read_" + fmt, max_pages=4, total_rows=60, B=2, Hkv=8, D=128, n_pages=10, page_size=16)
    for p in ("page_table", "rows", "k_out", "v_out") + planes:
        assert c.with_(**{p: None}) == NULL, p
    for bad in (dict(max_pages=0), dict(total_rows=0), dict(total_rows=1 << 31), dict(B=0), dict(B=(1 << 24) + 1), dict(Hkv=0), dict(D=40), dict(n_pages=0), dict(page_size=20)):
        assert c.with_(**bad) == SHAPE, bad
    for bad in (dict(page_table=P2), dict(rows=P2), dict(k_out=P8), dict(v_out=P8)):
        assert c.with_(**bad) == ALIGN, bad


@pytest.mark.parametrize("fmt", ["f16", "q8_0"])
def test_attention_refusals(lib, fmt):
    planes = ("k_cache", "v_cache") if fmt == "f16" else ("k_qs", "k_d", "v_qs", "v_d")
    c = Call(lib, "mx_attn_decode_" + fmt, q_stride=4096, max_pages=4, B=2, Hq=32, Hkv=8, D=128, n_pages=10, page_size=16, max_len=64, window=0, scale=0.1, ws_bytes=1 << 40)
    for p in ("q", "page_table", "seq_lens", "out") + planes:
        assert c.with_(**{p: None}) == NULL, p
    for bad in (dict(B=0), dict(B=65536), dict(Hq=0), dict(Hkv=0), dict(Hq=33), dict(Hq=65536), dict(D=264), dict(D=24), dict(q_stride=4088), dict(q_stride=4097), dict(max_pages=0),
                dict(n_pages=0), dict(page_size=40), dict(n_pages=1 << 28, page_size=16), dict(D=16, Hq=1, Hkv=1, q_stride=16)):
        assert c.with_(**bad) == SHAPE, bad
    for bad in (dict(q=P8), dict(out=P8), dict(out_q8=0x1004), dict(page_table=P2), dict(seq_lens=P2), dict(sinks=P2)):
        assert c.with_(**bad) == ALIGN, bad


def test_attention_workspace(lib):
    import ctypes as C
    l, _ = lib
    n = C.c_uint64()
    assert l.mx_attn_decode_ws_bytes(2, 32, 8, 128, 64, 0, None) == NULL
    for bad in ((0, 32, 8, 128), (2, 32, 0, 128), (2, 33, 8, 128), (2, 32, 8, 130), (2, 32, 8, 512)):
        assert l.mx_attn_decode_ws_bytes(*bad, 64, 0, C.addressof(n)) == SHAPE
    for B, Hq, Hkv, D, L, W in ((1, 32, 8, 128, 100000, 0), (64, 32, 8, 128, 8192, 0), (1, 64, 8, 64, 4000, 128), (1, 1, 1, 16, 1, 0), (3, 16, 2, 256, 9999, 0), (1, 40, 1, 64, 1 << 31, 0)):
        assert l.mx_attn_decode_ws_bytes(B, Hq, Hkv, D, L, W, C.addressof(n)) == OK
        for fmt in ("f16", "q8_0"):
            if not n.value:
                continue
            c = Call(lib, "mx_attn_decode_" + fmt, q_stride=Hq * D, max_pages=4, B=B, Hq=Hq, Hkv=Hkv, D=D, n_pages=10, page_size=16, max_len=L, window=W, scale=0.1, out_q8=None)
            if fmt == "q8_0" and D % 32:
                continue
            assert c.with_(ws_bytes=n.value - 1) == WORKSPACE and c.with_(ws=None, ws_bytes=n.value) == NULL and c.with_(ws=P8, ws_bytes=n.value) == ALIGN


def freqs(lib, n_rot, base=10000.0, scale=1.0, ext=0.0, attn=1.0, fast=32.0, slow=1.0, ctx=0, factors=None):
    f, m = np.zeros(n_rot // 2), np.zeros(1)
    fac = None if factors is None else np.ascontiguousarray(factors, np.float32)
    rc = lib[0].mx_rope_freqs(n_rot, base, scale, ext, attn, fast, slow, ctx, None if fac is None else fac.ctypes.data, f.ctypes.data, m.ctypes.data)
    return rc, f, float(m[0])


def test_frequencies(lib):
    rc, f, m = freqs(lib, 64, 500000.0)
    np.testing.assert_allclose(f, 500000.0 ** (-np.arange(32) / 32.0), rtol=1e-14)
    assert rc == OK and m == 1.0
    rc, g, m = freqs(lib, 64, 500000.0, scale=0.25, attn=1.5)
    np.testing.assert_allclose(g, f / 4, rtol=1e-14)
    assert m == 1.5
    div = np.linspace(1, 8, 32)
    np.testing.assert_allclose(freqs(lib, 64, 500000.0, factors=div)[1], f / div.astype(np.float32), rtol=1e-14)


def test_frequencies_of_a_stretched_context(lib):
    """YaRN: the fast pairs as trained, the slow ones at scale, a straight line between, the factor on the values."""
    n, base, ctx, s = 64, 150000.0, 4096, 1 / 32.0
    rc, f, m = freqs(lib, n, base, scale=s, ext=1.0, ctx=ctx)
    plain = base ** (-np.arange(n // 2) * 2.0 / n)
    turns = ctx * plain / (2 * math.pi)               # of a pair within the trained context
    low, high = math.floor(n * math.log(ctx / (32 * 2 * math.pi)) / (2 * math.log(base))), math.ceil(n * math.log(ctx / (2 * math.pi)) / (2 * math.log(base)))
    share = f / plain                                 # 1: as trained, s: slowed down
    assert rc == OK and 0 < low < high < n // 2
    np.testing.assert_allclose(share[: low + 1], 1.0, rtol=1e-14)
    np.testing.assert_allclose(share[high:], s, rtol=1e-14)
    np.testing.assert_allclose(np.diff(share[low: high + 1]), (s - 1) / (high - low), rtol=1e-9)
    assert (share[turns > 32] == 1).all() and np.allclose(share[turns < 0.5], s)
    assert abs(m - (1 + 0.1 * math.log(32))) < 1e-15


def test_frequency_refusals(lib):
    assert lib[0].mx_rope_freqs(64, 1e4, 1.0, 0.0, 1.0, 32.0, 1.0, 0, None, None, P16) == NULL
    for bad in (dict(n_rot=24), dict(n_rot=272), dict(n_rot=0), dict(base=1.0), dict(scale=0.0), dict(scale=float("nan")), dict(ext=-1.0), dict(ext=1.0, ctx=0), dict(ext=2.0, ctx=1),
                dict(ext=1.0, ctx=4096, fast=0.5), dict(ext=1.0, ctx=4096, slow=0.0)):
        args = {"n_rot": 64, **bad}
        assert freqs(lib, args.pop("n_rot"), **args)[0] == SHAPE, bad


@pytest.mark.parametrize("fmt", ["f16", "q8_0"])
def test_in_place_needs_one_stride(lib, fmt):
    """Rows that are read with one stride and written from the same address with another would be overwritten before they are read."""
    r = Call(lib, "mx_rope", T=2, n_heads=8, D=128, x_stride=2048, y_stride=1024, n_rot=128, interleaved=0, mscale=1.0)
    assert r.with_() == r.with_(x_stride=1024, y_stride=2048) == r.with_(T=600, x_stride=1032) == SHAPE
    c = Call(lib, "mx_rope_kv_write_" + fmt, **{**HEADS, "q_stride": 6144})
    assert c.with_() == c.with_(T=600) == c.with_(q_stride=4096, q_out_stride=4104) == SHAPE
