"""Entry points of the Q4_0 cache, the residual's norm and the routing without a GPU: refusals before any HIP call."""
import pytest

from test_kv_capi import ALIGN, HEADS, NULL, P2, P8, SHAPE, WORKSPACE, Call, lib  # noqa: F401

PLANES = ("k_qs", "k_d", "v_qs", "v_d")


def test_write_refusals(lib):  # noqa: F811
    c, w = Call(lib, "mx_rope_kv_write_q4_0", **HEADS), Call(lib, "mx_kv_write_q4_0", **HEADS)
    for p in ("q", "k", "v", "q_out", "positions", "slots", "freqs") + PLANES:
        assert c.with_(**{p: None}) == NULL, p
    for p in ("k", "v", "slots") + PLANES:
        assert w.with_(**{p: None}) == NULL, p
    for bad in (dict(T=0), dict(Hkv=0), dict(D=0), dict(D=288), dict(D=112, n_rot=16), dict(D=48, n_rot=16), dict(n_rot=8), dict(q_stride=4088), dict(k_stride=1016), dict(v_stride=1025),
                dict(n_pages=0), dict(page_size=24), dict(n_pages=1 << 27, page_size=16), dict(T=1 << 26), dict(T=1 << 23, D=96, n_rot=96)):
        assert c.with_(**bad) == SHAPE, bad
        if set(bad) <= {"T", "Hkv", "k_stride", "v_stride", "n_pages", "page_size"}:
            assert w.with_(**bad) == SHAPE, bad
    for bad in (dict(q=P8), dict(k=P8), dict(v=P2), dict(slots=P2)) + tuple({p: 0x1001} for p in PLANES) + tuple({p: P8} for p in PLANES):
        assert c.with_(**bad) == ALIGN, bad
    assert c.with_(q=0x2000, q_out=0x2000, q_out_stride=5000 // 8 * 8) == SHAPE


def test_read_refusals(lib):  # noqa: F811
    c = Call(lib, "mx_kv_read_q4_0", max_pages=4, total_rows=60, B=2, Hkv=8, D=128, n_pages=10, page_size=16)
    for p in ("page_table", "rows", "k_out", "v_out") + PLANES:
        assert c.with_(**{p: None}) == NULL, p
    for bad in (dict(max_pages=0), dict(total_rows=0), dict(total_rows=1 << 31), dict(B=0), dict(Hkv=0), dict(D=40), dict(D=112), dict(n_pages=0), dict(page_size=20), dict(total_rows=1 << 28, B=1)):
        assert c.with_(**bad) == SHAPE, bad
    for bad in (dict(page_table=P2), dict(rows=P2), dict(k_out=P8), dict(v_out=P8), dict(k_qs=P8), dict(v_d=P8)):
        assert c.with_(**bad) == ALIGN, bad


def test_attention_refusals(lib):  # noqa: F811
    c = Call(lib, "mx_attn_decode_q4_0", q_stride=4096, max_pages=4, B=2, Hq=32, Hkv=8, D=128, n_pages=10, page_size=16, max_len=64, window=0, scale=0.1, ws_bytes=1 << 40)
    for p in ("q", "page_table", "seq_lens", "out") + PLANES:
        assert c.with_(**{p: None}) == NULL, p
    for bad in (dict(B=0), dict(B=65536), dict(Hq=33), dict(D=264), dict(D=48), dict(q_stride=4088), dict(max_pages=0), dict(n_pages=0), dict(page_size=40), dict(n_pages=1 << 28, page_size=16)):
        assert c.with_(**bad) == SHAPE, bad
    for bad in (dict(q=P8), dict(out=P8), dict(out_q8=0x1004), dict(page_table=P2), dict(seq_lens=P2), dict(sinks=P2), dict(k_qs=P8), dict(k_d=P8)):
        assert c.with_(**bad) == ALIGN, bad
    assert c.with_(max_len=100000, ws_bytes=100) == WORKSPACE
    import ctypes
    n, query = ctypes.c_uint64(), lib[0].mx_attn_decode_q4_0_ws_bytes
    assert query(2, 32, 8, 128, 512, 0, ctypes.addressof(n)) == 0 and n.value == 0
    assert query(2, 32, 8, 128, 100000, 0, ctypes.addressof(n)) == 0 and n.value > 0
    assert c.with_(max_len=100000, ws_bytes=n.value - 1) == WORKSPACE
    assert query(2, 32, 8, 128, 100000, 0, None) == NULL
    for bad in ((0, 32, 8, 128), (65536, 32, 8, 128), (2, 33, 8, 128), (2, 32, 0, 128), (2, 32, 8, 48), (2, 32, 8, 288)):
        assert query(*bad, 1000, 0, ctypes.addressof(n)) == SHAPE, bad
    assert c.with_(max_len=100000, ws=None) == NULL


def test_norm_refusals(lib):  # noqa: F811
    c = Call(lib, "mx_add_rms_norm_f32w_q8", n_rows=4, hidden=128, eps=1e-5, halves=0)
    for p in ("x", "residual", "w", "sum", "q8_out"):
        assert c.with_(**{p: None}) == NULL, p
    for bad in (dict(n_rows=0), dict(n_rows=1 << 25), dict(n_rows=1 << 24, hidden=2048), dict(n_rows=1 << 22, hidden=8192), dict(n_rows=1 << 22, hidden=1 << 20), dict(hidden=0), dict(hidden=48), dict(hidden=100)):
        assert c.with_(**bad) == SHAPE, bad
    for bad in (dict(x=P8), dict(residual=P8), dict(w=P8), dict(sum=P2), dict(y=P8), dict(q8_out=0x1004), dict(q8_out=P8, halves=1)):
        assert c.with_(**bad) == ALIGN, bad


def test_route_refusals(lib):  # noqa: F811
    c = Call(lib, "mx_moe_route", n_tokens=4, n_experts=64, k=8, n_groups=1, topk_groups=1, flags=0, scale=1.0)
    for p in ("logits", "topk_idx", "topk_w"):
        assert c.with_(**{p: None}) == NULL, p
    for bad in (dict(n_tokens=0), dict(n_tokens=1 << 26), dict(n_experts=0), dict(n_experts=1025), dict(k=0), dict(k=65), dict(n_experts=4, k=5), dict(n_groups=0), dict(n_groups=3), dict(n_groups=65, n_experts=130),
                dict(topk_groups=0), dict(topk_groups=2), dict(n_groups=16, topk_groups=1, k=5), dict(flags=16), dict(flags=1 << 31)):
        assert c.with_(**bad) == SHAPE, bad
    for bad in (dict(logits=0x1001), dict(logits=P2, flags=8), dict(bias=P2), dict(topk_idx=P2), dict(topk_w=0x1001)):
        assert c.with_(**bad) == ALIGN, bad
    r = Call(lib, "mx_moe_router_logits", n_tokens=4, hidden=128, n_experts=64)
    for p in ("x", "W_gate", "logits"):
        assert r.with_(**{p: None}) == NULL, p
    for bad in (dict(n_tokens=0), dict(n_tokens=65536), dict(hidden=0), dict(hidden=126), dict(n_experts=0), dict(n_experts=1025)):
        assert r.with_(**bad) == SHAPE, bad
    for bad in (dict(x=P2), dict(W_gate=P8), dict(logits=P2)):
        assert r.with_(**bad) == ALIGN, bad
