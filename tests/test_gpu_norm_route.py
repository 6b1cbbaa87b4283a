"""GPU: the residual's addition with the norm and its 8-bit stream, and routing by scores, bias and groups."""
import numpy as np
import pytest
import torch

import oracle as O
from gpu_util import dev, host

pytestmark = pytest.mark.gpu


def f16(rng, *shape, scale=1.0):
    return O.round_fp16((rng.standard_normal(shape) * scale).astype(np.float32)).astype(np.float16)


@pytest.mark.parametrize("T,H", [(1, 32), (3, 64), (5, 992), (2, 1024), (7, 1056), (1, 4096), (333, 2880), (4, 5120), (2, 6144), (9, 7200), (3, 8192), (2, 8224), (1, 16384), (2050, 128), (77, 160), (9, 512), (5, 544), (2, 32768), (3, 32800), (1100, 1024)])
@pytest.mark.parametrize("halves", [False, True])
def test_add_rms_norm(mx, T, H, halves):
    """The sum is one fp32 addition rounded to fp16; the norm has the bits of rms_norm_f32w_q8 of that sum, the stream those of the quantizers on it."""
    rng = np.random.default_rng(T + H)
    x, res, w = f16(rng, T, H), f16(rng, T, H, scale=4.0), (1 + 0.3 * rng.standard_normal(H)).astype(np.float32)
    x[0, :32] = res[0, :32] = 0
    h, y, q8 = mx.ops.add_rms_norm_f32w_q8(dev(x), dev(res), dev(w), 1e-5, halves=halves)
    want = (x.astype(np.float32) + res.astype(np.float32)).astype(np.float16)
    assert np.array_equal(host(h).view(np.uint16), want.view(np.uint16))
    assert torch.equal(y, mx.ops.rms_norm_f32w_q8(h, dev(w), 1e-5)[0])
    assert torch.equal(q8, (mx.ops.quantize_q8_1s if halves else mx.ops.quantize_q8_1)(y))
    s = want.astype(np.float64)
    exact = s / np.sqrt((s * s).mean(1, keepdims=True) + 1e-5) * w
    # the rounding to fp16; the mean's 32-bit sum of H squares, the root and two products: (H + 6) 2^-24, half of it behind the root
    assert (np.abs(host(y) - exact) <= np.abs(exact) * (2.0 ** -11 + (H / 2 + 6) * 2.0 ** -24) + 2.0 ** -25).all()


@pytest.mark.parametrize("H", [64, 4096, 9216])
def test_in_place_and_without_rows(mx, H):
    rng = np.random.default_rng(H)
    x, res, w = dev(f16(rng, 5, H)), dev(f16(rng, 5, H)), dev(np.ones(H, np.float32))
    h, y, q8 = mx.ops.add_rms_norm_f32w_q8(x, res, w, 1e-6)
    h2, y2, q2 = mx.ops.add_rms_norm_f32w_q8(x, res, w, 1e-6, want_y=False)
    assert y2 is None and torch.equal(h, h2) and torch.equal(q8, q2)
    for target in (0, 1):
        a, b = x.clone(), res.clone()
        out = ((a, b)[target], torch.empty_like(x), torch.empty_like(q8))
        mx.ops.add_rms_norm_f32w_q8(a, b, w, 1e-6, out=out)
        assert torch.equal(out[0], h) and torch.equal(out[1], y) and torch.equal(out[2], q8)
        assert torch.equal((b, a)[target], (res, x)[target])


@pytest.mark.parametrize("H", [128, 1024, 33024])
def test_one_tensor_for_both(mx, H):
    x, w = dev(f16(np.random.default_rng(H), 3, H)), dev(np.ones(H, np.float32))
    h, y, q8 = mx.ops.add_rms_norm_f32w_q8(x, x.clone(), w, 1e-6)
    for got in (mx.ops.add_rms_norm_f32w_q8(x, x, w, 1e-6), mx.ops.add_rms_norm_f32w_q8(x, x, w, 1e-6, out=(x, torch.empty_like(x), torch.empty_like(q8)))):
        assert all(torch.equal(a, b) for a, b in zip(got, (h, y, q8)))


def test_rows_without_numbers_leave_others_alone(mx):
    rng = np.random.default_rng(1)
    x, res, w = f16(rng, 6, 256), f16(rng, 6, 256), np.ones(256, np.float32)
    want = host(mx.ops.add_rms_norm_f32w_q8(dev(x), dev(res), dev(w), 1e-5)[1])
    x[1, 7], x[3, 200], res[4, 0], x[5] = np.nan, np.inf, 65504, -res[5]
    x[4, 0] = 65504                                             # the sum is beyond fp16
    h, y, _ = (host(t) for t in mx.ops.add_rms_norm_f32w_q8(dev(x), dev(res), dev(w), 1e-5))
    assert np.array_equal(y[[0, 2]], want[[0, 2]]) and np.isnan(y[1]).all() and (y[5] == 0).all()
    assert np.isinf(h[3, 200]) and np.isinf(h[4, 0]) and np.isnan(y[3, 200]) and (np.delete(y[3], 200) == 0).all()


def test_norm_offsets_beyond_32_bits(mx):
    H, T = 8192, (1 << 32) // 8192 + 3
    x, res, w = torch.zeros(T, H, dtype=torch.float16, device="cuda"), torch.ones(T, H, dtype=torch.float16, device="cuda"), torch.ones(H, device="cuda")
    rng = np.random.default_rng(3)
    at = torch.tensor([0, 1, T - 4, T - 1], device="cuda")
    x[at], res[at] = dev(f16(rng, 4, H)), dev(f16(rng, 4, H))
    want = mx.ops.add_rms_norm_f32w_q8(x[at], res[at], w, 1e-5, want_y=False)
    q8 = torch.empty(T * (H // 32) * 40, dtype=torch.uint8, device="cuda")
    mx.ops.add_rms_norm_f32w_q8(x, res, w, 1e-5, out=(res, None, q8))
    assert torch.equal(res[at], want[0]) and torch.equal(q8.view(T, -1)[at], want[2].view(4, -1)) and (res[T - 2] == 1).all()


def test_norm_refusals(mx):
    x, w = torch.zeros(4, 64, dtype=torch.float16, device="cuda"), torch.ones(64, device="cuda")
    fn = mx.ops.add_rms_norm_f32w_q8
    fn(x, x.clone(), w, 1e-5)
    q8 = torch.empty(4 * 2 * 40, dtype=torch.uint8, device="cuda")
    for args in ((x.float(), x, w), (x, x[:3], w), (x, x, w[:32]), (x, x, w.half()), (x.cpu(), x, w), (x, x.t().contiguous().t(), w)):
        with pytest.raises(ValueError):
            fn(*args, 1e-5)
    for out in ((x[:3], None, q8), (x.clone(), x.clone()[:2], q8), (x.clone(), None, q8[:40]), (x.clone(), None, q8.float())):
        with pytest.raises(ValueError):
            fn(x, x, w, 1e-5, out=out)
    with pytest.raises(ValueError):
        fn(x, x, w, 1e-5, halves=True, out=(x.clone(), None, q8))
    with pytest.raises(mx.ops.MxError):
        fn(x[:, :48].contiguous(), x[:, :48].contiguous(), w[:48].contiguous(), 1e-5)
    with pytest.raises(mx.ops.MxError):
        fn(torch.zeros(0, 64, dtype=torch.float16, device="cuda"), torch.zeros(0, 64, dtype=torch.float16, device="cuda"), w, 1e-5)


# ------------------------------------------------------------------------------------------------------------------- routing
def route(logits, k, score="softmax", bias=None, n_groups=1, topk_groups=1, group_score="max", renormalize=True, scale=1.0):
    """-> (ids, weights in fp64, whether a token's choice is clear: its border wider than what 64-bit exponentials may be off)."""
    x = np.asarray(logits, np.float64)
    T, E = x.shape
    if score == "sigmoid":
        s = 1 / (1 + np.exp(-x))
    else:
        e = np.where(np.isneginf(x), 0.0, np.exp(x - np.where(np.isneginf(x.max(1)), 0.0, x.max(1))[:, None]))
        s = e / np.maximum(e.sum(1, keepdims=True), 1e-300)
    c = s if bias is None else s + np.asarray(bias, np.float64)
    open_ = np.ones((T, E), bool)
    if n_groups > 1:
        by = np.sort(c.reshape(T, n_groups, -1), -1)[..., ::-1]
        worth = by[..., 0] + by[..., 1] if group_score == "top2" and by.shape[-1] > 1 else by[..., 0]
        keep = np.argsort(-worth, 1, kind="stable")[:, :topk_groups]
        open_ = np.zeros((T, n_groups), bool)
        np.put_along_axis(open_, keep, True, 1)
        open_ = np.repeat(open_, E // n_groups, 1)
    ids = np.sort(np.argsort(np.where(open_, -c, np.inf), 1, kind="stable")[:, :k], 1)
    w = np.take_along_axis(s, ids, 1)
    return ids, scale * (w / (w.sum(1, keepdims=True) + 1e-20) if renormalize else w)


def check_route(mx, logits, k, what, **more):
    dm = {**more, "bias": None if more.get("bias") is None else dev(more["bias"])}
    idx, w = mx.ops.moe_route(dev(logits), k, **dm)
    ids, want = route(logits, k, **more)
    assert np.array_equal(host(idx), ids), "%s: %d tokens routed otherwise" % (what, (host(idx) != ids).any(1).sum())
    # one rounding to fp16 (2^-11, 2^-25 below the normal range); the factor is an fp32 number
    assert (np.abs(host(w) - want) <= want * (2.0 ** -11 + 2.0 ** -24) + 2.0 ** -25).all(), what
    return idx, w


@pytest.mark.parametrize("T,E,k,groups,kept", [(1, 1, 1, 1, 1), (1, 128, 8, 1, 1), (7, 60, 4, 1, 1), (33, 32, 4, 1, 1), (5, 1000, 64, 1, 1), (300, 256, 8, 8, 4), (3, 160, 6, 5, 3), (64, 64, 64, 64, 64),
                                             (9, 512, 10, 2, 1), (2, 1024, 16, 64, 7), (4097, 96, 3, 3, 2), (5, 1020, 30, 34, 5)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("f32", [False, True])
def test_route(mx, T, E, k, groups, kept, score, f32):
    rng = np.random.default_rng(E + k)
    logits = (rng.standard_normal((T, E)) * 2).astype(np.float32)
    logits = logits if f32 else logits.astype(np.float16)        # fp16: many equal ones
    bias = (0.1 * rng.standard_normal(E)).astype(np.float32)
    check_route(mx, logits, k, "plain", score=score, n_groups=groups, topk_groups=kept)
    check_route(mx, logits, k, "bias", score=score, bias=bias, n_groups=groups, topk_groups=kept, group_score="top2", renormalize=False, scale=2.5)
    check_route(mx, logits, k, "both", score=score, bias=bias * 30, n_groups=groups, topk_groups=kept, group_score="top2", scale=0.3)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_ties_go_to_the_lowest_id(mx, score):
    logits = np.zeros((3, 256), np.float16)
    logits[1, 64:] = 1.0
    logits[2, [3, 9, 200, 255]] = 2.0
    for groups, kept in ((1, 1), (8, 3)):
        for worth in ("max", "top2"):
            check_route(mx, logits, 5, "ties", score=score, n_groups=groups, topk_groups=kept, group_score=worth)


def test_choices_that_32_bits_cannot_tell(mx):
    """Sigmoids and biases whose sums differ by 2^-40 and less."""
    rng = np.random.default_rng(2)
    T, E = 500, 128
    logits = np.repeat((rng.standard_normal((T, 1)) * 3), E, 1).astype(np.float32)
    bias = np.zeros(E, np.float32)
    bias[rng.permutation(E)[:60]] = 2.0 ** -30 * rng.integers(1, 50, 60)
    check_route(mx, logits, 8, "close", score="sigmoid", bias=bias)
    logits = 30 + np.sort(rng.random((T, E)), 1).astype(np.float32)[:, rng.permutation(E)]        # 1 - sigmoid near 1e-13
    check_route(mx, logits, 8, "saturated", score="sigmoid")


def test_masked_experts_and_no_numbers(mx):
    """Experts of logit -infinity have score 0 and are taken last, by id; a bias of -infinity puts one out of the way too; a NaN lies below all of them."""
    rng = np.random.default_rng(3)
    logits = rng.standard_normal((4, 64)).astype(np.float32)
    logits[0, 5:] = -np.inf
    logits[1] = -np.inf
    bias = np.zeros(64, np.float32)
    for score in ("softmax", "sigmoid"):
        check_route(mx, logits, 8, "masked", score=score)
        check_route(mx, logits, 8, "masked", score=score, n_groups=4, topk_groups=2, group_score="top2")
    logits = rng.standard_normal((4, 64)).astype(np.float32)
    bias[10:] = -np.inf
    check_route(mx, logits, 8, "bias", score="sigmoid", bias=bias)
    check_route(mx, logits, 12, "bias", score="sigmoid", bias=bias)
    logits[2, :60] = np.nan
    idx, w = mx.ops.moe_route(dev(logits), 6, score="sigmoid", renormalize=False)
    assert host(idx)[2].tolist() == [0, 1, 60, 61, 62, 63] and np.isnan(host(w)[2, :2]).all() and np.isfinite(host(w)[2, 2:]).all()
    logits[3, 7] = np.nan                                        # a softmax over a NaN has no scores: ids by number
    idx, w = mx.ops.moe_route(dev(logits), 6, n_groups=8, topk_groups=2)
    assert host(idx)[3].tolist() == [0, 1, 2, 3, 4, 5] and np.isnan(host(w)[3]).all()


def test_a_token_is_routed_alike_in_every_batch(mx):
    rng = np.random.default_rng(4)
    logits, bias = dev(rng.standard_normal((1000, 256)).astype(np.float32)), dev((0.1 * rng.standard_normal(256)).astype(np.float32))
    call = lambda x: mx.ops.moe_route(x, 8, score="sigmoid", bias=bias, n_groups=8, topk_groups=4, group_score="top2")  # noqa: E731
    idx, w = call(logits)
    for at in (slice(0, 1), slice(7, 8), slice(3, 500)):
        i, v = call(logits[at].contiguous())
        assert torch.equal(i, idx[at]) and torch.equal(v, w[at])


def test_logits_are_the_routers(mx):
    """moe_router_logits gives what moe_router goes by; over them the softmax form chooses as it does."""
    rng = np.random.default_rng(5)
    for T, E, H in ((1, 128, 2048), (70, 60, 516), (600, 128, 2048)):
        x, W = dev(f16(rng, T, H)), dev((0.05 * rng.standard_normal((E, H))).astype(np.float32))
        logits = mx.ops.moe_router_logits(x, W)
        exact = host(x).astype(np.float64) @ host(W).astype(np.float64).T
        assert np.abs(host(logits) - exact).max() <= 2.0 ** -20 * np.sqrt(H)
        idx, w = mx.ops.moe_router(x, W, E, 4)
        i, v = mx.ops.moe_route(logits, 4)
        assert torch.equal(i, idx) and (v.float() - w.float()).abs().max() <= 2.0 ** -10


def test_route_captured(mx):
    rng = np.random.default_rng(6)
    logits = dev(rng.standard_normal((17, 160)).astype(np.float16))
    call = lambda: mx.ops.moe_route(logits, 6, n_groups=8, topk_groups=3)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        idx, w = call()
    for seed in range(4):
        logits.copy_(dev(np.random.default_rng(seed).standard_normal((17, 160)).astype(np.float16)))
        i, v = call()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(i, idx) and torch.equal(v, w)


def test_route_offsets_beyond_32_bits(mx):
    T, E = (1 << 32) // 1024 + 5, 1024
    logits = torch.zeros(T, E, dtype=torch.float16, device="cuda")
    at = torch.tensor([0, 7, T - 5, T - 2, T - 1], device="cuda")
    logits[at] = dev(np.random.default_rng(4).standard_normal((5, E)).astype(np.float16))
    idx, w = mx.ops.moe_route(logits, 8, n_groups=8, topk_groups=2)
    want = mx.ops.moe_route(logits[at], 8, n_groups=8, topk_groups=2)
    assert torch.equal(idx[at], want[0]) and torch.equal(w[at], want[1]) and torch.equal(idx[T - 3], torch.arange(8, dtype=torch.int32, device="cuda"))


def test_route_refusals(mx):
    x = torch.zeros(3, 64, device="cuda")
    mx.ops.moe_route(x, 4)
    for more in (dict(score="other"), dict(group_score="sum"), dict(bias=torch.zeros(63, device="cuda")), dict(bias=torch.zeros(64, device="cuda").half())):
        with pytest.raises(ValueError):
            mx.ops.moe_route(x, 4, **more)
    for bad in (x.double(), x.cpu(), x.t().contiguous().t()):
        with pytest.raises(ValueError):
            mx.ops.moe_route(bad, 4)
    for k, more in ((65, {}), (0, {}), (4, dict(n_groups=3)), (4, dict(n_groups=0)), (4, dict(n_groups=8, topk_groups=9)), (4, dict(n_groups=8, topk_groups=0)), (9, dict(n_groups=8, topk_groups=1))):
        with pytest.raises(mx.ops.MxError):
            mx.ops.moe_route(x, k, **more)
    with pytest.raises(mx.ops.MxError):
        mx.ops.moe_route(torch.zeros(3, 1025, device="cuda"), 4)
    with pytest.raises(mx.ops.MxError):
        mx.ops.moe_route(x[:0], 4)
    with pytest.raises(ValueError):
        mx.ops.moe_router_logits(torch.zeros(3, 64, device="cuda").half(), torch.zeros(8, 60, device="cuda"))
