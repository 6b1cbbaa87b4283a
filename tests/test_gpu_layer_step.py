"""GPU: a decoder layer's token steps, the operators in the order they are used in: residual + norm -> projections -> rotation and append to a Q4_0 cache -> attention -> projection -> residual + norm -> router -> experts."""
import numpy as np
import pytest
import torch

import kv_util as U
import oracle as O
import q4_util as Q
from gpu_util import check, dev, host
from test_gpu_moe import check_rows, make_experts
from test_gpu_norm_route import route

pytestmark = pytest.mark.gpu

H, HQ, HKV, D, PS, PAGES, E, K, EF = 512, 8, 2, 64, 16, 5, 32, 4, 256


class Layer:
    def __init__(self, mx, B, seed):
        from machx_inference_engine_amd import synth
        self.ops, self.B = mx.ops, B
        rng = np.random.default_rng(seed)
        self.Wqkv, self.Wo = synth.normal_weights("q8_0", (HQ + 2 * HKV) * D, H, seed=seed), synth.normal_weights("q8_0", H, HQ * D, seed=seed + 1)
        self.Wqkv_soa = [dev(t) for t in self.ops.repack_block32_to_soa("q8_0", host(self.Wqkv))]
        self.experts = [make_experts(O.Q8_0, s, E, *nk) for s, nk in ((seed + 100, (EF, H)), (seed + 200, (EF, H)), (seed + 300, (H, EF)))]
        self.banks = [(dev(x[1]), dev(x[2])) for x in self.experts]
        self.norms = [dev((1 + 0.1 * rng.standard_normal(H)).astype(np.float32)) for _ in range(2)]
        self.gate, self.bias = dev((0.05 * rng.standard_normal((E, H))).astype(np.float32)), dev((0.02 * rng.standard_normal(E)).astype(np.float32))
        self.sinks = dev(rng.standard_normal(HQ).astype(np.float32))
        self.freqs, self.mscale = self.ops.rope_freqs(D)
        self.freqs = self.freqs.cuda()
        self.pages = rng.permutation(B * PAGES).reshape(B, PAGES).astype(np.int32)
        self.table = dev(self.pages)

    def heads(self, qkv):
        return [p.unflatten(1, (-1, D)) for p in qkv.view(-1, (HQ + 2 * HKV) * D).split((HQ * D, HKV * D, HKV * D), 1)]

    def step(self, x, residual, pos, slots, lens, cache):
        """One token of each sequence -> everything that the steps leave."""
        ops, B = self.ops, self.B
        total, y, xq = ops.add_rms_norm_f32w_q8(x, residual, self.norms[0], 1e-5)
        q, k, v = self.heads(ops.gemv_q8_0_q8_batched(xq, self.Wqkv, H, (HQ + 2 * HKV) * D, B))
        qr = ops.rope_kv_write(q, k, v, pos, slots, cache, self.freqs, mscale=self.mscale)
        stream = torch.empty(B * HQ * D // 32 * 40, dtype=torch.uint8, device="cuda")
        a = ops.attn_decode(qr, cache, self.table, lens, sinks=self.sinks, out_q8=stream)
        o = ops.gemv_q8_0_q8_batched(stream, self.Wo, HQ * D, H, B)
        total2, y2, yq = ops.add_rms_norm_f32w_q8(o.view(B, H), total, self.norms[1], 1e-5)
        logits = ops.moe_router_logits(y2, self.gate)
        ids, w = ops.moe_route(logits, K, "sigmoid", self.bias, 8, 4, "top2", True, 2.5)
        (gq, gd), (uq, ud), (dq, dd) = self.banks
        h = ops.moe_gate_up_silu_q8(yq, gq, gd, uq, ud, H * EF, H * EF // 32, ids, B, K, H, EF, n_experts=E)
        down = ops.moe_down_q8_f16(h, dq, dd, H * EF, H * EF // 32, ids, w, B, K, EF, H, n_experts=E)
        return dict(total=total, y=y, q=q, k=k, v=v, qr=qr, a=a, o=o, total2=total2, y2=y2, yq=yq, logits=logits, ids=ids, w=w, h=h, down=down, out=ops.moe_reduce_q8(down, B, K, H))

    def prompt(self, lens, cache, seed):
        """Prompts of lens[b] tokens: appended at once, read back for the attention over them."""
        rng = np.random.default_rng(seed)
        rows = np.concatenate(([0], np.cumsum(lens))).astype(np.int32)
        x = dev(rng.standard_normal((rows[-1], H)).astype(np.float16))
        pos = np.concatenate([np.arange(n) for n in lens]).astype(np.int32)
        slots = np.concatenate([self.pages[b][np.arange(n) // PS] * PS + np.arange(n) % PS for b, n in enumerate(lens)]).astype(np.int32)
        _, _, xq = self.ops.add_rms_norm_f32w_q8(x, torch.zeros_like(x), self.norms[0], 1e-5, halves=True, want_y=False)
        q, k, v = self.heads(self.ops.gemm_q8_rows("q8_0_soa", xq, self.Wqkv_soa, len(x), H, (HQ + 2 * HKV) * D))
        self.ops.rope_kv_write(q, k, v, dev(pos), dev(slots), cache, self.freqs, mscale=self.mscale)
        kr, vr = self.ops.kv_read(cache, self.table, dev(rows), int(rows[-1]))
        # what was read is the encoding of what was written: the rotated keys in 64 bits are off by their own rounding, which may move a code on its border by a step
        codes, d = Q.q4_0(host(v))
        assert np.array_equal(host(vr).astype(np.float64), O.round_fp16(Q.values(codes, d).astype(np.float32)).astype(np.float64))
        kw = U.rope(host(k), pos, host(self.freqs), False, self.mscale)
        m = np.abs(kw).reshape(kw.shape[:-1] + (-1, 32)).max(-1).repeat(32, -1)
        # half a step of m / 8, a whole one past the last code (8 x / m in [7.5, 8] has none of its own); the two roundings to fp16 of the value, the scale's and the product's
        assert (np.abs(host(kr) - kw) <= m / 8 * (1 + 2.0 ** -8) + 2.0 ** -9 * m).all()


def slots_of(layer, pos):
    return dev((layer.pages[np.arange(layer.B), pos // PS] * PS + pos % PS).astype(np.int32))


def check_step(layer, got, x, residual, pos, cache):
    g = {n: host(t) for n, t in got.items()}
    f64 = lambda t: np.asarray(t, np.float64)  # noqa: E731
    for s, y, a, b, w in (("total", "y", x, residual, 0), ("total2", "y2", g["o"].reshape(layer.B, H), g["total"], 1)):
        assert np.array_equal(g[s], (np.asarray(a, np.float32) + np.asarray(b, np.float32)).astype(np.float16))
        t = f64(g[s])
        exact = t / np.sqrt((t * t).mean(1, keepdims=True) + 1e-5) * host(layer.norms[w])
        assert (np.abs(g[y] - exact) <= np.abs(exact) * (2.0 ** -11 + (H / 2 + 6) * 2.0 ** -24) + 2.0 ** -25).all()
    assert np.array_equal(g["yq"], O.quantize_q8_1(g["y2"].astype(np.float32)))
    freqs = host(layer.freqs)
    want = U.rope(g["q"], pos, freqs, False, layer.mscale)
    assert (np.abs(g["qr"] - want) <= 2.0 ** -11 * np.abs(want) + 2.0 ** -25 + U.rope_tol(g["q"], freqs, False, layer.mscale)).all()
    want, tol = Q.attention(g["qr"], cache, layer.pages, pos + 1, PS, D ** -0.5, 0, host(layer.sinks))
    assert (np.abs(g["a"] - want) <= tol).all()
    at = f64(g["y2"]) @ f64(host(layer.gate)).T
    # H products and additions in 32 bits
    assert (np.abs(g["logits"] - at) <= (H + 2) * 2.0 ** -24 * (np.abs(f64(g["y2"])) @ np.abs(f64(host(layer.gate))).T)).all()
    ids, w = route(g["logits"], K, "sigmoid", host(layer.bias), 8, 4, "top2", True, 2.5)
    assert np.array_equal(g["ids"], ids) and (np.abs(g["w"] - w) <= w * (2.0 ** -11 + 2.0 ** -24) + 2.0 ** -25).all()
    rb = H // 32 * 40
    gate, up = ([O.gemv_q8chain(O.Q8_0, bank[0][e], g["yq"][t * rb:(t + 1) * rb], H, EF)[0].astype(np.float32) for t in range(layer.B) for e in ids[t]] for bank in layer.experts[:2])
    check(g["h"].astype(np.float32), O.swiglu_np(np.stack(gate), np.stack(up)), "gate and up of the chosen experts")
    hq, hrb = O.quantize_q8_1(g["h"].astype(np.float32)), EF // 32 * 40
    down = np.stack([float(g["w"].ravel()[s]) * O.gemv_q8chain(O.Q8_0, layer.experts[2][0][e], hq[s * hrb:(s + 1) * hrb], EF, H)[0] for s, e in enumerate(ids.ravel())])
    check(g["down"].astype(np.float32), down, "weighted down products")


@pytest.mark.parametrize("B,lens", [(1, [37]), (3, [0, 15, 60]), (16, list(range(0, 64, 4)))])
def test_layer_step(mx, B, lens):
    """A prompt, then tokens one at a time, each stage against its plain form."""
    layer = Layer(mx, B, 40 + B)
    cache = mx.ops.kv_cache("q4_0", B * PAGES, HKV, PS, D)
    layer.prompt(lens, cache, 1)
    pos = np.array(lens, np.int32)
    rng = np.random.default_rng(2)
    x, residual = (dev(rng.standard_normal((B, H)).astype(np.float16)) for _ in range(2))
    for _ in range(5):
        got = layer.step(x, residual, dev(pos), slots_of(layer, pos), dev(pos + 1), cache)
        check_step(layer, got, host(x), host(residual), pos, cache)
        x, residual, pos = got["out"], got["total2"], pos + 1


@pytest.mark.parametrize("T", [1, 3, 70])
def test_prompt_through_the_experts(mx, T):
    """Routed, packed on the device, through the grouped products: the rows of the token by token form."""
    layer, ops = Layer(mx, 1, 60), mx.ops
    rng = np.random.default_rng(T)
    x, residual = (dev(rng.standard_normal((T, H)).astype(np.float16)) for _ in range(2))
    _, y, yq = ops.add_rms_norm_f32w_q8(x, residual, layer.norms[1], 1e-5)
    ids, w = ops.moe_route(ops.moe_router_logits(y, layer.gate), K, bias=layer.bias, n_groups=4, topk_groups=2)
    off, si, wp, t2p = ops.moe_build_packing_device(ids, w, E)
    for a, b in zip((off, si, wp, t2p), O.build_moe_packing(host(ids), host(w).astype(np.float32), E)):
        assert np.array_equal(host(a).astype(np.float64), np.asarray(b, np.float64))
    (gq, gd), (uq, ud), (dq, dd) = layer.banks
    rows = ops.quantize_q8_1(ops.moe_gather_rows(y, si, T * K, H))
    packed = ops.moe_prefill_gate_up_silu_q8(rows, gq, gd, uq, ud, H * EF, H * EF // 32, off, T * K, E, H, EF)
    h = torch.cat([ops.moe_gate_up_silu_q8(yq.view(T, -1)[t].contiguous(), gq, gd, uq, ud, H * EF, H * EF // 32, ids[t].contiguous(), 1, K, H, EF, n_experts=E) for t in range(T)])
    check_rows(host(packed)[host(t2p)], host(h), "grouped gate and up")
    out = ops.moe_prefill_down_q8(ops.quantize_q8_1(packed), dq, dd, H * EF, H * EF // 32, off, wp, T * K, E, H, EF)
    hq = ops.quantize_q8_1(packed[t2p.long()])
    down = torch.cat([ops.moe_down_q8(hq.view(T, -1)[t].contiguous(), dq, dd, H * EF, H * EF // 32, ids[t].contiguous(), w[t].contiguous(), 1, K, EF, H, n_experts=E) for t in range(T)])
    check_rows(host(out)[host(t2p)], host(down), "grouped down")


def test_captured_step(mx):
    """The step captured once, replayed over growing sequences on a cache of its own; between the replays the program's eager steps, which every replay has to agree with bit for bit."""
    B = 5
    layer = Layer(mx, B, 90)
    eager, own = (mx.ops.kv_cache("q4_0", B * PAGES, HKV, PS, D) for _ in range(2))
    pos = np.array([0, 3, 16, 31, 50], np.int32)
    layer.prompt(pos, eager, 3)
    for a, b in zip(own, eager):
        a.copy_(b)
    rng = np.random.default_rng(4)
    x, residual = (dev(rng.standard_normal((B, H)).astype(np.float16)) for _ in range(2))
    static = [x.clone(), residual.clone(), dev(pos), slots_of(layer, pos), dev(pos + 1)]
    scratch = tuple(t.clone() for t in own)
    layer.step(*static, scratch)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        replayed = layer.step(*static, own)
    for _ in range(8):
        now = (x, residual, dev(pos), slots_of(layer, pos), dev(pos + 1))
        got = layer.step(*now, eager)
        for a, b in zip(static, now):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        for name in got:
            assert torch.equal(got[name], replayed[name]), name
        for a, b in zip(eager, own):
            assert torch.equal(a, b)
        x, residual, pos = got["out"], got["total2"], pos + 1
