"""GPU: attention of one token over the paged cache (fp16 and Q8_0), against softmax and sums in 64 bits."""
import numpy as np
import pytest
import torch

import kv_util as U
import oracle as O
from gpu_util import dev, host

pytestmark = pytest.mark.gpu


def case(fmt, lens, Hkv, G, D, ps, seed, k_scale=1.0):
    rng = np.random.default_rng(seed)
    table, n_pages = U.pages_of(lens, ps, rng)
    cache = U.random_cache(fmt, rng, n_pages, Hkv, ps, D, k_scale)
    cache = U.keep_only(cache, table, lens, ps)
    q = O.round_fp16(rng.standard_normal((len(lens), Hkv * G, D)).astype(np.float32)).astype(np.float16)
    return rng, table, cache, q


def near(got, want, tol, what):
    got = np.asarray(got, np.float64)
    assert np.isfinite(got).all(), what + ": not finite"
    off = np.abs(got - want)
    worst = np.unravel_index(np.argmax(off - tol), off.shape)
    assert (off <= tol).all(), "%s: at %s %.6e instead of %.6e, %.2e allowed (%d of %d)" % (what, worst, got[worst], want[worst], tol[worst], (off > tol).sum(), off.size)


LENS = {"one": [1], "edges": [0, 1, 15, 16, 17, 31, 32, 33, 47, 48, 63, 64, 65, 127, 128, 129], "none": [0, 0, 0], "mid": [700], "ragged": [1000, 3, 257, 0, 513, 64],
        "long": [9001, 12]}


@pytest.mark.parametrize("fmt", ["f16", "q8_0"])
@pytest.mark.parametrize("lens", sorted(LENS))
@pytest.mark.parametrize("Hkv,G,D,ps", [(8, 4, 128, 16), (4, 8, 128, 64), (2, 8, 64, 32), (2, 8, 256, 16), (1, 1, 64, 16), (3, 5, 96, 48), (1, 16, 128, 256)])
def test_attn_decode(mx, fmt, lens, Hkv, G, D, ps):
    lens = LENS[lens]
    rng, table, cache, q = case(fmt, lens, Hkv, G, D, ps, 100 + D + len(lens))
    y = mx.ops.attn_decode(dev(q), cache, dev(table), dev(np.array(lens, np.int32)))
    want, tol = U.attention(q, cache, table, lens, ps, D ** -0.5)
    near(host(y), want, tol, "attention")
    assert (host(y)[np.array(lens) == 0] == 0).all()


@pytest.mark.parametrize("fmt,D", [("f16", 16), ("f16", 48), ("f16", 80), ("f16", 112), ("f16", 144), ("f16", 208), ("f16", 240), ("q8_0", 32), ("q8_0", 160), ("q8_0", 192), ("q8_0", 224)])
@pytest.mark.parametrize("G", [1, 7])
def test_odd_heads(mx, fmt, D, G):
    lens = [130, 0, 19, 1]
    rng, table, cache, q = case(fmt, lens, 2, G, D, 16, D)
    y = mx.ops.attn_decode(dev(q), cache, dev(table), dev(np.array(lens, np.int32)))
    near(host(y), *U.attention(q, cache, table, lens, 16, D ** -0.5), "D=%d G=%d" % (D, G))


@pytest.mark.parametrize("fmt", ["f16", "q8_0"])
@pytest.mark.parametrize("G", [17, 24, 40])
def test_more_heads_in_a_group_than_a_tile_holds(mx, fmt, G):
    lens = [77, 200]
    rng, table, cache, q = case(fmt, lens, 1, G, 64, 16, G)
    y = mx.ops.attn_decode(dev(q), cache, dev(table), dev(np.array(lens, np.int32)))
    near(host(y), *U.attention(q, cache, table, lens, 16, 0.125), "G=%d" % G)


@pytest.mark.parametrize("fmt", ["f16", "q8_0"])
@pytest.mark.parametrize("window", [1, 5, 16, 33, 128, 1000])
@pytest.mark.parametrize("with_sinks", [False, True])
def test_window_and_sinks(mx, fmt, window, with_sinks):
    lens = [0, 1, 4, 5, 6, 127, 128, 129, 300, 1500]
    rng, table, cache, q = case(fmt, lens, 2, 8, 64, 16, window)
    sinks = rng.standard_normal(16).astype(np.float32) * 3 if with_sinks else None
    y = mx.ops.attn_decode(dev(q), cache, dev(table), dev(np.array(lens, np.int32)), window=window, sinks=None if sinks is None else dev(sinks))
    near(host(y), *U.attention(q, cache, table, lens, 16, 0.125, window, sinks), "window %d" % window)


@pytest.mark.parametrize("fmt", ["f16", "q8_0"])
@pytest.mark.parametrize("B,Hkv,G,D", [(150, 1, 4, 64), (70, 2, 24, 128), (65, 1, 2, 256), (300, 3, 1, 96), (3000, 1, 1, 32)])
def test_many_ragged_sequences_in_equal_shares(mx, fmt, B, Hkv, G, D):
    """More sequences than a wave has lanes, empty ones among them (the first and the last too), shares that end in the middle of some and span others."""
    rng = np.random.default_rng(B)
    lens = [int(n) if rng.random() < 0.8 else 0 for n in np.exp(rng.uniform(0, np.log(900 if B < 1000 else 40), B))]
    lens[0] = lens[-1] = 0
    lens[B // 2] = 2500
    rng, table, cache, q = case(fmt, lens, Hkv, G, D, 16, B)
    sinks = rng.standard_normal(Hkv * G).astype(np.float32)
    y = mx.ops.attn_decode(dev(q), cache, dev(table), dev(np.array(lens, np.int32)), sinks=dev(sinks))
    near(host(y), *U.attention(q, cache, table, lens, 16, D ** -0.5, sinks=sinks), "B=%d" % B)


@pytest.mark.parametrize("fmt", ["f16", "q8_0"])
@pytest.mark.parametrize("n", [513, 544, 640, 1024, 1025, 4096, 16385])
def test_one_sequence_in_shares(mx, fmt, n):
    """Lengths around those at which the number of shares changes, with a length in front of what max_len says and behind it."""
    rng, table, cache, q = case(fmt, [n], 2, 4, 64, 32, n)
    for m in (n, n - 1, n // 2, 33, 1, 0):
        lens = np.array([m], np.int32)
        want, tol = U.attention(q, cache, table, lens, 32, 0.125)
        for max_len in (n, 600):
            near(host(mx.ops.attn_decode(dev(q), cache, dev(table), dev(lens), max_len=max_len)), want, tol, "%d of %d, max_len %d" % (m, n, max_len))


def test_a_large_batch_of_short_sequences(mx):
    lens = [i % 4 for i in range(20000)]
    rng, table, cache, q = case("f16", lens, 1, 1, 16, 16, 67)
    y = mx.ops.attn_decode(dev(q), cache, dev(table), dev(np.array(lens, np.int32)))
    near(host(y), *U.attention(q, cache, table, lens, 16, 0.25), "20000 sequences")


def test_pages_of_sixteen_times_any_number(mx):
    for ps in (16, 48, 80, 112, 1008, 4096):
        lens = [700, 1001, 0, ps + 1]
        rng, table, cache, q = case("q8_0", lens, 1, 4, 64, ps, ps)
        y = mx.ops.attn_decode(dev(q), cache, dev(table), dev(np.array(lens, np.int32)), window=900)
        near(host(y), *U.attention(q, cache, table, lens, ps, 0.125, 900), "pages of %d" % ps)


def test_refusals(mx):
    ops = mx.ops
    cache, tab, lens = ops.kv_cache("f16", 4, 2, 16, 64), dev(np.zeros((3, 4), np.int32)), dev(np.ones(3, np.int32))
    q = torch.zeros(3, 8, 64, dtype=torch.float16, device="cuda")
    ok = dict(q=q, cache=cache, page_table=tab, seq_lens=lens)
    ops.attn_decode(**ok)
    for bad in (dict(q=q.float()), dict(q=q.cpu()), dict(q=q[:2]), dict(q=q[..., :48]), dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)), dict(page_table=tab.long()),
                dict(page_table=tab[:, ::2]), dict(page_table=tab[:2]), dict(seq_lens=lens[:2]), dict(seq_lens=lens.cpu()), dict(sinks=torch.zeros(7, device="cuda")),
                dict(sinks=torch.zeros(8, device="cuda").half()), dict(out=q[:2]), dict(out=q.float()), dict(out=torch.zeros(3, 9, 64, device="cuda").half()[:, :8]),
                dict(out_q8=torch.zeros(5, dtype=torch.uint8, device="cuda")), dict(cache=cache[:1]), dict(cache=(cache[0], cache[1][:3])),
                dict(cache=(cache[0].transpose(1, 2), cache[1].transpose(1, 2))), dict(cache=(cache[0].float(), cache[1])), dict(cache=(cache[0].cpu(), cache[1])),
                dict(cache=ops.kv_cache("q8_0", 4, 2, 16, 64)[:3])):
        with pytest.raises(ValueError):
            ops.attn_decode(**{**ok, **bad})
    for bad in (dict(q=torch.zeros(3, 7, 64, dtype=torch.float16, device="cuda")), dict(max_len=100000, ws=torch.zeros(16, device="cuda")), dict(cache=ops.kv_cache("f16", 4, 2, 24, 64)),
                dict(q=torch.zeros(3 * 516, dtype=torch.float16, device="cuda").as_strided((3, 8, 64), (516, 64, 1)))):
        with pytest.raises(mx.ops.MxError):
            ops.attn_decode(**{**ok, **bad})


@pytest.mark.parametrize("fmt", ["f16", "q8_0"])
def test_what_the_window_left_behind_is_not_read(mx, fmt):
    """Pages in front of the window are given back: their entries name no page, and NaN lies in the slots in front of it."""
    ps, window, n = 16, 40, 203
    rng, table, cache, q = case(fmt, [n], 2, 4, 128, ps, 9)
    want, tol = U.attention(q, cache, table, [n], ps, 128 ** -0.5, window)
    lo = n - window
    for t in range(lo):
        for c in cache:
            if c.dtype == torch.float16:
                c[int(table[0, t // ps]), :, t % ps] = float("nan")
    table[0, : lo // ps] = -7
    y = mx.ops.attn_decode(dev(q), cache, dev(table), dev(np.array([n], np.int32)), window=window)
    near(host(y), want, tol, "window")


@pytest.mark.parametrize("fmt", ["f16", "q8_0"])
def test_pages_outside_the_cache_are_masked(mx, fmt):
    ps, lens = 16, [100, 64, 33, 500]
    rng, table, cache, q = case(fmt, lens, 2, 4, 64, ps, 31)
    table[0, 2], table[0, 3], table[3, 0], table[3, 17] = -1, 10 ** 6, -2 ** 31, 2 ** 31 - 1
    table[1, :] = -1                                           # nothing is left of this one
    y = mx.ops.attn_decode(dev(q), cache, dev(table), dev(np.array(lens, np.int32)))
    near(host(y), *U.attention(q, cache, table, lens, ps, 0.125), "bad pages")
    assert (host(y)[1] == 0).all()
    sinks = dev(np.full(8, -2.0, np.float32))
    assert (host(mx.ops.attn_decode(dev(q), cache, dev(table), dev(np.array(lens, np.int32)), sinks=sinks))[1] == 0).all()


@pytest.mark.parametrize("fmt", ["f16", "q8_0"])
def test_lengths_outside_their_range(mx, fmt):
    """Longer than the table: cut; negative: empty; longer than max_len: right all the same."""
    ps = 16
    rng, table, cache, q = case(fmt, [64, 64, 64, 50], 2, 4, 64, ps, 33)
    lens = np.array([65, 2 ** 31 - 1, -5, 50], np.int32)
    want, tol = U.attention(q, cache, table, np.minimum(lens, 64), ps, 0.125)
    for max_len in (None, 64, 1, 0, 100000):
        y = mx.ops.attn_decode(dev(q), cache, dev(table), dev(lens), max_len=max_len)
        near(host(y), want, tol, "max_len %s" % max_len)


@pytest.mark.parametrize("fmt", ["f16", "q8_0"])
def test_max_len_that_is_too_small_or_too_large(mx, fmt):
    lens = [3000, 1, 2047]
    rng, table, cache, q = case(fmt, lens, 1, 8, 128, 64, 35)
    want, tol = U.attention(q, cache, table, lens, 64, 128 ** -0.5)
    for max_len in (1, 100, 3000, 1 << 20):
        near(host(mx.ops.attn_decode(dev(q), cache, dev(table), dev(np.array(lens, np.int32)), max_len=max_len)), want, tol, "max_len %d" % max_len)


@pytest.mark.parametrize("fmt", ["f16", "q8_0"])
@pytest.mark.parametrize("scale", [0.0, 0.125, 3.0, -1.0])
def test_steep_and_flat_softmax(mx, fmt, scale):
    """Scores up to hundreds apart: the running maximum moves, and most weights vanish."""
    lens = [900, 37]
    rng, table, cache, q = case(fmt, lens, 2, 4, 64, 16, 41, k_scale=4.0)
    y = mx.ops.attn_decode(dev(q), cache, dev(table), dev(np.array(lens, np.int32)), scale=scale)
    near(host(y), *U.attention(q, cache, table, lens, 16, scale), "scale %g" % scale)


@pytest.mark.parametrize("fmt", ["f16", "q8_0"])
def test_small_values_keep_their_precision(mx, fmt):
    """Values below fp16's normal range, Q8_0 scales among them: nothing is rounded together with the scale."""
    lens = [333, 5]
    rng, table, cache, q = case(fmt, lens, 1, 4, 64, 16, 43)
    if fmt == "f16":
        cache[1].mul_(2.0 ** -14)
    else:
        cache[3].mul_(2.0 ** -14)
    want, tol = U.attention(q, cache, table, lens, 16, 0.125)
    near(host(mx.ops.attn_decode(dev(q), cache, dev(table), dev(np.array(lens, np.int32)))), want, tol, "small values")


@pytest.mark.parametrize("fmt", ["f16", "q8_0"])
@pytest.mark.parametrize("n", [480, 6000])
@pytest.mark.parametrize("gap", [17.5, 20.0])
def test_many_small_weights_are_not_lost(mx, fmt, n, gap):
    """The first token of every tile outweighs each of the others by e^gap, which is below fp16's smallest step, but only they have values.  Of a value: its rounding,
    2^-20 for the parts and sums and the score's error as elsewhere (one product, 2^-24 of it, and 2^-21 in its exponential); of all values 2^-40 of the largest weight."""
    kv = np.zeros((2, 1, 1, -(-n // 16) * 16, 64), np.float32)
    kv[0, ..., 0] = -gap
    kv[0, 0, 0, ::32, 0] = 0.0
    kv[1] = 512.0
    kv[1, 0, 0, ::32] = 0.0
    cache = tuple(dev(t.astype(np.float16)) for t in kv) if fmt == "f16" else tuple(dev(p) for t in kv for p in U.q8_0(t))
    q = np.zeros((1, 2, 64), np.float16)
    q[..., 0] = 8.0
    table, lens, ps = np.zeros((1, 1), np.int32), np.array([n], np.int32), kv.shape[3]
    want, _ = U.attention(q, cache, table, lens, ps, 0.125)
    tol = want * (2.0 ** -11 + 2.0 ** -20 + 3 * gap * (2.0 ** -21 + 80 * 2.0 ** -24)) + 2.0 ** -25 + 2.0 ** -40 * 512 * 32
    near(host(mx.ops.attn_decode(dev(q), cache, dev(table), dev(lens))), want, tol, "small weights")


@pytest.mark.parametrize("fmt", ["f16", "q8_0"])
def test_scores_of_many_sizes(mx, fmt):
    """Scores from 2^-8 to 2^29, of either sign, one sequence each: around them the distance between neighbouring 32-bit numbers passes 1.  All of a sequence are equal, so the
    result is the mean of its values; a score's rounding is the same for all."""
    B, n, ps = 76, 520, 544
    size = np.concatenate([s * 2.0 ** np.arange(-8, 30) for s in (1, -1)])
    kv = np.zeros((2, 1, 1, ps, 64), np.float32)
    kv[0, ..., 0] = 127.0 * 128
    kv[1] = np.random.default_rng(5).integers(-127, 128, (ps, 64))
    kv[1, ..., ::32] = 127.0
    cache = tuple(dev(t.astype(np.float16)) for t in kv) if fmt == "f16" else tuple(dev(p) for t in kv for p in U.q8_0(t))
    q = np.zeros((B, 2, 64), np.float16)
    q[..., 0] = (size * 2.0 ** -14 / (127.0 / 128))[:, None]
    table, lens = np.zeros((B, 1), np.int32), np.full(B, n, np.int32)
    want = U.stored(cache)[1][0, 0, :n].mean(0)
    y = host(mx.ops.attn_decode(dev(q), cache, dev(table), dev(lens), scale=1.0)).astype(np.float64)
    near(y, np.broadcast_to(want, y.shape), np.abs(want) * 2.0 ** -11 + 2.0 ** -20 * 127, "equal scores")


def test_nan_and_infinity_of_a_sequence_stay_with_it(mx):
    lens = [70, 70, 70]
    for fmt in ("f16", "q8_0"):
        rng, table, cache, q = case(fmt, lens, 2, 4, 64, 16, 47)
        want, tol = U.attention(q, cache, table, lens, 16, 0.125)
        (cache[0] if fmt == "f16" else cache[1])[int(table[1, 2]), 1, 3, 0] = float("nan")
        y = host(mx.ops.attn_decode(dev(q), cache, dev(table), dev(np.array(lens, np.int32))))
        assert np.isnan(y[1, 4:]).all()
        y[1, 4:] = want[1, 4:]
        near(y, want, tol, "the other heads and sequences")


@pytest.mark.parametrize("fmt", ["f16", "q8_0"])
@pytest.mark.parametrize("lens,G,D", [([5, 0, 900], 4, 128), ([2000], 8, 64), ([33], 16, 256), ([100, 3], 2, 96)])
def test_q8_stream_is_the_quantizer_s(mx, fmt, lens, G, D):
    rng, table, cache, q = case(fmt, lens, 2, G, D, 16, 51)
    n = len(lens) * 2 * G * D
    stream = torch.full((n // 32 * 40,), 99, dtype=torch.uint8, device="cuda")
    y = mx.ops.attn_decode(dev(q), cache, dev(table), dev(np.array(lens, np.int32)), out_q8=stream)
    assert torch.equal(stream, mx.ops.quantize_q8_1(y))


def test_strided_queries_and_given_buffers(mx):
    lens = [900, 31, 0]
    rng, table, cache, q = case("f16", lens, 2, 4, 128, 16, 53)
    wide = torch.randn(3, 12 * 128, dtype=torch.float16, device="cuda")
    wide[:, 128: 9 * 128] = dev(q).view(3, -1)
    part, args = wide[:, 128: 9 * 128].view(3, 8, 128), (cache, dev(table), dev(np.array(lens, np.int32)))
    want = mx.ops.attn_decode(dev(q), *args)
    need = mx.ops.attn_decode_ws_bytes(3, 8, 2, 128, table.shape[1] * 16)
    ws = torch.full((max(16, need) // 4,), float("nan"), device="cuda")
    out = torch.full((4, 8, 128), 5.0, dtype=torch.float16, device="cuda")
    mx.ops.attn_decode(part, *args, out=out[:3], ws=ws)
    assert torch.equal(out[:3], want) and (out[3] == 5).all()


def test_the_same_bits_every_time_and_on_every_stream(mx):
    lens = [5000, 700, 1, 0, 2500]
    rng, table, cache, q = case("q8_0", lens, 2, 8, 128, 64, 57)
    args = (dev(q), cache, dev(table), dev(np.array(lens, np.int32)))
    want = mx.ops.attn_decode(*args)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(mx.ops.attn_decode(*args))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in got)


def test_two_captured_graphs_that_grow(mx):
    """Two graphs captured after one another, replayed in turns and on two streams, with lengths that change in their buffers."""
    rng, table, cache, q = case("f16", [1000, 1000], 2, 4, 128, 16, 59)
    tab, graphs = dev(table), []
    for i in range(2):
        lens, qi = dev(np.array([1, 1], np.int32)), dev(q).clone()
        mx.ops.attn_decode(qi, cache, tab, lens)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = mx.ops.attn_decode(qi, cache, tab, lens)
        graphs.append((g, lens, qi, out))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for n in (1, 17, 400, 1000, 3):
        for i, (g, lens, qi, out) in enumerate(graphs):
            lens.copy_(torch.tensor([n, max(0, n - 5 * i)], dtype=torch.int32))
            qi.normal_()
        torch.cuda.synchronize()
        for (g, *_), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for g, lens, qi, out in graphs:
            assert torch.equal(out, mx.ops.attn_decode(qi, cache, tab, lens)), n


@pytest.mark.parametrize("fmt", ["f16", "q8_0"])
def test_offsets_past_32_bits(mx, fmt):
    """The last pages of a plane of more than 4 GiB, through writing, attention and reading back."""
    Hkv, D, ps = 8, 128, 64
    n_pages = (2 ** 32 // (Hkv * D * ps * (2 if fmt == "f16" else 1))) + 3
    cache = tuple(torch.empty(s, dtype=t, device="cuda") for s, t in
                  (((n_pages, Hkv, ps, D), torch.float16),) * 2) if fmt == "f16" else tuple(
        torch.empty(s, dtype=t, device="cuda") for _ in range(2) for s, t in (((n_pages, Hkv, ps, D), torch.int8), ((n_pages, Hkv, ps, D // 32), torch.float16)))
    rng = np.random.default_rng(61)
    table = np.array([[n_pages - 1, 0, n_pages - 2]], np.int32)
    n = 150
    k, v = (O.round_fp16(rng.standard_normal((n, Hkv, D)).astype(np.float32)).astype(np.float16) for _ in range(2))
    t = np.arange(n)
    mx.ops.kv_write(dev(k), dev(v), dev((table[0, t // ps].astype(np.int64) * ps + t % ps).astype(np.int32)), cache)
    small = tuple(c[torch.tensor([n_pages - 1, 0, n_pages - 2], device="cuda")] for c in cache)   # the same pages in a cache of three
    tiny = dev(np.array([[0, 1, 2]], np.int32))
    rows = dev(np.array([0, n], np.int32))
    got, want = mx.ops.kv_read(cache, dev(table), rows, n), mx.ops.kv_read(small, tiny, rows, n)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    if fmt == "f16":
        assert torch.equal(got[0], dev(k)) and torch.equal(got[1], dev(v))
    q, lens = dev(rng.standard_normal((1, 32, D)).astype(np.float16)), dev(np.array([n], np.int32))
    assert torch.equal(mx.ops.attn_decode(q, cache, dev(table), lens), mx.ops.attn_decode(q, small, tiny, lens))


@pytest.mark.parametrize("fmt", ["f16", "q8_0"])
def test_a_decode_step_between_its_projections(mx, fmt):
    """Norm, q/k/v products, rotation and cache, attention, output projection, token after token, through the entry points as a layer calls
    them; against the same layer in 64 bits on the values that the products gave."""
    from machx_inference_engine_amd import synth
    ops, H, Hq, Hkv, D, ps, B = mx.ops, 512, 8, 2, 64, 16, 3
    rng = np.random.default_rng(71)
    Wqkv, Wo = synth.normal_weights("q8_0", (Hq + 2 * Hkv) * D, H, seed=72), synth.normal_weights("q8_0", H, Hq * D, seed=73)
    freqs, mscale = ops.rope_freqs(D, base=10000.0)
    f, table = freqs.cuda(), rng.permutation(6).reshape(B, 2).astype(np.int32)
    cache, tab, norm_w = ops.kv_cache(fmt, 6, Hkv, ps, D), dev(table), torch.ones(H, device="cuda")
    cache[0].fill_(float("nan")) if fmt == "f16" else cache[1].fill_(float("nan"))
    stream = torch.empty(B * Hq * D // 32 * 40, dtype=torch.uint8, device="cuda")
    keys, values = [], []
    for t in range(20):
        x = torch.randn(B, H, dtype=torch.float16, device="cuda")
        _, xq = ops.rms_norm_f32w_q8(x, norm_w, 1e-5)
        qkv = ops.gemv_q8_0_q8_batched(xq, Wqkv, H, (Hq + 2 * Hkv) * D, B)
        q, k, v = (p.view(B, -1, D) for p in qkv.split((Hq * D, Hkv * D, Hkv * D), 1))
        pos, slots = np.full(B, t, np.int32), (table[:, t // ps] * ps + t % ps).astype(np.int32)
        qr = ops.rope_kv_write(q, k, v, dev(pos), dev(slots), cache, f, mscale=mscale)
        y = ops.attn_decode(qr, cache, tab, dev(pos + 1), out_q8=stream)
        want, tol = U.attention(host(qr), cache, table, pos + 1, ps, D ** -0.5)
        near(host(y), want, tol, "token %d" % t)
        assert torch.equal(ops.gemv_q8_0_q8_batched(stream, Wo, Hq * D, H, B), ops.gemv_q8_0_q8_batched(ops.quantize_q8_1(y), Wo, Hq * D, H, B))
        keys.append(U.rope(host(k), pos, host(f), False))
        values.append(host(v).astype(np.float64))
    # the cache holds every token's rotated keys and values
    got = [host(g).astype(np.float64).reshape(B, 20, Hkv, D) for g in ops.kv_read(cache, tab, dev(np.arange(0, 20 * B + 1, 20, dtype=np.int32)), 20 * B)]
    for g, w in zip(got, (np.stack(keys, 1), np.stack(values, 1))):
        step = np.abs(w).reshape(w.shape[:-1] + (-1, 32)).max(-1).repeat(32, -1) / 127
        # fp16: half a step of it, twice (rotation, and the reference's 32-bit part of it far below); Q8_0: half a step of the block, its scale's rounding, and
        # the value's own two roundings to fp16
        assert (np.abs(g - w) <= 2.0 ** -10 * np.abs(w) + 2.0 ** -24 + (0.5 * step * (1 + 2.0 ** -9) + 2.0 ** -10 * np.abs(w) if fmt == "q8_0" else 0)).all()


@pytest.mark.parametrize("D", [32, 64, 96, 128, 160, 256])
def test_largest_values_of_a_q8_0_cache(mx, D):
    """65504 is stored as 127 * 516 = 65532, which fp16 does not hold: weighed with others it counts as that, alone it rounds to infinity, and the block's other values are
    what they are.  Signs alternate from token to token and weights are nearly equal, so that sums of two or more are finite."""
    lens, Hkv, G, ps = [1000, 3, 40, 2], 2, 4, 16
    rng = np.random.default_rng(81 + D)
    table, n_pages = U.pages_of(lens + [1], ps, rng)
    cache = mx.ops.kv_cache("q8_0", n_pages, Hkv, ps, D)
    for b, n in enumerate(lens + [1]):
        t = np.arange(n)
        k, v = ((rng.uniform(-1, 1, (n, Hkv, D)) * s).astype(np.float16) for s in (0.05, 30000))
        v[..., ::5] = np.where(t % 2, -65504, 65504)[:, None, None]
        mx.ops.kv_write(dev(k), dev(v), dev((table[b, t // ps] * ps + t % ps).astype(np.int32)), cache)
    q = rng.standard_normal((5, Hkv * G, D)).astype(np.float16)
    want, tol = U.attention(q, cache, table, lens + [1], ps, D ** -0.5)
    y = host(mx.ops.attn_decode(dev(q), cache, dev(table), dev(np.array(lens + [1], np.int32))))
    near(y[:4], want[:4], tol[:4], "largest values")
    assert (want[4, :, ::5] == 65532).all() and (y[4, :, ::5] == np.inf).all()
    y[4, :, ::5] = want[4, :, ::5] = 0
    near(y[4], want[4], tol[4], "beside the largest values")


@pytest.mark.parametrize("steep", [1.0, 15.0])
@pytest.mark.parametrize("D,G,ps", [(64, 8, 16), (48, 3, 32), (128, 4, 16), (112, 2, 48), (256, 2, 16), (128, 17, 64)])
def test_infinite_values_of_an_fp16_cache(mx, D, G, ps, steep):
    """An element is infinite where one token's value is, whatever that token's weight, and NaN where infinities of either sign or a NaN are; all others are what they were."""
    lens = [900, 40, 5, 1, 0, 130]
    rng, table, cache, q = case("f16", lens, 2, G, D, ps, 83 + D, k_scale=steep)
    for b, n in enumerate(lens):
        for t in rng.integers(0, max(n, 1), 6) if n else ():
            for i, x in enumerate((np.inf, -np.inf, np.inf if rng.random() < 0.5 else -np.inf, np.nan)):
                cache[1][int(table[b, t // ps]), int(rng.integers(0, 2)), int(t) % ps, 4 * i + int(rng.integers(0, 2))] = float(x)
    with np.errstate(invalid="ignore"):
        want, tol = U.attention(q, cache, table, lens, ps, D ** -0.5)
    y = host(mx.ops.attn_decode(dev(q), cache, dev(table), dev(np.array(lens, np.int32)))).astype(np.float64)
    bad = ~np.isfinite(want)
    assert bad.any() and np.array_equal(y[bad], want[bad], equal_nan=True)
    near(np.where(bad, 0, y), np.where(bad, 0, want), np.where(bad, 1, tol), "beside infinities")


@pytest.mark.parametrize("D", [64, 96, 256])
def test_a_q8_0_block_that_holds_no_number(mx, D):
    """A value block written with a NaN or an infinity is NaN for every head that reads it; the blocks beside it and the other heads are what they were."""
    lens, Hkv, G, ps = [700, 20], 2, 3, 16
    rng = np.random.default_rng(91 + D)
    table, n_pages = U.pages_of(lens, ps, rng)
    cache = mx.ops.kv_cache("q8_0", n_pages, Hkv, ps, D)
    bad = np.zeros((2, Hkv * G, D), bool)
    for b, n in enumerate(lens):
        t = np.arange(n)
        k, v = (rng.standard_normal((n, Hkv, D)).astype(np.float16) for _ in range(2))
        v[n // 2, b, 33 * b + 5] = (np.nan, -np.inf)[b]
        bad[b, b * G: (b + 1) * G, 32 * b: 32 * b + 32] = True
        mx.ops.kv_write(dev(k), dev(v), dev((table[b, t // ps] * ps + t % ps).astype(np.int32)), cache)
    q = rng.standard_normal((2, Hkv * G, D)).astype(np.float16)
    with np.errstate(invalid="ignore"):
        want, tol = U.attention(q, cache, table, lens, ps, D ** -0.5)
    y = host(mx.ops.attn_decode(dev(q), cache, dev(table), dev(np.array(lens, np.int32))))
    assert np.isnan(y[bad]).all()
    near(np.where(bad, 0, y), np.where(bad, 0, want), np.where(bad, 1, tol), "beside the block")
