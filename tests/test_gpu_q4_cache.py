"""GPU: the Q4_0 key-value cache, written with and without rotation and read back, and the attention of one token over it, against plain forms in 64 bits."""
import gc

import numpy as np
import pytest
import torch

import kv_util as U
import oracle as O
import q4_util as Q
from gpu_util import dev, host

pytestmark = pytest.mark.gpu


def rows(rng, T, H, D, scale=1.0):
    return O.round_fp16((rng.standard_normal((T, H, D)) * scale).astype(np.float32)).astype(np.float16)


def slots_for(rng, T, n_pages, ps):
    return rng.permutation(n_pages * ps)[:T].astype(np.int32)


def near(got, want, tol, what):
    got = np.asarray(got, np.float64)
    assert np.isfinite(got).all(), what + ": not finite"
    off = np.abs(got - want)
    worst = np.unravel_index(np.argmax(off - tol), off.shape)
    assert (off <= tol).all(), "%s: at %s %.6e instead of %.6e, %.2e allowed (%d of %d)" % (what, worst, got[worst], want[worst], tol[worst], (off > tol).sum(), off.size)


# ------------------------------------------------------------------------------------------------------------------- writing and reading
@pytest.mark.parametrize("T,Hkv,D,ps", [(1, 8, 128, 16), (13, 1, 32, 48), (200, 3, 96, 16), (37, 8, 64, 256), (5, 2, 256, 32), (700, 2, 64, 16), (512, 1, 96, 64), (1000, 3, 128, 32), (600, 1, 192, 16)])
@pytest.mark.parametrize("kind", ["normal", "borders", "all"])
def test_kv_write(mx, T, Hkv, D, ps, kind):
    """The planes are the exact encoding of the rows bit for bit; every other slot is as it was.  "borders": 8 x / m + 8.5 is a whole number for every second element, and many share the largest
    magnitude; "all": every fp16 number."""
    rng = np.random.default_rng(T + D)
    n_pages = -(-T // ps) + 2
    k, v = rows(rng, T, Hkv, D), rows(rng, T, Hkv, D, 3.0)
    if kind == "borders":
        k, v = (((rng.integers(0, 33, k.shape) - 16) / 16 * s).astype(np.float16) for s in (1.0, 2.0 ** -20))
    if kind == "all":
        k = rng.integers(0, 0x7C00, k.shape).astype(np.uint16).view(np.float16) * rng.choice([1, -1], k.shape).astype(np.float16)
    k[0, 0, :32] = 0                       # a block of zeros
    slots = slots_for(rng, T, n_pages, ps)
    cache = Q.random_cache(rng, n_pages, Hkv, ps, D)
    want = [t.clone() for t in cache]
    at = torch.from_numpy(slots).cuda().long()
    for w, p in zip(want, Q.q4_0(k) + Q.q4_0(v)):
        w[at // ps, :, at % ps] = dev(p)
    mx.ops.kv_write(dev(k), dev(v), dev(slots), cache)
    for c, w in zip(cache, want):
        assert torch.equal(c.view(torch.uint8), w.view(torch.uint8))


def test_codes_are_the_weight_formats(mx):
    """Beside a border, where that encoder's 32-bit quotient may round to the other side, they are the encoding of the weights of that name."""
    rng = np.random.default_rng(8)
    x = rows(rng, 64, 2, 128)
    blocks = O.quantize(O.Q4_0, x.astype(np.float32).reshape(-1, 128)).reshape(-1, 18)
    codes, d = Q.q4_0(x)
    assert np.array_equal(d.reshape(-1).view(np.uint16), blocks[:, :2].copy().view(np.uint16).ravel())
    b = x.astype(np.float64).reshape(-1, 32)
    m = np.take_along_axis(b, np.abs(b).argmax(1)[:, None], 1)
    t = b * -8 / m + 8.5
    clear = (np.abs(t - np.round(t)) > 1e-5).all(1)
    assert clear.mean() > 0.9 and np.array_equal(codes.reshape(-1, 16)[clear], blocks[clear, 2:])


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("T,Hq,Hkv,D,n_rot,ps", [(1, 32, 8, 128, 128, 16), (9, 64, 8, 64, 64, 32), (50, 7, 1, 96, 48, 16), (21, 16, 2, 256, 64, 64), (3, 5, 5, 32, 16, 16), (700, 8, 2, 64, 64, 16),
                                                  (530, 6, 3, 128, 64, 48), (512, 4, 1, 96, 96, 32), (600, 2, 2, 256, 64, 16)])
def test_rope_kv_write_is_rope_then_write(mx, inter, T, Hq, Hkv, D, n_rot, ps):
    """One launch gives the bits of rope and kv_write, whether the rows are parts of a fused projection or not, and with q rotated in place."""
    rng = np.random.default_rng(T + Hq)
    n_pages = -(-T // ps) + 1
    qkv = dev(rows(rng, T, 1, (Hq + 2 * Hkv) * D)).view(T, -1)
    q, k, v = (t.view(T, -1, D) for t in qkv.split((Hq * D, Hkv * D, Hkv * D), 1))
    pos, slots, f = dev(rng.integers(0, 100000, T).astype(np.int32)), dev(slots_for(rng, T, n_pages, ps)), dev(U.freqs(n_rot))
    a = Q.random_cache(rng, n_pages, Hkv, ps, D)
    b, c = tuple(t.clone() for t in a), tuple(t.clone() for t in a)
    want = mx.ops.rope(q, pos, f, interleaved=inter, mscale=0.75)
    mx.ops.kv_write(mx.ops.rope(k, pos, f, interleaved=inter, mscale=0.75), v, slots, a)
    assert torch.equal(mx.ops.rope_kv_write(q, k, v, pos, slots, b, f, interleaved=inter, mscale=0.75), want)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    kept = qkv.clone()
    mx.ops.rope_kv_write(q, k, v, pos, slots, c, f, interleaved=inter, mscale=0.75, q_out=q)
    assert all(torch.equal(x, y) for x, y in zip(a, c)) and torch.equal(q, want) and torch.equal(qkv[:, Hq * D:], kept[:, Hq * D:])


@pytest.mark.parametrize("T", [6, 600])
def test_blocks_without_numbers_and_slots_outside(mx, T):
    """A block that holds a NaN or an infinity reads back as NaN, its neighbours as they are; a slot outside the cache writes nothing."""
    rng = np.random.default_rng(T)
    k, v = rows(rng, T, 2, 64), rows(rng, T, 2, 64)
    k[1, 0, 3], k[2, 1, 40], v[0, 1, 63], v[3, 0, 0] = np.nan, np.inf, -np.inf, np.nan
    slots = np.arange(T, dtype=np.int32)[::-1].copy()
    slots[4], slots[5] = -1, 16 * 40
    cache = mx.ops.kv_cache("q4_0", 40, 2, 16, 64)
    mx.ops.kv_write(dev(k), dev(v), dev(slots), cache)
    K, V = mx.ops.kv_read(cache, dev(np.arange(40, dtype=np.int32)[None]), dev(np.array([0, T], np.int32)), T)
    K, V = host(K).astype(np.float64)[::-1], host(V).astype(np.float64)[::-1]
    for got, x in ((K, k), (V, v)):
        want = Q.values(*Q.q4_0(np.nan_to_num(x, nan=0, posinf=0, neginf=0)))
        bad = ~np.isfinite(x.reshape(T, 2, 2, 32)).all(-1, keepdims=True).repeat(32, -1).reshape(x.shape)
        want[4] = want[5] = 0.0
        bad[4] = bad[5] = False
        assert np.array_equal(np.isnan(got), bad)
        assert np.array_equal(got[~bad], want.astype(np.float32).astype(np.float16).astype(np.float64)[~bad])


@pytest.mark.parametrize("lens,Hkv,D,ps", [([1, 0, 17, 33], 2, 64, 16), ([5, 48, 0, 0, 100], 1, 32, 48), ([40], 3, 96, 16), ([31, 32], 1, 256, 32), ([9000, 1], 4, 128, 64), ([i % 5 for i in range(150)], 1, 32, 16),
                                           ([70000], 8, 128, 256)])
def test_kv_read(mx, lens, Hkv, D, ps):
    """The products of codes and scales, which 32 bits hold exactly, rounded once; rows behind the last sequence are as they were, bad pages read as zeros."""
    rng = np.random.default_rng(D + len(lens))
    table, n_pages = U.pages_of(lens, ps, rng)
    cache = tuple(torch.randint(0, 256, (n_pages, Hkv, ps, D // 2), dtype=torch.uint8, device="cuda") if i % 2 == 0 else torch.randn(n_pages, Hkv, ps, D // 32, device="cuda").half() for i in range(4))
    total, spare = sum(lens), 3
    if sum(lens) > 100:
        table[0, -1 if lens[0] == max(lens) else 0] = -5
    out = tuple(torch.full((total + spare, Hkv, D), 7.0, dtype=torch.float16, device="cuda") for _ in range(2))
    rows_ = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    mx.ops.kv_read(cache, dev(table), dev(rows_), total + spare, out=out)
    b, t = np.repeat(np.arange(len(lens)), lens), np.concatenate([np.arange(n) for n in lens])
    page = torch.from_numpy(table).cuda().long()[torch.from_numpy(b).cuda(), torch.from_numpy(t // ps).cuda()]
    good, at = page >= 0, torch.from_numpy(t % ps).cuda()
    for o, codes, d in zip(out, cache[::2], cache[1::2]):
        c = codes[page.clamp(min=0), :, at].unflatten(-1, (-1, 16))
        want = ((torch.cat((c & 15, c >> 4), -1).float() - 8) * d[page.clamp(min=0), :, at].float()[..., None]).flatten(-2).half()
        want[~good] = 0
        assert torch.equal(o[:total], want) and (o[total:] == 7).all()


# ------------------------------------------------------------------------------------------------------------------- attention
def case(lens, Hkv, G, D, ps, seed, k_scale=1.0):
    rng = np.random.default_rng(seed)
    table, n_pages = U.pages_of(lens, ps, rng)
    cache = Q.keep_only(Q.random_cache(rng, n_pages, Hkv, ps, D, k_scale), table, lens, ps)
    return rng, table, cache, rows(rng, len(lens), Hkv * G, D)


def attend(mx, q, cache, table, lens, **more):
    return mx.ops.attn_decode(dev(q), cache, dev(table), dev(np.array(lens, np.int32)), **more)


LENS = {"one": [1], "edges": [0, 1, 15, 16, 17, 31, 32, 33, 47, 48, 63, 64, 65, 127, 128, 129], "none": [0, 0, 0], "mid": [700], "ragged": [1000, 3, 257, 0, 513, 64], "long": [9001, 12]}


@pytest.mark.parametrize("lens", sorted(LENS))
@pytest.mark.parametrize("Hkv,G,D,ps", [(8, 4, 128, 16), (4, 8, 128, 64), (2, 8, 64, 32), (2, 8, 256, 16), (1, 1, 64, 16), (3, 5, 96, 48), (1, 16, 128, 256)])
def test_attn_decode(mx, lens, Hkv, G, D, ps):
    lens = LENS[lens]
    rng, table, cache, q = case(lens, Hkv, G, D, ps, 100 + D + len(lens))
    want, tol = Q.attention(q, cache, table, lens, ps, D ** -0.5)
    for max_len in (None, 1 << 20):          # the longest of them, and a length that asks for parts
        y = attend(mx, q, cache, table, lens, max_len=max_len)
        near(host(y), want, tol, "max_len %s" % max_len)
        assert (host(y)[np.array(lens) == 0] == 0).all()


@pytest.mark.parametrize("D", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("G", [1, 7, 17, 40])
def test_every_width_of_head(mx, D, G):
    lens = [130, 0, 19, 1, 800]
    rng, table, cache, q = case(lens, 2, G, D, 16, D + G)
    want, tol = Q.attention(q, cache, table, lens, 16, D ** -0.5)
    for max_len in (None, 1 << 20):          # whole, in parts
        near(host(attend(mx, q, cache, table, lens, max_len=max_len)), want, tol, "D=%d G=%d max_len %s" % (D, G, max_len))


@pytest.mark.parametrize("D", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("G,Hkv", [(1, 40), (7, 3), (17, 8), (4, 64)])
def test_few_sequences_up_to_a_thousand_tokens(mx, D, G, Hkv):
    """Fewer workgroups than CUs, of more than two tiles a wave: no parts for heads of up to 128, whatever the lengths are in the end."""
    lens, most = ([1024, 0, 300, 97] if D <= 128 else [512, 0, 300, 97])[:256 // (Hkv * (1 + G // 17))], 1024 if D <= 128 else 512
    rng, table, cache, q = case(lens, Hkv, G, D, 16, 3 * D + G)
    assert mx.ops.attn_decode_ws_bytes(len(lens), Hkv * G, Hkv, D, most, fmt="q4_0") == 0
    assert mx.ops.attn_decode_ws_bytes(len(lens), Hkv * G, Hkv, D, most + 1, fmt="q4_0") > 0
    sinks = rng.standard_normal(Hkv * G).astype(np.float32)
    for window in (0, 260):
        stream = torch.empty(q.size // 32 * 40, dtype=torch.uint8, device="cuda")
        y = attend(mx, q, cache, table, lens, window=window, sinks=dev(sinks), max_len=most, out_q8=stream)
        near(host(y), *Q.attention(q, cache, table, lens, 16, D ** -0.5, window, sinks), "D=%d G=%d window %d" % (D, G, window))
        assert torch.equal(stream, mx.ops.quantize_q8_1(y)) and (host(y)[np.array(lens) == 0] == 0).all()


@pytest.mark.parametrize("window", [1, 5, 16, 33, 128, 1000])
@pytest.mark.parametrize("with_sinks", [False, True])
def test_window_and_sinks(mx, window, with_sinks):
    lens = [0, 1, 4, 5, 6, 127, 128, 129, 300, 1500]
    rng, table, cache, q = case(lens, 2, 8, 64, 16, window)
    sinks = rng.standard_normal(16).astype(np.float32) * 3 if with_sinks else None
    y = attend(mx, q, cache, table, lens, window=window, sinks=None if sinks is None else dev(sinks))
    near(host(y), *Q.attention(q, cache, table, lens, 16, 0.125, window, sinks), "window %d" % window)


@pytest.mark.parametrize("B,Hkv,G,D", [(150, 1, 4, 64), (70, 2, 24, 128), (65, 1, 2, 256), (300, 3, 1, 96), (3000, 1, 1, 32)])
def test_many_ragged_sequences_in_equal_shares(mx, B, Hkv, G, D):
    rng = np.random.default_rng(B)
    lens = [int(n) if rng.random() < 0.8 else 0 for n in np.exp(rng.uniform(0, np.log(900 if B < 1000 else 40), B))]
    lens[0] = lens[-1] = 0
    lens[B // 2] = 2500
    rng, table, cache, q = case(lens, Hkv, G, D, 16, B)
    sinks = rng.standard_normal(Hkv * G).astype(np.float32)
    near(host(attend(mx, q, cache, table, lens, sinks=dev(sinks))), *Q.attention(q, cache, table, lens, 16, D ** -0.5, sinks=sinks), "B=%d" % B)


@pytest.mark.parametrize("n", [513, 1025, 4096, 16385])
def test_one_sequence_in_shares(mx, n):
    """Lengths in front of what max_len says and behind it."""
    rng, table, cache, q = case([n], 2, 4, 64, 32, n)
    for m in (n, n - 1, n // 2, 33, 1, 0):
        want, tol = Q.attention(q, cache, table, [m], 32, 0.125)
        for max_len in (n, 600, 1, 0):
            near(host(attend(mx, q, cache, table, [m], max_len=max_len)), want, tol, "%d of %d, max_len %d" % (m, n, max_len))


def test_pages_of_sixteen_times_any_number(mx):
    for ps in (16, 48, 80, 112, 1008, 4096):
        lens = [700, 1001, 0, ps + 1]
        rng, table, cache, q = case(lens, 1, 4, 64, ps, ps)
        near(host(attend(mx, q, cache, table, lens, window=900)), *Q.attention(q, cache, table, lens, ps, 0.125, 900), "pages of %d" % ps)


def test_what_the_window_left_behind_is_not_read(mx):
    ps, window, n = 16, 40, 203
    rng, table, cache, q = case([n], 2, 4, 128, ps, 9)
    want, tol = Q.attention(q, cache, table, [n], ps, 128 ** -0.5, window)
    for t in range(n - window):
        for c in (cache[1], cache[3]):
            c[int(table[0, t // ps]), :, t % ps] = float("nan")
    table[0, : (n - window) // ps] = -7
    near(host(attend(mx, q, cache, table, [n], window=window)), want, tol, "window")


def test_pages_outside_the_cache_and_lengths_outside_their_range(mx):
    ps, lens = 16, [100, 64, 33, 500]
    rng, table, cache, q = case(lens, 2, 4, 64, ps, 31)
    table[0, 2], table[0, 3], table[3, 0], table[3, 17] = -1, 10 ** 6, -2 ** 31, 2 ** 31 - 1
    table[1, :] = -1                                           # nothing is left of this one
    y = attend(mx, q, cache, table, lens)
    near(host(y), *Q.attention(q, cache, table, lens, ps, 0.125), "bad pages")
    assert (host(y)[1] == 0).all()
    assert (host(attend(mx, q, cache, table, lens, sinks=dev(np.full(8, -2.0, np.float32))))[1] == 0).all()
    rng, table, cache, q = case([64, 64, 64, 50], 2, 4, 64, ps, 33)
    lens = np.array([65, 2 ** 31 - 1, -5, 50], np.int64)
    want, tol = Q.attention(q, cache, table, np.minimum(lens, 64), ps, 0.125)
    for max_len in (None, 64, 1, 100000):
        near(host(attend(mx, q, cache, table, lens, max_len=max_len)), want, tol, "max_len %s" % max_len)


def test_what_lies_behind_the_end_changes_no_bit(mx):
    """Codes and scales behind a sequence's end, infinite ones too, which would move what the weights are scaled by."""
    lens = [333, 5, 1000]
    rng, table, cache, q = case(lens, 2, 4, 64, 48, 5)
    other = Q.random_cache(rng, cache[0].shape[0], 2, 48, 64)
    for i in (1, 3):
        other[i].mul_(3000.0)
        other[i][..., ::2] = float("inf")
    for b, n in enumerate(lens):
        t = torch.arange(n, device="cuda")
        page, at = torch.from_numpy(table[b]).cuda().long()[t // 48], t % 48
        for o, c in zip(other, cache):
            o[page, :, at] = c[page, :, at]
    assert torch.equal(attend(mx, q, cache, table, lens), attend(mx, q, other, table, lens))


@pytest.mark.parametrize("scale", [0.0, 0.125, 3.0, -1.0])
def test_steep_and_flat_softmax(mx, scale):
    lens = [900, 37]
    rng, table, cache, q = case(lens, 2, 4, 64, 16, 41, k_scale=4.0)
    near(host(attend(mx, q, cache, table, lens, scale=scale)), *Q.attention(q, cache, table, lens, 16, scale), "scale %g" % scale)


@pytest.mark.parametrize("size", [2.0 ** -24, 2.0 ** -14, 2.0 ** -6, 2.0 ** 8, 2.0 ** 13])
def test_queries_of_any_size(mx, size):
    """Queries are scaled to fp16's range by powers of two; one of their elements is far smaller than the others."""
    lens = [300, 700]
    rng, table, cache, q = case(lens, 2, 4, 64, 16, 44)
    q = (q.astype(np.float64) * size).astype(np.float16)
    q[:, 1::3, ::7] = np.float16(2.0 ** -24)
    q[0, 3] = 0
    assert np.isfinite(q).all()
    near(host(attend(mx, q, cache, table, lens, scale=0.125 / size)), *Q.attention(q, cache, table, lens, 16, 0.125 / size), "queries of %g" % size)


@pytest.mark.parametrize("by", [2.0 ** -14, 2.0 ** 6, 2.0 ** 13])
def test_values_of_any_size(mx, by):
    """Scales below fp16's normal range, and those at whose size weights are scaled down; in the second half of the sequences first, one block of each head alone."""
    lens = [333, 5, 2100]
    rng, table, cache, q = case(lens, 1, 4, 64, 16, 43)
    for b, n in enumerate(lens):
        t = torch.arange(n // 2, n, device="cuda")
        cache[3][torch.from_numpy(table[b]).cuda().long()[t // 16], :, t % 16, 1] *= by
    want, tol = Q.attention(q, cache, table, lens, 16, 0.125)
    assert np.abs(want).max() < 65000
    near(host(attend(mx, q, cache, table, lens)), want, tol, "values of %g" % by)


def test_the_largest_values(mx):
    """Scales written elsewhere, up to fp16's largest: results beyond fp16 are infinite, others are numbers."""
    lens = [64, 700]
    rng, table, cache, q = case(lens, 1, 2, 64, 16, 45)
    cache[3][..., 0] = torch.where(cache[3][..., 0] == cache[3][..., 0], 65504.0, float("nan")).half()
    want, tol = Q.attention(q, cache, table, lens, 16, 0.125)
    got = host(attend(mx, q, cache, table, lens)).astype(np.float64)
    large = np.abs(want) > 65520 + tol
    small = np.abs(want) < 65504 - tol
    assert large.any() and small.any()
    assert np.array_equal(got[large], np.sign(want[large]) * np.inf)
    assert (np.abs(got - want)[small] <= tol[small]).all()


@pytest.mark.parametrize("n", [480, 6000])
@pytest.mark.parametrize("gap", [17.5, 20.0])
def test_many_small_weights_are_not_lost(mx, n, gap):
    """The first token of every tile outweighs each of the others by e^gap, which is below fp16's smallest step, but only they have values."""
    kv = np.zeros((2, 1, 1, -(-n // 16) * 16, 64), np.float32)
    kv[0, ..., 0] = -gap
    kv[0, 0, 0, ::32, 0] = 0.0
    kv[1] = 4.0
    kv[1, 0, 0, ::32] = 0.0
    cache = tuple(dev(p) for t in kv for p in Q.q4_0(O.round_fp16(t)))
    q = np.zeros((1, 2, 64), np.float16)
    q[..., 0] = 8.0
    table, lens, ps = np.zeros((1, 1), np.int32), [n], kv.shape[3]
    near(host(attend(mx, q, cache, table, lens)), *Q.attention(q, cache, table, lens, ps, 0.125), "small weights")


def test_scores_of_many_sizes(mx):
    """Scores up to 2^22, beyond which a maximum that lies 15 below would not be one."""
    for size in (1e3, 1e5, 1e6, 4e6):
        lens = [200, 33]
        rng, table, cache, q = case(lens, 1, 4, 64, 16, 47)
        K, V = Q.stored(cache)
        y = host(attend(mx, q, cache, table, lens, scale=size / 64)).astype(np.float64)
        assert np.isfinite(y).all()
        want, _ = Q.attention(q, cache, table, lens, 16, size / 64)
        for b, n in enumerate(lens):                       # where one token stands out by more than scores are off, the result is its value
            t = np.arange(n)
            k = K[table[b][t // 16], 0, t % 16]
            for h in range(4):
                x = np.sort(size / 64 * (k @ q[b, h].astype(np.float64)))
                if x[-1] - x[-2] > 40 + 2.0 ** -12 * abs(x[-1]):
                    assert (np.abs(y[b, h] - want[b, h]) <= 2.0 ** -11 * np.abs(want[b, h]) + 2.0 ** -19 * 8).all()


def test_values_that_are_no_numbers(mx):
    """They make their own block of the heads that read them NaN and leave everything else as it is."""
    lens = [100, 700, 40]
    rng, table, cache, q = case(lens, 2, 3, 96, 16, 51)
    clean = host(attend(mx, q, cache, table, lens))
    cache[3][int(table[0, 2]), 1, 3, 2] = float("nan")
    cache[3][int(table[1, 40]), 0, 7, 0] = float("inf")
    got = host(attend(mx, q, cache, table, lens))
    bad = np.zeros(got.shape, bool)
    bad[0, 3:, 64:] = True
    bad[1, :3, :32] = True
    assert np.array_equal(np.isnan(got), bad)
    # an infinite scale asks for no other weights than the largest there is: other results differ by their last bits at most
    want, tol = Q.attention(q, tuple(torch.nan_to_num(c, nan=0.0, posinf=0.0) if c.dtype == torch.float16 else c for c in cache), table, lens, 16, 96 ** -0.5)
    assert (np.abs(got.astype(np.float64) - clean) <= tol + 2.0 ** -10 * np.abs(clean) + 2.0 ** -20)[~bad].all()
    cache[1][int(table[2, 0]), 0, 0, 0] = float("nan")       # a key: everything of its heads
    assert np.isnan(host(attend(mx, q, cache, table, lens))[2, :3]).all()
    q[0, 0, 0], q[1, 5, 95] = np.inf, np.nan
    got = host(attend(mx, q, cache, table, lens))
    assert np.isnan(got[0, 0]).all() and np.isnan(got[1, 5]).all() and np.isfinite(got[1, 3:5]).all()


def test_strided_queries_and_the_stream_of_the_result(mx):
    lens = [100, 2000, 0, 31]
    rng, table, cache, _ = case(lens, 2, 4, 64, 16, 61)
    row = dev(rows(rng, 4, 1, 12 * 64)).view(4, 12 * 64)
    q = row[:, 128:128 + 512].view(4, 8, 64)
    stream = torch.zeros(4 * 8 * 64 // 32 * 40, dtype=torch.uint8, device="cuda")
    out = torch.empty(4, 8, 64, dtype=torch.float16, device="cuda")
    y = mx.ops.attn_decode(q, cache, dev(table), dev(np.array(lens, np.int32)), out=out, out_q8=stream)
    assert y is out and torch.equal(y, mx.ops.attn_decode(q.contiguous(), cache, dev(table), dev(np.array(lens, np.int32))))
    assert torch.equal(stream, mx.ops.quantize_q8_1(y.view(-1)))


def test_large_offsets(mx):
    """A cache of more than 2^32 codes: offsets take 64 bits."""
    n_pages, ps, Hkv, D = 4200, 1024, 8, 128
    cache = mx.ops.kv_cache("q4_0", n_pages, Hkv, ps, D)
    assert cache[0].numel() * 2 > 2 ** 32
    rng = np.random.default_rng(3)
    k, v = rows(rng, 40, Hkv, D), rows(rng, 40, Hkv, D)
    slots = (n_pages - 1) * ps + 500 + np.arange(40, dtype=np.int32)
    mx.ops.kv_write(dev(k), dev(v), dev(slots), cache)
    table, lens = np.full((1, 1), n_pages - 1, np.int32), [540]
    q = rows(rng, 1, 32, D)
    got = host(attend(mx, q, cache, table, lens, window=40))
    small = tuple(t[n_pages - 1:].clone() for t in cache)
    near(got, *Q.attention(q, small, np.zeros((1, 1), np.int32), lens, ps, D ** -0.5, 40), "far page")
    K, V = mx.ops.kv_read(cache, dev(table), dev(np.array([0, 540], np.int32)), 540)
    assert np.array_equal(host(K)[500:].astype(np.float64), Q.values(*Q.q4_0(k)).astype(np.float16).astype(np.float64))
    del cache, small
    torch.cuda.empty_cache()


def test_streams_and_captured_graphs(mx):
    """Two calls at once with a workspace each, and a step captured once and replayed with other contents, beside the program's own eager calls."""
    lens = [3000, 700, 1, 1200]
    rng, table, cache, q = case(lens, 2, 8, 128, 16, 71)
    tab, n, f = dev(table), dev(np.array(lens, np.int32)), dev(U.freqs(128))
    size = mx.ops.attn_decode_ws_bytes(4, 16, 2, 128, 3000, fmt="q4_0")
    assert size > 0
    qs = [dev(rows(rng, 4, 16, 128)) for _ in range(2)]
    want = [mx.ops.attn_decode(t, cache, tab, n, max_len=3000) for t in qs]
    streams, ws, got = [torch.cuda.Stream() for _ in qs], [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in qs], [None, None]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = mx.ops.attn_decode(qs[i], cache, tab, n, max_len=3000, ws=ws[i])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    slots = np.array([int(table[b, (m - 1) // 16]) * 16 + (m - 1) % 16 for b, m in enumerate(lens)], np.int32)
    x = dev(rows(rng, 4, 20, 128))
    parts = x[:, :16], x[:, 16:18], x[:, 18:]
    pos, slots, out = dev(np.array(lens, np.int32) - 1), dev(slots), torch.empty(4, 16, 128, dtype=torch.float16, device="cuda")

    def step(to, w):
        r = mx.ops.rope_kv_write(*parts, pos, slots, cache, f)
        return mx.ops.attn_decode(r, cache, tab, n, max_len=3000, out=to, ws=w)
    step(out, ws[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(out, ws[0])
    for seed in range(4):
        x.copy_(dev(rows(np.random.default_rng(seed), 4, 20, 128)))
        eager = step(torch.empty_like(out), ws[1]).clone()
        out.fill_(-1)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


def test_refusals(mx):
    ops = mx.ops
    cache, tab, lens = ops.kv_cache("q4_0", 4, 2, 16, 64), dev(np.zeros((3, 4), np.int32)), dev(np.ones(3, np.int32))
    q = torch.zeros(3, 8, 64, dtype=torch.float16, device="cuda")
    k = torch.zeros(3, 2, 64, dtype=torch.float16, device="cuda")
    ok = dict(q=q, cache=cache, page_table=tab, seq_lens=lens)
    ops.attn_decode(**ok)
    qs8 = ops.kv_cache("q8_0", 4, 2, 16, 64)
    for bad in (dict(q=q[..., :32]), dict(cache=cache[:3]), dict(cache=(cache[0], cache[1], qs8[2], cache[3])), dict(cache=(qs8[0], cache[1], cache[2], cache[3])),
                dict(cache=(cache[0], qs8[1][..., :1], cache[2], cache[3])), dict(cache=(cache[0].transpose(1, 2),) + cache[1:]), dict(cache=(cache[0].cpu(),) + cache[1:]),
                dict(cache=(cache[0][..., :16],) + cache[1:])):
        with pytest.raises(ValueError):
            ops.attn_decode(**{**ok, **bad})
    for bad in (dict(cache=ops.kv_cache("q4_0", 4, 2, 24, 64)), dict(max_len=100000, ws=torch.zeros(16, device="cuda")), dict(q=torch.zeros(3, 7, 64, dtype=torch.float16, device="cuda"))):
        with pytest.raises(mx.ops.MxError):
            ops.attn_decode(**{**ok, **bad})
    for fn in (lambda: ops.kv_cache("q4_0", 4, 2, 16, 80), lambda: ops.kv_cache("q4_1", 4, 2, 16, 64), lambda: ops.kv_write(k[..., :32], k, lens, cache), lambda: ops.kv_write(k, k, lens.long(), cache),
               lambda: ops.kv_read(cache, tab, dev(np.zeros(3, np.int32)), 5)):
        with pytest.raises(ValueError):
            fn()


@pytest.mark.parametrize("fmt", ["f16", "q8_0", "q4_0"])
def test_a_new_cache_takes_its_own_bytes(mx, fmt):
    gc.collect()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    cache = mx.ops.kv_cache(fmt, 512, 8, 64, 128)
    size = sum(t.numel() * t.element_size() for t in cache)
    # torch's allocator may hand out a block of up to 1 MiB more for each
    assert size <= torch.cuda.max_memory_allocated() - before <= size + (len(cache) << 20) and len({t.data_ptr() for t in cache}) == len(cache) and all((t == 0).all() for t in cache)
    with pytest.raises(ValueError):
        mx.ops.attn_decode_ws_bytes(1, 8, 8, 128, 4096, fmt="q4")


def test_queries_that_are_no_numbers(mx):
    """Such a head is NaN, its neighbours in the same products have the bits that they have beside a number; without tokens it is zeros."""
    lens = [0, 40, 700, 1]
    rng, table, cache, q = case(lens, 2, 8, 128, 16, 5)
    want = host(attend(mx, q, cache, table, lens))
    heads = {1: np.inf, 6: np.nan, 11: -np.inf}
    for h, x in heads.items():
        q[:, h, 3 * h % 128] = x
    y = host(attend(mx, q, cache, table, lens))
    others = [h for h in range(16) if h not in heads]
    assert np.isnan(y[1:, list(heads)]).all() and (y[0] == 0).all() and np.array_equal(y[:, others].view(np.uint16), want[:, others].view(np.uint16))
