"""GPU: rotary positions, writing the paged key-value cache (fp16 and Q8_0) and reading it back, against plain forms in 64 bits."""
import numpy as np
import pytest
import torch

import kv_util as U
import oracle as O
from gpu_util import dev, host

pytestmark = pytest.mark.gpu


def rows(rng, T, H, D, scale=1.0):
    return O.round_fp16((rng.standard_normal((T, H, D)) * scale).astype(np.float32)).astype(np.float16)


def near(got, want, tol, what):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    limit = tol + 2.0 ** -11 * np.abs(want) + 2.0 ** -25
    off = np.abs(got - want)
    assert (off <= limit).all(), "%s: off by %.3e where %.3e is allowed (%d of %d)" % (what, off.max(), limit.flat[np.argmax(off - limit)], (off > limit).sum(), off.size)


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("T,H,D,n_rot", [(1, 40, 128, 128), (3, 1, 16, 16), (7, 3, 64, 64), (5, 18, 256, 64), (2, 5, 80, 32), (33, 7, 96, 96), (4, 9, 112, 48),
                                         (300, 40, 128, 128), (6, 2, 256, 256), (2, 65, 32, 16), (512, 3, 64, 64), (777, 5, 128, 32),
                                         (600, 9, 80, 48), (513, 2, 256, 128), (70001, 2, 16, 16)])
def test_rope(mx, T, H, D, n_rot, inter):
    rng = np.random.default_rng(T * 1000 + D + n_rot)
    x, f = rows(rng, T, H, D), U.freqs(n_rot, 500000.0)
    pos = np.concatenate([[0], rng.integers(0, 1 << 20, T)])[:T].astype(np.int32) if T > 1 else np.array([131071], np.int32)
    y = mx.ops.rope(dev(x), dev(pos), dev(f), interleaved=inter, mscale=1.25)
    near(host(y), U.rope(x, pos, f, inter, np.float64(np.float32(1.25))), U.rope_tol(x, f, inter, 1.25), "rope")
    assert np.array_equal(host(y)[..., n_rot:].view(np.uint16), x[..., n_rot:].view(np.uint16))


@pytest.mark.parametrize("inter", [False, True])
def test_rope_keeps_far_angles(mx, inter):
    """Positions up to 2^31 - 1, where 32-bit angles have lost every digit."""
    rng = np.random.default_rng(5)
    pos = np.array([2 ** 31 - 1, 2 ** 30 + 7, 16777217, -3, 0, 1], np.int32)
    x, f = rows(rng, len(pos), 4, 64), U.freqs(64)
    # 64-bit angles up to 2^31 radians are off by 2^31 * 2^-53 radians from their own rounding, and as much again on the way to turns
    y = mx.ops.rope(dev(x), dev(pos), dev(f), interleaved=inter)
    near(host(y), U.rope(x, pos, f, inter), U.rope_tol(x, f, inter) + 2.0 ** -19 * np.abs(x).max(), "far positions")


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("T", [37, 600])
@pytest.mark.parametrize("H,D,n_rot", [(40, 128, 128), (70, 64, 32), (3, 256, 256), (5, 96, 48)])
def test_rope_in_place_and_strided(mx, T, H, D, n_rot, inter):
    rng = np.random.default_rng(11)
    wide = (H + 5) * D + 8
    buf = dev(rows(rng, T, 1, wide)).view(T, wide)
    f, pos = dev(U.freqs(n_rot)), dev(np.arange(100, 100 + T, dtype=np.int32))
    part = buf[:, 8 + 2 * D: 8 + (H + 2) * D].view(T, H, D)
    want = mx.ops.rope(part.contiguous(), pos, f, interleaved=inter)
    before = buf.clone()
    y = torch.full((T, H + 2, D), 7.0, dtype=torch.float16, device="cuda")
    mx.ops.rope(part, pos, f, interleaved=inter, y=y[:, :H])
    assert torch.equal(y[:, :H], want) and (y[:, H:] == 7).all() and torch.equal(buf, before)
    mx.ops.rope(part, pos, f, interleaved=inter, y=part)
    assert torch.equal(part, want)
    before[:, 8 + 2 * D: 8 + (H + 2) * D] = want.view(T, -1)
    assert torch.equal(buf, before), "what lies beside the rotated heads has changed"


def test_a_nan_stays_in_its_pair(mx):
    x = torch.ones(2, 3, 64, dtype=torch.float16, device="cuda")
    x[1, 1, 5] = float("nan")
    x[0, 2, 40] = float("inf")
    for inter in (False, True):
        y = mx.ops.rope(x, dev(np.array([3, 4], np.int32)), dev(U.freqs(64)), interleaved=inter)
        bad = set(map(tuple, torch.nonzero(~torch.isfinite(y)).tolist()))
        a, b = (4, 41) if inter else (37, 8)
        assert bad == {(1, 1, 5), (1, 1, a), (0, 2, 40), (0, 2, b)}


def slots_for(rng, T, n_pages, ps):
    return rng.permutation(n_pages * ps)[:T].astype(np.int32)


@pytest.mark.parametrize("fmt", ["f16", "q8_0"])
@pytest.mark.parametrize("T,Hkv,D,ps", [(1, 8, 128, 16), (13, 1, 32, 48), (200, 3, 96, 16), (37, 8, 64, 256), (5, 2, 256, 32), (700, 2, 64, 16), (512, 1, 96, 64),
                                         (1000, 3, 128, 32)])
def test_kv_write(mx, fmt, T, Hkv, D, ps):
    """The planes are the oracle's encoding of the rows bit for bit; every other slot is as it was."""
    rng = np.random.default_rng(T + D)
    n_pages = -(-T // ps) + 2
    k, v = rows(rng, T, Hkv, D), rows(rng, T, Hkv, D, 3.0)
    k[0, 0, :32] = 0                       # a block of zeros
    slots = slots_for(rng, T, n_pages, ps)
    cache = U.random_cache(fmt, rng, n_pages, Hkv, ps, D)
    want = [t.clone() for t in cache]
    planes = (k, v) if fmt == "f16" else U.q8_0(k) + U.q8_0(v)
    at = torch.from_numpy(slots).cuda().long()
    for w, p in zip(want, planes):
        w[at // ps, :, at % ps] = dev(p)
    mx.ops.kv_write(dev(k), dev(v), dev(slots), cache)
    for c, w in zip(cache, want):
        assert torch.equal(c, w)


@pytest.mark.parametrize("fmt", ["f16", "q8_0"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("T,Hq,Hkv,D,n_rot,ps", [(1, 32, 8, 128, 128, 16), (9, 64, 8, 64, 64, 32), (50, 7, 1, 96, 48, 16), (21, 16, 2, 256, 64, 64), (3, 5, 5, 32, 16, 16), (700, 8, 2, 64, 64, 16),
                                                  (530, 6, 3, 128, 64, 48), (512, 4, 1, 96, 96, 32), (600, 2, 2, 256, 64, 16)])
def test_rope_kv_write_is_rope_then_write(mx, fmt, inter, T, Hq, Hkv, D, n_rot, ps):
    """One launch gives the bits of rope and kv_write, whether the rows are parts of a fused projection or not, and with q rotated in place."""
    rng = np.random.default_rng(T + Hq)
    n_pages = -(-T // ps) + 1
    qkv = dev(rows(rng, T, 1, (Hq + 2 * Hkv) * D)).view(T, -1)
    q, k, v = (t.view(T, -1, D) for t in qkv.split((Hq * D, Hkv * D, Hkv * D), 1))
    pos, slots, f = dev(rng.integers(0, 100000, T).astype(np.int32)), dev(slots_for(rng, T, n_pages, ps)), dev(U.freqs(n_rot))
    a, b = U.random_cache(fmt, rng, n_pages, Hkv, ps, D), None
    b, c = tuple(t.clone() for t in a), tuple(t.clone() for t in a)
    want = mx.ops.rope(q, pos, f, interleaved=inter, mscale=0.75)
    mx.ops.kv_write(mx.ops.rope(k, pos, f, interleaved=inter, mscale=0.75), v, slots, a)
    assert torch.equal(mx.ops.rope_kv_write(q, k, v, pos, slots, b, f, interleaved=inter, mscale=0.75), want)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    mx.ops.rope_kv_write(q, k, v, pos, slots, c, f, interleaved=inter, mscale=0.75, q_out=q)
    assert torch.equal(q, want) and all(torch.equal(x, y) for x, y in zip(a, c))


@pytest.mark.parametrize("fmt", ["f16", "q8_0"])
def test_slots_outside_the_cache_are_skipped(mx, fmt):
    rng = np.random.default_rng(3)
    T, Hkv, D, ps, n_pages = 6, 2, 64, 16, 2
    k, v = dev(rows(rng, T, Hkv, D)), dev(rows(rng, T, Hkv, D))
    cache = U.random_cache(fmt, rng, n_pages, Hkv, ps, D)
    want = tuple(t.clone() for t in cache)
    mx.ops.kv_write(k[2:3], v[2:3], dev(np.array([31], np.int32)), want)
    mx.ops.kv_write(k, v, dev(np.array([-1, 32, 31, -2 ** 31, 2 ** 31 - 1, 33], np.int32)), cache)
    assert all(torch.equal(a, b) for a, b in zip(cache, want))


def test_q8_0_write_of_extremes(mx):
    """Ties, subnormals, the largest fp16 values, and blocks with a NaN or an infinity, which read back as NaN."""
    D, ps = 32, 16
    x = np.zeros((6, 1, D), np.float16)
    x[0, 0] = (np.arange(D) - 16) * 0.25
    x[0, 0, 0] = 127.0 / 2                                   # amax / 127 = 1 / 2: every other value is a tie
    x[1, 0] = np.linspace(-6e-8, 6e-8, D)
    x[2, 0] = np.linspace(-65472, 65472, D)
    x[3, 0, 7], x[3, 0, 8] = np.nan, 3
    x[4, 0, 9], x[4, 0, 8] = -np.inf, 3
    x[5, 0] = 1
    cache = mx.ops.kv_cache("q8_0", 1, 1, ps, D)
    mx.ops.kv_write(dev(x), dev(x), dev(np.arange(6, dtype=np.int32)), cache)
    qs, d = U.q8_0(x[[0, 1, 2, 5]])
    pick = [0, 1, 2, 5]
    assert np.array_equal(host(cache[0])[0, 0, pick], qs[:, 0]) and np.array_equal(host(cache[1])[0, 0, pick].view(np.uint16), d[:, 0].view(np.uint16))
    k, v = mx.ops.kv_read(cache, dev(np.zeros((1, 1), np.int32)), dev(np.array([0, 6], np.int32)), 6)
    assert torch.equal(torch.isnan(k).all(-1)[:, 0].cpu(), torch.tensor([False, False, False, True, True, False])) and torch.equal(k.isnan(), v.isnan())
    assert torch.isfinite(k[pick]).all()


@pytest.mark.parametrize("fmt", ["f16", "q8_0"])
@pytest.mark.parametrize("Hkv,D,ps,lens", [(8, 128, 16, [1]), (2, 64, 48, [0, 5, 48, 0, 0, 97, 16]), (1, 256, 16, [333, 0]), (3, 96, 256, [17, 255, 256, 257, 1, 1, 1]),
                                           (1, 32, 32, [(i * 7) % 23 for i in range(200)]), (1, 32, 16, [3] * 5000), (8, 128, 32, [8000, 300])])
def test_kv_read(mx, fmt, Hkv, D, ps, lens):
    rng = np.random.default_rng(len(lens) + D)
    table, n_pages = U.pages_of(lens, ps, rng)
    cache = U.keep_only(U.random_cache(fmt, rng, n_pages, Hkv, ps, D), table, lens, ps)
    start = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    total = int(start[-1]) + 5
    out = tuple(torch.full((total, Hkv, D), 9.0, dtype=torch.float16, device="cuda") for _ in range(2))
    got = mx.ops.kv_read(cache, dev(table), dev(start), total, out=out)
    for g, s in zip(got, U.stored(cache)):
        want = np.concatenate([s[table[b][np.arange(n) // ps], :, np.arange(n) % ps] for b, n in enumerate(lens)])
        assert np.array_equal(host(g)[: total - 5].view(np.uint16), want.astype(np.float16).view(np.uint16))
        assert (host(g)[total - 5:] == 9).all(), "rows behind the last sequence were written"


@pytest.mark.parametrize("fmt", ["f16", "q8_0"])
def test_kv_read_of_bad_pages_gives_zeros(mx, fmt):
    rng = np.random.default_rng(8)
    ps, Hkv, D = 16, 2, 64
    cache = U.random_cache(fmt, rng, 4, Hkv, ps, D)
    table = np.array([[2, -1, 4, 1], [2 ** 31 - 1, 0, 3, -2 ** 31]], np.int32)
    k, _ = mx.ops.kv_read(cache, dev(table), dev(np.array([0, 70, 130], np.int32)), 130)     # 70 tokens of a table that holds 64
    k, s = host(k).astype(np.float64), U.stored(cache)[0].astype(np.float16).astype(np.float64)
    for b, (r0, n) in enumerate(((0, 70), (70, 60))):
        for t in range(n):
            page = table[b, t // ps] if t < 64 else -1
            assert np.array_equal(k[r0 + t], s[page, :, t % ps] if 0 <= page < 4 else np.zeros((Hkv, D))), (b, t)


def test_write_then_read_and_a_captured_step(mx):
    """A write is seen by the read behind it on the same stream, also when both are replayed from a graph with new inputs in the same buffers."""
    rng = np.random.default_rng(21)
    B, Hq, Hkv, D, ps = 5, 8, 2, 64, 16
    lens = [40, 3, 17, 16, 1]
    table, n_pages = U.pages_of(lens, ps, rng)
    last = np.array([n - 1 for n in lens], np.int32)
    slots = dev(np.array([table[b, t // ps] * ps + t % ps for b, t in enumerate(last)], np.int32))
    start, total, f = dev(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)), sum(lens), dev(U.freqs(D))
    for fmt in ("f16", "q8_0"):
        cache = U.random_cache(fmt, rng, n_pages, Hkv, ps, D)
        new = [dev(rows(rng, B, h, D)) for h in (Hq, Hkv, Hkv)]
        pos, tab = dev(last.copy()), dev(table)

        def step():
            q = mx.ops.rope_kv_write(*new, pos, slots, cache, f)
            return (q,) + mx.ops.kv_read(cache, tab, start, total)

        step()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for _ in range(3):
            for t in new:
                t.copy_(torch.randn_like(t))
            graph.replay()
            torch.cuda.synchronize()
            replayed = [t.clone() for t in out]
            assert all(torch.equal(a, b) for a, b in zip(replayed, step()))


def test_refusals(mx):
    ops = mx.ops
    x, pos, f = torch.zeros(3, 4, 64, dtype=torch.float16, device="cuda"), dev(np.zeros(3, np.int32)), dev(U.freqs(64))
    for bad in (dict(x=x.float()), dict(x=x.cpu()), dict(x=x.transpose(1, 2).contiguous().transpose(1, 2)),
                dict(positions=pos.long()), dict(positions=pos[:2]), dict(freqs=f.float()), dict(freqs=f.cpu()), dict(y=x[:2]), dict(y=x.float())):
        with pytest.raises(ValueError):
            ops.rope(**{**dict(x=x, positions=pos, freqs=f), **bad})
    for bad in (dict(freqs=dev(U.freqs(128))), dict(freqs=dev(U.freqs(24))), dict(x=x[:0], positions=pos[:0])):
        with pytest.raises(mx.ops.MxError):
            ops.rope(**{**dict(x=x, positions=pos, freqs=f), **bad})
    cache, slots = ops.kv_cache("q8_0", 2, 4, 16, 64), dev(np.arange(3, dtype=np.int32))
    ok = dict(q=x, k=x, v=x, positions=pos, slots=slots, cache=cache, freqs=f)
    ops.rope_kv_write(**ok)
    for bad in (dict(k=x[:, :2]), dict(v=x[:2]), dict(q=x[..., :32]), dict(slots=slots[:2]), dict(slots=slots.long()), dict(positions=pos[:1]), dict(cache=cache[:2]),
                dict(cache=cache[:3]), dict(cache=(cache[0], cache[1], cache[2], cache[3][..., :1])), dict(q_out=x[:2]), dict(cache=tuple(t.cpu() for t in cache))):
        with pytest.raises(ValueError):
            ops.rope_kv_write(**{**ok, **bad})
    with pytest.raises(ValueError):
        ops.kv_write(x[:, :1], x, slots, cache)
    tab, rows = dev(np.zeros((2, 1), np.int32)), dev(np.array([0, 3, 5], np.int32))
    for bad in (dict(rows=rows[:2]), dict(rows=rows.long()), dict(page_table=tab.long()), dict(out=(x, x)), dict(cache=cache[:3])):
        with pytest.raises(ValueError):
            ops.kv_read(**{**dict(cache=cache, page_table=tab, rows=rows, total_rows=5), **bad})
    with pytest.raises(mx.ops.MxError):
        ops.kv_read(cache, tab, rows, 0)
    with pytest.raises(ValueError):
        ops.kv_cache("q8_0", 2, 4, 16, 80)
    with pytest.raises(mx.ops.MxError):
        ops.rope_freqs(24)


@pytest.mark.parametrize("T", [5, 600])
def test_rows_beside_each_other_keep_their_neighbours(mx, T):
    """q, k and v as parts of wider rows, q_out as a part of another: what lies between them is neither read as theirs nor written."""
    rng = np.random.default_rng(T)
    Hq, Hkv, D, ps = 4, 2, 64, 16
    wide = torch.full((T, 1024), float("nan"), dtype=torch.float16, device="cuda")
    parts = [wide[:, 64: 64 + Hq * D], wide[:, 384: 384 + Hkv * D], wide[:, 640: 640 + Hkv * D]]
    for p in parts:
        p.copy_(dev(rows(rng, T, 1, p.shape[1])).view(T, -1))
    q, k, v = (p.view(T, -1, D) for p in parts)
    to = torch.full((T, 512), 3.0, dtype=torch.float16, device="cuda")
    cache = mx.ops.kv_cache("f16", -(-T // ps), Hkv, ps, D)
    pos, slots, f = dev(np.arange(T, dtype=np.int32)), dev(np.arange(T, dtype=np.int32)), dev(U.freqs(D))
    mx.ops.rope_kv_write(q, k, v, pos, slots, cache, f, q_out=to[:, 128: 128 + Hq * D].view(T, Hq, D))
    assert torch.equal(to[:, 128: 384].view(T, Hq, D), mx.ops.rope(q.contiguous(), pos, f))
    assert (to[:, :128] == 3).all() and (to[:, 384:] == 3).all()
    at = torch.arange(T, device="cuda")
    assert torch.equal(cache[0][at // ps, :, at % ps], mx.ops.rope(k.contiguous(), pos, f)) and torch.equal(cache[1][at // ps, :, at % ps], v.contiguous())
