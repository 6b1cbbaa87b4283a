"""Plain forms in 64 bits of the rotary, cache and one-token attention operators, and caches to run them on."""
import numpy as np
import torch

import oracle as O
from gpu_util import dev


def freqs(n_rot, base=10000.0):
    return base ** (-2.0 * np.arange(n_rot // 2) / n_rot)


def rope(x, pos, f, inter, mscale=1.0):
    """x [T, H, D] -> fp64 rows, not rounded."""
    x = np.asarray(x, np.float64)
    n = 2 * len(f)
    a = np.asarray(pos, np.float64)[:, None] * f
    c, s = mscale * np.cos(a)[:, None], mscale * np.sin(a)[:, None]
    i0, i1 = (np.arange(0, n, 2), np.arange(1, n, 2)) if inter else (np.arange(n // 2), np.arange(n // 2, n))
    y = x.copy()
    y[..., i0] = x[..., i0] * c - x[..., i1] * s
    y[..., i1] = x[..., i0] * s + x[..., i1] * c
    return y


def rope_tol(x, f, inter, mscale=1.0):
    """Beside the rounding to fp16 (half a step, 2^-11 of the value; 2^-25 below its normal range), which the caller counts: each of the two products
    has its sine's rounding (2^-24) and its own, the sum one more; the sines themselves are off by 2^-34."""
    x = np.abs(np.asarray(x, np.float64))
    n = 2 * len(f)
    i0, i1 = (np.arange(0, n, 2), np.arange(1, n, 2)) if inter else (np.arange(n // 2), np.arange(n // 2, n))
    size = np.zeros_like(x)
    size[..., i0] = size[..., i1] = mscale * (x[..., i0] + x[..., i1])
    return size * (3 * 2.0 ** -24 + 2.0 ** -33)


def q8_0(x):
    """Q8_0 planes (int8 [..., D], fp16 [..., D / 32]) of fp16 values, by the oracle's encoder of that weight format."""
    x = np.asarray(x, np.float32)
    blocks = O.quantize(O.Q8_0, x.reshape(-1, x.shape[-1])).reshape(-1, 34)
    return blocks[:, 2:].copy().view(np.int8).reshape(x.shape), blocks[:, :2].copy().view(np.float16).reshape(x.shape[:-1] + (x.shape[-1] // 32,))


def stored(planes):
    """What a cache's planes stand for, fp64 [pages, heads, page size, D] for keys and for values."""
    p = [t.detach().cpu().numpy() for t in planes]
    if len(p) == 2:
        return [t.astype(np.float64) for t in p]
    return [p[i].astype(np.float64) * np.repeat(p[i + 1].astype(np.float64), 32, -1) for i in (0, 2)]


def random_cache(fmt, rng, n_pages, Hkv, ps, D, k_scale=1.0):
    """A cache of normal values; Q8_0 planes are their encoding."""
    k, v = (O.round_fp16((rng.standard_normal((n_pages, Hkv, ps, D)) * s).astype(np.float32)) for s in (k_scale, 1.0))
    if fmt == "f16":
        return tuple(dev(t.astype(np.float16)) for t in (k, v))
    return tuple(dev(t) for x in (k, v) for t in q8_0(x))


def poison(cache):
    """The same cache with NaN everywhere (scales of Q8_0)."""
    bad = tuple(torch.full_like(t, float("nan")) if t.dtype == torch.float16 else torch.full_like(t, 77) for t in cache)
    return bad


def pages_of(lens, ps, rng, spare=2):
    """(page table [B, max_pages] of shuffled pages, page count); entries behind a sequence's end name no page of the cache."""
    need = [-(-max(0, n) // ps) for n in lens]
    n_pages = sum(need) + spare
    order, table, at = rng.permutation(n_pages), np.full((len(lens), max(1, max(need))), -1, np.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = order[at: at + n]
        at += n
    return table, n_pages


def keep_only(cache, table, lens, ps):
    """The cache with NaN in every slot that no sequence owns."""
    out = poison(cache)
    for b, n in enumerate(lens):
        t = torch.arange(max(0, n), device="cuda")
        page, at = torch.from_numpy(table[b]).cuda().long()[t // ps], t % ps
        for o, c in zip(out, cache):
            o[page, :, at] = c[page, :, at]
    return out


def attention(q, cache, table, lens, ps, scale, window=0, sinks=None, k_rounded=None):
    """-> (out, tolerance) in fp64 [B, Hq, D].  The tolerance: one rounding of the result to fp16 (2^-11 of it, 2^-25 below the normal range), 2^-20 for the weights' and
    values' two fp16 parts and the sums, 2^-25 of the largest weight where a weight's second part is below fp16's range, and what the 32-bit scores are off,
    e: D + 16 roundings of 2^-24 of the products' magnitudes, and 2^-21 of the score itself in its exponential."""
    q = np.asarray(q, np.float64)
    K, V = stored(cache)
    B, Hq, D = q.shape
    Hkv = K.shape[1]
    G, n_pages = Hq // Hkv, K.shape[0]
    out, tol = np.zeros((B, Hq, D)), np.full((B, Hq, D), 2.0 ** -25)
    for b in range(B):
        n = min(max(0, int(lens[b])), table.shape[1] * ps)
        t = np.arange(max(0, n - window) if window else 0, n)
        page = table[b][t // ps]
        t, page = t[(page >= 0) & (page < n_pages)], page[(page >= 0) & (page < n_pages)]
        if not len(t):
            continue
        for h in range(Hq):
            k, v = K[page, h // G, t % ps], V[page, h // G, t % ps]
            x = scale * (k @ q[b, h])
            e = (D + 16) * 2.0 ** -24 * abs(scale) * (np.abs(k) @ np.abs(q[b, h])).max() + 2.0 ** -21 * np.abs(x).max()
            top = max(x.max(), sinks[h]) if sinks is not None else x.max()
            p = np.exp(x - top)
            total = p.sum() + (np.exp(sinks[h] - top) if sinks is not None else 0.0)
            out[b, h] = p @ v / total
            size = p @ np.abs(v) / total
            tol[b, h] += 2.0 ** -11 * np.abs(out[b, h]) + size * (2.0 ** -20 + 3 * e) + 2.0 ** -25 * np.abs(v).sum(0) / total
    return out, tol
