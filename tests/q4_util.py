"""Plain forms in 64 bits of the Q4_0 cache and the attention over it, and caches to run them on."""
import numpy as np
import torch

import kv_util as U
import oracle as O
from gpu_util import dev


def q4_0(x):
    """Q4_0 planes (uint8 [..., D / 2], fp16 [..., D / 32]) of fp16 values; codes by exact quotients: 8 x / m is a ratio of two 11-bit numbers, which 64 bits tell from every border."""
    x = np.asarray(x, np.float64)
    b = x.reshape(x.shape[:-1] + (-1, 32))
    m = np.take_along_axis(b, np.abs(b).argmax(-1)[..., None], -1)
    code = np.minimum(15, np.floor(np.where(m == 0, 8.0, b * -8 / np.where(m == 0, 1, m) + 8.5))).astype(np.uint8)
    d = np.where(m == 0, -0.0, m / -8)[..., 0].astype(np.float16)
    return (code[..., :16] | code[..., 16:] << 4).reshape(x.shape[:-1] + (-1,)), d


def values(codes, d):
    """What planes stand for, fp64 [..., D]."""
    c = np.asarray(codes).reshape(codes.shape[:-1] + (-1, 16))
    v = np.concatenate((c & 15, c >> 4), -1).astype(np.float64) - 8
    return (v * np.asarray(d, np.float64)[..., None]).reshape(codes.shape[:-1] + (-1,))


def stored(cache):
    p = [t.detach().cpu().numpy() for t in cache]
    return values(p[0], p[1]), values(p[2], p[3])


def random_cache(rng, n_pages, Hkv, ps, D, k_scale=1.0):
    """The encoding of normal values."""
    return tuple(dev(t) for s in (k_scale, 1.0) for t in q4_0(O.round_fp16((rng.standard_normal((n_pages, Hkv, ps, D)) * s).astype(np.float32))))


def keep_only(cache, table, lens, ps):
    """The cache with NaN for the scales, and other codes, in every slot that no sequence owns."""
    return U.keep_only(cache, table, lens, ps)


def attention(q, cache, table, lens, ps, scale, window=0, sinks=None):
    """-> (out, tolerance) in fp64 [B, Hq, D].  The tolerance: one rounding of the result to fp16 (2^-11 of it, 2^-25 below the normal range), and, with `size` the weighted mean of 23 |d|, what
    products of codes up to 15 and of the offset 8 are made of,
      2^-20 of size for the two fp16 parts of weights times scales and the sums,
      3 e of size for what the 32-bit scores are off: 34 roundings in a block's product, one for each block behind it and four more, 2^-24 each of 23 |d| sum |q|, and 2^-21 of the score in its exponential,
      2^-39 2^k of 23 |d| a token and unit of the largest weight, the last bits of parts below fp16's normal range; 2^k: the largest scale, 1 at least."""
    q = np.asarray(q, np.float64)
    K, V = stored(cache)
    kd, vd = (np.abs(cache[i].detach().cpu().numpy().astype(np.float64)) for i in (1, 3))
    B, Hq, D = q.shape
    Hkv, n_pages = K.shape[1], K.shape[0]
    G = Hq // Hkv
    out, tol = np.zeros((B, Hq, D)), np.full((B, Hq, D), 2.0 ** -25)
    for b in range(B):
        n = min(max(0, int(lens[b])), table.shape[1] * ps)
        t = np.arange(max(0, n - window) if window else 0, n)
        page = table[b][t // ps]
        ok = (page >= 0) & (page < n_pages)
        t, page = t[ok], page[ok]
        if not len(t):
            continue
        for h in range(Hq):
            k, v, dk, dv = K[page, h // G, t % ps], V[page, h // G, t % ps], kd[page, h // G, t % ps], vd[page, h // G, t % ps]
            x = scale * (k @ q[b, h])
            e = (38 + D // 32) * 2.0 ** -24 * abs(scale) * (23 * dk @ np.abs(q[b, h]).reshape(-1, 32).sum(1)).max() + 2.0 ** -21 * np.abs(x).max()
            top = max(x.max(), sinks[h]) if sinks is not None else x.max()
            p = np.exp(x - top)
            total = p.sum() + (np.exp(sinks[h] - top) if sinks is not None else 0.0)
            out[b, h] = p @ v / total
            size = 23 * np.repeat(p @ dv, 32) / total
            tol[b, h] += 2.0 ** -11 * np.abs(out[b, h]) + size * (2.0 ** -20 + 3 * e) + 2.0 ** -39 * max(1.0, dv.max()) * 23 * np.repeat(dv.sum(0), 32) * np.exp(x.max() - top) / total
    return out, tol
