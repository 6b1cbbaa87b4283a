"""GPU: scales of a Q4_0 cache that are no numbers, infinite ones among them."""
import numpy as np
import pytest
import torch

import q4_util as Q
from gpu_util import dev, host
from test_gpu_q4_cache import attend, case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,G", [(32, 1), (64, 8), (96, 2), (128, 4), (256, 2)])
@pytest.mark.parametrize("sign", [1, -1])
def test_infinite_scales_of_keys(mx, D, G, sign):
    """Every head that reads one is NaN, whichever side of zero its token's score would lie on; heads and sequences that do not have the bits that they have without."""
    lens = [300, 1500, 40, 1, 0]
    rng, table, cache, q = case(lens, 2, G, D, 16, D + G)
    q = np.concatenate([q[:, :G], -q[:, :G]], 1)                       # the second key-value head's queries are the first's with the other sign
    for codes, d in (cache[:2], cache[2:]):
        codes[:, 1], d[:, 1] = codes[:, 0], d[:, 0]
    for most in (None, 1 << 20):                                       # whole, in parts
        want = host(attend(mx, q, cache, table, lens, max_len=most))
        c = tuple(t.clone() for t in cache)
        for b, t in ((0, 100), (1, 1499), (3, 0)):
            c[1][int(table[b, t // 16]), :, t % 16, D // 32 - 1] = sign * float("inf")
        got = host(attend(mx, q, c, table, lens, max_len=most))
        assert np.isnan(got[[0, 1, 3]]).all() and np.array_equal(got[[2, 4]].view(np.uint16), want[[2, 4]].view(np.uint16))
        # outside the window it is not read
        win = host(attend(mx, q, c, table, lens, max_len=most, window=30))
        assert np.isfinite(win[[0, 2]]).all() and np.isnan(win[[1, 3]]).all()


@pytest.mark.parametrize("T", [70, 20000])
def test_reading_back(mx, T):
    """A block whose scale is infinite or NaN reads back as NaN whole, its neighbours as they are; the largest number that a scale may be gives infinities, and zeros where codes are 8."""
    rng = np.random.default_rng(T)
    n_pages, Hkv, D = -(-T // 16), 4, 128
    cache = Q.random_cache(rng, n_pages, Hkv, 16, D)
    table, ends = dev(rng.permutation(n_pages).astype(np.int32)[None]), dev(np.array([0, T], np.int32))
    want = mx.ops.kv_read(cache, table, ends, T)
    odd = [float("inf"), -float("inf"), float("nan"), 65504.0]
    at = torch.from_numpy(rng.integers(0, 40, tuple(cache[1].shape))).cuda()
    for d in (cache[1], cache[3]):
        for i, x in enumerate(odd):
            d[at == i] = x
    got = mx.ops.kv_read(cache, table, ends, T)
    t = torch.arange(T, device="cuda")
    page = table[0].long()[t // 16]
    of = at[page, :, t % 16].repeat_interleave(32, -1)                 # [T, Hkv, D]: what stands in an element's scale
    for w, g, codes in zip(want, got, cache[::2]):
        assert torch.equal(g[of > 3], w[of > 3]) and g[of < 3].isnan().all()
        c = codes[page, :, t % 16].unflatten(-1, (-1, 16))
        c = torch.cat((c & 15, c >> 4), -1).flatten(-2).float() - 8
        assert torch.equal(g[of == 3], (c * 65504.0).half()[of == 3])
