"""Launches that one call cannot hold, without a GPU."""
from test_kv_capi import SHAPE, Call, lib  # noqa: F401


def test_route_tokens(lib):  # noqa: F811
    """A workgroup of 256 threads takes four tokens, and a launch holds fewer than 2^32 threads."""
    c = Call(lib, "mx_moe_route", n_experts=64, k=8, n_groups=1, topk_groups=1, flags=0, scale=1.0)
    for n in ((1 << 26) - 3, (1 << 26) - 2, (1 << 26) - 1, 1 << 26, (1 << 32) - 1):
        assert (n + 3) // 4 * 256 >= 1 << 32 and c.with_(n_tokens=n) == SHAPE, n
