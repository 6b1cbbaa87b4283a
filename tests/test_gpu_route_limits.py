"""GPU: routing at the largest number of tokens that a call takes, and router logits on the current device only."""
import numpy as np
import pytest
import torch

from gpu_util import dev

pytestmark = pytest.mark.gpu


def test_the_most_tokens(mx):
    T, E = (1 << 26) - 4, 2
    logits = torch.zeros(T, E, dtype=torch.float16, device="cuda")
    at = torch.tensor([0, 5, T // 2 + 1, T - 2, T - 1], device="cuda")
    logits[at] = dev(np.array([[1, 2], [3, 1], [-1, 1], [0, 2], [2, 0]], np.float16))
    idx, w = mx.ops.moe_route(logits, 1, renormalize=False)
    want = mx.ops.moe_route(logits[at], 1, renormalize=False)
    assert torch.equal(idx[at], want[0]) and torch.equal(w[at], want[1]) and want[0].flatten().tolist() == [1, 0, 1, 1, 0]
    assert int(idx.sum()) == 3 and int((w == 0.5).sum()) == T - 5
    with pytest.raises(mx.ops.MxError):
        mx.ops.moe_route(torch.zeros(T + 1, 1, dtype=torch.float16, device="cuda"), 1)


def test_router_logits_on_the_current_device(mx, monkeypatch):
    """A tensor of another device than the current one is refused before a launch, as the other routing calls do: here the current device says that it is another."""
    x, W = torch.zeros(3, 64, device="cuda").half(), torch.zeros(8, 64, device="cuda")
    mx.ops.moe_router_logits(x, W)
    monkeypatch.setattr(mx.ops, "_current_device", lambda: x.get_device() + 1)
    monkeypatch.setattr(mx.ops, "_stream_of", lambda dev: 0)
    monkeypatch.setattr(mx.ops, "lib", None)                    # nothing may be called
    with pytest.raises(ValueError):
        mx.ops.moe_router_logits(x, W)


def test_router_logits_refusals(mx):
    x, W = torch.zeros(3, 64, device="cuda").half(), torch.zeros(8, 64, device="cuda")
    for bad in ((x.float(), W), (x.cpu(), W), (x, W.half()), (x, W.cpu()), (x.t().contiguous().t(), W), (x, W.t().contiguous().t()), (x[:, :60].contiguous(), W)):
        with pytest.raises(ValueError):
            mx.ops.moe_router_logits(*bad)
