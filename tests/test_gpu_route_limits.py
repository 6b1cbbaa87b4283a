"""GPU: routing at the largest number of tokens that a call takes."""
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
