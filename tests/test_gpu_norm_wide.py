"""GPU: the residual's norm over rows that fill the LDS a workgroup may take without asking, eager and captured before any eager call of that width."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hidden", [31744, 31776, 32768, 32800])
@pytest.mark.parametrize("halves", [False, True])
def test_wide_rows(mx, hidden, halves):
    g = torch.Generator(device="cuda").manual_seed(hidden)
    x, res = (torch.randn(5, hidden, device="cuda", generator=g).half() for _ in range(2))
    w = 1 + 0.3 * torch.randn(hidden, device="cuda", generator=g)
    out = torch.empty_like(x), torch.empty_like(x), torch.empty(5 * hidden // 32 * (48 if halves else 40), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mx.ops.add_rms_norm_f32w_q8(x, res, w, 1e-5, halves=halves, out=out)
    for _ in range(3):
        x.copy_(torch.randn(5, hidden, device="cuda", generator=g).half())
        h, y, q8 = mx.ops.add_rms_norm_f32w_q8(x, res, w, 1e-5, halves=halves)
        for t in out:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(h, (x.float() + res.float()).half()) and torch.equal(y, mx.ops.rms_norm_f32w_q8(h, w, 1e-5)[0])
        assert torch.equal(q8, (mx.ops.quantize_q8_1s if halves else mx.ops.quantize_q8_1)(y)) and all(torch.equal(a, b) for a, b in zip(out, (h, y, q8)))
