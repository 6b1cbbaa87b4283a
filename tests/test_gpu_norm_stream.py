"""GPU: the 8-bit stream that the norms and gated activations emit beside their rows is the quantizer's of those rows, over enough blocks to meet the products that round
otherwise by way of fp32 than at once."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def normal(seed, *shape):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, device="cuda", generator=g)


@pytest.mark.parametrize("rows,hidden", [(1024, 4096), (333, 2880), (4096, 128)])
@pytest.mark.parametrize("seed", [1, 2])
def test_rms_norm(mx, rows, hidden, seed):
    x, w = normal(seed, rows, hidden).half(), 1 + 0.3 * normal(seed + 10, hidden)
    y, q8 = mx.ops.rms_norm_f32w_q8(x, w, 1e-6)
    assert torch.equal(q8, mx.ops.quantize_q8_1(y))


@pytest.mark.parametrize("rows,hidden", [(1024, 4096), (32768, 128)])
@pytest.mark.parametrize("seed", [3, 4])
def test_gated_rms_norm(mx, rows, hidden, seed):
    x, z, w = normal(seed, rows, hidden), normal(seed + 10, rows, hidden).half(), (1 + 0.3 * normal(seed + 20, hidden)).half()
    y, q8 = mx.ops.gated_rms_norm_q8(x, z, w, 1e-6)
    assert torch.equal(q8, mx.ops.quantize_q8_1(y))


@pytest.mark.parametrize("n", [1 << 18, 1 << 22])
@pytest.mark.parametrize("oai", [False, True])
def test_gated_activations(mx, n, oai):
    gate, up = (3 * normal(5, n)).half(), (3 * normal(6, n)).half()
    y, q8 = mx.ops.swiglu_q8(gate, up, oai=oai)
    assert torch.equal(q8, mx.ops.quantize_q8_1(y)) and torch.equal(mx.ops.swiglu_q8(gate, up, oai=oai, want_y=False)[1], q8)
