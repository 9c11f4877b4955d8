"""Layer norm and 8-bit activations on CPU: the statements against 64 bits, and what the entry points refuse."""
import pytest
import torch

from savanna_b200 import ops


def test_layernorm_statement():
    g = torch.Generator().manual_seed(0)
    x, w, b = (torch.randn(*s, generator=g) for s in ((5, 33), (33,), (33,)))
    xd = x.double()
    want = (xd - xd.mean(-1, keepdim=True)) / torch.sqrt(xd.var(-1, correction=0, keepdim=True) + 1e-5) * w.double() + b.double()
    # a mean of 33 values and a square root: 64 roundings of values of a few units at most
    assert float((ops.layernorm(x, w, b, 1e-5).double() - want).abs().max()) <= 64 * 2.0 ** -24 * 16
    y, xr = ops.layernorm_residual(x, w, b, 1e-5)
    assert xr is x and torch.equal(y, ops.layernorm(x, w, b, 1e-5))


def test_layernorm_refusals():
    x, w = torch.randn(2, 8), torch.ones(8)
    for bad in ((x, w[:7], w), (x, w, torch.ones(8, 1)), (torch.randn(3, 0), w, w), (torch.tensor(1.0), w, w)):
        with pytest.raises(ValueError):
            ops.layernorm(*bad, 1e-5)
        with pytest.raises(ValueError):
            ops.layernorm_residual(*bad, 1e-5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (2, 2, 128), (5, 300)])
def test_activation_statement(shape, dtype):
    x = torch.randn(*shape, generator=torch.Generator().manual_seed(1)).to(dtype)
    q, scale = ops.act_quantize(x)
    back = ops.act_dequantize(q, scale, dtype)
    assert q.dtype == torch.int8 and q.shape == x.shape and back.dtype == dtype
    amax = x.double().abs().amax()
    assert float((back.double() - x.double()).abs().max()) <= float(amax) * (1 / 254 + 2 * torch.finfo(dtype).eps)


def test_activation_blocks_with_infinities_come_back_as_nan():
    x = torch.zeros(1, 256)
    x[0, 1], x[0, 130] = float("inf"), 2.0
    back = ops.act_dequantize(*ops.act_quantize(x), torch.float32)
    assert bool(back[0, :128].isnan().all()) and float(back[0, 130]) == 2.0


def test_activation_refusals():
    with pytest.raises(ValueError):
        ops.act_quantize(torch.zeros(3, 4, dtype=torch.int32))
    with pytest.raises(ValueError):
        ops.act_quantize(torch.zeros(3, 0))
    q, scale = ops.act_quantize(torch.randn(3, 200))
    for bad in ((q.float(), scale, torch.bfloat16), (q, scale[:, :1], torch.bfloat16), (q, scale.double(), torch.bfloat16), (q, scale, torch.float64)):
        with pytest.raises(ValueError):
            ops.act_dequantize(*bad)
