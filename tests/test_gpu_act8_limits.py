"""Activations in 8 bits: rows too long for 32-bit columns are refused; the longest that memory has room for beside its statement goes there and back."""
import pytest
import torch

from savanna_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("D", [2 ** 31 - 127, 2 ** 31, 2 ** 32 + 5])
def test_rows_that_are_too_long_are_refused(D):
    x = torch.ones(1, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError):
        ops.act_quantize(x.expand(D))
    with pytest.raises(ValueError):
        ops.act_dequantize(x.to(torch.int8).expand(D), x.float().expand((D + 127) // 128))


def test_a_row_of_2_to_30_values_and_a_few():
    n = 2 ** 30 + 77                                 # off vectors: single values; its offsets in bytes pass 2^31
    x = (torch.arange(n, device=DEV, dtype=torch.int32) % 253 - 126).to(torch.bfloat16)
    q, scale = ops.act_quantize(x)
    for at in (0, n // 2 // 128 * 128, n - 77 - 128, n - 77):
        part = x[at:at + 128]
        assert torch.equal(q[at:at + 128], torch.round(part.float() * (127.0 / part.float().abs().max())).to(torch.int8))
        assert torch.equal(scale[at // 128], part.float().abs().max() / 127.0)
    back = ops.act_dequantize(q, scale)
    # |x| <= 126: half a step of 126 / 127, and values of up to 126 have 8 bits: 2^-8 of them
    for at in range(0, n, 2 ** 28):
        a, b = x[at:at + 2 ** 28].float(), back[at:at + 2 ** 28].float()
        assert bool(((a - b).abs() <= 126 / 254 + 2.0 ** -8 * 127).all())
