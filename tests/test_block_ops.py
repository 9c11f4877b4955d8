"""Layer norm and 8-bit activations on CPU: the statements against 64 bits, and what the entry points refuse."""
import os

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


def _rpe_inputs(B=1, L=6, H=2, nb=8, far=4, causal=True):
    g = torch.Generator().manual_seed(2)
    n = far + 1 if causal else 2 * far + 1
    return torch.randn(B, L, H, 12, generator=g), torch.randn(nb, H, generator=g), torch.randint(0, nb, (n,), generator=g, dtype=torch.int32)


@pytest.mark.parametrize("causal", [True, False])
def test_attention_rpe_statement(causal):
    """Against the formula pair by pair, its gradient for the table against differences."""
    qkv, table, buckets = _rpe_inputs(causal=causal)
    qkv, table = qkv.double(), table.double().requires_grad_(True)
    far = 4
    q, k, v = qkv.split(4, dim=-1)
    want = torch.zeros(1, 6, 2, 4, dtype=torch.float64)
    for h in range(2):
        for i in range(6):
            js = range(i + 1) if causal else range(6)
            at = [min(i - j, far) if causal else max(-far, min(far, i - j)) + far for j in js]
            s = torch.stack([q[0, i, h] @ k[0, j, h] / 2 + 1.5 * table[int(buckets[a]), h] for j, a in zip(js, at)])
            want[0, i, h] = (torch.softmax(s, 0)[:, None] * torch.stack([v[0, j, h] for j in js])).sum(0).detach()
    got = ops.attention_rpe(qkv, table, buckets, 1.5, causal)
    # the statement computes in fp32: scores of a few units, six keys
    assert float((got - want).abs().max()) <= 64 * 2.0 ** -24 * 16
    w = torch.randn(got.shape, generator=torch.Generator().manual_seed(3)).double()
    (grad,) = torch.autograd.grad((got * w).sum(), table)
    with torch.no_grad():
        for b, h in ((0, 0), (int(buckets[0]), 1), (int(buckets[-1]), 0)):
            step = torch.zeros_like(table)
            step[b, h] = 0.05
            diff = ((ops.attention_rpe(qkv, table + step, buckets, 1.5, causal) - ops.attention_rpe(qkv, table - step, buckets, 1.5, causal)) * w).sum() / 0.1
            # third derivative times step^2 / 6 of sums of about 50 values, and fp32 differences divided by the step
            assert abs(float(diff - grad[b, h])) <= 0.05 ** 2 * 1.5 ** 3 * 50 + 64 * 2.0 ** -24 * 50 / 0.1


def test_attention_rpe_refusals():
    qkv, table, buckets = _rpe_inputs()
    both = torch.zeros(9, dtype=torch.int32)
    for bad in ((qkv[..., :11], table, buckets, 1.0, True), (qkv[0], table, buckets, 1.0, True), (qkv, table[:, :1], buckets, 1.0, True),
                (qkv, table, buckets.long(), 1.0, True), (qkv, table, buckets[:0], 1.0, True), (qkv, table, both[:8], 1.0, False),
                (qkv, table.to(torch.int32), buckets, 1.0, True), (qkv, table[0], buckets, 1.0, True)):
        with pytest.raises(ValueError):
            ops.attention_rpe(*bad)
    assert ops.attention_rpe(qkv, table, both, 1.0, False).shape == (1, 6, 2, 4)
    assert not ops.attention_rpe_covers(qkv, 4)


def test_attention_rpe_step_statement_is_the_last_row():
    qkv, table, buckets = _rpe_inputs(B=2)
    q, k, v = qkv.split(4, dim=-1)
    full = ops.attention_rpe(qkv, table, buckets, 1.5, True)
    for n in range(1, 7):
        lengths = torch.tensor([n, 0], dtype=torch.int32)
        got = ops.attention_rpe_step(q[:, n - 1], k, v, table, buckets, 1.5, lengths)
        assert float((got[0] - full[0, n - 1]).abs().max()) <= 64 * 2.0 ** -24 * 16 and float(got[1].abs().max()) == 0


def test_attention_rpe_step_statement_keeps_nan_and_empties_rows_without_keys():
    q, k, v = torch.randn(3, 2, 8), torch.randn(3, 5, 2, 8), torch.randn(3, 5, 2, 8)
    q[1, 0, 0] = float("nan")
    n = torch.tensor([0, 4, 5], dtype=torch.int32)
    out = ops.attention_rpe_step(q, k, v, torch.randn(4, 2), torch.arange(4, dtype=torch.int32), 1.0, n)
    assert float(out[0].abs().max()) == 0 and bool(out[1, 0].isnan().all()) and bool(out[1, 1].isfinite().all()) and bool(out[2].isfinite().all())


def test_attention_rpe_step_refusals():
    qkv, table, buckets = _rpe_inputs(B=2)
    q, k, v = qkv.split(4, dim=-1)
    q = q[:, 0]
    n = torch.tensor([1, 2], dtype=torch.int32)
    for bad in ((q[0], k, v, table, buckets), (q, k, v[:, :3], table, buckets), (q, k, v.double(), table, buckets), (q[..., :3], k, v, table, buckets),
                (q, k, v, table[:, :1], buckets), (q, k, v, table, buckets.long())):
        with pytest.raises(ValueError):
            ops.attention_rpe_step(*bad, 1.0, n)
    for bad in (n.long(), n[:1], torch.tensor([[1, 2]], dtype=torch.int32)):
        with pytest.raises(ValueError):
            ops.attention_rpe_step(q, k, v, table, buckets, 1.0, bad)


def test_attention_step_entry_refuses_caches_beyond_its_indexes():
    import ctypes

    from savanna_b200.ops import cuda_ops
    if not os.path.exists(cuda_ops._LIB_PATH):
        pytest.skip("library not built")
    entry, strides = ctypes.CDLL(cuda_ops._LIB_PATH).sb_attn_step, (ctypes.c_longlong * 3)(8, 8, 8)

    def call(T):                                     # no heads: nothing is launched
        return entry(None, None, None, None, None, 1, T, 0, 64, strides, strides, strides, 0, None, 2, None, 1, 0, ctypes.c_float(1), ctypes.c_float(1),
                     None, 1, None)
    assert call(2 ** 30) == 0 and call(2 ** 30 + 1) != 0 and call(-1) != 0
