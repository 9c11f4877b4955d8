"""Saved-tensor hooks that give back the same values in another layout, or other tensors: the backward passes of the plain transformer block's
operators read what was saved, whatever its strides, and refuse what was not."""
import math

import pytest
import torch

from savanna_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


def _other_strides(t):
    """The values of t with its dimensions in another order in memory; one-dimensional ones at every other place."""
    if t.dim() < 2:
        return torch.stack([t, t], -1)[..., 0]
    return t.transpose(-2, -1).contiguous().transpose(-2, -1) if t.dim() == 2 else t.transpose(0, 2).contiguous().transpose(0, 2)


def _off_16_bytes(t):
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:]
    return flat.copy_(t.reshape(-1)).view(t.shape)


def _hooks(unpack):
    return torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack)


def _rpe(B, L, H, causal, table_dtype=torch.float32):
    g = torch.Generator(device=DEV).manual_seed(L)
    qkv = torch.randn(B, L, H, 384, generator=g, device=DEV).to(BF).requires_grad_(True)
    table = (0.2 * torch.randn(16, H, generator=g, device=DEV)).to(table_dtype).requires_grad_(True)
    buckets = torch.randint(0, 16, (41 if causal else 81,), generator=g, device=DEV, dtype=torch.int32)
    return qkv, table, buckets, torch.randn(B, L, H, 128, generator=g, device=DEV).to(BF)


def _same(got, want):
    # dq is added up in an order that varies: a step of bf16 between two sums; dk, dv and the table's gradient are not
    assert torch.equal(got[1], want[1]) and torch.equal(got[0][..., 128:], want[0][..., 128:])
    a, b = got[0].double(), want[0].double()
    assert bool(((a - b).abs() <= 2.0 ** -7 * b.abs() + 2.0 ** -20 * b.abs().max()).all())


@pytest.mark.parametrize("table_dtype", [BF, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "both"])
@pytest.mark.parametrize("unpack", [_other_strides, _off_16_bytes], ids=["strides", "alignment"])
def test_attention_rpe_backward_of_other_layouts(unpack, causal, table_dtype):
    qkv, table, buckets, go = _rpe(2, 150, 3, causal, table_dtype)
    want = torch.autograd.grad(ops.attention_rpe(qkv, table, buckets, math.sqrt(128), causal), (qkv, table), go)
    with _hooks(unpack):
        o = ops.attention_rpe(qkv, table, buckets, math.sqrt(128), causal)
    _same(torch.autograd.grad(o, (qkv, table), go), want)


def test_attention_rpe_backward_of_expanded_tensors():
    """All tokens alike, given back as one token with strides of 0."""
    one, table, buckets, go = _rpe(1, 1, 2, True)
    qkv = one.detach().expand(2, 90, 2, 384).contiguous().requires_grad_(True)
    go = torch.randn(2, 90, 2, 128, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).to(BF)
    want = torch.autograd.grad(ops.attention_rpe(qkv, table, buckets, 1.0, True), (qkv, table), go)
    with _hooks(lambda t: t[:1, :1].expand(t.shape) if t.shape == qkv.shape else t):
        o = ops.attention_rpe(qkv, table, buckets, 1.0, True)
    _same(torch.autograd.grad(o, (qkv, table), go), want)


def test_attention_rpe_backward_refuses_other_tensors():
    qkv, table, buckets, go = _rpe(1, 40, 2, False)
    for change in (lambda t: t.cpu(), lambda t: t.float() if t.dtype == BF else t, lambda t: t[:, :30] if t.dim() == 4 else t,
                   lambda t: t[..., :20] if t.dim() == 3 else t, lambda t: t[:-1] if t.dtype == torch.int32 else t):
        with _hooks(change):
            o = ops.attention_rpe(qkv, table, buckets, 1.0, False)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(o, (qkv, table), go)


def _norm(T, D, dtype):
    g = torch.Generator(device=DEV).manual_seed(T + D)
    x, gy, gr = ((torch.randn(2, T, D, generator=g, device=DEV)).to(dtype) for _ in range(3))
    w, b = ((1 + 0.1 * torch.randn(D, generator=g, device=DEV)).to(dtype) for _ in range(2))
    return [t.requires_grad_(True) for t in (x, w, b)], gy, gr


@pytest.mark.parametrize("dtype", [BF, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("T,D", [(40, 64), (33, 1000), (17, 331)])
def test_layernorm_backward_of_other_strides(T, D, dtype):
    leaves, gy, gr = _norm(T, D, dtype)
    want = torch.autograd.grad(ops.layernorm_residual(*leaves, 1e-5), leaves, (gy, gr))
    with _hooks(_other_strides):
        y = ops.layernorm_residual(*leaves, 1e-5)
    for got, w in zip(torch.autograd.grad(y, leaves, (gy, gr)), want):
        assert torch.equal(got, w)


def test_layernorm_backward_refuses_other_tensors():
    leaves, gy, _ = _norm(20, 96, BF)
    for change in (lambda t: t.cpu(), lambda t: t.float() if t.dtype == BF else t, lambda t: t[:, :10] if t.dim() == 3 else t,
                   lambda t: t[:5] if t.dim() == 2 else t, lambda t: t[:40] if t.dim() == 1 else t):
        with _hooks(change):
            y = ops.layernorm(*leaves, 1e-5)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(y, leaves, gy)
