"""What the forward of attention with a relative position bias keeps for its backward: the output, what it lost in rounding, and the rows' log-sum-exp.

Up to 1024 tokens the probabilities enter their product as two bf16 values.  The first is off by 2^-8 of P at most, the second by 2^-8 of that: 2^-16 P.
In 32 bits P itself is off by 2^-18 (exponents of up to 32 units, 2^-24 of them each; two units of the exponential) and the sums over 64 steps of 16
keys, two products each, by 128 * 2^-24 = 2^-17.  What the output loses is kept in 256ths of a step of 2^-7 (of its power of two): half a 256th, 2^-16, or
a whole one where half a step was lost.  So, with A = sum_j P_j |v_j|,
    |o + lost - exact| <= (2^-16 + 2^-17 + 2^-18) A + 2^-15 |exact|
A single bf16 value would be off by 2^-8 P, which the oracle shows to lie outside."""
import math

import pytest
import torch

from savanna_b200 import ops
from savanna_b200.ops import reference as ref
from tests.test_gpu_rpe import _map

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


def _kept(qkv, table, buckets, scale, causal):
    """(o, lost, lse) as a saved-tensor hook sees them."""
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t) or t, lambda t: t):
        o = ops.attention_rpe(qkv.clone().requires_grad_(True), table, buckets, scale, causal)
    lost, = (t for t in saved if t.dtype == torch.int8)
    lse, = (t for t in saved if t.dtype == torch.float32 and t.dim() == 3)
    assert lost.shape == o.shape
    return o.detach(), lost, lse


def _inputs(B, L, H, causal, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    qkv = torch.randn(B, L, H, 384, generator=g, device=DEV)
    qkv[..., 256:] = 0.5 + torch.rand(B, L, H, 128, generator=g, device=DEV)          # values of one sign: no output near zero
    table = torch.randn(32, H, generator=g, device=DEV)
    return qkv.to(BF), table, _map(32, 64, causal)


def _probabilities(qkv, table, buckets, causal):
    L = qkv.shape[1]
    q, k, v = (t.double().transpose(1, 2) for t in qkv.split(128, dim=-1))
    s = q @ k.transpose(-1, -2) / math.sqrt(128) + ref.relative_bias(table.double(), buckets, 1.0, L, L, causal)
    if causal:
        s = s.masked_fill(torch.ones(L, L, dtype=torch.bool, device=DEV).triu(1), float("-inf"))
    return s, v


CASES = [(3, 17), (2, 130), (2, 300), (2, 777), (1, 1024)]


@pytest.mark.parametrize("causal", [True, False], ids=["causal", "both"])
@pytest.mark.parametrize("B,L", CASES)
def test_output_with_what_it_lost(B, L, causal):
    qkv, table, buckets = _inputs(B, L, 3, causal, L)
    o, lost, lse = _kept(qkv, table, buckets, 1.0, causal)
    s, v = _probabilities(qkv, table, buckets, causal)
    p = torch.softmax(s, -1)
    want = (p @ v).transpose(1, 2)
    bound = (2.0 ** -16 + 2.0 ** -17 + 2.0 ** -18) * (p @ v.abs()).transpose(1, 2) + 2.0 ** -15 * want.abs()
    got = (o.float().view(torch.int32) + 256 * lost.int()).view(torch.float32).double()
    worst = float(((got - want).abs() / bound).max())
    assert worst <= 1
    # exponents and their sum in 32 bits, a logarithm of up to 16 units
    off = float((lse.double() - torch.logsumexp(s, -1)).abs().max())
    assert off <= 2.0 ** -17 + 16 * 2.0 ** -23
    # one bf16 value of each probability, normalised by their sum
    one = torch.exp(s - s.amax(-1, keepdim=True)).to(BF).double()
    single = (one @ v / one.sum(-1, keepdim=True)).transpose(1, 2)
    outside = float(((single - want).abs() / bound).max())
    assert outside > 1


@pytest.mark.parametrize("causal", [True, False], ids=["causal", "both"])
@pytest.mark.parametrize("B,L", CASES[1:])
def test_what_the_output_lost_is_rounded_to_its_nearest_256th(B, L, causal):
    """The mean of what is left, in 256ths of a step: 0 where it was rounded, 1/2 where it was cut off.  2^17 values or more, each within 1/2 of its
    rounding and, with the error above, within 2 in all: their mean varies by 2 / 2^8.5 = 0.006; sums in 32 bits that were cut off instead of
    rounded would shift it by up to 128 * 2^-24 / 2 of the value, 1/8 of a 256th of a step."""
    qkv, table, buckets = _inputs(B, L, 4, causal, L)
    o, lost, _ = _kept(qkv, table, buckets, 1.0, causal)
    s, v = _probabilities(qkv, table, buckets, causal)
    want = (torch.softmax(s, -1) @ v).transpose(1, 2)
    many = torch.arange(L, device=DEV) >= 16         # the first rows of a causal sequence are averages of a few values
    left = (want.float().view(torch.int32) - o.float().view(torch.int32)).double() / 256 - lost.double()
    mean = float(left[:, many].mean())
    assert abs(mean) <= 0.25
    # and one that lost nothing says so
    if causal:
        assert torch.equal(o[:, 0], qkv[:, 0, :, 256:]) and int(lost[:, 0].abs().max()) == 0
