"""Attention of one new token over a cache against its definition in 64 bits.

Tolerance: scores are sums of hd products in 32 bits (hd * 2^-24 of the sum of magnitudes) and exponents of up to a few hundred; a
relative error of 2^-13 of each weight covers scores of up to 2^9 in units of log2 with the exponential's own two units.  The sums of up to T weighted
values add at most 2^-13 of the weighted magnitudes (chains of T / (4 * 2) + 40 additions, T <= 20000).  Then the output's rounding."""
import math

import pytest
import torch

from savanna_b200 import ops
from savanna_b200.ops import reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _case(B, T, H, hd, dtype, far=128, nb=32, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    q, k, v = (torch.randn(*s, generator=g, device=DEV).to(dtype) for s in ((B, H, hd), (B, T, H, hd), (B, T, H, hd)))
    table = torch.randn(nb, H, generator=g, device=DEV).to(dtype)
    buckets = torch.randint(0, nb, (far + 1,), generator=g, device=DEV, dtype=torch.int32)
    lengths = torch.randint(0, T + 1, (B,), generator=g, device=DEV, dtype=torch.int32)
    return q, k, v, table, buckets, lengths


def _check(got, q, k, v, table, buckets, scale, lengths):
    B, T, H, hd = k.shape
    for b in range(B):
        n = T if lengths is None else max(0, min(T, int(lengths[b])))
        if n == 0:
            assert float(got[b].abs().max()) == 0
            continue
        d = torch.arange(n - 1, -1, -1, device=DEV).clamp(max=buckets.shape[0] - 1)
        s = torch.einsum("hd,thd->ht", q[b].double(), k[b, :n].double()) / math.sqrt(hd) + table.double()[buckets.long()[d]].t() * scale
        p = torch.softmax(s, -1)
        want = torch.einsum("ht,thd->hd", p, v[b, :n].double())
        mag = torch.einsum("ht,thd->hd", p, v[b, :n].double().abs())
        half = torch.finfo(got.dtype).eps / 2
        bound = half * want.abs() + 3 * 2.0 ** -13 * mag + torch.finfo(got.dtype).smallest_normal
        err = (got[b].double() - want).abs()
        assert bool((err <= bound).all()), f"row {b} of {n} keys: {float((err / bound).max()):.3g} of the bound"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("hd", [8, 64, 72, 128, 200, 256])
def test_lengths_from_none_to_long(hd, dtype):
    for B, T, H in ((1, 1, 1), (3, 2, 2), (5, 33, 3), (2, 257, 4), (9, 700, 2), (1, 3001, 1), (1, 20000, 2), (40, 130, 16), (200, 65, 8)):
        q, k, v, table, buckets, lengths = _case(B, T, H, hd, dtype, seed=B + T)
        for n in (lengths, None):
            _check(ops.attention_rpe_step(q, k, v, table, buckets, 1.5, n), q, k, v, table, buckets, 1.5, n)


@pytest.mark.parametrize("far", [0, 1, 5, 2000])
def test_maps(far):
    q, k, v, table, buckets, lengths = _case(4, 900, 2, 128, torch.bfloat16, far=far)
    _check(ops.attention_rpe_step(q, k, v, table.float(), buckets, 2.0, lengths), q, k, v, table, buckets, 2.0, lengths)


def test_what_lies_behind_the_last_key_is_not_looked_at():
    for T in (300, 9000):
        q, k, v, table, buckets, _ = _case(3, T, 2, 128, torch.bfloat16)
        lengths = torch.tensor([0, 17, T - 100], device=DEV, dtype=torch.int32)
        want = ops.attention_rpe_step(q, k, v, table, buckets, 1.0, lengths)
        for b, n in enumerate(lengths.tolist()):
            k[b, n:], v[b, n:] = float("nan"), float("inf")
        assert torch.equal(want, ops.attention_rpe_step(q, k, v, table, buckets, 1.0, lengths))
        # lengths outside of the cache are clamped
        out = ops.attention_rpe_step(q[:2], k[:2, :17], v[:2, :17], table, buckets, 1.0, torch.tensor([-5, 10 ** 6], device=DEV, dtype=torch.int32))
        assert torch.equal(out, want[:2]) or float((out - want[:2]).abs().max()) <= 2.0 ** -7 * float(want.abs().max())
        assert float(out[0].abs().max()) == 0


def test_buckets_of_minus_infinity_may_empty_a_row():
    q, k, v, table, buckets, _ = _case(2, 40, 2, 64, torch.bfloat16)
    buckets.fill_(3)
    table[3] = float("-inf")
    assert float(ops.attention_rpe_step(q, k, v, table, buckets, 1.0).abs().max()) == 0
    buckets[0] = 4                                   # the newest key alone is left
    got = ops.attention_rpe_step(q, k, v, table, buckets, 1.0)
    assert torch.equal(got, v[:, -1])


@pytest.mark.parametrize("B,T,H", [(300, 40, 4), (2, 900, 2), (1, 9000, 2)], ids=["one block", "cluster", "two kernels"])
@pytest.mark.parametrize("where", ["q", "k", "v", "overflow", "table"])
def test_nan_stays_visible_in_its_row(B, T, H, where):
    q, k, v, table, buckets, _ = _case(B, T, H, 64, torch.bfloat16, seed=7)
    want = ops.attention_rpe_step(q, k, v, table, buckets, 1.0)
    hit = torch.zeros(B, H, dtype=torch.bool, device=DEV)
    if where == "table":
        table[int(buckets[0]), 1] = float("nan")     # of the newest key
        hit[:, 1] = True
    else:
        hit[-1, 1] = True
        if where == "q":
            q[-1, 1, 3] = float("nan")
        elif where == "overflow":                    # a score of +inf: inf - inf in the softmax
            q[-1, 1, 3], k[-1, T // 2, 1, 3] = 3e38, 3e38
        else:
            (k if where == "k" else v)[-1, T // 2, 1] = float("nan")
    got = ops.attention_rpe_step(q, k, v, table, buckets, 1.0)
    assert bool(got[hit].isnan().all())
    assert torch.equal(got[~hit], want[~hit])


def test_strided_caches_and_queries():
    g = torch.Generator(device=DEV).manual_seed(4)
    qkv = torch.randn(3, 2, 3 * 128, generator=g, device=DEV).to(torch.bfloat16)
    cache = torch.randn(3, 2, 500, 2, 2 * 128, generator=g, device=DEV).to(torch.bfloat16)          # room for more tokens than there are
    q, k, v = qkv[..., :128], cache[:, 0, :333, :, :128], cache[:, 1, :333, :, 128:]
    _, _, _, table, buckets, lengths = _case(3, 333, 2, 128, torch.bfloat16)
    assert torch.equal(ops.attention_rpe_step(q, k, v, table, buckets, 1.0, lengths),
                       ops.attention_rpe_step(q.contiguous(), k.contiguous(), v.contiguous(), table, buckets, 1.0, lengths))
    odd = torch.empty(3, 333, 2, 129, device=DEV, dtype=torch.bfloat16)[..., 1:]
    odd.copy_(k)                                     # off 16-byte boundaries: the statement
    want = ref.attention_rpe_step(q, odd, v, table, buckets, 1.0, lengths)
    assert torch.equal(ops.attention_rpe_step(q, odd, v, table, buckets, 1.0, lengths), want)


def test_offsets_beyond_32_bits():
    """The last sequence of a cache of more than 2^31 values."""
    B, T, H, hd = 9, 2 ** 16, 32, 128                 # 9 * 2^28 values, 4.8 GB each
    k = torch.empty(B, T, H, hd, device=DEV, dtype=torch.bfloat16)
    q, kk, vv, table, buckets, _ = _case(1, 300, H, hd, torch.bfloat16)
    k[-1, :300] = kk[0]
    lengths = torch.zeros(B, device=DEV, dtype=torch.int32)
    lengths[-1] = 300
    out = ops.attention_rpe_step(q.expand(B, H, hd), k, k, table, buckets, 1.0, lengths)
    assert float(out[:-1].abs().max()) == 0
    _check(out[-1:], q, k[-1:, :300], k[-1:, :300], table, buckets, 1.0, None)


def test_guarded_buffers_streams_and_graphs():
    from savanna_b200.ops import cuda_ops
    for B, T, H in ((2, 100, 2), (6, 1500, 4), (1, 9000, 2)):
        args = _case(B, T, H, 128, torch.bfloat16)
        args, lengths = args[:5], args[5]
        with cuda_ops.guarded_allocations():
            want = ops.attention_rpe_step(*args, 1.0, lengths)
            assert cuda_ops.check_guards() >= 1
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = ops.attention_rpe_step(*args, 1.0, lengths)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(want, again)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = ops.attention_rpe_step(*args, 1.0, lengths)
        lengths.copy_(lengths // 2)                  # a graph follows the lengths on the device
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, ops.attention_rpe_step(*args, 1.0, lengths))


def test_agrees_with_the_last_row_of_the_training_form():
    g = torch.Generator(device=DEV).manual_seed(6)
    qkv = torch.randn(2, 290, 3, 384, generator=g, device=DEV).to(torch.bfloat16)
    table = torch.randn(32, 3, generator=g, device=DEV)
    buckets = torch.randint(0, 32, (101,), generator=g, device=DEV, dtype=torch.int32)
    full = ops.attention_rpe(qkv, table, buckets, 1.0, True)[:, -1]
    q, k, v = qkv.split(128, dim=-1)
    one = ops.attention_rpe_step(q[:, -1], k, v, table, buckets, 1.0)
    # roundings of the training form's weights and of both outputs: 2^-8 each of values below max |v|
    assert float((full.float() - one.float()).abs().max()) <= 4 * 2.0 ** -8 * float(v.abs().max())


def test_gradients_run_the_statement():
    q, k, v, table, buckets, lengths = _case(2, 20, 2, 64, torch.bfloat16)
    table.requires_grad_(True)
    out = ops.attention_rpe_step(q, k, v, table, buckets, 1.0, lengths)
    out.float().sum().backward()
    assert table.grad is not None


def test_empty_batch_and_cache():
    q, k, v, table, buckets, _ = _case(2, 0, 2, 64, torch.bfloat16)
    assert float(ops.attention_rpe_step(q, k, v, table, buckets).abs().max()) == 0
    assert ops.attention_rpe_step(q[:0], k[:0], v[:0], table, buckets).shape == (0, 2, 64)


def test_refusals():
    q, k, v, table, buckets, n = _case(2, 6, 2, 64, torch.bfloat16)
    for bad in ((q[0], k, v, table, buckets), (q, k, v[:, :3], table, buckets), (q, k, v.half(), table, buckets), (q[..., :8], k, v, table, buckets),
                (q, k, v, table[:, :1], buckets), (q, k, v, table, buckets.long()), (q, k.cpu(), v, table, buckets)):
        with pytest.raises(ValueError):
            ops.attention_rpe_step(*bad, 1.0, n)
    for bad in (n.long(), n[:1], n.cpu()):
        with pytest.raises(ValueError):
            ops.attention_rpe_step(q, k, v, table, buckets, 1.0, bad)


@pytest.mark.filterwarnings("ignore")
def test_traced_on_new_inputs():
    q, k, v, table, buckets, n = _case(2, 40, 2, 64, torch.bfloat16)

    def f(x):
        return ops.attention_rpe_step(x, k, v, table, buckets, 1.0, n)
    traced = torch.jit.trace(f, q, check_trace=False)
    assert torch.equal(traced(-q), f(-q))
