"""Attention with a learned relative position bias on CUDA against its definition in 64 bits.

Tolerances.  With h = 2^-9 * 1.0 the largest relative rounding of a bf16 value is 2^-8 / 2 * 2 = 2^-8 of its size at most (eps / 2): the
probabilities P and the score gradients dS enter their products rounded to bf16, the outputs are rounded once more.  So
    |o - o'|  <= 2 h' sum_j P_j |v_j - o|  + h' |o|       (the row is normalised by the rounded P's sum)
and for the gradients, each a sum over products with one rounded factor (relative error h') and one delta that is off by at most
2 h' sum_j P_j |dP_j - delta| =: e, with h' = 2^-8:
    |dq| error <= scale sum_j (h' |dS_j| + P_j e) |k_j|,   |dk| the same over i with |q_i|,   |dv| <= h' sum_i P_ij |do_i|,
plus h' |dS_j| and h' P_ij again for the backward's own P, whose divisor is the sum of the rounded ones (off by h' at most, where one key has nearly
all the weight), plus h' of the result, and 2^-13 of the sums of magnitudes for the 32-bit exponentials (an error of 2^-24 times exponents of up to 2^11, and
the two-unit error of ex2).  The table's gradient sums dS: sum over the pairs (h'/... the sums are of unrounded dS) (2^-13 |dS| + P e)."""
import math

import pytest
import torch

from savanna_b200 import ops
from savanna_b200.ops import reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16
H1 = 2.0 ** -8
SMALL = 2.0 ** -13


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _map(nb, maxd, causal):
    side = nb if causal else nb // 2
    exact = max(1, side // 2)
    d = torch.arange(maxd + 1, dtype=torch.float64)
    far = exact + torch.floor(torch.log(d.clamp(min=1) / exact) / math.log(max(maxd, exact + 1) / exact) * (side - exact) + 1e-9)
    b = torch.where(d < exact, d, far.clamp(max=side - 1)).to(torch.int32)
    return (b if causal else torch.cat([b[1:].flip(0) + side, b])).to(DEV)


def _case(B, L, H, nb, maxd, causal, seed=0, table_dtype=BF):
    g = _gen(seed)
    qkv = torch.randn(B, L, H, 384, generator=g, device=DEV).to(BF)
    table = (0.2 * torch.randn(nb, H, generator=g, device=DEV)).to(table_dtype)
    go = torch.randn(B, L, H, 128, generator=g, device=DEV).to(BF)
    return qkv, table, _map(nb, maxd, causal), go


def _exact(qkv, table, buckets, scale, causal, go):
    """(value, bound) of o, dqkv, dtable in 64 bits."""
    B, L, H, _ = qkv.shape
    sm = 1 / math.sqrt(128)
    q, k, v = (t.double().transpose(1, 2) for t in qkv.split(128, dim=-1))
    bias = ref.relative_bias(table.double(), buckets, scale, L, L, causal)
    s = q @ k.transpose(-1, -2) * sm + bias
    if causal:
        s = s.masked_fill(torch.ones(L, L, dtype=torch.bool, device=DEV).triu(1), float("-inf"))
    p = torch.softmax(s, -1)
    o = p @ v
    g = go.double().transpose(1, 2)
    dp = g @ v.transpose(-1, -2)
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    e = 2 * H1 * ds.abs().sum(-1, keepdim=True) + SMALL * (p * dp.abs()).sum(-1, keepdim=True)
    # sum_j P_j |v_j - o| <= sum_j P_j |v_j| + |o|, and no more than that where one key has nearly all the weight
    spread = torch.minimum(p @ v.abs() + o.abs(), 2 * torch.sqrt(((p @ (v * v)) - o * o).clamp(min=0)) + SMALL * (p @ v.abs()))
    bo = 2 * H1 * spread + H1 * o.abs() + SMALL * (p @ v.abs())
    # dP and delta are sums of 128 products in 32 bits, each off by up to 128 * 2^-24 * sum |do_d v_d|, however small the sum itself is (where
    # the softmax has a single key, dP - delta is 0 and this all that is left): together 2^-16 of that sum, averaged over the row in delta
    mag = g.abs() @ v.abs().transpose(-1, -2)
    e = e + 2.0 ** -16 * (p * mag).sum(-1, keepdim=True)
    err = 2 * H1 * ds.abs() + p * e + SMALL * (p * (dp.abs() + delta.abs())) + 2.0 ** -16 * p * mag
    dq, dk, dv = ds @ k * sm, ds.transpose(-1, -2) @ q * sm, p.transpose(-1, -2) @ g
    bq = sm * (err @ k.abs()) + H1 * dq.abs()
    bk = sm * (err.transpose(-1, -2) @ q.abs()) + H1 * dk.abs()
    bv = (2 * H1 + SMALL) * (p.transpose(-1, -2) @ g.abs()) + H1 * dv.abs()
    # by distance, then by bucket
    i = torch.arange(L, device=DEV)
    d = i[:, None] - i[None, :]
    far = buckets.shape[0] - 1 if causal else buckets.shape[0] // 2
    at = (d.clamp(0, far) if causal else d.clamp(-far, far) + far).reshape(-1)
    n, nb = buckets.shape[0], table.shape[0]
    one = (p * e + H1 * ds.abs() + SMALL * (p * (dp.abs() + delta.abs())) + 2.0 ** -16 * p * mag + SMALL * ds.abs()).sum(0).reshape(H, -1)
    gd = torch.zeros(n, H, dtype=torch.float64, device=DEV).index_add_(0, at, ds.sum(0).reshape(H, -1).t())
    bd = torch.zeros(n, H, dtype=torch.float64, device=DEV).index_add_(0, at, one.t())
    # what all distances add up to (their errors: exactly, they add up to 0) is taken off each in proportion to its share of P
    mass = torch.zeros(n, H, dtype=torch.float64, device=DEV).index_add_(0, at, p.sum(0).reshape(H, -1).t()) / (B * L)
    bd = bd + (mass + 1e-4) * bd.sum(0)
    gt = torch.zeros(nb, H, dtype=torch.float64, device=DEV).index_add_(0, buckets.long(), gd) * scale
    bt = torch.zeros(nb, H, dtype=torch.float64, device=DEV).index_add_(0, buckets.long(), bd) * abs(scale)
    return (o.transpose(1, 2), bo.transpose(1, 2)), (torch.cat([dq, dk, dv], -1).transpose(1, 2), torch.cat([bq, bk, bv], -1).transpose(1, 2)), \
        (gt, bt + torch.finfo(table.dtype).eps / 2 * gt.abs() + 1e-12)


def _inside(got, want, bound, what):
    err = (got.double() - want).abs()
    bad = ~(err <= bound + 1e-30)
    worst = (err / (bound + 1e-30)).nan_to_num(float("inf")).max()
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {float(worst):.3g} of the bound"


def _run(qkv, table, buckets, scale, causal, go):
    qkv, table = qkv.clone().requires_grad_(True), table.clone().requires_grad_(True)
    o = ops.attention_rpe(qkv, table, buckets, scale, causal)
    return (o.detach(), *torch.autograd.grad(o, (qkv, table), go))


def _status_ok():
    from savanna_b200.ops import cuda_ops
    torch.cuda.synchronize()
    cuda_ops.check_status()


LENGTHS = [1, 2, 3, 17, 63, 64, 65, 127, 128, 129, 200, 255, 256, 257, 383, 385, 511, 513, 777, 1300]


@pytest.mark.parametrize("causal", [True, False], ids=["causal", "both"])
@pytest.mark.parametrize("L", LENGTHS)
def test_values_and_gradients(L, causal):
    for maxd in (64, 128, 250):
        B, H = (2, 2) if L < 600 else (1, 2)
        c = _case(B, L, H, 32, maxd, causal, seed=L + maxd)
        got = _run(*c[:3], math.sqrt(128), causal, c[3])
        _status_ok()
        for name, v, (want, bound) in zip(("o", "dqkv", "dtable"), got, _exact(*c[:3], math.sqrt(128), causal, c[3])):
            _inside(v, want, bound, f"{name} maxd {maxd}")
        with torch.no_grad():
            assert torch.equal(ops.attention_rpe(*c[:3], math.sqrt(128), causal), got[0])


@pytest.mark.parametrize("causal", [True, False], ids=["causal", "both"])
@pytest.mark.parametrize("maxd,nb", [(0, 1), (1, 2), (7, 8), (500, 64), (1024, 32)])
def test_maps_from_one_distance_to_the_longest(maxd, nb, causal):
    c = _case(1, 700, 3, nb if causal else 2 * nb, maxd, causal, seed=maxd, table_dtype=torch.float32)
    got = _run(*c[:3], 3.0, causal, c[3])
    _status_ok()
    for name, v, (want, bound) in zip(("o", "dqkv", "dtable"), got, _exact(*c[:3], 3.0, causal, c[3])):
        _inside(v, want, bound, name)


@pytest.mark.parametrize("causal", [True, False], ids=["causal", "both"])
@pytest.mark.parametrize("L", [1023, 1024, 1025])
def test_where_the_probabilities_stop_entering_in_two_parts(L, causal):
    c = _case(1, L, 2, 32, 128, causal, seed=L)
    got = _run(*c[:3], math.sqrt(128), causal, c[3])
    _status_ok()
    for name, v, (want, bound) in zip(("o", "dqkv", "dtable"), got, _exact(*c[:3], math.sqrt(128), causal, c[3])):
        _inside(v, want, bound, name)
    with torch.no_grad():
        assert torch.equal(ops.attention_rpe(*c[:3], math.sqrt(128), causal), got[0])


def test_one_token_has_a_gradient_for_its_value_alone():
    for causal in (True, False):
        qkv, table, buckets, go = _case(3, 1, 5, 32, 128, causal)
        o, dqkv, dt = _run(qkv, table, buckets, 11.0, causal, go)
        assert torch.equal(o, qkv[..., 256:]) and torch.equal(dqkv[..., 256:], go)
        assert float(dqkv[..., :256].abs().max()) == 0 and float(dt.abs().max()) == 0


def test_a_bucket_of_minus_infinity_masks_its_keys_and_may_empty_a_row():
    """Distance 0 masked: the first row of a causal sequence has no key left and is zero."""
    qkv, table, buckets, go = _case(2, 300, 2, 32, 128, True)
    table[0] = float("-inf")
    o, dqkv, _ = _run(qkv, table, buckets, 2.0, True, go)
    _status_ok()
    assert float(o[:, 0].abs().max()) == 0 and not bool(o.isnan().any()) and not bool(dqkv.isnan().any())
    keep = ref.attention_rpe(qkv, table, buckets, 2.0, True)
    # both round to bf16, the kernel's probabilities too: 2^-8 of values and averages of up to the largest |v|
    assert float((o.float() - keep.float()).abs().max()) <= 3 * H1 * float(qkv[..., 256:].abs().max())


@pytest.mark.parametrize("value", [torch.finfo(torch.float32).min / 16, -1e9])
def test_a_bucket_of_the_lowest_values_masks_its_keys(value):
    qkv, table, buckets, go = _case(1, 300, 2, 32, 128, True, table_dtype=torch.float32)
    table[5] = value
    o, dqkv, dt = _run(qkv, table, buckets, 1.0, True, go)
    _status_ok()
    assert not bool(o.isnan().any()) and not bool(dqkv.isnan().any()) and not bool(dt.isnan().any())
    (want, bound), (wg, bg), (wt, bt) = _exact(qkv, table, buckets, 1.0, True, go)
    _inside(o, want, bound, "o")
    _inside(dqkv, wg, bg, "dqkv")
    _inside(dt, wt, bt, "dtable")


def test_table_types_agree_and_other_types_are_converted():
    qkv, table, buckets, go = _case(1, 260, 2, 32, 128, True)
    a = _run(qkv, table, buckets, 4.0, True, go)
    b = _run(qkv, table.float(), buckets, 4.0, True, go)
    c = _run(qkv, table.half(), buckets, 4.0, True, go)
    assert torch.equal(a[0], b[0]) and a[2].dtype == BF and b[2].dtype == torch.float32 and c[2].dtype == torch.float16
    assert torch.equal(a[2], b[2].to(BF))


def test_table_gradient_is_repeatable_and_buffers_are_left_alone():
    from savanna_b200.ops import cuda_ops
    for causal in (True, False):
        c = _case(2, 333, 3, 32, 100, causal)
        with cuda_ops.guarded_allocations():
            first = _run(*c[:3], 2.0, causal, c[3])
            assert cuda_ops.check_guards() >= 6
        for _ in range(3):
            again = _run(*c[:3], 2.0, causal, c[3])
            assert torch.equal(first[0], again[0]) and torch.equal(first[2], again[2])
    _status_ok()


def test_strided_output_gradient_and_other_stream():
    qkv, table, buckets, go = _case(2, 200, 2, 32, 64, True)
    want = _run(qkv, table, buckets, 2.0, True, go)
    odd = torch.empty(2, 200, 2, 129, device=DEV, dtype=BF)[..., 1:]
    odd.copy_(go)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(qkv, table, buckets, 2.0, True, odd)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(want[0], got[0]) and torch.equal(want[2], got[2])
    expanded = _run(qkv, table, buckets, 2.0, True, torch.ones(1, 1, 1, 1, device=DEV, dtype=BF).expand(2, 200, 2, 128))
    same = _run(qkv, table, buckets, 2.0, True, torch.ones(2, 200, 2, 128, device=DEV, dtype=BF))
    assert torch.equal(expanded[2], same[2])


def test_odd_strides_of_dimensions_of_size_one_and_gradients_off_16_bytes():
    qkv, table, buckets, go = _case(1, 150, 2, 32, 64, True)

    def run(x, g):
        x, t = x.detach().requires_grad_(True), table.clone().requires_grad_(True)
        o = ops.attention_rpe(x, t, buckets, 2.0, True)
        return (o.detach(), *torch.autograd.grad(o, (x, t), g))

    def after(t, start, end):                        # the same values in the middle of a longer row
        row = torch.zeros(1, start + t.numel() + end, device=DEV, dtype=BF)[:, start: start + t.numel()]
        row.copy_(t.view(1, -1))
        return row.view(t.shape)
    want = run(qkv, go)
    for x, g in ((after(qkv, 0, 3), go), (qkv, after(go, 0, 5)), (qkv, after(go, 1, 0)), (after(qkv, 8, 1), after(go, 3, 2))):
        assert x.is_contiguous() and g.is_contiguous()
        got = run(x, g)
        _status_ok()
        assert torch.equal(want[0], got[0]) and torch.equal(want[2], got[2])
        # dq is added up in an order that varies: a step of bf16 between two sums; dk and dv are not
        assert torch.equal(want[1][..., 128:], got[1][..., 128:])
        assert bool(((want[1].double() - got[1].double()).abs() <= 2.0 ** -7 * want[1].double().abs() + 2.0 ** -20 * want[1].abs().max()).all())


def test_captured_forward_and_backward():
    qkv, table, buckets, go = _case(1, 400, 2, 32, 128, True)
    want = _run(qkv, table, buckets, 2.0, True, go)
    ql, tl = qkv.clone().requires_grad_(True), table.clone().requires_grad_(True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = ops.attention_rpe(ql, tl, buckets, 2.0, True)
        gq, gt = torch.autograd.grad(o, (ql, tl), go)
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(o, want[0]) and torch.equal(gt, want[2])
    _status_ok()


def test_shapes_that_the_kernels_do_not_cover_run_the_statement():
    g = _gen(1)
    buckets = _map(32, 128, True)
    for qkv in (torch.randn(1, 20, 2, 3 * 64, generator=g, device=DEV).to(BF), torch.randn(1, 20, 2, 384, generator=g, device=DEV)):
        table = torch.randn(32, 2, generator=g, device=DEV)
        assert torch.equal(ops.attention_rpe(qkv, table, buckets, 2.0, True), ref.attention_rpe(qkv, table, buckets, 2.0, True))
    far = _map(32, 4000, True)
    qkv = torch.randn(1, 20, 2, 384, generator=g, device=DEV).to(BF)
    assert not ops.attention_rpe_covers(qkv, 4000) and ops.attention_rpe(qkv, torch.randn(32, 2, device=DEV), far, 2.0, True).shape == (1, 20, 2, 128)


def test_empty_batch():
    qkv = torch.empty(0, 5, 2, 384, device=DEV, dtype=BF, requires_grad=True)
    table = torch.randn(32, 2, device=DEV, requires_grad=True)
    o = ops.attention_rpe(qkv, table, _map(32, 128, True), 1.0, True)
    gq, gt = torch.autograd.grad(o, (qkv, table), torch.empty_like(o))
    assert o.shape == (0, 5, 2, 128) and gq.shape == qkv.shape and float(gt.abs().sum()) == 0


def test_refusals():
    qkv, table, buckets, _ = _case(1, 6, 2, 8, 4, True)
    both = torch.zeros(9, dtype=torch.int32, device=DEV)
    for bad in ((qkv[..., :383], table, buckets, 1.0, True), (qkv[0], table, buckets, 1.0, True), (qkv, table[:, :1], buckets, 1.0, True),
                (qkv, table, buckets.long(), 1.0, True), (qkv, table, buckets[:0], 1.0, True), (qkv, table, both[:8], 1.0, False),
                (qkv, table.to(torch.int32), buckets, 1.0, True), (qkv, table[0], buckets, 1.0, True), (qkv, table.cpu(), buckets, 1.0, True),
                (qkv, table, buckets.cpu(), 1.0, True)):
        with pytest.raises(ValueError):
            ops.attention_rpe(*bad)


def test_buckets_that_do_not_exist_have_no_bias_and_no_gradient():
    qkv, table, buckets, go = _case(1, 150, 2, 32, 128, True)
    odd = buckets.clone()
    odd[buckets == 3], odd[buckets == 9] = -1, 40
    zero = table.clone()
    zero[3], zero[9] = 0, 0
    a, b = _run(qkv, table, odd, 2.0, True, go), _run(qkv, zero, buckets, 2.0, True, go)
    assert torch.equal(a[0], b[0])
    keep = torch.ones(32, dtype=torch.bool, device=DEV)
    keep[3] = keep[9] = False
    assert torch.equal(a[2][keep], b[2][keep]) and float(a[2][~keep].abs().max()) == 0


@pytest.mark.filterwarnings("ignore")
def test_traced_on_new_inputs():
    qkv, table, buckets, _ = _case(1, 70, 2, 32, 64, True)
    other = _case(1, 70, 2, 32, 64, True, seed=9)[0]

    def f(x):
        return ops.attention_rpe(x, table, buckets, 2.0, True)
    traced = torch.jit.trace(f, qkv, check_trace=False)
    assert torch.equal(traced(other), f(other))


@pytest.mark.parametrize("causal", [True, False], ids=["causal", "both"])
def test_second_derivatives(causal):
    """create_graph goes through elementary operations, whose gradients are those of the statement."""
    qkv, table, buckets, go = _case(1, 20, 2, 32, 16, causal, table_dtype=torch.float32)

    def second(f):
        a, t = qkv.clone().requires_grad_(True), table.clone().requires_grad_(True)
        ga, gt = torch.autograd.grad(f(a, t), (a, t), go, create_graph=True)
        return torch.autograd.grad(ga.float().square().sum() + gt.square().sum(), (a, t))
    got = second(lambda a, t: ops.attention_rpe(a, t, buckets, 2.0, causal))
    want = second(lambda a, t: ref.attention_rpe(a, t, buckets, 2.0, causal))
    for x, y in zip(got, want):                      # the same sums in another order, then bf16
        assert (x.float() - y.float()).norm() <= 2 * H1 * y.float().norm()


def test_forward_mode_runs_the_statement():
    qkv, table, buckets, _ = _case(1, 12, 2, 32, 16, True, table_dtype=torch.float32)
    t = torch.randn_like(table)
    f = lambda v: ops.attention_rpe(qkv, v, buckets, 2.0, True)  # noqa: E731
    p = lambda v: ref.attention_rpe(qkv, v, buckets, 2.0, True)  # noqa: E731
    assert torch.equal(torch.func.jvp(f, (table,), (t,))[1], torch.func.jvp(p, (table,), (t,))[1])
