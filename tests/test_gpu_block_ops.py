"""Layer norm and 8-bit activations on CUDA against their definitions in 64 bits.

Tolerances count roundings.  With u = 2^-24 (fp32) and h = eps / 2 of the output's type: a sum of n values in fp32 is off by at most
(its longest chain of additions) * u * sum |values|; chains here are at most 64 values of a thread, 5 + 5 steps of a tree and, over
the rows, the rows of a block and 32 partial rows.  The final rounding adds h * |value| (and half a smallest subnormal step in fp16)."""
import pytest
import torch

from savanna_b200 import ops
from savanna_b200.ops import reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _floor(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def _inside(got, want, bound, what):
    """Element by element, in 64 bits."""
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {float((err / bound.clamp(min=1e-300)).max()):.3g} of the bound"


def _norm_case(rows, D, dtype, seed=0, mean=0.5):
    g = _gen(seed)
    x = (torch.randn(rows, D, generator=g, device=DEV) + mean).to(dtype)
    w = (1 + 0.1 * torch.randn(D, generator=g, device=DEV)).to(dtype)
    b = (0.1 * torch.randn(D, generator=g, device=DEV)).to(dtype)
    gy = torch.randn(rows, D, generator=g, device=DEV).to(dtype)
    gr = torch.randn(rows, D, generator=g, device=DEV).to(dtype)
    return x, w, b, gy, gr


def _norm_exact(x, w, b, gy, gr, eps, dtype):
    """Values and bounds of y, dx, dw, db."""
    x, w, b, gy = (t.double() for t in (x, w, b, gy))
    rows, D = x.shape
    m = x.mean(-1, keepdim=True)
    var = ((x - m) ** 2).mean(-1, keepdim=True)
    r = 1 / torch.sqrt(var + eps)
    xh = (x - m) * r
    y = xh * w + b
    # the mean is off by 80 u mean|x| at most; the variance's relative error is twice that of the differences, 160 u (mean |x| r)^2 / ... is
    # covered by the same term on xh: |d xh| <= 96 u r (|x| + mean|x|) + 100 u |xh| (1 + mean|x| r)
    ax = x.abs().mean(-1, keepdim=True)
    dxh = 96 * U * r * (x.abs() + ax) + 100 * U * xh.abs() * (1 + ax * r)
    h, lo = _half(dtype), _floor(dtype)
    out = {"y": (y, h * y.abs() + lo + w.abs() * dxh + 4 * U * (b.abs() + y.abs()))}
    g = gy * w
    c1, c2 = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
    dx = r * (g - c1 - xh * c2) + (gr.double() if gr is not None else 0)
    d1 = 80 * U * g.abs().mean(-1, keepdim=True)
    d2 = (g.abs() * dxh).mean(-1, keepdim=True) + 80 * U * (g * xh).abs().mean(-1, keepdim=True)
    rr = 100 * U * (1 + ax * r)                                                  # relative error of rstd
    ddx = r * (d1 + xh.abs() * d2 + dxh * c2.abs()) + (rr + 8 * U) * r * (g.abs() + c1.abs() + (xh * c2).abs())
    out["dx"] = (dx, h * dx.abs() + lo + ddx + 4 * U * dx.abs() + (4 * U * gr.double().abs() if gr is not None else 0))
    dw, db = (gy * xh).sum(0), gy.sum(0)
    chain = rows + 64
    out["dw"] = (dw, h * dw.abs() + lo + (gy.abs() * dxh).sum(0) + chain * U * (gy * xh).abs().sum(0))
    out["db"] = (db, h * db.abs() + lo + chain * U * gy.abs().sum(0))
    return out


WIDTHS = [1, 2, 3, 4, 6, 8, 12, 33, 64, 100, 136, 256, 257, 1000, 1024, 1027, 2048, 2056, 4096, 4104, 5001, 8191, 8192, 8196, 12000, 12001, 16370, 16372, 16383, 16384]


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("D", WIDTHS)
def test_layernorm_values_and_gradients(D, dtype):
    for rows in (1, 2, 5, 333 if D > 2048 else 1301):
        for residual in (False, True):
            x, w, b, gy, gr = _norm_case(rows, D, dtype, seed=D + rows)
            want = _norm_exact(x, w, b, gy, gr if residual else None, 1e-5, dtype)
            leaves = [t.requires_grad_(True) for t in (x, w, b)]
            if residual:
                y, xr = ops.layernorm_residual(*leaves, 1e-5)
                assert torch.equal(xr, x)
                got = torch.autograd.grad((y, xr), leaves, (gy, gr))
            else:
                y = ops.layernorm(*leaves, 1e-5)
                got = torch.autograd.grad(y, leaves, gy)
            for name, v in zip(("y", "dx", "dw", "db"), (y.detach(), *got)):
                assert v.dtype == dtype
                _inside(v, *want[name], f"{name} rows {rows} residual {residual}")
            with torch.no_grad():
                assert torch.equal(ops.layernorm(x, w, b, 1e-5), y)


def test_layernorm_of_rows_far_from_zero():
    """A mean a thousand times the spread: the difference of two sums of squares would leave nothing of the variance."""
    x, w, b, gy, _ = _norm_case(64, 4096, torch.float32, mean=1000.0)
    want = _norm_exact(x, w, b, gy, None, 1e-5, torch.float32)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = ops.layernorm(*leaves, 1e-5)
    got = torch.autograd.grad(y, leaves, gy)
    for name, v in zip(("y", "dx", "dw", "db"), (y.detach(), *got)):
        _inside(v, *want[name], name)
    assert float((y.detach().double() - want["y"][0]).abs().max()) < 2e-3


def test_layernorm_constant_rows_and_nan():
    x = torch.full((3, 128), 2.0, device=DEV, dtype=torch.bfloat16)
    w, b = torch.ones(128, device=DEV, dtype=torch.bfloat16), torch.full((128,), 0.5, device=DEV, dtype=torch.bfloat16)
    assert torch.equal(ops.layernorm(x, w, b, 1e-5), torch.full_like(x, 0.5))
    x[1, 5] = float("nan")
    y = ops.layernorm(x, w, b, 1e-5)
    assert bool(y[1].isnan().all()) and not bool(y[0].isnan().any()) and not bool(y[2].isnan().any())


def test_layernorm_views_empty_and_three_dimensions():
    g = _gen(3)
    big = torch.randn(4, 6, 200, generator=g, device=DEV).to(torch.bfloat16)
    w, b = torch.randn(96, generator=g, device=DEV).to(torch.bfloat16), torch.randn(96, generator=g, device=DEV).to(torch.bfloat16)
    for x in (big[:, 1:5, 3:99], big.transpose(0, 1)[..., 8:104], big.flatten()[1:1 + 96 * 20].view(20, 96)):
        y = ops.layernorm(x, w, b, 1e-5)
        assert y.shape == x.shape
        assert torch.equal(y, ops.layernorm(x.clone(memory_format=torch.contiguous_format), w, b, 1e-5))
    leaves = [t.clone().requires_grad_(True) for t in (big[:0, :, :96], w, b)]
    y = ops.layernorm(*leaves, 1e-5)
    dx, dw, db = torch.autograd.grad(y, leaves, torch.empty_like(y))
    assert y.shape == (0, 6, 96) and dx.shape == (0, 6, 96) and float(dw.abs().sum()) == 0 and float(db.abs().sum()) == 0


def test_layernorm_residual_uses_either_gradient_alone():
    x, w, b, gy, gr = _norm_case(40, 512, torch.bfloat16)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y, xr = ops.layernorm_residual(*leaves, 1e-5)
    only = torch.autograd.grad(xr, leaves, gr, allow_unused=True, retain_graph=True)
    assert torch.equal(only[0], gr) and only[1] is None and only[2] is None
    _inside(torch.autograd.grad(y, leaves, gy)[0], *_norm_exact(x.detach(), w.detach(), b.detach(), gy, None, 1e-5, torch.bfloat16)["dx"], "dx")


def test_layernorm_is_repeatable_in_guarded_buffers_and_in_graphs():
    from savanna_b200.ops import cuda_ops
    x, w, b, gy, gr = _norm_case(777, 1000, torch.bfloat16)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]

    def step():
        y, xr = ops.layernorm_residual(*leaves, 1e-5)
        return (y.detach(), *torch.autograd.grad((y, xr), leaves, (gy, gr)))
    with cuda_ops.guarded_allocations():
        want = step()
        assert cuda_ops.check_guards() >= 5
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(want, again))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(want, held))


def test_layernorm_module_runs_the_kernels():
    from savanna_b200.models.norms import LayerNorm
    from savanna_b200.ops import cuda_ops
    g = _gen(5)
    m = LayerNorm(384, 1e-5, dtype=torch.bfloat16, device=DEV)
    with torch.no_grad():
        m.weight.normal_(generator=g)
        m.bias.normal_(generator=g)
    x = torch.randn(2, 37, 384, generator=g, device=DEV).to(torch.bfloat16).requires_grad_(True)
    before = cuda_ops.launch_count()
    y = m(x)
    u, xr = m.forward_with_residual(x)
    assert cuda_ops.launch_count() - before == 2 and torch.equal(u, y)
    (u.float().sum() + 2 * xr.float().sum()).backward()
    want = torch.nn.functional.layer_norm(x.detach().float(), (384,), m.weight.detach().float(), m.bias.detach().float(), 1e-5)
    # both round the same 32-bit value, off by a few u: at most one step of bf16 apart
    assert bool(((y.float() - want).abs() <= 2 * _half(torch.bfloat16) * want.abs() + 1e-5).all())
    assert m.weight.grad is not None and m.bias.grad is not None


# ----------------------------------------------------------------------------- 8-bit activations


def _blocks(t, n):
    return torch.nn.functional.pad(t, (0, n * 128 - t.shape[-1])).view(*t.shape[:-1], n, 128)


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (2, 128), (5, 129), (2, 3, 1000), (999, 1003), (64, 4096), (1, 16384)])
def test_activations_come_back_within_half_a_step(shape, dtype):
    g = _gen(sum(shape))
    x = (torch.randn(*shape, generator=g, device=DEV) * torch.exp(torch.randn(shape[-1], generator=g, device=DEV))).to(dtype)
    q, scale = ops.act_quantize(x)
    back = ops.act_dequantize(q, scale, dtype)
    n = -(-shape[-1] // 128)
    assert q.dtype == torch.int8 and q.shape == x.shape and scale.shape == (*shape[:-1], n) and back.dtype == dtype
    amax = _blocks(x.double(), n).abs().amax(-1)
    _inside(scale, amax / 127, 2 * U * amax / 127, "scale")
    assert int(_blocks(q.int(), n).abs().amax(-1).min()) == 127
    # half a step of amax / 127; x * (127 / amax) is off by 3 u of up to 127, the product q * scale by 2 u; then x's own rounding
    a = amax.repeat_interleave(128, -1)[..., : shape[-1]]
    _inside(back, x.double(), a / 254 + 8 * U * a + _half(dtype) * back.double().abs() + _floor(dtype), "x")


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "fp16", "fp32"])
def test_activations_vector_and_scalar_paths_agree(dtype):
    g = _gen(9)
    flat = torch.randn(40 * 264 + 1, generator=g, device=DEV).to(dtype)
    a, b = flat[:-1].clone().view(40, 264), flat[1:].view(40, 264)
    b.copy_(a)                                                # the same values off a 16-byte boundary
    for x, y in zip(ops.act_quantize(a), ops.act_quantize(b)):
        assert torch.equal(x, y)


def test_activations_zero_infinite_and_nan_blocks():
    x = torch.zeros(4, 256, device=DEV, dtype=torch.bfloat16)
    x[1, 3], x[2, 200], x[3, 0] = float("inf"), float("nan"), 1.0
    x[1, 130] = 5.0
    q, scale = ops.act_quantize(x)
    back = ops.act_dequantize(q, scale, torch.bfloat16)
    assert torch.equal(back[0], x[0]) and torch.equal(back[3], x[3])
    assert bool(back[1, :128].isnan().all()) and bool(back[2, 128:].isnan().all())
    assert float(back[1, 130]) == 5.0 and not bool(back[2, :128].isnan().any())


def test_activations_guarded_and_empty():
    from savanna_b200.ops import cuda_ops
    with cuda_ops.guarded_allocations():
        for shape in ((7, 130), (3, 256), (0, 64), (1, 8)):
            x = torch.randn(*shape, device=DEV).to(torch.bfloat16)
            q, scale = ops.act_quantize(x)
            assert ops.act_dequantize(q, scale).shape == shape
        assert cuda_ops.check_guards() > 0


def test_refusals():
    x, w = torch.randn(2, 8, device=DEV), torch.ones(8, device=DEV)
    for bad in ((x, w[:7], w), (x, w, torch.ones(8, 1, device=DEV)), (torch.randn(3, 0, device=DEV), w, w), (torch.tensor(1.0, device=DEV), w, w)):
        with pytest.raises(ValueError):
            ops.layernorm(*bad, 1e-5)
        with pytest.raises(ValueError):
            ops.layernorm_residual(*bad, 1e-5)
    for bad in (torch.zeros(3, 4, dtype=torch.int32, device=DEV), torch.zeros(3, 0, device=DEV), torch.tensor(1.0, device=DEV)):
        with pytest.raises(ValueError):
            ops.act_quantize(bad)
    q, scale = ops.act_quantize(torch.randn(3, 200, device=DEV))
    for bad in ((q.float(), scale, torch.bfloat16), (q, scale[:, :1], torch.bfloat16), (q, scale.double(), torch.bfloat16), (q, scale, torch.float64),
                (q, scale.cpu(), torch.bfloat16)):
        with pytest.raises(ValueError):
            ops.act_dequantize(*bad)


def test_types_and_sizes_that_the_kernels_do_not_cover_run_pytorchs():
    g = _gen(8)
    with pytest.raises(RuntimeError):                # as there
        ops.layernorm(torch.randn(3, 64, device=DEV).to(torch.bfloat16), torch.randn(64, device=DEV), torch.randn(64, device=DEV), 1e-5)
    for x, w in ((torch.randn(2, 20000, generator=g, device=DEV), torch.randn(20000, generator=g, device=DEV)),
                 (torch.randn(2, 10, generator=g, device=DEV).double(), torch.randn(10, generator=g, device=DEV).double())):
        want = torch.nn.functional.layer_norm(x, (x.shape[-1],), w, w, 1e-5)
        assert torch.equal(ops.layernorm(x, w, w, 1e-5), want)
        y, xr = ops.layernorm_residual(x, w, w, 1e-5)
        assert torch.equal(y, want) and xr is x


@pytest.mark.filterwarnings("ignore")
def test_traced_operators_run_on_new_inputs():
    w, b = torch.randn(64, device=DEV), torch.randn(64, device=DEV)

    def f(x):
        return ops.act_dequantize(*ops.act_quantize(ops.layernorm(x, w, b, 1e-5)), torch.float32)
    g = _gen(2)
    x, z = torch.randn(5, 64, generator=g, device=DEV), torch.randn(5, 64, generator=g, device=DEV)
    traced = torch.jit.trace(f, x, check_trace=False)
    assert torch.equal(traced(z), f(z)) and not torch.equal(traced(z), f(x))


def test_values_halfway_between_two_codes_go_to_the_even_one():
    """With amax = 127 a code is the value itself: halves are ties."""
    x = torch.arange(-127, 128, device=DEV).float().div(2).repeat(2)[:384].clone()
    x[::128] = 127.0
    for dtype in (torch.float16, torch.float32):
        q, scale = ops.act_quantize(x.to(dtype).view(1, 384))
        assert torch.equal(scale, torch.ones_like(scale)) and torch.equal(q[0].float(), torch.round(x))


@pytest.mark.parametrize("D", [33, 100, 1027, 4095])
def test_layernorm_of_odd_widths_leaves_neighbours_alone(D):
    """A row of NaN between others, and nothing written outside: vectors reach into the rows before and behind."""
    from savanna_b200.ops import cuda_ops
    for rows in (1, 3, 40):
        x, w, b, gy, gr = _norm_case(rows, D, torch.bfloat16, seed=rows)
        want = _norm_exact(x, w, b, gy, gr, 1e-5, torch.bfloat16)
        bad = rows // 2
        x[bad], gy[bad], gr[bad] = float("nan"), float("inf"), float("nan")
        leaves = [t.requires_grad_(True) for t in (x, w, b)]
        with cuda_ops.guarded_allocations():
            y, xr = ops.layernorm_residual(*leaves, 1e-5)
            dx, dw, db = torch.autograd.grad((y, xr), leaves, (gy, gr))
            assert cuda_ops.check_guards() >= 5
        keep = torch.arange(rows, device=DEV) != bad
        for name, v in (("y", y.detach()), ("dx", dx)):
            assert bool(v[bad].isnan().all())
            _inside(v[keep], want[name][0][keep], want[name][1][keep], name)
        assert bool(dw.isnan().all())


@pytest.mark.parametrize("residual", [False, True])
def test_layernorm_second_derivatives(residual):
    g = _gen(4)
    x, w, b = (torch.randn(*s, generator=g, device=DEV) for s in ((6, 40), (40,), (40,)))
    r, q = torch.randn(6, 40, generator=g, device=DEV), torch.randn(6, 40, generator=g, device=DEV)

    def second(f, t):
        leaves = [v.clone().to(t).requires_grad_(True) for v in (x, w, b)]
        y, xr = f(*leaves)
        dx, dw, db = torch.autograd.grad((y * r.to(t)).sum() + (xr * xr).sum(), leaves, create_graph=True)
        return torch.autograd.grad((dx * q.to(t)).sum() + (dw * dw).sum(), leaves, allow_unused=True)
    plain = lambda x, w, b: (torch.nn.functional.layer_norm(x, (40,), w, b, 1e-5), x)  # noqa: E731
    own = (lambda x, w, b: ops.layernorm_residual(x, w, b, 1e-5)) if residual else (lambda x, w, b: (ops.layernorm(x, w, b, 1e-5), x))
    for a, c in zip(second(own, torch.float32), second(plain, torch.float64)):
        if c is None or float(c.abs().max()) == 0:
            assert a is None or float(a.abs().max()) <= 1e-3
        else:                                        # 40-term sums of products of up to five factors in fp32: a few hundred roundings
            assert float((a.double() - c).abs().max()) <= 1024 * U * float(c.abs().max()) * 8


def test_layernorm_leaves_transforms_and_autocast_to_pytorch():
    g = _gen(6)
    x, w, b = torch.randn(4, 32, generator=g, device=DEV), torch.randn(32, generator=g, device=DEV), torch.randn(32, generator=g, device=DEV)
    t = torch.randn(4, 32, generator=g, device=DEV)
    f = lambda v: ops.layernorm(v, w, b, 1e-5)  # noqa: E731
    p = lambda v: torch.nn.functional.layer_norm(v, (32,), w, b, 1e-5)  # noqa: E731
    assert torch.allclose(torch.func.jvp(f, (x,), (t,))[1], torch.func.jvp(p, (x,), (t,))[1])
    assert torch.allclose(torch.vmap(f)(x), p(x), atol=1e-5)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert f(x.to(torch.bfloat16).float()).dtype == p(x).dtype == torch.float32
    with torch.autocast("cuda", dtype=torch.bfloat16):
        h = [v.to(torch.bfloat16) for v in (x, w, b)]
        assert ops.layernorm(*h, 1e-5).dtype == torch.nn.functional.layer_norm(h[0], (32,), h[1], h[2], 1e-5).dtype


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("T,D", [(743, 7091), (1000, 1024), (3000, 200)])
def test_codes_are_those_of_the_statement(T, D, dtype):
    from savanna_b200.ops import reference as ref
    g = torch.Generator(device=DEV).manual_seed(T)
    x = (torch.randn(T, D, generator=g, device=DEV) * torch.exp2(torch.randint(-60, 60, (T, 1), generator=g, device=DEV))).to(dtype)
    x = x.nan_to_num(0.0, 1000.0, -1000.0)           # what fp16 does not hold
    q, scale = ops.act_quantize(x)
    for want, s in (ref.act_quantize(x), [t.to(DEV) for t in ref.act_quantize(x.cpu())]):
        assert torch.equal(q, want)
        # amax / 127 by a division or by a product with 1 / 127
        assert float(((scale - s).abs() / s.clamp(min=1e-30)).max()) <= 2 * 2.0 ** -23
