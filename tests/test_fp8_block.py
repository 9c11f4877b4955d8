"""8-bit operands with a scale for each block of 128 on the CPU: the statement against the definition in 64 bits, its gradients, and refusals."""
import pytest
import torch

from savanna_b200 import ops
from tests.fp8_block_oracle import blockwise, close_sum, half_step, tiles

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _randn(*shape, seed=0, dtype=torch.bfloat16, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 130), (2, 5, 128), (7, 300), (64,)])
def test_rows(shape, dtype):
    x = _randn(*shape, dtype=dtype)
    q, s = ops.fp8_block_quantize(x)
    assert q.shape == x.shape and q.dtype == torch.float8_e4m3fn and s.shape == x.shape[:-1] + (-(-x.shape[-1] // 128),)
    want = blockwise(x.double(), x.dim() - 1)
    got = ops.fp8_block_dequantize(q, s, torch.float32).double()
    if dtype != torch.float32:          # quotients of 16-bit values fall on the same code; the scale and its product carry a rounding each
        assert ((got - want).abs() <= 2.0 ** -22 * want.abs()).all()
    else:
        assert ((got - x.double()).abs() <= 2.0 ** -4 * x.double().abs() * (1 + 2.0 ** -20) + s.double().amax() * 2.0 ** -10).all()


@pytest.mark.parametrize("shape", [(1, 1), (128, 128), (130, 300), (5, 1000)])
def test_tiles(shape):
    w = _randn(*shape)
    q, s = ops.fp8_block_quantize_weight(w)
    assert s.shape == (-(-shape[0] // 128), -(-shape[1] // 128))
    want = tiles(w.double())
    assert ((ops.fp8_block_dequantize(q, s, torch.float32).double() - want).abs() <= 2.0 ** -22 * want.abs()).all()


def test_zeros_and_what_is_not_finite():
    x = torch.zeros(3, 300)
    x[1, 5], x[2, 200] = float("inf"), float("nan")
    q, s = ops.fp8_block_quantize(x)
    back = ops.fp8_block_dequantize(q, s, torch.float32)
    assert (back[0] == 0).all() and back[1, :128].isnan().all() and (back[1, 128:] == 0).all()
    assert back[2, 128:256].isnan().all() and (back[2, :128] == 0).all()


def test_huge_and_tiny_values_keep_their_relative_precision():
    x = torch.tensor([[3e38, 1e38, -3.3e38, 1e36], [1e-37, 3e-38, 0.0, 1e-30]])
    back = ops.fp8_block_dequantize(*ops.fp8_block_quantize(x), torch.float32)
    assert (back[0] - x[0]).abs().max() <= 2.0 ** -4 * 3.3e38 and back.isfinite().all()
    assert (back[1] - x[1]).abs().max() <= 2.0 ** -4 * 1e-30 + 2.0 ** -110


def _close(got, want, tol):
    assert got.shape == want.shape
    assert (got.double() - want).norm() <= tol * want.norm().clamp(min=1e-30)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,K,N", [(1, 1, 1), (5, 130, 7), (150, 260, 140)])
def test_linear_and_its_gradients(T, K, N, dtype):
    x, w, b, r, gy = (_randn(*s, seed=i, dtype=dtype) for i, s in enumerate([(T, K), (N, K), (N,), (T, N), (T, N)]))
    leaves = [t.requires_grad_() for t in (x, w, b, r)]
    y = ops.linear_fp8_block(x, w, b, r)
    gx, gw, gb, gr = torch.autograd.grad(y, leaves, gy)
    xd, wd, gd = x.detach().double(), w.detach().double(), gy.double()
    wq = tiles(wd)
    # one rounding of the result; fp32 operands may fall on the neighbouring code where the definition in 64 bits lies beside a border
    tol = 2 * half_step(dtype) + (1e-3 if dtype == torch.float32 else 1e-5)
    _close(y, blockwise(xd, 1) @ wq.t() + b.detach().double() + r.detach().double(), tol)
    _close(gx, blockwise(gd, 1) @ wq, tol)
    _close(gw, blockwise(gd, 0).t() @ blockwise(xd, 0), tol)
    _close(gb, gd.sum(0), tol)
    assert torch.equal(gr, gy)


@pytest.mark.parametrize("form", ["te", "classic"])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_and_projection(form, residual):
    T, K, N = 9, 300, 40
    x, r, g, w = (_randn(*s, seed=i).float() for i, s in enumerate([(T, K), (T, K), (K,), (N, K)]))
    r = r if residual else None
    q, s, kept = ops.rmsnorm_fp8_block(x, g, 1e-5, form, r)
    h = x if r is None else x + r
    assert torch.equal(kept, h)
    ms = h.double().square().mean(-1, keepdim=True)
    y = h.double() / ((ms + 1e-5).sqrt() if form == "te" else ms.sqrt() + 1e-5) * g.double()
    _close(ops.fp8_block_dequantize(q, s, torch.float32), blockwise(y, 1), 1e-3)
    out, kept = ops.norm_linear_fp8_block(x, g, 1e-5, form, w, None, r)
    _close(out, blockwise(y, 1) @ tiles(w.double()).t(), 1e-3)
    assert torch.equal(kept, h)


def test_gradient_of_the_norm_and_its_residual():
    T, K, N = 9, 300, 40
    x, r, g, w, gy, gs = (_randn(*s, seed=i).float() for i, s in enumerate([(T, K), (T, K), (K,), (N, K), (T, N), (T, K)]))
    leaves = [t.requires_grad_() for t in (x, r, g, w)]
    y, s = ops.norm_linear_fp8_block(x, g, 1e-5, "te", w, None, r)
    gx, gr, gg, gw = torch.autograd.grad((y, s), leaves, (gy, gs))
    h = (x + r).detach().double().requires_grad_()
    gain = g.detach().double().requires_grad_()
    n = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-5) * gain
    dn = blockwise(gy.double(), 1) @ tiles(w.detach().double())
    wx, wg = torch.autograd.grad((n, h), (h, gain), (dn, gs.double()))
    _close(gx, wx, 1e-3)
    _close(gg, wg, 1e-3)
    assert torch.equal(gx, gr)
    _close(gw, blockwise(gy.double(), 0).t() @ blockwise(n.detach(), 0), 1e-3)


def test_kept_weight_gives_the_same_result_and_passes_gradients_to_the_input():
    x, w = _randn(5, 200), _randn(70, 200, seed=1)
    kept = ops.fp8_block_quantize_weight(w)
    x.requires_grad_()
    a, b = ops.linear_fp8_block(x, w), ops.linear_fp8_block(x, kept)
    assert torch.equal(a, b)
    assert torch.equal(*(torch.autograd.grad(y, x, torch.ones_like(y))[0] for y in (a, b)))
    with torch.no_grad():
        assert torch.equal(ops.linear_fp8_block(ops.fp8_block_quantize(x), kept), a)
        assert ops.linear_fp8_block(ops.fp8_block_quantize(x), kept, dtype=torch.float32).dtype == torch.float32


def refusals(device):
    x, w, b = _randn(4, 200).to(device), _randn(70, 200).to(device), _randn(70).to(device)
    q, s = ops.fp8_block_quantize(x)
    wq, ws = ops.fp8_block_quantize_weight(w)
    g = _randn(200).to(device)
    return [
        lambda: ops.fp8_block_quantize(x.int()),
        lambda: ops.fp8_block_quantize(x[0, 0]),
        lambda: ops.fp8_block_quantize(x[:, :0]),
        lambda: ops.fp8_block_quantize(x.double()),
        lambda: ops.fp8_block_quantize_weight(w[0]),
        lambda: ops.fp8_block_dequantize(q, s[:, :1]),
        lambda: ops.fp8_block_dequantize(q, s.half()),
        lambda: ops.fp8_block_dequantize(x, s),
        lambda: ops.fp8_block_dequantize(q, s, torch.int32),
        lambda: ops.rmsnorm_fp8_block(x, g[:5], 1e-5),
        lambda: ops.rmsnorm_fp8_block(x, g.float(), 1e-5),
        lambda: ops.rmsnorm_fp8_block(x, g, 1e-5, "other"),
        lambda: ops.rmsnorm_fp8_block(x, g, 1e-5, "te", x[:2]),
        lambda: ops.rmsnorm_fp8_block(x, g, 1e-5, "te", x.float()),
        lambda: ops.linear_fp8_block(x, w[:, :100]),
        lambda: ops.linear_fp8_block(x, w.float()),
        lambda: ops.linear_fp8_block(x, w[0]),
        lambda: ops.linear_fp8_block(x, w[:0]),
        lambda: ops.linear_fp8_block(x, w, b[:3]),
        lambda: ops.linear_fp8_block(x, w, b.float()),
        lambda: ops.linear_fp8_block(x, w, None, x),
        lambda: ops.linear_fp8_block(x, w, dtype=torch.float32),
        lambda: ops.linear_fp8_block((q, s), w, dtype=torch.int8),
        lambda: ops.linear_fp8_block((q, s[:, :1]), (wq, ws)),
        lambda: ops.linear_fp8_block(x, (wq, ws[:, :1])),
        lambda: ops.linear_fp8_block(x, (wq, s)),
        lambda: ops.linear_fp8_block((q, s), w.clone().requires_grad_()),
        lambda: ops.linear_fp8_block((q, s.clone().requires_grad_()), (wq, ws)),
        lambda: ops.fp8_block_dequantize(wq, ws.clone().requires_grad_()),
        lambda: ops.norm_linear_fp8_block(x, g, 1e-5, "te", w, b.float()),
        lambda: ops.norm_linear_fp8_block(x, g, 1e-5, "te", w[:, :100]),
        lambda: ops.norm_linear_fp8_block(x, g, 1e-5, "none", w),
        lambda: ops.norm_linear_fp8_block(x, g, 1e-5, "te", w, b, x[:1]),
    ]


@pytest.mark.parametrize("i", range(len(refusals("cpu"))))
def test_refusals(i):
    with pytest.raises(ValueError):
        refusals("cpu")[i]()


def test_no_second_derivative():
    x = _randn(4, 130).float().requires_grad_()
    y = ops.linear_fp8_block(x, _randn(6, 130).float())
    g, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_recipe_key():
    import os
    from savanna_b200.config import GlobalConfig
    tiny = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "configs", "baseline", "tiny_sh2_cpu.yml")
    cfg = GlobalConfig.from_ymls([tiny], {"global_num_gpus": 1, "fp8_recipe": "block128", "use_fp8_linears": True})
    assert cfg.fp8_recipe == "block128"
