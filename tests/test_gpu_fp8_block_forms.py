"""Every form of the block-scaled products where its rings wrap and its tiles end inside: which form a size runs by is asserted beside its values."""
import pytest
import torch

from savanna_b200 import ops
from savanna_b200.ops import cuda_ops, reference as ref
from tests.fp8_block_oracle import blockwise, close_sum, half_step, tiles

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _randn(*shape, seed=0, dtype=torch.bfloat16, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def _whole(q, s):
    return ref.fp8_block_dequantize(q, s, torch.float64)


def _takes_few(T, N):
    return bool(cuda_ops.require().sb_gemm_fp8_block_takes_few(T, N))


def _by_pairs(M, N):
    return bool(cuda_ops.require().sb_gemm_fp8_block_goes_by_pairs(M, N))


def test_wide_products_of_more_than_31_tokens_go_by_tiles():
    """Where the tiles' kernel was the faster one."""
    assert not any(_takes_few(T, 12288) for T in (32, 33, 64))
    assert all(_takes_few(T, 12288) for T in (1, 16, 17, 31)) and all(_takes_few(T, 8192) for T in (1, 32, 64))


def test_weight_gradients_have_a_rule_of_their_own():
    """128 x 128 tiles where they take half as many waves again: [2304, 2304] of 8192 tokens 81 us, by pairs 91."""
    pairs = cuda_ops.require().sb_gemm_fp8_block_weight_goes_by_pairs
    assert not any(pairs(*s) for s in ((2304, 2304), (1333, 4096), (3712, 3712), (4480, 4224), (1024, 1024)))
    assert all(pairs(*s) for s in ((2048, 2048), (4096, 4096), (12288, 4096), (1096, 2104)))
    assert all(_by_pairs(*s) for s in ((3712, 3712), (4480, 4224), (4096, 4096))) and not _by_pairs(512, 4096)


# k-blocks of a CTA: fewer than its stages, more, more than twice as many, more than its accumulators and than a group of 16 scales, more than two groups
FEW = [(T, K, N, kbs) for T in (1, 16, 17, 32, 33, 64) for K, N, kbs in ((2900, 130, 3), (6100, 130, 6), (10200, 261, 10), (17300, 100, 17), (33700, 130, 33))]
FEW += [(3, 4100, 19000, 33), (31, 2100, 18990, 17), (64, 4100, 5000, 9)]


@pytest.mark.parametrize("T,K,N,kbs", FEW)
@pytest.mark.parametrize("dtype", TYPES)
def test_few_tokens(T, K, N, kbs, dtype):
    parts = cuda_ops.require().sb_gemm_fp8_block_few_parts(N, K)
    assert _takes_few(T, N) and -(-(-(-K // 128)) // parts) == kbs
    x, w, b, r = (_randn(*s, seed=i, dtype=dtype) for i, s in enumerate([(T, K), (N, K), (N,), (T, N)]))
    xq, wq = ops.fp8_block_quantize(x), ops.fp8_block_quantize_weight(w)
    a, c = _whole(*xq), _whole(*wq)
    want, terms = a @ c.t(), a.abs() @ c.abs().t()
    with torch.no_grad():
        y = ops.linear_fp8_block(x, wq)                           # behind the quantiser, weights read ahead
        close_sum(y, want, terms, dtype, "product")
        assert torch.equal(ops.linear_fp8_block(xq, wq, dtype=dtype), y)
        full = want + b.double() + r.double()
        close_sum(ops.linear_fp8_block(x, wq, b, r), full, terms + b.double().abs() + r.double().abs(), dtype, "with bias and residual")
    cuda_ops.check_status()


@pytest.mark.parametrize("T,K,N", [(1104, 2104, 1096), (1090, 2103, 1101), (2300, 640, 1800)])
@pytest.mark.parametrize("dtype", TYPES)
def test_gradients_by_pairs(T, K, N, dtype):
    """Input gradient [T, K] or weight gradient [N, K] (or both) by 256 x 256 tiles that end inside, fresh and added in place."""
    assert _by_pairs(T, K) or _by_pairs(N, K) or _by_pairs(T, N)
    if T < 2000:
        assert _by_pairs(T, K) and cuda_ops.require().sb_gemm_fp8_block_weight_goes_by_pairs(N, K)
    x, b, gy = (_randn(*s, seed=i, dtype=dtype) for i, s in ((0, (T, K)), (2, (N,)), (4, (T, N))))
    w = torch.nn.Parameter(_randn(N, K, seed=1, dtype=dtype))
    x.requires_grad_(), b.requires_grad_()
    y = ops.linear_fp8_block(x, w, b)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), gy)
    with torch.no_grad():
        wq, rows, grow = (_whole(*q) for q in (ops.fp8_block_quantize_weight(w), ops.fp8_block_quantize(x), ops.fp8_block_quantize(gy)))
        close_sum(y, rows @ wq.t() + b.double(), rows.abs() @ wq.abs().t() + b.double().abs(), dtype, "y")
        close_sum(gx, grow @ wq, grow.abs() @ wq.abs(), dtype, "dx")
        close_sum(gb, gy.double().sum(0), gy.double().abs().sum(0), dtype, "db")
        gcol, xcol = (_whole(*ref.fp8_block_quantize(t.detach().t().contiguous())).t() for t in (gy, x))
        want, terms = gcol.t() @ xcol, gcol.abs().t() @ xcol.abs()
        start = _randn(N, K, seed=7, dtype=dtype)
        w._fuse_grad_accum, w.grad = True, start.clone()
    ops.linear_fp8_block(x, w, b).backward(gy)
    total = want + start.double()
    if dtype == torch.float32:           # some codes beside a border fall on the other side than the statement's
        assert (gw.double() - want).norm() <= 1e-3 * want.norm() and (w.grad.double() - total).norm() <= 1e-3 * total.norm()
    else:
        close_sum(gw, want, terms, dtype, "dw")
        close_sum(w.grad, total, terms + start.double().abs(), dtype, "dw in place")
    cuda_ops.check_status()


@pytest.mark.parametrize("T,K,N", [(1104, 2104, 1096), (1090, 2103, 1101)])
def test_pairs_write_nothing_outside(T, K, N):
    with cuda_ops.guarded_allocations():
        for dtype in TYPES:
            x, w = _randn(T, K, dtype=dtype).requires_grad_(), _randn(N, K, seed=1, dtype=dtype).requires_grad_()
            y = ops.linear_fp8_block(x, w)
            torch.autograd.grad(y, (x, w), torch.ones_like(y))
        assert cuda_ops.check_guards() > 0
    cuda_ops.check_status()


@pytest.mark.parametrize("form", ["te", "classic"])
def test_norm_and_projection_of_rows_beyond_the_norms_kernel(form):
    x, g, w = _randn(20, 20000), _randn(20000, seed=1), _randn(48, 20000, seed=2)
    y, s = ops.norm_linear_fp8_block(x, g, 1e-5, form, w)
    ms = x.double().square().mean(-1, keepdim=True)
    n = x.double() / ((ms + 1e-5).sqrt() if form == "te" else ms.sqrt() + 1e-5) * g.double()
    want = blockwise(n, 1) @ tiles(w.double()).t()
    assert torch.equal(s, x)
    # the result's rounding, and a few values beside a border that have the neighbouring code
    assert (y.double() - want).norm() <= (2 * half_step(torch.bfloat16) + 1e-3) * want.norm()


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("shape", [(0, 130), (2, 0, 256)])
def test_norms_of_no_rows(shape, residual):
    D = shape[-1]
    x, g, w, b = torch.empty(shape, device="cuda", dtype=torch.bfloat16), _randn(D), _randn(9, D, seed=1), _randn(9, seed=2)
    r = torch.empty_like(x) if residual else None
    q, s, kept = ops.rmsnorm_fp8_block(x, g, 1e-5, "te", r)
    assert q.shape == kept.shape == x.shape and s.shape == shape[:-1] + (-(-D // 128),)
    leaves = [t.requires_grad_() for t in (x, r, g, w, b) if t is not None]
    y, s = ops.norm_linear_fp8_block(x, g, 1e-5, "te", w, b, r)
    assert y.shape == shape[:-1] + (9,) and s.shape == x.shape
    grads = torch.autograd.grad((y, s), leaves, (torch.empty_like(y), torch.empty_like(s)))
    assert all(a.shape == t.shape and (a == 0).all() for a, t in zip(grads, leaves))
