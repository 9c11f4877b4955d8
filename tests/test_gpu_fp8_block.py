"""8-bit operands with a scale for each block of 128 on the GPU: quantisers, norm, product and gradients against the definition in 64 bits."""
import pytest
import torch

from savanna_b200 import ops
from savanna_b200.ops import reference as ref
from tests.fp8_block_oracle import blockwise, close_sum, half_step, tiles
from tests.test_fp8_block import refusals

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _randn(*shape, seed=0, dtype=torch.bfloat16, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def _whole(q, s):
    return ref.fp8_block_dequantize(q, s, torch.float64)


def _same_bits(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


# ------------------------------------------------------------------------------------------------ quantisers


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,C", [(1, 1), (3, 130), (257, 128), (5, 1000), (130, 4099), (1, 16384), (300, 264)])
def test_rows_have_the_statements_codes(R, C, dtype):
    x = _randn(R, C, dtype=dtype) * _randn(C, seed=1, dtype=dtype).exp()
    q, s = ops.fp8_block_quantize(x)
    want_q, want_s = ref.fp8_block_quantize(x)
    assert torch.equal(s, want_s)
    if dtype != torch.float32:           # a quotient of 16-bit values is never so near a border that its last bit matters
        assert _same_bits(q, want_q)
    else:
        assert (q.float() - want_q.float()).abs().max() <= 32 and (q.float() != want_q.float()).float().mean() < 1e-3
    for out in TYPES:
        assert torch.equal(ops.fp8_block_dequantize(q, s, out), ref.fp8_block_dequantize(q, s, out))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,K", [(1, 1), (128, 128), (130, 300), (7, 1000), (260, 4096)])
def test_tiles_have_the_statements_codes(N, K, dtype):
    w = _randn(N, K, dtype=dtype)
    q, s = ops.fp8_block_quantize_weight(w)
    want_q, want_s = ref.fp8_block_quantize_weight(w)
    assert torch.equal(s, want_s)
    if dtype != torch.float32:
        assert _same_bits(q, want_q)
    assert torch.equal(ops.fp8_block_dequantize(q, s, dtype), ref.fp8_block_dequantize(q, s, dtype))


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_offsets_and_leading_dimensions(dtype):
    base = _randn(6, 10, 700, dtype=dtype)
    for x in (base[:, :, 3:259], base.transpose(0, 1), base[::2, 1::3, 8:520], base[..., ::2], base[0, 0, :1].expand(5, 1), base[:1, 0].expand(9, 700)):
        q, s = ops.fp8_block_quantize(x)
        want_q, want_s = ref.fp8_block_quantize(x)
        assert q.shape == x.shape and torch.equal(s, want_s)
        assert _same_bits(q, want_q) or dtype == torch.float32


def test_blocks_that_are_zero_or_not_finite():
    x = torch.zeros(200, 300, device="cuda")
    x[1, 5], x[2, 200], x[150, 299] = float("inf"), float("nan"), -float("inf")
    back = ops.fp8_block_dequantize(*ops.fp8_block_quantize(x), torch.float32)
    want = ref.fp8_block_dequantize(*ref.fp8_block_quantize(x), torch.float32)
    assert torch.equal(back.isnan(), want.isnan()) and (back.nan_to_num() == 0).all()
    w = ops.fp8_block_dequantize(*ops.fp8_block_quantize_weight(x), torch.float32)
    assert w[:128, :256].isnan().all() and w[128:, 256:].isnan().all() and (w[128:, :256] == 0).all()


def test_huge_and_tiny_values():
    x = torch.tensor([[3e38, 1e38, -3.3e38, 1e36], [1e-37, 3e-38, 0.0, 1e-30]], device="cuda")
    q, s = ops.fp8_block_quantize(x)
    want_q, want_s = ref.fp8_block_quantize(x)
    assert torch.equal(s, want_s) and torch.equal(q.float(), want_q.float())


def test_empty():
    x = torch.empty(0, 130, device="cuda", dtype=torch.bfloat16)
    q, s = ops.fp8_block_quantize(x)
    assert q.shape == (0, 130) and s.shape == (0, 2) and ops.fp8_block_dequantize(q, s).shape == (0, 130)
    w = _randn(9, 130).requires_grad_()
    y = ops.linear_fp8_block(x.requires_grad_(), w)
    gx, gw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert y.shape == (0, 9) and gx.shape == x.shape and (gw == 0).all()


# ------------------------------------------------------------------------------------------------ norm


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("form", ["te", "classic"])
@pytest.mark.parametrize("T,D", [(1, 1), (3, 127), (9, 1000), (2, 1029), (130, 4096), (5, 16384), (4, 8200)])
def test_norm(T, D, form, dtype):
    x, r = _randn(T, D, dtype=dtype, std=3.0), _randn(T, D, seed=1, dtype=dtype)
    g = _randn(D, seed=2, dtype=dtype)
    for res in (r, None):
        q, s, kept = ops.rmsnorm_fp8_block(x, g, 1e-5, form, res)
        h = x if res is None else x + res
        assert torch.equal(kept, h) and q.shape == x.shape and s.shape == (T, -(-D // 128))
        ms = h.double().square().mean(-1, keepdim=True)
        y = h.double() / ((ms + 1e-5).sqrt() if form == "te" else ms.sqrt() + 1e-5) * g.double()
        amax = torch.stack([b.abs().amax(-1) for b in y.split(128, -1)], -1)
        # the row's sum of squares and root: below 2^-18 of it for 16384 values added by threads, warps and blocks
        assert ((s.double() * 448 - amax).abs() <= 2.0 ** -18 * amax + 2.0 ** -99).all()
        step = s.double().repeat_interleave(128, -1)[:, :D] * 2.0 ** -10
        assert ((_whole(q, s) - y).abs() <= (2.0 ** -4 + 2.0 ** -17) * y.abs() + step).all()


def test_norm_of_strided_rows_and_of_a_width_beyond_the_kernel():
    base = _randn(5, 3, 600)
    x, r, g = base[:, 1, 5:505], base[:, 2, :500], _randn(500, seed=3)
    q, s, kept = ops.rmsnorm_fp8_block(x, g, 1e-5, "te", r)
    q2, s2, kept2 = ops.rmsnorm_fp8_block(x.contiguous(), g, 1e-5, "te", r.contiguous())
    assert torch.equal(kept, kept2) and torch.equal(s, s2) and _same_bits(q, q2)
    wide, g = _randn(2, 20000), _randn(20000, seed=1)
    q, s, _ = ops.rmsnorm_fp8_block(wide, g, 1e-5)
    assert q.shape == wide.shape and s.shape == (2, 157)


# ------------------------------------------------------------------------------------------------ product


SIZES = [(1, 128, 128), (1, 4096, 264), (2, 129, 1), (7, 1000, 520), (16, 300, 130), (33, 4096, 1000), (64, 16, 8), (77, 127, 257), (128, 256, 256),
         (129, 520, 300), (300, 1, 260), (513, 1027, 650), (1333, 640, 4096), (3000, 256, 1000)]


@pytest.mark.parametrize("T,K,N", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
def test_product(T, K, N, dtype):
    x, w, b, r = (_randn(*s, seed=i, dtype=dtype) for i, s in enumerate([(T, K), (N, K), (N,), (T, N)]))
    xq, wq = ops.fp8_block_quantize(x), ops.fp8_block_quantize_weight(w)
    a, c = _whole(*xq), _whole(*wq)
    want, terms = a @ c.t(), a.abs() @ c.abs().t()
    with torch.no_grad():
        close_sum(ops.linear_fp8_block(x, wq), want, terms, dtype, "product")
        close_sum(ops.linear_fp8_block(xq, wq, dtype=dtype), want, terms, dtype, "product of codes")
        full = want + b.double() + r.double()
        close_sum(ops.linear_fp8_block(x, w, b, r), full, terms + b.double().abs() + r.double().abs(), dtype, "with bias and residual")


def test_product_of_operands_in_other_strides():
    x, w = _randn(40, 384), _randn(70, 384, seed=1)
    (q, s), (wq, ws) = ops.fp8_block_quantize(x), ops.fp8_block_quantize_weight(w)
    want = ops.linear_fp8_block((q, s), (wq, ws))
    odd = torch.empty(40, 391, dtype=torch.uint8, device="cuda")[:, 3:387]
    odd.copy_(q.view(torch.uint8))
    cols = ws.t().contiguous().t()
    assert torch.equal(ops.linear_fp8_block((odd.view(torch.float8_e4m3fn), s.contiguous()), (wq, cols)), want)
    q3, s3 = ops.fp8_block_quantize(x.view(2, 20, 384))
    r = _randn(2, 20, 80, seed=2)[..., 3:73]
    assert torch.equal(ops.linear_fp8_block((q3, s3), (wq, ws), None, r), (want.view(2, 20, 70).float() * 0 + ops.linear_fp8_block((q, s), (wq, ws), None, r.reshape(40, 70)).view(2, 20, 70).float()).to(want.dtype))


def test_scales_that_are_not_finite_show_in_their_rows_and_columns_alone():
    x, w = _randn(200, 256), _randn(300, 256, seed=1)
    x[3, 7], w[140, 9] = float("inf"), float("nan")
    y = ops.linear_fp8_block(x, w)
    bad = torch.zeros(200, 300, dtype=torch.bool, device="cuda")
    bad[3], bad[:, 128:256] = True, True
    assert torch.equal(y.isfinite(), ~bad)


# ------------------------------------------------------------------------------------------------ gradients


@pytest.mark.parametrize("T,K,N", [(1, 128, 64), (5, 130, 7), (77, 1000, 520), (300, 257, 129), (777, 1027, 650), (2000, 768, 2304)])
@pytest.mark.parametrize("dtype", TYPES)
def test_gradients(T, K, N, dtype):
    x, w, b, r, gy = (_randn(*s, seed=i, dtype=dtype) for i, s in enumerate([(T, K), (N, K), (N,), (T, N), (T, N)]))
    leaves = [t.requires_grad_() for t in (x, w, b, r)]
    y = ops.linear_fp8_block(x, w, b, r)
    gx, gw, gb, gr = torch.autograd.grad(y, leaves, gy)
    with torch.no_grad():
        wq = _whole(*ops.fp8_block_quantize_weight(w))
        grow = _whole(*ops.fp8_block_quantize(gy))
        gcol, xcol = (_whole(*ref.fp8_block_quantize(t.t().contiguous())).t() for t in (gy, x))
        close_sum(gx, grow @ wq, grow.abs() @ wq.abs(), dtype, "dx")
        terms = gcol.abs().t() @ xcol.abs()
        if dtype == torch.float32:       # some codes beside a border fall on the other side than the statement's
            assert (gw.double() - gcol.t() @ xcol).norm() <= 1e-3 * (gcol.t() @ xcol).norm()
        else:
            close_sum(gw, gcol.t() @ xcol, terms, dtype, "dw")
        close_sum(gb, gy.double().sum(0), gy.double().abs().sum(0), dtype, "db")
        assert torch.equal(gr, gy)


@pytest.mark.parametrize("T,K,N", [(1, 128, 64), (77, 1000, 520), (2000, 768, 2304), (300, 4096, 129)])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("form", ["te", "classic"])
def test_gradients_through_the_norm(T, K, N, residual, form):
    x, r, g, w, b, gy, gs = (_randn(*s, seed=i) for i, s in enumerate([(T, K), (T, K), (K,), (N, K), (N,), (T, N), (T, K)]))
    r = r if residual else None
    leaves = [t.requires_grad_() for t in (x, r, g, w, b) if t is not None]
    y, s = ops.norm_linear_fp8_block(x, g, 1e-5, form, w, b, r)
    got = dict(zip([n for n in ("x", "r", "g", "w", "b") if n != "r" or residual], torch.autograd.grad((y, s), leaves, (gy, gs))))
    h = (x if r is None else x + r).detach()
    assert torch.equal(s, h)
    hd, gain = h.double().requires_grad_(), g.detach().double().requires_grad_()
    ms = hd.square().mean(-1, keepdim=True)
    n = hd / ((ms + 1e-5).sqrt() if form == "te" else ms.sqrt() + 1e-5) * gain
    wq = tiles(w.detach().double())
    want_y = blockwise(n.detach(), 1) @ wq.t() + b.detach().double()
    dn = blockwise(gy.double(), 1) @ wq
    wx, wg = torch.autograd.grad((n, hd), (hd, gain), (dn, gs.double()))
    ww = blockwise(gy.double(), 0).t() @ blockwise(n.detach(), 0)
    # one rounding to bf16 each, one more of the norm's output gradient; a few values beside a border have the neighbouring code
    for name, a, e, tol in (("y", y, want_y, 2.0), ("dx", got["x"], wx, 3.0), ("dg", got["g"], wg, 4.0), ("dw", got["w"], ww, 2.0),
                            ("db", got["b"], gy.double().sum(0), 2.0)):
        assert (a.detach().double() - e).norm() <= tol * half_step(torch.bfloat16) * e.norm(), name
    if residual:
        assert torch.equal(got["x"], got["r"])


def test_norms_of_other_types_and_widths():
    for dtype, K in ((torch.float16, 256), (torch.bfloat16, 131), (torch.float32, 512), (torch.float32, 1), (torch.bfloat16, 20000)):
        x, g, w = _randn(20, K, dtype=dtype).requires_grad_(), _randn(K, seed=1, dtype=dtype).requires_grad_(), _randn(48, K, seed=2, dtype=dtype).requires_grad_()
        y, s = ops.norm_linear_fp8_block(x, g, 1e-5, "te", w)
        assert y.dtype == dtype and torch.equal(s, x)
        gx, gg, gw = torch.autograd.grad(y, (x, g, w), torch.ones_like(y))
        h, gain = x.detach().double().requires_grad_(), g.detach().double().requires_grad_()
        n = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-5) * gain
        wx, wg = torch.autograd.grad(n, (h, gain), blockwise(torch.ones_like(y).double(), 1) @ tiles(w.detach().double()))
        for a, e in ((gx, wx), (gg, wg), (gw, blockwise(torch.ones_like(y).double(), 0).t() @ blockwise(n.detach(), 0))):
            assert (a.double() - e).norm() <= (2 * half_step(dtype) + 1e-3) * e.norm()


def test_gradients_of_some_inputs_and_through_a_kept_weight():
    x, w, b = _randn(50, 200).requires_grad_(), _randn(70, 200, seed=1).requires_grad_(), _randn(70, seed=2).requires_grad_()
    gy = _randn(50, 70, seed=3)
    all_ = torch.autograd.grad(ops.linear_fp8_block(x, w, b), (x, w, b), gy)
    for i, t in enumerate((x, w, b)):
        assert torch.equal(torch.autograd.grad(ops.linear_fp8_block(x, w, b), t, gy)[0], all_[i])
    assert torch.equal(torch.autograd.grad(ops.linear_fp8_block(x, ops.fp8_block_quantize_weight(w), b), x, gy)[0], all_[0])
    # output gradients in other strides: a transposed one, a broadcast one
    assert torch.equal(torch.autograd.grad(ops.linear_fp8_block(x, w, b), x, gy.t().contiguous().t())[0], all_[0])
    one = torch.ones((), device="cuda", dtype=torch.bfloat16).expand(50, 70)
    assert torch.equal(torch.autograd.grad(ops.linear_fp8_block(x, w, b), w, one)[0], torch.autograd.grad(ops.linear_fp8_block(x, w, b), w, one.contiguous())[0])


def test_saved_tensors_through_hooks_that_change_strides():
    x, w = _randn(130, 200).requires_grad_(), _randn(70, 200, seed=1).requires_grad_()
    gy = _randn(130, 70, seed=3)
    want = torch.autograd.grad(ops.linear_fp8_block(x, w), (x, w), gy)

    def pack(t):
        u = t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t
        return t.dtype, u.cpu().t().contiguous()

    def unpack(p):
        u = p[1].cuda().t()
        return u.view(p[0]) if p[0] == torch.float8_e4m3fn else u
    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        y = ops.linear_fp8_block(x, w)
    for a, b in zip(torch.autograd.grad(y, (x, w), gy), want):
        assert torch.equal(a, b)


def test_second_derivative_is_refused():
    x = _randn(4, 130).requires_grad_()
    y = ops.linear_fp8_block(x, _randn(6, 130))
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(y.sum(), x, create_graph=True)


# ------------------------------------------------------------------------------------------------ where and when


def test_captured_and_replayed():
    x, r, g, w = _randn(40, 512), _randn(40, 512, seed=1), _randn(512, seed=2), _randn(300, 512, seed=3)
    kept = ops.fp8_block_quantize_weight(w)
    with torch.no_grad():
        ops.norm_linear_fp8_block(x, g, 1e-5, "te", kept, None, r)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, s = ops.norm_linear_fp8_block(x, g, 1e-5, "te", kept, None, r)
            z = ops.linear_fp8_block(s, w=w.t().contiguous().t()[:, :512])
        for seed in (5, 6):
            x.copy_(_randn(40, 512, seed=seed))
            graph.replay()
            want_y, want_s = ops.norm_linear_fp8_block(x, g, 1e-5, "te", kept, None, r)
            assert torch.equal(y, want_y) and torch.equal(s, want_s) and torch.equal(z, ops.linear_fp8_block(want_s, w))


def test_training_step_captured_and_replayed():
    x, w, gy = _randn(200, 256).requires_grad_(), _randn(300, 256, seed=1).requires_grad_(), _randn(200, 300, seed=2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(ops.linear_fp8_block(x, w), (x, w), gy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(ops.linear_fp8_block(x, w), (x, w), gy)
    with torch.no_grad():
        gy.copy_(_randn(200, 300, seed=7))
    graph.replay()
    for a, b in zip(got, torch.autograd.grad(ops.linear_fp8_block(x, w), (x, w), gy)):
        assert torch.equal(a, b)


def test_two_streams_at_once():
    xs = [_randn(100, 1024, seed=i) for i in range(2)]
    w = ops.fp8_block_quantize_weight(_randn(2000, 1024, seed=9))
    want = [ops.linear_fp8_block(x, w) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(ops.linear_fp8_block(xs[i], w))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in range(2) for y in got[i])


@pytest.mark.parametrize("T,K,N", [(1, 128, 130), (5, 1000, 129), (130, 300, 257), (300, 520, 300)])
def test_nothing_is_written_outside_of_the_outputs(T, K, N):
    from savanna_b200.ops import cuda_ops
    with cuda_ops.guarded_allocations():
        for dtype in TYPES:
            x, w, b = _randn(T, K, dtype=dtype).requires_grad_(), _randn(N, K, seed=1, dtype=dtype).requires_grad_(), _randn(N, seed=2, dtype=dtype).requires_grad_()
            y = ops.linear_fp8_block(x, w, b)
            torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
            q, s, _ = ops.rmsnorm_fp8_block(x.detach(), w[0].detach(), 1e-5, "te", x.detach())
            ops.fp8_block_dequantize(q, s, dtype)
        assert cuda_ops.check_guards() > 0
    cuda_ops.check_status()


@pytest.mark.parametrize("i", range(len(refusals("cpu"))))
def test_refusals(i):
    with pytest.raises(ValueError):
        refusals("cuda")[i]()


# ------------------------------------------------------------------------------------------------ as models use them


@pytest.fixture
def recipe():
    from savanna_b200.ops import cuda_ops
    cuda_ops.set_fp8_recipe("block128")
    yield cuda_ops
    cuda_ops.set_fp8_recipe("delayed")


def test_norm_projection_gate_projection_in_a_row(recipe):
    """A gated MLP by the operators one after the other, and by the model's entry point under the recipe: the same bits."""
    T, D, F = 70, 256, 384
    x, g, w12, w3, b = (_randn(*s, seed=i, std=v) for i, (s, v) in enumerate([((2, T // 2, D), 1.0), ((D,), 0.1), ((2 * F, D), 0.05), ((D, F), 0.05), ((D,), 0.1)]))
    leaves = [t.requires_grad_() for t in (x, g, w12, w3, b)]
    gy = _randn(2, T // 2, D, seed=9)
    y = ops.mlp_gated(x, g, 1e-5, "te", w12, w3, b, "silu", fp8=True)
    got = torch.autograd.grad(y, leaves, gy)
    ab, s = ops.norm_linear_fp8_block(x, g, 1e-5, "te", w12)
    z = ops.linear_fp8_block(ops.glu_act_packed(ab, "silu"), w3, b, s)
    assert torch.equal(y, z)
    for a, e in zip(got, torch.autograd.grad(z, leaves, gy)):
        assert torch.equal(a, e)


def test_recipe_sees_changed_weights(recipe):
    x, w = _randn(20, 256), torch.nn.Parameter(_randn(64, 256, seed=1))
    with torch.no_grad():
        a = ops.linear(x, w, fp8=True)
        w.mul_(2.0)
        assert torch.equal(ops.linear(x, w, fp8=True).float(), 2.0 * a.float())
        w.data.view(torch.int16).bitwise_xor_(-0x8000)            # the sign bits, past PyTorch's version counter, as a fused step writes
        recipe.bump_param_epoch()
        assert torch.equal(ops.linear(x, w, fp8=True).float(), -2.0 * a.float())


def test_weight_gradient_added_in_place(recipe):
    for T, K, N in ((77, 256, 264), (1000, 520, 300), (300, 129, 65)):
        x, w, gy = _randn(T, K), torch.nn.Parameter(_randn(N, K, seed=1)), _randn(T, N, seed=2)
        fresh, = torch.autograd.grad(ops.linear_fp8_block(x, w), w, gy)
        w._fuse_grad_accum = True
        start = _randn(N, K, seed=3)
        w.grad = start.clone()
        ops.linear(x, w, fp8=True).backward(gy)
        gcol, xcol = (_whole(*ref.fp8_block_quantize(t.t().contiguous())).t() for t in (gy, x))
        want = start.double() + gcol.t() @ xcol
        close_sum(w.grad, want, gcol.abs().t() @ xcol.abs() + start.double().abs(), torch.bfloat16, "accumulated")
        assert not torch.equal(w.grad, fresh)


def test_training_under_the_recipe_tracks_bf16(recipe):
    import os
    from savanna_b200.config import GlobalConfig
    from savanna_b200.data.synthetic import acgt_batch
    from savanna_b200.parallel import state
    from savanna_b200.train.trainer import Trainer
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    over = {"global_num_gpus": 1, "use_fp8_linears": True, "use_fp8_input_projections": True, "use_fp8_output_projections": True, "use_fp8_mlp_projections": True,
            "fp8_recipe": "block128"}
    cfg = GlobalConfig.from_ymls([os.path.join(root, "configs", "baseline", "tiny_sh2_gpu.yml")], over)
    tr = Trainer(cfg, load=False)
    batches = iter([{"text": acgt_batch(cfg.train_micro_batch_size_per_gpu, cfg.seq_length, seed=i).cuda()} for i in range(3)])
    before = recipe.launch_count()
    losses = [float(tr.train_step(batches)) for _ in range(3)]
    state.destroy_model_parallel()
    assert all(torch.isfinite(torch.tensor(losses))) and recipe.launch_count() > before
    recipe.check_status()
    assert any(getattr(p, "_fp8_block_cache", None) is not None for p in tr.model.parameters())


def test_recipe_in_a_captured_graph_leaves_no_codes_behind(recipe):
    x, w = _randn(20, 256), torch.nn.Parameter(_randn(64, 256, seed=1))
    with torch.no_grad():
        ops.linear(x, torch.nn.Parameter(_randn(64, 256, seed=5)), fp8=True)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = ops.linear(x, w, fp8=True)
        eager = ops.linear(x, w, fp8=True).clone()                # before any replay
        graph.replay()
        assert torch.equal(y, eager)
        w.mul_(2.0)
        graph.replay()
        assert torch.equal(y.float(), 2.0 * eager.float())


def test_recipe_on_two_streams(recipe):
    x, w = _randn(20, 256), torch.nn.Parameter(_randn(64, 256, seed=1))
    with torch.no_grad():
        want = ops.linear_fp8_block(x, w)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        got = [ops.linear(x, w, fp8=True)]
        with torch.cuda.stream(side):
            got.append(ops.linear(x, w, fp8=True))
        torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


# ------------------------------------------------------------------------------------------------ sizes


def test_more_than_two_to_the_31_values():
    """The last rows of tensors whose offsets pass 32 bits are those of the same rows by themselves."""
    T, D, N = 270001, 8192, 128
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("wants 40 GB")
    g = _randn(D, seed=1)
    x = torch.empty(T, D, device="cuda", dtype=torch.bfloat16)
    x[-1000:] = _randn(1000, D)
    x[:-1000] = 1.0
    tail = x[-300:].clone()
    q, s, kept = ops.rmsnorm_fp8_block(x, g, 1e-5, "te", x)
    q1, s1, kept1 = ops.rmsnorm_fp8_block(tail, g, 1e-5, "te", tail)
    assert _same_bits(q[-300:], q1) and torch.equal(s[-300:], s1) and torch.equal(kept[-300:], kept1)
    del kept
    assert torch.equal(ops.fp8_block_dequantize(q, s)[-300:], ops.fp8_block_dequantize(q1, s1))
    w = ops.fp8_block_quantize_weight(_randn(N, D, seed=2))
    with torch.no_grad():
        assert torch.equal(ops.linear_fp8_block((q, s), w)[-200:], ops.linear_fp8_block((q1[100:], s1[100:]), w))
    del q, s
    q, s = ops.fp8_block_quantize(x)
    q1, s1 = ops.fp8_block_quantize(tail)
    assert _same_bits(q[-300:], q1) and torch.equal(s[-300:], s1)
    del q, s
    # a wide result, its input gradient and the weight gradient over all tokens
    h = torch.zeros(T, 128, device="cuda", dtype=torch.bfloat16)
    h[-200:] = _randn(200, 128, seed=3)
    h.requires_grad_()
    w = _randn(D, 128, seed=4).requires_grad_()
    gy = x
    y = ops.linear_fp8_block(h, w)
    short = h[-200:].detach().requires_grad_()
    y1 = ops.linear_fp8_block(short, w)
    assert torch.equal(y[-200:], y1)
    gh, gw = torch.autograd.grad(y, (h, w), gy)
    assert torch.equal(gh[-200:], torch.autograd.grad(y1, short, gy[-200:].contiguous())[0])
    # columns of the last tokens alone: the others' activations are zero, and blocks of tokens begin where T - 200 is no multiple of 128
    n0 = (T - 200) // 128 * 128
    gcol, xcol = (_whole(*ref.fp8_block_quantize(t[n0:].detach().t().contiguous())).t() for t in (gy, h))
    close_sum(gw, gcol.t() @ xcol, gcol.abs().t() @ xcol.abs(), torch.bfloat16, "dw")
