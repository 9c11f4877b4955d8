"""Performance cases of projections on 8-bit operands with a scale for each block of 128, and of the norm that writes such operands.

A case is a plain dict.  `kind` selects the operator:

  norm         RMS norm of x + residual into e4m3 with a scale for 128 values of a row, and the way back   ops.rmsnorm_fp8_block, ops.fp8_block_dequantize
  linear       projection: with a weight kept in 8 bits (serving), or forward + backward with one that training changes     ops.linear_fp8_block
  norm_linear  projection of the norm of x + residual, serving or forward + backward                        ops.norm_linear_fp8_block

Activations and output gradients are quantised by 1 x 128 values along the contraction of their product, weights by 128 x 128 tiles.
`run` computes the plain form in elementary 32-bit operations where `own` is false, and calls the framework where it is true.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 128                 # values that share a scale
TOP = 448.0                 # largest e4m3 value
TINY = 2.0 ** -100          # least magnitude that a scale is made for
EPS = 1e-5


def listed():
    return [
        # one decode step of eight sequences
        dict(name="norm_step", kind="norm", T=8, D=4096, dtype="bf16"),
        # the residual stream of the 7B model, one sequence of training
        dict(name="norm_8k", kind="norm", T=8192, D=4096, dtype="bf16"),
        # a fp16 run of a small model: a width that ends inside a block, a ragged batch
        dict(name="norm_odd", kind="norm", T=999, D=1000, dtype="fp16"),
        # decoding one sequence: the input projection of the 7B model
        dict(name="linear_step", kind="linear", T=1, K=4096, N=12288, dtype="bf16", bias=False, train=False),
        # decoding sixteen: the MLP's output projection
        dict(name="linear_step_batch", kind="linear", T=16, K=11264, N=4096, dtype="bf16", bias=False, train=False),
        # a prompt of an odd length through the output projection
        dict(name="linear_prefill", kind="linear", T=1333, K=4096, N=4096, dtype="bf16", bias=True, train=False),
        # a small fp16 model whose sizes end inside blocks
        dict(name="linear_odd", kind="linear", T=77, K=1000, N=520, dtype="fp16", bias=True, train=False),
        # the input projection of the 7B model in training, one 8192-token sequence
        dict(name="linear_train_8k", kind="linear", T=8192, K=4096, N=12288, dtype="bf16", bias=False, train=True),
        # fine-tuning a small model on a ragged batch, odd sizes in every direction
        dict(name="linear_train_odd", kind="linear", T=777, K=1027, N=650, dtype="bf16", bias=True, train=True),
        # norm, residual and projection of a 4096-wide block in training
        dict(name="norm_linear_train_8k", kind="norm_linear", T=8192, K=4096, N=4096, dtype="bf16", bias=False, train=True),
        # the same in a narrow model
        dict(name="norm_linear_train_small", kind="norm_linear", T=2000, K=768, N=2304, dtype="bf16", bias=True, train=True),
        # decoding four sequences through norm and input projection
        dict(name="norm_linear_step", kind="norm_linear", T=4, K=4096, N=12288, dtype="bf16", bias=False, train=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi, step):
    """A width of lo .. hi: half of them multiples of 128, as those of most models, the others of `step`."""
    d = _log(rng, lo, hi)
    step = rng.choice([step, 128])
    return max(step, d // step * step)


def draw(rng):
    kind = rng.choice(["norm", "linear", "linear", "linear", "norm_linear", "norm_linear"])
    if kind == "norm":
        D = _width(rng, 64, 16384, 1)
        return dict(kind=kind, T=_log(rng, 1, max(1, min(65536, 8192 * 4096 // D))), D=D, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    train = rng.random() < 0.5
    # a norm's backward pass goes by rows of eights
    K = _width(rng, 128, 16384, 8 if kind == "norm_linear" else 1)
    N = _width(rng, 128, 16384, 1)
    most = 8192 * 4096 * (12288 if kind == "linear" else 4096)
    while K * N * 16 > most:
        N = max(128, N // 2)
    T = _log(rng, 1, max(1, min(16384, most // (K * N))))
    if not train and rng.random() < 0.5:
        T = _log(rng, 1, 64)
    dtype = "bf16" if kind == "norm_linear" else rng.choice(["bf16", "bf16", "fp16"])
    return dict(kind=kind, T=T, K=K, N=N, dtype=dtype, bias=rng.random() < 0.3, train=train)


# ------------------------------------------------------------------------------------------------ inputs


def _randn(g, *shape, std=1.0, mean=0.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=g, device=DEV) * std + mean).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 31)
    c = dict(case)
    dt, T, D = TYPES[c["dtype"]], c["T"], c.get("D") or c.get("K")
    # the residual stream: channels of unequal size, a few of them large
    size = torch.exp(0.5 * torch.randn(D, generator=g, device=DEV)) * torch.where(torch.rand(D, generator=g, device=DEV) < 0.01, 20.0, 1.0)
    st = dict(case=c, x=(torch.randn(T, D, generator=g, device=DEV) * size).to(dt))
    if c["kind"] != "linear":
        st["res"] = (torch.randn(T, D, generator=g, device=DEV) * size).to(dt)
        st["g"] = _randn(g, D, std=0.1, mean=1.0, dtype=dt)
    if c["kind"] == "norm":
        return st
    N = c["N"]
    w = _randn(g, N, D, std=1.0 / math.sqrt(D), dtype=dt)
    st["b"] = _randn(g, N, std=0.1, dtype=dt) if c["bias"] else None
    if c["train"]:
        st["w"] = w
        st["gy"] = _randn(g, T, N, dtype=dt)
        if c["kind"] == "norm_linear":
            st["gs"] = _randn(g, T, D, dtype=dt)
        for n in ("x", "res", "g", "w", "b"):
            if st.get(n) is not None:
                st[n].requires_grad_(True)
    else:
        st["w"] = _tiles(w)          # the weight as a server loads it: e4m3 and one scale a tile
    return st


# ------------------------------------------------------------------------------------------------ one pass


def _run_own(st):
    from savanna_b200 import ops
    c = st["case"]
    if c["kind"] == "norm":
        with torch.no_grad():
            q, scale, s = ops.rmsnorm_fp8_block(st["x"], st["g"], EPS, "te", st["res"])
            return dict(y=ops.fp8_block_dequantize(q, scale, st["x"].dtype), s=s)
    if not c["train"]:
        with torch.no_grad():
            if c["kind"] == "linear":
                return ops.linear_fp8_block(st["x"], st["w"], st["b"])
            y, s = ops.norm_linear_fp8_block(st["x"], st["g"], EPS, "te", st["w"], st["b"], st["res"])
            return dict(y=y, s=s)
    names = [n for n in ("x", "res", "g", "w", "b") if st.get(n) is not None]
    leaves = [st[n] for n in names]
    if c["kind"] == "linear":
        y = ops.linear_fp8_block(st["x"], st["w"], st["b"])
        return dict(zip(["y"] + ["d" + n for n in names], (y,) + torch.autograd.grad(y, leaves, st["gy"])))
    y, s = ops.norm_linear_fp8_block(st["x"], st["g"], EPS, "te", st["w"], st["b"], st["res"])
    return dict(zip(["y", "s"] + ["d" + n for n in names], (y, s) + torch.autograd.grad((y, s), leaves, (st["gy"], st["gs"]))))


def _code(v, amax):
    """(e4m3 values of v with its scale, the scale).  The quotient is formed so that one halfway between two codes is met exactly."""
    amax = amax.clamp(min=TINY)
    return (v * TOP / amax).clamp(-TOP, TOP).to(torch.float8_e4m3fn), amax * (1.0 / TOP)


def _rows(x):
    """x [R, C] fp32 as its 8-bit form stands for it: a scale for 128 values of a row."""
    R, C = x.shape
    n = -(-C // BLOCK)
    v = torch.nn.functional.pad(x, (0, n * BLOCK - C)).view(R, n, BLOCK)
    q, scale = _code(v, v.abs().amax(-1, keepdim=True))
    return (q.float() * scale).view(R, n * BLOCK)[:, :C]


def _cols(x):
    return _rows(x.t()).t()


def _tiles(w):
    """w [N, K] -> (e4m3 [N, K], scale [N / 128, K / 128])."""
    N, K = w.shape
    n, k = -(-N // BLOCK), -(-K // BLOCK)
    v = torch.nn.functional.pad(w.float(), (0, k * BLOCK - K, 0, n * BLOCK - N)).view(n, BLOCK, k, BLOCK)
    q, scale = _code(v, v.abs().amax((1, 3), keepdim=True))
    return q.view(n * BLOCK, k * BLOCK)[:N, :K].contiguous(), scale.view(n, k)


def _whole(q, scale):
    N, K = q.shape
    return q.float() * scale.repeat_interleave(BLOCK, 0)[:N].repeat_interleave(BLOCK, 1)[:, :K]


def _plain_norm(st):
    s = (st["x"].detach().float() + st["res"].detach().float()).to(st["x"].dtype)
    sf = s.float()
    r = 1.0 / torch.sqrt((sf * sf).mean(-1, keepdim=True) + EPS)
    return s, sf * r * st["g"].detach().float(), r


def _plain(st):
    c, dt = st["case"], st["x"].dtype
    if c["kind"] == "norm":
        s, y, _ = _plain_norm(st)
        return dict(y=_rows(y).to(dt), s=s)
    norm = c["kind"] == "norm_linear"
    if norm:
        s, a, r = _plain_norm(st)
    else:
        a = st["x"].detach().float()
    w = _whole(*(_tiles(st["w"].detach()) if c["train"] else st["w"]))
    y = _rows(a) @ w.t()
    if st["b"] is not None:
        y = y + st["b"].detach().float()
    out = dict(y=y.to(dt))
    if norm:
        out["s"] = s
    if not c["train"]:
        return out if norm else out["y"]
    gy = st["gy"].float()
    da = _rows(gy) @ w
    out["dw"] = (_cols(gy).t() @ _cols(a)).to(dt)
    if st["b"] is not None:
        out["db"] = gy.sum(0).to(dt)
    if not norm:
        out["dx"] = da.to(dt)
        return out
    xh = s.float() * r
    out["dg"] = (da * xh).sum(0).to(dt)
    t = da * st["g"].detach().float()
    out["dx"] = (r * (t - xh * (t * xh).mean(-1, keepdim=True)) + st["gs"].float()).to(dt)
    out["dres"] = out["dx"]
    return out


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _plain(state)


# ------------------------------------------------------------------------------------------------ work, and the definition in 64 bits


def work(case):
    c = case
    T, size = c["T"], 4 if c["dtype"] == "fp32" else 2
    if c["kind"] == "norm":
        D = c["D"]
        # x and the residual in, their sum and the 8-bit form out; that form in again, its values out
        return dict(bytes=T * D * (4 * size + 2) + size * D + 8 * T * -(-D // BLOCK), flops=T * D * 10)
    K, N = c["K"], c["N"]
    norm = c["kind"] == "norm_linear"
    streams = T * K * size * (3 if norm else 1) + T * N * size             # x, (residual, sum), y
    if not c["train"]:
        return dict(bytes=streams + N * K + 4 * -(-N // BLOCK) * -(-K // BLOCK), flops=2 * T * N * K)
    back = T * N * size + T * K * size * (2 if norm else 1) + 2 * N * K * size   # dy, (ds,) dx; w and dw
    return dict(bytes=streams + back, flops=6 * T * N * K)


def _e4m3(v):
    """Nearest e4m3 value, half to even, in 64 bits: steps of an eighth of the power of two, the smallest 2^-9."""
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (e - 1).clamp(min=-6) - 3)
    return (torch.round(v / step) * step).clamp(-TOP, TOP)


def _exact_block(x, dim):
    out = torch.empty_like(x)
    for i in range(0, x.shape[dim], BLOCK):
        part = x.narrow(dim, i, min(BLOCK, x.shape[dim] - i))
        amax = part.abs().amax(dim, keepdim=True).clamp(min=TINY)
        out.narrow(dim, i, part.shape[dim]).copy_(_e4m3(part * TOP / amax) * (amax / TOP))
    return out


def _exact_tiles(w):
    out = torch.empty_like(w)
    for i in range(0, w.shape[0], BLOCK):
        part = torch.nn.functional.pad(w[i:i + BLOCK], (0, -w.shape[1] % BLOCK))
        amax = part.abs().amax(0).view(-1, BLOCK).amax(1).clamp(min=TINY).repeat_interleave(BLOCK)
        out[i:i + BLOCK] = (_e4m3(part * TOP / amax) * (amax / TOP))[:, :w.shape[1]]
    return out


def exact(case, seed):
    st = prepare(case, seed)
    c = case
    with torch.no_grad():
        x = st["x"].detach().double()
        out = {}
        if c["kind"] != "linear":
            out["s"] = x + st["res"].detach().double()
            s = out["s"].to(st["x"].dtype).double()                        # the stream as it is kept
            gain = st["g"].detach().double()
            rms = (s.square().mean(-1, keepdim=True) + EPS) ** 0.5
            x = s / rms * gain
            if c["kind"] == "norm":
                return dict(out, y=_exact_block(x, 1))
        if c["train"]:
            w = _exact_tiles(st["w"].detach().double())
        else:
            q, scale = st["w"]
            k, n = torch.arange(c["K"], device=DEV) // BLOCK, torch.arange(c["N"], device=DEV) // BLOCK
            w = q.double() * scale.double()[n][:, k]
        out["y"] = torch.einsum("tk,nk->tn", _exact_block(x, 1), w)
        if st["b"] is not None:
            out["y"] += st["b"].detach().double()
        if not c["train"]:
            return out if c["kind"] == "norm_linear" else out["y"]
        gy = st["gy"].double()
        out["dw"] = torch.einsum("tn,tk->nk", _exact_block(gy, 0), _exact_block(x, 0))
        dx = torch.einsum("tn,nk->tk", _exact_block(gy, 1), w)
        if st["b"] is not None:
            out["db"] = gy.sum(0)
        if c["kind"] == "norm_linear":
            h = s / rms
            out["dg"] = torch.einsum("tk,tk->k", dx, h)
            dx = dx * gain
            dx = (dx - h * (dx * h).mean(-1, keepdim=True)) / rms + st["gs"].double()
            out["dres"] = dx
        out["dx"] = dx
        return out
