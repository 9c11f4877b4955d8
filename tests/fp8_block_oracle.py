"""The definition of 8-bit operands with a scale for each block of 128 in 64 bits, apart from the framework's code."""
import torch

TOP, TINY, BLOCK = 448.0, 2.0 ** -100, 128


def e4m3(v):
    """Nearest e4m3 value, half to even."""
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (e - 1).clamp(min=-6) - 3)
    return (torch.round(v / step) * step).clamp(-TOP, TOP)


def blockwise(x, dim):
    """x (float64) as its 8-bit form stands for it, a scale for 128 values along `dim`."""
    out = torch.empty_like(x)
    for i in range(0, x.shape[dim], BLOCK):
        n = min(BLOCK, x.shape[dim] - i)
        part = x.narrow(dim, i, n)
        amax = part.abs().amax(dim, keepdim=True).clamp(min=TINY)
        out.narrow(dim, i, n).copy_(e4m3(part * TOP / amax) * (amax / TOP))
    return out


def tiles(w):
    out = torch.empty_like(w)
    for i in range(0, w.shape[0], BLOCK):
        for j in range(0, w.shape[1], BLOCK):
            part = w[i:i + BLOCK, j:j + BLOCK]
            amax = part.abs().max().clamp(min=TINY)
            out[i:i + BLOCK, j:j + BLOCK] = e4m3(part * TOP / amax) * (amax / TOP)
    return out


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def close_sum(got, want, terms, dtype, what, roundings=1):
    """got (of `dtype`) against a sum in 64 bits whose terms have the magnitudes `terms` in all: one rounding to the type (`roundings` of them);
    scales carry a rounding each to 24 bits, and the fp32 sums of 128 products and of the blocks at most 2^-23 for each of some 130 additions,
    together below 2^-15 of the terms' magnitude."""
    # below the type's smallest normal value a rounding is off by half its smallest step
    floor = torch.finfo(dtype).smallest_normal * half_step(dtype)
    bound = roundings * (half_step(dtype) * want.abs() + floor) + 2.0 ** -15 * terms
    err = (got.double() - want).abs()
    assert got.shape == want.shape and bool((err <= bound).all()), f"{what}: {float((err / bound.clamp(min=1e-300)).max())} of the bound"
