"""What the fp8 recipes keep on a weight, on the CPU: dropped with the weight, and ended where weights are written."""
import re

import torch

from savanna_b200 import ops


def test_every_copy_that_a_recipe_keeps_goes_with_the_parameters():
    import os
    from savanna_b200.parallel.zero_partitioned import UnitFlat
    with open(os.path.join(os.path.dirname(ops.__file__), "cuda_ops.py")) as fh:
        names = set(re.findall(r"\bw\.(_\w*cache)\b", fh.read()))
    assert {"_fp8_cache", "_mx_cache", "_fp8_block_cache"} <= names
    params = [torch.nn.Parameter(torch.randn(8, 16)) for _ in range(2)]
    flat = UnitFlat(params, 1, 0, {}, "unit", free_params=True, free_grads=True, tp=1)
    for p in params:
        for n in names:
            setattr(p, n, object())
    flat.release_params()
    assert not [n for p in params for n in names if getattr(p, n) is not None]


def test_block_scaled_recipes_leave_the_fused_tensor_parallel_projections_out():
    """Those take per-tensor scales: the caller gathers or scatters around the block-scaled projection."""
    from savanna_b200.ops import cuda_ops
    x, w = torch.randn(4, 8, 16), torch.randn(24, 16)
    try:
        for name in ("mxfp8", "block128"):
            cuda_ops.set_fp8_recipe(name)
            assert cuda_ops.linear_allgather(x, w, None, 1, True) is None and cuda_ops.linear_reducescatter(x, w, 1, True) is None
    finally:
        cuda_ops.set_fp8_recipe("delayed")


def test_unchanged_weights_end_with_the_outer_context_and_with_an_error():
    from savanna_b200.ops import cuda_ops
    assert cuda_ops._UNCHANGED is None
    with cuda_ops.weights_unchanged():
        outer = cuda_ops._UNCHANGED
        with cuda_ops.weights_unchanged():
            assert cuda_ops._UNCHANGED is outer
        assert cuda_ops._UNCHANGED is outer
    assert cuda_ops._UNCHANGED is None
    try:
        with cuda_ops.weights_unchanged():
            raise KeyError
    except KeyError:
        pass
    assert cuda_ops._UNCHANGED is None
    with cuda_ops.weights_unchanged():
        assert cuda_ops._UNCHANGED is not outer
