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


def _in_thread(call):
    import threading
    out = []
    t = threading.Thread(target=lambda: out.append(call()))
    t.start()
    t.join()
    return out[0]


def test_unchanged_weights_end_with_the_outer_context_and_with_an_error():
    from savanna_b200.ops import cuda_ops
    assert cuda_ops._unchanged() is None
    with cuda_ops.weights_unchanged():
        outer = cuda_ops._unchanged()
        assert outer is not None
        with cuda_ops.weights_unchanged():
            assert cuda_ops._unchanged() is outer
        assert cuda_ops._unchanged() is outer
    assert cuda_ops._unchanged() is None
    try:
        with cuda_ops.weights_unchanged():
            raise KeyError
    except KeyError:
        pass
    assert cuda_ops._unchanged() is None
    with cuda_ops.weights_unchanged():
        assert cuda_ops._unchanged() not in (None, outer)


def test_unchanged_weights_of_one_thread_are_no_others():
    """Contexts that overlap in two threads leave nothing open, and hold for one of them alone."""
    import threading
    from savanna_b200.ops import cuda_ops
    inside, go = threading.Event(), threading.Event()
    seen = []

    def other():
        with cuda_ops.weights_unchanged():
            seen.append(cuda_ops._unchanged())
            inside.set()
            go.wait(30)
            seen.append(cuda_ops._unchanged())
    t = threading.Thread(target=other)
    with cuda_ops.weights_unchanged():
        assert cuda_ops._unchanged() is not None and _in_thread(cuda_ops._unchanged) is None
        t.start()
        assert inside.wait(30)
    assert cuda_ops._unchanged() is None
    go.set()
    t.join()
    assert seen == [None, None] and cuda_ops._unchanged() is None


def test_unchanged_weights_hold_in_the_backward_pass():
    """Checkpointed blocks run again there, by the autograd engine."""
    from savanna_b200.ops import cuda_ops
    seen = []

    class Again(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return x * 2

        @staticmethod
        def backward(ctx, g):
            seen.append(cuda_ops._unchanged())
            return g * 2
    x = torch.ones(3, requires_grad=True)
    with cuda_ops.weights_unchanged():
        mark = cuda_ops._unchanged()
        Again.apply(x).sum().backward()
        _in_thread(lambda: Again.apply(x).sum().backward())
    Again.apply(x).sum().backward()
    assert seen == [mark, mark, None]
