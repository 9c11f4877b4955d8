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
