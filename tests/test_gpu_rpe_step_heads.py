"""Attention step over a cache: head sizes that leave lanes of a key's group without columns, against the definition in 64 bits (tolerance: that of
`tests/test_gpu_rpe_step.py`)."""
import pytest
import torch

from savanna_b200 import ops
from tests.test_gpu_rpe_step import _case, _check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [8, 40, 64, 72, 96, 128, 136, 200, 256])
@pytest.mark.parametrize("B,T,H", [(20, 40, 4), (2, 900, 2), (1, 9000, 2)], ids=["one block", "cluster", "two kernels"])
def test_a_key_of_infinity_away_from_the_query_has_no_weight(B, T, H, hd):
    """A score of -inf: the row is that of the other keys, for every head size (in some of them lanes have no columns of their own)."""
    q, k, v, table, buckets, lengths = _case(B, T, H, hd, torch.bfloat16, seed=hd)
    lengths = lengths.clamp(min=T // 2 + 1)
    q[..., 1] = q[..., 1].abs() + 0.5                # bf16 values of at least one half: 0.5 * -inf = -inf
    k[:, T // 3, :, 1] = float("-inf")
    for n in (lengths, None):
        got = ops.attention_rpe_step(q, k, v, table, buckets, 1.0, n)
        assert bool(got.isfinite().all())
        _check(got, q, k, v, table, buckets, 1.0, n)
