"""Attention with a relative position bias where a score is NaN or +inf: the whole row of its softmax is NaN, and with it the row's output and query
gradient and the gradients of all keys and values that the row sees.  Other rows, heads and sequences are not touched."""
import pytest
import torch

from tests.test_gpu_rpe import _case, _run

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("causal", [True, False], ids=["causal", "both"])
@pytest.mark.parametrize("L", [40, 300, 1100])
@pytest.mark.parametrize("where", ["q", "k", "infinite key", "table"])
def test_a_score_that_is_not_a_number_shows_in_all_that_depends_on_it(where, L, causal):
    qkv, table, buckets, go = _case(2, L, 2, 32, 20, causal, table_dtype=torch.float32)
    at = L // 3
    i = torch.arange(L, device=DEV)
    sees = (i[:, None] >= i[None, :]) | (not causal)
    bad = torch.zeros(2, 2, L, dtype=torch.bool, device=DEV)         # rows whose softmax is NaN, [B, H, L]
    if where == "q":
        qkv[1, at, 1, 3] = float("nan")
        bad[1, 1, at] = True
    elif where == "table":                           # of the distance 5
        table[int(buckets[5 if causal else 25]), 1] = float("nan")
        hit = (buckets == buckets[5 if causal else 25]).nonzero().flatten() - (0 if causal else 20)
        d = (i[:, None] - i[None, :]).clamp(-20, 20)
        bad[:, 1] = (torch.isin(d, hit) & sees).any(-1)
    else:
        qkv[..., 3] = qkv[..., 3].abs() + 0.5
        qkv[1, at, 1, 131] = float("nan") if where == "k" else float("inf")
        bad[1, 1] = sees[:, at]
    o, dqkv, dt = _run(qkv, table, buckets, 2.0, causal, go)
    rows = bad.transpose(1, 2)                       # [B, L, H]
    keys = (bad[..., None] & sees).any(-2).transpose(1, 2)
    assert torch.equal(o.isnan().any(-1), rows) and torch.equal(o.isnan().all(-1), rows)
    assert bool(dqkv[..., :128][rows].isnan().all())
    assert bool(dqkv[..., 128:][keys].isnan().all())
    assert bool(dqkv[..., 256:][~keys].isfinite().all())
    assert bool(dt[:, 1].isnan().any()) and bool(dt[:, 0].isfinite().all()) and bool(dqkv[:, :, 0].isfinite().all())
