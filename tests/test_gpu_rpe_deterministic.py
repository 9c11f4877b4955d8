"""Attention with a relative position bias under torch.use_deterministic_algorithms: gradients that repeat themselves bit by bit."""
import pytest
import torch

from savanna_b200 import ops
from savanna_b200.ops import reference as ref
from tests.test_gpu_rpe import _case, _run

pytestmark = pytest.mark.gpu


@pytest.fixture
def deterministic():
    was, warn = torch.are_deterministic_algorithms_enabled(), torch.is_deterministic_algorithms_warn_only_enabled()
    torch.use_deterministic_algorithms(True, warn_only=True)       # cuBLAS wants a variable of the environment otherwise
    yield
    torch.use_deterministic_algorithms(was, warn_only=warn)


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "both"])
def test_gradients_repeat_themselves(causal, deterministic):
    c = _case(2, 1500, 2, 32, 128, causal, table_dtype=torch.float32)
    first = _run(*c[:3], 3.0, causal, c[3])
    for _ in range(6):
        for a, b in zip(first, _run(*c[:3], 3.0, causal, c[3])):
            assert torch.equal(a, b)
    q, t = c[0].clone().requires_grad_(True), c[1].clone().requires_grad_(True)
    o = ref.attention_rpe(q, t, c[2], 3.0, causal)
    for a, b in zip(first, (o, *torch.autograd.grad(o, (q, t), c[3]))):
        assert torch.equal(a, b)


@pytest.mark.filterwarnings("ignore")
def test_without_gradients_the_kernels_run(deterministic):
    c = _case(1, 200, 2, 32, 64, True)
    with torch.no_grad():
        got = ops.attention_rpe(*c[:3], 3.0, True)
    torch.use_deterministic_algorithms(False)
    with torch.no_grad():
        assert torch.equal(got, ops.attention_rpe(*c[:3], 3.0, True))
