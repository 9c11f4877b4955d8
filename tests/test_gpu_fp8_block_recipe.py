"""`fp8_recipe: block128` where weights change, are traced, captured, partitioned or loaded: the codes of a weight are those of the weight as it is."""
import pytest
import torch

from savanna_b200 import ops

pytestmark = pytest.mark.gpu


def _randn(*shape, seed=0, dtype=torch.bfloat16, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


@pytest.fixture
def recipe():
    from savanna_b200.ops import cuda_ops
    cuda_ops.set_fp8_recipe("block128")
    yield cuda_ops
    cuda_ops.set_fp8_recipe("delayed")


class _Projections(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.g, self.w, self.b = (torch.nn.Parameter(_randn(*s, seed=i)) for i, s in enumerate([(256,), (64, 256), (64,)]))

    def forward(self, x):
        return ops.linear(x, self.w, self.b, fp8=True), ops.norm_linear(x, self.g, 1e-5, "te", self.w, None, True)[0]


def test_traced_graph_sees_changed_weights(recipe):
    x, m = _randn(20, 256, seed=7), _Projections()
    with torch.no_grad():
        m.b.zero_()
        m(x)                                                      # a call that may keep codes
        f = torch.jit.trace(m, (x,), check_trace=False)
        before = f(x)
        m.w.mul_(2.0)
        recipe.bump_param_epoch()
        for a, b in zip(f(x), before):
            assert torch.equal(a.float(), 2.0 * b.float())


# ------------------------------------------------------------------------------------------------ optimizers

