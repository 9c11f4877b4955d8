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


# ------------------------------------------------------------------------------------------------ written past PyTorch's counters


def test_weights_written_through_their_data(recipe):
    x, g, w = _randn(20, 256), _randn(256, seed=2), torch.nn.Parameter(_randn(64, 256, seed=1))
    with torch.no_grad():
        before = ops.linear(x, w, fp8=True), ops.norm_linear(x, g, 1e-5, "te", w, None, True)[0]
        w.data.mul_(2.0)                                          # a version counter of its own
        after = ops.linear(x, w, fp8=True), ops.norm_linear(x, g, 1e-5, "te", w, None, True)[0]
    for a, b in zip(after, before):
        assert torch.equal(a.float(), 2.0 * b.float())


def test_weights_written_by_a_replayed_graph(recipe):
    x, w = _randn(20, 256), torch.nn.Parameter(_randn(64, 256, seed=1))
    with torch.no_grad():
        ops.linear(x, torch.nn.Parameter(_randn(64, 256, seed=5)), fp8=True)
        torch.cuda.synchronize()
        update = torch.cuda.CUDAGraph()
        with torch.cuda.graph(update):
            w.mul_(2.0)
        before = ops.linear(x, w, fp8=True).float()
        update.replay()
        assert torch.equal(ops.linear(x, w, fp8=True).float(), 2.0 * before)


def test_weights_are_quantised_once_where_they_do_not_change(recipe):
    x, w = _randn(20, 256), torch.nn.Parameter(_randn(64, 256, seed=1))

    def launches(call):
        before = recipe.launch_count()
        y = call()
        return recipe.launch_count() - before, y
    with torch.no_grad():
        alone, want = launches(lambda: ops.linear(x, w, fp8=True))
        with recipe.weights_unchanged():
            first, a = launches(lambda: ops.linear(x, w, fp8=True))
            with recipe.weights_unchanged():                      # the outer one's codes hold in it
                again, b = launches(lambda: ops.linear(x, w, fp8=True))
            after, c = launches(lambda: ops.linear(x, w, fp8=True))
        assert first == alone and again == after == alone - 1
        assert all(torch.equal(y, want) for y in (a, b, c))
        w.data.mul_(2.0)
        with recipe.weights_unchanged():
            assert torch.equal(ops.linear(x, w, fp8=True).float(), 2.0 * want.float())
        w.data.mul_(2.0)
        assert torch.equal(ops.linear(x, w, fp8=True).float(), 4.0 * want.float())


@pytest.mark.parametrize("forward_inside", [False, True])
def test_checkpointed_forward_and_its_recomputation_on_different_sides(recipe, forward_inside):
    import contextlib
    from torch.utils.checkpoint import checkpoint
    m, x = _Projections(), _randn(20, 256, seed=7).requires_grad_()
    leaves = [x] + list(m.parameters())

    def loss(run):
        return sum(y.float().square().sum() for y in run(x))
    want = torch.autograd.grad(loss(m), leaves)
    sides = [recipe.weights_unchanged, contextlib.nullcontext]
    with sides[not forward_inside]():
        y = loss(lambda t: checkpoint(m, t, use_reentrant=False))
    with sides[forward_inside]():
        got = torch.autograd.grad(y, leaves)
    for a, e in zip(got, want):
        assert torch.equal(a, e)


def test_traced_graph_from_between_two_updates(recipe):
    x, m = _randn(20, 256, seed=7), _Projections()
    with torch.no_grad():
        m.b.zero_()
        with recipe.weights_unchanged():
            m(x)
            f = torch.jit.trace(m, (x,), check_trace=False)
            before = f(x)
        m.w.data.mul_(2.0)
        for a, b in zip(f(x), before):
            assert torch.equal(a.float(), 2.0 * b.float())


# ------------------------------------------------------------------------------------------------ optimizers

_OVER = {"global_num_gpus": 1, "train_micro_batch_size_per_gpu": 1, "use_fp8_linears": True, "use_fp8_input_projections": True, "use_fp8_output_projections": True,
         "use_fp8_mlp_projections": True}


def _trainer(over):
    import os
    from savanna_b200.config import GlobalConfig
    from savanna_b200.train.trainer import Trainer
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    return Trainer(GlobalConfig.from_ymls([os.path.join(root, "configs", "baseline", "tiny_sh2_gpu.yml")], dict(_OVER, **over)), load=False)


def _batches(cfg, n, first=0):
    from savanna_b200.data.synthetic import acgt_batch
    return iter([{"text": acgt_batch(cfg.train_micro_batch_size_per_gpu, cfg.seq_length, seed=first + i, pin=True)} for i in range(n)])


@pytest.fixture
def trainers():
    from savanna_b200.ops import cuda_ops
    from savanna_b200.parallel import state
    yield _trainer
    state.destroy_model_parallel()
    cuda_ops.set_fp8_recipe("delayed")


def _trace(over, n=6):
    from savanna_b200.parallel import state
    tr = _trainer(over)
    d = _batches(tr.cfg, n * tr.gas)
    out = [float(tr.train_step(d)) for _ in range(n)]
    state.destroy_model_parallel()
    return out


@pytest.mark.parametrize("fp8_recipe", ["delayed", "mxfp8", "block128"])
@pytest.mark.parametrize("stage", [2, 3])
def test_optimizer_on_the_host_under_partitioned_stages(trainers, fp8_recipe, stage):
    """The update is written by the CPU and gathered into flat buffers: the next step's projections run on it."""
    over = {"fp8_recipe": fp8_recipe, "gradient_accumulation_steps": 2}
    want = _trace(dict(over, zero_optimization={"stage": 1}))
    got = _trace(dict(over, zero_optimization={"stage": stage, "offload_optimizer": {"device": "cpu"}}))
    assert max(abs(a - b) for a, b in zip(want, got)) < 2e-2 * max(want), (want, got)


@pytest.mark.parametrize("stage", [1, 2, 3])
def test_weights_rewritten_from_optimizer_state(trainers, stage):
    """`sync_params_from_master` and `load_state_dict` rewrite flat buffers or shards: no projection keeps codes of what was there.  (Under the
    other recipes the model also runs projections with an amax history, which no two losses share.)"""
    from savanna_b200.ops import cuda_ops
    tr = trainers({"fp8_recipe": "block128", "zero_optimization": {"stage": stage}})

    def loss():
        return tr.evaluate(_batches(tr.cfg, 1, 50), iters=1)["lm_loss"]
    tr.train_step(_batches(tr.cfg, 1))
    saved = [g.master.clone() for g in tr.optimizer.groups]
    tr.optimizer.sync_params_from_master()                        # flat buffers without what rounding to bf16 may have added
    want = loss()
    for i in range(4):
        tr.train_step(_batches(tr.cfg, 1, 1 + i))
    assert abs(loss() - want) > 1e-2                              # and the codes of these weights may be kept now
    sd = tr.optimizer.state_dict()
    for g, m in zip(tr.optimizer.groups, saved):
        g.master.copy_(m)
    if stage == 1:
        tr.optimizer.sync_params_from_master()
    else:
        tr.optimizer.load_state_dict(dict(sd, single_partition_of_fp32_groups=[m.clone() for m in saved]))
    assert loss() == want
    for i in range(2):
        tr.train_step(_batches(tr.cfg, 1, 1 + i))
    loss()
    for g, m in zip(tr.optimizer.groups, saved):
        g.master.copy_(m)
    epoch = cuda_ops.PARAM_EPOCH
    tr.optimizer.sync_params_from_master()
    assert cuda_ops.PARAM_EPOCH > epoch and loss() == want


@pytest.mark.parametrize("fp8_recipe", ["delayed", "mxfp8", "block128"])
def test_other_optimizers_are_followed(recipe, fp8_recipe):
    """A step of SGD that doubles the weight doubles its projection."""
    from savanna_b200.train.optimizers import DataParallelOptimizer
    recipe.set_fp8_recipe(fp8_recipe)
    x, w = _randn(32, 256), torch.nn.Parameter(_randn(64, 256, seed=1))
    opt = DataParallelOptimizer(torch.optim.SGD([w], lr=1.0), 0.0, None, 1)
    w.grad = -w.detach().clone()
    with torch.no_grad():
        before = [ops.linear(x, w, fp8=True).float() for _ in range(2)][1]
        opt.step()
        assert torch.equal(ops.linear(x, w, fp8=True).float(), 2.0 * before)


def test_released_units_keep_no_codes(trainers):
    tr = trainers({"fp8_recipe": "block128", "zero_optimization": {"stage": 3}})
    for i in range(2):
        tr.train_step(_batches(tr.cfg, 1, i))
    tr.evaluate(_batches(tr.cfg, 1, 9), iters=1)
    flats = [f for u in tr.optimizer.units[1:] for f in u.flats]
    assert flats and all(f.full.untyped_storage().size() == 0 for f in flats)
    kept = [p for f in flats for p in f.params if getattr(p, "_fp8_block_cache", None) is not None]
    assert not kept


def test_kept_codes_are_those_of_the_weights_they_stand_for(trainers):
    """After steps and an evaluation: whatever is kept on a parameter is a fresh quantisation of it."""
    tr = trainers({"fp8_recipe": "block128", "zero_optimization": {"stage": 1}, "gradient_accumulation_steps": 2})
    for i in range(3):
        tr.train_step(_batches(tr.cfg, 2, 2 * i))
    tr.evaluate(_batches(tr.cfg, 1, 9), iters=1)
    kept = [(p, p._fp8_block_cache[1]) for p in tr.model.parameters() if getattr(p, "_fp8_block_cache", None) is not None]
    assert kept
    for p, (q, s) in kept:
        want_q, want_s = ops.fp8_block_quantize_weight(p.detach())
        assert torch.equal(s, want_s) and torch.equal(q.view(torch.uint8), want_q.view(torch.uint8))


def test_partitioned_stage_3_matches_stage_1(trainers):
    over = {"fp8_recipe": "block128", "gradient_accumulation_steps": 2}
    want = _trace(dict(over, zero_optimization={"stage": 1}))
    got = _trace(dict(over, zero_optimization={"stage": 3}, checkpoint_activations=True, checkpoint_num_layers=2))
    assert max(abs(a - b) for a, b in zip(want, got)) < 2e-2 * max(want), (want, got)


def test_training_follows_bf16(trainers):
    """The loss of 30 steps under the recipe stays beside that in bf16: as near as the block-scaled hardware format has to."""
    plain = _trace({k: False for k in _OVER if k.startswith("use_fp8")} | {"train_micro_batch_size_per_gpu": 2}, 30)
    block = _trace({"fp8_recipe": "block128", "train_micro_batch_size_per_gpu": 2}, 30)
    assert abs(plain[-1] - block[-1]) < 0.06 * plain[-1], (plain[-1], block[-1])
    assert max(abs(a - b) for a, b in zip(plain, block)) < 0.2, (plain, block)
    assert plain != block


# ------------------------------------------------------------------------------------------------ traced


class _Codes(_Projections):
    def forward(self, x):
        q, s, _ = ops.rmsnorm_fp8_block(x, self.g, 1e-5)
        return ops.linear_fp8_block((q, s), self.w, self.b), ops.norm_linear_fp8_block(x, self.g, 1e-5, "te", self.w, self.b)[0]


def test_traced_calls_with_codes_under_no_grad(recipe):
    """A parameter in the projection of an input given as codes is no reason to refuse it where no gradient is wanted."""
    m = _Codes()
    with torch.no_grad():
        traced = torch.jit.trace(m, (_randn(20, 256, seed=7),), check_trace=False)
        y = _randn(20, 256, seed=8)
        for a, e in zip(traced(y), m(y)):
            assert torch.equal(a, e) and not a.requires_grad


def test_traced_without_gradients_and_run_with_them(recipe):
    m, x = _Projections(), _randn(20, 256, seed=7)
    with torch.no_grad():
        f = torch.jit.trace(m, (x,), check_trace=False)
    got, want = (torch.autograd.grad([y.float().square().sum() for y in g(x)], list(m.parameters())) for g in (f, m))
    for a, e in zip(got, want):
        assert torch.equal(a, e)


class _KeptCodes(_Projections):
    def __init__(self):
        super().__init__()
        self.q, self.s = ops.fp8_block_quantize_weight(self.w.detach())

    def forward(self, x):
        q, s, _ = ops.rmsnorm_fp8_block(x, self.g, 1e-5)
        return ops.linear_fp8_block((q, s), (self.q, self.s))


def test_traced_codes_want_no_gradient(recipe):
    """Codes of an input that wants a gradient carry none, traced as otherwise."""
    m, x = _KeptCodes(), _randn(20, 256, seed=7)
    assert torch.equal(torch.jit.trace(m, (x,), check_trace=False)(x), m(x))


# ------------------------------------------------------------------------------------------------ loaded for generation


@pytest.mark.parametrize("fp8_recipe", ["mxfp8", "block128"])
def test_loaded_checkpoints_run_their_recipe(trainers, fp8_recipe, tmp_path):
    import os
    from savanna_b200.ckpt import save_checkpoint
    from savanna_b200.inference.load import load_for_inference
    from savanna_b200.ops import cuda_ops
    tr = trainers({"fp8_recipe": fp8_recipe, "zero_optimization": {"stage": 1}, "save": str(tmp_path)})
    tr.train_step(_batches(tr.cfg, 1))
    save_checkpoint(tr, 1)
    tokens = next(_batches(tr.cfg, 1, 5))["text"][:, :96].long().cuda()
    tr.model.eval()
    positions = torch.arange(96, device="cuda")
    with torch.no_grad():
        want = tr.model(tokens, positions)
        cuda_ops.set_fp8_recipe("delayed")
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        model, _, cfg = load_for_inference(str(tmp_path), [os.path.join(root, "configs", "baseline", "tiny_sh2_gpu.yml")], overrides=dict(_OVER, fp8_recipe=fp8_recipe))
        assert cfg.fp8_recipe == fp8_recipe and cuda_ops.FP8_RECIPE == fp8_recipe
        if fp8_recipe == "block128":                             # the other's model has projections with an amax history too
            assert torch.equal(model(tokens, positions), want)
