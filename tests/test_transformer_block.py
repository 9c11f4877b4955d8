"""The transformer block of `norm: layernorm`, the `global` operator with `pos_emb: rpe`, and checkpoints in 8 bits: the operators as a
model uses them together, in training and in cached generation."""
import os

import pytest
import torch

from savanna_b200 import ops
from savanna_b200.config import GlobalConfig
from savanna_b200.inference.cached import CachedDecoder
from savanna_b200.models import build_model
from savanna_b200.models.rope import RelativePositionBias, are_consecutive, consecutive_positions, mark_consecutive
from savanna_b200.ops import reference as ref
from savanna_b200.parallel import state

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _model(yml, device=None, **over):
    cfg = GlobalConfig.from_ymls([os.path.join(ROOT, "configs", "baseline", yml)],
                                 {"global_num_gpus": 1, "norm": "layernorm", "pos_emb": "rpe", "operator_config": [[["global"], 2]], "num_layers": 2,
                                  **over})
    cfg.build_tokenizer()
    torch.manual_seed(0)
    model = build_model(cfg, device=device)
    with torch.no_grad():                            # norms and tables that matter
        for n, p in model.named_parameters():
            if "norm" in n:
                p.add_(0.2 * torch.randn(p.shape, generator=torch.Generator().manual_seed(p.numel())).to(p))
    return cfg, model


def _tokens(B, n, device=None):
    return torch.randint(0, 256, (B, n), generator=torch.Generator().manual_seed(n)).to(device or "cpu")


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("nb,maxd", [(32, 128), (16, 100), (64, 300), (8, 5)])
def test_bucket_map_has_the_bucket_of_every_distance(nb, maxd, causal):
    m = RelativePositionBias(1.0, causal, nb, maxd, heads=2)
    far, buckets = m.far, m.bucket_map()
    assert far == maxd and buckets.dtype == torch.int32 and buckets.shape == ((far + 1,) if causal else (2 * far + 1,))
    L = 2 * far + 50
    want = m.bias(torch.arange(L), torch.arange(L))
    assert torch.equal(want, ref.relative_bias(m.weight, buckets, m.scale, L, L, causal))
    assert m.bucket_map() is buckets
    m.max_distance = 2 * maxd
    assert m.bucket_map().shape[0] != buckets.shape[0]


def test_no_bucket_map_where_buckets_do_not_grow():
    m = RelativePositionBias(1.0, True, 32, 16, heads=2)
    assert m.far == -1
    with pytest.raises(ValueError):
        m.bucket_map()


def test_marks_of_consecutive_positions():
    p = consecutive_positions(5)
    assert torch.equal(p, torch.arange(5)) and are_consecutive(p)
    assert not are_consecutive(torch.arange(5)) and not are_consecutive(p.flip(0)) and not are_consecutive(p.detach())
    assert are_consecutive(mark_consecutive(p.detach()))
    p[0] = 7
    assert not are_consecutive(p)
    with torch.inference_mode():
        assert are_consecutive(consecutive_positions(3))


def test_cached_generation_with_relative_positions_follows_the_model():
    _, model = _model("tiny_sh2_cpu.yml")
    model.eval()
    toks = _tokens(2, 40)
    dec = CachedDecoder(model)
    with torch.no_grad():
        got = dec.prefill(toks[:, :30])
        for n in range(30, 40):
            want = model(toks[:, :n])[:, -1].float()
            # two layers of fp32 sums in another order: a few hundred roundings of values of a few units
            assert float((got - want).abs().max()) <= 512 * 2.0 ** -24 * float(want.abs().max().clamp(min=1))
            got = dec.step(toks[:, n])


def test_cached_generation_refuses_what_it_does_not_cover():
    for over in ({"pos_emb": "alibi"}, {"rpe_max_distance": 16}):
        _, model = _model("tiny_sh2_cpu.yml", **over)
        with pytest.raises(NotImplementedError):
            CachedDecoder(model)


def _by_hand(model, toks, labels, chunks):
    """Gradients of the blocks' parameters when each chunk's backward pass runs at its input as 8 bits give it back."""
    pos = consecutive_positions(toks.shape[1], toks.device)
    blocks = model.blocks()
    with torch.no_grad():
        ins, x = [], model.embedding(toks, pos)
        for s in range(0, len(blocks), chunks):
            ins.append(x)
            for b in blocks[s:s + chunks]:
                x = b(x, pos)
    x = x.detach().requires_grad_(True)
    ops.cross_entropy(model.logits(x), labels).mean().backward()
    g = x.grad
    for i in reversed(range(len(ins))):
        h = ops.act_dequantize(*ops.act_quantize(ins[i]), ins[i].dtype).requires_grad_(True)
        y = h
        for b in blocks[i * chunks:(i + 1) * chunks]:
            y = b(y, pos)
        y.backward(g)
        g = h.grad
    return {n: p.grad.clone() for n, p in model.named_parameters() if p.grad is not None and ".mixer." in n or ".mlp." in n}


def _compare_8bit(yml, device, same, **over):
    cfg, model = _model(yml, device, checkpoint_activations=True, checkpoint_num_layers=1, checkpoint_in_8bit=True, **over)
    model.train()
    toks = _tokens(2, cfg.seq_length if device is None else 200, device)
    labels = toks.roll(-1, 1)
    want = _by_hand(model, toks, labels, 1)
    for p in model.parameters():
        p.grad = None
    # inputs reach the re-entrant checkpoint with gradients only where the embedding has them
    ops.cross_entropy(model(toks), labels).mean().backward()
    seen = 0
    for n, p in model.named_parameters():
        if n in want and want[n].abs().max() > 0:
            assert same(p.grad, want[n]), n
            seen += 1
    assert seen >= 10
    state.destroy_model_parallel()


@pytest.mark.parametrize("host", [False, True])
def test_checkpoints_in_8_bits_recompute_at_what_they_kept(host):
    _compare_8bit("tiny_sh2_cpu.yml", None, torch.equal, checkpoint_in_cpu=host)


def test_checkpoints_in_8_bits_refuse_partitioned_activations(monkeypatch):
    _, model = _model("tiny_sh2_cpu.yml", checkpoint_activations=True, checkpoint_in_8bit=True, partition_activations=True)
    monkeypatch.setattr(state, "get_model_parallel_world_size", lambda: 2)
    with pytest.raises(NotImplementedError):
        model._checkpoint_storage()


# ----------------------------------------------------------------------------- CUDA


def _gpu(**over):
    return _model("tiny_sh2_gpu.yml", "cuda", **{"hidden_size": 256, "num_attention_heads": 2, "attention_dropout": 0.0, "hidden_dropout": 0.0, **over})


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
def test_model_step_runs_the_kernels_and_agrees_with_the_statements(causal):
    from savanna_b200.ops import cuda_ops
    _, model = _gpu(pretraining_strategy="AR" if causal else "MLM")
    toks = _tokens(2, 300, "cuda")
    labels = toks.roll(-1, 1)

    def step():
        for p in model.parameters():
            p.grad = None
        logits = model(toks)
        ops.cross_entropy(logits, labels).mean().backward()
        return logits.detach().float(), {n: p.grad.float().clone() for n, p in model.named_parameters() if p.grad is not None}
    from unittest import mock
    with mock.patch.object(cuda_ops, "attention_rpe", wraps=cuda_ops.attention_rpe) as used, \
            mock.patch.object(cuda_ops, "layernorm_residual", wraps=cuda_ops.layernorm_residual) as norms:
        got = step()
    assert used.call_count == 2 and norms.call_count >= 2
    ops.set_backend("torch")
    try:
        want = step()
    finally:
        ops.set_backend("auto")
    # both round every activation to bf16, at different places: 2.2 % of the logits (2-norm), gradients through twice as many roundings
    assert (got[0] - want[0]).norm() <= 2.2e-2 * want[0].norm()
    for n, g in want[1].items():
        if g.norm() > 0:
            assert (got[1][n] - g).norm() <= 6e-2 * g.norm(), (n, float((got[1][n] - g).norm() / g.norm()))
    cuda_ops.check_status()


@pytest.mark.gpu
def test_positions_that_are_not_consecutive_take_the_materialised_scores():
    from savanna_b200.ops import cuda_ops
    from unittest import mock
    _, model = _gpu()
    model.eval()
    toks = _tokens(1, 100, "cuda")
    with torch.no_grad(), mock.patch.object(cuda_ops, "attention_rpe", wraps=cuda_ops.attention_rpe) as used:
        a = model(toks, torch.arange(100, device="cuda"))
        assert used.call_count == 0
        b = model(toks)
        assert used.call_count == 2
        c = model(toks, 3 * torch.arange(100, device="cuda"))
        assert used.call_count == 2
    assert (a.float() - b.float()).norm() <= 2.2e-2 * a.float().norm()
    assert (a.float() - c.float()).norm() > 5e-2 * a.float().norm()


@pytest.mark.gpu
def test_cached_generation_on_the_kernels_follows_the_model():
    from savanna_b200.ops import cuda_ops
    from unittest import mock
    _, model = _gpu()
    model.eval()
    toks = _tokens(3, 170, "cuda")
    dec = CachedDecoder(model)
    with torch.no_grad(), mock.patch.object(cuda_ops, "attention_rpe_step", wraps=cuda_ops.attention_rpe_step) as used:
        got = dec.prefill(toks[:, :150])
        assert dec._fused is None
        for n in range(150, 170):
            want = model(toks[:, :n])[:, -1].float()
            assert (got - want).norm() <= 2.2e-2 * want.norm()
            got = dec.step(toks[:, n])
        assert used.call_count == 40


@pytest.mark.gpu
def test_bucket_map_is_there_for_other_streams():
    rpe = RelativePositionBias(1.0, heads=2, device="cuda")
    want = rpe.bucket_map().cpu()
    rpe._map = None
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(first):
        torch.cuda._sleep(200_000_000)               # a tenth of a second before the map's values
        rpe.bucket_map()
    with torch.cuda.stream(second):
        got = rpe.bucket_map().clone()
    torch.cuda.synchronize()
    assert torch.equal(got.cpu(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("host", [False, True])
def test_checkpoints_in_8_bits_on_the_kernels(host):
    # the query gradient is added up in an order that varies: a few units of its 32-bit sums, then one rounding to bf16 that may fall on
    # either side, carried through the projections: 2^-8 of the 2-norm, twice
    _compare_8bit("tiny_sh2_gpu.yml", "cuda", lambda a, b: (a.float() - b.float()).norm() <= 2 * 2.0 ** -8 * b.float().norm(),
                  hidden_size=256, num_attention_heads=2, attention_dropout=0.0, hidden_dropout=0.0, checkpoint_in_cpu=host)


@pytest.mark.gpu
def test_captured_training_step_of_a_model():
    _, model = _gpu()
    toks = _tokens(1, 130, "cuda")
    labels = toks.roll(-1, 1)
    params = [p for p in model.parameters() if p.requires_grad]

    def step():
        loss = ops.cross_entropy(model(toks), labels).mean()
        return loss, torch.autograd.grad(loss, params, allow_unused=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = float(step()[0])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, grads = step()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert abs(float(loss) - want) <= 1e-5 * abs(want) and all(bool(g.isfinite().all()) for g in grads if g is not None)
