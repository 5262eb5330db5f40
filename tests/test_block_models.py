"""The decoder-block options (sliding window with first tokens, scaled embedding, norms on both sides, residual scale and gate) in
the LLaMA and OLMo-2 models: formulas, receptive field, parallel runs, command line, refusals. CPU."""
import argparse

import pytest
import torch

from maltos_b200.models import LlamaConfig, LlamaForCausalLM, OlmoConfig, OlmoForCausalLM
from maltos_b200.ops.embedding import ScaledEmbedding
from tests.dist_utils import run_distributed

SIZES = dict(vocab_size=96, hidden_size=64, intermediate_size=128, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
             max_position_embeddings=32)
OPTIONS = dict(sliding_window=5, sink_tokens=2, full_attention_every=2, embedding_scale=3.0, residual_scale=0.5, residual_gate=True)


def _model(kind, cls=None, seed=0, **options):
    import maltos_b200.models as M

    torch.manual_seed(seed)
    config = (LlamaConfig if kind == "llama" else OlmoConfig)(**{**SIZES, **options})
    model = (getattr(M, cls) if cls else (LlamaForCausalLM if kind == "llama" else OlmoForCausalLM))(config)
    with torch.no_grad():
        for name, p in model.named_parameters():
            if p.dim() == 1:                     # norms and gates away from one
                p.add_(0.2 * torch.randn(p.shape, generator=torch.Generator().manual_seed(len(name))))
    return model


def _ids(B=2, S=16, seed=7):
    return torch.randint(0, 96, (B, S), generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("kind", ["llama", "olmo"])
def test_options_left_alone_change_nothing(kind):
    plain, window = _model(kind), _model(kind, sliding_window=32)
    assert type(plain.embed_tokens) is torch.nn.Embedding
    assert [n for n, _ in plain.named_parameters()] == [n for n, _ in window.named_parameters()]
    a, b = plain(_ids()), window(_ids())
    torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-5)      # a window of the whole row is causal attention


@pytest.mark.parametrize("kind", ["llama", "olmo"])
def test_receptive_field(kind):
    """One windowed layer: a token reaches the next window - 1 positions, and all later ones if it is a first token."""
    model = _model(kind, num_hidden_layers=1, sliding_window=4, sink_tokens=1)
    ids = _ids(1)
    base = model(ids)
    for at, reached in ((0, range(0, 16)), (3, range(3, 7)), (8, range(8, 12))):
        other = ids.clone()
        other[0, at] = (other[0, at] + 1) % 96
        changed = (model(other) - base).abs().amax(-1)[0] > 0
        assert changed.nonzero().flatten().tolist() == list(reached)
    docs = torch.tensor([[0] * 8 + [1] * 7 + [-1]])
    pos = torch.tensor([list(range(8)) + list(range(7)) + [0]])
    base = model({"input_ids": ids, "sequence_ids": docs, "position_ids": pos})
    other = ids.clone()
    other[0, 8] = (other[0, 8] + 1) % 96         # first token of the second document
    changed = (model({"input_ids": other, "sequence_ids": docs, "position_ids": pos}) - base).abs().amax(-1)[0] > 0
    assert changed.nonzero().flatten().tolist() == list(range(8, 15))


def test_llama_block_is_the_formula():
    model = _model("llama", num_hidden_layers=1, post_block_norm=True, residual_scale=0.3, residual_gate=True, embedding_scale=2.0)
    layer, ids = model.layers[0], _ids()
    assert isinstance(model.embed_tokens, ScaledEmbedding)

    def norm(t, w):
        return w * t / (t.square().mean(-1, keepdim=True) + model.config.rms_norm_eps).sqrt()

    x = 2.0 * model.embed_tokens.weight[ids]
    n1, n2 = layer.post_attention_layernorm, layer.post_feedforward_layernorm
    x = x + 0.3 * n1.gate * norm(layer.self_attn(norm(x, layer.input_layernorm.weight)), n1.after_weight)
    x = x + 0.3 * n2.gate * norm(layer.mlp(norm(x, n1.weight)), n2.after_weight)
    torch.testing.assert_close(model(ids), model.lm_head(norm(x, model.norm.weight)), rtol=1e-4, atol=1e-5)


def test_olmo_block_is_the_formula():
    model = _model("olmo", num_hidden_layers=1, residual_scale=0.3, residual_gate=True)
    layer, ids = model.layers[0], _ids()

    def norm(t, w):
        return w * t / (t.square().mean(-1, keepdim=True) + model.config.rms_norm_eps).sqrt()

    x = model.embed_tokens.weight[ids]
    n1, n2 = layer.post_attention_layernorm, layer.post_feedforward_layernorm
    rotary = (model.rotary_emb.cos, model.rotary_emb.sin)
    x = x + 0.3 * n1.gate * norm(layer.self_attn(x, rotary=rotary), n1.after_weight)
    x = x + 0.3 * n2.gate * norm(layer.mlp(x), n2.after_weight)
    torch.testing.assert_close(model(ids), model.lm_head(norm(x, model.norm.weight)), rtol=1e-4, atol=1e-5)


def test_full_attention_every_and_flops():
    model = _model("llama", num_hidden_layers=4, **{**OPTIONS, "full_attention_every": 3})
    assert [layer.self_attn.attn_core.window for layer in model.layers] == [5, 5, None, 5]
    assert model.flops_per_token() < _model("llama", num_hidden_layers=4).flops_per_token()


def _worker(rank, world, kind, variant, options):
    import maltos_b200  # noqa: F401
    from maltos_b200.runtime import MeshConfig, RuntimeCore
    from maltos_b200.runtime.plugins.tp import TensorParallelPlugin
    from maltos_b200.runtime.plugins.tp_sp import TpSpPlugin
    from maltos_b200.runtime.plugins.zero3 import Zero3Plugin
    from maltos_b200.train.cli import _zero3_wrap_classes

    name = ("Llama" if kind == "llama" else "Olmo") + "ForCausalLM" + {"tp": "Tp", "sp": "TpSp", "zero3": ""}[variant]
    model = _model(kind, name, **options)
    ids = _ids()
    batch = {"input_ids": ids, "labels": ids.roll(-1, 1)}
    if variant == "zero3":
        batch = {k: v[rank:rank + 1] for k, v in batch.items()}
        plugin, mesh = Zero3Plugin(wrap_cls=_zero3_wrap_classes()), MeshConfig(dp=world)
    else:
        plugin, mesh = (TensorParallelPlugin() if variant == "tp" else TpSpPlugin()), MeshConfig(tp=world)
    rt = RuntimeCore(model=model, mesh=mesh, plugins=[plugin], optimizer_factory=lambda p: torch.optim.SGD(p, lr=0.1))
    rt.setup()
    losses = []
    for _ in range(2):
        loss, _ = rt.run_step(batch)
        rt.step_optimizer()
        losses.append(float(loss))
    rt.close()
    return losses


@pytest.mark.parametrize("kind,variant", [("llama", "tp"), ("llama", "sp"), ("olmo", "sp"), ("llama", "zero3"), ("olmo", "zero3")])
def test_parallel_runs_match_a_single_process(kind, variant):
    options = dict(OPTIONS, post_block_norm=True) if kind == "llama" else dict(OPTIONS)
    model = _model(kind, **options)
    ids = _ids()
    batch = {"input_ids": ids, "labels": ids.roll(-1, 1)}
    optimizer = torch.optim.SGD(model.parameters(), lr=0.1)
    want = []
    for _ in range(2):
        loss = model(batch)
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        want.append(float(loss))
    got = run_distributed(_worker, 2, kind, variant, options)
    if variant == "zero3":                       # each rank has the loss of its own row, rows have the same number of targets
        got = [[sum(x) / 2 for x in zip(*got)]]
    for losses in got:
        # fp32 sums in another order; the second loss has a step of every gradient behind it
        assert all(abs(a - b) < 5e-5 for a, b in zip(losses, want)), (losses, want)


def test_context_parallel_cores_refuse_a_window():
    from maltos_b200.runtime.layers.attn_masking_utils import refuse_windowed_core

    refuse_windowed_core("layers.0.self_attn", _model("llama").layers[0].self_attn.attn_core)
    with pytest.raises(ValueError, match="sliding_window"):
        refuse_windowed_core("layers.0.self_attn", _model("llama", sliding_window=4).layers[0].self_attn.attn_core)


@pytest.mark.parametrize("bad", [dict(sliding_window=0), dict(sink_tokens=1), dict(sliding_window=2, sink_tokens=-1), dict(full_attention_every=2),
                                 dict(sliding_window=2, full_attention_every=0), dict(embedding_scale=0.0)])
def test_refused_options(bad):
    for config in (LlamaConfig, OlmoConfig):
        with pytest.raises(ValueError):
            config(**{**SIZES, **bad})


def test_command_line(tmp_path):
    from maltos_b200.train.cli import _build_model, validate_args
    from maltos_b200.train.flags import parse_args_from

    recipe = tmp_path / "r.yaml"
    recipe.write_text("model: {type: llama, hidden_size: 64, num_heads: 4, num_layers: 2, intermediate_size: 128, vocab_size: 96, sliding_window: 8,\n"
                      "        sink_tokens: 2, full_attention_every: 2, embedding_scale: 8.0, post_block_norm: true, residual_scale: 0.5, residual_gate: true}\n"
                      "data: {seq_len: 32}\n")
    args = parse_args_from(["--config", str(recipe)], require_data=False)
    validate_args(args, 1)
    model = _build_model(args)
    assert [layer.self_attn.attn_core.window for layer in model.layers] == [8, None] and model.embed_tokens.scale == 8.0
    assert model.layers[0].post_feedforward_layernorm.gate is not None and model.layers[0].post_attention_layernorm.scale == 0.5
    args = parse_args_from(["--config", str(recipe), "--model", "olmo2", "--no-post-block-norm"], require_data=False)
    validate_args(args, 1)
    assert _build_model(args).layers[1].joined
    for extra, what in ((["--model", "olmo2"], "post-block-norm"), (["--model", "tiny", "--no-post-block-norm"], "sliding-window")):
        with pytest.raises(ValueError, match=what):
            validate_args(parse_args_from(["--config", str(recipe), *extra], require_data=False), 1)
    args = parse_args_from(["--config", str(recipe), "--cp-size", "2"], require_data=False)
    with pytest.raises(ValueError, match="sliding-window"):
        validate_args(args, 2)
    assert isinstance(args, argparse.Namespace)
