"""Options of the decoder block outlive a run: they stand beside the runtime spec, a resume without them is refused, and conversions
keep the tensors that they made. CPU."""
import json

import pytest
import torch
from safetensors import safe_open

from maltos_b200.state.checkpoint import load_model_options, save_model_options, save_runtime_spec, save_sharded_checkpoint
from maltos_b200.tools import convert_checkpoint
from maltos_b200.train import cli
from maltos_b200.train.flags import apply_model_options, build_model_options, build_runtime_spec, parse_args_from, parse_runtime_spec_args
from tests.test_control_plane_cpu import _Loader, _runtime

SIZES = ["--model", "llama", "--dim", "64", "--n-heads", "4", "--n-layers", "2", "--hidden-size", "128", "--vocab-size", "96", "--seq-len", "32",
         "--precision", "fp32"]
OPTIONS = ["--sliding-window", "8", "--sink-tokens", "2", "--embedding-scale", "8.0", "--post-block-norm", "--residual-scale", "0.5", "--residual-gate"]


@pytest.fixture(autouse=True)
def _gradients():
    with torch.enable_grad():          # the conversion's command line turns them off for its process
        yield
    torch.set_grad_enabled(True)


def _args(*extra):
    return parse_args_from([*SIZES, *extra], require_data=False)


def _checkpoint(root, args, options=True):
    model = cli._build_model(args)
    runtime = cli._build_runtime(args, model, torch.device("cpu"))
    runtime.setup()
    save_runtime_spec(root, build_runtime_spec(args))
    if options:
        save_model_options(root, build_model_options(args))
    save_sharded_checkpoint(runtime.state_manager, root / "step_00000001")
    runtime.close()
    return dict(model.state_dict())


def _logical(path):
    out = {}
    for f in path.glob("*.safetensors"):
        with safe_open(f, "pt") as s:
            out |= {k: s.get_tensor(k) for k in s.keys()}
    return out


def test_options_of_the_command_line():
    assert build_model_options(_args()) == {}
    args = _args(*OPTIONS)
    options = build_model_options(args)
    assert options == dict(sliding_window=8, sink_tokens=2, embedding_scale=8.0, post_block_norm=True, residual_scale=0.5, residual_gate=True)
    again = apply_model_options(parse_runtime_spec_args(json.loads(json.dumps(build_runtime_spec(args)))), json.loads(json.dumps(options)))
    assert build_model_options(again) == options
    with pytest.raises(ValueError, match="unknown"):
        apply_model_options(_args(), {"window": 3})


def test_one_root_one_set_of_options(tmp_path):
    save_model_options(tmp_path, {})
    assert load_model_options(tmp_path) is None and not list(tmp_path.iterdir())
    save_model_options(tmp_path, {"sliding_window": 8})
    save_model_options(tmp_path, {"sliding_window": 8})
    assert load_model_options(tmp_path / "step_00000001") == {"sliding_window": 8}
    for other in ({}, {"sliding_window": 9}):
        with pytest.raises(ValueError, match="different"):
            save_model_options(tmp_path, other)


def test_conversion_keeps_what_the_options_made(tmp_path):
    args = _args(*OPTIONS)
    state = _checkpoint(tmp_path / "run", args)
    convert_checkpoint.main(["runtime-to-logical", "--checkpoint", str(tmp_path / "run" / "step_00000001"), "--output", str(tmp_path / "logical")])
    logical = _logical(tmp_path / "logical")
    assert set(logical) == set(state) and any("after_weight" in k for k in logical) and any(k.endswith("gate") for k in logical)
    assert all(torch.equal(logical[k], state[k]) for k in state)
    recipe = tmp_path / "recipe.yaml"
    recipe.write_text("model: {type: llama}\n")
    convert_checkpoint.main(["logical-to-runtime", "--config", str(recipe), "--checkpoint", str(tmp_path / "logical"), "--output", str(tmp_path / "back"),
                             "--", *SIZES, *OPTIONS])
    assert load_model_options(tmp_path / "back" / "step_00000000") == build_model_options(args)


def test_conversion_without_the_record_is_refused(tmp_path):
    _checkpoint(tmp_path, _args(*OPTIONS), options=False)
    with pytest.raises(ValueError, match="model_options.json"):
        convert_checkpoint.main(["runtime-to-logical", "--checkpoint", str(tmp_path / "step_00000001"), "--output", str(tmp_path / "logical")])


def test_a_resume_needs_the_same_options(tmp_path):
    from maltos_b200.train.trainer import Trainer, TrainerConfig

    def trainer(options, root, steps, resume=None, weights_only=False):
        config = TrainerConfig(max_steps=steps, checkpoint_every=2, checkpoint_dir=root, resume_from=resume, load_weights_only=weights_only)
        return Trainer(runtime=_runtime(), dataloader=_Loader(), config=config, runtime_spec={"version": 1}, model_options=options)

    first = trainer({"sliding_window": 8}, tmp_path / "a", 2)
    first.setup()
    first.fit()
    last = tmp_path / "a" / "step_00000002"
    for options in ({}, {"sliding_window": 8, "sink_tokens": 1}):
        with pytest.raises(ValueError, match="--sliding-window 8"):
            trainer(options, tmp_path / "a", 4, last).setup()
    trainer({}, tmp_path / "b", 2, last, weights_only=True).setup()          # other options over the same weights, in a root of its own
    again = trainer({"sliding_window": 8}, tmp_path / "a", 4, last)
    again.setup()
    again.fit()
    assert again.runtime.state.step_context.step == 4
    plain = trainer({}, tmp_path / "c", 2)
    plain.setup()
    plain.fit()
    assert not (tmp_path / "c" / "model_options.json").exists()
    trainer({"sliding_window": 8}, tmp_path / "c", 4, tmp_path / "c" / "step_00000002").setup()   # nothing recorded: taken at its word
