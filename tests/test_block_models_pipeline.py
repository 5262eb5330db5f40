"""The decoder-block options across pipeline stages: which layers have a window follows the layer's place in the whole model, and every
kind of parameter gets its gradient. CPU."""
import pytest
import torch

from tests.dist_utils import run_distributed
from tests.test_block_models import OPTIONS, _ids, _model


def _worker(rank, world, kind, schedule, options):
    import maltos_b200  # noqa: F401
    from maltos_b200.parallel import ParallelPlan, PipelineScheduleConfig
    from maltos_b200.runtime import MeshConfig, RuntimeCore
    from maltos_b200.runtime.plugins.pp import PipelineParallelPlugin

    ids = _ids()
    rt = RuntimeCore(model=_model(kind, **options), mesh=MeshConfig(pp=world), plan=ParallelPlan(pp_schedule=PipelineScheduleConfig(microbatches=2)),
                     plugins=[PipelineParallelPlugin(schedule=schedule)], optimizer_factory=lambda p: torch.optim.SGD(p, lr=0.1))
    rt.setup()
    losses = []
    for _ in range(3):
        rt.run_step({"input_ids": ids, "labels": ids.roll(-1, 1)})
        rt.step_optimizer()
        losses.append(rt.collect_metrics()["loss"])
    rt.close()
    return losses


@pytest.mark.parametrize("kind,schedule", [("llama", "afab"), ("llama", "1f1b"), ("olmo", "1f1b")])
def test_pipeline_stages_match_a_single_process(kind, schedule):
    options = dict(OPTIONS, num_hidden_layers=4, full_attention_every=3, **({"post_block_norm": True} if kind == "llama" else {}))
    model, ids = _model(kind, **options), _ids()
    optimizer = torch.optim.SGD(model.parameters(), lr=0.1)
    want = []
    for _ in range(3):
        loss = model({"input_ids": ids, "labels": ids.roll(-1, 1)})
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        want.append(loss.item())
    for losses in run_distributed(_worker, 2, kind, schedule, options):
        # fp32 sums in another order; the later losses have steps of every gradient behind them
        assert all(abs(a - b) < 5e-5 for a, b in zip(losses, want)), (losses, want)
