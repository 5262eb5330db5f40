"""A token id outside a scaled embedding's table ends a training run (the kernels read it as zeros and record it)."""
import pytest
import torch

from maltos_b200.ops import _lib
from maltos_b200.runtime import MeshConfig, RuntimeCore
from maltos_b200.train.trainer import Trainer, TrainerConfig

pytestmark = pytest.mark.gpu


class _Loader:
    def __init__(self, bad_at):
        self.i, self.bad_at = 0, bad_at

    def next_batch(self, cp_rank=None):
        ids = torch.randint(0, 64, (2, 32), generator=torch.Generator().manual_seed(self.i))
        if self.i == self.bad_at:
            ids[1, 3] = 64
        self.i += 1
        return {"input_ids": ids, "labels": torch.zeros_like(ids)}

    def state_dict(self):
        return {"i": self.i}

    def load_state_dict(self, state):
        self.i = int(state["i"])


@pytest.mark.parametrize("bad_at", [None, 2])
def test_a_bad_token_id_ends_the_run(tmp_path, bad_at):
    from maltos_b200 import models as M

    torch.manual_seed(0)
    model = M.LlamaForCausalLM(M.LlamaConfig(vocab_size=64, hidden_size=128, intermediate_size=256, num_hidden_layers=1, num_attention_heads=2,
                                             num_key_value_heads=2, max_position_embeddings=32, embedding_scale=4.0, sliding_window=8))
    _lib.fetch_status(raise_on_error=False)
    runtime = RuntimeCore(model=model, mesh=MeshConfig(), device="cuda", dtype=torch.bfloat16, optimizer_factory=lambda p: torch.optim.SGD(p, lr=0.01))
    trainer = Trainer(runtime=runtime, dataloader=_Loader(bad_at), runtime_spec={"v": 1},
                      config=TrainerConfig(max_steps=4, checkpoint_every=1, checkpoint_dir=tmp_path))
    trainer.setup()
    if bad_at is None:
        trainer.fit()
    else:
        with pytest.raises(_lib.DeviceStatusError, match="index out of bounds.*detail 64"):
            trainer.fit()
    assert len(list(tmp_path.glob("step_*"))) == (4 if bad_at is None else bad_at)
