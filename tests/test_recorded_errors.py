"""What kernels record instead of trapping stops a training run: the trainer asks after every optimizer step. CPU."""
import pytest

from maltos_b200.ops import _lib
from tests.test_control_plane_cpu import _trainer


def test_the_trainer_asks_after_every_step_and_saves_no_bad_one(tmp_path, monkeypatch):
    asked = []

    def recorded(device):
        asked.append(str(device))
        if len(asked) == 4:
            raise _lib.DeviceStatusError("kernel status 4 (index out of bounds)")

    monkeypatch.setattr(_lib, "raise_recorded_errors", recorded)
    trainer, _, loader = _trainer(tmp_path, max_steps=6)                # a checkpoint every second step
    with pytest.raises(_lib.DeviceStatusError):
        trainer.fit()
    assert asked == ["cpu"] * 4 and loader.closed
    assert [p.name for p in sorted(tmp_path.glob("step_*"))] == ["step_00000002"]


def test_nothing_to_ask_on_the_cpu(monkeypatch):
    monkeypatch.setattr(_lib, "fetch_status", lambda: pytest.fail("no device to ask"))
    _lib.raise_recorded_errors("cpu")
