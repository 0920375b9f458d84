"""Which form a captured training step takes next to a process group, on the CPU: nothing is captured here."""
import os
from types import SimpleNamespace

import pytest
import torch
import torch.distributed as dist

from ofq_amd import engine


@pytest.fixture
def no_device_stream(monkeypatch):
    monkeypatch.setattr(torch.cuda, "Stream", lambda *a, **k: object())


def _step(dp, mode):
    opt = SimpleNamespace(advance_for_replay=lambda: None)
    return engine.GraphedTrainStep(torch.nn.Linear(2, 2), opt, loss_fn=lambda *a: None, dp=dp, mode=mode)


@pytest.mark.parametrize("mode", ["full", "segmented", "split"])
def test_collectives_are_never_captured(no_device_stream, mode):
    """A captured collective takes RCCL's stream into the capture while c10d's watchdog may still query events recorded on it."""
    synced = SimpleNamespace(sync=True, world=1)
    assert _step(synced, mode).mode == ("split" if mode == "split" else "segmented")
    for dp in (None, SimpleNamespace(sync=False, world=1)):
        assert _step(dp, mode).mode == "full"
    with pytest.raises(ValueError):
        _step(synced, "whole")


def test_capture_mode_next_to_a_live_process_group():
    """Event queries of c10d's watchdog count as errors of a capture in mode "global": with a group alive it is thread-local, with or without
    a DataParallel in the step."""
    assert engine._capture_error_mode() == "global"
    store = dist.HashStore()
    dist.init_process_group("gloo", store=store, rank=0, world_size=1)
    try:
        assert engine._capture_error_mode() == "thread_local"
    finally:
        dist.destroy_process_group()
    assert engine._capture_error_mode() == "global"
