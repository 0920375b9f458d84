"""What a captured FusedMuon step holds and what it follows, on the CPU: the books of the capture, no launch."""
import pytest
import torch

from ofq_amd.optim import FusedMuon


def _captured(monkeypatch):
    p, v = torch.nn.Parameter(torch.zeros(3, 4)), torch.nn.Parameter(torch.zeros(3))
    opt = FusedMuon([{"params": [v], "use_muon": False}, {"params": [p]}], lr=0.1)
    opt.state[v]["step"] = torch.tensor(1.0)
    opt.begin_capture(torch.device("cpu"))
    opt._captured_hyper(opt.param_groups[0], [v])
    opt._capture_muon(opt.param_groups[1])
    stored = []

    class Lib:
        ofq_adamw_hyper_pack = staticmethod(lambda *a: 0)
        ofq_store_f32 = staticmethod(lambda *a: stored.append(a) or 0)
    from ofq_amd import ops
    monkeypatch.setattr(ops, "lib", lambda: Lib)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    return opt, v, stored


def test_a_replay_follows_the_learning_rate_and_the_decay(monkeypatch):
    opt, v, stored = _captured(monkeypatch)
    opt.param_groups[1]["lr"], opt.param_groups[1]["weight_decay"] = 0.05, 0.2
    opt.advance_for_replay()
    assert len(stored) == 1 and float(opt.state[v]["step"]) == 2


@pytest.mark.parametrize("name,value", [("momentum", 0.9), ("nesterov", False), ("ns_steps", 4), ("eps", 1e-6), ("adjust_lr_fn", "match_rms_adamw"),
                                        ("ns_coefficients", (1.5, -0.5, 0.0))])
def test_a_replay_refuses_what_the_captured_launches_cannot_follow(monkeypatch, name, value):
    """A momentum schedule, for one: the captured launches hold the old value.  Nothing has been advanced when it is refused."""
    opt, v, stored = _captured(monkeypatch)
    opt.param_groups[1][name] = value
    with pytest.raises(RuntimeError, match="capture"):
        opt.advance_for_replay()
    assert not stored and float(opt.state[v]["step"]) == 1
