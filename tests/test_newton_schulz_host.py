"""What optim.orthogonalize, optim.FusedMuon and engine.make_optimizer refuse, and the groups of a model, on the CPU."""
import numpy as np
import pytest
import torch

from ofq_amd import _lib, ops
from ofq_amd.optim import FusedMuon, _check_newton_schulz, orthogonalize


@pytest.mark.parametrize("kw,error", [
    (dict(steps=-1), ValueError), (dict(steps=101), ValueError), (dict(steps=2.0), ValueError), (dict(eps=0.0), ValueError),
    (dict(eps=float("nan")), ValueError), (dict(coefficients=(1.0, 2.0)), ValueError), (dict(coefficients=(float("inf"), 0.0, 0.0)), ValueError),
    (dict(coefficients=(10.0, 5.0, 5.0)), ValueError), (dict(coefficients=(1.0, -60.0, 0.0)), ValueError), (dict(), RuntimeError),
])
def test_orthogonalize_refusals(kw, error):
    with pytest.raises(error, match="orthogonalize"):
        orthogonalize(torch.randn(4, 5), **kw)


@pytest.mark.parametrize("shape", [(), (3,), (2, 3, 4)])
def test_orthogonalize_takes_matrices_only(shape):
    with pytest.raises(ValueError, match="matrices only"):
        orthogonalize(torch.zeros(shape))


def test_usual_coefficients_are_in_range():
    for c in ((3.4445, -4.7750, 2.0315), (1.5, -0.5, 0.0), (2.0, -1.5, 0.5), (1.875, -1.25, 0.375)):
        _check_newton_schulz("x", c, 12, 1e-7)


@pytest.mark.parametrize("kw", [dict(lr=-1.0), dict(weight_decay=-1.0), dict(momentum=1.0), dict(betas=(1.0, 0.9)), dict(adamw_eps=-1.0),
                                dict(ns_steps=-1), dict(eps=0.0), dict(adjust_lr_fn="other"), dict(ns_coefficients=(9.0, 9.0, 9.0))])
def test_muon_hyper_parameters(kw):
    with pytest.raises(ValueError):
        FusedMuon([torch.nn.Parameter(torch.zeros(3, 4))], **kw)


def test_muon_groups_hold_matrices():
    v = torch.nn.Parameter(torch.zeros(3))
    with pytest.raises(ValueError, match="use_muon=False"):
        FusedMuon([v])
    opt = FusedMuon([{"params": [v], "use_muon": False}])
    with pytest.raises(ValueError):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(2, 2, 2))]})
    assert len(opt.param_groups) == 1
    p = torch.nn.Parameter(torch.zeros(2, 2))
    opt.add_param_group({"params": [p]})
    with pytest.raises(ValueError, match="twice"), pytest.warns(UserWarning):
        q = torch.nn.Parameter(torch.zeros(2, 2))
        opt.add_param_group({"params": [q, q]})
    opt.set_frozen(v, torch.ones(3))
    with pytest.raises(RuntimeError, match="freeze"):
        opt.set_frozen(p, torch.ones(2, 2))
    opt.set_frozen(p, None)
    with pytest.raises(RuntimeError, match="no captured step"):
        opt.advance_for_replay()


def test_muon_has_no_cpu_fallback():
    p = torch.nn.Parameter(torch.zeros(3, 4))
    opt = FusedMuon([p])
    p.grad = torch.ones_like(p)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        opt.step()


def test_make_optimizer_choices():
    from ofq_amd import engine
    from test_host_logic import _tiny
    model = _tiny()
    with pytest.raises(ValueError, match="adamw"):
        engine.make_optimizer(model, opt="sgd")
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        engine.make_optimizer(model, opt="muon")
    groups = engine.muon_param_groups(model, 0.05)
    names = {id(p): n for n, p in model.named_parameters()}
    got = [{names[id(p)] for p in g["params"]} for g in groups]
    assert got[0] and all(n.startswith("blocks.") and n.endswith(".weight") for n in got[0])
    assert set().union(*got) == {n for n, p in model.named_parameters() if p.requires_grad} and sum(map(len, got)) == len(set().union(*got))
    assert "head.weight" in got[2] and "patch_embed.proj.weight" in got[2] and "pos_embed" in got[1] | got[2]
    assert [g["weight_decay"] for g in groups] == [0.05, 0.0, 0.05]


def test_entry_refuses_bad_arguments_on_the_host():
    lib = _lib.load()
    t = np.zeros(2, dtype=ops.NS_ENTRY)
    assert lib.ofq_newton_schulz_entry_bytes() == ops.NS_ENTRY.itemsize
    assert lib.ofq_newton_schulz_ws_bytes(t.ctypes.data, 2) == 0                     # no rows
    t["rows"], t["cols"] = 64, 128
    # planes: two of X (two buffers) and one each of A and B, two 16-bit planes each; records and partial sums in front
    planes = 2 * 2 * (2 * 64 * 128 + 2 * 64 * 64) * 2
    assert planes < lib.ofq_newton_schulz_ws_bytes(t.ctypes.data, 2) <= planes + 2048
    args = (5, 3.4445, -4.775, 2.0315, 1e-7, 0.1, 0.0, 0.9, 0, None, None)
    assert lib.ofq_newton_schulz(t.ctypes.data, 2, 0, *args, None, 0, None) != 0     # no tensors
    assert lib.ofq_newton_schulz(None, 0, 0, *args, None, 0, None) != 0
    t["rows"] = (1 << 20) + 1
    assert lib.ofq_newton_schulz_ws_bytes(t.ctypes.data, 2) == 0
