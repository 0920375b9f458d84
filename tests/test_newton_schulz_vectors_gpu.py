"""orthogonalize and FusedMuon on vectors (matrices of one row or one column), alone and among others: their chain is a scalar's."""
import math

import numpy as np
import pytest
import torch

from test_newton_schulz_gpu import NS, TOL16, definition, far, matrix, muon_reference, tol

pytestmark = pytest.mark.gpu
AS_FLOATS = tuple(float(np.float32(c)) for c in NS)        # as the entry takes the coefficients


@pytest.fixture(scope="module", autouse=True)
def lib():
    assert torch.cuda.is_available(), "the -m gpu tests need a HIP device"
    import ofq_amd.ops as ops
    ops.lib()


VECTORS = [(1, 1), (1, 2), (3, 1), (1, 63), (64, 1), (1, 65), (129, 1), (1, 1000), (5000, 1), (1, 300001)]


@pytest.mark.parametrize("shape", VECTORS)
@pytest.mark.parametrize("steps", [0, 1, 5, 8])
def test_a_vector_is_off_by_its_last_rounding(shape, steps):
    """64 bits up to the result: half a step of fp32 (2^-24), or of bf16 (2^-8)."""
    from ofq_amd.optim import orthogonalize
    g = matrix(*shape)
    want = definition(g, steps, AS_FLOATS)
    out = orthogonalize(g.cuda(), steps=steps).double().cpu()
    assert bool(((out - want).abs() <= 2.0 ** -24 * (1 + 2.0 ** -20) * want.abs()).all())
    h = g.bfloat16()
    want = definition(h, steps, AS_FLOATS)
    out = orthogonalize(h.cuda(), steps=steps).double().cpu()
    assert bool(((out - want).abs() <= 2.0 ** -8 * want.abs()).all())


def test_vectors_among_matrices():
    """In any place of the list, the longest and the shortest of it; matrices keep their own precision; vectors alone; the same bits twice."""
    from ofq_amd.optim import orthogonalize
    shapes = [(65, 1), (100, 80), (1, 129), (1, 9000), (64, 64), (1, 1), (200, 65), (7, 1)]
    mats = [matrix(*s, seed=i) for i, s in enumerate(shapes)]
    dev = [m.cuda() for m in mats]
    outs = orthogonalize(dev)
    for m, o in zip(mats, outs):
        assert far(o, definition(m)) <= (tol(m.shape) if min(m.shape) > 1 else 2.0 ** -22)
    assert all(torch.equal(a, b) for a, b in zip(outs, orthogonalize(dev)))
    alone = [k for k, m in enumerate(mats) if min(m.shape) == 1]
    for k, o in zip(alone, orthogonalize([dev[k] for k in alone])):
        assert torch.equal(o, outs[k])
    half = orthogonalize([m.bfloat16() for m in dev])
    for m, o in zip(mats, half):
        assert far(o, definition(m.bfloat16())) <= TOL16


def test_zero_nan_and_tiny_vectors():
    from ofq_amd.optim import orthogonalize
    v = [torch.zeros(1, 70), matrix(90, 1), matrix(1, 40, seed=2) * 1e-30, torch.zeros(5, 1), matrix(1, 33, seed=3) * 1e36]
    v[1][5, 0] = math.nan
    outs = orthogonalize([t.cuda() for t in v], eps=1e-40)
    assert not bool(outs[0].any()) and not bool(outs[3].any()) and not bool(torch.isfinite(outs[1]).any())
    for k in (2, 4):
        assert far(outs[k], definition(v[k], eps=1e-40)) <= 2.0 ** -22
    small = orthogonalize(v[2].cuda())                   # below eps: divided by eps, and grown by a^5 at most
    assert float(small.norm()) <= 3.5 ** 5 * 1e-29 / 1e-7


@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_on_vectors(nesterov):
    from ofq_amd.optim import FusedMuon
    shapes = [(1, 300), (65, 1), (96, 64), (1, 1)]
    ps = [torch.nn.Parameter(0.05 * matrix(*s, seed=9).cuda()) for s in shapes]
    opt = FusedMuon(ps, lr=0.02, momentum=0.95, weight_decay=0.1, nesterov=nesterov)
    want = [(p.detach().cpu().double(), torch.zeros(p.shape, dtype=torch.float64)) for p in ps]
    for t in range(3):
        for i, p in enumerate(ps):
            p.grad = matrix(*p.shape, seed=100 * t + i, rank=8).cuda()
            want[i] = muon_reference(*want[i], p.grad.cpu(), nesterov=nesterov)
        opt.step()
    for p, (w, m) in zip(ps, want):
        # momentum: a rounding or two a step; the update is lr sqrt(rows / columns) times a unit vector, its direction as good as the momentum's
        assert far(opt.state[p]["momentum_buffer"], m) <= 8 * 2.0 ** -24
        update = 3 * 0.02 * math.sqrt(max(1.0, p.shape[0] / p.shape[1])) * math.sqrt(min(p.shape)) * 1.3
        assert float((p.detach().cpu().double() - w).norm()) <= (tol(p.shape) if min(p.shape) > 1 else 2.0 ** -20) * update + 8 * 2.0 ** -24 * float(w.norm())
