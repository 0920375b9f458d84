"""orthogonalize and FusedMuon where max(|U|_F, eps) lies at the lower end of fp32's range."""
import pytest
import torch

from test_newton_schulz_gpu import TOL32, definition, far, matrix

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def lib():
    assert torch.cuda.is_available(), "the -m gpu tests need a HIP device"
    import ofq_amd.ops as ops
    ops.lib()


@pytest.mark.parametrize("eps", [1e-40, 1e-44, 1e-36, 1e-7])
@pytest.mark.parametrize("shape", [(64, 64), (100, 80), (70, 200)])
def test_a_zero_matrix_stays_zero(shape, eps):
    from ofq_amd.optim import orthogonalize
    for dtype in (torch.float32, torch.bfloat16):
        out = orthogonalize(torch.zeros(shape, dtype=dtype, device="cuda"), eps=eps)
        assert not bool(out.any())


@pytest.mark.parametrize("scale", [1e-37, 1e-38, 3e-36, 1e33, 1e36])
def test_norms_at_the_ends_of_the_range(scale):
    """100 x 80 of them have about 90 times that norm, with zero padding in both directions.  Elements under 2^-126 enter as they are."""
    from ofq_amd.optim import orthogonalize
    g = matrix(100, 80) * scale
    assert far(orthogonalize(g.cuda(), eps=1e-40), definition(g, eps=1e-40)) <= TOL32


def test_muon_leaves_a_parameter_without_a_gradient_value_finite():
    """Gradient and momentum all zero: the update is zero, the parameter only decays."""
    from ofq_amd.optim import FusedMuon
    p = torch.nn.Parameter(matrix(96, 70).cuda())
    before = p.detach().clone()
    opt = FusedMuon([p], lr=0.1, weight_decay=0.5, eps=1e-40)
    p.grad = torch.zeros_like(p)
    opt.step()
    # p (1 - lr wd): three roundings of 2^-24
    assert float((p.detach() - 0.95 * before).abs().max()) <= 3 * 2.0 ** -24 * float(before.abs().max())
