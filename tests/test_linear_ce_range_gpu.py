"""linear_cross_entropy in fp32 where an operand lies near the ends of fp32's range."""
import pytest
import torch

from test_linear_ce_gpu import GRAD_TOL, LOSS_TOL, call, make, reference

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def lib():
    assert torch.cuda.is_available(), "the -m gpu tests need a HIP device"
    import ofq_amd.ops as ops
    ops.lib()


@pytest.mark.parametrize("sx,sw", [(1e36, 1e-36), (1e35, 1e-35), (1e-35, 1e35), (2e37, 1e-37), (1e-36, 1e36), (1e36, 1e-37), (1e-20, 1e-20), (1e36, 1e-10)])
@pytest.mark.parametrize("T,V", [(6, 100), (40, 100)])
def test_operands_near_the_ends_of_the_range(T, V, sx, sw):
    """The power of two that brings a tensor to its planes' scale is taken off again wherever the result is a float: a loss and gradients that
    are finite in 64 bits (and below 3e38) are finite and right.  Elements under 2^-126 are steps of 2^-149; an operand of 1e-37 has
    elements there itself, which enter as they are."""
    x, w, b, y = make(T, 64, V, "fp32")
    x, w = x * sx, w * sw
    if sx * sw > 1:                      # logits of 1e26: the largest alone counts, its gradients are zeros and ones
        b = None
    got, want = call(x, w, b, y), reference(x, w, b, y)
    zmax = float((x.double() @ w.double().t()).abs().max()) + 2
    assert abs(float(got[0]) - float(want[0])) <= LOSS_TOL * zmax
    for a, c in zip(got[1:], want[1:]):
        assert bool(torch.isfinite(a).all())
        assert float((a.double().cpu() - c).norm()) <= GRAD_TOL["fp32"] * float(c.norm()) + 2.0 ** -149 * T * c.numel() ** 0.5
