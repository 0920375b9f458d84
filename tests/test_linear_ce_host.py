"""What linear_cross_entropy refuses, on the CPU: every refusal comes before a launch."""
import pytest
import torch

from ofq_amd.functional import linear_cross_entropy
from ofq_amd.quantization.utils import LinearCrossEntropy

X, W, Y = torch.randn(4, 8), torch.randn(5, 8), torch.tensor([0, 1, 2, -100])


@pytest.mark.parametrize("kw,error", [
    (dict(reduction="max"), ValueError), (dict(label_smoothing=-0.1), ValueError), (dict(label_smoothing=1.5), ValueError),
    (dict(label_smoothing=float("nan")), ValueError), (dict(weight=torch.randn(5, 9)), ValueError), (dict(weight=torch.randn(8)), ValueError),
    (dict(weight=torch.randn(0, 8)), ValueError), (dict(target=Y.int()), ValueError), (dict(target=Y[:3]), ValueError),
    (dict(target=torch.rand(4, 5)), ValueError), (dict(bias=torch.randn(4)), ValueError), (dict(bias=torch.randn(5, 1)), ValueError),
    (dict(input=X.double()), RuntimeError), (dict(input=X.half(), weight=W.half()), RuntimeError), (dict(input=X.bfloat16()), RuntimeError),
    (dict(bias=torch.randn(5).bfloat16()), RuntimeError), (dict(), RuntimeError),
])
def test_refusals(kw, error):
    args = dict(input=X, weight=W, target=Y)
    args.update(kw)
    with pytest.raises(error, match="linear_cross_entropy"):
        linear_cross_entropy(**args)


def test_module_has_the_functions_checks():
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        LinearCrossEntropy()(X, W, Y)


def test_entries_refuse_bad_arguments_on_the_host():
    from ofq_amd import _lib
    lib = _lib.load()
    assert lib.ofq_linear_ce_kept_bytes(0, 8, 5, 0, 1, 1) == 0 and lib.ofq_linear_ce_fwd_ws_bytes(4, 0, 5, 0) == 0
    assert lib.ofq_linear_ce_bwd_ws_bytes(4, 8, (1 << 24) + 1, 0, 1, 1) == 0
    # bf16 whose rows are whole chunks is used in place; anything else is packed
    kept = lambda *a: lib.ofq_linear_ce_kept_bytes(*a, 0)
    assert kept(64, 64, 1024, 1, 0) - kept(64, 64, 1024, 1, 1) == 1024 * 64 * 2 and kept(64, 63, 1024, 1, 1) == kept(64, 64, 1024, 1, 0)
    # logits up to 128 MB stay for the backward, more do not
    with_z = lambda *a: lib.ofq_linear_ce_kept_bytes(*a, 1)
    assert with_z(64, 256, 1024, 0, 1) - kept(64, 256, 1024, 0, 1) == 64 * 1024 * 4
    assert with_z(64, 64, 1024, 0, 1) == kept(64, 64, 1024, 0, 1)                # (a product over 64 is sooner done again)
    assert with_z(4096, 256, 16384, 0, 1) == kept(4096, 256, 16384, 0, 1) and with_z(4096, 256, 8192, 0, 1) > kept(4096, 256, 8192, 0, 1)
    none = [None] * 4
    assert lib.ofq_linear_ce_fwd(*none, 4, 8, 5, 0, 0, -100, 0.0, 1, 1, None, None, 0, None, 0, None) != 0
    assert lib.ofq_linear_ce_bwd(*[None] * 4, 0, 4, 8, 5, 0, 0, 0.0, 1, None, None, None, None, 0, None) != 0
