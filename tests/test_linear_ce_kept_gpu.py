"""What the forward pass of linear_cross_entropy keeps where no gradient is to come."""
import pytest
import torch

from test_linear_ce_gpu import make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def lib():
    assert torch.cuda.is_available(), "the -m gpu tests need a HIP device"
    import ofq_amd.ops as ops
    ops.lib()


def kept_bytes(fn):
    """Size of what one forward pass keeps, as the library's caller allocated it."""
    from ofq_amd import ops
    seen, real = [], ops.linear_ce_fwd

    def spy(*a, **k):
        out = real(*a, **k)
        seen.append(out[1].numel())
        return out
    ops.linear_ce_fwd = spy
    try:
        loss = fn()
    finally:
        ops.linear_ce_fwd = real
    assert len(seen) == 1
    return seen[0], loss


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("T,D", [(3, 320), (300, 320), (300, 512)])
def test_without_gradients_nothing_is_kept_for_them(T, D, dtype):
    """Validation: weights that are parameters, under no_grad and inference_mode.  The logits are not kept, and the loss is the same bits.
    (A bf16 product over 320 is sooner done again than its logits are read: those are not kept for a backward either.)"""
    from ofq_amd import ops
    from ofq_amd.functional import linear_cross_entropy
    x, w, b, y = make(T, D, 9100, dtype)
    x, y = x.cuda(), y.cuda()
    w, b = torch.nn.Parameter(w.cuda()), torch.nn.Parameter(b.cuda())
    trained, loss = kept_bytes(lambda: linear_cross_entropy(x, w, y, bias=b))
    lib, b16 = ops.lib(), int(dtype == "bf16")
    assert trained == lib.ofq_linear_ce_kept_bytes(T, D, 9100, b16, 1, 1)
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            size, alone = kept_bytes(lambda: linear_cross_entropy(x, w, y, bias=b))
        assert size == lib.ofq_linear_ce_kept_bytes(T, D, 9100, b16, 1, 0)
        assert trained - size >= (T * 9100 * 4 if T == 3 or dtype == "fp32" or D == 512 else 0)
        assert not alone.requires_grad and torch.equal(alone, loss.detach())
