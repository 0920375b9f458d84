"""The input-gradient GEMM (ofq_qgemm_bf16s_nt) on rows shorter than its k-step: what lies behind an operand's last row is NaN here,
so a product that reads it shows it.  K = 8 is the patch embedding of an eight-channel stem."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "the -m gpu tests need a HIP device"
    import ofq_amd.ops as ops
    ops.lib()
    return ops


def _tailed(t, fill):
    """A copy of t at the head of a larger allocation that holds `fill` behind it."""
    buf = torch.full((t.numel() + 256,), fill, dtype=t.dtype, device="cuda")
    buf[:t.numel()] = t.reshape(-1)
    return buf[:t.numel()].view(t.shape)


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("scale", [True, False])
@pytest.mark.parametrize("M,N,K", [(196, 768, 8), (1, 384, 16), (130, 300, 24), (196, 100, 8), (257, 768, 40)])
def test_short_rows_read_nothing_behind_the_operands(ops, M, N, K, scale, f16):
    g = torch.Generator().manual_seed(M + N + K)
    A = torch.randn(M, K, generator=g)
    B = torch.randint(-127, 128, (N, K), generator=g).float()
    s = torch.rand(K, generator=g) + 0.5
    ref = (A.double() * (s.double() if scale else 1.0)) @ B.double().t()
    a = _tailed(A.cuda(), float("nan"))
    b = _tailed(B.cuda().to(torch.float16 if f16 else torch.bfloat16), float("nan"))
    ks = _tailed(s.cuda(), float("nan")) if scale else None
    out = ops.qgemm_bf16s_nt(a, b, ks, 1.0, amax=ops.amax_for(a) if f16 else None)
    # two fp16 planes: 2^-22 of the largest |A s| per element at most, over K products with codes of up to 127; the three bf16 planes
    # and the fp32 accumulation (K + 2 roundings of 2^-24 of the largest partial sum) lie below that
    tol = float((A.abs() * (s if scale else 1.0)).max()) * 127 * K * 2.0 ** -21
    assert float((out.double().cpu() - ref).abs().max()) <= tol
