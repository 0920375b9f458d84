"""linear_cross_entropy with reduction="none": incoming gradients of unlike and of tiny size, each row of dx held by its own norm."""
import pytest
import torch

from test_linear_ce_gpu import DTYPES, GRAD_TOL, call, far, make, reference

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def lib():
    assert torch.cuda.is_available(), "the -m gpu tests need a HIP device"
    import ofq_amd.ops as ops
    ops.lib()


def decades(T, low, high, seed=3):
    """Weights of both signs, 10^low to 10^high, the ends among them, a zero too where there is room for it."""
    g = torch.Generator().manual_seed(seed)
    w = 10.0 ** (low + (high - low) * torch.rand(T, generator=g)) * (torch.randint(0, 2, (T,), generator=g) * 2 - 1)
    w[0], w[-1] = 10.0 ** low, 10.0 ** high
    if T > 4:
        w[2] = 0.0
    return w


def rows_are_right(dx, x, w, b, y, grad, smoothing, dtype):
    """Row t of dx is g_t sum_v G_tv W_v.  fp32: G is off by 2^-22 of 1 + |x| |w| (the logit's own error) + |z - lse| / 2 (the exponential's
    argument) + 4 (two planes each of G and W, the product of the low planes, the sums), of its own size; the target's 1 - p cancels, so its
    G counts as 1.  bf16: G and the result are rounded to 2^-8 of themselves (half steps) on top of that."""
    x, w = x.double(), w.double()
    live = y != -100
    z = x @ w.t() + (0.0 if b is None else b.double())
    lse = torch.logsumexp(z, 1, keepdim=True)
    G = (z - lse).exp() - smoothing / w.shape[0]
    size = G.abs() + smoothing / w.shape[0]
    at = torch.arange(len(y))[live]
    G[at, y[live]] -= 1 - smoothing
    size[at, y[live]] = 1.0
    c = 2.0 ** -22 * (5 + (x.abs() @ w.abs().t()).max(1).values + (z - lse).abs().max(1).values / 2) + (2.0 ** -7 if dtype == "bf16" else 0.0)
    want = torch.where(live, grad.double(), 0.0)[:, None] * (G @ w)
    bound = grad.double().abs() * c * (size @ w.norm(dim=1)) + (2.0 ** -149 if dtype == "fp32" else 2.0 ** -133) * w.shape[1]
    err = (dx.detach().double().cpu() - want).norm(dim=1)
    assert bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("T,D,V", [(3, 64, 200), (9, 64, 5000), (140, 96, 333), (300, 320, 9100), (700, 72, 300), (1025, 192, 4100), (4200, 64, 9001)])
def test_weights_over_twelve_decades(T, D, V, dtype):
    """Every tile form, dx in one and in several parts, one piece of the vocabulary and two, few rows."""
    x, w, b, y = make(T, D, V, dtype, ignored=0.1 if T > 4 else 0.0)
    grad = decades(T, -12, 0)
    got = call(x, w, b, y, 0.1, "none", grad)
    want = reference(x, w, b, y, 0.1, "none", grad)
    rows_are_right(got[1], x, w, b, y, grad, 0.1, dtype)
    for k in (1, 2, 3):
        assert got[k].dtype == DTYPES[dtype] and far(got[k], want[k]) <= GRAD_TOL[dtype]
    dead = (y == -100) | (grad == 0)
    assert not bool(got[1].cpu()[dead].any())


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("low,high", [(-36, -36), (-35, -35), (-37.5, -36.5), (-37.8, -37.2), (-36, 0), (20, 32), (20, 37.3)])
@pytest.mark.parametrize("T,D,V", [(3, 64, 300), (5, 64, 300), (40, 64, 300), (300, 320, 9100)])
def test_tiny_and_huge_weights(T, D, V, low, high, dtype):
    """A gradient that is finite stays so, whatever the largest incoming one is.  The last places of an element under 2^-126 are steps of
    2^-149 (bf16: 2^-133): one half for each of the sums that go into it."""
    x, w, b, y = make(T, D, V, dtype)
    grad = decades(T, low, high)
    step = 2.0 ** -149 if dtype == "fp32" else 2.0 ** -133
    got = call(x, w, b, y, 0.0, "none", grad)
    want = reference(x, w, b, y, 0.0, "none", grad)
    assert all(bool(torch.isfinite(t).all()) for t in got)
    rows_are_right(got[1], x, w, b, y, grad, 0.0, dtype)
    for k in (1, 2, 3):
        floor = step * T * want[k].numel() ** 0.5
        assert float((got[k].double().cpu() - want[k]).norm()) <= GRAD_TOL[dtype] * float(want[k].norm()) + floor


@pytest.mark.parametrize("reduction", ["sum", "mean"])
@pytest.mark.parametrize("grad", [1e-36, 1e-34, 1e30])
def test_tiny_and_huge_incoming_gradients(grad, reduction):
    x, w, b, y = make(40, 64, 300, "fp32")
    got = call(x, w, b, y, 0.0, reduction, grad)
    want = reference(x, w, b, y, 0.0, reduction, grad)
    for k in (1, 2, 3):
        floor = 2.0 ** -149 * 40 * want[k].numel() ** 0.5
        # (grad / n is one float of its own: 2^-149 of it where it lies under 2^-126)
        own = 2.0 ** -149 / (grad / 40) if reduction == "mean" else 0.0
        assert float((got[k].double().cpu() - want[k]).norm()) <= (GRAD_TOL["fp32"] + own) * float(want[k].norm()) + floor


def test_large_weights_on_small_rows():
    """What counts for dW is a row's weight times the row: the largest weights on the smallest rows, over eight decades each way."""
    x, w, b, y = make(200, 96, 400, "fp32")
    size = 10.0 ** torch.linspace(-4, 0, 200)
    x = x * size[:, None]
    grad = 1e-3 / size ** 2
    got = call(x, w, b, y, 0.0, "none", grad)
    want = reference(x, w, b, y, 0.0, "none", grad)
    for k in (1, 2, 3):
        assert far(got[k], want[k]) <= GRAD_TOL["fp32"]
    rows_are_right(got[1], x, w, b, y, grad, 0.0, "fp32")


def test_a_weight_that_is_no_number_stays_in_its_row():
    """dx of the other rows is what it is without that row."""
    x, w, b, y = make(100, 64, 300, "fp32")
    grad = torch.rand(100, generator=torch.Generator().manual_seed(1)) + 0.5
    for bad in (float("nan"), float("inf")):
        g = grad.clone()
        g[17] = bad
        dx = call(x, w, b, y, 0.0, "none", g)[1].cpu()
        keep = torch.arange(100) != 17
        assert not bool(torch.isfinite(dx[17]).any())
        x2, y2, g2 = x[keep], y[keep], grad[keep]
        rows_are_right(dx[keep], x2, w, b, y2, g2, 0.0, "fp32")


def test_weighted_rows_twice_and_replayed():
    """The gradients may be taken twice, and a captured pass follows the weights in its static buffer."""
    from ofq_amd.functional import linear_cross_entropy
    x, w, b, y = make(150, 96, 300, "fp32", ignored=0.2)
    xs, ws, bs = (t.cuda().requires_grad_() for t in (x, w, b))
    ys, g = y.cuda(), decades(150, -6, 0).cuda()
    rows = linear_cross_entropy(xs, ws, ys, bias=bs, reduction="none")
    one = torch.autograd.grad(rows, (xs, ws, bs), g, retain_graph=True)
    two = torch.autograd.grad(rows, (xs, ws, bs), g)
    assert all(torch.equal(a, c) for a, c in zip(one, two))
    del rows, one, two

    def step():
        rows = linear_cross_entropy(xs, ws, ys, bias=bs, reduction="none")
        return torch.autograd.grad(rows, (xs, ws, bs), g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (5, 6, 7):
        h = decades(150, -9, 3, seed)
        g.copy_(h)
        graph.replay()
        eager = call(x, w, b, y, 0.0, "none", h)[1:]
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, eager))
