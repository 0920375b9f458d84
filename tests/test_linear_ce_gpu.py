"""functional.linear_cross_entropy, LinearCrossEntropy and LSQ_QLinear4head.loss against the definition in 64 bits."""
import math

import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
# Norm of the error over the norm of the result.
#   fp32: an operand in two fp16 planes is off by 2^-22 of itself at most, the dropped product of the two low planes by 2^-22, an fp32
#   accumulation of n MFMAs by about sqrt(n) 2^-24; __expf by 2^-22 (1 + |z - lse| / 4) for the differences that carry weight: together
#   below 16 steps of 2^-22.
#   bf16: G and the result are rounded once each, 2^-9 rms of at most 2^-8 each; twice that.
GRAD_TOL = {"fp32": 16 * 2.0 ** -22, "bf16": 4 * 2.0 ** -8}
LOSS_TOL = 16 * 2.0 ** -22                 # of the largest |lse| or |logit| that goes into it; exact products for bf16 inputs


@pytest.fixture(scope="module", autouse=True)
def lib():
    assert torch.cuda.is_available(), "the -m gpu tests need a HIP device"
    import ofq_amd.ops as ops
    ops.lib()


def make(T, D, V, dtype, bias=True, seed=0, ignored=0.0):
    g = torch.Generator().manual_seed(seed + 7 * T + D + V)
    x = torch.randn(T, D, generator=g)
    w = torch.randn(V, D, generator=g) * (1.5 / math.sqrt(D))
    b = torch.randn(V, generator=g) * 0.5 if bias else None
    y = torch.randint(0, V, (T,), generator=g)
    if ignored:
        y[torch.rand(T, generator=g) < ignored] = -100
    dt = DTYPES[dtype]
    return x.to(dt), w.to(dt), None if b is None else b.to(dt), y


def reference(x, w, b, y, smoothing=0.0, reduction="mean", grad=None, ignore=-100):
    """Loss and gradients from the formulas, in 64 bits on the CPU; ignored rows are left out before anything is computed."""
    x, w = x.double(), w.double()
    T, V = y.numel(), w.shape[0]
    live = (y != ignore).nonzero().squeeze(1)
    xl, yl = x[live], y[live]
    z = xl @ w.t() + (0.0 if b is None else b.double())
    lse = torch.logsumexp(z, 1, keepdim=True)
    want = torch.full_like(z, smoothing / V)
    want[torch.arange(len(live)), yl] += 1.0 - smoothing
    rows = torch.zeros(T, dtype=torch.float64)
    rows[live] = lse.squeeze(1) - (1 - smoothing) * z.gather(1, yl[:, None]).squeeze(1) - (smoothing * z.mean(1) if smoothing else 0.0)
    if reduction == "none":
        loss, wt = rows, grad.double()[live]
    elif reduction == "sum":
        loss, wt = rows.sum(), torch.full((len(live),), float(grad) if grad is not None else 1.0, dtype=torch.float64)
    else:
        n = max(len(live), 1)
        loss, wt = rows.sum() / len(live) if len(live) else torch.tensor(math.nan), \
            torch.full((len(live),), (float(grad) if grad is not None else 1.0) / n, dtype=torch.float64)
    G = ((z - lse).exp() - want) * wt[:, None]
    dx = torch.zeros_like(x)
    dx[live] = G @ w
    return loss, dx, G.t() @ xl, G.sum(0)


def call(x, w, b, y, smoothing=0.0, reduction="mean", grad=None, ignore=-100):
    from ofq_amd.functional import linear_cross_entropy
    xs, ws = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    bs = None if b is None else b.cuda().requires_grad_()
    loss = linear_cross_entropy(xs, ws, y.cuda(), bias=bs, ignore_index=ignore, label_smoothing=smoothing, reduction=reduction)
    leaves = [xs, ws] + ([] if b is None else [bs])
    g = None if grad is None else torch.as_tensor(grad, dtype=torch.float32).cuda()
    return (loss,) + torch.autograd.grad(loss, leaves, g)


def far(a, b):
    a, b = a.detach().double().cpu(), b.double()
    assert a.shape == b.shape
    n = float(b.norm())
    return float((a - b).norm()) / n if n else float((a - b).norm())


def check(got, want, dtype, zmax):
    assert got[0].dtype == torch.float32
    assert float((got[0].detach().double().cpu() - want[0]).abs().max()) <= LOSS_TOL * max(zmax, 1.0)
    for a, b in zip(got[1:], want[1:]):
        assert a.dtype == DTYPES[dtype]
        assert far(a, b) <= GRAD_TOL[dtype]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("T,D,V", [(1, 1, 1), (1, 64, 2), (1, 33, 129), (2, 7, 3), (63, 64, 127), (64, 128, 128), (65, 65, 129), (127, 100, 517),
                                   (128, 384, 1000), (129, 192, 1000), (257, 31, 300), (300, 256, 2049), (513, 72, 4100)])
def test_loss_and_gradients(T, D, V, dtype):
    x, w, b, y = make(T, D, V, dtype)
    zmax = float((x.double() @ w.double().t()).abs().max()) + 2
    check(call(x, w, b, y), reference(x, w, b, y), dtype, zmax)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("smoothing", [0.0, 0.1, 1.0])
def test_reductions_smoothing_bias_and_ignored_rows(dtype, bias, reduction, smoothing):
    x, w, b, y = make(140, 96, 333, dtype, bias=bias, ignored=0.3)
    grad = {"mean": -3.0, "sum": 0.125, "none": torch.linspace(-1.0, 2.0, 140)}[reduction]
    zmax = 140 * (float((x.double() @ w.double().t()).abs().max()) + 2) if reduction == "sum" else 16.0
    check(call(x, w, b, y, smoothing, reduction, grad), reference(x, w, b, y, smoothing, reduction, grad), dtype, zmax)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_many_pieces_of_the_vocabulary(dtype):
    """T large enough for the vocabulary to be cut: 8192 rows of two planes leave pieces of 4096 columns."""
    T, D, V = 8192, 64, 9001
    x, w, b, y = make(T, D, V, dtype, ignored=0.1)
    got = call(x, w, b, y, 0.05)
    want = reference(x, w, b, y, 0.05)
    check(got, want, dtype, 16.0)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("ignored", [False, True])
@pytest.mark.parametrize("T,D,V", [(1, 64, 2), (1, 4160, 300), (2, 128, 5000), (3, 511, 777), (4, 2048, 1030), (4, 8192, 65), (5, 516, 777), (7, 33, 64),
                                   (8, 1000, 129), (8, 4100, 500), (9, 512, 777)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_few_rows(T, D, V, ignored, reduction, dtype):
    """Up to eight rows (bf16: four) take the logits and the gradients in one pass over the weights each: rows of whole 16 bytes and others, columns beyond
    4096, vocabularies smaller than the grid, rows that do not count."""
    x, w, b, y = make(T, D, V, dtype)
    if ignored and T > 1:
        y[T // 2] = -100
    grad = torch.linspace(-1.0, 2.0, T) if reduction == "none" else None
    zmax = float((x.double() @ w.double().t()).abs().max()) + 2
    check(call(x, w, b, y, 0.1, reduction, grad), reference(x, w, b, y, 0.1, reduction, grad), dtype, zmax)


@pytest.mark.parametrize("T,D,V", [(1, 64, 2), (2, 96, 3), (3, 128, 700), (33, 96, 130), (64, 320, 75)])
def test_gradients_of_few_rows_are_off_by_their_own_rounding_alone(T, D, V):
    """bf16, up to 64 rows: G is held to 16 bits.  An element of a gradient is off by half a step of its own (2^-8 relative) and by what G's two
    roundings (2^-8 of 2^-8), the logits (products of bf16 are exact, their sums and exponentials off by 2^-20) and fp32 sums leave of
    sum |G| |W|: together below 2^-15 of that."""
    x, w, b, y = make(T, D, V, "bf16")
    got = call(x, w, b, y, 0.1, "sum")
    want = reference(x, w, b, y, 0.1, "sum")
    z = x.double() @ w.double().t() + b.double()
    G = torch.softmax(z, 1) - 0.1 / V
    G[torch.arange(T), y] -= 0.9
    for a, c, size in ((got[1], want[1], G.abs() @ w.double().abs()), (got[2], want[2], G.abs().t() @ x.double().abs())):
        assert bool(((a.double().cpu() - c).abs() <= 2.0 ** -8 * c.abs() + 2.0 ** -15 * size).all())


def test_few_rows_with_one_gradient_alone():
    from ofq_amd.functional import linear_cross_entropy
    x, w, _, y = make(2, 128, 500, "bf16")
    both = call(x, w, None, y)
    xs, ws = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    dx, = torch.autograd.grad(linear_cross_entropy(xs, ws.detach(), y.cuda()), [xs])
    dw, = torch.autograd.grad(linear_cross_entropy(xs.detach(), ws, y.cuda()), [ws])
    assert torch.equal(dx, both[1]) and torch.equal(dw, both[2])


def test_gradient_agrees_with_differences():
    """fp32 loss along a direction: central differences of the 64-bit loss against the kernel's gradient."""
    x, w, b, y = make(37, 48, 90, "fp32", ignored=0.2)
    got = call(x, w, b, y, 0.1)
    g = torch.Generator().manual_seed(1)
    for k, t in enumerate((x, w, b)):
        d = torch.randn(t.shape, generator=g).double()
        h = 1e-5
        args = [[x.double(), w.double(), b.double()] for _ in range(2)]
        args[0][k] = t.double() + h * d
        args[1][k] = t.double() - h * d
        diff = (reference(*args[0], y, 0.1)[0] - reference(*args[1], y, 0.1)[0]) / (2 * h)
        # differences: h^2 of the third derivative and 2^-53 / h; the kernel: its gradient tolerance times |d|
        tol = 1e-8 + GRAD_TOL["fp32"] * float(got[1 + k].double().norm()) * float(d.norm())
        assert abs(float((got[1 + k].double().cpu() * d).sum()) - float(diff)) <= tol


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_ignored_rows_may_hold_anything(dtype, value):
    x, w, b, y = make(70, 64, 200, dtype, ignored=0.5)
    want = call(x, w, b, y)
    dirty = x.clone()
    dirty[y == -100] = value
    got = call(dirty, w, b, y)
    for a, c in zip(got, want):
        assert torch.equal(a, c)
    assert not got[1][(y == -100).cuda()].any()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("T,live", [(300, 1), (300, 63), (300, 64), (300, 65), (300, 129), (9001, 70)])
def test_the_rows_that_count_anywhere_among_many(T, live, dtype):
    """As many rows as end on, in front of and behind a padding step, spread over the batch (and past what one pass of the numbering holds)."""
    D, V = 256, 130
    x, w, b, y = make(T, D, V, dtype)
    keep = torch.zeros(T, dtype=torch.bool)
    keep[torch.randperm(T, generator=torch.Generator().manual_seed(live))[:live]] = True
    keep[-1], keep[0] = True, False
    y[~keep] = -100
    x[~keep] = math.nan
    check(call(x, w, b, y, 0.1), reference(x, w, b, y, 0.1), dtype, 32.0)
    g = torch.rand(T, generator=torch.Generator().manual_seed(1)) - 0.5
    got = call(x, w, b, y, 0.0, "none", g)
    check(got, reference(x, w, b, y, 0.0, "none", g), dtype, 32.0)
    assert not bool(got[0].detach().cpu()[~keep].any()) and not bool(got[1].cpu()[~keep].any())


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("T,D,V", [(512, 512, 33000), (300, 320, 9100), (1025, 192, 4100)])
def test_logits_that_stay_for_the_backward(T, D, V, dtype):
    """Every tile form a kept grid has, with rests in both directions; without a backward pass nothing is kept and the loss is the same."""
    from ofq_amd.functional import linear_cross_entropy
    x, w, b, y = make(T, D, V, dtype, ignored=0.1)
    got = call(x, w, b, y, 0.1)
    check(got, reference(x, w, b, y, 0.1), dtype, 32.0)
    with torch.no_grad():
        assert torch.equal(linear_cross_entropy(x.cuda(), w.cuda(), y.cuda(), bias=b.cuda(), label_smoothing=0.1), got[0].detach())


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_no_rows_at_all(reduction):
    x, w, b, y = make(4, 64, 50, "fp32")
    got = call(x[:0], w, b, y[:0], 0.0, reduction, torch.ones(0) if reduction == "none" else None)
    assert got[0].shape == ((0,) if reduction == "none" else ())
    assert math.isnan(float(got[0])) if reduction == "mean" else not bool(got[0].any())
    if reduction != "mean":
        assert not any(bool(g.any()) for g in got[1:])


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_an_overflowed_gradient_stays_in_the_rows_that_count(dtype):
    """A loss scale that overflowed sends Inf in: rows that do not count still get zeros, the others nothing finite that is not zero."""
    x, w, b, y = make(70, 64, 90, dtype, ignored=0.3)
    dead = y == -100
    for reduction, grad in (("mean", math.inf), ("none", torch.full((70,), math.inf))):
        dx = call(x, w, b, y, 0.0, reduction, grad)[1].float().cpu()
        assert not bool(dx[dead].any()) and not bool(torch.isfinite(dx[~dead]).any())


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_a_graph_replayed_with_other_numbers_of_rows(dtype):
    """The number of rows that count is read on the device: a captured pass follows it from all rows to none."""
    from ofq_amd.functional import linear_cross_entropy
    x, w, _, y = make(260, 256, 300, dtype)
    xs, ws, ys = x.cuda().requires_grad_(), w.cuda().requires_grad_(), y.cuda()

    def step():
        loss = linear_cross_entropy(xs, ws, ys, reduction="sum")
        return (loss.detach(),) + torch.autograd.grad(loss, (xs, ws))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for live in (260, 100, 0, 1, 200):
        t = y.clone()
        t[live:] = -100
        ys.copy_(t)
        graph.replay()
        eager = call(x, w, None, t, 0.0, "sum")
        torch.cuda.synchronize()
        for a, c in zip(out, eager):
            assert torch.equal(a, c.detach())


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_no_live_row(dtype):
    x, w, b, y = make(5, 64, 10, dtype)
    y[:] = -100
    for reduction, expect in (("mean", math.nan), ("sum", 0.0), ("none", 0.0)):
        got = call(x, w, b, y, reduction=reduction, grad=torch.ones(5) if reduction == "none" else 1.0)
        assert bool(torch.isnan(got[0]).all()) if math.isnan(expect) else not bool(got[0].any())
        assert not any(bool(t.any()) for t in got[1:])


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_masked_classes_and_other_ignore_index(dtype):
    """A bias of -inf takes a class out; ignore_index may be an ordinary class number."""
    x, w, b, y = make(50, 64, 140, dtype)
    b = b.float()
    b[7], b[130:] = -math.inf, -math.inf
    y[y == 7] = 8
    y[y >= 130] = 3
    y[:10] = 0
    got = call(x, w, b.to(DTYPES[dtype]), y, ignore=0)
    keep = [v for v in range(130) if v != 7]
    at = torch.zeros(140, dtype=torch.int64)
    at[keep] = torch.arange(len(keep))
    loss, dx, dw, db = reference(x, w[keep], b.to(DTYPES[dtype])[keep], torch.where(y == 0, -100, at[y]))
    assert abs(float(got[0]) - float(loss)) <= LOSS_TOL * 16
    assert far(got[1], dx) <= GRAD_TOL[dtype] and far(got[2][keep], dw) <= GRAD_TOL[dtype] and far(got[3][keep], db) <= GRAD_TOL[dtype]
    gone = [7] + list(range(130, 140))
    assert not got[2][gone].any() and not got[3][gone].any()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_a_target_outside_the_vocabulary_is_loud(dtype):
    x, w, b, y = make(9, 64, 20, dtype)
    for bad in (20, -1, 2 ** 40):
        yy = y.clone()
        yy[4] = bad
        assert math.isnan(float(call(x, w, b, yy)[0]))
        rows = call(x, w, b, yy, reduction="none", grad=torch.ones(9))
        assert torch.isnan(rows[0]).tolist() == [i == 4 for i in range(9)]
        assert all(bool(torch.isfinite(t.float()).all()) for t in rows[1:])


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("scale", [1e-12, 1e6])
def test_scales_far_from_one(dtype, scale):
    x, w, b, y = make(40, 64, 100, dtype)
    x, w = (x.float() * scale).to(DTYPES[dtype]), (w.float() / scale).to(DTYPES[dtype])
    got, want = call(x, w, b, y), reference(x, w, b, y)
    check(got, want, dtype, 16.0)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_large_logits_do_not_overflow(dtype):
    x, w, b, y = make(33, 64, 150, dtype)
    x = (x.float() * 300).to(DTYPES[dtype])
    want = reference(x, w, b, y)
    got = call(x, w, b, y)
    zmax = float((x.double() @ w.double().t()).abs().max())
    assert abs(float(got[0]) - float(want[0])) <= LOSS_TOL * zmax
    # an error of LOSS_TOL zmax in z is one of that relative size in exp z
    for a, c in zip(got[1:], want[1:]):
        assert far(a, c) <= GRAD_TOL[dtype] + 4 * LOSS_TOL * zmax


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_strides_offsets_and_leading_dimensions(dtype):
    """Inputs that are views: columns of a wider tensor, a transposed weight, a 3-d input, addresses that are not multiples of 16 bytes."""
    from ofq_amd.functional import linear_cross_entropy
    x, w, b, y = make(60, 64, 130, dtype, ignored=0.1)
    base = linear_cross_entropy(x.cuda(), w.cuda(), y.cuda(), bias=b.cuda(), reduction="none")
    wide = torch.zeros(60, 70, dtype=x.dtype, device="cuda")
    wide[:, 3:67] = x.cuda()
    off = torch.zeros(130 * 64 + 1, dtype=w.dtype, device="cuda")
    off[1:] = w.cuda().reshape(-1)
    yy = torch.stack([y, y], 1).cuda()[:, 0]
    xv, wv = wide[:, 3:67].requires_grad_(), off[1:].view(130, 64).requires_grad_()
    for xx, ww in ((xv, w.cuda().requires_grad_()), (x.cuda().requires_grad_(), w.cuda().t().contiguous().t().requires_grad_()),
                   (x.cuda().requires_grad_(), wv)):
        rows = linear_cross_entropy(xx.view(4, 15, 64) if xx.is_contiguous() else xx, ww, yy.view(4, 15) if xx.is_contiguous() else yy,
                                    bias=b.cuda(), reduction="none")
        assert torch.equal(rows.reshape(-1), base)
        gx, gw = torch.autograd.grad(rows.sum(), (xx, ww))
        _, dx, dw, _ = reference(x, w, b, y, 0.0, "none", torch.ones(60))
        assert far(gx, dx) <= GRAD_TOL[dtype] and far(gw, dw) <= GRAD_TOL[dtype]


def test_bias_in_fp32_beside_bf16():
    x, w, b, y = make(50, 64, 130, "bf16")
    from ofq_amd.functional import linear_cross_entropy
    bs = (b.float() + 0.001).cuda().requires_grad_()
    loss = linear_cross_entropy(x.cuda(), w.cuda(), y.cuda(), bias=bs)
    g, = torch.autograd.grad(loss, (bs,))
    want = reference(x, w, bs.detach().cpu(), y)
    assert g.dtype == torch.float32 and abs(float(loss) - float(want[0])) <= LOSS_TOL * 16 and far(g, want[3]) <= GRAD_TOL["bf16"]


def test_only_the_gradients_asked_for():
    from ofq_amd.functional import linear_cross_entropy
    x, w, b, y = make(30, 64, 100, "fp32")
    full = call(x, w, b, y)
    for k in range(3):
        t = [x.cuda(), w.cuda(), b.cuda()]
        t[k].requires_grad_()
        loss = linear_cross_entropy(t[0], t[1], y.cuda(), bias=t[2])
        g, = torch.autograd.grad(loss, (t[k],))
        assert torch.equal(g, full[1 + k])
    with torch.no_grad():
        assert torch.equal(linear_cross_entropy(x.cuda(), w.cuda(), y.cuda(), bias=b.cuda()), full[0].detach())


def test_same_bits_every_time_and_on_another_stream():
    x, w, b, y = make(700, 96, 5000, "fp32", ignored=0.1)
    first = call(x, w, b, y)
    s = torch.cuda.Stream()
    for stream in (torch.cuda.current_stream(), s, s):
        with torch.cuda.stream(stream):
            again = call(x, w, b, y)
        stream.synchronize()
        for a, c in zip(first, again):
            assert torch.equal(a, c)


def test_weight_changed_between_forward_and_backward_is_refused():
    from ofq_amd.functional import linear_cross_entropy
    x, w, b, y = make(8, 64, 20, "bf16")
    ws = w.cuda().requires_grad_()
    loss = linear_cross_entropy(x.cuda(), ws, y.cuda())
    with torch.no_grad():
        ws.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_weights_that_come_back_at_another_alignment():
    """A saved-tensor hook may hand the backward a copy: at another alignment than the forward's (which had packed it) it is refused; one
    that went to the host and back is as good as the original."""
    from ofq_amd.functional import linear_cross_entropy
    x, w, _, y = make(40, 64, 300, "bf16")
    xs, ys = x.cuda().requires_grad_(), y.cuda()
    odd = torch.empty(300 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(300, 64).copy_(w.cuda()).requires_grad_()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.clone()):
        loss = linear_cross_entropy(xs, odd, ys)
        with pytest.raises(RuntimeError, match="ofq_linear_ce_bwd"):
            loss.backward()
    want = call(x, w, None, y)
    ws = w.cuda().requires_grad_()
    with torch.autograd.graph.save_on_cpu():
        dx, dw = torch.autograd.grad(linear_cross_entropy(xs, ws, ys), [xs, ws])
    assert torch.equal(dx, want[1]) and torch.equal(dw, want[2])


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_captured_forward_and_backward_replayed(dtype):
    """The graph replayed with other inputs in its static buffers, with eager work and synchronisations between the replays."""
    from ofq_amd.functional import linear_cross_entropy
    batches = [make(200, 64, 700, dtype, seed=s, ignored=0.2) for s in range(4)]
    x, w, b, y = (t.cuda() for t in batches[0])
    for t in (x, w, b):
        t.requires_grad_()

    def step():
        loss = linear_cross_entropy(x, w, y, bias=b, label_smoothing=0.1)
        return (loss.detach(),) + torch.autograd.grad(loss, (x, w, b))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for n in range(3):
        for bx, bw, bb, by in batches:
            with torch.no_grad():
                x.copy_(bx), w.copy_(bw), b.copy_(bb), y.copy_(by)
            graph.replay()
            eager = call(bx, bw, bb, by, 0.1)
            torch.cuda.synchronize()
            for a, c in zip(out, eager):
                assert torch.equal(a, c.detach())


def test_two_losses_in_one_backward():
    """Two heads over the same hidden states, their gradients accumulated, as a distilled model has them."""
    from ofq_amd.functional import linear_cross_entropy
    x, w, b, y = make(50, 64, 130, "fp32")
    _, w2, _, _ = make(50, 64, 130, "fp32", seed=5)
    xs, a, c = x.cuda().requires_grad_(), w.cuda().requires_grad_(), w2.cuda().requires_grad_()
    (linear_cross_entropy(xs, a, y.cuda()) + 0.5 * linear_cross_entropy(xs, c, y.cuda(), reduction="sum")).backward()
    r1, r2 = reference(x, w, None, y), reference(x, w2, None, y, 0.0, "sum", 0.5)
    assert far(xs.grad, r1[1] + r2[1]) <= GRAD_TOL["fp32"] and far(a.grad, r1[2]) <= GRAD_TOL["fp32"] and far(c.grad, r2[2]) <= GRAD_TOL["fp32"]


def test_module_and_quantised_head():
    """LSQ_QLinear4head.loss equals cross entropy on the head's own logits, with every parameter's gradient."""
    from ofq_amd.quantization.modules.qlinear import LSQ_QLinear4head
    from ofq_amd.quantization.utils import LinearCrossEntropy
    torch.manual_seed(3)
    head = LSQ_QLinear4head(m=nn.Linear(64, 130), weight_bits=8, input_bits=8, weight_quant_method="lsq", input_quant_method="lsq",
                            pretrained_initialized=True).cuda()
    x = torch.randn(24, 64, device="cuda")
    y = torch.randint(0, 130, (24,), device="cuda")
    with torch.no_grad():
        head(x)
    params = list(head.parameters())
    got = head.loss(x, y, label_smoothing=0.1)
    grads = torch.autograd.grad(got, params)
    want = torch.nn.functional.cross_entropy(head(x), y, label_smoothing=0.1)
    ref = torch.autograd.grad(want, params)
    assert abs(float(got) - float(want)) <= 2 * LOSS_TOL * 16
    scale = max(float(r.norm()) for r in ref)
    for a, c in zip(grads, ref):
        # both are fp32 results of different summation orders; a step's gradient is a sum of cancelling terms, so by the common scale
        assert float((a - c).norm()) <= 1e-4 * scale
    mod = LinearCrossEntropy(label_smoothing=0.1)
    w = torch.randn(130, 64, device="cuda")
    assert abs(float(mod(x, w, y)) - float(torch.nn.functional.cross_entropy(x.double() @ w.double().t(), y, label_smoothing=0.1))) \
        <= LOSS_TOL * 64
