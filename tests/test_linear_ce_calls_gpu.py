"""Calls of linear_cross_entropy that its documentation allows: no batch dimension, broadcast and tied operands, two calls at once, two captured
graphs in turn, and what a pass holds in memory."""
import pytest
import torch

from test_linear_ce_gpu import GRAD_TOL, LOSS_TOL, call, far, make, reference

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def lib():
    assert torch.cuda.is_available(), "the -m gpu tests need a HIP device"
    import ofq_amd.ops as ops
    ops.lib()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_one_row_without_a_batch_dimension(dtype, reduction):
    from ofq_amd.functional import linear_cross_entropy
    x, w, b, y = make(1, 72, 300, dtype)
    xs = x[0].cuda().requires_grad_()
    loss = linear_cross_entropy(xs, w.cuda(), y[0].cuda(), bias=b.cuda(), reduction=reduction)
    g, = torch.autograd.grad(loss, (xs,))
    want = reference(x, w, b, y)
    assert loss.shape == () and g.shape == (72,)
    assert abs(float(loss.detach()) - float(want[0])) <= LOSS_TOL * 16 and far(g, want[1][0]) <= GRAD_TOL[dtype]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("T", [4, 40, 100])
def test_broadcast_operands(T, dtype):
    """One row for all of the batch, one bias for all classes: the gradient is the sum over what was broadcast."""
    from ofq_amd.functional import linear_cross_entropy
    x, w, b, y = make(T, 64, 130, dtype)
    row, one = x[:1].cuda().requires_grad_(), b[:1].cuda().requires_grad_()
    loss = linear_cross_entropy(row.expand(T, 64), w.cuda(), y.cuda(), bias=one.expand(130), reduction="sum")
    gr, go = torch.autograd.grad(loss, (row, one))
    want = reference(x[:1].expand(T, 64), w, b[:1].expand(130), y, 0.0, "sum")
    assert far(gr, want[1].sum(0, keepdim=True)) <= GRAD_TOL[dtype]
    # the sum over all classes of a bias gradient is zero: what is left are the roundings of its 130 elements
    size = float(want[3].abs().sum())
    assert abs(float(go)) <= GRAD_TOL[dtype] * size


def test_tied_rows_and_weights():
    """The hidden states are rows of the weight itself: one leaf, two gradients, one of them through an index that takes a row twice."""
    from ofq_amd.functional import linear_cross_entropy
    _, w, b, y = make(90, 64, 200, "fp32")
    at = torch.randint(0, 200, (90,), generator=torch.Generator().manual_seed(2))
    at[1] = at[0]
    ws = w.cuda().requires_grad_()
    g, = torch.autograd.grad(linear_cross_entropy(ws[at.cuda()], ws, y.cuda(), bias=b.cuda()), (ws,))
    _, dx, dw, _ = reference(w[at], w, b, y)
    assert far(g, dw.index_add(0, at, dx)) <= 2 * GRAD_TOL["fp32"]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_two_calls_at_once(dtype):
    """Forward and backward passes of two problems interleaved on two streams, the host never waiting in between."""
    from ofq_amd.functional import linear_cross_entropy
    probs = [make(300, 320, 4100, dtype, seed=s, ignored=0.1) for s in (1, 2)]
    want = [call(*p, 0.1) for p in probs]
    dev = [[t.cuda() for t in p] for p in probs]
    for d in dev:
        for t in d[:3]:
            t.requires_grad_()
    streams = [torch.cuda.Stream() for _ in probs]
    torch.cuda.synchronize()
    out = [[], []]
    for _ in range(4):
        losses = []
        for d, s in zip(dev, streams):
            with torch.cuda.stream(s):
                losses.append(linear_cross_entropy(d[0], d[1], d[3], bias=d[2], label_smoothing=0.1))
        for k, (d, s) in enumerate(zip(dev, streams)):
            with torch.cuda.stream(s):
                out[k].append((losses[k].detach(),) + torch.autograd.grad(losses[k], d[:3]))
    torch.cuda.synchronize()
    for k in range(2):
        for got in out[k]:
            assert all(torch.equal(a, c.detach()) for a, c in zip(got, want[k]))


def test_two_captured_graphs_in_turn():
    """Each graph holds its own scratch: replayed alternately, with eager work in between, both keep their results."""
    from ofq_amd.functional import linear_cross_entropy
    probs = [make(260, 256, 3000, "fp32", seed=1, ignored=0.1), make(70, 128, 5000, "bf16", seed=2)]
    steps, graphs, outs = [], [], []
    for p in probs:
        x, w, b, y = (t.cuda() for t in p)
        for t in (x, w, b):
            t.requires_grad_()

        def step(x=x, w=w, b=b, y=y):
            loss = linear_cross_entropy(x, w, y, bias=b, reduction="sum")
            return (loss.detach(),) + torch.autograd.grad(loss, (x, w, b))
        steps.append(step)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for step in steps:
            step()
    torch.cuda.current_stream().wait_stream(side)
    for step in steps:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step())
    eager = [step() for step in steps]
    for k in (0, 1, 1, 0, 1, 0):
        graphs[k].replay()
        steps[1 - k]()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(outs[k], eager[k]))


@pytest.mark.parametrize("dtype,T,D,V", [("bf16", 2048, 256, 65536), ("fp32", 2048, 256, 65536)])
def test_what_a_pass_holds(dtype, T, D, V):
    """The peak of a pass, forward and backward: what its own size queries say, its gradients and the loss; below the logits alone, in the type
    that their cross entropy needs."""
    from ofq_amd import ops
    from ofq_amd.functional import linear_cross_entropy
    x, w, _, y = make(T, D, V, dtype, bias=False)
    x, w, y = x.cuda().requires_grad_(), w.cuda().requires_grad_(), y.cuda()

    def step():
        return torch.autograd.grad(linear_cross_entropy(x, w, y), (x, w))
    step()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    base = torch.cuda.memory_allocated()
    grads = step()
    torch.cuda.synchronize()
    peak = torch.cuda.max_memory_allocated() - base
    L, b16, size = ops.lib(), int(dtype == "bf16"), 2 if dtype == "bf16" else 4
    kept = L.ofq_linear_ce_kept_bytes(T, D, V, b16, 1, 1)
    fwd, bwd = L.ofq_linear_ce_fwd_ws_bytes(T, D, V, b16), L.ofq_linear_ce_bwd_call_ws_bytes(T, D, V, b16, 1, 1, 1, 0)
    assert peak <= kept + max(fwd, bwd + (T + V) * D * size) + (1 << 21)
    assert peak < T * V * 4
    assert len(grads) == 2
