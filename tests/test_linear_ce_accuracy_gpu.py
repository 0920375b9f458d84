"""bf16 gradients of linear_cross_entropy held to the roundings that they have, and to nothing more: as a whole by the norm, and element by
element, the classes behind the last whole 64 among them.  The checks themselves are tried on the CPU with mistakes in their input."""
import math

import pytest
import torch

from test_linear_ce_gpu import call, make, reference

STEP = 2.0 ** -8                           # half a step of bf16, relative


def graph_of(x, w, b, y, smoothing, reduction):
    """G in 64 bits over what all rows share, and that factor."""
    z = x.double() @ w.double().t() + (0.0 if b is None else b.double())
    G = torch.softmax(z, 1) - smoothing / w.shape[0]
    live = y != -100
    G[torch.arange(len(y))[live], y[live]] -= 1 - smoothing
    G[~live] = 0
    unit = 1 - smoothing if smoothing <= 0.5 else 1.0
    return G / unit, unit / (int(live.sum()) if reduction == "mean" else 1)


def check_roundings(got, x, w, b, y, smoothing, reduction):
    """got: dx, dW, db in bf16.  G over the shared factor is rounded to bf16 (up to 64 rows: to two bf16 planes, 16 bits), the result is
    rounded to bf16; sums, logits and exponentials are fp32's.
    By norm: the error of those two roundings done in 64 bits, one after the other, plus 2^-13: a G that fp32 (2^-20 of it) puts on
    the other side of a tie moves by 2^-8 of itself, and one in 2^11 does: 2^-8 2^-5.5.
    By element: half a step of the result, half a step (16 bits: 2^-15) of each G, and 2^-15 of the terms for fp32's errors."""
    G, f = graph_of(x, w, b, y, smoothing, reduction)
    one_plane = len(y) > 64
    R = G.bfloat16().double() if one_plane else G
    X = torch.where((y != -100)[:, None], x.double(), 0.0)
    for name, a, exact, rounded, size in (("dx", got[0], G @ w.double(), R @ w.double(), G.abs() @ w.double().abs()),
                                          ("dW", got[1], G.t() @ X, R.t() @ X, G.abs().t() @ X.abs()),
                                          ("db", got[2], G.sum(0), G.sum(0), G.abs().sum(0))):
        a = a.detach().double().cpu()
        exact, rounded, size = exact * f, rounded * f, size * f
        n = float(exact.norm())
        bound = float((exact.bfloat16().double() - exact).norm()) + float((rounded - exact).norm()) + 2.0 ** -13 * n
        err = (a - exact).abs()
        assert float(err.norm()) <= bound, (name, "norm", float(err.norm()) / n, bound / n)
        per = STEP * exact.abs() + ((STEP if one_plane else 0.0) + 2.0 ** -15) * size * (1 + STEP)
        assert bool((err <= per).all()), (name, "element", float((err / per).max()))


def tail_targets(T, V, seed=1):
    """Targets among the classes behind the last whole 64."""
    first = V // 64 * 64
    assert first < V
    return torch.randint(first, V, (T,), generator=torch.Generator().manual_seed(seed))


CASES = [(1, 64, 65), (4, 128, 127), (5, 64, 1001), (64, 192, 1000), (65, 64, 9001), (140, 320, 333), (255, 128, 333), (300, 192, 1000), (512, 512, 33000), (1025, 128, 4100),
         (2100, 64, 40001)]


@pytest.mark.gpu
@pytest.mark.parametrize("T,D,V", CASES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("smoothing,reduction", [(0.0, "mean"), (0.1, "mean"), (0.3, "sum")])
def test_bf16_gradients_have_their_roundings_alone(T, D, V, tail, smoothing, reduction):
    """W in place (D a multiple of 64) and packed, every tile form, one piece and two; with targets behind the last whole 64 classes those rows of W
    carry dx."""
    x, w, b, y = make(T, D, V, "bf16", ignored=0.0 if T < 5 else 0.1)
    if tail:
        y = torch.where(y == -100, y, tail_targets(T, V))
    got = call(x, w, b, y, smoothing, reduction)
    check_roundings(got[1:], x, w, b, y, smoothing, reduction)


def simulated(x, w, b, y, smoothing, reduction, mistake=None):
    """What the kernels do, in 64 bits on the CPU."""
    G, f = graph_of(x, w, b, y, smoothing, reduction)
    if mistake == "shared factor in G":
        G, f = G * f, 1.0
    R = G.bfloat16().double() if len(y) > 64 else G
    if mistake == "a class lost from dx":
        lost = R.clone()
        lost[:, -1] = 0
        dx = lost @ w.double()
    else:
        dx = R @ w.double()
    dw = R.t() @ torch.where((y != -100)[:, None], x.double(), 0.0)
    if mistake == "a row of dW left at zero":
        dw[-1] = 0
    return (dx * f).bfloat16(), (dw * f).bfloat16(), (G.sum(0) * f).bfloat16()


@pytest.mark.parametrize("T,D,V", [(255, 128, 333), (255, 64, 1001)])
@pytest.mark.parametrize("mistake", [None, "shared factor in G", "a class lost from dx", "a row of dW left at zero"])
def test_the_check_sees_a_mistake(T, D, V, mistake):
    """(1/255 lies in the middle between two numbers of bf16.)"""
    x, w, b, _ = make(T, D, V, "bf16")
    y = tail_targets(T, V)
    got = simulated(x, w, b, y, 0.0, "mean", mistake)
    if mistake is None:
        check_roundings(got, x, w, b, y, 0.0, "mean")
        loss, dx, dw, db = reference(x, w, b, y)
        G, f = graph_of(x, w, b, y, 0.0, "mean")
        assert math.isfinite(float(loss)) and torch.allclose(G.sum(0) * f, db) and torch.allclose(G @ w.double() * f, dx)
    else:
        with pytest.raises(AssertionError):
            check_roundings(got, x, w, b, y, 0.0, "mean")
