"""optim.orthogonalize and optim.FusedMuon against the definition in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

NS = (3.4445, -4.7750, 2.0315)
# Norm of the error over the norm of the result.  One rounding of X (two fp16 planes: 2^-22 of an element) is multiplied on its way by at
# most the growth of a singular value over the chain, a^5 = 485 where it stays small, over the growth of the whole matrix, which ends
# at norm sqrt(rank) from norm 1: for the matrices here, whose rank is at least 1 and whose singular values are spread, below 30.  Three
# products a step and five steps: 15 roundings at random add to sqrt(15).  30 * 4 * 2^-22 = 2.9e-5; ranks of 64 and more stay below 1e-5
# (the bound that is used for them), being divided by sqrt(rank) of 8 and more.
TOL32, TOL32_SMALL = 1e-5, 2.9e-5
# bf16: one rounding of the result, off by 2^-9 at most (half a step): rms below that
TOL16 = 2.0 ** -8


@pytest.fixture(scope="module", autouse=True)
def lib():
    assert torch.cuda.is_available(), "the -m gpu tests need a HIP device"
    import ofq_amd.ops as ops
    ops.lib()


def definition(u, steps=5, coefficients=NS, eps=1e-7):
    a, b, c = coefficients
    x = u.double()
    x = x / max(float(x.norm()), eps)
    flip = x.shape[0] > x.shape[1]
    x = x.t() if flip else x
    for _ in range(steps):
        q = x @ x.t()
        x = a * x + (b * q + c * (q @ q)) @ x
    return x.t() if flip else x


def far(a, b):
    a, b = a.detach().double().cpu(), b.double()
    assert a.shape == b.shape
    n = float(b.norm())
    return float((a - b).norm()) / n if n else float((a - b).norm())


def tol(shape):
    return TOL32 if min(shape) >= 64 else TOL32_SMALL


def matrix(r, c, seed=0, rank=None):
    g = torch.Generator().manual_seed(seed + 31 * r + c)
    m = torch.randn(r, c, generator=g)
    if rank:
        k = min(rank, r, c)
        m = 0.1 * m + torch.randn(r, k, generator=g) @ torch.randn(k, c, generator=g)
    return m


SHAPES = [(1, 1), (1, 2), (2, 1), (1, 300), (300, 1), (3, 5), (63, 65), (64, 64), (65, 63), (127, 129), (128, 128), (128, 1000), (129, 127),
          (192, 192), (200, 65), (257, 255), (384, 1536), (1000, 130)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("rank", [None, 4])
def test_one_matrix_fp32(shape, rank):
    from ofq_amd.optim import orthogonalize
    g = matrix(*shape, rank=rank)
    out = orthogonalize(g.cuda())
    assert out.dtype == torch.float32 and far(out, definition(g)) <= tol(shape)


def test_a_list_is_each_of_its_matrices():
    """All shapes and both types in one call: each is its own definition's, twice the same bits (alone a matrix may differ by roundings: a
    launch takes its tile form by the number of its tiles); the same tensor twice is two results."""
    from ofq_amd.optim import orthogonalize
    mats = [matrix(*s, seed=i).cuda() for i, s in enumerate(SHAPES)]
    mats += [m.bfloat16() for m in mats[::2]] + [mats[3], mats[3], torch.zeros(0, 5, device="cuda"), torch.zeros(7, 0, device="cuda")]
    keep = [m.clone() for m in mats]
    outs = orthogonalize(mats)
    assert len(outs) == len(mats)
    for m, o, k in zip(mats, outs, keep):
        assert torch.equal(m, k) and o.dtype == m.dtype and o.shape == m.shape
        if m.numel():
            want = definition(m.cpu())
            assert far(o, want) <= (TOL16 if m.dtype == torch.bfloat16 else tol(m.shape))
    assert outs[-4].data_ptr() != outs[-3].data_ptr() and torch.equal(outs[-4], outs[-3])
    assert all(torch.equal(a, b) for a, b in zip(outs, orthogonalize(mats)))


def test_more_matrices_than_one_upload_holds():
    from ofq_amd.optim import orthogonalize
    mats = [matrix(3 + i % 5, 4 + i % 7, seed=i) for i in range(101)]
    for m, o in zip(mats, orthogonalize([m.cuda() for m in mats])):
        assert far(o, definition(m)) <= TOL32_SMALL


@pytest.mark.parametrize("steps,coefficients", [(0, NS), (1, NS), (2, NS), (6, NS), (12, (1.5, -0.5, 0.0)), (10, (2.0, -1.5, 0.5)), (3, (1.875, -1.25, 0.375))])
def test_steps_and_coefficients(steps, coefficients):
    from ofq_amd.optim import orthogonalize
    for shape in ((90, 70), (64, 200)):
        g = matrix(*shape)
        out = orthogonalize(g.cuda(), steps=steps, coefficients=coefficients)
        assert far(out, definition(g, steps, coefficients)) <= TOL32


@pytest.mark.parametrize("scale", [1e-30, 1e-15, 1e15, 1e30])
def test_scales_far_from_one(scale):
    """The norm is taken in 64 bits: neither the squares of 1e-30 nor those of 1e30 leave its range; below eps the matrix is divided by eps."""
    from ofq_amd.optim import orthogonalize
    g = matrix(100, 80) * scale
    if scale < 1e-7:
        out = orthogonalize(g.cuda(), eps=1e-40)
        assert far(out, definition(g, eps=1e-40)) <= TOL32
        small = orthogonalize(g.cuda())
        assert bool(torch.isfinite(small).all()) and float(small.norm()) < 1e-2
    else:
        assert far(orthogonalize(g.cuda()), definition(g)) <= TOL32


def test_zero_nan_and_inf_stay_in_their_matrix():
    from ofq_amd.optim import orthogonalize
    mats = [matrix(70, 70), torch.zeros(70, 90), matrix(65, 130, seed=2), matrix(30, 20, seed=3)]
    mats[0][3, 4] = math.nan
    mats[2][64, 129] = math.inf
    outs = orthogonalize([m.cuda() for m in mats])
    assert bool(torch.isnan(outs[0]).any()) and not bool(outs[1].any()) and not bool(torch.isfinite(outs[2]).all())
    assert far(outs[3], definition(mats[3])) <= TOL32_SMALL


def test_views_and_another_stream():
    from ofq_amd.optim import orthogonalize
    base = matrix(200, 300).cuda()
    views = [base.t(), base[10:90, 5:77], base[::2, ::3], base.reshape(-1)[1:4097].view(64, 64)]
    want = orthogonalize([v.contiguous().clone() for v in views])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = orthogonalize(views)
    s.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------------------------- the optimiser
LR, MU, WD = 0.02, 0.95, 0.1


def muon_reference(p, m, g, lr=LR, mu=MU, wd=WD, nesterov=True, rms=False):
    p, m, g = p.double(), m.double(), g.double()
    m = mu * m + (1 - mu) * g
    o = definition(mu * m + (1 - mu) * g if nesterov else m)
    s = 0.2 * math.sqrt(max(p.shape)) if rms else math.sqrt(max(1.0, p.shape[0] / p.shape[1]))
    return p * (1 - lr * wd) - lr * s * o, m


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("rms", [True, False])
def test_muon_steps(nesterov, rms):
    from ofq_amd.optim import FusedMuon
    shapes = [(64, 64), (192, 768), (768, 192), (129, 65), (1, 40), (40, 1)]
    ps = [torch.nn.Parameter(0.05 * matrix(*s, seed=9).cuda()) for s in shapes]
    opt = FusedMuon(ps, lr=LR, momentum=MU, weight_decay=WD, nesterov=nesterov, adjust_lr_fn="match_rms_adamw" if rms else None)
    want = [(p.detach().cpu().double(), torch.zeros(p.shape, dtype=torch.float64)) for p in ps]
    for t in range(3):
        for i, p in enumerate(ps):
            p.grad = None if (t == 1 and i == 2) else matrix(*p.shape, seed=100 * t + i, rank=8).cuda()
            if p.grad is not None:
                want[i] = muon_reference(*want[i], p.grad.cpu(), nesterov=nesterov, rms=rms)
        opt.step()
    for p, (w, m) in zip(ps, want):
        # three steps of momentum (a rounding or two each), and three updates whose size next to the weights is at most lr s |O| / |p|
        assert far(opt.state[p]["momentum_buffer"], m) <= 8 * 2.0 ** -24
        s = 0.2 * math.sqrt(max(p.shape)) if rms else math.sqrt(max(1.0, p.shape[0] / p.shape[1]))
        update = 3 * LR * s * math.sqrt(min(p.shape)) * 1.3
        assert float((p.detach().cpu().double() - w).norm()) <= tol(p.shape) * update + 8 * 2.0 ** -24 * float(w.norm())


def test_adamw_groups_equal_fused_adamw():
    from ofq_amd.optim import FusedAdamW, FusedMuon
    def params():
        return [torch.nn.Parameter(matrix(5, 7).cuda()), torch.nn.Parameter(matrix(9, 1)[:, 0].cuda())]
    a, b = params(), params()
    hidden = torch.nn.Parameter(matrix(64, 64).cuda())
    one = FusedAdamW(a, lr=1e-2, weight_decay=0.05, eps=1e-6, betas=(0.8, 0.9))
    two = FusedMuon([{"params": [hidden]}, {"params": b, "use_muon": False}], lr=1e-2, weight_decay=0.05, adamw_eps=1e-6, betas=(0.8, 0.9))
    for t in range(3):
        for p, q in zip(a, b):
            p.grad = torch.randn_like(p)
            q.grad = p.grad.clone()
        hidden.grad = torch.randn_like(hidden)
        one.step(), two.step()
    for p, q in zip(a, b):
        assert torch.equal(p, q) and torch.equal(one.state[p]["exp_avg_sq"], two.state[q]["exp_avg_sq"])
    state = two.state_dict()
    again = FusedMuon([{"params": [hidden]}, {"params": b, "use_muon": False}])
    again.load_state_dict(state)
    assert torch.equal(again.state[hidden]["momentum_buffer"], two.state[hidden]["momentum_buffer"])


def test_captured_step_follows_the_learning_rate():
    """A captured step of both rules, replayed with a learning rate that changes, against eager steps: the same bits."""
    from ofq_amd.optim import FusedMuon

    def build():
        ps = [torch.nn.Parameter(matrix(*s, seed=4).cuda()) for s in ((64, 96), (130, 70), (33,) * 2)]
        v = torch.nn.Parameter(matrix(50, 1)[:, 0].cuda())
        for p in ps + [v]:
            p.grad = torch.zeros_like(p)
        return ps + [v], FusedMuon([{"params": ps}, {"params": [v], "use_muon": False}], lr=LR)
    (ea, eo), (ca, co) = build(), build()
    grads = [[torch.randn(p.shape, generator=torch.Generator().manual_seed(10 * t + i)).cuda() for i, p in enumerate(ea)] for t in range(6)]

    def load(ps, t):
        for p, g in zip(ps, grads[t]):
            p.grad.copy_(g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        load(ca, 0)
        co.step()
    torch.cuda.current_stream().wait_stream(side)
    load(ea, 0)
    eo.step()
    co.begin_capture(torch.device("cuda", torch.cuda.current_device()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        co.step()
    for t in range(1, 6):
        for opt in (eo, co):
            for group in opt.param_groups:
                group["lr"] = LR / t
        load(ca, t)
        co.advance_for_replay()
        graph.replay()
        load(ea, t)
        eo.step()
        torch.cuda.synchronize()
        for p, q in zip(ea, ca):
            assert torch.equal(p, q)
            for k in eo.state[p]:
                assert torch.equal(eo.state[p][k], co.state[q][k])


def test_step_guard_leaves_everything_as_it_is():
    from ofq_amd import ops
    from ofq_amd.optim import FusedMuon
    p = torch.nn.Parameter(matrix(70, 65).cuda())
    opt = FusedMuon([p], lr=LR)
    p.grad = torch.randn_like(p)
    opt.step()
    before, mom = p.detach().clone(), opt.state[p]["momentum_buffer"].clone()
    dev = p.device
    had = ops._guard_words.get(dev.index)
    try:
        word = torch.ones(1, dtype=torch.int32, device=dev)
        ops._guard_words[dev.index] = word
        opt.step()
        assert torch.equal(p.detach(), before) and torch.equal(opt.state[p]["momentum_buffer"], mom)
        word.zero_()
        opt.step()
        assert not torch.equal(p.detach(), before)
    finally:
        if had is None:
            ops._guard_words.pop(dev.index)
        else:
            ops._guard_words[dev.index] = had


def test_a_training_step_with_both_ends():
    """The two ends of a step together: a quantised model's hidden layers under FusedMuon through engine.make_optimizer, its loss from
    the hidden states through the classifier's fused loss; gradients against the logits' own cross entropy, then the update."""
    from functools import partial
    from types import SimpleNamespace

    import torch.nn as nn
    from ofq_amd import engine
    from ofq_amd.deit import DistilledVisionTransformer
    torch.manual_seed(0)
    model = DistilledVisionTransformer(img_size=224, patch_size=16, embed_dim=64, depth=2, num_heads=2, mlp_ratio=4, qkv_bias=True,
                                       num_classes=50, norm_layer=partial(nn.LayerNorm, eps=1e-6), act_layer=nn.GELU)
    args = SimpleNamespace(qmodules=engine.default_qmodules(2), wq_mode="statsq", wq_enable=True, wq_bitw=4, aq_enable=True, aq_mode="lsq",
                           aq_bitw=4, wq_per_channel=True, aq_per_channel=True, model_type="deit", pretrained_initialized=True,
                           qk_reparam=True, qk_reparam_type=0)
    model = engine.get_qat_model(model, args).cuda()
    img, y = torch.randn(4, 3, 224, 224, device="cuda"), torch.randint(0, 50, (4,), device="cuda")
    engine.setup_alpha(model, img)
    model.train()
    opt = engine.make_optimizer(model, lr=1e-3, opt="muon")
    muon = {id(p) for p in opt.param_groups[0]["params"]}
    named = dict(model.named_parameters())
    assert {n for n, p in named.items() if id(p) in muon} == {n for n, p in named.items()
                                                              if n.startswith("blocks.") and n.endswith(".weight") and p.dim() == 2}
    assert sum(len(g["params"]) for g in opt.param_groups) == len([p for p in named.values() if p.requires_grad])

    def loss_fn(out, target, soft):
        return sum(nn.functional.cross_entropy(o, target) for o in out[:2])
    before = {n: p.detach().clone() for n, p in named.items()}
    for _ in range(2):
        loss = engine.train_step(model, opt, img, y, None, loss_fn)
        assert bool(torch.isfinite(loss))
    moved = [n for n, p in named.items() if p.grad is not None and bool(p.grad.any()) and torch.equal(p, before[n])]
    assert not moved
    for n, p in named.items():
        if id(p) in muon:
            assert set(opt.state[p]) == {"momentum_buffer"}
    # the head's fused loss against its logits, on the hidden states the head sees
    seen = {}
    hook = model.head.register_forward_pre_hook(lambda m, a: seen.update(x=a[0].detach()))
    with torch.no_grad():
        model(img)
    hook.remove()
    head = model.head
    params = list(head.parameters())
    fused = head.loss(seen["x"], y)
    plain = nn.functional.cross_entropy(head(seen["x"]), y)
    assert abs(float(fused) - float(plain)) <= 1e-5
    ga, gb = torch.autograd.grad(fused, params), torch.autograd.grad(plain, params)
    scale = max(float(g.norm()) for g in gb)
    assert all(float((a - b).norm()) <= 1e-4 * scale for a, b in zip(ga, gb))


def test_a_captured_training_step_under_both_rules():
    """engine.GraphedTrainStep with the optimiser of opt="muon", the learning rate changing: losses, parameters and momentum are the
    eager steps', bit for bit."""
    import copy
    from functools import partial
    from types import SimpleNamespace

    import torch.nn as nn
    from ofq_amd import engine
    from ofq_amd.deit import DistilledVisionTransformer
    torch.manual_seed(0)
    base = DistilledVisionTransformer(img_size=224, patch_size=16, embed_dim=64, depth=2, num_heads=2, mlp_ratio=4, qkv_bias=True,
                                      num_classes=50, norm_layer=partial(nn.LayerNorm, eps=1e-6), act_layer=nn.GELU)
    args = SimpleNamespace(qmodules=engine.default_qmodules(2), wq_mode="statsq", wq_enable=True, wq_bitw=4, aq_enable=True, aq_mode="lsq",
                           aq_bitw=4, wq_per_channel=True, aq_per_channel=True, model_type="deit", pretrained_initialized=True,
                           qk_reparam=True, qk_reparam_type=0)
    base = engine.get_qat_model(base, args).cuda()
    g = torch.Generator().manual_seed(1)
    batches = [(torch.randn(4, 3, 224, 224, generator=g).cuda(), torch.randint(0, 50, (4,), generator=g).cuda(),
                torch.randn(4, 50, generator=g).cuda()) for _ in range(2)]
    engine.setup_alpha(base, batches[0][0])
    from ofq_amd.quantization.utils import KDLossSoftandHard
    results = []
    for graphed in (False, True):
        model = copy.deepcopy(base).train()
        opt = engine.make_optimizer(model, lr=1e-3, opt="muon")
        loss_fn = KDLossSoftandHard()
        gs = engine.GraphedTrainStep(model, opt, loss_fn, warmup=2) if graphed else None
        losses = []
        for i in range(6):
            for group in opt.param_groups:
                group["lr"] = 1e-3 * (1 - 0.1 * i)
            img, y, soft = batches[i % 2]
            loss = gs(img, y, soft) if graphed else engine.train_step(model, opt, img, y, soft, loss_fn)
            losses.append(float(loss.detach()))
        state = [opt.state[p].get("momentum_buffer") for p in model.parameters()]
        results.append((losses, [p.detach().clone() for p in model.parameters()], state))
    (la, pa, sa), (lb, pb, sb) = results
    assert la == lb
    assert all(torch.equal(a, b) for a, b in zip(pa, pb))
    assert sum(a is not None for a in sa) > 0
    assert all((a is None and b is None) or torch.equal(a, b) for a, b in zip(sa, sb))


def test_train_command_with_muon(tmp_path):
    """train.py --opt muon: two epochs of two steps, and a run resumed after the first goes on with the same losses."""
    import contextlib
    import io

    from ofq_amd import train_cli
    common = ["--model", "deit_tiny_distilled_patch16_224", "--batch-size", "4", "--steps-per-epoch", "2", "--val-steps", "1",
              "--lr", "5e-4", "--weight-decay", "0.05", "--aq-enable", "--aq-mode", "lsq", "--aq-per-channel", "--aq_clip_learnable",
              "--aq-bitw", "3", "--wq-enable", "--wq-per-channel", "--wq-bitw", "3", "--wq-mode", "statsq", "--model_type", "deit",
              "--quantized", "--qk_reparam", "--qk_reparam_type", "0", "--log-interval", "1", "--warmup-epochs", "0", "--opt", "muon"]

    def run(extra):
        buf = io.StringIO()
        with contextlib.redirect_stdout(buf):
            train_cli.main(common + extra)
        return [float(l.split("Loss:")[1].split()[0]) for l in buf.getvalue().splitlines() if l.startswith("Train:")]
    full = run(["--epochs", "2", "--output", str(tmp_path / "full")])
    run(["--epochs", "1", "--output", str(tmp_path / "half")])
    rest = run(["--epochs", "2", "--resume", str(tmp_path / "half" / "last.pth.tar"), "--output", str(tmp_path / "res")])
    assert len(full) == 4 and rest == pytest.approx(full[2:], rel=1e-6)
