"""linear_cross_entropy on the GPU against F.cross_entropy(F.linear(...)) in double precision on the CPU's definition.

Tolerances.  u = torch.finfo(dtype).eps / 2, products exact, fp32 accumulation.
  loss       the operands are the same in both, so what differs is fp32 arithmetic: a logit's accumulation is off by at most
             width * 2^-24 * sum |x w| <= width * 2^-24 * |x| |w| (worst order), lse and the rest by a few 2^-24 of the largest logit
  gradients  dz is rounded once (u |dz|), the result once (u), both accumulated in fp32.  Norm-wise over a whole gradient:
             |d dx| <= u | |dz| |W| | + u |dx|, so each is held to (|dz| |W|) u + u |dx| + the logits' error, elementwise.
             Kept exponentials (large calls) are rounded once more before dz: u p, except at the label.
             A probability below fp32's smallest normal number, 2^-126, may be flushed to zero by the exponential and the products
             (hardware exp2; 1e-38 of a gradient): 2^-126 of the other operand's magnitudes, doubled.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _inputs(n, d, v, dtype, bias, seed=0, ignored=0.2):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((n, d), generator=g)
    w = torch.randn((v, d), generator=g) * 2 / math.sqrt(d)
    t = torch.randint(0, v, (n,), generator=g)
    x += w[t] * torch.rand((n, 1), generator=g) * 3
    t[torch.rand(n, generator=g) < ignored] = -100
    b = torch.randn(v, generator=g) if bias else None
    return [None if o is None else o.to(dtype).to(DEV) for o in (x, w, b)] + [t.to(DEV)]


def _oracle(x, w, b, t, up, smoothing=0.0, reduction="mean", ignore=-100):
    """(loss, dx, dw, db, |dz| |W|, |dz|^T |x|, sum |dz|) in double precision."""
    xd, wd = x.detach().double(), w.detach().double()
    z = xd @ wd.t()
    if b is not None:
        z = z + b.detach().double()
    has = t != ignore
    tt = t.clamp(0, w.shape[0] - 1)
    lse = torch.logsumexp(z, 1)
    rows = lse - (1 - smoothing) * z.gather(1, tt[:, None])[:, 0]
    if smoothing:
        rows = rows - smoothing * z.mean(1)
    rows = torch.where(has, rows, torch.zeros_like(rows))
    count = max(int(has.sum()), 1) if reduction == "mean" else 1
    loss = rows if reduction == "none" else rows.sum() / count
    p = torch.exp(z - lse[:, None])
    dz = p - smoothing / w.shape[0]
    dz = dz.scatter_add(1, tt[:, None], torch.full_like(lse, smoothing - 1)[:, None])
    gr = (up.double() if reduction == "none" else up.double().expand(x.shape[0])) / count
    dz = torch.where(has[:, None], dz * gr[:, None], torch.zeros_like(dz))
    xz = torch.where(has[:, None], xd, torch.zeros_like(xd))
    # an error e of a logit, and of lse, changes dz by at most 2 p e
    pg = torch.where(has[:, None], p * gr[:, None].abs(), torch.zeros_like(p))
    return loss, (dz @ wd, dz.t() @ xz, dz.sum(0)), (dz.abs() @ wd.abs(), dz.abs().t() @ xz.abs(), dz.abs().sum(0)), \
        (pg @ wd.abs(), pg.t() @ xz.abs(), pg.sum(0))


def _logit_error(x, w, b):
    e = x.shape[1] * 2.0 ** -24 * float(x.double().norm(dim=1).max()) * float(w.double().norm(dim=1).max())
    top = float(x.double().norm(dim=1).max()) * float(w.double().norm(dim=1).max()) + (0 if b is None else float(b[b.abs() < 1e30].abs().max()))
    return e + 8 * 2.0 ** -24 * (top + math.log(w.shape[0]) + 1)


def _check(x, w, b, t, smoothing=0.0, reduction="mean", up=None, ignore=-100, kept=False):
    from yolov6_amd.models.losses.loss_ce import linear_cross_entropy
    leaves = [o.detach().requires_grad_() for o in (x, w, b) if o is not None]
    loss = linear_cross_entropy(leaves[0], leaves[1], t, leaves[2] if b is not None else None, label_smoothing=smoothing, reduction=reduction,
                                ignore_index=ignore)
    if up is None:
        up = torch.ones_like(loss)
    grads = torch.autograd.grad(loss, leaves, up)
    torch.cuda.synchronize()
    want, exact, spread, soft = _oracle(x, w, b, t, up, smoothing, reduction, ignore)
    err = _logit_error(x, w, b)
    assert loss.dtype == torch.float32 and loss.shape == want.shape
    assert float((loss.detach().double() - want).abs().max() if loss.numel() else 0) <= 2 * err * (1 if reduction != "sum" else x.shape[0])
    u = torch.finfo(x.dtype).eps / 2
    tiny = torch.finfo(x.dtype).tiny * u * 2
    # fp32 products accumulate `length` terms: length * 2^-24 of the sum of magnitudes
    for got, leaf, ex, sp, so, length in zip(grads, leaves, exact, spread, soft, (w.shape[0], x.shape[0], x.shape[0])):
        assert got.dtype == leaf.dtype and got.shape == leaf.shape
        flush = 2.0 ** -125 * (length * float(max(x.double().nan_to_num().abs().max(), w.double().abs().max(), 1.0)) * float(up.abs().max()) + 1)
        slack = (u * so if kept else 0) + u * sp + u * ex.abs() + 2 * err * so + length * 2.0 ** -24 * sp + 2 ** -20 * so * 2 + tiny + flush
        over = (got.double() - ex).abs() - slack * 1.01
        assert bool((over <= 0).all()), (tuple(leaf.shape), float(over.max()), float(ex.abs().max()))
    return loss, grads


SHAPES = [(1, 1, 1), (1, 8, 2), (2, 16, 3), (5, 64, 17), (63, 63, 64), (64, 64, 65), (129, 72, 127), (128, 128, 128), (130, 200, 129),
          (257, 512, 1000), (33, 515, 513), (3, 1024, 4097), (300, 31, 2)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,d,v", SHAPES)
def test_value_and_gradients(n, d, v, dtype):
    x, w, b, t = _inputs(n, d, v, dtype, True, seed=n + d + v)
    _check(x, w, b, t, up=torch.tensor(1024.0 if dtype == torch.float16 else 1.0, device=DEV))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("smoothing", [0.0, 0.1, 1.0])
@pytest.mark.parametrize("bias", [False, True])
def test_options(dtype, reduction, smoothing, bias):
    x, w, b, t = _inputs(150, 96, 333, dtype, bias, seed=3)
    up = None
    if reduction == "none":
        up = torch.linspace(-2, 3, 150, device=DEV)
        up[::7] = 0
    _check(x, w, b, t, smoothing, reduction, up)


def _keeps(n, d, v, dtype):
    """Whether such a call keeps exponentials."""
    return d >= 64 and v >= 512 and n * v >= 1 << 19 if dtype == torch.float32 else d >= 128 and v >= 1024 and n * v >= 1 << 22


# (rows, width, classes): every tile size, several pieces of the vocabulary (over 128 MB of dz), splits of both gradient products
LARGE = [(2100, 72, 33000), (4097, 40, 20011), (1100, 1032, 2057), (20000, 64, 81), (40, 136, 70001), (3000, 512, 4100)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,d,v", LARGE)
def test_pieces_tiles_and_splits(n, d, v, dtype):
    x, w, b, t = _inputs(n, d, v, dtype, True, seed=v)
    _check(x, w, b, t, smoothing=0.1, up=torch.tensor(16.0 * n if dtype == torch.float16 else 1.0, device=DEV), kept=_keeps(n, d, v, dtype))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [24, 25])
def test_views(dtype, d):
    """Rows of a wider buffer (at odd addresses), columns of a transposed one, one row for all, more than two dimensions."""
    from yolov6_amd.models.losses.loss_ce import linear_cross_entropy
    x, w, b, t = _inputs(90, 80, 70, dtype, True, seed=d)
    for cut in (x[:, 3:3 + d], x[::2, 1:1 + d], x.t()[:d].t(), x[:1, 5:5 + d].expand(30, d)):
        for wcut in (w[:, 7:7 + d], w.t()[:d].t(), w[:1, :d].expand(70, d)):
            _check(cut, wcut, b, t[:cut.shape[0]], reduction="sum")
    flat = x[:, :d].contiguous()
    cube = flat.view(3, 5, 6, d).requires_grad_()
    loss = linear_cross_entropy(cube, w[:, :d], t.view(3, 5, 6), b, reduction="none")
    assert loss.shape == (3, 5, 6)
    (g,) = torch.autograd.grad(loss.sum(), cube)
    _, grads = _check(flat, w[:, :d], b, t, reduction="none")
    assert torch.equal(g.view(90, d), grads[0])
    one = linear_cross_entropy(flat[0], w[:, :d], t[0], b, reduction="none")
    assert one.shape == () and torch.equal(one, loss.view(-1)[0].detach())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_rows_without_a_label(dtype):
    """They are not read: what is in them reaches nothing; all rows without one: loss 0, gradients 0."""
    from yolov6_amd.models.losses.loss_ce import linear_cross_entropy
    x, w, b, t = _inputs(200, 48, 90, dtype, True, seed=1, ignored=0.4)
    _, clean = _check(x, w, b, t)
    x[t == -100] = math.nan
    x[0 if int(t[0]) == -100 else int((t == -100).nonzero()[0]), 0] = math.inf
    leaves = [o.detach().requires_grad_() for o in (x, w, b)]
    loss = linear_cross_entropy(leaves[0], leaves[1], t, leaves[2])
    grads = torch.autograd.grad(loss, leaves)
    assert bool(torch.isfinite(loss.detach())) and all(torch.equal(a, c) for a, c in zip(grads, clean))
    none = torch.full_like(t, 7)
    for reduction in ("mean", "sum", "none"):
        loss = linear_cross_entropy(leaves[0], leaves[1], none, leaves[2], ignore_index=7, reduction=reduction)
        grads = torch.autograd.grad(loss.sum(), leaves)
        assert int(loss.count_nonzero()) == 0 and all(int(g.count_nonzero()) == 0 for g in grads)
    empty = leaves[0][:0]
    loss = linear_cross_entropy(empty, leaves[1], t[:0], leaves[2])
    grads = torch.autograd.grad(loss, leaves)
    assert float(loss.detach()) == 0.0 and all(int(g.count_nonzero()) == 0 for g in grads)
    assert linear_cross_entropy(empty, leaves[1], t[:0], leaves[2], reduction="none").shape == (0,)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_what_is_not_finite(dtype):
    from yolov6_amd.models.losses.loss_ce import linear_cross_entropy
    x, w, b, t = _inputs(70, 32, 300, dtype, True, seed=2, ignored=0.0)
    # classes switched off by a bias of -infinity (whole tiles of them among others): finite everywhere
    off = b.clone()
    off[64:200] = -math.inf
    off[t.unique()] = 0.0
    _check(x, w, off, t)
    lowest = b.clone()
    lowest[64:200] = torch.finfo(dtype).min
    lowest[t.unique()] = 0.0
    _check(x, w, lowest, t)
    # a label whose class is switched off: infinite loss, as torch
    off[t[3]] = -math.inf
    rows = linear_cross_entropy(x, w, t, off, reduction="none")
    want = torch.nn.functional.cross_entropy(x.float() @ w.float().t() + off.float(), t, reduction="none")
    assert torch.equal(rows.isinf(), want.isinf()) and torch.equal(rows.isnan(), want.isnan()) and bool(rows[3].isinf())
    # every class off: NaN, as torch;  a NaN feature: its row alone
    assert bool(linear_cross_entropy(x, w, t, torch.full_like(b, -math.inf), reduction="none").isnan().all())
    bad = x.clone()
    bad[5, 7] = math.nan
    rows = linear_cross_entropy(bad, w, t, b, reduction="none")
    assert bool(rows[5].isnan()) and int(rows.isnan().sum()) == 1
    # a label that is no class: NaN there, and in the gradients
    for wrong in (300, -1, 1 << 40):
        tt = t.clone()
        tt[9] = wrong
        xg = x.detach().requires_grad_()
        rows = linear_cross_entropy(xg, w, tt, b, reduction="none")
        assert bool(rows[9].isnan()) and int(rows.isnan().sum()) == 1
        (g,) = torch.autograd.grad(linear_cross_entropy(xg, w, tt, b), xg)
        assert bool(g[9].isnan().all())
    # large logits: exp of nothing overflows
    _check(x * 30, w * 30, b, t, reduction="sum")


@pytest.mark.parametrize("want", [(0,), (1,), (2,), (0, 1), (1, 2), (0, 2)])
def test_gradients_that_are_asked_for(want):
    from yolov6_amd.models.losses.loss_ce import linear_cross_entropy
    ops = _inputs(130, 64, 257, torch.bfloat16, True, seed=4)
    _, every = _check(*ops)
    leaves = [o.detach().requires_grad_(k in want) for k, o in enumerate(ops[:3])]
    loss = linear_cross_entropy(leaves[0], leaves[1], ops[3], leaves[2])
    got = torch.autograd.grad(loss, [leaves[k] for k in want], retain_graph=True)
    again = torch.autograd.grad(loss, [leaves[k] for k in want])
    for k, g, a in zip(want, got, again):
        # (fewer gradients may be cut into other tiles: the same sums in another order)
        assert torch.equal(g, a) and float((g.double() - every[k].double()).abs().max()) <= 2.0 ** -7 * float(every[k].abs().max())


def test_gradient_by_differences():
    """Central differences of the double-precision loss at bf16-rounded points are not exact here, so of the fp32 kernel's own loss: an
    fp32 sum of 24 rows is off by 1e-6 of its 60 or so, over a step of 2^-5 by 2e-3 at most."""
    from yolov6_amd.models.losses.loss_ce import linear_cross_entropy
    x, w, b, t = _inputs(24, 16, 40, torch.float32, True, seed=6)
    leaves = [o.detach().requires_grad_() for o in (x, w, b)]
    grads = torch.autograd.grad(linear_cross_entropy(leaves[0], leaves[1], t, leaves[2], reduction="sum", label_smoothing=0.1), leaves)
    g = torch.Generator().manual_seed(1)
    for k in range(3):
        way = torch.randn(leaves[k].shape, generator=g).to(DEV)
        way /= way.norm()
        ends = []
        for h in (2.0 ** -5, -2.0 ** -5):
            moved = [o.detach() + (h * way if i == k else 0) for i, o in enumerate(leaves)]
            ends.append(float(linear_cross_entropy(moved[0], moved[1], t, moved[2], reduction="sum", label_smoothing=0.1)))
        # third derivatives along a unit direction are at most of the order of the logits' cubes: h^2 / 6 of it is within 1e-2
        assert abs((ends[0] - ends[1]) / 2.0 ** -4 - float((grads[k] * way).sum())) <= 2e-3 + 1e-2


def test_same_inputs_same_bits():
    ops = _inputs(1500, 200, 5003, torch.bfloat16, True, seed=8)
    first = _check(*ops)
    for _ in range(2):
        again = _check(*ops)
        assert torch.equal(first[0], again[0]) and all(torch.equal(a, c) for a, c in zip(first[1], again[1]))


def test_once_differentiable():
    from yolov6_amd.models.losses.loss_ce import linear_cross_entropy
    x, w, b, t = _inputs(10, 16, 12, torch.float32, True)
    x.requires_grad_()
    (g,) = torch.autograd.grad(linear_cross_entropy(x, w, t, b), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.sum().backward()


def test_autocast_and_the_torch_op():
    import yolov6_amd.torch_ops  # noqa: F401
    from yolov6_amd.models.losses.loss_ce import linear_cross_entropy
    x, w, b, t = _inputs(100, 40, 333, torch.float32, True, seed=9)
    leaves = [o.detach().requires_grad_() for o in (x, w, b)]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = linear_cross_entropy(leaves[0], leaves[1], t, leaves[2])
    grads = torch.autograd.grad(loss, leaves)
    low = [o.bfloat16() for o in (x, w, b)]
    want, wgrads = _check(*low, t)
    assert torch.equal(loss, want) and all(g.dtype == torch.float32 and torch.equal(g, c.float()) for g, c in zip(grads, wgrads))
    for reduction in ("mean", "none"):
        want, wgrads = _check(*low, t, reduction=reduction)
        leaves = [o.detach().requires_grad_() for o in low]
        loss, _ = torch.ops.yolov6_hip.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2], -100, 0.0, reduction)
        grads = torch.autograd.grad(loss.sum(), leaves)
        assert torch.equal(loss, want) and all(torch.equal(g, c) for g, c in zip(grads, wgrads))
    loss, _ = torch.ops.yolov6_hip.linear_cross_entropy(low[0].requires_grad_(), low[1], t, None, -100, 0.0, "mean")
    assert torch.autograd.grad(loss, low[0])[0].shape == low[0].shape


def test_the_torch_op_under_compile():
    import yolov6_amd.torch_ops  # noqa: F401

    def step(x, w, t, b):
        loss, _ = torch.ops.yolov6_hip.linear_cross_entropy(x * 2, w, t, b, -100, 0.1, "mean")
        return loss * 3

    x, w, b, t = _inputs(64, 48, 200, torch.bfloat16, True, seed=12)
    got = []
    for f in (step, torch.compile(step, backend="aot_eager", fullgraph=True)):
        leaves = [o.detach().requires_grad_() for o in (x, w, b)]
        loss = f(leaves[0], leaves[1], t, leaves[2])
        got.append([loss.detach(), *torch.autograd.grad(loss, leaves)])
    assert all(torch.equal(a, c) for a, c in zip(*got))


def test_another_stream_and_graphs():
    """A side stream; then two captured steps whose replays alternate with eager ones on new inputs."""
    from yolov6_amd.models.losses.loss_ce import linear_cross_entropy

    def step(ops):
        leaves = [o.detach().requires_grad_() for o in ops[:3]]
        loss = linear_cross_entropy(leaves[0], leaves[1], ops[3], leaves[2], label_smoothing=0.1)
        return [loss.detach(), *torch.autograd.grad(loss, leaves)]

    sets = [_inputs(300, 72, 1001, torch.bfloat16, True, seed=20), _inputs(64, 512, 130, torch.bfloat16, True, seed=21)]
    eager = [step(o) for o in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [step(o) for o in sets]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for e, o in zip(eager, other) for a, c in zip(e, o))
    graphs, outs = [], []
    for o in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(o))
        graphs.append(g)
    for turn in range(3):
        for k, o in enumerate(sets):
            fresh = _inputs(o[0].shape[0], o[0].shape[1], o[1].shape[0], torch.bfloat16, True, seed=30 + turn)
            for a, c in zip(o, fresh):
                a.copy_(c)
        for g in graphs:
            g.replay()
        for k, o in enumerate(sets):
            want = step(o)
            torch.cuda.synchronize()
            assert all(torch.equal(a, c) for a, c in zip(outs[k], want)), (turn, k)


def test_a_training_run_of_all_of_them():
    """Backbone features -> linear_cross_entropy under autocast and a loss scale -> clipped FusedSGD step, against torch's operators in double
    precision on the rounded operands: the first step's gradients and update; then the loop runs, skips an overflow and goes on."""
    from yolov6_amd.models.losses.loss_ce import linear_cross_entropy
    from yolov6_amd.solver import FusedSGD, LossScaler, clip_grad_norm_, grad_norm
    from yolov6_amd.train_engine import ParamArena
    torch.manual_seed(0)
    model = torch.nn.Sequential(torch.nn.Linear(32, 64), torch.nn.ReLU(), torch.nn.Linear(64, 500)).to(DEV)
    ref = [p.detach().double().requires_grad_() for p in model.parameters()]
    arena = ParamArena(model)
    opt, scaler = FusedSGD(model, arena, lr=0.1, weight_decay=0.0), LossScaler(DEV, init_scale=1024.0)
    x, t = torch.randn(96, 32, device=DEV), torch.randint(0, 500, (96,), device=DEV)
    t[::5] = -100
    head = model[2]

    def step():
        opt.zero_grad()
        feats = torch.relu(model[0](x))
        with torch.autocast("cuda", dtype=torch.float16):
            loss = linear_cross_entropy(feats, head.weight, t, head.bias, label_smoothing=0.1)
        scaler.scale_loss(loss).backward()
        return loss.detach()

    loss = step()
    h = torch.relu(x.double() @ ref[0].t() + ref[1])
    want = torch.nn.functional.cross_entropy(h.half().double() @ ref[2].half().double().t() + ref[3].half().double(), t, label_smoothing=0.1)
    # (through the straight rounding of h and the head, the gradients are those of the unrounded graph up to fp16: 2^-11 a factor)
    full = torch.nn.functional.cross_entropy(h @ ref[2].t() + ref[3], t, label_smoothing=0.1)
    full.backward()
    assert abs(float(loss) - float(want)) <= 1e-5 * float(want)
    total = float(grad_norm([p.grad for p in model.parameters()])) / 1024
    exact = float(torch.cat([r.grad.reshape(-1) for r in ref]).norm())
    assert abs(total - exact) <= 8 * 2.0 ** -11 * exact
    norm = opt.step(scaler, max_norm=0.5 * exact)
    assert abs(float(norm) - total) <= 2.0 ** -20 * total
    scaler.update()
    for p, r in zip(model.parameters(), ref):
        moved = -0.1 * (1 + 0.937) * 0.5 * r.grad
        assert float((p.detach().double() - r.detach() - moved).norm()) <= 8 * 2.0 ** -11 * float(moved.norm()) + 2.0 ** -22 * float(r.detach().norm())
    for _ in range(3):
        step()
        clip_grad_norm_(model.parameters(), 1.0)
        opt.step(scaler, max_norm=1.0)
        scaler.update()
    before = arena.data.clone()
    step()
    arena.grad[3] = math.inf
    opt.step(scaler, max_norm=1.0)
    scaler.update()
    assert torch.equal(before, arena.data) and float(scaler.scale) == 512.0
    step()
    opt.step(scaler, max_norm=1.0)
    assert not torch.equal(before, arena.data) and bool(torch.isfinite(arena.data).all())


@pytest.mark.parametrize("d", [16, 160])
def test_rows_in_pieces(d):
    """More rows than one piece of the tiles' statistics holds (256 MB)."""
    n, v = 131072 + 300, 33000
    x, w, b, t = _inputs(n, d, v, torch.bfloat16, True, seed=11, ignored=0.0)
    t[-300:] = -100
    t[77] = -100
    from yolov6_amd.models.losses.loss_ce import linear_cross_entropy
    leaves = [o.detach().requires_grad_() for o in (x, w, b)]
    rows = linear_cross_entropy(leaves[0], leaves[1], t, leaves[2], reduction="none")
    up = torch.zeros(n, device=DEV)
    pick = torch.tensor([0, 5, 77, 65535, 65536, 100000, 130000, 131071, 131072 + 5], device=DEV)
    up[pick] = 1.0
    grads = torch.autograd.grad(rows, leaves, up)
    total = linear_cross_entropy(x, w, t, b, reduction="sum")
    err = _logit_error(x, w, b)
    want = torch.cat([torch.nn.functional.cross_entropy(x[k:k + 8192].double() @ w.double().t() + b.double(), t[k:k + 8192], reduction="none")
                      for k in range(0, n, 8192)])
    assert float((rows.detach().double() - want).abs().max()) <= 2 * err
    assert abs(float(total) - float(want.sum())) <= 2 * err * n
    # rows whose upstream gradient is 0 add nothing: the gradients are those of the picked rows alone
    _, exact, spread, soft = _oracle(x[pick], w, b, t[pick], up[pick], reduction="none")
    u = torch.finfo(torch.bfloat16).eps / 2
    others = torch.ones(n, dtype=torch.bool, device=DEV)
    others[pick] = False
    assert int(grads[0][others].count_nonzero()) == 0
    for got, ex, sp, so in zip((grads[0][pick], grads[1], grads[2]), exact, spread, soft):
        kept = u * so if d >= 128 else 0
        assert bool(((got.double() - ex).abs() <= 1.01 * (kept + u * sp + u * ex.abs() + 2 * err * so + v * 2.0 ** -24 * sp + 2.0 ** -19 * so + 2.0 ** -100)).all())


def test_a_weight_beyond_4_gigabytes():
    """Offsets past 32 bits in the weight and its gradient."""
    n, d, v = 5, 16384, 140001
    g = torch.Generator(device=DEV).manual_seed(0)
    w = torch.empty((v, d), dtype=torch.bfloat16, device=DEV)
    for k in range(0, v, 10000):
        w[k:k + 10000] = torch.randn((min(10000, v - k), d), generator=g, device=DEV) / 128
    x = torch.randn((n, d), generator=g, device=DEV).bfloat16().requires_grad_()
    t = torch.tensor([0, 70000, 131072, v - 1, -100], device=DEV)
    w.requires_grad_()
    from yolov6_amd.models.losses.loss_ce import linear_cross_entropy
    loss = linear_cross_entropy(x, w, t, reduction="sum")
    dx, dw = torch.autograd.grad(loss, [x, w])
    z = torch.cat([x.detach().double() @ w.detach()[k:k + 10000].double().t() for k in range(0, v, 10000)], 1)[:4]
    lse = torch.logsumexp(z, 1)
    err = _logit_error(x.detach(), w.detach()[:1000], None) * 1.5
    assert abs(float(loss) - float((lse - z[torch.arange(4), t[:4]]).sum())) <= 8 * err
    dz = torch.exp(z - lse[:, None])
    dz[torch.arange(4), t[:4]] -= 1
    u = torch.finfo(torch.bfloat16).eps / 2
    want = torch.zeros((4, d), dtype=torch.float64, device=DEV)
    spread = torch.zeros_like(want)
    for k in range(0, v, 10000):
        part, xs = dz[:, k:k + 10000], x.detach()[:4].double()
        ex, sp = part.t() @ xs, part.abs().t() @ xs.abs()
        assert bool(((dw[k:k + 10000].double() - ex).abs() <= 1.01 * (u * sp + u * ex.abs() + 2 * err * sp + 2.0 ** -120)).all()), k
        want += part @ w.detach()[k:k + 10000].double()
        spread += part.abs() @ w.detach()[k:k + 10000].double().abs()
    assert bool(((dx[:4].double() - want).abs() <= 1.01 * (u * spread + u * want.abs() + 2 * err * spread + v * 2.0 ** -24 * spread)).all())
    assert int(dx[4].count_nonzero()) == 0


@pytest.mark.parametrize("top", [1.0, 30.0, 1000.0])
def test_small_losses_of_large_logits(top):
    """A label far above the others: the loss is log(1 + sum exp(z - z_t)), whatever z_t is.  Logits are exact here (one feature, values of few
    bits): the sum of exponentials is off by 4 * 2^-24 of itself or so, the loss by that."""
    from yolov6_amd.models.losses.loss_ce import linear_cross_entropy
    for classes in (3, 100, 5000):
        w = torch.full((classes, 1), top - 8.0, device=DEV)
        w[7 % classes] = top
        x, t = torch.ones((2, 1), device=DEV), torch.tensor([7 % classes, 0], device=DEV)
        got = linear_cross_entropy(x, w, t, reduction="none")
        want = torch.log1p((classes - 1) * torch.exp(torch.tensor(-8.0, dtype=torch.float64)))
        assert abs(float(got[0]) - float(want)) <= 8 * 2.0 ** -24 * (1 + float(want)), classes
        assert abs(float(got[1]) - float(want) - (0 if 7 % classes == 0 else 8.0)) <= 8 * 2.0 ** -24 * (9 + float(want))


@pytest.mark.parametrize("smooth", [0.0, 0.1])
@pytest.mark.parametrize("top", [1.0, 30.0, 1000.0])
def test_gradients_of_rows_that_are_almost_right(top, smooth):
    """p - 1 of the label is minus the others' share, which is small and keeps its digits; exact logits as above.  The share is a quotient of sums
    (8 * 2^-24 of itself at most), the smoothing's terms add two roundings of 0.1 at most."""
    from yolov6_amd.models.losses.loss_ce import linear_cross_entropy
    for classes in (3, 100, 5000):
        w = torch.full((classes, 1), top - 12.0, device=DEV)
        w[2] = top
        w.requires_grad_()
        linear_cross_entropy(torch.ones((1, 1), device=DEV), w, torch.tensor([2], device=DEV), label_smoothing=smooth, reduction="sum").backward()
        z = w.detach().double().cpu().flatten()
        p = torch.softmax(z, 0)
        want = p - smooth / classes
        want[2] = -(torch.exp(z[0] - z[2]) * (classes - 1) * p[2]) + smooth - smooth / classes
        off = (w.grad.double().cpu().flatten() - want).abs()
        bound = 16 * 2.0 ** -24 * p + 4 * 2.0 ** -24 * smooth
        bound[2] = 16 * 2.0 ** -24 * (1 - p[2]).abs() + 4 * 2.0 ** -24 * smooth
        assert bool((off <= bound + 1e-30).all()), (classes, off.max(), want[:4])


# rows, width, classes of calls that keep exponentials: whole and odd sizes, tiles of 128 and 256, two pieces, several rows of statistics
KEPT = [(4100, 256, 4200), (300, 264, 60001), (9000, 300, 2101), (2050, 520, 33003)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("reduction,smoothing", [("mean", 0.0), ("none", 0.1)])
@pytest.mark.parametrize("n,d,v", KEPT)
def test_kept_exponentials(n, d, v, reduction, smoothing, dtype):
    x, w, b, t = _inputs(n, d, v, dtype, True, seed=n)
    up = torch.tensor(16.0 * n if dtype == torch.float16 else 1.0, device=DEV)
    if reduction == "none":
        up = torch.linspace(-2, 3, n, device=DEV)
        up[::7] = 0
    _check(x, w, b, t, smoothing, reduction, up, kept=True)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_kept_exponentials_with_masked_classes(dtype):
    """Classes at minus infinity that fill whole tiles, begin and end inside one; large logits; no bias gradient asked for."""
    from yolov6_amd.models.losses.loss_ce import linear_cross_entropy
    n, d, v = 4100, 256, 4200
    x, w, b, t = _inputs(n, d, v, dtype, True, seed=2)
    b[100:1500] = -math.inf
    b[2000:2007] = -math.inf
    t[(t >= 0) & torch.isinf(b[t.clamp(0)])] = 3000
    x[5] *= 30
    _check(x, w, b, t, up=torch.tensor(16.0 * n if dtype == torch.float16 else 1.0, device=DEV), kept=True)
    # a row that is not finite reaches the other rows' dx not at all, and a NaN row is one
    x[7, 3] = math.nan
    t[7] = 2500
    leaf, wl = x.requires_grad_(), w.requires_grad_()
    linear_cross_entropy(leaf, wl, t, b, reduction="sum").backward()
    assert bool(leaf.grad[7].isnan().all()) and bool(leaf.grad[torch.arange(n, device=DEV) != 7].isfinite().all())


def test_kept_exponentials_twice_and_in_a_graph():
    """retain_graph: what the forward kept is not used up; a captured step replayed on new inputs."""
    from yolov6_amd.models.losses.loss_ce import linear_cross_entropy
    n, d, v = 4100, 256, 4200
    x, w, b, t = _inputs(n, d, v, torch.bfloat16, True, seed=4)
    x, w, b = x.requires_grad_(), w.requires_grad_(), b.requires_grad_()
    loss = linear_cross_entropy(x, w, t, b)
    one = torch.autograd.grad(loss, (x, w, b), retain_graph=True)
    two = torch.autograd.grad(loss, (x, w, b))
    assert all(bool((p == q).all()) for p, q in zip(one, two))
    del loss
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.autograd.grad(linear_cross_entropy(x, w, t, b), (x, w, b))
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = torch.autograd.grad(linear_cross_entropy(x, w, t, b), (x, w, b))
    for seed in (5, 6, 7):
        fresh = _inputs(n, d, v, torch.bfloat16, True, seed=seed)
        with torch.no_grad():
            for p, q in zip((x, w, b, t), fresh):
                p.copy_(q)
        g.replay()
        got = [h.clone() for h in held]
        eager = torch.autograd.grad(linear_cross_entropy(x, w, t, b), (x, w, b))
        torch.cuda.synchronize()
        assert all(bool((p == q).all()) for p, q in zip(got, eager)), seed


def test_exponentials_kept_in_part():
    """Over 2 GiB of them: the first pieces are kept, the others formed again; bf16, rows past 32-bit offsets."""
    x, w, b, t = _inputs(20000, 256, 60000, torch.bfloat16, True, seed=9)
    _check(x, w, b, t, kept=True)


def test_capture_beside_a_living_eager_graph_is_refused():
    """The engine would make the capture wait for the eager graph's stream and end the process at the capture's end."""
    from yolov6_amd.models.losses.loss_ce import linear_cross_entropy
    x, w, b, t = _inputs(64, 40, 30, torch.bfloat16, True, seed=6)
    for k in range(3):
        ops = [o.detach().requires_grad_(i == k) for i, o in enumerate((x, w, b))]
        loss = linear_cross_entropy(ops[0], ops[1], t, ops[2])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            torch.zeros(1, device=DEV)
            with pytest.raises(RuntimeError, match="eager graph"):
                linear_cross_entropy(ops[0], ops[1], t, ops[2])
        want = torch.autograd.grad(loss, ops[k])[0]
        del loss
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held = torch.autograd.grad(linear_cross_entropy(ops[0], ops[1], t, ops[2]), ops[k])[0]
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want)


@pytest.mark.parametrize("n,d,v,dtype", [(1101, 136, 4003, torch.float16), (1101, 129, 4003, torch.bfloat16), (523, 71, 1005, torch.float32)])
def test_kept_exponentials_of_odd_sizes(n, d, v, dtype):
    """Just enough of them, in the order of the rows and in another, and each gradient by itself."""
    from yolov6_amd.models.losses.loss_ce import linear_cross_entropy
    assert _keeps(n, d, v, dtype)
    x, w, b, t = _inputs(n, d, v, dtype, True, seed=n)
    up = torch.tensor(16.0 * n if dtype == torch.float16 else 1.0, device=DEV)
    _, every = _check(x, w, b, t, smoothing=0.1, up=up, kept=True)
    u = torch.finfo(dtype).eps / 2
    for k in range(3):
        leaves = [o.detach().requires_grad_(i == k) for i, o in enumerate((x, w, b))]
        (got,) = torch.autograd.grad(linear_cross_entropy(leaves[0], leaves[1], t, leaves[2], label_smoothing=0.1), leaves[k], up)
        # (one gradient alone may be cut into other tiles: the same sums in another order, rounded once)
        assert bool(((got.double() - every[k].double()).abs() <= 2 * u * every[k].double().abs() + 2.0 ** -12 * float(every[k].abs().max())).all())
    _check(x[:, :d - 8].t().contiguous().t(), w[:, 8:], None, t, reduction="sum", up=torch.tensor(4.0, device=DEV), kept=True)
