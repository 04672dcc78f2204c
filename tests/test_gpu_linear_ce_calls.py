"""Calls of linear_cross_entropy that its documentation allows, beside those of test_gpu_linear_ce.py: where no tolerance is named, results
are compared bit for bit with those of a call that is tested there.  Elsewhere the tolerances are that file's (_check)."""
import math

import pytest
import torch

from tests.test_gpu_linear_ce import DEV, _check, _inputs

pytestmark = pytest.mark.gpu


def _loss(leaves, t, **options):
    from yolov6_amd.models.losses.loss_ce import linear_cross_entropy
    return linear_cross_entropy(leaves[0], leaves[1], t, leaves[2], **options)


def _op_loss(leaves, t, *options):
    import yolov6_amd.torch_ops  # noqa: F401
    return torch.ops.yolov6_hip.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2], *(options or (-100, 0.0, "mean")))[0]


def _leaves(ops, *dtypes):
    return [o.detach().clone().to(k).requires_grad_() for o, k in zip(ops[:3], dtypes * 3 if len(dtypes) == 1 else dtypes)]


@pytest.mark.parametrize("compiled", [False, True])
@pytest.mark.parametrize("amp", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dtypes", [(torch.float32,), (torch.float16, torch.float32, torch.float32), (torch.bfloat16, torch.float32, torch.float16)])
def test_the_op_under_autocast(dtypes, amp, compiled):
    """Forward in the region, backward outside it, as a training loop has them: the bits of the plain function, gradients in the leaves' types."""
    ops = _inputs(100, 40, 333, torch.float32, True, seed=9)
    t = ops[3]
    want = _leaves(ops, *dtypes)
    with torch.autocast("cuda", dtype=amp):
        loss = _loss(want, t)
    grads = torch.autograd.grad(loss * 64, want)
    f = torch.compile(lambda x, w, b, t: _op_loss((x, w, b), t), backend="aot_eager", fullgraph=True) if compiled else lambda x, w, b, t: _op_loss((x, w, b), t)
    got = _leaves(ops, *dtypes)
    with torch.autocast("cuda", dtype=amp):
        op_loss = f(*got, t)
    op_grads = torch.autograd.grad(op_loss * 64, got)
    assert torch.equal(op_loss, loss) and all(a.dtype == c.dtype == o.dtype and torch.equal(a, c) for a, c, o in zip(op_grads, grads, got))


def test_the_op_backward_inside_autocast():
    """The region of the backward changes nothing: the operands are those of the forward."""
    ops = _inputs(100, 40, 333, torch.float32, True, seed=10)
    leaves = _leaves(ops, torch.float32)
    want = torch.autograd.grad(_loss(leaves, ops[3]), leaves)
    for f in (_loss, _op_loss):
        loss = f(leaves, ops[3])
        with torch.autocast("cuda", dtype=torch.bfloat16):
            got = torch.autograd.grad(loss, leaves)
        assert all(torch.equal(a, c) for a, c in zip(got, want))


def test_forward_mode_is_refused_by_the_op():
    ops = _inputs(10, 16, 12, torch.float32, True)
    with torch.autograd.forward_ad.dual_level():
        for k in range(3):
            duals = [torch.autograd.forward_ad.make_dual(o, torch.ones_like(o)) if i == k else o for i, o in enumerate(ops[:3])]
            for f in (_loss, _op_loss):
                with pytest.raises(RuntimeError, match="forward mode"):
                    f(duals, ops[3])


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,d,v", [(150, 96, 333), (4100, 256, 4200)])
def test_an_upstream_gradient_that_is_not_finite_stays_in_its_row(n, d, v, dtype, bad):
    """reduction none, as F.cross_entropy: the row's dx and the sums over all rows (dW, db) are not finite, the other rows' dx are theirs."""
    ops = _inputs(n, d, v, dtype, True, seed=3, ignored=0.2)
    t = ops[3]
    t[5] = 7
    up = torch.linspace(-2, 3, n, device=DEV)
    up[5] = 0.0
    leaves = _leaves(ops, dtype)
    want = torch.autograd.grad(_loss(leaves, t, reduction="none"), leaves, up)
    up[5] = bad
    got = torch.autograd.grad(_loss(leaves, t, reduction="none"), leaves, up)
    others = torch.arange(n, device=DEV) != 5
    assert torch.equal(got[0][others], want[0][others]) and not bool(got[0][5].isfinite().any())
    assert not bool(got[1].isfinite().any()) and not bool(got[2].isfinite().any())
    # all of them, and beside zeros only
    for value in (bad, 0.0):
        up = torch.full((n,), value, device=DEV)
        up[5] = bad
        got = torch.autograd.grad(_loss(leaves, t, reduction="none"), leaves, up)
        labelled = t != -100
        rows = labelled if value != 0.0 else ~others
        assert not bool(got[0][rows].isfinite().any()) and int(got[0][~rows].count_nonzero()) == 0


@pytest.mark.parametrize("n", [4096, 4097, 8192 + 15, 600_001, 1 << 20, (1 << 20) + 1, (1 << 22) + 4097])
@pytest.mark.parametrize("share", [0.0, 0.5, 0.999])
def test_many_rows(n, share):
    """Labelled rows are counted block by block: two classes and one feature, so that value and gradient have closed forms, at rows before, at
    and behind the borders of those blocks.  Logits +-x/2 of few bits: loss log(1 + exp(-+x)), off by 8 * 2^-24 of 1 + its size."""
    g = torch.Generator(device=DEV).manual_seed(n)
    x = (torch.randint(-64, 65, (n, 1), generator=g, device=DEV) / 16.0).requires_grad_()
    w = torch.tensor([[0.5], [-0.5]], device=DEV)
    t = torch.randint(0, 2, (n,), generator=g, device=DEV)
    t[torch.rand(n, generator=g, device=DEV) < share] = -100
    rows = _loss((x, w, None), t, reduction="none")
    (dx,) = torch.autograd.grad(rows, x, torch.ones_like(rows))
    z = x.detach().double().flatten() * torch.where(t == 1, -1.0, 1.0)           # label's logit - the other's
    want = torch.where(t == -100, torch.zeros_like(z), torch.nn.functional.softplus(-z, threshold=100.0))
    assert bool(((rows.detach().double() - want).abs() <= 8 * 2.0 ** -24 * (1 + want)).all())
    slope = torch.where(t == -100, torch.zeros_like(z), -torch.sigmoid(-z) * torch.where(t == 1, -1.0, 1.0))
    # two products of a probability (8 * 2^-24 of it) and 0.5, exact; the two planes' sums in fp32
    assert bool(((dx.double().flatten() - slope).abs() <= 16 * 2.0 ** -24 * slope.abs() + 2.0 ** -100).all())
    total = _loss((x.detach(), w, None), t, reduction="sum")
    assert abs(float(total) - float(want.sum())) <= 8 * 2.0 ** -24 * float((1 + want).sum()) + 2.0 ** -24 * float(want.sum())
    assert torch.equal(total.isfinite(), torch.ones((), dtype=torch.bool, device=DEV))


def test_time_grows_with_the_rows():
    """Eight times the rows take about eight times as long: a count that every block makes for itself takes sixty-four."""
    def us(n):
        x = torch.zeros((n, 8), dtype=torch.float16, device=DEV)
        w, t = torch.zeros((2, 8), dtype=torch.float16, device=DEV), torch.zeros(n, dtype=torch.int64, device=DEV)
        best = math.inf
        for _ in range(4):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            _loss((x, w, None), t, reduction="none")
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b) * 1000)
        return best
    times = [us(n) for n in (1 << 20, 1 << 23)]
    print("us", times)
    assert times[1] <= 16 * times[0], times


def test_bias_gradient_of_many_rows_with_kept_exponentials():
    """Thousands of partial sums of a class: joined in a fixed order, and right."""
    x, w, b, t = _inputs(100_003, 128, 1040, torch.bfloat16, True, seed=17)
    first = _check(x, w, b, t, reduction="sum", kept=True)
    leaves = _leaves((x, w, b), torch.bfloat16)
    again = torch.autograd.grad(_loss(leaves, t, reduction="sum"), leaves)
    assert all(torch.equal(a, c) for a, c in zip(first[1], again))


class _Misplaced(torch.autograd.graph.saved_tensors_hooks):
    """Hands every saved tensor back one element behind the start of a wider buffer."""

    def __init__(self):
        def unpack(t):
            if t.dim() != 2:
                return t
            buf = torch.zeros((t.shape[0], t.shape[1] + 3), dtype=t.dtype, device=t.device)
            buf[:, 1:1 + t.shape[1]] = t
            return buf[:, 1:1 + t.shape[1]]
        super().__init__(lambda t: t, unpack)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,d,v,cut", [(70, 40, 130, 0), (70, 40, 130, 1), (70, 37, 130, 0), (40, 136, 110_003, 0), (40, 136, 110_003, 3)])
@pytest.mark.parametrize("hooks", [torch.autograd.graph.save_on_cpu, _Misplaced])
@pytest.mark.parametrize("form", [_loss, _op_loss])
def test_operands_that_come_back_elsewhere(form, hooks, n, d, v, cut, dtype):
    """Saved-tensor hooks hand the backward the same values at other addresses and pitches: the same bits."""
    ops = _inputs(n, d + cut, v, dtype, True, seed=d)
    x, w = (o[:, cut:].detach().requires_grad_() for o in ops[:2])       # (views of a wider buffer: other pitch, odd start)
    leaves = (x, w, ops[2].detach().requires_grad_())
    want = torch.autograd.grad(_loss(leaves, ops[3]), leaves)
    with hooks():
        loss = form(leaves, ops[3])
    got = torch.autograd.grad(loss, leaves)
    assert all(torch.equal(a, c) for a, c in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_the_features_go_when_the_caller_drops_them(dtype):
    """The backward reads the labelled rows as the forward gathered them: an activation lives no longer than its caller keeps it."""
    ops = _inputs(4000, 500, 30, dtype, True, seed=3)
    leaves = _leaves(ops, dtype)
    want = torch.autograd.grad(_loss(leaves, ops[3]), leaves)
    feats = leaves[0] + 0
    loss = _loss((feats, *leaves[1:]), ops[3])
    torch.cuda.synchronize()
    held, size = torch.cuda.memory_allocated(), feats.numel() * feats.element_size()
    del feats
    assert held - torch.cuda.memory_allocated() >= size
    assert all(torch.equal(a, c) for a, c in zip(torch.autograd.grad(loss, leaves), want))


@pytest.mark.parametrize("how", ["backward", "grad"])
def test_capture_beside_a_living_graph_of_a_side_stream(how):
    """Warm-up on a side stream whose loss is still held, as in torch's recipe: that stream joins the capture.  Replays alternate with eager
    steps on new inputs."""
    x, w, b, t = _inputs(64, 40, 300, torch.bfloat16, True, seed=6)
    leaves = _leaves((x, w, b), torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        loss = _loss(leaves, t)
        loss.backward()
    torch.cuda.current_stream().wait_stream(side)
    for o in leaves:
        o.grad = None
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        inner = _loss(leaves, t)
        if how == "backward":
            inner.backward()
            held = [o.grad for o in leaves]
        else:
            held = torch.autograd.grad(inner, leaves)
    for seed in (7, 8, 9):
        fresh = _inputs(64, 40, 300, torch.bfloat16, True, seed=seed)
        with torch.no_grad():
            for p, q in zip((*leaves, t), fresh):
                p.copy_(q)
        g.replay()
        torch.cuda.synchronize()
        others = _leaves(leaves, torch.bfloat16)
        want = torch.autograd.grad(_loss(others, t), others)
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(held, want)), seed
    assert math.isfinite(float(loss.detach()))


def test_the_op_captured_beside_a_living_eager_graph_is_refused():
    x, w, b, t = _inputs(64, 40, 30, torch.bfloat16, True, seed=6)
    for k in range(3):
        ops = [o.detach().requires_grad_(i == k) for i, o in enumerate((x, w, b))]
        loss = _op_loss(ops, t)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            torch.zeros(1, device=DEV)
            with pytest.raises(RuntimeError, match="eager graph"):
                _op_loss(ops, t)
            with pytest.raises(RuntimeError, match="eager graph"), torch.autocast("cuda", dtype=torch.float16):
                _op_loss(ops, t)
            with torch.no_grad():
                value = _op_loss(ops, t)                     # no gradient, no accumulator
        want = torch.autograd.grad(loss, ops[k])[0]
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(value, loss.detach())
        del loss
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held = torch.autograd.grad(_op_loss(ops, t), ops[k])[0]
        for _ in range(3):
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(held, want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("reduction,smoothing", [("mean", 0.0), ("none", 0.1)])
def test_recompute(dtype, reduction, smoothing, monkeypatch):
    """Nothing of [rows, classes] is kept, and the gradients have one rounding less: the tolerance is that of calls that keep nothing."""
    from functools import partial
    from yolov6_amd.models.losses import loss_ce
    n, d, v = 4100, 264, 4200
    ops = _inputs(n, d, v, dtype, True, seed=n)
    up = torch.tensor(16.0 * n if dtype == torch.float16 else 1.0, device=DEV)
    if reduction == "none":
        up = torch.linspace(-2, 3, n, device=DEV)
    logits = n * v * ops[0].element_size()
    leaves = _leaves(ops, dtype)
    for recompute in (False, True):
        for form in (_loss, _op_loss):
            before = torch.cuda.memory_allocated()
            if form is _loss:
                loss = _loss(leaves, ops[3], recompute=recompute)
            else:
                loss = _op_loss(leaves, ops[3], -100, 0.0, "mean", recompute)
            torch.cuda.synchronize()
            held = torch.cuda.memory_allocated() - before
            assert held < logits / 2 if recompute else held >= logits
            del loss
    monkeypatch.setattr(loss_ce, "linear_cross_entropy", partial(loss_ce.linear_cross_entropy, recompute=True))
    _, want = _check(*ops, smoothing, reduction, up, kept=False)
    loss = _op_loss(leaves, ops[3], -100, smoothing, reduction, True)
    got = torch.autograd.grad(loss, leaves, up)
    assert all(torch.equal(a, c) for a, c in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,d,v", [(70, 32, 300), (300, 64, 1500), (2100, 72, 33000), (4100, 256, 4200)])
def test_classes_at_the_lowest_value_fill_tiles(n, d, v, dtype):
    """A bias of the type's lowest value switches classes off, whole tiles of them: finite everywhere, with and without gradients.  All of them
    at it: as likely as each other, log(classes), off by 8 * 2^-24 of 1 + that.  One at the highest: 0 or that value."""
    x, w, b, t = _inputs(n, d, v, dtype, True, seed=v)
    lo, hi = 20, v - 30
    b[lo:hi] = torch.finfo(dtype).min
    t[(t >= lo) & (t < hi)] = 5
    _check(x, w, b, t, kept=(d >= 128))
    rows = _loss((x, w, b), t, reduction="none")
    want = torch.nn.functional.cross_entropy(x.double() @ w.double().t() + b.double(), t, reduction="none")
    from tests.test_gpu_linear_ce import _logit_error
    assert bool(((rows.double() - want).abs() <= 2 * _logit_error(x, w, b)).all())
    every = torch.full_like(b, torch.finfo(dtype).min)
    rows = _loss((x, w, every), t, reduction="none")
    want = torch.where(t == -100, 0.0, math.log(v))
    assert bool(((rows.double() - want).abs() <= 8 * 2.0 ** -24 * (1 + want)).all())
    one = torch.zeros_like(b)
    one[lo] = torch.finfo(dtype).max
    t[::3] = lo
    rows = _loss((x / 64, w, one), t, reduction="none")
    want = torch.where((t == -100) | (t == lo), 0.0, torch.finfo(dtype).max)
    assert bool(((rows.double() - want).abs() <= 2.0 ** -23 * want).all())


_FIRST = """
import torch
from yolov6_amd import clip_grad_norm_, linear_cross_entropy
x, w, b, t = (torch.randn(4100, 256, device="cuda").{t}(), torch.randn(4200, 256, device="cuda").mul(0.1).{t}(), torch.randn(4200, device="cuda").{t}(),
              torch.randint(0, 4200, (4100,), device="cuda"))
leaves = [o.requires_grad_() for o in (x, w, b)]
p = torch.nn.Parameter(torch.zeros(1000, device="cuda"))
first = torch.randn(1000, device="cuda")
p.grad = first.clone()
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    held = torch.autograd.grad(linear_cross_entropy(x, w, t, b), leaves)
    norm = clip_grad_norm_([p], 1.0)
for _ in range(3):
    p.grad.copy_(first)
    g.replay()
    torch.cuda.synchronize()
    want = torch.autograd.grad(linear_cross_entropy(x, w, t, b), leaves)
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(held, want))
    assert abs(float(norm) - float(first.double().norm())) <= 2.0 ** -23 * float(norm)
print("as the first call")
"""


@pytest.mark.parametrize("dtype", ["bfloat16", "float"])
def test_captured_as_the_first_call_of_a_process(dtype):
    """No warm-up: the library, its kernels' limits and the extension come up inside the capture."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", _FIRST.replace("{t}", dtype)], cwd=root, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "as the first call" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]


@pytest.mark.parametrize("which", ["weight", "saved", "bias"])
@pytest.mark.parametrize("change", ["host", "shape", "type"])
def test_what_a_hook_must_not_hand_back(which, change):
    """Another device, shape or type than it was given: refused before anything is launched."""
    ops = _inputs(64, 40, 50, torch.bfloat16, True, seed=3)
    leaves = _leaves(ops, torch.bfloat16)

    def unpack(t):
        mine = {"weight": t.dim() == 2, "saved": t.dtype == torch.uint8, "bias": t.dim() == 1 and t.dtype == torch.bfloat16}[which]
        return t if not mine else t.cpu() if change == "host" else t[:-1] if change == "shape" else t.half() if t.dtype != torch.uint8 else t.to(torch.int8)

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        loss = _loss(leaves, ops[3])
    with pytest.raises(RuntimeError, match="yolov6_amd"):
        torch.autograd.grad(loss, leaves)
    torch.cuda.synchronize()


def test_what_the_backward_op_refuses():
    import yolov6_amd.torch_ops  # noqa: F401
    x, w, b, t = _inputs(64, 40, 50, torch.bfloat16, True, seed=3)
    loss, saved = torch.ops.yolov6_hip.linear_cross_entropy(x, w, t, b, -100, 0.0, "none")
    back = torch.ops.yolov6_hip.linear_cross_entropy_backward
    good = torch.ones_like(loss)
    back(good, x, w, t, b, saved, -100, 0.0, "none", False)
    for grad, kept in ((good[:-1], saved), (good.cpu(), saved), (good, saved.cpu()), (good, saved[:-256]), (good, saved[::2]), (good, saved.to(torch.int8)),
                       (torch.ones((), device=DEV), saved)):
        with pytest.raises(RuntimeError, match="yolov6_amd"):
            back(grad, x, w, t, b, kept, -100, 0.0, "none", False)
    torch.cuda.synchronize()
