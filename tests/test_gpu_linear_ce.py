"""linear_cross_entropy on the GPU against F.cross_entropy(F.linear(...)) in double precision on the CPU's definition.

Tolerances.  u = torch.finfo(dtype).eps / 2, products exact, fp32 accumulation.
  loss       the operands are the same in both, so what differs is fp32 arithmetic: a logit's accumulation is off by at most
             width * 2^-24 * sum |x w| <= width * 2^-24 * |x| |w| (worst order), lse and the rest by a few 2^-24 of the largest logit
  gradients  dz is rounded once (u |dz|), the result once (u), both accumulated in fp32.  Norm-wise over a whole gradient:
             |d dx| <= u | |dz| |W| | + u |dx|, so each is held to (|dz| |W|) u + u |dx| + the logits' error, elementwise.
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
    top = float(x.double().norm(dim=1).max()) * float(w.double().norm(dim=1).max()) + (0 if b is None else float(b.abs().max()))
    return e + 8 * 2.0 ** -24 * (top + math.log(w.shape[0]) + 1)


def _check(x, w, b, t, smoothing=0.0, reduction="mean", up=None, ignore=-100):
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
        slack = u * sp + u * ex.abs() + 2 * err * so + length * 2.0 ** -24 * sp + 2 ** -20 * so * 2 + tiny
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
