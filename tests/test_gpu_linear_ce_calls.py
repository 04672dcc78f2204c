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
