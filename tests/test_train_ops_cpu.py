"""Refusals of the training operators that need no GPU: operands are checked before the library is called."""
import math

import pytest
import torch

from yolov6_amd.models.losses.loss_ce import linear_cross_entropy
from yolov6_amd.solver import clip_grad_norm_, grad_norm


def _operands(n=4, d=8, v=5, dtype=torch.float32):
    return torch.zeros(n, d, dtype=dtype), torch.zeros(v, d, dtype=dtype), torch.zeros(n, dtype=torch.int64), torch.zeros(v, dtype=dtype)


def test_linear_cross_entropy_refusals(hip_lib):
    x, w, t, b = _operands()
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        linear_cross_entropy(x, w, t, b)
    for bad, what in (((x.double(), w.double(), t, b.double()), "one type"), ((x.half(), w, t, b), "one type"), ((x, w, t, b.half()), "one type"),
                      ((x, w, t.int(), b), "int64"), ((x[:, :7], w, t, b), "fit together"), ((x, w, t[:3], b), "fit together"),
                      ((x, w, t, b[:4]), "fit together"), ((x, w[0], t, b), "fit together"), ((x, w[:0], t, b[:0]), "no class"),
                      ((x[:, :0], w[:, :0], t, b), "no class")):
        with pytest.raises(RuntimeError, match=what):
            linear_cross_entropy(*bad)
    with pytest.raises(RuntimeError, match="reduction"):
        linear_cross_entropy(x, w, t, b, reduction="batchmean")
    for e in (-0.1, 1.5, math.nan):
        with pytest.raises(RuntimeError, match="label_smoothing"):
            linear_cross_entropy(x, w, t, b, label_smoothing=e)


def test_native_refusals(hip_lib):
    """The C entry's own checks, before anything is launched."""
    import ctypes as C
    from yolov6_amd import _lib
    d = _lib.LinearCeDesc()
    d.x = d.weight = d.target = d.loss = d.grad_out = d.dx = 4096
    d.rows, d.width, d.classes, d.x_pitch, d.w_pitch, d.reduction = 4, 8, 5, 8, 8, 2
    assert hip_lib.y6_linear_ce_workspace_bytes(C.byref(d), 0) > 0 and hip_lib.y6_linear_ce_workspace_bytes(C.byref(d), 1) > 0
    d.workspace, d.workspace_bytes = 4096, 16
    assert hip_lib.y6_linear_ce_backward(C.byref(d), None) == -1 and b"null" in hip_lib.y6_last_error()
    d.saved, d.saved_bytes = 4096, 1 << 20
    for call in (hip_lib.y6_linear_ce_forward, hip_lib.y6_linear_ce_backward):
        assert call(C.byref(d), None) == -1 and b"workspace" in hip_lib.y6_last_error()
    for field, value, what in (("dtype", 2, b"dtype"), ("rows", 0, b"rows"), ("classes", 0, b"classes"), ("width", 0, b"wide"), ("w_pitch", 7, b"pitch"),
                               ("smoothing", 1.5, b"smoothing"), ("reduction", 5, b"reduction"), ("weight", 4097, b"aligned"), ("x", None, b"null")):
        keep = getattr(d, field)
        setattr(d, field, value)
        assert hip_lib.y6_linear_ce_forward(C.byref(d), None) == -1 and what in hip_lib.y6_last_error(), field
        assert hip_lib.y6_linear_ce_workspace_bytes(C.byref(d), 1) == 0
        setattr(d, field, keep)
    d.workspace_bytes, d.saved_bytes = 1 << 20, 16
    for call in (hip_lib.y6_linear_ce_forward, hip_lib.y6_linear_ce_backward):
        assert call(C.byref(d), None) == -1 and b"saved" in hip_lib.y6_last_error()
    lst = _lib.GradList((C.c_void_p * 2)(4096, 4100), (C.c_int64 * 2)(8, 8), (C.c_int32 * 2)(1, 1), 2, 0)
    assert hip_lib.y6_grad_clip(C.byref(lst), 1.0, 4096, 1 << 20, 4096, None) == -1 and b"share memory" in hip_lib.y6_last_error()
    assert hip_lib.y6_grad_clip(C.byref(lst), -1.0, 4096, 1 << 20, 4096, None) == -1 and b"max_norm" in hip_lib.y6_last_error()
    assert hip_lib.y6_grad_norm(C.byref(lst), 4096, 8, 4096, None) == -1 and b"workspace" in hip_lib.y6_last_error()
    lst.norm_type = 7
    assert hip_lib.y6_grad_norm(C.byref(lst), 4096, 1 << 20, 4096, None) == -1 and b"norm" in hip_lib.y6_last_error()


def test_gradient_refusals(hip_lib):
    p = torch.nn.Parameter(torch.zeros(4))
    p.grad = torch.zeros(4)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        clip_grad_norm_([p], 1.0)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        grad_norm([p.grad])
    with pytest.raises(RuntimeError, match="type"):
        grad_norm([p.grad], 0.5)
    with pytest.raises(RuntimeError, match="max_norm"):
        clip_grad_norm_([p], -2.0)
    with pytest.raises(RuntimeError, match="fp16, bf16 or fp32"):
        grad_norm([p.grad.double()])
    assert float(clip_grad_norm_([torch.nn.Parameter(torch.zeros(4))], 1.0)) == 0.0



def test_forward_mode_is_refused(hip_lib):
    """A dual operand's tangent would vanish: refused before anything else is looked at."""
    x, w, t, b = _operands()
    with torch.autograd.forward_ad.dual_level():
        for k in range(3):
            ops = [torch.autograd.forward_ad.make_dual(o, torch.ones_like(o)) if i == k else o for i, o in enumerate((x, w, b))]
            with pytest.raises(RuntimeError, match="forward mode"):
                linear_cross_entropy(ops[0], ops[1], t, ops[2])
            with pytest.raises(RuntimeError, match="forward mode"):
                grad_norm([ops[k]])


def test_a_copied_weight_is_a_larger_saved_buffer(hip_lib):
    """What the host side goes by when a weight comes back from saved-tensor hooks at another address."""
    import ctypes as C
    from yolov6_amd import _lib
    for dtype in (0, 1, 3):
        for rows, width, classes, pitch, at in ((1, 8, 1, 8, 4096), (4, 8, 5, 8, 4096), (4, 8, 5, 8, 4100), (4, 7, 5, 9, 4096), (3000, 512, 4096, 512, 1 << 20)):
            d = _lib.LinearCeDesc()
            d.x = d.target = 4096
            d.weight, d.rows, d.width, d.classes, d.x_pitch, d.w_pitch, d.dtype = at, rows, width, classes, width, pitch, dtype
            plain = hip_lib.y6_linear_ce_saved_bytes(C.byref(d))
            d.flags = 1
            copied = hip_lib.y6_linear_ce_saved_bytes(C.byref(d))
            needs = dtype == 1 or (width * 2) % 16 or (pitch * 2) % 16 or at % 16
            assert plain > 0 and (copied == plain if needs else copied >= plain + classes * width * 2)
            d.weight, d.w_pitch = 8192, width
            assert hip_lib.y6_linear_ce_saved_bytes(C.byref(d)) == copied


def test_recompute_keeps_nothing_of_rows_by_classes(hip_lib):
    import ctypes as C
    from yolov6_amd import _lib
    for dtype, size in ((0, 2), (1, 4), (3, 2)):
        d = _lib.LinearCeDesc()
        d.x = d.target = d.weight = 4096
        d.rows, d.width, d.classes, d.x_pitch, d.w_pitch, d.dtype = 8192, 512, 8192, 512, 512, dtype
        kept = hip_lib.y6_linear_ce_saved_bytes(C.byref(d))
        d.flags = 2
        without = hip_lib.y6_linear_ce_saved_bytes(C.byref(d))
        assert kept >= 8192 * 8192 * size and 0 < without <= 2 * 8192 * 512 * 6 + (1 << 20)


def test_sizes_whose_launches_would_leave_32_bits_are_refused(hip_lib):
    """Up to 2^30 rows were accepted; a launch of theirs has 2^36 threads.  The largest that are taken, and one more."""
    import ctypes as C
    from yolov6_amd import _lib
    d = _lib.LinearCeDesc()
    d.x = d.target = d.weight = 4096
    d.width = d.x_pitch = d.w_pitch = 8
    for rows, classes, good in (((1 << 26) - 16, 5, True), ((1 << 26) - 15, 5, False), (1 << 30, 2, False), (4, (1 << 30) - 512, True), (4, 1 << 30, False)):
        d.rows, d.classes = rows, classes
        for size in (hip_lib.y6_linear_ce_saved_bytes(C.byref(d)), hip_lib.y6_linear_ce_workspace_bytes(C.byref(d), 0), hip_lib.y6_linear_ce_workspace_bytes(C.byref(d), 1)):
            assert (size > 0) == good, (rows, classes)
        if not good:
            assert b"rows" in hip_lib.y6_last_error()


def test_sparse_gradients_are_refused(hip_lib):
    p = torch.nn.Parameter(torch.zeros(4, 3))
    p.grad = torch.sparse_coo_tensor([[1]], [[1.0, 2.0, 3.0]], (4, 3))
    for call in (lambda: clip_grad_norm_([p], 1.0), lambda: grad_norm([p.grad])):
        with pytest.raises(RuntimeError, match="dense"):
            call()
