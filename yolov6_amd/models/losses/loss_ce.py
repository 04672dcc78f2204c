"""Softmax cross entropy of a linear classifier over many classes: value and gradients without keeping the logits.

    loss = linear_cross_entropy(features, weight, target, bias)     # = F.cross_entropy(F.linear(features, weight, bias), target)
    loss.backward()

For classifiers whose [rows, classes] logits are what fills the memory and the time of a step: pretraining the backbone on a large
label set, dense labels with a large vocabulary.  The detection losses (loss.py) keep their sigmoid scores.  The reference has no
softmax classifier; the semantics are torch's, except that the mean over no labelled row is 0 (as ComputeLoss's terms are without
targets), not a NaN.  Kernels: csrc/linear_ce.hip (y6_linear_ce_forward / _backward).
"""
import ctypes as C

import torch

from ... import _lib

_TYPES = {torch.float16: _lib.Y6_F16, torch.bfloat16: _lib.Y6_BF16, torch.float32: _lib.Y6_F32}
_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def _ptr(t):
    return None if t is None else t.data_ptr()


def _desc(x, weight, bias, target, ignore_index, smoothing, reduction):
    n, d = x.shape
    desc = _lib.LinearCeDesc()
    desc.x, desc.weight, desc.bias, desc.target = _ptr(x), _ptr(weight), _ptr(bias), _ptr(target)
    desc.rows, desc.width, desc.classes, desc.dtype = n, d, weight.shape[0], _TYPES[x.dtype]
    desc.x_pitch = x.stride(0) if n > 1 else d
    desc.w_pitch = weight.stride(0) if weight.shape[0] > 1 else d
    desc.ignore_index, desc.smoothing, desc.reduction = ignore_index, smoothing, reduction
    return desc


def _call(name, desc, backward):
    lib = _lib.load()
    size = lib.y6_linear_ce_workspace_bytes(C.byref(desc), backward)
    if size == 0:
        _lib.check(-1, name)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")          # (the callers have made x's device the current one)
    desc.workspace, desc.workspace_bytes = ws.data_ptr(), size
    _lib.check(getattr(lib, f"y6_linear_ce_{name}")(C.byref(desc), _lib.current_stream_ptr()), f"linear_ce_{name}")


def _forward(x, weight, bias, target, ignore_index, smoothing, reduction, want_lse):
    """(loss, lse or None) of checked operands."""
    n = x.shape[0]
    if n == 0:
        return x.new_zeros((0,) if reduction == 0 else (), dtype=torch.float32), None
    with torch.cuda.device(x.device):
        loss = torch.empty((n,) if reduction == 0 else (), dtype=torch.float32, device=x.device)
        lse = torch.empty(n, dtype=torch.float32, device=x.device) if want_lse else None
        desc = _desc(x, weight, bias, target, ignore_index, smoothing, reduction)
        desc.loss, desc.lse = _ptr(loss), _ptr(lse)
        _call("forward", desc, 0)
    return loss, lse


def _backward(grad, x, weight, bias, target, lse, ignore_index, smoothing, reduction, want):
    """Gradients of (x, weight, bias), None where `want` says so."""
    n, d = x.shape
    if n == 0:
        return tuple(torch.zeros_like(t) if w and t is not None else None for t, w in zip((x, weight, bias), want))
    with torch.cuda.device(x.device):
        dx = torch.empty((n, d), dtype=x.dtype, device=x.device) if want[0] else None
        dw = torch.empty(weight.shape, dtype=x.dtype, device=x.device) if want[1] else None
        db = torch.empty(weight.shape[0], dtype=x.dtype, device=x.device) if want[2] and bias is not None else None
        if dx is None and dw is None and db is None:
            return None, None, None
        grad = grad.to(torch.float32).contiguous()
        desc = _desc(x, weight, bias, target, ignore_index, smoothing, reduction)
        desc.lse, desc.grad_out, desc.dx, desc.dw, desc.dbias = _ptr(lse), _ptr(grad), _ptr(dx), _ptr(dw), _ptr(db)
        _call("backward", desc, 1)
    return dx, dw, db


class _LinearCrossEntropyFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, target, ignore_index, smoothing, reduction):
        need = any(ctx.needs_input_grad[:3])
        loss, lse = _forward(x, weight, bias, target, ignore_index, smoothing, reduction, need)
        if need:
            ctx.save_for_backward(x, weight, bias, target, lse)
            ctx.options = (ignore_index, smoothing, reduction)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        x, weight, bias, target, lse = ctx.saved_tensors
        return (*_backward(grad, x, weight, bias, target, lse, *ctx.options, ctx.needs_input_grad[:3]), None, None, None, None)


def _rows_dense(t):
    """t with its last dimension dense and its rows apart: the view itself where it is that."""
    if t.shape[1] > 1 and t.stride(1) != 1:
        return t.contiguous()
    return t


def _checked(features, weight, target, bias, label_smoothing, reduction):
    """Operands as the kernels take them: features [rows, width], weight [classes, width], target [rows]."""
    if reduction not in _REDUCTIONS:
        raise RuntimeError(f"yolov6_amd: linear_cross_entropy reduction {reduction!r} ('mean', 'sum' or 'none')")
    if not 0.0 <= label_smoothing <= 1.0:
        raise RuntimeError(f"yolov6_amd: linear_cross_entropy label_smoothing {label_smoothing} is not in [0, 1]")
    if features.dtype not in _TYPES or weight.dtype != features.dtype or (bias is not None and bias.dtype != features.dtype):
        raise RuntimeError("yolov6_amd: linear_cross_entropy takes features, weight and bias of one type, fp16, bf16 or fp32 (got "
                           f"{features.dtype}, {weight.dtype}{'' if bias is None else f', {bias.dtype}'})")
    if target.dtype != torch.int64:
        raise RuntimeError(f"yolov6_amd: linear_cross_entropy labels are int64 (got {target.dtype})")
    if features.dim() < 1 or weight.dim() != 2 or features.shape[-1] != weight.shape[1] or target.shape != features.shape[:-1] or \
            (bias is not None and tuple(bias.shape) != (weight.shape[0],)):
        raise RuntimeError(f"yolov6_amd: linear_cross_entropy features {tuple(features.shape)}, weight {tuple(weight.shape)}, target "
                           f"{tuple(target.shape)}{'' if bias is None else f', bias {tuple(bias.shape)}'} do not fit together")
    if weight.shape[0] < 1 or weight.shape[1] < 1:
        raise RuntimeError(f"yolov6_amd: linear_cross_entropy weight {tuple(weight.shape)} has no class or no column")
    for name, t in (("features", features), ("weight", weight), ("target", target), ("bias", bias)):
        if t is not None:
            _lib.require_gpu_tensor(t, name)
            if t.device != features.device:
                raise RuntimeError(f"yolov6_amd: linear_cross_entropy {name} on {t.device}, features on {features.device}")


def linear_cross_entropy(features, weight, target, bias=None, *, ignore_index=-100, label_smoothing=0.0, reduction="mean"):
    """F.cross_entropy(F.linear(features, weight, bias), target, ...) without the logits.

    features [..., width], weight [classes, width], bias [classes] or None, in one type (fp16, bf16, fp32; under autocast they are cast
    to its type); target [...] int64.  Returns fp32: a scalar ('mean' over the labelled rows, 'sum'), or [...] ('none').  Gradients
    come in the operands' type, once differentiable; under a loss scale (LossScaler) as usual.  Rows labelled ignore_index have loss
    0, a zero gradient, and are not read: a NaN in them goes nowhere.  A label that is neither a class nor ignore_index makes its
    row's loss and the gradients NaN (no host check: nothing synchronises).  Products of 16-bit operands accumulate in fp32; the
    gradient of the logits is rounded to the operands' type once, where the matrix instructions of the two gradient products take
    it.  Works on any view with a dense last dimension; others are copied."""
    if torch.is_autocast_enabled("cuda"):
        dtype = torch.get_autocast_dtype("cuda")
        features, weight, bias = features.to(dtype), weight.to(dtype), None if bias is None else bias.to(dtype)
    _checked(features, weight, target, bias, label_smoothing, reduction)
    x = _rows_dense(features.reshape(-1, features.shape[-1]))
    w = _rows_dense(weight)
    if w.shape[0] > 1 and w.stride(0) < w.shape[1]:
        w = w.contiguous()                                   # an expanded weight
    b = None if bias is None else bias.contiguous()
    loss = _LinearCrossEntropyFn.apply(x, w, b, target.reshape(-1).contiguous(), int(ignore_index), float(label_smoothing), _REDUCTIONS[reduction])
    return loss.reshape(target.shape) if reduction == "none" else loss
