"""The `torch.library` seam SURVEY 8b sketched (`TORCH_LIBRARY(yolov6_hip, m)`), for the STATELESS operators of the hot path.

    import yolov6_amd.torch_ops                      # registers the namespace
    dets, index, count = torch.ops.yolov6_hip.nms_batched(pred, 0.03, 0.65, None, False, True, 300)
    labels, boxes, scores, fg = torch.ops.yolov6_hip.tal_assign(pd_scores, pd_bboxes, anc_points, gt_labels, gt_bboxes, mask_gt,
                                                                 13, 1.0, 6.0, 1e-9)
    y = torch.ops.yolov6_hip.conv2d_bias_act(x_nchw, weight, bias, "relu", 1)
    loss, _ = torch.ops.yolov6_hip.linear_cross_entropy(features, weight, target, bias, -100, 0.0, "mean")      # differentiable

Each op is a dispatcher-visible custom op (schema, CUDA-only implementation, fake / meta kernel for shape inference), so
`torch.compile` traces THROUGH callers of them (they stay opaque calls into libyolov6_hip.so), `torch.ops.yolov6_hip.*` works from
TorchScript-free C++ / Python callers alike, and errors surface as `RuntimeError` - what the reference's assigner fallback catches
(yolov6/models/losses/loss.py:105).  The implementations are the SAME ctypes bindings the module mirrors use (utils/nms.py,
assigners/*.py, engine.PlanBuilder): one code path, two doors.  What is NOT here: the whole-model plans (`Model.forward`) and the
training graph - they own buffers, packed weights and streams, which is state a functional op cannot carry; they stay behind
`HipModule`.

Replaces / mirrors: `non_max_suppression` (yolov6/utils/nms.py:31-105), `TaskAlignedAssigner.forward` (assigners/tal_assigner.py:22-106),
`ATSSAssigner.forward` (assigners/atss_assigner.py:22-93), `ConvModule.forward_fuse` / the RepVGG deploy conv (layers/common.py:51-54,
:247-248)."""
from typing import List, Optional, Tuple

import torch
from torch import Tensor

NAMESPACE = "yolov6_hip"
__all__ = ["nms_batched", "tal_assign", "atss_assign", "conv2d_bias_act", "linear_cross_entropy"]


@torch.library.custom_op(f"{NAMESPACE}::nms_batched", mutates_args=(), device_types="cuda")
def nms_batched(pred: Tensor, conf_thres: float, iou_thres: float, classes: Optional[List[int]], agnostic: bool, multi_label: bool,
                max_det: int) -> Tuple[Tensor, Tensor, Tensor]:
    """(dets [B, max_det, 6] f32 xyxy/conf/cls, index [B, max_det] i32 = anchor * nc + cls, count [B] i32): the device-side result
    of `non_max_suppression`; rows past `count[b]` are 0 / -1."""
    from .utils.nms import nms_raw
    return nms_raw(pred, conf_thres, iou_thres, classes, agnostic, multi_label, max_det)


@nms_batched.register_fake
def _(pred, conf_thres, iou_thres, classes, agnostic, multi_label, max_det):
    B = pred.shape[0]
    return (pred.new_empty((B, max_det, 6), dtype=torch.float32), pred.new_empty((B, max_det), dtype=torch.int32),
            pred.new_empty((B,), dtype=torch.int32))


def _assign_fake(ref: Tensor, B: int, A: int, C: int):
    return (ref.new_empty((B, A), dtype=torch.int64), ref.new_empty((B, A, 4), dtype=torch.float32),
            ref.new_empty((B, A, C), dtype=torch.float32), ref.new_empty((B, A), dtype=torch.bool))


@torch.library.custom_op(f"{NAMESPACE}::tal_assign", mutates_args=(), device_types="cuda")
def tal_assign(pd_scores: Tensor, pd_bboxes: Tensor, anc_points: Tensor, gt_labels: Tensor, gt_bboxes: Tensor, mask_gt: Tensor,
               topk: int, alpha: float, beta: float, eps: float) -> Tuple[Tensor, Tensor, Tensor, Tensor]:
    """(target_labels [B, A] i64, target_bboxes [B, A, 4] f32, target_scores [B, A, C] f32, fg_mask [B, A] bool)."""
    from .assigners import TaskAlignedAssigner
    G = gt_bboxes.shape[1]
    out = TaskAlignedAssigner(topk=topk, num_classes=pd_scores.shape[-1], alpha=alpha, beta=beta, eps=eps)(
        pd_scores, pd_bboxes, anc_points, gt_labels, gt_bboxes, mask_gt)
    lab, box, sc, fg = out
    if G == 0:        # (the module mirrors the reference's float early-out; the op's schema is fixed)
        lab, fg = lab.long(), fg.bool()
    return lab, box.float(), sc.float(), fg


@tal_assign.register_fake
def _(pd_scores, pd_bboxes, anc_points, gt_labels, gt_bboxes, mask_gt, topk, alpha, beta, eps):
    B, A, C = pd_scores.shape
    return _assign_fake(pd_scores, B, A, C)


@torch.library.custom_op(f"{NAMESPACE}::atss_assign", mutates_args=(), device_types="cuda")
def atss_assign(anc_bboxes: Tensor, n_level_bboxes: List[int], gt_labels: Tensor, gt_bboxes: Tensor, mask_gt: Tensor,
                pd_bboxes: Optional[Tensor], topk: int, num_classes: int) -> Tuple[Tensor, Tensor, Tensor, Tensor]:
    from .assigners import ATSSAssigner
    lab, box, sc, fg = ATSSAssigner(topk=topk, num_classes=num_classes)(anc_bboxes, n_level_bboxes, gt_labels, gt_bboxes, mask_gt, pd_bboxes)
    return lab.long(), box.float(), sc.float(), fg.bool()


@atss_assign.register_fake
def _(anc_bboxes, n_level_bboxes, gt_labels, gt_bboxes, mask_gt, pd_bboxes, topk, num_classes):
    return _assign_fake(anc_bboxes, gt_bboxes.shape[0], anc_bboxes.shape[0], num_classes)


@torch.library.custom_op(f"{NAMESPACE}::conv2d_bias_act", mutates_args=(), device_types="cuda")
def conv2d_bias_act(x: Tensor, weight: Tensor, bias: Optional[Tensor], act: str, stride: int) -> Tensor:
    """conv (k in {1, 3}, pad k//2, stride 1 / 2) + bias + activation ("relu" | "silu" | "hardswish" | "none") of an NCHW fp16
    tensor as one fused HIP launch; NCHW fp16 out.  A functional op packs the weights on every call: the module mirrors (which cache
    a plan) are the fast path - this door is for callers that want the single operator."""
    from .engine import NCHWInput, PlanBuilder
    if act not in ("relu", "silu", "hardswish", "none"):
        raise RuntimeError(f"yolov6_hip::conv2d_bias_act: unknown activation {act!r}")
    pb = PlanBuilder(x.device)
    y = pb.conv(NCHWInput(x.contiguous()), weight, bias, stride=stride, act=None if act == "none" else act)
    out = pb.to_nchw(y, x.dtype if x.dtype in (torch.float16, torch.float32) else torch.float16)
    plan = pb.finalize(out, autotune=False)
    return plan.run().clone()


@conv2d_bias_act.register_fake
def _(x, weight, bias, act, stride):
    B, _, H, W = x.shape
    k = weight.shape[-1]
    Ho, Wo = (H + 2 * (k // 2) - k) // stride + 1, (W + 2 * (k // 2) - k) // stride + 1
    return x.new_empty((B, weight.shape[0], Ho, Wo))


@torch.library.custom_op(f"{NAMESPACE}::linear_cross_entropy", mutates_args=(), device_types="cuda")
def linear_cross_entropy(features: Tensor, weight: Tensor, target: Tensor, bias: Optional[Tensor], ignore_index: int, label_smoothing: float,
                         reduction: str, recompute: bool = False) -> Tuple[Tensor, Tensor]:
    """(loss, bytes that the backward takes over): models/losses/loss_ce.py with a schema.  They are made whether a backward follows or not, up to
    2 GiB of them unless `recompute`: a caller that wants the value alone calls models/losses/loss_ce.py without gradients.  Under autocast the operands are cast first."""
    from . import _lib
    return _lib.torch_host().linear_cross_entropy_forward(features, weight, target, bias, ignore_index, label_smoothing, reduction, recompute)


@linear_cross_entropy.register_fake
def _(features, weight, target, bias, ignore_index, label_smoothing, reduction, recompute=False):
    return (features.new_empty(target.shape if reduction == "none" else (), dtype=torch.float32),
            features.new_empty((torch.library.get_ctx().new_dynamic_size(),), dtype=torch.uint8))


@torch.library.custom_op(f"{NAMESPACE}::linear_cross_entropy_backward", mutates_args=(), device_types="cuda")
def linear_cross_entropy_backward(grad: Tensor, features: Tensor, weight: Tensor, target: Tensor, bias: Optional[Tensor], saved: Tensor,
                                  ignore_index: int, label_smoothing: float, reduction: str,
                                  recompute: bool) -> Tuple[Tensor, Tensor, Tensor]:
    from . import _lib
    return _lib.torch_host().linear_cross_entropy_backward(grad, features, weight, target, bias, saved, ignore_index, label_smoothing, reduction,
                                                             recompute)


@linear_cross_entropy_backward.register_fake
def _(grad, features, weight, target, bias, saved, ignore_index, label_smoothing, reduction, recompute):
    return (features.new_empty(features.shape), weight.new_empty(weight.shape), weight.new_empty((0,) if bias is None else (weight.shape[0],)))


def _ce_capture(features, weight, bias):
    """What models/losses/loss_ce.py refuses under stream capture, for a call that a backward may follow."""
    if torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing():
        from . import _lib
        _lib.torch_host().linear_cross_entropy_refuse_outer_graph(features, weight, bias)


def _ce_setup(ctx, inputs, output):
    features, weight, target, bias, *ctx.options = inputs
    _ce_capture(features, weight, bias)
    ctx.mark_non_differentiable(output[1])
    ctx.save_for_backward(features, weight, target, bias, output[1])


def _ce_grad(ctx, grad, _):
    features, weight, target, bias, saved = ctx.saved_tensors
    dx, dw, db = torch.ops.yolov6_hip.linear_cross_entropy_backward(grad, features, weight, target, bias, saved, *ctx.options)
    return dx, dw, None, None if bias is None else db, None, None, None, None


linear_cross_entropy.register_autograd(_ce_grad, setup_context=_ce_setup)


def _ce_autocast(features, weight, target, bias, *options):
    """The casts come before the op, so that they are differentiated and its backward sees the operands of its forward, wherever it runs."""
    if torch.is_grad_enabled():
        _ce_capture(features, weight, bias)                  # (what is cast is a leaf no longer)
    dtype = torch.get_autocast_dtype("cuda")
    with torch._C._ExcludeDispatchKeyGuard(torch._C.DispatchKeySet(torch._C.DispatchKey.AutocastCUDA)):
        return torch.ops.yolov6_hip.linear_cross_entropy(features.to(dtype), weight.to(dtype), target, None if bias is None else bias.to(dtype), *options)


_fragment = torch.library.Library(NAMESPACE, "FRAGMENT")      # (the kernel is there as long as this object)
_fragment.impl("linear_cross_entropy", _ce_autocast, "AutocastCUDA")
