"""Softmax cross entropy of a linear classifier over many classes: value and gradients in tiles, without the logits.

    loss = linear_cross_entropy(features, weight, target, bias)     # = F.cross_entropy(F.linear(features, weight, bias), target)
    loss.backward()

For classifiers whose [rows, classes] logits are what fills the memory and the time of a step: a head over a large label set, dense labels
with a large vocabulary.  The detection losses (loss.py) keep their sigmoid scores.  The reference has no
softmax classifier; the semantics are torch's, except that the mean over no labelled row is 0 (as ComputeLoss's terms are without
targets), not a NaN.  Kernels: csrc/linear_ce.hip (y6_linear_ce_forward / _backward); the
autograd node and the operands' checks: csrc/torch_host.cpp.

Memory of a training call beside its operands and gradients, `size` the bytes of an element.
  From the forward to the end of the graph (y6_linear_ce_saved_bytes):
    the labelled rows gathered, rows x width x size (fp32: x 6 bytes);
    a copy of the weight where its rows do not start at 16-byte borders (fp32: always, classes x width x 6 bytes);
    in calls large enough that the backward gains by it, exponentials of rows x classes x size, up to 2 GiB for each loss that is alive: what
    the logits of the operands' type would take (and a few percent for their scales).  `recompute=True` keeps none of them, and the backward forms the scores again.
  During the backward: one piece of the logits' gradient, rows x piece x 2 bytes (fp32: x 6), pieces cut for 128 to 256 MB but not below 256 classes, so
    more from 2^19 rows on (fp32: from 170 thousand); in several pieces or splits the features' gradient in fp32, rows x width x 4 x splits; splits of a
    piece of the weight's gradient likewise.
  During the forward: the tiles' statistics, at most 256 MB, half as much again with label smoothing.
"""
from ... import _lib


def linear_cross_entropy(features, weight, target, bias=None, *, ignore_index=-100, label_smoothing=0.0, reduction="mean", recompute=False):
    """F.cross_entropy(F.linear(features, weight, bias), target, ...) without the logits.

    features [..., width], weight [classes, width], bias [classes] or None, in one type (fp16, bf16, fp32; under autocast they are cast
    to its type); target [...] int64.  Returns fp32: a scalar ('mean' over the labelled rows, 'sum'), or [...] ('none').  Gradients
    come in the operands' type, once differentiable, in reverse mode (dual tensors are refused); under a loss scale (LossScaler) as usual.
    Rows labelled ignore_index have loss 0, a zero gradient, and are not read: a NaN in them goes nowhere.  A label that is neither a class
    nor ignore_index makes its row's loss and the gradients NaN (no host check: nothing synchronises).  With 'none', an upstream gradient
    that is not finite reaches its own row of the features' gradient and the gradients of weight and bias, as in torch.

    Products of 16-bit operands accumulate in fp32; the gradient of the logits is rounded to the operands' type where the matrix instructions
    of the two gradient products take it.  recompute=False: large calls keep exponentials for the backward (memory: above), which round the
    probabilities of the classes that are not the label once more before that; recompute=True keeps none and takes 1.1 to 1.2 times
    as long (4096 x 1024 x 32000 in bf16: 1148 us, 968 with them).  Under stream capture no eager graph over the operands that was made on the default stream may be alive (an error).
    Works on any view with a dense last dimension; others are copied."""
    return _lib.torch_host().linear_cross_entropy(features, weight, target, bias, ignore_index, label_smoothing, reduction, bool(recompute))
