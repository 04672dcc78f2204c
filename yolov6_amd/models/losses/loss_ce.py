"""Softmax cross entropy of a linear classifier over many classes: value and gradients without the logits in memory.

    loss = linear_cross_entropy(features, weight, target, bias)     # = F.cross_entropy(F.linear(features, weight, bias), target)
    loss.backward()

For classifiers whose [rows, classes] logits are what fills the memory and the time of a step: pretraining the backbone on a large
label set, dense labels with a large vocabulary.  The detection losses (loss.py) keep their sigmoid scores.  The reference has no
softmax classifier; the semantics are torch's, except that the mean over no labelled row is 0 (as ComputeLoss's terms are without
targets), not a NaN.  Kernels: csrc/linear_ce.hip (y6_linear_ce_forward / _backward); the
autograd node and the operands' checks: csrc/torch_host.cpp.

Memory of a training call beside its operands and gradients: the labelled rows gathered, at most 2 GiB of exponentials in the operands'
type (they live from the forward to the end of the graph), and at most 256 MB of dz during the backward.
"""
from ... import _lib


def linear_cross_entropy(features, weight, target, bias=None, *, ignore_index=-100, label_smoothing=0.0, reduction="mean"):
    """F.cross_entropy(F.linear(features, weight, bias), target, ...) without the logits.

    features [..., width], weight [classes, width], bias [classes] or None, in one type (fp16, bf16, fp32; under autocast they are cast
    to its type); target [...] int64.  Returns fp32: a scalar ('mean' over the labelled rows, 'sum'), or [...] ('none').  Gradients
    come in the operands' type, once differentiable, in reverse mode (dual tensors are refused); under a loss scale (LossScaler) as usual.  Rows labelled ignore_index have loss
    0, a zero gradient, and are not read: a NaN in them goes nowhere.  A label that is neither a class nor ignore_index makes its
    row's loss and the gradients NaN (no host check: nothing synchronises).  With 'none', an upstream gradient that is not
    finite reaches its own row of the features' gradient and the gradients of weight and bias, as in torch.  Products of 16-bit operands accumulate in fp32; the
    gradient of the logits is rounded to the operands' type where the matrix instructions of the two gradient products take it (in
    large calls the probabilities of the other classes once before that, when they are kept for the backward).  Under stream capture no
    eager graph over the operands that was made on the default stream may be alive (an error).  Works on any view with a dense last dimension; others are copied."""
    return _lib.torch_host().linear_cross_entropy(features, weight, target, bias, ignore_index, label_smoothing, reduction)
