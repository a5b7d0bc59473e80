"""Softmax cross entropy of a linear scorer over many classes on the HIP target, and its gradients.

Not in the reference, which stops at the features of the last layer.  Vertex classification scores every vertex
against the class weights; link prediction scores a batch of queries against the embeddings of all vertices.  With N
rows and V classes the logits are an N x V matrix that is far larger than the operands; the loss never stores it:

    l[n, v] = <Hidden[n], Weight[v]>        lse[n] = log(sum_v exp l[n, v])        Loss[n] = lse[n] - l[n, Label[n]]
    G[n, v] = dLoss[n] * (exp(l[n, v] - lse[n]) - [v = Label[n]])     dHidden = G Weight     dWeight = G^T Hidden

A label outside [0, V) (such as -1) marks a row to ignore: its loss is zero, its row of dHidden is zero and it adds
nothing to dWeight.  Operands are float32 or bfloat16, losses and statistics float32.

The gradient keeps G for a piece of the vocabulary (all of it where that and the copies of the operands fit 4 GiB) in the
module's workspace: 2 bytes per row and class for bfloat16, 4 for float32.  bfloat16 rounds G to bfloat16.  float32 keeps
G / dLoss to 2^-23 of itself and 2^-50, and elements of Weight and of dLoss * Hidden to 2^-23 of themselves and 2^-50 of
the matrix's largest: probabilities or features less than 2^-27 of the largest lose relative accuracy.
"""
import torch

from .. import _lib
from ..runtime import NDArray
from . import _common as C

_TYPES = {k: C.ELEMENT_TYPES[k] for k in ("float32", "bfloat16")}


class _LinearCrossEntropyBase(C.DenseBase):
    def _parse(self, input_placeholders, compute_args, schedule_args):
        C.check_known_keys(compute_args, (), "compute_args")
        C.check_known_keys(schedule_args, (), "schedule_args")
        if len(input_placeholders) != 3:
            raise ValueError("expected placeholders for Hidden, Weight and Label")
        hidden, weight, label = input_placeholders
        self._element = C.typed(hidden.dtype, _TYPES, "Hidden")
        if C.typed(weight.dtype, _TYPES, "Weight") != self._element:
            raise TypeError("Hidden and Weight must have one type, got %s and %s" % (hidden.dtype, weight.dtype))
        self._index = C.typed(label.dtype, C.INDEX_TYPES, "Label")
        hs, ws, ls = (tuple(int(s) for s in p.shape) for p in input_placeholders)
        if len(hs) != 2 or len(ws) != 2 or hs[1] != ws[1] or hs[1] < 1 or ws[0] < 1:
            raise ValueError("Hidden and Weight must have shapes (N, D) and (V, D), got %s and %s" % (hs, ws))
        if ls != hs[:1]:
            raise ValueError("Label must have shape %s, got %s" % (hs[:1], ls))
        if hs[0] > 1 << 22 or hs[1] > 1 << 16 or ws[0] >= 0x7fff0000:
            raise ValueError("Hidden %s and Weight %s are beyond what the kernels index" % (hs, ws))
        self._hidden_shape, self._weight_shape, self._label_shape = hs, ws, ls
        self._sizes = (hs[0], ws[0], hs[1])

    def _checked_operands(self, hidden, weight, label):
        return (C.check_typed_operand(hidden, self._hidden_shape, self._element[0], self._ctx, "Hidden"),
                C.check_typed_operand(weight, self._weight_shape, self._element[0], self._ctx, "Weight"),
                C.check_typed_operand(label, self._label_shape, self._index[0], self._ctx, "Label"))


class LinearCrossEntropyhip(_LinearCrossEntropyBase):
    """build([Hidden (N, D), Weight (V, D), Label (N,) of int32 or int64]); run([hidden, weight, label]) returns the
    module-owned float32 arrays (loss (N,), lse (N,)); lse is what the gradient's run takes."""

    def build(self, input_placeholders, compute_args=None, schedule_args=None):
        self._parse(input_placeholders, compute_args, schedule_args)
        self._space = self._workspace("fg_linear_ce_workspace", *self._sizes, self._element[1])
        self._loss, self._lse = (NDArray(torch.empty(self._label_shape, dtype=torch.float32, device=self._ctx)) for _ in range(2))
        self.out_tvm = self._loss
        self._built = True

    def _checked(self, arrays):
        if len(arrays) != 3:
            raise ValueError("expected 3 input arrays (Hidden, Weight, Label)")
        operands = self._checked_operands(*arrays)
        for out in (self._loss, self._lse):
            C.check_apart(out.tensor, operands, "the module's output")
        return operands

    def _launch(self, tensors):
        hidden, weight, label = tensors
        _lib.check(_lib.lib().fg_linear_ce(
            *self._sizes, hidden.data_ptr(), weight.data_ptr(), label.data_ptr(), self._loss.tensor.data_ptr(),
            self._lse.tensor.data_ptr(), self._element[1], self._index[1], self._space.data_ptr(),
            self._space.numel(), self._stream()))
        return self._loss, self._lse


class LinearCrossEntropyGradhip(_LinearCrossEntropyBase):
    """build() as for the loss; run([hidden, weight, label, lse, dloss]) with the forward pass's lse (N,) and the
    gradient dloss (N,) of the losses (1 / N each for their mean) returns the module-owned (dHidden, dWeight), of the
    operands' type.  The logits are computed again, a piece of the vocabulary at a time."""

    def build(self, input_placeholders, compute_args=None, schedule_args=None):
        self._parse(input_placeholders, compute_args, schedule_args)
        self._space = self._workspace("fg_linear_ce_grad_workspace", *self._sizes, self._element[1])
        self._dhidden = NDArray(torch.empty(self._hidden_shape, dtype=self._element[0], device=self._ctx))
        self._dweight = NDArray(torch.empty(self._weight_shape, dtype=self._element[0], device=self._ctx))
        self.out_tvm = self._dhidden
        self._built = True

    def _checked(self, arrays):
        if len(arrays) != 5:
            raise ValueError("expected 5 input arrays (Hidden, Weight, Label, LogSumExp, LossGrad)")
        operands = self._checked_operands(*arrays[:3]) + tuple(
            C.check_typed_operand(x, self._label_shape, torch.float32, self._ctx, what)
            for x, what in zip(arrays[3:], ("LogSumExp", "LossGrad")))
        for out in (self._dhidden, self._dweight):
            C.check_apart(out.tensor, operands, "the module's output")
        return operands

    def _launch(self, tensors):
        hidden, weight, label, lse, dloss = tensors
        _lib.check(_lib.lib().fg_linear_ce_grad(
            *self._sizes, hidden.data_ptr(), weight.data_ptr(), label.data_ptr(), lse.data_ptr(), dloss.data_ptr(),
            self._dhidden.tensor.data_ptr(), self._dweight.tensor.data_ptr(), self._element[1], self._index[1],
            self._space.data_ptr(), self._space.numel(), self._stream()))
        return self._dhidden, self._dweight
