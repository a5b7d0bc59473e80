"""Lookup of learned vertex embeddings on the HIP target, and its gradient.

Not in the reference, whose features are inputs.  A graph model without input features learns one row per vertex
(or entity): a mini-batch looks the rows of its sampled vertices up, and the backward pass adds the gradients of
equal ids into the table's gradient.

Ids outside [0, V) are padding: they look up zeros and add nothing to the gradient, so -1 pads ragged batches.
Elements are float32, bfloat16 or float16; sums are held in float32 and rounded once.  Like every module here a
module owns its output (and workspace), which the next run overwrites.
"""
import torch

from .. import _lib
from ..runtime import NDArray
from . import _common as C


def _parse(input_placeholders):
    if len(input_placeholders) != 2:
        raise ValueError("expected placeholders for Table and Ids")
    table, ids = input_placeholders
    element = C.typed(table.dtype, C.ELEMENT_TYPES, "Table")
    index = C.typed(ids.dtype, C.INDEX_TYPES, "Ids")
    shape = tuple(int(s) for s in table.shape)
    if len(shape) != 2 or min(shape) < 1:
        raise ValueError("Table must have shape (num_rows, row_len), got %s" % (shape,))
    if shape[0] >= C.INT32_MAX or shape[1] > 1 << 20:
        raise ValueError("Table of shape %s is beyond what the kernels index" % (shape,))
    ids_shape = tuple(int(s) for s in ids.shape)
    n = 1
    for s in ids_shape:
        n *= s
    if n < 0 or n > 0x7fff0000:
        raise ValueError("Ids of shape %s are beyond what the kernels index" % (ids_shape,))
    return element, index, shape, ids_shape, n


class EmbeddingLookuphip(C.DenseBase):
    """Out[i, :] = scale * Table[Ids[i], :].

    EmbeddingLookuphip(scale).build([placeholder((V, D), dtype), placeholder(ids_shape, "int32" or "int64")]);
    run([table, ids]) returns the module-owned array of shape ids_shape + (D,).
    """

    def __init__(self, scale=1.0):
        super().__init__()
        self._scale = float(scale)

    def build(self, input_placeholders, compute_args=None, schedule_args=None):
        C.check_known_keys(compute_args, (), "compute_args")
        C.check_known_keys(schedule_args, (), "schedule_args")
        self._element, self._index, self._shape, self._ids_shape, self._n = _parse(input_placeholders)
        self.out_tvm = NDArray(torch.empty(self._ids_shape + self._shape[1:], dtype=self._element[0], device=self._ctx))
        self._built = True

    def _checked(self, arrays):
        if len(arrays) != 2:
            raise ValueError("expected 2 input arrays (Table, Ids)")
        table = C.check_typed_operand(arrays[0], self._shape, self._element[0], self._ctx, "Table")
        ids = C.check_typed_operand(arrays[1], self._ids_shape, self._index[0], self._ctx, "Ids")
        C.check_apart(self.out_tvm.tensor, (table, ids), "the module's output")
        return table, ids

    def _launch(self, tensors):
        table, ids = tensors
        _lib.check(_lib.lib().fg_embedding_lookup(
            self._shape[0], self._shape[1], self._n, table.data_ptr(), ids.data_ptr(), self.out_tvm.tensor.data_ptr(),
            self._scale, self._element[1], self._index[1], self._stream()))
        return self.out_tvm


class EmbeddingLookupGradhip(C.DenseBase):
    """Gradient of EmbeddingLookuphip for the table: dTable[v, :] = scale * sum over i with Ids[i] = v of dOut[i, :].

    build() as for the lookup.  run([ids, dout]) returns the module-owned dTable (V, D), every row of it written;
    run([ids, dout, grad]) adds to the caller's grad (V, D) instead, touching the looked-up rows only, and returns
    it: for gradients accumulated over several batches, and for a table that has another gradient already.
    The ids are sorted on the device in every run and equal ids are added in the order of the batch, so results do
    not depend on timing.
    """

    def __init__(self, scale=1.0):
        super().__init__()
        self._scale = float(scale)

    def build(self, input_placeholders, compute_args=None, schedule_args=None):
        C.check_known_keys(compute_args, (), "compute_args")
        C.check_known_keys(schedule_args, (), "schedule_args")
        self._element, self._index, self._shape, self._ids_shape, self._n = _parse(input_placeholders)
        self._space = self._workspace("fg_embedding_grad_workspace", self._shape[0], self._shape[1], self._n)
        self.out_tvm = None      # made by the first run that needs it: accumulating runs do not
        self._built = True

    def _own(self):
        if self.out_tvm is None:
            self.out_tvm = NDArray(torch.empty(self._shape, dtype=self._element[0], device=self._ctx))
        return self.out_tvm

    def _checked(self, arrays):
        if len(arrays) not in (2, 3):
            raise ValueError("expected 2 or 3 input arrays (Ids, OutGrad and optionally TableGrad)")
        ids = C.check_typed_operand(arrays[0], self._ids_shape, self._index[0], self._ctx, "Ids")
        dout = C.check_typed_operand(arrays[1], self._ids_shape + self._shape[1:], self._element[0], self._ctx, "OutGrad")
        if len(arrays) == 2:
            grad = self._own()
        else:
            C.check_typed_operand(arrays[2], self._shape, self._element[0], self._ctx, "TableGrad")
            grad = arrays[2] if isinstance(arrays[2], NDArray) else NDArray(arrays[2])
        C.check_apart(grad.tensor, (ids, dout), "the table's gradient")
        return ids, dout, grad, len(arrays) == 3

    def _launch(self, tensors):
        ids, dout, grad, accumulate = tensors
        _lib.check(_lib.lib().fg_embedding_grad(
            self._shape[0], self._shape[1], self._n, ids.data_ptr(), dout.data_ptr(), grad.tensor.data_ptr(),
            self._scale, int(accumulate), self._element[1], self._index[1], self._space.data_ptr(),
            self._space.numel(), self._stream()))
        return grad
