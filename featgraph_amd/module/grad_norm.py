"""Global norm of many gradients on the HIP target, and clipping by it.

Not in the reference, which has no training step.  norm = sqrt(sum of the squares of all elements of all tensors),
added in float64; clipping multiplies every element by min(1, max_norm / (norm + eps)).  The tensors may differ in
shape and in type (float32, bfloat16, float16).
"""
import bisect
import ctypes
import math

import numpy as np
import torch

from .. import _lib
from ..runtime import NDArray, as_tensor
from . import _common as C


class GradNormhip(C.DenseBase):
    """build([placeholder of every tensor]); run([tensors]) returns the module-owned float32 norm, of shape ()."""

    def build(self, input_placeholders, compute_args=None, schedule_args=None):
        self._parse(input_placeholders, compute_args, schedule_args)
        self._allocate()
        self._built = True

    def _parse(self, input_placeholders, compute_args, schedule_args, keys=()):
        args = C.check_known_keys(compute_args, keys, "compute_args")
        C.check_known_keys(schedule_args, (), "schedule_args")
        if len(input_placeholders) > 1 << 17:
            raise ValueError("at most %d tensors per call, got %d" % (1 << 17, len(input_placeholders)))
        types = [C.typed(p.dtype, C.ELEMENT_TYPES, "gradients") for p in input_placeholders]
        self._shapes = [torch.Size(int(s) for s in p.shape) for p in input_placeholders]
        self._expected = [(shape, t[0], shape.numel() * t[0].itemsize) for shape, t in zip(self._shapes, types)]
        self._list = (_lib.Tensor * max(1, len(types)))()
        for entry, shape, t in zip(self._list, self._shapes, types):
            entry.n, entry.dtype = shape.numel(), t[1]
        # the list's address columns (data, out) as an array, so that a call sets all of them at once
        words = np.frombuffer(self._list, dtype=np.uint64).reshape(-1, ctypes.sizeof(_lib.Tensor) // 8)
        self._data, self._out = words[:len(types), 0], words[:len(types), 1]
        return args

    def _allocate(self):
        self._space = self._workspace("fg_grad_norm_workspace")
        self._norm = NDArray(torch.empty((), dtype=torch.float32, device=self._ctx))
        self.out_tvm = self._norm

    def _checked(self, arrays):
        """(tensors, their addresses) of the operands."""
        if len(arrays) != len(self._expected):
            raise ValueError("expected %d input arrays, got %d" % (len(self._expected), len(arrays)))
        ctx, tensors, at = self._ctx, [], []
        for x, (shape, dtype, _) in zip(arrays, self._expected):
            t = x if isinstance(x, torch.Tensor) else as_tensor(x)
            if t.shape != shape or t.dtype != dtype or t.device != ctx or not t.is_contiguous():
                C.check_typed_operand(t, shape, dtype, ctx, "gradient %d" % len(tensors))
            tensors.append(t)
            at.append(t.data_ptr())
        return tensors, at

    def _launch(self, operands):
        tensors, at = operands
        self._data[:] = at
        _lib.check(_lib.lib().fg_grad_norm(len(tensors), self._list, self._norm.tensor.data_ptr(),
                                           self._space.data_ptr(), self._space.numel(), self._stream()))
        return self._norm


class ClipGradNormhip(GradNormhip):
    """Out_t = min(1, max_norm / (norm + eps)) * Grad_t for every tensor t.

    ClipGradNormhip(max_norm).build([placeholder of every tensor]); run([tensors]) returns (norm, [clipped arrays]),
    module-owned.  build(..., {"in_place": True}) overwrites the tensors of the call instead and returns them; they
    must not overlap, and where the norm is below max_norm they are left as they are without being written.
    """

    def __init__(self, max_norm, eps=1e-6):
        super().__init__()
        self._max_norm, self._eps = float(max_norm), float(eps)
        if not (self._max_norm >= 0 and self._eps >= 0 and math.isfinite(self._eps)):
            raise ValueError("max_norm and eps must not be negative, got %r and %r" % (max_norm, eps))

    def build(self, input_placeholders, compute_args=None, schedule_args=None):
        args = self._parse(input_placeholders, compute_args, schedule_args, ("in_place",))
        self._in_place = bool(args.get("in_place", False))
        self._allocate()
        self._clipped = None
        if not self._in_place:
            self._clipped = [NDArray(torch.empty(shape, dtype=t, device=self._ctx)) for shape, t, _ in self._expected]
            self._out[:] = [c.tensor.data_ptr() for c in self._clipped]
            spans = sorted([(c.tensor.data_ptr(), size) for c, (_, _, size) in zip(self._clipped, self._expected) if size] +
                           [(self._norm.tensor.data_ptr(), 4)])
            self._out_begin, self._out_end = [b for b, _ in spans], [b + n for b, n in spans]
        self._built = True

    def _checked(self, arrays):
        tensors, at = super()._checked(arrays)
        if self._in_place:
            end = 0
            for begin, size in sorted([(b, size) for b, (_, _, size) in zip(at, self._expected) if size] +
                                      [(self._norm.tensor.data_ptr(), 4)]):
                if begin < end:
                    raise ValueError("the gradients overlap each other or the module's norm")
                end = begin + size
        else:
            begins, ends = self._out_begin, self._out_end
            for begin, (_, _, size) in zip(at, self._expected):
                i = bisect.bisect_left(begins, begin + size) - 1
                if size and i >= 0 and ends[i] > begin:      # the outputs are disjoint: the last one that starts below
                    raise ValueError("a gradient overlaps the module's outputs")
        return tensors, at

    def _launch(self, operands):
        tensors, at = operands
        self._data[:] = at
        if self._in_place:
            self._out[:] = at
        _lib.check(_lib.lib().fg_grad_clip(len(tensors), self._list, self._max_norm, self._eps,
                                           self._norm.tensor.data_ptr(), self._space.data_ptr(), self._space.numel(),
                                           self._stream()))
        return self._norm, (self._clipped if not self._in_place else [NDArray(t) for t in tensors])
