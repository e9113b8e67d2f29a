"""Linears of routed rows: every group (an element, a fine-tuned variant, an expert) with matrices of its own.

``GroupedLinear`` (``smx_grouped_*``) takes rows in the order of a ``RowRouting``, as its ``dispatch`` leaves them and its ``combine`` takes them back. Like
the linears with adapters it works on CUDA tensors (float32 or float64) and on torch's current stream of their device, waits for nothing, can be
captured into CUDA graphs (after a first call of a kind on a GPU) and is not recorded by autograd: its backward pass is a method.
"""
from __future__ import annotations

import ctypes
from collections import namedtuple

from . import _lib
from .adapters import RowRouting, _apart, _call, _out, _precision, _ptr, _rows, _stream, _values
from .mace import SymmetrixError

GroupedGradients = namedtuple("GroupedGradients", ["x", "weights"])


class GroupedLinear:
    """A linear of all degrees with matrices for every group: ``y = x weights_l[g]`` for every component of the rows of group ``g``.

    ``weights`` is a list with a contiguous tensor ``[groups, in_l, out_l]`` per degree, ``components`` the rows per atom of every degree (default 1, 3, 5,
    ...). A row of ``x`` holds the components of degree 0, then those of degree 1, and so on, ``in_l`` channels each; ``y`` the same with ``out_l``.

    The tensors themselves are kept and read in every call: values changed in place count from the next call on."""

    def __init__(self, weights, components=None):
        import torch
        weights = list(weights)
        if not weights or len(weights) > _lib.GROUPED_MAX_DEGREES:
            raise ValueError(f"weights needs one tensor for each of 1 .. {_lib.GROUPED_MAX_DEGREES} degrees")
        first = _values(weights[0], "weights[0]", (None, None, None))
        self.dtype, self.device, self.num_groups = first.dtype, first.device, first.shape[0]
        if not 1 <= self.num_groups <= _lib.ROUTE_MAX_GROUPS:
            raise ValueError(f"weights[0] has shape {tuple(first.shape)}: 1 .. {_lib.ROUTE_MAX_GROUPS} groups are supported")
        for q, w in enumerate(weights):
            if not _values(w, f"weights[{q}]", (self.num_groups, None, None), self.dtype, self.device).is_contiguous():
                raise ValueError(f"weights[{q}] must be contiguous")
        self.weights = tuple(weights)
        self.components = [2 * l + 1 for l in range(len(weights))] if components is None else [int(c) for c in components]
        if len(self.components) != len(weights) or any(not 1 <= c <= 1024 for c in self.components):
            raise ValueError("components needs a number in 1 .. 1024 for each degree")
        self.in_channels, self.out_channels = [w.shape[1] for w in weights], [w.shape[2] for w in weights]
        if any(not 1 <= n <= 1 << 20 for n in self.in_channels + self.out_channels):
            raise ValueError("a degree needs 1 .. 1048576 channels")
        self.in_width = sum(c * i for c, i in zip(self.components, self.in_channels))
        self.out_width = sum(c * o for c, o in zip(self.components, self.out_channels))
        self._library = _lib.load()
        self._index = self.device.index
        self._home = _stream(self._index)
        self._status = torch.zeros(1, dtype=torch.int32, device=self.device)
        f = self._fixed = _lib.GroupedCall()
        f.precision, f.num_degrees, f.num_groups, f.status = _precision(self.dtype), len(weights), self.num_groups, self._status.data_ptr()
        for d, w, c in zip(f.degrees, weights, self.components):
            d.components, d.in_channels, d.out_channels = c, w.shape[1], w.shape[2]
        self._shapes = tuple(tuple(w.shape) for w in weights)

    def check(self) -> None:
        """Waits for the current stream and raises ``SymmetrixError`` if a bounded wait inside a kernel ran out in a call since the last check:
        what such a call lost holds NaN. (Calls themselves never wait, so they cannot tell.)"""
        code = int(self._status.item())
        if code:
            self._status.zero_()
            raise SymmetrixError(_lib.SMX_ERR_CUDA, f"a bounded wait ran out in a device kernel (code {code}); results are invalid")

    def _begin(self, routing):
        if not isinstance(routing, RowRouting):
            raise ValueError("routing must be a RowRouting")
        if routing.device != self.device:
            raise ValueError(f"routing is on {routing.device}, expected {self.device}")
        if routing.num_groups != self.num_groups:
            raise ValueError(f"routing has {routing.num_groups} groups, the linear {self.num_groups}")
        call = _lib.GroupedCall.from_buffer_copy(self._fixed)
        for d, w, shape in zip(call.degrees, self.weights, self._shapes):
            if w.requires_grad or w.shape != shape or w.dtype is not self.dtype or w.get_device() != self._index or not w.is_contiguous():
                if not _values(w, "weights", shape, self.dtype, self.device).is_contiguous():
                    raise ValueError("weights must be contiguous")
            d.weight = w.data_ptr()                  # (as it is now: a program may have given the tensor other memory)
        call.num_rows, call.offsets = routing._pairs, routing._offsets
        stream = _stream(self._index)
        call.stream = stream
        if stream != self._home:
            import torch
            self._status.record_stream(torch.cuda.current_stream(self._index))
        if stream != routing._home:
            routing._use()
        return call

    def forward(self, x, routing: RowRouting, out=None):
        """``y`` of ``x`` ``[rows * slots, in_width]`` in the order of ``routing``. Rows behind the last group are zero, or left as they were in ``out``."""
        call = self._begin(routing)
        n = routing._pairs
        x, call.x_stride = _rows(x, "x", (n, self.in_width), self.dtype, self.device)
        if out is None:
            y, call.y_stride, call.zero_tail = x.new_empty((n, self.out_width)), self.out_width, 1
        else:
            y, call.y_stride = _out(out, "out", (n, self.out_width), self.dtype, self.device)
            _apart(y, x, *self.weights)
        call.x, call.y = _ptr(x), _ptr(y)
        _call(self._library.smx_grouped_forward, self._index, ctypes.byref(call))
        return y

    def backward(self, x, grad_y, routing: RowRouting, want_x: bool = True, want_weights: bool = True):
        """Gradients ``(x, weights)`` of a forward pass with the same ``x``, routing and matrices, None where not wanted; rows behind the last group and
        matrices of groups without rows get zeros. ``x`` is not read (and may be None) without ``want_weights``."""
        call = self._begin(routing)
        n = routing._pairs
        grad_y, call.grad_y_stride = _rows(grad_y, "grad_y", (n, self.out_width), self.dtype, self.device)
        call.grad_y = _ptr(grad_y)
        grad_x = grad_weights = None
        if want_x:
            grad_x, call.grad_x_stride = grad_y.new_empty((n, self.in_width)), self.in_width
            call.grad_x = _ptr(grad_x)
        if want_weights:
            x, call.x_stride = _rows(x, "x", (n, self.in_width), self.dtype, self.device)
            call.x = _ptr(x)
            # one allocation for all degrees, each on a multiple of 16 bytes
            g, at, grad_weights = self.num_groups, 0, []
            sizes = [g * i * o for i, o in zip(self.in_channels, self.out_channels)]
            flat = grad_y.new_empty(sum(-(-s // 4) * 4 for s in sizes))
            base, size = flat.data_ptr(), flat.element_size()
            for d, s, i, o in zip(call.degrees, sizes, self.in_channels, self.out_channels):
                d.grad_weight = base + size * at
                grad_weights.append(flat.as_strided((g, i, o), (i * o, o, 1), at))
                at += -(-s // 4) * 4
            need = self._library.smx_grouped_workspace_bytes(ctypes.byref(call), 1)
            if need < 0:
                raise ValueError("the sizes exceed what smx_grouped_backward supports")
            if need:
                ws = grad_y.new_empty(-(-need // size))
                call.workspace, call.workspace_bytes = ws.data_ptr(), need
        _call(self._library.smx_grouped_backward, self._index, ctypes.byref(call))
        return GroupedGradients(grad_x, grad_weights)
